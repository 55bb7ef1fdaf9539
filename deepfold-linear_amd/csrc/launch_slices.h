// A launch of more threads than a grid's x dimension may have, in several.  Plain C++ (tests/test_launch_slices.py builds it
// with g++).
#pragma once

namespace dfl {

// Workgroups of `threads` that one launch may have side by side: grid times workgroup stays below 2^32.
constexpr long long launch_most(int threads) { return ((1ll << 32) - 1) / threads; }

// launch(first, count) for workgroups first .. first + count - 1 of `blocks`; ends at the first that does not return 0.
template <class F> auto launch_slices(long long blocks, int threads, F launch) -> decltype(launch(0ll, 0ll)) {
  const long long most = launch_most(threads);
  decltype(launch(0ll, 0ll)) e{};
  for (long long first = 0; first < blocks; first += most) {
    e = launch(first, blocks - first < most ? blocks - first : most);
    if (e) break;
  }
  return e;
}

}  // namespace dfl
