// The numbers of a scan's launches for the tests, as the kernels make them (tests/test_scan_launches.py builds and loads this).
#include "../deepnet_amd/csrc/scan_launch.h"

extern "C" {
unsigned tag(unsigned long long launch) { return scan_tag(launch); }
unsigned long long next(unsigned long long launch) { return scan_next(launch); }
// The launch that `n` others have gone before.
unsigned long long after(unsigned long long launch, unsigned long long n) {
  for (unsigned long long k = 0; k < n; ++k) launch = scan_next(launch);
  return launch;
}
}
