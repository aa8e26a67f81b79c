// The numbers of a scan's launches (scan.hip), by which a link is known as this launch's.
#pragma once

// A launch is counted from 0 to 2^32 - 2 and again, so that its number is never 0, which is what words hold that nobody has written, and comes
// back after all the others.
constexpr unsigned scan_tag(unsigned long long launch) { return (unsigned)launch + 1u; }
// The launch after one.
constexpr unsigned long long scan_next(unsigned long long launch) { return launch < 0xfffffffeull ? launch + 1 : 0; }
