// Which bins of the sampler's histogram can hold the token at which the mass reaches
// top-p of all of it, from bounds of each bin's mass.  Plain arithmetic without CUDA
// types, so that a host program can run a CTA's threads one after another.
//
// The bounds are integers, 2^30 times a mass, rounded outwards bin by bin.  Prefix
// sums of integers do not depend on how bins are dealt to threads: the sum a thread
// starts from is the sum its neighbour ends on, so one bin of the CTA, whoever holds
// it, crosses a given mass, and every CTA of a cluster names the same one.  (Sums
// rounded once per thread leave gaps of some units in which two threads see the
// crossing, and which of them is heard is a race.)
#pragma once

#include <cmath>

namespace wfd {

template <int PER>
struct SampleBounds {
  unsigned long long lo[PER], hi[PER];  // of each bin
  unsigned long long lo_sum, hi_sum;    // of the thread's bins
};

// The bins bin .. bin + PER - 1 with counts c: bin b's weights lie within half a bin, g
// in log2, of 2^(-g b), up to 1e-4 for the rounding of the bin and of the power; low: 0
// where the steps have no size (a bin may then hold any weight up to 1), else 0.9999.
template <int PER>
__host__ __device__ __forceinline__ SampleBounds<PER> sample_bounds(const unsigned int (&c)[PER], int bin, float g, double low) {
  constexpr double F = 1073741824.0;
  SampleBounds<PER> r;
  r.lo_sum = r.hi_sum = 0;
  for (int e = 0; e < PER; ++e) {
    const float b = (float)(bin + e);
    r.lo[e] = r.hi[e] = 0;
    if (c[e] != 0) {
      r.lo[e] = (unsigned long long)((double)c[e] * (double)exp2f(-g * (b + 0.5f)) * low * F);
      r.hi[e] = (unsigned long long)((double)c[e] * (double)exp2f(-g * fmaxf(b - 0.5f, 0.f)) * 1.0001 * F) + 1;
    }
    r.lo_sum += r.lo[e];
    r.hi_sum += r.hi[e];
  }
  return r;
}

// lo0, hi0: sums over the bins before `bin`; lo_all, hi_all: over all bins.  first(b):
// the first bin whose upper sum reaches top-p of the least the row can weigh; last(b):
// the first bin whose lower sum reaches top-p of the most.  Each is called for one bin
// of the row at most.  The margin, 2^-20 of the largest weight, covers the 2^-45 by which
// each of up to 2^19 weights is rounded in the exact sums, 2^-26 together.
template <int PER, typename First, typename Last>
__host__ __device__ __forceinline__ void sample_bracket(const SampleBounds<PER>& s, unsigned long long lo0, unsigned long long hi0,
                                               unsigned long long lo_all, unsigned long long hi_all, float top_p,
                                               int bin, First first, Last last) {
  constexpr double margin = 1024.0;
  const double p = top_p > 0.f ? (double)top_p : 0.0;
  const double from = p * (double)lo_all - margin, to = p * (double)hi_all + margin;
  for (int e = 0; e < PER; ++e) {
    const unsigned long long lo1 = lo0 + s.lo[e], hi1 = hi0 + s.hi[e];
    if ((double)hi1 >= from && ((double)hi0 < from || bin + e == 0)) first(bin + e);
    if ((double)lo1 >= to && (double)lo0 < to) last(bin + e);
    lo0 = lo1;
    hi0 = hi1;
  }
}

}  // namespace wfd
