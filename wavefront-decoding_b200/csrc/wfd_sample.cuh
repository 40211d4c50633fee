// K12 — sampling with temperature, top-k, top-p and min-p from given uniform
// numbers: one id per row of logits.
//
// For a row x with maximum m0: w_i = exp((x_i - m0) / T); in the order "x
// descending, index ascending" top-k keeps the first k, top-p those whose
// predecessors weigh less than p of what top-k kept, min-p those with w_i >= m;
// the id is the first index, in index order, at which the kept weight so far
// exceeds u times all of it.  Nothing is sorted: each filter is one threshold
// in a total order of distinct 64-bit keys (value, then index).
//
// Precision.  A vocabulary has ~1e5 borders between ids, so sums off by 1e-7 would
// move an id in 1 % of the rows.  Weights are computed in 64 bits (a 128-entry table
// of 2^(j/128) and a Taylor polynomial of degree 4 on |r| <= ln 2 / 256, 1.2e-15)
// and held as integers, 2^44 times the weight: sums are exact in any order, so the
// id depends on the row, its parameters and u alone, not on how threads or CTAs
// are laid out.  Weights below 2^-45 of the largest are zero; V <= 2^19 keeps sums
// in 63 bits.
//
// Finding a threshold: a histogram of counts over 2048 equal steps of m0 - x (32-bit
// shared-memory atomics, no exponentials) locates the bin of the k-th token exactly,
// and the bin where the mass crosses p to within the bins' own width (a bin's weights
// lie within 2^(45/2048)); one exact pass then gives the mass kept by top-k and,
// for the few bins in question, each bin's; the tokens of the one bin that holds the
// threshold are sorted (at most 2048; denser bins, ties above all, are first
// narrowed by the same step on the 64-bit keys).
//
// A row is worked on by a cluster of 1 to 8 CTAs, a slice of the vocabulary each,
// joined through distributed shared memory: as many as keep every SM busy.  The
// first pass comes from HBM, the later ones from L1 / L2.  Bound by the 64-bit
// arithmetic of the exact passes (11 operations a token) and by the number of
// dependent passes for a few rows.
#pragma once

#include <cooperative_groups.h>

#include "wfd_model.cuh"

namespace wfd {

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = 2048;
constexpr int kSampleList = 2048;
constexpr int kSampleMaxV = 1 << 19;
constexpr int kSampleTile = kSampleThreads * 8;  // tokens of one step of a CTA
constexpr double kSampleOne = 17592186044416.0;  // 2^44
constexpr float kSampleRange = 31.3f;            // > 45 ln 2: weights beyond are zero

struct SampleParams {
  const void* x;
  int32_t* out;
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const int32_t* row_seq;
  const int32_t* row_pos;
  int32_t* err;
  long long ldx;
  int n, V, vec;  // vec: 16-byte loads are aligned
  int n_params, u_stride, u_cols, seq_stride, pos_stride;
  int slice;  // tokens per CTA of a row's cluster, a multiple of kSampleTile
};

struct SampleShared {
  double tab[128];                       // 2^(j/128)
  unsigned int cnt[kSampleBins];         // tokens per bin
  unsigned int mlo[kSampleBins];         // exact mass per bin, two 32-bit halves
  unsigned int mhi[kSampleBins];
  unsigned long long key[kSampleList];   // leader: tokens of the threshold's bin
  unsigned long long wt[kSampleList];    // ... and their weights
  unsigned long long part[4][kSampleWarps];
  unsigned long long red[8];             // CTA results, read by the cluster
  unsigned long long bc[4];              // leader's decisions
  unsigned int n_list;
  float fmx, fmn;
};

__device__ __forceinline__ float sample_value(float v) { return isnan(v) ? -__int_as_float(0x7f800000) : v + 0.f; }
// larger key = larger value, then smaller index (v is not NaN; -0 has become +0)
__device__ __forceinline__ unsigned long long sample_key(float v, int i) {
  const uint32_t b = __float_as_uint(v);
  return ((unsigned long long)(b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u)) << 32) | (uint32_t)~i;
}

template <typename T>
struct SampleRow {
  const T* x;
  int lo, hi, vec;
  bool pinf;  // the maximum is +inf: its tokens share the row
  // f(v, index) for this thread's tokens of [lo, hi); warps take 256 consecutive
  // tokens, lanes 8 consecutive ones
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    const float NEG_INF = -__int_as_float(0x7f800000);
    for (int t = lo + (int)threadIdx.x * 8; t < hi; t += kSampleTile) {
      float v[8];
      load8(t, v);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (v[i] > NEG_INF) f(v[i], t + i);
    }
  }
  __device__ __forceinline__ void load8(int t, float (&v)[8]) const {
    const float INF = __int_as_float(0x7f800000);
    if (vec && t + 8 <= hi) {
      Vec8<T>::load(x + t, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = t + i < hi ? to_f<T>(x[t + i]) : -INF;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = sample_value(v[i]);
      if (pinf) v[i] = v[i] == INF ? 0.f : -INF;
    }
  }
};

// Weight of a value: exp((v - m0) / T) for c = 128 log2(e) / T, v - m0 within the range.
struct SampleWeight {
  const double* tab;
  double m0, c;
  __device__ __forceinline__ double operator()(float v) const {
    const double z = ((double)v - m0) * c;
    const double big = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds z to an integer
    const double zn = z + big;
    const int n = __double2loint(zn);
    const double r = z - (zn - big);  // 128 log2 of what is left, |r| <= 1/2
    constexpr double q = 0.6931471805599453094 / 128.0;
    const double p = fma(r, fma(r, fma(r, fma(r, q * q * q * q / 24.0, q * q * q / 6.0), q * q / 2.0), q), 1.0);
    const double w = p * tab[n & 127];
    return __hiloint2double(__double2hiint(w) + (n >> 7) * (1 << 20), __double2loint(w));
  }
  // 2^44 w, to the nearest integer (w <= 1)
  __device__ __forceinline__ static unsigned long long fixed(double w) {
    return (unsigned long long)(__double_as_longlong(w + 256.0) - __double_as_longlong(256.0));
  }
};

// Sums of N values over the CTA, in every thread.
template <int N>
__device__ __forceinline__ void sample_sum(unsigned long long (&v)[N], SampleShared& s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (lane == 0) s.part[i][warp] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = 0;
    for (int w = 0; w < kSampleWarps; ++w) v[i] += s.part[i][w];
  }
}

// Exclusive prefix of v over the CTA's threads, and the total.
__device__ __forceinline__ unsigned long long sample_scan(unsigned long long v, unsigned long long& total,
                                                          SampleShared& s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  __syncthreads();
  if (lane == 31) s.part[0][warp] = incl;
  __syncthreads();
  unsigned long long before = 0;
  total = 0;
  for (int w = 0; w < kSampleWarps; ++w) {
    before += w < warp ? s.part[0][w] : 0;
    total += s.part[0][w];
  }
  return before + incl - v;
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_rows_kernel(const SampleParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cl = cg::this_cluster();
  extern __shared__ __align__(16) unsigned char sample_smem[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(sample_smem);
  unsigned long long* tsum = reinterpret_cast<unsigned long long*>(&s + 1);  // kept mass of each 256 tokens
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int r = (int)(blockIdx.x / C);
  const float NEG_INF = -__int_as_float(0x7f800000), INF = -NEG_INF;
  if (tid < 128) s.tab[tid] = exp2((double)tid / 128.0);
  for (int i = tid; i < kSampleBins; i += kSampleThreads) s.cnt[i] = s.mlo[i] = s.mhi[i] = 0;
  if (tid == 0) s.n_list = 0;
  griddep_wait();

  // ---- this row's parameters
  const int pr = p.row_seq != nullptr ? p.row_seq[(long long)r * p.seq_stride] : r;
  const int pc = p.row_pos != nullptr ? p.row_pos[(long long)r * p.pos_stride] : 0;
  if (pr < 0 || pr >= p.n_params || pc < 0 || pc >= p.u_cols) {  // cluster-uniform
    if (rank == 0 && tid == 0) {
      set_error(p.err, kErrBadRows);
      p.out[r] = -1;
    }
    return;
  }
  const float Tf = p.temperature != nullptr ? p.temperature[pr] : 1.f;
  const float uf = p.u[(long long)pr * p.u_stride + pc];
  const int k = p.top_k != nullptr ? p.top_k[pr] : 0;
  const float tp = p.top_p != nullptr ? p.top_p[pr] : 1.f;
  const double minp = p.min_p != nullptr ? fmin((double)p.min_p[pr], 1.0) : 0.0;

  SampleRow<T> row;
  row.x = static_cast<const T*>(p.x) + (long long)r * p.ldx;
  row.lo = min(p.V, rank * p.slice);
  row.hi = min(p.V, row.lo + p.slice);
  row.vec = p.vec;
  row.pinf = false;

  // ---- maximum (its first index) and smallest finite value
  unsigned long long best = 0;
  float mn = INF;
  row.each([&](float v, int i) {
    const unsigned long long q = sample_key(v, i);
    best = q > best ? q : best;
    mn = fminf(mn, v);
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long y = __shfl_xor_sync(0xffffffffu, best, o);
    best = y > best ? y : best;
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
  }
  if (lane == 0) {
    s.part[0][warp] = best;
    s.part[1][warp] = __float_as_uint(mn);
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kSampleWarps; ++w) {
      best = s.part[0][w] > best ? s.part[0][w] : best;
      mn = fminf(mn, __uint_as_float((uint32_t)s.part[1][w]));
    }
    s.red[0] = best;
    s.fmn = mn;
  }
  cl.sync();
  best = 0;
  mn = INF;
  for (int c = 0; c < C; ++c) {
    const SampleShared* o = cl.map_shared_rank(&s, c);
    best = o->red[0] > best ? o->red[0] : best;
    mn = fminf(mn, o->fmn);
  }
  const uint32_t bk32 = (uint32_t)(best >> 32);
  float m0 = best == 0 ? NEG_INF : __uint_as_float((bk32 & 0x80000000u) ? bk32 ^ 0x80000000u : ~bk32);
  if (best == 0 || !(Tf > 0.f)) {  // nothing to sample from, or greedy
    if (rank == 0 && tid == 0) p.out[r] = best == 0 ? -1 : (int)~(uint32_t)best;
    cl.sync();  // the others may still read this CTA's result
    return;
  }
  if (m0 == INF) {
    row.pinf = true;
    m0 = mn = 0.f;
  }
  SampleWeight weight;
  weight.tab = s.tab;
  weight.m0 = (double)m0;
  weight.c = 128.0 * 1.4426950408889634074 / (double)Tf;
  const float dmax = kSampleRange * Tf;

  // bins of equal steps of m0 - v over the values that have a weight
  const float D = fminf(m0 - mn, dmax);
  const float scale = D > 0.f ? fminf((float)kSampleBins / D, 3.0e38f) : 0.f;
  auto bin_of = [&](float v) { return min(kSampleBins - 1, (int)((m0 - v) * scale)); };
  unsigned long long least = 0;  // tokens with a key below this are filtered out

  // The key of one threshold: of all tokens of bin b with key >= least, in order,
  // the last one before which the sum (of counts, or of weights) is below `need`;
  // `before` is the sum over the bins above.  Called by the whole cluster.
  auto threshold = [&](int b, bool mass, unsigned long long before, unsigned long long need) -> unsigned long long {
    SampleShared* lead = cl.map_shared_rank(&s, 0);
    unsigned long long klo = least, khi = ~0ull;
    for (int depth = 0; depth < 8; ++depth) {
      row.each([&](float v, int i) {
        if (m0 - v <= dmax && bin_of(v) == b) {
          const unsigned long long q = sample_key(v, i);
          if (q >= klo && q <= khi) {
            const unsigned int at = atomicAdd(&lead->n_list, 1u);
            if (at < (unsigned)kSampleList) {
              lead->key[at] = q;
              lead->wt[at] = mass ? SampleWeight::fixed(weight(v)) : 1ull;
            }
          }
        }
      });
      cl.sync();
      const unsigned int n = lead->n_list;
      cl.sync();  // every CTA has read it
      if (n <= (unsigned)kSampleList) {
        if (rank == 0) {  // sort descending by key, then walk
          int m = 32;
          while (m < (int)n) m <<= 1;
          for (int i = (int)n + tid; i < m; i += kSampleThreads) {
            s.key[i] = 0;
            s.wt[i] = 0;
          }
          __syncthreads();
          for (int w = 2; w <= m; w <<= 1) {
            for (int j = w >> 1; j > 0; j >>= 1) {
              for (int i = tid; i < m / 2; i += kSampleThreads) {
                const int a = 2 * i - (i & (j - 1)), c = a + j;
                const unsigned long long ka = s.key[a], kc = s.key[c];
                if ((ka < kc) == ((a & w) == 0)) {
                  s.key[a] = kc;
                  s.key[c] = ka;
                  const unsigned long long t = s.wt[a];
                  s.wt[a] = s.wt[c];
                  s.wt[c] = t;
                }
              }
              __syncthreads();
            }
          }
          constexpr int PER = kSampleList / kSampleThreads;
          unsigned long long v[PER], sum = 0, total;
#pragma unroll
          for (int e = 0; e < PER; ++e) {
            const int i = tid * PER + e;
            v[e] = i < (int)n ? s.wt[i] : 0;
            sum += v[e];
          }
          unsigned long long run = before + sample_scan(sum, total, s);
          if (tid == 0) s.bc[0] = s.key[0];  // the first is always kept
          __syncthreads();
          // the last kept token: kept, and the next one (if any) is not
#pragma unroll
          for (int e = 0; e < PER; ++e) {
            const int i = tid * PER + e;
            const unsigned long long nextrun = run + v[e];
            if (i < (int)n && run < need && (i + 1 == (int)n || !(nextrun < need))) s.bc[0] = s.key[i];
            run = nextrun;
          }
          if (tid == 0) s.n_list = 0;
        }
        cl.sync();
        const unsigned long long q = lead->bc[0];
        cl.sync();
        return q;
      }
      // too many: the range of their keys, then counts and sums over 1024 to 2048
      // equal steps of it
      unsigned long long a = ~0ull, z = 0;
      row.each([&](float v, int i) {
        if (m0 - v <= dmax && bin_of(v) == b) {
          const unsigned long long q = sample_key(v, i);
          if (q >= klo && q <= khi) {
            a = q < a ? q : a;
            z = q > z ? q : z;
          }
        }
      });
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long ya = __shfl_xor_sync(0xffffffffu, a, o), yz = __shfl_xor_sync(0xffffffffu, z, o);
        a = ya < a ? ya : a;
        z = yz > z ? yz : z;
      }
      __syncthreads();
      if (lane == 0) {
        s.part[0][warp] = a;
        s.part[1][warp] = z;
      }
      for (int i = tid; i < kSampleBins; i += kSampleThreads) s.cnt[i] = s.mlo[i] = s.mhi[i] = 0;
      __syncthreads();
      if (tid == 0) {
        for (int w = 0; w < kSampleWarps; ++w) {
          a = s.part[0][w] < a ? s.part[0][w] : a;
          z = s.part[1][w] > z ? s.part[1][w] : z;
        }
        s.red[0] = a;
        s.red[1] = z;
        s.n_list = 0;
      }
      cl.sync();
      klo = ~0ull;
      khi = 0;
      for (int c = 0; c < C; ++c) {
        const SampleShared* o = cl.map_shared_rank(&s, c);
        klo = o->red[0] < klo ? o->red[0] : klo;
        khi = o->red[1] > khi ? o->red[1] : khi;
      }
      const int bits = 64 - __clzll((long long)(khi - klo));
      const int shift = bits > 11 ? bits - 11 : 0;
      row.each([&](float v, int i) {
        if (m0 - v <= dmax && bin_of(v) == b) {
          const unsigned long long q = sample_key(v, i);
          if (q >= klo && q <= khi) {
            const int g = kSampleBins - 1 - (int)((q - klo) >> shift);  // descending
            atomicAdd(&s.cnt[g], 1u);
            if (mass) {
              const unsigned long long w = SampleWeight::fixed(weight(v));
              const unsigned int old = atomicAdd(&s.mlo[g], (unsigned int)w);
              atomicAdd(&s.mhi[g], (unsigned int)(w >> 32) + (old + (unsigned int)w < old ? 1u : 0u));
            }
          }
        }
      });
      cl.sync();
      if (rank == 0) {
        constexpr int PER = kSampleBins / kSampleThreads;
        unsigned long long v[PER], c[PER], sum = 0, total;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const int g = tid * PER + e;
          v[e] = c[e] = 0;
          for (int o = 0; o < C; ++o) {
            const SampleShared* os = cl.map_shared_rank(&s, o);
            c[e] += os->cnt[g];
            v[e] += ((unsigned long long)os->mhi[g] << 32) + os->mlo[g];
          }
          if (!mass) v[e] = c[e];
          sum += v[e];
        }
        unsigned long long run = before + sample_scan(sum, total, s);
        if (tid == 0) s.bc[1] = kSampleBins - 1;
        __syncthreads();
        // the last non-empty step that begins below `need` holds the threshold
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          if (c[e] > 0 && run < need) atomicMin(&s.bc[1], (unsigned long long)(kSampleBins - 1 - (tid * PER + e)));
          run += v[e];
        }
        __syncthreads();
        // the sum above it
        unsigned long long above = 0;
        const int g0 = kSampleBins - 1 - (int)s.bc[1];
#pragma unroll
        for (int e = 0; e < PER; ++e) above += (tid * PER + e < g0) ? v[e] : 0;
        unsigned long long one[1] = {above};
        sample_sum<1>(one, s);
        if (tid == 0) s.bc[2] = before + one[0];
      }
      cl.sync();
      const unsigned long long step = lead->bc[1];
      before = lead->bc[2];
      const unsigned long long base = klo;
      klo = base + (step << shift);
      khi = base + ((step + 1) << shift) - 1;
      cl.sync();
    }
    return least;
  };

  const bool use_k = k > 0 && k < p.V, use_p = tp < 1.f;
  if (use_k || use_p) {
    row.each([&](float v, int) {
      if (m0 - v <= dmax) atomicAdd(&s.cnt[bin_of(v)], 1u);
    });
    cl.sync();
    // counts of the whole row, this thread's bins
    constexpr int PER = kSampleBins / kSampleThreads;
    unsigned int c[PER];
    unsigned long long sum = 0, n_all;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      c[e] = 0;
      for (int o = 0; o < C; ++o) c[e] += cl.map_shared_rank(&s, o)->cnt[tid * PER + e];
      sum += c[e];
    }
    const unsigned long long at = sample_scan(sum, n_all, s);
    if (use_k && n_all > (unsigned long long)k) {
      unsigned long long run = at;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        if (run < (unsigned long long)k && run + c[e] >= (unsigned long long)k) {
          s.bc[2] = tid * PER + e;
          s.bc[3] = run;
        }
        run += c[e];
      }
      __syncthreads();
      const int b = (int)s.bc[2];
      const unsigned long long before = s.bc[3];
      // what lies behind the k-th token's bin is gone; in it, the first k - before stay
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (tid * PER + e > b) c[e] = 0;
        else if (tid * PER + e == b) c[e] = (unsigned int)(k - before);
      cl.sync();  // every CTA has read the counts
      least = threshold(b, false, before, (unsigned long long)k);
    } else {
      cl.sync();
    }
    if (use_p) {
      // bounds of the mass up to each bin: its weights lie in [wl, wh]
      const float g = scale > 0.f ? 1.4426950408889634f / (scale * Tf) : 0.f;  // log2 weight of one bin
      double lo = 0.0, hi = 0.0, wl[PER], wh[PER];
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int b = tid * PER + e;
        wh[e] = c[e] ? (double)c[e] * (double)exp2f(-g * (float)b) * 1.0001 : 0.0;
        wl[e] = c[e] ? (double)c[e] * (double)exp2f(-g * (float)(b + 1)) * 0.9999 : 0.0;
        lo += wl[e];
        hi += wh[e];
      }
      // prefix sums as integers (2^30 per unit, rounded outwards) so that the scan above serves
      unsigned long long tl, th;
      const double F = 1073741824.0;
      unsigned long long pl = sample_scan((unsigned long long)(lo * F), tl, s);
      unsigned long long ph = sample_scan((unsigned long long)(hi * F) + 1, th, s);
      __syncthreads();
      if (tid == 0) {
        s.bc[2] = kSampleBins - 1;
        s.bc[3] = kSampleBins - 1;
      }
      __syncthreads();
      const double first = (double)tp * (double)tl - 2.0 * kSampleThreads, last = (double)tp * (double)(th + kSampleThreads);
      double rl = (double)pl, rh = (double)ph;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        rl += wl[e] * F;
        rh += wh[e] * F + 1.0;
        if (rh + kSampleThreads >= first) atomicMin(&s.bc[2], (unsigned long long)(tid * PER + e));
        if (rl - kSampleThreads >= last) atomicMin(&s.bc[3], (unsigned long long)(tid * PER + e));
      }
      for (int i = tid; i < kSampleBins; i += kSampleThreads) s.mlo[i] = s.mhi[i] = 0;
      __syncthreads();
      const int b0 = (int)s.bc[2], b1 = (int)s.bc[3];
      // exact: the mass that top-k kept, the mass above bin b0, and of each bin b0..b1
      unsigned long long z[2] = {0, 0};
      row.each([&](float v, int i) {
        if (m0 - v <= dmax && sample_key(v, i) >= least) {
          const unsigned long long w = SampleWeight::fixed(weight(v));
          const int b = bin_of(v);
          z[0] += w;
          if (b < b0) {
            z[1] += w;
          } else if (b <= b1) {
            const unsigned int old = atomicAdd(&s.mlo[b], (unsigned int)w);
            atomicAdd(&s.mhi[b], (unsigned int)(w >> 32) + (old + (unsigned int)w < old ? 1u : 0u));
          }
        }
      });
      sample_sum<2>(z, s);
      if (tid == 0) {
        s.red[2] = z[0];
        s.red[3] = z[1];
      }
      cl.sync();
      unsigned long long Z = 0, above = 0;
      for (int o = 0; o < C; ++o) {
        const SampleShared* os = cl.map_shared_rank(&s, o);
        Z += os->red[2];
        above += os->red[3];
      }
      // tokens are kept while the mass before them is below `need`
      unsigned long long need = (unsigned long long)ceil((double)tp * (double)Z);
      if (!(tp > 0.f) || need < 1) need = 1;
      unsigned long long v[PER], bsum = 0, tot;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int b = tid * PER + e;
        v[e] = 0;
        if (b >= b0 && b <= b1)
          for (int o = 0; o < C; ++o) {
            const SampleShared* os = cl.map_shared_rank(&s, o);
            v[e] += ((unsigned long long)os->mhi[b] << 32) + os->mlo[b];
          }
        bsum += v[e];
      }
      unsigned long long run = above + sample_scan(bsum, tot, s);
      __syncthreads();
      if (tid == 0) {
        s.bc[2] = 0;
        s.bc[3] = above;
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        // the bin in which the mass reaches `need` (one at most)
        if (v[e] > 0 && run < need && run + v[e] >= need) {
          s.bc[2] = tid * PER + e + 1;
          s.bc[3] = run;
        }
        run += v[e];
      }
      __syncthreads();
      const int b = (int)s.bc[2] - 1;
      const unsigned long long before = s.bc[3];
      cl.sync();  // every CTA has read the masses and results
      if (b >= 0) least = threshold(b, true, before, need);
    }
  }

  // ---- kept mass of every 256 tokens, then the id
  const int tiles = (p.slice + kSampleTile - 1) / kSampleTile;
  unsigned long long mass[1] = {0};
  for (int t = 0; t < tiles; ++t) {
    const int t0 = row.lo + t * kSampleTile + tid * 8;
    unsigned long long w8 = 0;
    if (t0 < row.hi) {
      float v[8];
      row.load8(t0, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (v[i] > NEG_INF && m0 - v[i] <= dmax && sample_key(v[i], t0 + i) >= least) {
          const double w = weight(v[i]);
          w8 += w >= minp ? SampleWeight::fixed(w) : 0ull;
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w8 += __shfl_xor_sync(0xffffffffu, w8, o);
    if (lane == 0) {
      tsum[t * kSampleWarps + warp] = w8;
      mass[0] += w8;
    }
  }
  sample_sum<1>(mass, s);
  if (tid == 0) s.red[4] = mass[0];
  cl.sync();
  unsigned long long Z = 0, mine = 0;
  for (int o = 0; o < C; ++o) {
    const unsigned long long z = cl.map_shared_rank(&s, o)->red[4];
    if (o < rank) mine += z;
    Z += z;
  }
  // the id is the first index at which the mass exceeds `target`
  unsigned long long target = uf > 0.f ? (unsigned long long)((double)fminf(uf, 1.f) * (double)Z) : 0ull;
  if (target >= Z) target = Z - 1;
  if (target >= mine && target < mine + mass[0]) {  // in this CTA's slice
    unsigned long long run = mine;
    if (warp == 0) {
      // 32 groups at a time until the one that holds the target
      const int n = tiles * kSampleWarps;
      for (int g0 = 0; g0 < n; g0 += 32) {
        const unsigned long long v = g0 + lane < n ? tsum[g0 + lane] : 0;
        unsigned long long incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned long long y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, run + incl > target);
        if (hit) {
          const int l = __ffs(hit) - 1;
          const int g = g0 + l;
          run += __shfl_sync(0xffffffffu, incl - v, l);
          // this group's tokens: 8 per lane
          const int t0 = row.lo + (g / kSampleWarps) * kSampleTile + (g % kSampleWarps) * 256 + lane * 8;
          float v8[8];
          unsigned long long w8[8], sum = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) v8[i] = NEG_INF;
          if (t0 < row.hi) row.load8(t0, v8);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            w8[i] = 0;
            if (v8[i] > NEG_INF && m0 - v8[i] <= dmax && sample_key(v8[i], t0 + i) >= least) {
              const double w = weight(v8[i]);
              w8[i] = w >= minp ? SampleWeight::fixed(w) : 0ull;
            }
            sum += w8[i];
          }
          unsigned long long inc = sum;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
          }
          unsigned long long at = run + inc - sum;
          const unsigned own = __ballot_sync(0xffffffffu, at + sum > target);
          if (lane == __ffs(own) - 1) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if (at <= target && at + w8[i] > target) p.out[r] = t0 + i;
              at += w8[i];
            }
          }
          break;
        }
        run += __shfl_sync(0xffffffffu, incl, 31);
      }
    }
  }
  cl.sync();  // no CTA leaves while another reads its shared memory
}

}  // namespace wfd
