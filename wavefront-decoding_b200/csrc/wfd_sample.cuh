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
// move an id in 1 % of the rows.  Weights are computed in 64 bits (a 32-entry table of
// 2^(j/32) and a Taylor polynomial of degree 5 on |r| <= ln 2 / 64, 2.2e-15)
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
// threshold are listed and each is told what lies before it (at most 512; denser
// bins, ties above all, are first narrowed by the same step on the 64-bit keys).  The
// exact pass also leaves the mass of every 256 tokens before the bins in question, so
// what they keep is all that is added before the id is looked up.
//
// A row is worked on by a cluster of 1 to 8 CTAs, a slice of the vocabulary each,
// joined through distributed shared memory: as many as keep every SM busy.  The first
// pass copies the slice to shared memory (where it fits), the later ones read it
// there.  Only tokens that count are weighed: a lane takes its own in turn (weighing all of
// them cost 28 thousand cycles a row of which 400 tokens weigh, this 7).  128 rows of
// 50304 bf16 logits with temperatures of 0.5 to 1.5, top-k, top-p and min-p take 66 us a call,
// one fp32 row of 32000 with top-p 13 to 16, 32 rows of 131071, half masked, 51: bound by the
// instructions of the exact pass where every token weighs (40 to 100 a token, an SM
// issuing 51 % of its cycles), by the dependent passes and cluster barriers otherwise.
// (Eight independent weights at a time, the bins' masses in a loop of their own: 70 us.)
#pragma once

#include <cooperative_groups.h>

#include "wfd_model.cuh"
#include "wfd_sample_bins.cuh"

namespace wfd {

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = 2048;
constexpr int kSampleList = kSampleThreads;
constexpr int kSampleMaxV = 1 << 19;
constexpr int kSampleTile = kSampleThreads * 8;  // tokens of one step of a CTA
constexpr int kSampleDense = 4;  // of the 8 tokens of the busiest lane
constexpr int kSampleSmem = 112 * 1024;  // dynamic shared memory: two CTAs an SM
static_assert(kSampleMaxV / 256 * 8 + 64 * 1024 <= kSampleSmem, "an uncached row");
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
  const void* norm_x;  // rows whose RMS divides the logits, or null
  int norm_ld, norm_d;
  float norm_eps;
  int slice;  // tokens per CTA of a row's cluster, a multiple of kSampleTile
  int cached; // the slice is kept in shared memory
};

struct SampleShared {
  unsigned int cnt[kSampleBins];         // tokens per bin
  unsigned int mlo[kSampleBins];         // exact mass per bin, two 32-bit halves
  unsigned int mhi[kSampleBins];
  ulonglong2 list[kSampleList];          // leader: tokens (key, weight) of the threshold's bin
  unsigned long long part[4][kSampleWarps];
  unsigned long long red[8];             // CTA results, read by the cluster
  unsigned long long bc[6];              // decisions (0, 1: the leader's thresholds for top-k and top-p)
  unsigned int n_list[2];
  float fmx, fmn;
};

__device__ __forceinline__ float sample_value(float v) { return isnan(v) ? -__int_as_float(0x7f800000) : v + 0.f; }
// larger key = larger value, then smaller index (v is not NaN; -0 has become +0)
__device__ __forceinline__ unsigned long long sample_key(float v, int i) {
  const uint32_t b = __float_as_uint(v);
  return ((unsigned long long)(b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u)) << 32) | (uint32_t)~i;
}

// The CTA's slice [lo, hi) of a row, 8 consecutive tokens to a thread; x is where the
// values are, in global or shared memory.  What is past hi, NaN, or -inf reads as -inf.
template <typename T>
struct SampleRow {
  const T* x;   // of token 0 of the row
  int lo, hi, vec;
  bool pinf;   // the maximum is +inf: its tokens share the row
  bool clean;  // the values hold no NaN and no -0
  template <typename F>
  __device__ __forceinline__ void each8(F f) const {  // f(v[8], index of v[0])
    for (int t = lo + (int)threadIdx.x * 8; t < hi; t += kSampleTile) {
      float v[8];
      load8(t, v);
      f(v, t);
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
    if (!clean) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = sample_value(v[i]);
    }
    if (pinf) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = v[i] == INF ? 0.f : -INF;
    }
  }
  __device__ __forceinline__ float load1(int t) const {  // a token inside the slice
    const float INF = __int_as_float(0x7f800000);
    float v = to_f<T>(x[t]);
    if (!clean) v = sample_value(v);
    return pinf ? (v == INF ? 0.f : -INF) : v;
  }
};

// Weight of a value: exp((v - m0) / T) for c = 32 log2(e) / T, v - m0 within the range.
// Every lane of the warp calls: lane j holds 2^(j/32), and the table is read by shuffles
// (two cycles a warp, whatever the entries).
struct SampleWeight {
  double tab, m0, c;
  __device__ __forceinline__ double operator()(float v) const {
    const double z = ((double)v - m0) * c;
    const double big = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds z to an integer
    const double zn = z + big;
    const int n = __double2loint(zn);
    const double r = z - (zn - big);  // 32 log2 of what is left, |r| <= 1/2
    constexpr double q = 0.6931471805599453094 / 32.0;
    const double p =
        fma(r, fma(r, fma(r, fma(r, fma(r, q * q * q * q * q / 120.0, q * q * q * q / 24.0), q * q * q / 6.0), q * q / 2.0), q), 1.0);
    const double w = p * __shfl_sync(0xffffffffu, tab, n & 31);
    return __hiloint2double(__double2hiint(w) + (n >> 5) * (1 << 20), __double2loint(w));
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

// ... of two values at once.
__device__ __forceinline__ void sample_scan2(unsigned long long a, unsigned long long b, unsigned long long& pa,
                                             unsigned long long& pb, unsigned long long& ta, unsigned long long& tb,
                                             SampleShared& s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long ia = a, ib = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long ya = __shfl_up_sync(0xffffffffu, ia, o), yb = __shfl_up_sync(0xffffffffu, ib, o);
    if (lane >= o) {
      ia += ya;
      ib += yb;
    }
  }
  __syncthreads();
  if (lane == 31) {
    s.part[0][warp] = ia;
    s.part[1][warp] = ib;
  }
  __syncthreads();
  pa = ia - a;
  pb = ib - b;
  ta = tb = 0;
  for (int w = 0; w < kSampleWarps; ++w) {
    pa += w < warp ? s.part[0][w] : 0;
    pb += w < warp ? s.part[1][w] : 0;
    ta += s.part[0][w];
    tb += s.part[1][w];
  }
}

// Root mean square of a row of d values, in every thread; each CTA of a row sums in the
// same order.
template <typename T>
__device__ __forceinline__ float sample_rms(const T* x, int d, float eps, SampleShared& s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float ss = 0.f;
  for (int c = threadIdx.x * 8; c < d; c += kSampleThreads * 8) {
    float v[8];
    Vec8<T>::load(x + c, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (lane == 0) s.part[2][warp] = __float_as_uint(ss);
  __syncthreads();
  float tot = 0.f;
  for (int w = 0; w < kSampleWarps; ++w) tot += __uint_as_float((uint32_t)s.part[2][w]);
  return sqrtf(tot / (float)d + eps);
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_rows_kernel(const SampleParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cl = cg::this_cluster();
  extern __shared__ __align__(16) unsigned char sample_smem[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(sample_smem);
  unsigned long long* tsum = reinterpret_cast<unsigned long long*>(&s + 1);  // kept mass of each 256 tokens
  T* cache = reinterpret_cast<T*>(tsum + p.slice / 256);                     // the slice, where p.cached
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int r = (int)(blockIdx.x / C);
  const float NEG_INF = -__int_as_float(0x7f800000), INF = -NEG_INF;
  for (int i = tid; i < kSampleBins; i += kSampleThreads) s.cnt[i] = s.mlo[i] = s.mhi[i] = 0;
  if (tid < 2) s.n_list[tid] = 0;
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
  float Tf = p.temperature != nullptr ? p.temperature[pr] : 1.f;
  const float uf = p.u[(long long)pr * p.u_stride + pc];
  const int k = p.top_k != nullptr ? p.top_k[pr] : 0;
  const float tp = p.top_p != nullptr ? p.top_p[pr] : 1.f;
  const double minp = p.min_p != nullptr ? fmin((double)p.min_p[pr], 1.0) : 0.0;

  if (p.norm_x != nullptr) {  // logits x_i / rms: into the temperature, which leaves the order of the tokens alone
    const float rms = sample_rms(static_cast<const T*>(p.norm_x) + (long long)r * p.norm_ld, p.norm_d, p.norm_eps, s);
    if (Tf > 0.f) Tf = fmaxf(Tf * rms, 1e-45f);
  }

  SampleRow<T> row;
  row.x = static_cast<const T*>(p.x) + (long long)r * p.ldx;
  row.lo = min(p.V, rank * p.slice);
  row.hi = min(p.V, row.lo + p.slice);
  row.vec = p.vec;
  row.pinf = row.clean = false;

  // ---- maximum and smallest finite value
  float mx = NEG_INF, mn = INF;
  constexpr int U = 4;  // groups in flight: this pass reads HBM
  for (int t0 = row.lo + tid * 8; t0 < row.hi; t0 += U * kSampleTile) {
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) row.load8(t0 + u * kSampleTile, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * kSampleTile;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        mx = fmaxf(mx, v[u][i]);
        mn = fminf(mn, v[u][i] > NEG_INF ? v[u][i] : INF);
      }
      if (p.cached && t < row.hi) Vec8<T>::store(cache + (t - row.lo), v[u]);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
  }
  if (lane == 0) {
    s.part[0][warp] = __float_as_uint(mx);
    s.part[1][warp] = __float_as_uint(mn);
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kSampleWarps; ++w) {
      mx = fmaxf(mx, __uint_as_float((uint32_t)s.part[0][w]));
      mn = fminf(mn, __uint_as_float((uint32_t)s.part[1][w]));
    }
    s.fmx = mx;
    s.fmn = mn;
  }
  cl.sync();
  float m0 = NEG_INF;
  mn = INF;
  for (int c = 0; c < C; ++c) {
    const SampleShared* o = cl.map_shared_rank(&s, c);
    m0 = fmaxf(m0, o->fmx);
    mn = fminf(mn, o->fmn);
  }
  if (m0 == NEG_INF) {  // nothing to sample from
    if (rank == 0 && tid == 0) p.out[r] = -1;
    cl.sync();  // the others may still read this CTA's result
    return;
  }
  if (p.cached && row.hi > row.lo) {  // (every thread reads back what it wrote itself)
    row.x = cache - row.lo;
    row.vec = 1;
    row.clean = true;
    row.hi = min(row.lo + p.slice, (row.hi + 7) & ~7);  // the last group is padded with -inf
  }
  if (m0 == INF) {
    row.pinf = true;
    m0 = mn = 0.f;
  }
  if (!(Tf > 0.f)) {  // greedy: the first index of the maximum
    int at = 0x7fffffff;
    row.each8([&](float(&v)[8], int t) {
#pragma unroll
      for (int i = 7; i >= 0; --i)
        if (v[i] == m0) at = min(at, t + i);
    });
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) s.part[2][warp] = (unsigned long long)at;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kSampleWarps; ++w) at = min(at, (int)s.part[2][w]);
      s.red[5] = (unsigned long long)at;
    }
    cl.sync();
    if (rank == 0 && tid == 0) {
      for (int c = 0; c < C; ++c) at = min(at, (int)cl.map_shared_rank(&s, c)->red[5]);
      p.out[r] = at;
    }
    cl.sync();
    return;
  }
  SampleWeight weight;
  weight.tab = exp2((double)lane / 32.0);
  weight.m0 = (double)m0;
  weight.c = 32.0 * 1.4426950408889634074 / (double)Tf;
  const float dmax = kSampleRange * Tf;

  // bins of equal steps of m0 - v over the values that have a weight
  const float D = fminf(m0 - mn, dmax);
  const float scale = D > 0.f ? fminf((float)(kSampleBins - 1) / D, 3.0e38f) : 0.f;
  // the nearest of kSampleBins steps: adding 2^23 leaves the integer in the low bits
  // (a scale of 0 makes NaN of an infinite distance: the last bin)
  constexpr float kBin0 = 8388608.f;
  auto step_of = [&](float v) { return fminf(fmaf(m0 - v, scale, kBin0), kBin0 + (float)(kSampleBins - 1)); };
  auto bin_of = [&](float v) { return (int)(__float_as_uint(step_of(v)) & (kSampleBins - 1)); };
  auto weighs = [&](float v) { return v > NEG_INF && m0 - v <= dmax; };
  unsigned long long least = 0;  // tokens with a key below this are filtered out
  const int tiles = p.slice / kSampleTile;
  // f(v, weight, tile, index) for the tokens that `want`, few of them: each lane takes its own
  // in turn, so a warp spends as many rounds on 256 tokens as its busiest lane has
  auto each_of = [&](auto want, auto f) {
    for (int k = 0; k < tiles; ++k) {
      const int t = row.lo + k * kSampleTile + tid * 8;
      unsigned todo = 0;
      if (t < row.hi) {
        float v[8];
        row.load8(t, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) todo |= want(v[i], t + i) ? 1u << i : 0u;
      }
      while (__any_sync(0xffffffffu, todo != 0)) {
        const bool on = todo != 0;
        const int i = on ? __ffs(todo) - 1 : 0;
        todo &= todo - 1;
        const float v = on ? row.load1(t + i) : m0;
        const double w = weight(v);
        if (on) f(v, w, k, t + i);
      }
    }
  };
  auto add_mass = [&](int g, unsigned long long w) {  // 64-bit sum in two 32-bit halves
    const unsigned int old = atomicAdd(&s.mlo[g], (unsigned int)w);
    atomicAdd(&s.mhi[g], (unsigned int)(w >> 32) + (old + (unsigned int)w < old ? 1u : 0u));
  };

  // The key of one threshold (which 0: top-k, 1: top-p): of all tokens of bin b with
  // key >= least, in order, the last one before which the sum (of counts, or of
  // weights) is below `need`; `before` is the sum over the bins above.  Called by the
  // whole cluster.
  auto threshold = [&](int which, int b, unsigned long long before, unsigned long long need) -> unsigned long long {
    SampleShared* lead = cl.map_shared_rank(&s, 0);
    unsigned long long klo = least, khi = ~0ull;
    for (int depth = 0; depth < 8; ++depth) {
      auto inside = [&](float v, int i) {
        if (!(weighs(v) && bin_of(v) == b)) return false;
        const unsigned long long q = sample_key(v, i);
        return q >= klo && q <= khi;
      };
      each_of(inside, [&](float v, double w, int, int i) {
        const unsigned int at = atomicAdd(&lead->n_list[which], 1u);
        if (at < (unsigned)kSampleList)
          lead->list[at] = make_ulonglong2(sample_key(v, i), which ? SampleWeight::fixed(w) : 1ull);
      });
      cl.sync();
      const unsigned int n = lead->n_list[which];
      if (n <= (unsigned)kSampleList) {
        if (rank == 0) {
          // what lies before each token: `per` neighbouring lanes share one token's sum
          int per = 32;
          while (per > 1 && per * (int)n > kSampleThreads) per >>= 1;
          const int i = tid / per, part = tid % per;
          const ulonglong2 me = i < (int)n ? s.list[i] : make_ulonglong2(0, 0);
          unsigned long long sum = 0;
          for (int j = part; j < (int)n; j += per) {
            const ulonglong2 o = s.list[j];
            sum += o.x > me.x ? o.y : 0;
          }
          for (int o = per >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          // the smallest key that is kept (the first token of the bin always is)
          unsigned long long kept = i < (int)n && (before + sum < need || sum == 0) ? me.x : ~0ull;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long y = __shfl_xor_sync(0xffffffffu, kept, o);
            kept = y < kept ? y : kept;
          }
          if (lane == 0) s.part[0][warp] = kept;
          __syncthreads();
          if (tid == 0) {
            for (int w = 1; w < kSampleWarps; ++w) kept = s.part[0][w] < kept ? s.part[0][w] : kept;
            s.bc[which] = kept;
          }
        }
        cl.sync();
        return lead->bc[which];
      }
      // too many: the range of their keys, then counts and sums over 1024 to 2048
      // equal steps of it
      cl.sync();  // every CTA has read the count, and whatever it still needed of the bins
      unsigned long long a = ~0ull, z = 0;
      row.each8([&](float(&v)[8], int t) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (weighs(v[i]) && bin_of(v[i]) == b) {
            const unsigned long long q = sample_key(v[i], t + i);
            if (q >= klo && q <= khi) {
              a = q < a ? q : a;
              z = q > z ? q : z;
            }
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
        s.n_list[which] = 0;
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
      each_of(inside, [&](float v, double w, int, int i) {
        const int g = kSampleBins - 1 - (int)((sample_key(v, i) - klo) >> shift);  // descending
        atomicAdd(&s.cnt[g], 1u);
        if (which) add_mass(g, SampleWeight::fixed(w));
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
          if (!which) v[e] = c[e];
          sum += v[e];
        }
        unsigned long long run = before + sample_scan(sum, total, s);
        if (tid == 0) s.bc[4] = kSampleBins - 1;
        __syncthreads();
        // the last non-empty step that begins below `need` holds the threshold
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          if (c[e] > 0 && run < need) atomicMin(&s.bc[4], (unsigned long long)(kSampleBins - 1 - (tid * PER + e)));
          run += v[e];
        }
        __syncthreads();
        // the sum above it
        unsigned long long above = 0;
        const int g0 = kSampleBins - 1 - (int)s.bc[4];
#pragma unroll
        for (int e = 0; e < PER; ++e) above += (tid * PER + e < g0) ? v[e] : 0;
        unsigned long long one[1] = {above};
        sample_sum<1>(one, s);
        if (tid == 0) s.bc[5] = before + one[0];
      }
      cl.sync();
      const unsigned long long step = lead->bc[4];
      before = lead->bc[5];
      const unsigned long long base = klo;
      klo = base + (step << shift);
      khi = base + ((step + 1) << shift) - 1;
      for (int i = tid; i < kSampleBins; i += kSampleThreads) s.cnt[i] = s.mlo[i] = s.mhi[i] = 0;
      cl.sync();
    }
    return least;
  };

  // One pass over what top-k kept.  Z: its mass; above: the mass of the bins before b0;
  // mlo, mhi: that of each bin b0..b1; tsum: for every 256 tokens, the mass of those
  // before b0 that min-p keeps too.
  unsigned long long mass = 0;  // this warp's tsum, summed (lane 0)
  auto weigh = [&](int b0, int b1, unsigned long long& Z, unsigned long long& above) {
    const float f0 = kBin0 + (float)b0, f1 = kBin0 + (float)b1;
    unsigned long long z[2] = {0, 0};
    for (int k = 0; k < tiles; ++k) {
      const int t = row.lo + k * kSampleTile + tid * 8;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = NEG_INF;
      if (t < row.hi) row.load8(t, v);
      unsigned todo = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        todo |= weighs(v[i]) && (least == 0 || sample_key(v[i], t + i) >= least) ? 1u << i : 0u;
      unsigned long long sure = 0;
      auto one = [&](float vi, bool on) {
        const double w = weight(on ? vi : m0);
        const unsigned long long f = on ? SampleWeight::fixed(w) : 0;
        const float st = step_of(vi);
        const bool in0 = st < f0;
        z[0] += f;
        z[1] += in0 ? f : 0;
        sure += in0 && w >= minp ? f : 0;
        const bool inner = on && !in0 && st <= f1;
        if (__any_sync(0xffffffffu, inner)) {
          if (inner) add_mass(__float_as_uint(st) & (kSampleBins - 1), f);
        }
      };
      const int rounds = __reduce_max_sync(0xffffffffu, __popc(todo));
      if (rounds >= kSampleDense) {
#pragma unroll
        for (int i = 0; i < 8; ++i) one(v[i], todo >> i & 1);
      } else {
        for (int q = 0; q < rounds; ++q) {
          const bool on = todo != 0;
          const int i = on ? __ffs(todo) - 1 : 0;
          todo &= todo - 1;
          one(on ? row.load1(t + i) : m0, on);
        }
      }
      if (rounds > 0) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sure += __shfl_xor_sync(0xffffffffu, sure, o);
      }
      if (lane == 0) {
        tsum[k * kSampleWarps + warp] = sure;
        mass += sure;
      }
    }
    Z = z[0];
    above = z[1];
  };

  const bool use_k = k > 0 && k < p.V, use_p = tp < 1.f;
  if (use_k || use_p) {
    row.each8([&](float(&v)[8], int) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (weighs(v[i])) atomicAdd(&s.cnt[bin_of(v[i])], 1u);
    });
    cl.sync();
    // counts of the whole row, this thread's bins
    constexpr int PER = kSampleBins / kSampleThreads;
    static_assert(PER == 4, "one 16-byte vector of counts a thread");
    unsigned int c[PER] = {0, 0, 0, 0};
    for (int o = 0; o < C; ++o) {
      const uint4 q = reinterpret_cast<const uint4*>(cl.map_shared_rank(&s, o)->cnt)[tid];
      c[0] += q.x;
      c[1] += q.y;
      c[2] += q.z;
      c[3] += q.w;
    }
    unsigned long long n_all = 0, at = 0;
    if (use_k) at = sample_scan((unsigned long long)c[0] + c[1] + c[2] + c[3], n_all, s);
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
      least = threshold(0, b, before, (unsigned long long)k);
    }
    if (use_p) {
      // the bins in which the mass can cross top-p
      const float g = scale > 0.f ? (float)(weight.c / 32.0 / (double)scale) : 0.f;  // log2 weight of one bin
      const SampleBounds<PER> bd = sample_bounds(c, tid * PER, g, D < INF ? 0.9999 : 0.0);
      unsigned long long tl, th, pl, ph;
      sample_scan2(bd.lo_sum, bd.hi_sum, pl, ph, tl, th, s);
      __syncthreads();
      if (tid == 0) s.bc[2] = s.bc[3] = kSampleBins - 1;
      __syncthreads();
      sample_bracket(bd, pl, ph, tl, th, tp, tid * PER, [&](int b) { s.bc[2] = b; }, [&](int b) { s.bc[3] = b; });
      __syncthreads();
      const int b0 = (int)s.bc[2], b1 = (int)s.bc[3];
      unsigned long long z[2];
      weigh(b0, b1, z[0], z[1]);
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
      unsigned long long v[PER] = {0, 0, 0, 0}, tot;
      if (tid * PER + PER > b0 && tid * PER <= b1) {
        for (int o = 0; o < C; ++o) {
          const SampleShared* os = cl.map_shared_rank(&s, o);
          const uint4 l = reinterpret_cast<const uint4*>(os->mlo)[tid], h = reinterpret_cast<const uint4*>(os->mhi)[tid];
          v[0] += ((unsigned long long)h.x << 32) + l.x;
          v[1] += ((unsigned long long)h.y << 32) + l.y;
          v[2] += ((unsigned long long)h.z << 32) + l.z;
          v[3] += ((unsigned long long)h.w << 32) + l.w;
        }
      }
      const unsigned long long bsum = v[0] + v[1] + v[2] + v[3];
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
      if (b >= 0) least = threshold(1, b, before, need);
      // the tokens of these bins that are kept (each lane adds to its warp's sums)
      auto late = [&](float v, int i) {
        if (!weighs(v)) return false;
        const int q = bin_of(v);
        return q >= b0 && q <= b1 && (least == 0 || sample_key(v, i) >= least);
      };
      each_of(late, [&](float, double w, int tile, int) {
        if (w >= minp) atomicAdd(&tsum[tile * kSampleWarps + warp], SampleWeight::fixed(w));
        if (w >= minp) mass += SampleWeight::fixed(w);
      });
    }
  }
  if (!use_p) {
    unsigned long long z0, z1;
    weigh(kSampleBins, kSampleBins, z0, z1);
  }

  // ---- the id, from the kept mass of every 256 tokens
  auto kept = [&](float v, int i) { return weighs(v) && (least == 0 || sample_key(v, i) >= least); };
  unsigned long long total[1] = {mass};
  sample_sum<1>(total, s);
  if (tid == 0) s.red[4] = total[0];
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
  if (target >= mine && target < mine + total[0]) {  // in this CTA's slice
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
            const bool on = kept(v8[i], t0 + i);
            const double w = weight(on ? v8[i] : m0);
            w8[i] = on && w >= minp ? SampleWeight::fixed(w) : 0;
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
