// K11 — wavefront attention over the 8-bit slot cache on the 5th-generation tensor
// cores: bf16 queries, head_dim 128, or head_dim 64 with an even kv-head count
// (two heads as one 128-byte row, as K2's head pairs).
//
// The cached codes go from HBM to the tensor core as they are: TMA tiles of 128
// keys x 128 bytes feed tcgen05.mma kind::f8f6f4 (e4m3 x e4m3 -> f32), with no
// conversion pass.  The other operand keeps its precision by being split into two
// e4m3 pieces of 4 significant bits each, a row / column n of 8 bits becoming two
// columns n and NQP + n of the same MMA:
//     x 2^-e = x1 + x2 / 16,  x1 = e4m3(x 2^-e),  x2 = e4m3(16 (x 2^-e - x1))
// (e from the row's largest element, |x 2^-e| <= 448, so |16 (.. - x1)| <= 256).
//   Q: a bf16 value has 8 significant bits, so both pieces together are exact down
//      to 2^-23 of the row's largest element.
//   P: each piece is off by at most half a step, 2^-4 of its value: 2^-8 together,
//      what rounding P to bf16 costs, down to weights of 2^-16 of the largest (an
//      attention sink over 64k flat keys stays inside that).  The weights' sum is
//      taken of the unrounded weights in fp32.
// The minimum N of the instruction leaves room for the second piece, so a tile of
// 32 KB takes 8 MMAs, half of the bf16 kernel's for the same bytes.
//     S^T[128 keys x 2 NQP] = K . [Q1 | Q2]^T         (K-major, 4 k-steps of 32 bytes)
//     O^T[128 dims x 2 NQP] += V^T . [P1 | P2]^T       (both MN-major, 4 k-steps of 32 keys)
// Scales: a key's 2^{e_k} multiplies its finished score; its value scale joins the
// weight, t = s + e_v in log2 units, so that the running maximum is taken of t and
// the weights stay within e4m3's range: w = 2^(t - M + 8), M moved when a tile
// exceeds it by 3/4 (w <= 431 < 448).  The denominator needs 2^(s - M + 8) = w 2^{-e_v}.
// |e_v| <= 32 keeps that above the fp32 underflow for every key that matters.
//
// What bounds it: HBM.  A tile pair (256 keys, 64 KB) takes 1.5 us of an SM's share
// of the copy bandwidth; the softmax of a pair is one dependent chain through two
// named barriers, so each softmax thread works on two keys (one of either tile):
// the chain's latency is paid once per 64 KB, as in the bf16 kernel.
//
// Warp roles (one CTA per SM): 0 TMA producer; 1 TMEM owner and MMA issuer; 2 the
// Q operand of the next units (two buffers); 3 the keys' exponents (a ring of tile
// pairs); 4.. softmax, 4 warps per slice of the query columns.  Work split, merging and the self-planned start are K2's
// (UnitIter, CtaStart).  Every wait is bounded; no multicast, no cluster.
#pragma once

#include "wfd_q8_attn.cuh"

namespace wfd {

// Tensor maps of a code buffer: boxes of 256 rows (a tile pair), and of 128, 64, 32,
// 16 and 8 for its tail.
constexpr int kQ8Boxes = 6;
struct Q8Maps {
  CUtensorMap k[kQ8Boxes];
  CUtensorMap v[kQ8Boxes];
};

template <int NQP, int G>
struct Q8Cfg {
  static constexpr int N = 2 * NQP;                  // MMA columns: both pieces
  // Rings of tile pairs (256 keys x 128 bytes).  A K pair is done with after S, a V
  // pair only after the softmax and P.V, one pair later: twice the V pairs keep as
  // many of either in flight.
  static constexpr int KS = 2;
  static constexpr int VS = NQP == 16 ? 4 : 3;
  static constexpr int TILE_BYTES = kTcTile * 128;
  static constexpr int PAIR_BYTES = 2 * TILE_BYTES;
  static constexpr int Q_BYTES = N * 128;            // one of two buffers
  static constexpr int P_ROWB = N;                   // one key's row of P^T
  static constexpr int P_BYTES = 2 * kTcTile * P_ROWB;     // one group's
  static constexpr int P_SWZ_BITS = NQP == 16 ? 1 : 2;     // 32- / 64-byte swizzle
  static constexpr uint64_t P_LAYOUT = NQP == 16 ? 6 : 4;
  static constexpr int P_ATOM = 8 * P_ROWB;
  static constexpr int RED_FLOATS = G * 2 * 4 * NQP;
  static constexpr int EXP_RING = 4;                 // tile pairs of key / value exponents, one 32-bit word a key
  static constexpr int EXP_BYTES = EXP_RING * 2 * kTcTile * 4;
  static constexpr int MX_FLOATS = (NQP == 16 ? 8 : 16) * 2 * 16;  // per softmax warp: running maxima and rescale factors
  static constexpr int ML_FLOATS = 2 * NQP;          // the second group's maxima and sums at the end of a unit
  static constexpr int SMEM = (KS + VS) * PAIR_BYTES + 2 * Q_BYTES + G * P_BYTES + EXP_BYTES +
                              (2 * RED_FLOATS + 4 * NQP + MX_FLOATS + ML_FLOATS) * 4 + 1024;
  static constexpr int S_COL = 0;                    // S^T of tile pair buffer sb, half hf: (2 sb + hf) N
  static constexpr int O_COL = 4 * N;                // O^T of group g: O_COL + g N
  static constexpr int TMEM_COLS = NQP == 16 ? 256 : 512;
  static constexpr int PART_FLOATS = NQP * (128 + 2);
  static_assert(O_COL + G * N <= TMEM_COLS, "TMEM columns");
  static_assert(SMEM + 2048 <= 232448, "shared memory per CTA (dynamic + the kernel's static arrays)");
};

// Softmax warps: groups that take alternate tile pairs, each with its own maxima,
// sums and O (merged at the end of a unit), and slices of the query columns inside
// a group.  Up to 16 columns a pair's softmax is a chain of dependent steps, and two
// groups keep two pairs in it; 32 columns are bound by instruction issue, and four
// slices of 8 fill the schedulers with less state a thread.
__host__ __device__ constexpr int q8_groups(int na) { return na <= 16 ? 2 : 1; }
__host__ __device__ constexpr int q8_slices(int na) { return na <= 16 ? 1 : na / 8; }
__host__ __device__ constexpr int q8_tc_threads(int na) { return 128 + 128 * q8_groups(na) * q8_slices(na); }

// kind::f8f6f4, e4m3 x e4m3 -> f32, M = 128
__host__ __device__ constexpr uint32_t q8_idesc(int n, bool a_mn_major, bool b_mn_major) {
  return (1u << 4) | ((a_mn_major ? 1u : 0u) << 15) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(0), "r"(0), "r"(0), "r"(0));
}

// A value every lane holds, known to the compiler as warp-uniform: tcgen05.mma takes
// its operands in uniform registers, and moving them there from per-thread ones
// made the issue of one MMA cost 154 cycles against 41 (of which 32 are the reads
// of the A operand).
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }
// One lane of the (converged) warp, the same at every call.
__device__ __forceinline__ bool elect_lane() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(p));
  return p != 0;
}

// Bounded mbarrier wait by every lane of a warp, with a warp-uniform result: one
// probe and one vote when the phase has completed (every pair passes about ten of
// these; tc_wait's further load of the abort flag made them 200 cycles each).
// Otherwise it gives up at the spin limit (error word and CTA abort flag) or as soon
// as another role has aborted: the roles keep their control flow, issue no more
// work that depends on the wait, and every wait after it ends the same way.
__device__ __forceinline__ bool q8_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  for (uint32_t i = 1; i < kSpinLimit; ++i) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if (__any_sync(0xffffffffu, *abort_flag != 0)) return false;
  }
  set_error(err, kErrTimeout);
  *abort_flag = 1;
  return false;
}

// 32 TMEM lanes, N consecutive columns -> N registers per thread
template <int N>
__device__ __forceinline__ void tmem_cols(uint32_t taddr, float (&v)[N]) {
  if constexpr (N == 16) {
    tmem_ld<16>(taddr, v);
  } else {
    uint32_t r[N];
    if constexpr (N == 2)
      asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(taddr));
    else if constexpr (N == 4)
      asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                   : "r"(taddr));
    else
      asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                   : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                   : "r"(taddr));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __uint_as_float(r[i]);
  }
}

// Two fp32 values in one 64-bit register: one instruction for both (the softmax of
// 32 columns is bound by instruction issue).
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pk2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void up2(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 2^x, 0 far below; x <= 9 here (a NaN stays one)
__device__ __forceinline__ float ex2_ftz(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Two values as two pieces: codes of (a, b) in the low 16 bits of p1 and p2.
__device__ __forceinline__ void q8_split(f32x2 w, uint32_t& p1, uint32_t& p2) {
  float a, b;
  up2(w, a, b);
  p1 = e4m3x2(a, b);
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)p1, __NV_E4M3);
  const float2 f = __half22float2(__half2(h));
  const f32x2 r = fma2(pk2(f.x, f.y), pk2(-16.f, -16.f), mul2(w, pk2(16.f, 16.f)));  // 16 (w - f), exact
  up2(r, a, b);
  p2 = e4m3x2(a, b);
}

// A CTA's share of the work and where it starts, from the item table itself (K2's
// self-planned start: the plan kernel may still be running).  Called by the whole CTA.
struct SelfStart {
  long long wtot[32];
  Seg S0;
  long long base0, nbase0;
  int seg0, slot0, seq0, minpos;
};
template <int THREADS>
__device__ __forceinline__ long long self_start(const VerifyParams& p, SelfStart& sh, long long& share, long long& a,
                                                long long& b) {
  constexpr int IPT = (kSelfPlanMax + THREADS - 1) / THREADS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  wfd_item my[IPT];
  long long w[IPT], tsum = 0;
#pragma unroll
  for (int k = 0; k < IPT; ++k) {
    const int i = tid * IPT + k;
    w[k] = 0;
    if (i < p.n_segs) {
      my[k] = p.items[i];
      Seg s;
      w[k] = slot_segment(p, my[k], s);
    }
    tsum += w[k];
  }
  long long incl = tsum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) sh.wtot[warp] = incl;
  if (tid == 0) sh.minpos = 0x7fffffff;
  __syncthreads();
  long long before = 0, all = 0;
#pragma unroll
  for (int k = 0; k < THREADS / 32; ++k) {
    before += (k < warp) ? sh.wtot[k] : 0;
    all += sh.wtot[k];
  }
  const long long total = (long long)p.Hkv * all;
  share = 1;
  a = b = 0;
  if (total > 0) {
    share = max((total + gridDim.x - 1) / gridDim.x, (long long)kQ8MinShare);
    a = (long long)blockIdx.x * share;
    b = (a + share < total) ? a + share : total;
  }
  if (a < b) {  // the item that holds work index a, by the thread that holds the item
    long long pf = before + incl - tsum;
#pragma unroll
    for (int k = 0; k < IPT; ++k) {
      const int i = tid * IPT + k;
      if (w[k] > 0 && (long long)p.Hkv * pf <= a && a < (long long)p.Hkv * (pf + w[k])) {
        slot_segment(p, my[k], sh.S0);
        sh.base0 = (long long)p.Hkv * pf;
        sh.nbase0 = i + 1 <= p.n_segs - 1 ? (long long)p.Hkv * (pf + w[k]) : 0x7fffffffffffffffll;
        sh.seg0 = i;
        sh.slot0 = my[k].slot;
        sh.seq0 = my[k].seq;
      }
      pf += w[k];
    }
  }
  __syncthreads();
  if (a < b) {  // the lowest position any item writes on that (slot, sequence): below it nothing changes
    int mp = 0x7fffffff;
#pragma unroll
    for (int k = 0; k < IPT; ++k)
      if (w[k] > 0 && my[k].slot == sh.slot0 && my[k].seq == sh.seq0 && my[k].pos0 < mp) mp = my[k].pos0;
    if (mp != 0x7fffffff) atomicMin(&sh.minpos, mp);
  }
  __syncthreads();
  return total;
}

// The query columns of one unit: up to NQP vectors of one kv head, or up to NQP / 2
// of either head of a pair (head 0's first).
template <bool PAIR, int NQP>
struct UnitCols {
  int v0, nv1, nvec;
  __device__ __forceinline__ UnitCols(const VerifyParams& p, const Seg& S, int qg) {
    constexpr int gh = PAIR ? NQP / 2 : NQP;
    v0 = qg * gh;
    nv1 = min(gh, S.q_len * p.G - v0);
    nvec = PAIR ? 2 * nv1 : nv1;
  }
  __device__ __forceinline__ int head(int n) const { return PAIR && n >= nv1 ? 1 : 0; }
  __device__ __forceinline__ int vec(int n) const { return v0 + (PAIR && n >= nv1 ? n - nv1 : n); }
};

// NA: query columns the softmax works on (every unit has at most NA vectors).
template <int NQP, int NA, bool PAIR>
__global__ void __launch_bounds__(q8_tc_threads(NA), 1)
    q8_tc_kernel(const __grid_constant__ Q8Maps maps, const Q8AttnParams p) {
  constexpr int G = q8_groups(NA);   // softmax groups
  constexpr int H = q8_slices(NA);   // column slices of a group (4 warps each)
  using C = Q8Cfg<NQP, G>;
  constexpr int KS = C::KS, VS = C::VS;
  constexpr int N = C::N;
  constexpr int THREADS = q8_tc_threads(NA);
  constexpr int NL = NA / H;         // query columns per softmax thread
  constexpr int SMT = 128 * H;       // softmax threads of a group
  static_assert(4 * G * H * 32 <= C::MX_FLOATS && (G == 1 || NL * kTcTile * 4 <= C::P_BYTES), "the merge of two groups");
  static_assert(NL == 2 || NL == 4 || NL == 8 || NL == 16, "columns per softmax thread");
  static_assert(NA <= NQP, "active query columns");
  static_assert(KS == 2, "the K ring shares S's barriers");
  const float NEG_INF = -__int_as_float(0x7f800000);

  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* kts = smem;                                // KS K tile pairs
  unsigned char* vts = kts + KS * C::PAIR_BYTES;            // VS V tile pairs
  unsigned char* qs = vts + VS * C::PAIR_BYTES;             // 2 x Q operand (K-major, 128B swizzle)
  unsigned char* ps = qs + 2 * C::Q_BYTES;                  // P^T operand of a tile pair (MN-major), per group
  float* red = reinterpret_cast<float*>(ps + G * C::P_BYTES);  // [G][2][4][NQP] column maxima
  float* lred = red + C::RED_FLOATS;                        // [G][2][4][NQP] column sums
  float* ml = lred + C::RED_FLOATS;                         // [2][NQP] the second group's maxima and sums
  float* cscale = ml + C::ML_FLOATS;                     // [4][NQP] score scale of each column, per unit
  float* mxs = cscale + 4 * NQP;                            // [16][2][16] per softmax warp
  uint32_t* exps = reinterpret_cast<uint32_t*>(mxs + C::MX_FLOATS);  // [EXP_RING][2][128] exponents of a key

  __shared__ __align__(8) uint64_t bar_kfull[KS];
  __shared__ __align__(8) uint64_t bar_vfull[VS];
  __shared__ __align__(8) uint64_t bar_vempty[VS];
  __shared__ __align__(8) uint64_t bar_sfull[2];
  __shared__ __align__(8) uint64_t bar_sfree[2];
  __shared__ __align__(8) uint64_t bar_pfull[G];
  __shared__ __align__(8) uint64_t bar_ofull[G];
  __shared__ __align__(8) uint64_t bar_qready[4];  // unit's Q and column scales written
  __shared__ __align__(8) uint64_t bar_qfree[2];
  __shared__ __align__(8) uint64_t bar_drain;
  __shared__ __align__(8) uint64_t bar_efull[C::EXP_RING];   // a tile pair's exponents written
  __shared__ __align__(8) uint64_t bar_efree[C::EXP_RING];   // ... and read by every softmax warp
  __shared__ uint32_t s_tmem;
  __shared__ int s_rp[G][NQP];  // gapped windows: each query column's row position
  __shared__ volatile int s_abort;
  __shared__ int s_flag;
  __shared__ SelfStart s_start;

  const int tid = threadIdx.x, warp = (int)uniform((uint32_t)tid >> 5), lane = tid & 31;
  const bool self = p.items != nullptr;
  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.k[0])) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.v[0])) : "memory");
    for (int s = 0; s < KS; ++s) {
      mbar_init(&bar_kfull[s], 1);
    }
    for (int s = 0; s < VS; ++s) {
      mbar_init(&bar_vfull[s], 1);
      mbar_init(&bar_vempty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bar_sfull[s], 1);
      mbar_init(&bar_sfree[s], 4 * H);
      mbar_init(&bar_qfree[s], 1);
    }
    for (int s = 0; s < 4; ++s) mbar_init(&bar_qready[s], 1);
    for (int s = 0; s < C::EXP_RING; ++s) {
      mbar_init(&bar_efull[s], 1);
      mbar_init(&bar_efree[s], 4 * H);
    }
    for (int s = 0; s < G; ++s) {
      mbar_init(&bar_pfull[s], 1);
      mbar_init(&bar_ofull[s], 1);
    }
    mbar_init(&bar_drain, 1);
    fence_mbar_init();
    s_abort = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                 "r"(C::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (!self) griddep_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  long long share = 1, a = 0, b = 0;
  CtaStart cs{};
  int minpos = 0;
  if (self) {
    self_start<THREADS>(p, s_start, share, a, b);
    cs.S = s_start.S0;
    cs.base = s_start.base0;
    cs.nbase = s_start.nbase0;
    cs.seg = s_start.seg0;
    minpos = s_start.minpos;
  } else {
    cs = p.start[blockIdx.x];
    const long long total = (long long)p.Hkv * p.prefix[p.n_segs];
    if (total > 0) {
      share = max((total + gridDim.x - 1) / gridDim.x, (long long)kQ8MinShare);
      a = (long long)blockIdx.x * share;
      b = (a + share < total) ? a + share : total;
    }
  }
  const int seg0 = cs.seg;
  auto make_iter = [&]() {
    UnitIter r{a, b, seg0};
    if (a < b) {
      r.have = true;
      r.S = cs.S;
      r.base = cs.base;
      r.nbase = cs.nbase;
    }
    r.waited = !self;
    return r;
  };
  // before reading cache rows (or their exponents) [.., end) of the current
  // segment: the plan kernel's append may write rows from minpos on
  auto need_rows = [&](UnitIter& itr, int end) {
    if (!itr.waited && (itr.seg != seg0 || end > minpos)) {
      griddep_wait();
      itr.waited = true;
    }
  };

  Seg S;
  int u, r_lo, r_hi;
  long long ustart;
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    UnitIter itr = make_iter();
    uint32_t it = 0;
    uint32_t n_k = 0, n_v = 0;  // pairs whose loads were issued (prefixes of the sequence: issue stops at an abort)
    while (itr.next(p, S, u, r_lo, r_hi, ustart)) {
      const int h = u % p.Hkv;
      const int n_t = (r_hi - r_lo + 2 * kTcTile - 1) / (2 * kTcTile);
      const long long row0 = S.k_row0 + p.k_row_offset + r_lo;
      for (int t = 0; t < n_t; ++t, ++it) {
        need_rows(itr, r_lo + (t + 1) * 2 * kTcTile);
        const int row = (int)(row0 + (long long)t * 2 * kTcTile);
        // a last pair of at most 224 keys loads only those, in boxes of 128 / 64 / 32 /
        // 16 / 8 rows; what the stage holds past them is masked (V: zeroed)
        const int left = r_hi - r_lo - t * 2 * kTcTile;
        const int nr = left > 224 ? 2 * kTcTile : ((left + 7) & ~7);
        auto load = [&](unsigned char* dst, const CUtensorMap* m, uint64_t* bar) {
          mbar_arrive_expect_tx(bar, (uint32_t)(nr * 128));
          if (nr == 2 * kTcTile) {
            tma_load_3d(dst, m, 0, h, row, bar);
          } else {
            int off = 0;
            for (int pc = 1; pc < kQ8Boxes; ++pc) {
              const int pr = 256 >> pc;
              if (nr & pr) {
                tma_load_3d(dst + off * 128, m + pc, 0, h, row + off, bar);
                off += pr;
              }
            }
          }
        };
        const int ks = (int)(it % KS), vs = (int)(it % VS);
        // (the K ring is as deep as S: pair it - 2's S complete frees its K)
        bool go = it >= (uint32_t)KS ? q8_wait(&bar_sfull[ks], ((it / KS) - 1) & 1u, &s_abort, p.err) : !s_abort;
        if (go && lane == 0) {
          load(kts + ks * C::PAIR_BYTES, maps.k, &bar_kfull[ks]);
          n_k = it + 1;
          if (p.fail_waits && n_k == 1) {  // test hook: give up with this copy in flight
            set_error(p.err, kErrTimeout);
            s_abort = 1;
          }
        }
        __syncwarp();
        go = it >= (uint32_t)VS ? q8_wait(&bar_vempty[vs], ((it / VS) - 1) & 1u, &s_abort, p.err) : !s_abort;
        if (go && lane == 0) {
          load(vts + vs * C::PAIR_BYTES, maps.v, &bar_vfull[vs]);
          n_v = it + 1;
        }
        __syncwarp();
      }
    }
    // the MMA warp's commits land on these barriers before the CTA exits
    for (uint32_t j = (it > (uint32_t)VS ? it - VS : 0); j < it; ++j)
      q8_wait(&bar_vempty[j % VS], (j / VS) & 1u, &s_abort, p.err);
    // copies in flight land before the CTA exits, also after an abort
    if (lane == 0) {
      for (uint32_t j = (n_k > (uint32_t)KS ? n_k - KS : 0); j < n_k; ++j)
        if (!mbar_wait_bounded(&bar_kfull[j % KS], (j / KS) & 1u)) set_error(p.err, kErrTimeout);
      for (uint32_t j = (n_v > (uint32_t)VS ? n_v - VS : 0); j < n_v; ++j)
        if (!mbar_wait_bounded(&bar_vfull[j % VS], (j / VS) & 1u)) set_error(p.err, kErrTimeout);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    UnitIter itr = make_iter();
    uint32_t it = 0, units = 0;  // it: tile pairs before this unit
    constexpr uint32_t IDESC_S = q8_idesc(N, false, false);
    constexpr uint32_t IDESC_PV = q8_idesc(N, true, true);
    const uint32_t q_addr = smem_u32(qs);
    const uint32_t p_addr = smem_u32(ps);
    const uint32_t k_addr = smem_u32(kts);
    const uint32_t v_addr = smem_u32(vts);
    const uint32_t tm = uniform(tmem);
    while (itr.next(p, S, u, r_lo, r_hi, ustart)) {
      const int n_sub = (r_hi - r_lo + kTcTile - 1) / kTcTile;
      const int n_t = (n_sub + 1) >> 1;
      const int qb = (int)(units & 1u);
      const uint32_t qa = uniform(q_addr + (uint32_t)(qb * C::Q_BYTES));
      q8_wait(&bar_qready[units & 3u], (units >> 2) & 1u, &s_abort, p.err);
      tc_fence_after();
      // S of pair t + 1 goes out before P.V of pair t, whose weights the softmax is
      // still computing; but when its keys are late, P.V does not wait for them
      int ts = 0, tv = 0;
      while (tv < n_t) {
        bool do_s = ts < n_t, s_ok = false, p_ok = false;
        if (do_s && tv < ts) {
          const uint32_t i = it + ts, j = it + tv;
          for (uint32_t n = 0; n < kSpinLimit; ++n) {  // (every exit by a vote)
            s_ok = __all_sync(0xffffffffu, mbar_test_wait(&bar_kfull[i % KS], (i / KS) & 1u) &&
                                               (i < 2 || mbar_test_wait(&bar_sfree[i & 1u], ((i >> 1) - 1) & 1u)));
            if (s_ok) break;
            p_ok = __all_sync(0xffffffffu, mbar_test_wait(&bar_pfull[j % G], (j / G) & 1u));
            if (p_ok || __any_sync(0xffffffffu, s_abort != 0)) break;
          }
          do_s = !p_ok;
        }
        if (do_s) {
          const uint32_t i = it + ts;
          const int sb = (int)(i & 1u), ks = (int)(i % KS);
          const bool two = uniform(2 * ts + 1 < n_sub) != 0;
          bool go = s_ok;
          if (!s_ok) {
            go = q8_wait(&bar_kfull[ks], (i / KS) & 1u, &s_abort, p.err);
            if (i >= 2) go = q8_wait(&bar_sfree[sb], ((i >> 1) - 1) & 1u, &s_abort, p.err) && go;
          }
          tc_fence_after();
          const uint32_t k0 = uniform(k_addr + (uint32_t)(ks * C::PAIR_BYTES));
          const uint32_t d0 = uniform(tm + (uint32_t)(2 * sb * N));
          if (go && elect_lane()) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // 32 bytes of the row; the two tiles are independent accumulators
              umma_f8(d0, umma_desc(k0 + j * 32, 16, 1024, 2), umma_desc(qa + j * 32, 16, 1024, 2), IDESC_S,
                      j > 0 ? 1u : 0u);
              if (two)
                umma_f8(d0 + N, umma_desc(k0 + C::TILE_BYTES + j * 32, 16, 1024, 2),
                        umma_desc(qa + j * 32, 16, 1024, 2), IDESC_S, j > 0 ? 1u : 0u);
            }
            umma_commit(&bar_sfull[sb]);
            if (ts == n_t - 1) umma_commit(&bar_qfree[qb]);  // the unit's Q buffer may be rewritten
          }
          __syncwarp();
          ++ts;
        } else {
          const uint32_t i = it + tv;
          const int vs = (int)(i % VS);
          const bool two = uniform(2 * tv + 1 < n_sub) != 0;
          bool go = q8_wait(&bar_vfull[vs], (i / VS) & 1u, &s_abort, p.err);
          const int g = (int)(i % G);
          // (P of pair i written: the group has read S and the O of its pair before)
          if (!p_ok) go = q8_wait(&bar_pfull[g], (i / G) & 1u, &s_abort, p.err) && go;
          tc_fence_after();
          const uint32_t v0 = uniform(v_addr + (uint32_t)(vs * C::PAIR_BYTES));
          const uint32_t o0 = uniform(tm + (uint32_t)(C::O_COL + g * N));
          const uint32_t p0 = uniform(p_addr + (uint32_t)(g * C::P_BYTES));
          if (go && elect_lane()) {
            // k-step j: 32 keys, four 8-row groups of V and of P^T
#pragma unroll
            for (int j = 0; j < 4; ++j)
              umma_f8(o0, umma_desc(v0 + j * 4096, 16, 1024, 2),
                      umma_desc(p0 + j * 4 * C::P_ATOM, 16, C::P_ATOM, C::P_LAYOUT), IDESC_PV, j > 0 ? 1u : 0u);
            if (two) {
#pragma unroll
              for (int j = 4; j < 8; ++j)
                umma_f8(o0, umma_desc(v0 + j * 4096, 16, 1024, 2),
                        umma_desc(p0 + j * 4 * C::P_ATOM, 16, C::P_ATOM, C::P_LAYOUT), IDESC_PV, 1u);
            }
            umma_commit(&bar_ofull[g]);
            umma_commit(&bar_vempty[vs]);
          }
          __syncwarp();
          ++tv;
        }
      }
      it += n_t;
      ++units;
    }
    // every MMA complete before TMEM is freed and the CTA exits, also after an abort
    if (elect_lane()) {
      umma_commit(&bar_drain);
      if (!mbar_wait_bounded(&bar_drain, 0)) set_error(p.err, kErrTimeout);
    }
    __syncwarp();
  } else if (warp == 2) {
    // ------------------------------------------------------------ Q operand
    // Lane l holds bytes 4l..4l+3 of a 128-byte row.  Rows n and NQP + n: the two
    // pieces of query vector n.  The operand has two buffers (unit w is written once
    // the S MMAs of unit w - 2 are done), its barriers and the column scales four:
    // the softmax, two tile pairs behind the MMA warp, may still be in unit w - 3.
    UnitIter itr = make_iter();
    uint32_t units = 0;
    const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.q);
    while (itr.next(p, S, u, r_lo, r_hi, ustart)) {
      const int h = u % p.Hkv, qg = u / p.Hkv;
      const int qb = (int)(units & 1u);
      const bool go = units >= 2 ? q8_wait(&bar_qfree[qb], ((units >> 1) - 1) & 1u, &s_abort, p.err) : !s_abort;
      if (go) {
        const UnitCols<PAIR, NQP> uc(p, S, qg);
        unsigned char* qd = qs + qb * C::Q_BYTES;
        float* cd = cscale + (units & 3u) * NQP;
        constexpr int QB = NA < 8 ? NA : 8;  // vectors loaded at once
        for (int n0 = 0; n0 < NA; n0 += QB) {
          uint2 raw[QB];
#pragma unroll
          for (int i = 0; i < QB; ++i) {
            const int n = n0 + i;
            raw[i] = make_uint2(0, 0);
            if (n < uc.nvec) {
              const int e = uc.head(n), v = uc.vec(n);
              if (PAIR) {
                if ((lane >> 4) == e)
                  raw[i] = *reinterpret_cast<const uint2*>(
                      q + ((long long)(S.q_row0 + v / p.G) * p.Hq + (2 * h + e) * p.G + v % p.G) * 64 + (lane & 15) * 4);
              } else {
                raw[i] = *reinterpret_cast<const uint2*>(
                    q + ((long long)(S.q_row0 + v / p.G) * p.Hq + h * p.G + v % p.G) * 128 + lane * 4);
              }
            }
          }
#pragma unroll
          for (int i = 0; i < QB; ++i) {
            const int n = n0 + i;
            float f[4] = {__uint_as_float(raw[i].x << 16), __uint_as_float(raw[i].x & 0xffff0000u),
                          __uint_as_float(raw[i].y << 16), __uint_as_float(raw[i].y & 0xffff0000u)};
            const float am = fmaxf(fmaxf(fabsf(f[0]), fabsf(f[1])), fmaxf(fabsf(f[2]), fabsf(f[3])));
            const float amax = warp_max_f32(am);
            const bool bad = isnan(f[0]) || isnan(f[1]) || isnan(f[2]) || isnan(f[3]) || amax == -NEG_INF;
            // below 2^-90 the low piece loses bits of scores that are zero anyway
            const int e = max(-100, q8_exponent(amax));
            const float sc = exp2_int(-e);
            uint32_t a1, a2, b1, b2;
            q8_split(pk2(f[0] * sc, f[1] * sc), a1, a2);
            q8_split(pk2(f[2] * sc, f[3] * sc), b1, b2);
            const uint32_t off = (uint32_t)((((lane >> 2) ^ (n & 7)) << 4) + (lane & 3) * 4);
            *reinterpret_cast<uint32_t*>(qd + n * 128 + off) = a1 | (b1 << 16);
            *reinterpret_cast<uint32_t*>(qd + (NQP + n) * 128 + off) = a2 | (b2 << 16);
            // a vector that is not finite has no finite score: all of its output is NaN
            const bool any_bad = __any_sync(0xffffffffu, bad);
            if (lane == 0) cd[n] = any_bad ? __int_as_float(0x7fc00000) : p.scale_log2 * exp2_int(e);
          }
        }
        fence_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_qready[units & 3u]);
      ++units;
    }
    // the MMA warp's last commits land on these barriers before the CTA exits
    for (uint32_t k = (units > 2 ? units - 2 : 0); k < units; ++k)
      q8_wait(&bar_qfree[k & 1u], (k >> 1) & 1u, &s_abort, p.err);
  } else if (warp == 3) {
    // ------------------------------------------------------------ exponents
    // Word of a key: e_k, e_v of the (first) head, then of the pair's second head.
    // Loaded past L1 (the append may write neighbouring bytes), a tile pair ahead
    // of being stored; lane l takes keys l, l + 32, ...
    UnitIter itr = make_iter();
    uint32_t tt = 0;
    while (itr.next(p, S, u, r_lo, r_hi, ustart)) {
      const int h = u % p.Hkv;
      const int n_t = (r_hi - r_lo + 2 * kTcTile - 1) / (2 * kTcTile);
      const long long base = S.k_row0 * p.c.Hkv + (long long)(PAIR ? 2 * h : h) * p.c.max_seq;
      const signed char* kp = reinterpret_cast<const signed char*>(p.c.ke) + base;
      const signed char* vp = reinterpret_cast<const signed char*>(p.c.ve) + base;
      uint32_t w[8];
      auto load = [&](int t, uint32_t(&o)[8]) {
        need_rows(itr, min(r_hi, r_lo + (t + 1) * 2 * kTcTile));
        // all loads in flight at once: a key past the range reads the last one's
        int e[4][8] = {};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = min(r_lo + t * 2 * kTcTile + i * 32 + lane, r_hi - 1);
          e[0][i] = __ldcg(kp + key);
          e[1][i] = __ldcg(vp + key);
        }
        if (PAIR) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int key = p.c.max_seq + min(r_lo + t * 2 * kTcTile + i * 32 + lane, r_hi - 1);
            e[2][i] = __ldcg(kp + key);
            e[3][i] = __ldcg(vp + key);
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
          o[i] = (uint32_t)(e[0][i] & 255) | (uint32_t)(e[1][i] & 255) << 8 | (uint32_t)(e[2][i] & 255) << 16 |
                 (uint32_t)e[3][i] << 24;
      };
      load(0, w);
      for (int t = 0; t < n_t; ++t, ++tt) {
        uint32_t nx[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (t + 1 < n_t) load(t + 1, nx);
        const int slot = (int)(tt % C::EXP_RING);
        if (tt >= (uint32_t)C::EXP_RING) q8_wait(&bar_efree[slot], ((tt / C::EXP_RING) - 1) & 1u, &s_abort, p.err);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          exps[slot * 2 * kTcTile + i * 32 + lane] = w[i];
          w[i] = nx[i];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_efull[slot]);
      }
    }
  } else {
    // ------------------------------------------------------------ softmax warps
    const int sw = warp - 4;
    const int g = sw / (4 * H);         // group: pairs i with i % G == g
    const int sq = sw & 3;              // warp within its column slice
    const int col0 = ((sw >> 2) % H) * NL;  // first query column of this thread
    const int qd = warp & 3;            // TMEM lane quadrant this warp may access
    const int stid = tid - 128 - g * SMT;  // thread within the group
    const int my_row = qd * 32 + lane;  // key of either tile, then head dim, this thread owns
    const uint32_t tq = tmem + ((uint32_t)(qd * 32) << 16);
    unsigned char* pg = ps + g * C::P_BYTES;
    int* rp = s_rp[g];
    auto group_bar = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(1 + g), "n"(SMT) : "memory"); };
    auto all_bar = [&]() { asm volatile("bar.sync %0, %1;" ::"n"(1 + G), "n"(G * SMT) : "memory"); };
    UnitIter itr = make_iter();
    uint32_t it = 0, units = 0;  // it: tile pairs before this unit
    constexpr int NP = NL / 2;   // columns are worked on two at a time
    const f32x2 c16 = pk2(0.0625f, 0.0625f);
    // columns past the unit's vectors hold anything: an MMA column enters no other
    while (itr.next(p, S, u, r_lo, r_hi, ustart)) {
      const int h = u % p.Hkv, qg = u / p.Hkv;
      const int n_sub = (r_hi - r_lo + kTcTile - 1) / kTcTile;
      const int n_t = (n_sub + 1) >> 1;
      const UnitCols<PAIR, NQP> uc(p, S, qg);
      const int nvec = uc.nvec;
      if (nvec > NA && stid == 0) set_error(p.err, kErrBadRows);  // an item longer than the call's max_q
      const int c_first = (int)(ustart / share);
      const int c_last = (int)((ustart + S.k_len - 1) / share);
      const int n_contrib = p.invariant ? 1 : c_last - c_first + 1;
      int arrived = 0;
      // (the plan kernel clears the counters, so they are read after it only)
      if (n_contrib > 1 && stid == 0 && itr.waited) arrived = ld_relaxed_gpu(p.ws_cnt + c_first);

      if (p.row_pos != nullptr) {
        if (sq == 0 && lane < NL) {
          const int n = col0 + lane;
          rp[n] = n < nvec ? p.row_pos[(long long)(S.q_row0 + uc.vec(n) / p.G) * p.row_pos_stride] : -1;
        }
        group_bar();
      }
      q8_wait(&bar_qready[units & 3u], (units >> 2) & 1u, &s_abort, p.err);
      const float* csc = cscale + (units & 3u) * NQP + col0;
      // The running maximum of column col0 + j (j < NL) lives in lane j of every
      // softmax warp of the slice: what the exponentials subtract (8 below it) and the
      // pair's rescale factors reach the other lanes through shared memory.
      float m = NEG_INF;
      f32x2 lp[NP], oacc[NP];
#pragma unroll
      for (int j = 0; j < NP; ++j) lp[j] = oacc[j] = 0ull;
      auto add_o = [&](uint32_t i) {  // P.V of pair i joins O
        q8_wait(&bar_ofull[g], (i / G) & 1u, &s_abort, p.err);
        tc_fence_after();
        float o0[NL], o1[NL];
        tmem_cols<NL>(tq + (uint32_t)(C::O_COL + g * N + col0), o0);
        tmem_cols<NL>(tq + (uint32_t)(C::O_COL + g * N + NQP + col0), o1);
        tc_wait_ld();
        tc_fence_before();
#pragma unroll
        for (int j = 0; j < NP; ++j)
          oacc[j] = add2(oacc[j], fma2(pk2(o1[2 * j], o1[2 * j + 1]), c16, pk2(o0[2 * j], o0[2 * j + 1])));
      };
      // a per-head pair of values for the columns (2 j, 2 j + 1)
      auto by_head = [&](int j, float v0, float v1) {
        if constexpr (!PAIR) return pk2(v0, v0);
        return pk2(uc.head(col0 + 2 * j) ? v1 : v0, uc.head(col0 + 2 * j + 1) ? v1 : v0);
      };
      const int t0 = G == 1 ? 0 : (int)((it ^ (uint32_t)g) & 1u);  // this group's first pair
      for (int t = t0; t < n_t; t += G) {
        const uint32_t i = it + t;
        const int sb = (int)(i & 1u);
        const int k0 = r_lo + t * 2 * kTcTile;
        const int es = (int)(i % C::EXP_RING);
        q8_wait(&bar_efull[es], (i / C::EXP_RING) & 1u, &s_abort, p.err);
        const uint32_t ew[2] = {exps[es * 2 * kTcTile + my_row], exps[es * 2 * kTcTile + kTcTile + my_row]};
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_efree[es]);
        q8_wait(&bar_sfull[sb], (i >> 1) & 1u, &s_abort, p.err);
        tc_fence_after();
        f32x2 x[2][NP];
        {
          float hi[2][NL], lo[2][NL];
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            tmem_cols<NL>(tq + (uint32_t)((2 * sb + hf) * N + col0), hi[hf]);
            tmem_cols<NL>(tq + (uint32_t)((2 * sb + hf) * N + NQP + col0), lo[hf]);
          }
          tc_wait_ld();
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const float ka = exp2_int((int)(signed char)ew[hf]), kb = exp2_int((int)(signed char)(ew[hf] >> 16));
            const float va = (float)(signed char)(ew[hf] >> 8), vb = (float)(signed char)(ew[hf] >> 24);
#pragma unroll
            for (int j = 0; j < NP; ++j) {
              const f32x2 s = fma2(pk2(lo[hf][2 * j], lo[hf][2 * j + 1]), c16, pk2(hi[hf][2 * j], hi[hf][2 * j + 1]));
              const float2 cs = *reinterpret_cast<const float2*>(csc + 2 * j);
              x[hf][j] = fma2(mul2(s, by_head(j, ka, kb)), pk2(cs.x, cs.y), by_head(j, va, vb));
            }
          }
          // (after the scales are read: the Q warp may rewrite them once S is free)
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar_sfree[sb]);
        }
        // masking, as K2: nothing to do on a tile pair inside the unit and below the
        // causal frontier of the window's first row
        const int pair_last = k0 + 2 * kTcTile - 1;
        if (pair_last >= r_hi || col0 + NL > nvec || p.row_pos != nullptr || pair_last > S.k_len - S.q_len) {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const int key = k0 + hf * kTcTile + my_row;
            const int nlim = key < r_hi ? nvec : 0;
            const int thr = (key - (S.k_len - S.q_len)) * p.G;
#pragma unroll
            for (int j = 0; j < NP; ++j) {
              float y[2];
              up2(x[hf][j], y[0], y[1]);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int n = col0 + 2 * j + e;
                const bool see = n < nlim && (p.row_pos != nullptr ? key <= rp[n] : uc.vec(n) >= thr);
                y[e] = see ? y[e] : NEG_INF;
              }
              x[hf][j] = pk2(y[0], y[1]);
            }
          }
        }
        float* rb = red + (2 * g + ((i / G) & 1u)) * (4 * NQP);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          float a0, a1, b0, b1;
          up2(x[0][j], a0, a1);
          up2(x[1][j], b0, b1);
          const float r0 = warp_max_f32(fmaxf(a0, b0)), r1 = warp_max_f32(fmaxf(a1, b1));
          if (lane == 0) *reinterpret_cast<float2*>(rb + sq * NQP + col0 + 2 * j) = make_float2(r0, r1);
        }
        group_bar();
        if (t >= G) add_o(i - G);  // relative to the maximum before this pair; also frees P^T
        float* mw = mxs + sw * 32;
        float al = 1.f;
        if (lane < NL) {
          const int c = col0 + lane;
          const float mx = fmaxf(fmaxf(rb[c], rb[NQP + c]), fmaxf(rb[2 * NQP + c], rb[3 * NQP + c]));
          if (mx > m + 0.75f) {
            al = ex2_ftz(m - mx);
            m = mx;
          }
          mw[lane] = m == NEG_INF ? 0.f : 8.f - m;  // no key seen: exp2(-inf) = 0
          mw[16 + lane] = al;
        }
        const bool moved = __any_sync(0xffffffffu, al != 1.f);
        __syncwarp();
        if (moved) {
#pragma unroll
          for (int j = 0; j < NP; ++j) {
            const float2 aj = *reinterpret_cast<const float2*>(mw + 16 + 2 * j);
            lp[j] = mul2(lp[j], pk2(aj.x, aj.y));
            oacc[j] = mul2(oacc[j], pk2(aj.x, aj.y));
          }
        }
        if (pair_last >= r_hi && col0 == 0) {  // warp-uniform
          // rows past the range may hold anything: once the pair has landed, zero these keys' V rows
          q8_wait(&bar_vfull[i % VS], (i / VS) & 1u, &s_abort, p.err);
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            if (k0 + hf * kTcTile + my_row >= r_hi) {
              unsigned char* vrow = vts + (int)(i % VS) * C::PAIR_BYTES + (hf * kTcTile + my_row) * 128;
#pragma unroll
              for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(vrow + c * 16) = make_uint4(0, 0, 0, 0);
            }
          }
        }
        // weights 2^(t - M + 8); the denominator's leave the value scale out again.
        // (A pair of one tile: the other's are zero, and no MMA reads them.)
        uint32_t w1[2][(NL + 3) / 4], w2[2][(NL + 3) / 4];
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          const float2 mj = *reinterpret_cast<const float2*>(mw + 2 * j);
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const float ia = exp2_int(-(int)(signed char)(ew[hf] >> 8)), ib = exp2_int(-(int)(signed char)(ew[hf] >> 24));
            float d0, d1;
            up2(add2(x[hf][j], pk2(mj.x, mj.y)), d0, d1);
            const f32x2 w = pk2(ex2_ftz(d0), ex2_ftz(d1));
            lp[j] = fma2(w, by_head(j, ia, ib), lp[j]);
            uint32_t p1, p2;
            q8_split(w, p1, p2);
            if ((j & 1) == 0) {
              w1[hf][j / 2] = p1;
              w2[hf][j / 2] = p2;
            } else {
              w1[hf][j / 2] |= p1 << 16;
              w2[hf][j / 2] |= p2 << 16;
            }
          }
        }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const uint32_t rowo = (uint32_t)((hf * kTcTile + my_row) * C::P_ROWB);
          auto put = [&](int col, const uint32_t(&w)[(NL + 3) / 4]) {
            uint32_t off = rowo + (uint32_t)col;
            off ^= ((off >> 7) & ((1u << C::P_SWZ_BITS) - 1u)) << 4;
            if constexpr (NL == 16)
              *reinterpret_cast<uint4*>(pg + off) = make_uint4(w[0], w[1], w[2], w[3]);
            else if constexpr (NL == 8)
              *reinterpret_cast<uint2*>(pg + off) = make_uint2(w[0], w[1]);
            else if constexpr (NL == 4)
              *reinterpret_cast<uint32_t*>(pg + off) = w[0];
            else
              *reinterpret_cast<uint16_t*>(pg + off) = (uint16_t)w[0];
          };
          put(col0, w1[hf]);
          put(NQP + col0, w2[hf]);
        }
        fence_async_smem();
        group_bar();
        if (stid == 0) mbar_arrive(&bar_pfull[g]);
      }
      if (t0 < n_t) add_o(it + (uint32_t)(t0 + (n_t - 1 - t0) / G * G));
      it += n_t;
      ++units;

      // ---- column sums of the weights over the unit's keys
      float* lb = lred + (2 * g + (units & 1u)) * (4 * NQP);
      {
        float w[NL];
#pragma unroll
        for (int j = 0; j < NP; ++j) up2(lp[j], w[2 * j], w[2 * j + 1]);
        const float r = warp_col_sum<NL>(w, lane);
        if (lane < NL) lb[sq * NQP + col0 + reduced_col<NL>(lane)] = r;
      }
      group_bar();
      float mc[NL], lc[NL], oc[NL];
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const int n = col0 + j;
        mc[j] = __shfl_sync(0xffffffffu, m, j);
        lc[j] = lb[n] + lb[NQP + n] + lb[2 * NQP + n] + lb[3 * NQP + n];
      }
#pragma unroll
      for (int j = 0; j < NP; ++j) up2(oacc[j], oc[2 * j], oc[2 * j + 1]);
      if constexpr (G == 2) {
        // the second group hands its (m, l, O) over through shared memory (O in its own
        // P^T buffer, whose last P.V is done) and goes on to the next unit
        float* og = reinterpret_cast<float*>(ps + C::P_BYTES);
        if (g == 1) {
#pragma unroll
          for (int j = 0; j < NL; ++j) {
            og[j * kTcTile + my_row] = oc[j];
            if (my_row == 0) {
              ml[j] = mc[j];
              ml[NQP + j] = lc[j];
            }
          }
        }
        all_bar();
        if (g == 0) {
#pragma unroll
          for (int j = 0; j < NL; ++j) {
            const float m1 = ml[j], nm = fmaxf(mc[j], m1), ms = nm == NEG_INF ? 0.f : nm;
            const float wa = ex2_ftz(mc[j] - ms), wb = ex2_ftz(m1 - ms);
            lc[j] = lc[j] * wa + ml[NQP + j] * wb;
            oc[j] = oc[j] * wa + og[j * kTcTile + my_row] * wb;
            mc[j] = nm;
          }
        }
        all_bar();
        if (g == 1) continue;
      }
      const int dim = my_row;
      // output element of query column n held by this thread's O^T row, or -1
      auto out_at = [&](int n) -> long long {
        const int e = uc.head(n), v = uc.vec(n);
        const long long row = (long long)(S.q_row0 + v / p.G) * p.Hq + v % p.G;
        if (PAIR) return (dim >> 6) == e ? (row + (2 * h + e) * p.G) * 64 + (dim & 63) : -1;
        return (row + h * p.G) * 128 + dim;
      };
      auto put_out = [&](int n, float O, float L) {
        const long long oi = out_at(n);
        if (oi >= 0) static_cast<__nv_bfloat16*>(p.out)[oi] = __float2bfloat16_rn(L == 0.f ? 0.f : O / L);
      };
      if (n_contrib == 1) {
#pragma unroll
        for (int j = 0; j < NL; ++j)
          if (col0 + j < nvec) put_out(col0 + j, oc[j], lc[j]);
      } else {
        if (!itr.waited) {
          griddep_wait();
          itr.waited = true;
        }
        // 2: every other contributor had published when this CTA began the unit
        if (stid == 0) {
          s_flag = (arrived == n_contrib - 1) ? 2 : 0;
          if (s_flag == 2) fence_acq_rel_gpu();
        }
        group_bar();
        if (s_flag != 2) {
          const int slot = (ustart < a) ? 2 * (int)blockIdx.x : 2 * (int)blockIdx.x + 1;
          float* pb = p.ws_part + (size_t)slot * C::PART_FLOATS;
#pragma unroll
          for (int j = 0; j < NL; ++j) {
            if (col0 + j < nvec) {
              if (dim == 0) {
                pb[col0 + j] = mc[j];
                pb[NQP + col0 + j] = lc[j];
              }
              pb[2 * NQP + (col0 + j) * 128 + dim] = oc[j];
            }
          }
          __threadfence();
          group_bar();
          if (stid == 0) {
            const int prev = atomicAdd(p.ws_cnt + c_first, 1);
            s_flag = (prev == n_contrib - 1) ? 1 : 0;
          }
          group_bar();
        }
        if (s_flag) {
          __threadfence();
          // online merge in key order, whoever arrives last
          const int k_own = (int)blockIdx.x - c_first;
          float M[NL], Ls[NL], acc[NL];
#pragma unroll
          for (int j = 0; j < NL; ++j) {
            M[j] = NEG_INF;
            Ls[j] = 0.f;
            acc[j] = 0.f;
          }
          for (int k = 0; k < n_contrib; ++k) {
            const int cc = c_first + k;
            const float* base = p.ws_part + (size_t)(k == 0 ? 2 * cc + 1 : 2 * cc) * C::PART_FLOATS;
            float mk[NL], lk[NL], ok[NL];
#pragma unroll
            for (int j = 0; j < NL; ++j) {
              const int n = col0 + j;
              if (k == k_own) {
                mk[j] = mc[j];
                lk[j] = lc[j];
                ok[j] = oc[j];
              } else {
                mk[j] = n < nvec ? ld_cg_f32(base + n) : NEG_INF;
                lk[j] = n < nvec ? ld_cg_f32(base + NQP + n) : 0.f;
                ok[j] = n < nvec ? ld_cg_f32(base + 2 * NQP + n * 128 + dim) : 0.f;
              }
            }
#pragma unroll
            for (int j = 0; j < NL; ++j) {
              const float nm = fmaxf(M[j], mk[j]);
              const float ms = nm == NEG_INF ? 0.f : nm;
              const float wa = fast_exp2(M[j] - ms), wb = fast_exp2(mk[j] - ms);
              Ls[j] = Ls[j] * wa + lk[j] * wb;
              acc[j] = acc[j] * wa + ok[j] * wb;
              M[j] = nm;
            }
          }
#pragma unroll
          for (int j = 0; j < NL; ++j)
            if (col0 + j < nvec) put_out(col0 + j, acc[j], Ls[j]);
        }
        if (s_flag && stid == 0) p.ws_cnt[c_first] = 0;
        group_bar();  // s_flag is rewritten by the next unit
      }
    }
  }

  if (self) griddep_wait();  // stream order for what follows, whether or not this CTA needed the plan
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS) : "memory");
  }
}

}  // namespace wfd
