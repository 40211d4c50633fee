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
//   Q: a bf16 value has 8 significant bits, so both pieces together are exact until
//      the low one underflows: off by at most 2^-14 where the row's largest element
//      is 224 to 448, 2^-21.8 of it.
//   P: each piece is off by at most half a step, 2^-4 of its value: 2^-8 together,
//      what rounding P to bf16 costs.  A step's weights are scaled by that step's own
//      largest, 2^8 there, and O of the step joins the unit's in fp32
//      under 2^(step's maximum - M): where the low piece underflows, below 2^-14 of
//      the step's largest weight, a weight is off by at most 2^-22 of it, so the
//      256 keys of a step lose 2^-14 of it together, however many steps there are.
//      (Scaled by the running maximum instead, weights below 2^-22 of it were zero:
//      one key 15 nats above a flat prefix hid all of the rest.)  The weights' sum
//      is taken of the unrounded weights in fp32.
// The minimum N of the instruction leaves room for the second piece, so a tile of
// 32 KB takes 8 MMAs, half of the bf16 kernel's for the same bytes.
//     S^T[128 keys x 2 NQP] = K . [Q1 | Q2]^T         (K-major, 4 k-steps of 32 bytes)
//     O^T[128 dims x 2 NQP] += V^T . [P1 | P2]^T       (both MN-major, 4 k-steps of 32 keys)
// Scales: a key's 2^{e_k} multiplies its finished score; its value scale joins the
// weight, t = s + e_v in log2 units, so that the maxima are taken of t and the
// weights stay within e4m3's range: w = 2^(t - m + 8) <= 2^8, m the step's maximum.
// Sums are held relative to M, a maximum that moves only when a step's exceeds it by
// 16: what it leaves, w 2^(m - M) |code| <= 2^33 a key, is far inside fp32.  The
// denominator needs 2^(s - M + 8) = w 2^{-e_v} 2^(m - M); |e_v| <= 32 keeps that above
// the fp32 underflow for every key that matters.
//
// What bounds it: HBM; a step of 256 keys (64 KB of K and V) takes 1.5 us of an SM's
// share of the copy bandwidth.  Behind it come two chains:
//   * the softmax of a step is a dependent chain through two named barriers (1.5 us
//     by itself).  Up to 16 query columns, two CTAs share an SM, each with a pipeline
//     and a share of the work of its own, so that two chains, and the ends of units
//     (output rows written or merged), overlap; a thread works on two keys, one of
//     either tile, so that the chain is paid once per 64 KB.  32 columns need the
//     registers of one CTA, whose 16 softmax warps are bound by instruction issue;
//   * TMA keeps about 100 KB an SM in flight: 192 KB measured 12 % less bandwidth, and
//     tensor maps that promote to 256 bytes fetch the neighbouring head's half of each
//     pair of lines for nothing (53 % more DRAM traffic).
//
// Warp roles: 0 TMA producer; 1 TMEM owner and MMA issuer; 2 the Q operand of the next
// unit; 3 the keys' exponents; 4.. softmax.  Work split, merging and the self-planned
// start are K2's.  Every wait is bounded; no multicast, no cluster.
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

// CTAs an SM holds, column slices of the softmax (4 warps each), threads of a CTA.
__host__ __device__ constexpr int q8_ctas(int na) { return na <= 16 ? 2 : 1; }
__host__ __device__ constexpr int q8_slices(int na) { return na <= 16 ? 1 : 4; }
__host__ __device__ constexpr int q8_tc_threads(int na) { return 128 + 128 * q8_slices(na); }

template <int NQP, int NA>
struct Q8Cfg {
  static constexpr int N = 2 * NQP;                  // MMA columns: both pieces
  static constexpr int CTAS = q8_ctas(NA);
  static constexpr int T = NA == 16 ? 1 : 2;         // 128-key tiles of a step (16 columns a thread: one, for registers)
  static constexpr int TILE_BYTES = kTcTile * 128;
  static constexpr int STEP_BYTES = T * TILE_BYTES;  // K (or V) of a step
  // Rings of steps.  A K step is done with after S (of which there are as many
  // buffers), a V step only after the softmax and P.V.
  static constexpr int KS = CTAS == 2 && T == 2 ? 1 : 2;
  static constexpr int VS = CTAS == 2 && T == 2 ? 2 : T == 2 ? 3 : 4;
  static constexpr int Q_BYTES = N * 128;
  static constexpr int QB = CTAS == 2 ? 1 : 2;       // Q operand buffers
  static constexpr int P_ROWB = N;                   // one key's row of P^T
  static constexpr int P_BYTES = T * kTcTile * P_ROWB;
  static constexpr int P_SWZ_BITS = NQP == 16 ? 1 : 2;     // 32- / 64-byte swizzle
  static constexpr uint64_t P_LAYOUT = NQP == 16 ? 6 : 4;
  static constexpr int P_ATOM = 8 * P_ROWB;
  static constexpr int RED_FLOATS = 2 * 4 * NQP;     // double-buffered, 4 warps a slice
  static constexpr int WARPS = 4 * q8_slices(NA);    // softmax warps
  static constexpr int ER = 2;                       // exponent ring, in steps
  static constexpr int S_COL = 0;                    // S^T buffer s, tile hf: (T s + hf) N
  static constexpr int O_COL = KS * T * N;           // O^T
  static constexpr int TMEM_COLS = O_COL + N <= 128 ? 128 : O_COL + N <= 256 ? 256 : 512;
  static constexpr int PART_FLOATS = NQP * (128 + 2);
  static_assert(CTAS * TMEM_COLS <= 512 && O_COL + N <= TMEM_COLS, "TMEM columns");
};

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

// Work is counted in chunks of 256 keys of a unit (segment, query group, kv head),
// the last of a unit possibly shorter: a piece of a few keys takes as long as a whole
// step and is one more to merge, so units are cut at chunk borders only.  (Shares in
// keys, as K2's, took 36 us for 256 units of 65 keys, chunks 13.4 us.)
constexpr int kQ8Chunk256 = 256;
__device__ __forceinline__ int q8_chunks(int k_len) { return (k_len + kQ8Chunk256 - 1) / kQ8Chunk256; }

// A CTA's walk over its share [pos, end) of the work, in chunks: the pieces [r_lo,
// r_hi) (keys) of units, in order; a unit that follows in the same segment costs no
// division and no load.
struct Q8Stream {
  long long pos, end, base, nbase, ustart;
  Seg S;
  int seg, u, uc, r_lo, r_hi;  // uc: chunks of a unit of this segment
  int t, n;        // step of the piece, steps of the piece
  uint32_t step, unit;  // steps and units so far (the current one not counted)
  bool fresh;      // u not yet known in this segment
  bool live;
  bool waited;     // griddep_wait() executed by this thread

  __device__ __forceinline__ long long seg_base(const VerifyParams& p, int i) const {
    return i <= p.n_segs - 1 ? (long long)p.Hkv * p.prefix[i] : 0x7fffffffffffffffll;
  }
  __device__ __forceinline__ bool next_unit(const VerifyParams& p, int step_keys) {
    for (;;) {
      if (pos >= end) {
        live = false;
        return false;
      }
      if (pos >= nbase) {
        if (!waited) {  // the segment table and prefix are the plan kernel's outputs
          griddep_wait();
          waited = true;
        }
        while (pos >= nbase) {
          ++seg;
          base = nbase;
          nbase = seg_base(p, seg + 1);
        }
        S = p.segs[seg];
        fresh = true;
      }
      if (fresh) {
        uc = q8_chunks(S.k_len);
        u = pos == base ? 0 : (int)((pos - base) / uc);
        ustart = base + (long long)u * uc;
        fresh = false;
      } else {
        ++u;
        ustart += uc;
      }
      const long long uend = ustart + uc;
      if (p.invariant) {
        const bool mine = ustart >= pos;  // else it began in the share before this one, which takes it whole
        pos = uend;
        if (!mine) continue;
        r_lo = 0;
        r_hi = S.k_len;
      } else {
        r_lo = (int)(pos - ustart) * kQ8Chunk256;
        pos = uend < end ? uend : end;
        r_hi = min(S.k_len, (int)(pos - ustart) * kQ8Chunk256);
      }
      t = 0;
      n = (r_hi - r_lo + step_keys - 1) / step_keys;
      return true;
    }
  }
  // to the next step; returns whether there is one
  __device__ __forceinline__ bool advance(const VerifyParams& p, int step_keys) {
    ++step;
    if (++t < n) return true;
    ++unit;
    return next_unit(p, step_keys);
  }
};

// Where the CTA's share starts: from the item table itself (K2's self-planned start:
// the plan kernel may still be running).  Called by the whole CTA.
struct SelfStart {
  long long wtot[32];
  Seg S0;
  long long base0, nbase0;
  int seg0, slot0, seq0, minpos;
};
__device__ __forceinline__ void share_of(long long total, long long& share, long long& a, long long& b) {
  share = max((total + gridDim.x - 1) / gridDim.x, 1ll);
  a = min(total, (long long)blockIdx.x * share);
  b = min(total, a + share);
}
template <int THREADS>
__device__ __forceinline__ void self_start(const VerifyParams& p, SelfStart& sh, long long& share, long long& a,
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
      slot_segment(p, my[k], s);
      w[k] = (long long)s.n_qg * q8_chunks(s.k_len);
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
  share_of((long long)p.Hkv * all, share, a, b);
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
}

// Per softmax warp and column, of a step: what the exponents add, the factor of what
// the unit holds (1 unless M moved), the factor 2^(m - M) of what the step adds (of
// the last two steps: O joins one step late).
enum : int { kMxSub = 0, kMxMove = 16, kMxStep = 32 };
constexpr float kQ8Lead = 16.f;  // how far a step's maximum may exceed M

// Shared memory besides the tiles.
template <typename C, int NQP>
struct Q8Shared {
  uint32_t exps[C::ER][C::T * kTcTile];  // a step's exponents, one word a key
  float red[2][4][NQP];                  // column maxima of each warp
  float lred[2][4][NQP];                 // column sums
  float cscale[4][NQP];                  // score scale of each column, per unit
  float mx[C::WARPS][4][16];             // per softmax warp: kMxSub, kMxMove, kMxStep (two steps')
  uint64_t kfull[C::KS], vfull[C::VS], vempty[C::VS];
  uint64_t sfull[C::KS], sfree[C::KS];   // S of a step complete (its K free), and read by the softmax
  uint64_t pfull, ofull;                 // P written (so the O of the step before is read), P.V complete
  uint64_t qready[4], qfree[C::QB];      // a unit's Q operand and column scales written, its S MMAs done
  uint64_t efull[C::ER], efree[C::ER];   // a step's exponents written, and read by every softmax warp
  uint64_t drain;
  SelfStart start;
  uint32_t tmem;
  int vslot[C::ER];                      // where the step's V tiles are: slot, phase parity << 8
  int rp[NQP];                           // gapped windows: each query column's row position
  int abort;
  int flag;
};
template <int NQP, int NA>
constexpr int q8_smem() {
  using C = Q8Cfg<NQP, NA>;
  constexpr int bytes = (C::KS + C::VS) * C::STEP_BYTES + C::QB * C::Q_BYTES + C::P_BYTES + (int)sizeof(Q8Shared<C, NQP>);
  static_assert(C::CTAS * (bytes + 1024) <= 233472 && bytes <= 232448, "shared memory of an SM");
  return bytes;
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
__global__ void __launch_bounds__(q8_tc_threads(NA), q8_ctas(NA))
    q8_tc_kernel(const __grid_constant__ Q8Maps maps, const Q8AttnParams p) {
  using C = Q8Cfg<NQP, NA>;
  constexpr int T = C::T, KS = C::KS, VS = C::VS, N = C::N, ER = C::ER, QB = C::QB;
  constexpr int STEP = T * kTcTile;  // keys of a step
  constexpr int THREADS = q8_tc_threads(NA);
  constexpr int H = q8_slices(NA);   // column slices (4 warps each)
  constexpr int NL = NA / H;         // query columns per softmax thread
  constexpr int NP = NL / 2;         // ... worked on two at a time
  constexpr int SMT = 128 * H;       // softmax threads
  static_assert(NL == 2 || NL == 4 || NL == 8 || NL == 16, "columns per softmax thread");
  static_assert(NA <= NQP, "active query columns");
  const float NEG_INF = -__int_as_float(0x7f800000);

  extern __shared__ __align__(1024) unsigned char q8_raw[];
  unsigned char* kts = q8_raw;                               // KS steps of K
  unsigned char* vts = kts + KS * C::STEP_BYTES;             // VS steps of V
  unsigned char* qs = vts + VS * C::STEP_BYTES;              // QB x Q operand (K-major, 128B swizzle)
  unsigned char* ps = qs + QB * C::Q_BYTES;                  // P^T operand of a step (MN-major)
  Q8Shared<C, NQP>& sh = *reinterpret_cast<Q8Shared<C, NQP>*>(ps + C::P_BYTES);
  volatile int* abort_flag = &sh.abort;
  // the swizzled tiles rely on the declared alignment (no room is kept to make up for it)
  if ((smem_u32(q8_raw) & 1023u) != 0) {
    set_error(p.err, kErrTimeout);
    return;
  }

  const int tid = threadIdx.x, warp = (int)uniform((uint32_t)tid >> 5), lane = tid & 31;
  const bool self = p.items != nullptr;
  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.k[2 - T])) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.v[2 - T])) : "memory");
    for (int s = 0; s < KS; ++s) {
      mbar_init(&sh.kfull[s], 1);
      mbar_init(&sh.sfull[s], 1);
      mbar_init(&sh.sfree[s], 4 * H);
    }
    for (int s = 0; s < VS; ++s) {
      mbar_init(&sh.vfull[s], 1);
      mbar_init(&sh.vempty[s], 1);
    }
    mbar_init(&sh.pfull, 1);
    mbar_init(&sh.ofull, 1);
    for (int s = 0; s < 4; ++s) mbar_init(&sh.qready[s], 1);
    for (int s = 0; s < QB; ++s) mbar_init(&sh.qfree[s], 1);
    for (int s = 0; s < ER; ++s) {
      mbar_init(&sh.efull[s], 1);
      mbar_init(&sh.efree[s], 4 * H);
    }
    mbar_init(&sh.drain, 1);
    fence_mbar_init();
    sh.abort = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                 "r"(C::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (!self) griddep_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;

  long long share, a, b;
  if (self)
    self_start<THREADS>(p, sh.start, share, a, b);
  else
    share_of((long long)p.Hkv * p.prefix[p.n_segs], share, a, b);
  // every role walks the same steps
  Q8Stream s;
  s.pos = a;
  s.end = b;
  s.t = s.n = 0;
  s.step = s.unit = 0;
  s.fresh = true;
  s.waited = !self;
  s.live = a < b;
  if (s.live) {
    if (self) {
      s.S = sh.start.S0;
      s.base = sh.start.base0;
      s.nbase = sh.start.nbase0;
      s.seg = sh.start.seg0;
    } else {
      const CtaStart cs = p.start[blockIdx.x];
      s.S = cs.S;
      s.base = cs.base;
      s.nbase = cs.nbase;
      s.seg = cs.seg;
    }
    s.next_unit(p, STEP);
  }
  // before reading cache rows (or their exponents) below `end` of the current
  // segment: the plan kernel's append may write rows from minpos on
  auto need_rows = [&](int end) {
    if (!s.waited && (s.seg != sh.start.seg0 || end > sh.start.minpos)) {
      griddep_wait();
      s.waited = true;
    }
  };

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    uint32_t n_k = 0, n_v = 0;      // steps whose loads were issued (prefixes of the sequence: issue stops at an abort)
    uint32_t ks = 0, vs = 0, kp = 0, vp = 0;  // ring slots and phases
    while (s.live) {
      need_rows(s.r_lo + (s.t + 1) * STEP);
      const int h = s.u % p.Hkv;
      const int row = (int)(s.S.k_row0 + p.k_row_offset + s.r_lo + (long long)s.t * STEP);
      // a last step of few keys loads only those, in boxes of 128 / 64 / 32 / 16 / 8
      // rows; what the stage holds past them is masked (V: zeroed)
      const int left = s.r_hi - s.r_lo - s.t * STEP;
      const int nr = left > STEP - 32 ? STEP : ((left + 7) & ~7);
      auto load = [&](unsigned char* dst, const CUtensorMap* m, uint64_t* bar) {
        mbar_arrive_expect_tx(bar, (uint32_t)(nr * 128));
        if (nr == STEP) {
          tma_load_3d(dst, m + (2 - T), 0, h, row, bar);
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
      // (the K ring is as deep as S's: the S of step - KS complete frees its K)
      bool go = s.step >= (uint32_t)KS ? q8_wait(&sh.sfull[ks], kp ^ 1u, abort_flag, p.err) : !*abort_flag;
      go = __all_sync(0xffffffffu, go);
      if (go && lane == 0) {
        load(kts + ks * C::STEP_BYTES, maps.k, &sh.kfull[ks]);
        n_k = s.step + 1;
        if (p.fail_waits && n_k == 1) {  // test hook: give up with this copy in flight
          set_error(p.err, kErrTimeout);
          *abort_flag = 1;
        }
      }
      __syncwarp();
      go = s.step >= (uint32_t)VS ? q8_wait(&sh.vempty[vs], vp ^ 1u, abort_flag, p.err) : !*abort_flag;
      go = __all_sync(0xffffffffu, go);
      if (go && lane == 0) {
        load(vts + vs * C::STEP_BYTES, maps.v, &sh.vfull[vs]);
        n_v = s.step + 1;
      }
      __syncwarp();
      if (++ks == KS) {
        ks = 0;
        kp ^= 1u;
      }
      if (++vs == VS) {
        vs = 0;
        vp ^= 1u;
      }
      s.advance(p, STEP);
    }
    // the MMA warp's commits land on these barriers before the CTA exits
    for (uint32_t j = (s.step > (uint32_t)VS ? s.step - VS : 0); j < s.step; ++j)
      q8_wait(&sh.vempty[j % VS], (j / VS) & 1u, abort_flag, p.err);
    // copies in flight land before the CTA exits, also after an abort
    if (lane == 0) {
      for (uint32_t j = (n_k > (uint32_t)KS ? n_k - KS : 0); j < n_k; ++j)
        if (!mbar_wait_bounded(&sh.kfull[j % KS], (j / KS) & 1u)) set_error(p.err, kErrTimeout);
      for (uint32_t j = (n_v > (uint32_t)VS ? n_v - VS : 0); j < n_v; ++j)
        if (!mbar_wait_bounded(&sh.vfull[j % VS], (j / VS) & 1u)) set_error(p.err, kErrTimeout);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    // S in order, ahead of the softmax; P.V as soon as a step's weights are there.
    constexpr uint32_t IDESC_S = q8_idesc(N, false, false);
    constexpr uint32_t IDESC_PV = q8_idesc(N, true, true);
    const uint32_t q_addr = smem_u32(qs), p_addr = smem_u32(ps), k_addr = smem_u32(kts), v_addr = smem_u32(vts);
    const uint32_t tm = uniform(tmem);
    uint32_t ks = 0, kp = 0;           // of S's step
    uint32_t pv = 0, pvs = 0, pvp = 0; // P.V issued so far, its V slot and phase
    uint32_t two_tiles = 0;            // of the steps pv, pv + 1, ..: whether they have a second tile
    // P.V of the next step, if its weights and its V tiles are there (last: waits)
    auto try_pv = [&](uint32_t steps, bool last) -> bool {
      if (pv == steps) return false;
      bool go = __all_sync(0xffffffffu, mbar_test_wait(&sh.pfull, pv & 1u) && mbar_test_wait(&sh.vfull[pvs], pvp));
      if (!go && !last) return false;
      if (!go) {
        go = q8_wait(&sh.pfull, pv & 1u, abort_flag, p.err);
        go = q8_wait(&sh.vfull[pvs], pvp, abort_flag, p.err) && go;
      }
      const bool two = uniform(two_tiles & 1u) != 0;
      tc_fence_after();
      const uint32_t v0 = uniform(v_addr + pvs * C::STEP_BYTES);
      if (go && elect_lane()) {
        const uint32_t o0 = tm + (uint32_t)C::O_COL;
        // k-step j: 32 keys, four 8-row groups of V and of P^T
#pragma unroll
        for (int j = 0; j < 4; ++j)
          umma_f8(o0, umma_desc(v0 + j * 4096, 16, 1024, 2),
                  umma_desc(p_addr + j * 4 * C::P_ATOM, 16, C::P_ATOM, C::P_LAYOUT), IDESC_PV, j > 0 ? 1u : 0u);
        if (T == 2 && two) {
#pragma unroll
          for (int j = 4; j < 8; ++j)
            umma_f8(o0, umma_desc(v0 + j * 4096, 16, 1024, 2),
                    umma_desc(p_addr + j * 4 * C::P_ATOM, 16, C::P_ATOM, C::P_LAYOUT), IDESC_PV, 1u);
        }
        umma_commit(&sh.ofull);
        umma_commit(&sh.vempty[pvs]);
      }
      __syncwarp();
      two_tiles >>= 1;
      ++pv;
      if (++pvs == VS) {
        pvs = 0;
        pvp ^= 1u;
      }
      return true;
    };
    while (s.live) {
      const uint32_t qpar = (s.unit >> 2) & 1u, spar = ((s.step / KS) & 1u) ^ 1u;
      bool go = false;
      for (uint32_t n = 0; n < kSpinLimit; ++n) {  // (every exit by a vote)
        go = __all_sync(0xffffffffu, mbar_test_wait(&sh.kfull[ks], kp) &&
                                         (s.step < (uint32_t)KS || mbar_test_wait(&sh.sfree[ks], spar)) &&
                                         (s.t > 0 || mbar_test_wait(&sh.qready[s.unit & 3u], qpar)));
        if (go) break;
        if (!try_pv(s.step, false) && __any_sync(0xffffffffu, *abort_flag != 0)) break;
      }
      if (!go) q8_wait(&sh.kfull[ks], kp, abort_flag, p.err);  // an abort, or the spin limit
      tc_fence_after();
      const int left = s.r_hi - s.r_lo - s.t * STEP;
      const bool two = uniform(left > kTcTile) != 0;
      const uint32_t qb = s.unit % QB;
      const uint32_t k0 = uniform(k_addr + ks * C::STEP_BYTES);
      const uint32_t qa = uniform(q_addr + qb * C::Q_BYTES);
      const uint32_t d0 = uniform(tm + ks * (uint32_t)(T * N));
      if (go && elect_lane()) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // 32 bytes of the row; the tiles are independent accumulators
          umma_f8(d0, umma_desc(k0 + j * 32, 16, 1024, 2), umma_desc(qa + j * 32, 16, 1024, 2), IDESC_S,
                  j > 0 ? 1u : 0u);
          if (T == 2 && two)
            umma_f8(d0 + N, umma_desc(k0 + C::TILE_BYTES + j * 32, 16, 1024, 2), umma_desc(qa + j * 32, 16, 1024, 2),
                    IDESC_S, j > 0 ? 1u : 0u);
        }
        umma_commit(&sh.sfull[ks]);
        if (s.t == s.n - 1) umma_commit(&sh.qfree[qb]);  // the unit's Q buffer may be rewritten
      }
      __syncwarp();
      two_tiles |= (two ? 1u : 0u) << (s.step - pv);
      if (++ks == KS) {
        ks = 0;
        kp ^= 1u;
      }
      s.advance(p, STEP);
    }
    while (try_pv(s.step, true)) {
    }
    // every MMA complete before TMEM is freed and the CTA exits, also after an abort
    if (elect_lane()) {
      umma_commit(&sh.drain);
      if (!mbar_wait_bounded(&sh.drain, 0)) set_error(p.err, kErrTimeout);
    }
    __syncwarp();
  } else if (warp == 2) {
    // ------------------------------------------------------------ Q operand
    // Lane l holds bytes 4l..4l+3 of a 128-byte row.  Rows n and NQP + n: the two
    // pieces of query vector n.  An operand buffer is rewritten once the S MMAs of its
    // unit are done; the column scales and barriers have four turns, since the softmax
    // may still be a unit behind the MMA warp.
    const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.q);
    while (s.live) {
      const int h = s.u % p.Hkv, qg = s.u / p.Hkv;
      const uint32_t w = s.unit, qb = w % QB;
      const UnitCols<PAIR, NQP> uc(p, s.S, qg);
      unsigned char* qd = qs + qb * C::Q_BYTES;
      float* cd = sh.cscale[w & 3u];
      constexpr int NB = NA < 8 ? NA : 8;  // vectors loaded at once
      uint2 raw[NB];
      auto load = [&](int n0) {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const int n = n0 + i;
          raw[i] = make_uint2(0, 0);
          if (n < uc.nvec) {
            const int e = uc.head(n), v = uc.vec(n);
            const long long row = (long long)(s.S.q_row0 + v / p.G) * p.Hq + v % p.G;
            if (PAIR) {
              if ((lane >> 4) == e)
                raw[i] = *reinterpret_cast<const uint2*>(q + (row + (2 * h + e) * p.G) * 64 + (lane & 15) * 4);
            } else {
              raw[i] = *reinterpret_cast<const uint2*>(q + (row + h * p.G) * 128 + lane * 4);
            }
          }
        }
      };
      load(0);  // on its way while the buffer is still in use
      bool go = w >= (uint32_t)QB ? q8_wait(&sh.qfree[qb], ((w / QB) - 1) & 1u, abort_flag, p.err) : !*abort_flag;
      go = __all_sync(0xffffffffu, go);
      if (go) {
        for (int n0 = 0; n0 < NA; n0 += NB) {
          if (n0 > 0) load(n0);
#pragma unroll
          for (int i = 0; i < NB; ++i) {
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
      if (lane == 0) mbar_arrive(&sh.qready[w & 3u]);
      s.step += (uint32_t)s.n;
      ++s.unit;
      s.next_unit(p, STEP);
    }
    // the MMA warp's last commits land on these barriers before the CTA exits
    for (uint32_t k = (s.unit > (uint32_t)QB ? s.unit - QB : 0); k < s.unit; ++k)
      q8_wait(&sh.qfree[k % QB], (k / QB) & 1u, abort_flag, p.err);
  } else if (warp == 3) {
    // ------------------------------------------------------------ exponents
    // Word of a key: e_k, e_v of the (first) head, then of the pair's second head.
    // Loaded past L1 (the append may write neighbouring bytes), a step ahead of being
    // stored; lane l takes keys l, l + 32, ...  A key past the range reads the last one's.
    constexpr int NK = STEP / 32;
    uint32_t w[NK];
    uint32_t vs = 0, vp = 0, held = 0;  // V slot of the next step to load; of the step held in w
    auto store = [&](uint32_t i) {      // step i, held in w
      const int slot = (int)(i % ER);
      if (i >= (uint32_t)ER) q8_wait(&sh.efree[slot], ((i / ER) - 1) & 1u, abort_flag, p.err);
#pragma unroll
      for (int k = 0; k < NK; ++k) sh.exps[slot][k * 32 + lane] = w[k];
      if (lane == 0) sh.vslot[slot] = (int)held;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.efull[slot]);
    };
    while (s.live) {
      const int h = s.u % p.Hkv;
      const int k0 = s.r_lo + s.t * STEP;
      need_rows(min(s.r_hi, k0 + STEP));
      const long long base = s.S.k_row0 * p.c.Hkv + (long long)(PAIR ? 2 * h : h) * p.c.max_seq;
      const signed char* kp = reinterpret_cast<const signed char*>(p.c.ke) + base;
      const signed char* vq = reinterpret_cast<const signed char*>(p.c.ve) + base;
      int e[4][NK] = {};
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        const int key = min(k0 + i * 32 + lane, s.r_hi - 1);
        e[0][i] = __ldcg(kp + key);
        e[1][i] = __ldcg(vq + key);
        if (PAIR) {
          e[2][i] = __ldcg(kp + p.c.max_seq + key);
          e[3][i] = __ldcg(vq + p.c.max_seq + key);
        }
      }
      if (s.step > 0) store(s.step - 1);
#pragma unroll
      for (int i = 0; i < NK; ++i)
        w[i] = (uint32_t)(e[0][i] & 255) | (uint32_t)(e[1][i] & 255) << 8 | (uint32_t)(e[2][i] & 255) << 16 |
               (uint32_t)e[3][i] << 24;
      held = vs | vp << 8;
      if (++vs == VS) {
        vs = 0;
        vp ^= 1u;
      }
      s.advance(p, STEP);
    }
    if (s.step > 0) store(s.step - 1);
  } else {
    // ------------------------------------------------------------ softmax warps
    const int sw = warp - 4;
    const int sq = sw & 3;                  // warp within its column slice
    const int col0 = (sw >> 2) * NL;        // first query column of this thread
    const int qd = warp & 3;                // TMEM lane quadrant this warp may access
    const int stid = tid - 128;
    const int my_row = qd * 32 + lane;      // key of a tile, then head dim, this thread owns
    const uint32_t tq = tmem + ((uint32_t)(qd * 32) << 16);
    const int vid = (int)blockIdx.x;
    float* mw = sh.mx[sw][0];
    const f32x2 c16 = pk2(0.0625f, 0.0625f);
    // columns past the unit's vectors hold anything: an MMA column enters no other
    while (s.live) {
      const int h = s.u % p.Hkv, qg = s.u / p.Hkv;
      const Seg S = s.S;
      const int r_lo = s.r_lo, r_hi = s.r_hi, n_t = s.n;
      const long long ustart = s.ustart;
      const UnitCols<PAIR, NQP> uc(p, S, qg);
      const int nvec = uc.nvec;
      if (nvec > NA && stid == 0) set_error(p.err, kErrBadRows);  // an item longer than the call's max_q
      // the shares that hold keys of this unit
      const int c_first = ustart >= a ? vid : (int)(ustart / share);
      const int c_last = ustart + s.uc <= a + share ? vid : (int)((ustart + s.uc - 1) / share);
      const int n_contrib = p.invariant ? 1 : c_last - c_first + 1;
      int arrived = 0;
      // (the plan kernel clears the counters, so they are read after it only)
      if (n_contrib > 1 && stid == 0 && s.waited) arrived = ld_relaxed_gpu(p.ws_cnt + c_first);
      int frontier = S.k_len - S.q_len;  // the first row's position: keys up to it need no mask
      if (p.row_pos != nullptr) {
        if (sq == 0 && lane < NL) {
          const int n = col0 + lane;
          sh.rp[n] = n < nvec ? p.row_pos[(long long)(S.q_row0 + uc.vec(n) / p.G) * p.row_pos_stride] : -1;
        }
        softmax_bar<SMT>();
        // of these columns, the first row's position
        frontier = __reduce_min_sync(0xffffffffu, lane < NL && col0 + lane < nvec ? sh.rp[col0 + lane] : 0x7fffffff);
      }
      q8_wait(&sh.qready[s.unit & 3u], (s.unit >> 2) & 1u, abort_flag, p.err);
      const float* csc = sh.cscale[s.unit & 3u] + col0;
      // M of column col0 + j (j < NL) lives in lane j of every softmax warp of the
      // slice; a step's factors reach the other lanes through shared memory.
      float m = NEG_INF;
      f32x2 lp[NP], oacc[NP];
#pragma unroll
      for (int j = 0; j < NP; ++j) lp[j] = oacc[j] = 0ull;
      auto add_o = [&](uint32_t i, int t) {  // P.V of step i, the unit's t, joins O
        const float* ms = mw + kMxStep + 16 * (t & 1);
        q8_wait(&sh.ofull, i & 1u, abort_flag, p.err);
        tc_fence_after();
        float o0[NL], o1[NL];
        tmem_cols<NL>(tq + (uint32_t)(C::O_COL + col0), o0);
        tmem_cols<NL>(tq + (uint32_t)(C::O_COL + NQP + col0), o1);
        tc_wait_ld();
        tc_fence_before();
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          const float2 sj = *reinterpret_cast<const float2*>(ms + 2 * j);
          oacc[j] = fma2(fma2(pk2(o1[2 * j], o1[2 * j + 1]), c16, pk2(o0[2 * j], o0[2 * j + 1])), pk2(sj.x, sj.y), oacc[j]);
        }
      };
      // a per-head pair of values for the columns (2 j, 2 j + 1)
      auto by_head = [&](int j, float v0, float v1) {
        if constexpr (!PAIR) return pk2(v0, v0);
        return pk2(uc.head(col0 + 2 * j) ? v1 : v0, uc.head(col0 + 2 * j + 1) ? v1 : v0);
      };
      for (int t = 0; t < n_t; ++t) {
        const uint32_t i = s.step + (uint32_t)t;
        const int k0 = r_lo + t * STEP;
        const int es = (int)(i % ER), sb = (int)(i % KS);
        q8_wait(&sh.efull[es], (i / ER) & 1u, abort_flag, p.err);
        uint32_t ew[T];
#pragma unroll
        for (int hf = 0; hf < T; ++hf) ew[hf] = sh.exps[es][hf * kTcTile + my_row];
        const int vslot = sh.vslot[es];
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.efree[es]);
        q8_wait(&sh.sfull[sb], (i / KS) & 1u, abort_flag, p.err);
        tc_fence_after();
        f32x2 x[T][NP];
        {
          float hi[T][NL], lo[T][NL];
#pragma unroll
          for (int hf = 0; hf < T; ++hf) {
            tmem_cols<NL>(tq + (uint32_t)((T * sb + hf) * N + col0), hi[hf]);
            tmem_cols<NL>(tq + (uint32_t)((T * sb + hf) * N + NQP + col0), lo[hf]);
          }
          tc_wait_ld();
#pragma unroll
          for (int hf = 0; hf < T; ++hf) {
            const float ka = exp2_int((int)(signed char)ew[hf]), kb = exp2_int((int)(signed char)(ew[hf] >> 16));
            const float va = (float)(signed char)(ew[hf] >> 8), vb = (float)(signed char)(ew[hf] >> 24);
#pragma unroll
            for (int j = 0; j < NP; ++j) {
              const f32x2 y = fma2(pk2(lo[hf][2 * j], lo[hf][2 * j + 1]), c16, pk2(hi[hf][2 * j], hi[hf][2 * j + 1]));
              const float2 cs = *reinterpret_cast<const float2*>(csc + 2 * j);
              x[hf][j] = fma2(mul2(y, by_head(j, ka, kb)), pk2(cs.x, cs.y), by_head(j, va, vb));
            }
          }
          // (after the scales are read: the Q warp may rewrite them once S is free)
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.sfree[sb]);
        }
        // masking, as K2: nothing to do on a step inside the unit and below the causal
        // frontier of the window's first row
        const int last = k0 + STEP - 1;
        if (last >= r_hi || col0 + NL > nvec || last > frontier) {
#pragma unroll
          for (int hf = 0; hf < T; ++hf) {
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
                const bool see = n < nlim && (p.row_pos != nullptr ? key <= sh.rp[n] : uc.vec(n) >= thr);
                y[e] = see ? y[e] : NEG_INF;
              }
              x[hf][j] = pk2(y[0], y[1]);
            }
          }
        }
        float* rb = sh.red[i & 1u][0];
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          float m0, m1;
          up2(x[0][j], m0, m1);
          if constexpr (T == 2) {
            float b0, b1;
            up2(x[1][j], b0, b1);
            m0 = fmaxf(m0, b0);
            m1 = fmaxf(m1, b1);
          }
          m0 = warp_max_f32(m0);
          m1 = warp_max_f32(m1);
          if (lane == 0) *reinterpret_cast<float2*>(rb + sq * NQP + col0 + 2 * j) = make_float2(m0, m1);
        }
        softmax_bar<SMT>();
        if (t >= 1) add_o(i - 1, t - 1);  // relative to M before this step; also frees P^T
        float al = 1.f;
        if (lane < NL) {
          const int c = col0 + lane;
          const float mx = fmaxf(fmaxf(rb[c], rb[NQP + c]), fmaxf(rb[2 * NQP + c], rb[3 * NQP + c]));
          const bool none = mx == NEG_INF;  // no key seen: exp2(-inf) = 0
          const float sub = none ? 0.f : 8.f - mx;
          const float ms = 8.f - sub;  // the maximum that `sub` stands for: its rounding enters no ratio of steps
          if (!none && ms > m + kQ8Lead) {
            al = ex2_ftz(m - ms);
            m = ms;
          }
          mw[kMxSub + lane] = sub;
          mw[kMxMove + lane] = al;
          mw[kMxStep + 16 * (t & 1) + lane] = none ? 0.f : ex2_ftz(ms - m);
        }
        const bool moved = __any_sync(0xffffffffu, al != 1.f);
        __syncwarp();
        if (moved) {
#pragma unroll
          for (int j = 0; j < NP; ++j) {
            const float2 aj = *reinterpret_cast<const float2*>(mw + kMxMove + 2 * j);
            lp[j] = mul2(lp[j], pk2(aj.x, aj.y));
            oacc[j] = mul2(oacc[j], pk2(aj.x, aj.y));
          }
        }
        if (last >= r_hi && col0 == 0) {  // warp-uniform
          // rows past the range may hold anything: once the tiles have landed, zero these keys' V rows
          q8_wait(&sh.vfull[vslot & 255], (uint32_t)(vslot >> 8), abort_flag, p.err);
#pragma unroll
          for (int hf = 0; hf < T; ++hf) {
            if (k0 + hf * kTcTile + my_row >= r_hi) {
              unsigned char* vrow = vts + (vslot & 255) * C::STEP_BYTES + (hf * kTcTile + my_row) * 128;
#pragma unroll
              for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(vrow + c * 16) = make_uint4(0, 0, 0, 0);
            }
          }
        }
        // weights 2^(t - m + 8); the denominator's leave the value scale out again.
        // (A step of one tile: the other's are zero, and no MMA reads them.)
        uint32_t w1[T][(NL + 3) / 4], w2[T][(NL + 3) / 4];
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          const float2 mj = *reinterpret_cast<const float2*>(mw + kMxSub + 2 * j);
          const float2 sj = *reinterpret_cast<const float2*>(mw + kMxStep + 16 * (t & 1) + 2 * j);
          f32x2 ls = 0ull;  // the step's sum
#pragma unroll
          for (int hf = 0; hf < T; ++hf) {
            const float ia = exp2_int(-(int)(signed char)(ew[hf] >> 8)), ib = exp2_int(-(int)(signed char)(ew[hf] >> 24));
            float d0, d1;
            up2(add2(x[hf][j], pk2(mj.x, mj.y)), d0, d1);
            const f32x2 w = pk2(ex2_ftz(d0), ex2_ftz(d1));
            ls = fma2(w, by_head(j, ia, ib), ls);
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
          lp[j] = fma2(ls, pk2(sj.x, sj.y), lp[j]);
        }
#pragma unroll
        for (int hf = 0; hf < T; ++hf) {
          const uint32_t rowo = (uint32_t)((hf * kTcTile + my_row) * C::P_ROWB);
          auto put = [&](int col, const uint32_t(&w)[(NL + 3) / 4]) {
            uint32_t off = rowo + (uint32_t)col;
            off ^= ((off >> 7) & ((1u << C::P_SWZ_BITS) - 1u)) << 4;
            if constexpr (NL == 16)
              *reinterpret_cast<uint4*>(ps + off) = make_uint4(w[0], w[1], w[2], w[3]);
            else if constexpr (NL == 8)
              *reinterpret_cast<uint2*>(ps + off) = make_uint2(w[0], w[1]);
            else if constexpr (NL == 4)
              *reinterpret_cast<uint32_t*>(ps + off) = w[0];
            else
              *reinterpret_cast<uint16_t*>(ps + off) = (uint16_t)w[0];
          };
          put(col0, w1[hf]);
          put(NQP + col0, w2[hf]);
        }
        fence_async_smem();
        softmax_bar<SMT>();
        if (stid == 0) mbar_arrive(&sh.pfull);
      }
      add_o(s.step + (uint32_t)n_t - 1, n_t - 1);

      // ---- column sums of the weights over the unit's keys
      float* lb = sh.lred[s.unit & 1u][0];
      {
        float w[NL];
#pragma unroll
        for (int j = 0; j < NP; ++j) up2(lp[j], w[2 * j], w[2 * j + 1]);
        const float r = warp_col_sum<NL>(w, lane);
        if (lane < NL) lb[sq * NQP + col0 + reduced_col<NL>(lane)] = r;
      }
      softmax_bar<SMT>();
      float oc[NL];
#pragma unroll
      for (int j = 0; j < NP; ++j) up2(oacc[j], oc[2 * j], oc[2 * j + 1]);
      auto lsum = [&](int n) { return lb[n] + lb[NQP + n] + lb[2 * NQP + n] + lb[3 * NQP + n]; };
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
          if (col0 + j < nvec) put_out(col0 + j, oc[j], lsum(col0 + j));
      } else {
        if (!s.waited) {
          griddep_wait();
          s.waited = true;
        }
        // 2: every other contributor had published when this stream began the unit
        if (stid == 0) {
          sh.flag = (arrived == n_contrib - 1) ? 2 : 0;
          if (sh.flag == 2) fence_acq_rel_gpu();
        }
        softmax_bar<SMT>();
        if (sh.flag != 2) {
          const int slot = (ustart < a) ? 2 * vid : 2 * vid + 1;
          float* pb = p.ws_part + (size_t)slot * C::PART_FLOATS;
#pragma unroll
          for (int j = 0; j < NL; ++j) {
            const float mj = __shfl_sync(0xffffffffu, m, j);
            if (col0 + j < nvec) {
              if (dim == 0) {
                pb[col0 + j] = mj;
                pb[NQP + col0 + j] = lsum(col0 + j);
              }
              pb[2 * NQP + (col0 + j) * 128 + dim] = oc[j];
            }
          }
          __threadfence();
          softmax_bar<SMT>();
          if (stid == 0) {
            const int prev = atomicAdd(p.ws_cnt + c_first, 1);
            sh.flag = (prev == n_contrib - 1) ? 1 : 0;
          }
          softmax_bar<SMT>();
        }
        if (sh.flag) {
          __threadfence();
          // online merge in key order, whoever arrives last; up to 8 columns at a time,
          // whose loads of one contributor are all in flight together
          const int k_own = vid - c_first;
          constexpr int MC = NL < 8 ? NL : 8;
#pragma unroll
          for (int j0 = 0; j0 < NL; j0 += MC) {
            float M[MC], Ls[MC], acc[MC];
#pragma unroll
            for (int j = 0; j < MC; ++j) {
              M[j] = NEG_INF;
              Ls[j] = acc[j] = 0.f;
            }
            for (int k = 0; k < n_contrib; ++k) {
              const int cc = c_first + k;
              const float* base = p.ws_part + (size_t)(k == 0 ? 2 * cc + 1 : 2 * cc) * C::PART_FLOATS;
              float mk[MC], lk[MC], ok[MC];
#pragma unroll
              for (int j = 0; j < MC; ++j) {
                const int n = col0 + j0 + j;
                const float mj = __shfl_sync(0xffffffffu, m, j0 + j);
                mk[j] = mj;
                lk[j] = 0.f;
                ok[j] = oc[j0 + j];
                if (k != k_own && n < nvec) {
                  mk[j] = ld_cg_f32(base + n);
                  lk[j] = ld_cg_f32(base + NQP + n);
                  ok[j] = ld_cg_f32(base + 2 * NQP + n * 128 + dim);
                }
              }
#pragma unroll
              for (int j = 0; j < MC; ++j) {
                if (k == k_own) lk[j] = lsum(col0 + j0 + j);
                const float nm = fmaxf(M[j], mk[j]);
                const float ms = nm == NEG_INF ? 0.f : nm;
                const float wa = fast_exp2(M[j] - ms), wb = fast_exp2(mk[j] - ms);
                Ls[j] = Ls[j] * wa + lk[j] * wb;
                acc[j] = acc[j] * wa + ok[j] * wb;
                M[j] = nm;
              }
            }
#pragma unroll
            for (int j = 0; j < MC; ++j)
              if (col0 + j0 + j < nvec) put_out(col0 + j0 + j, acc[j], Ls[j]);
          }
        }
        if (sh.flag && stid == 0) p.ws_cnt[c_first] = 0;
        softmax_bar<SMT>();  // s_flag is rewritten by the next unit
      }
      s.step += (uint32_t)n_t;
      ++s.unit;
      s.next_unit(p, STEP);
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
