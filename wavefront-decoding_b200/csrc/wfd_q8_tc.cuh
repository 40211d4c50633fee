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
// Q operand of the next units (two buffers); 3.. softmax, 4 warps per slice of the
// query columns.  Work split, merging and the self-planned start are K2's
// (UnitIter, CtaStart).  Every wait is bounded; no multicast, no cluster.
#pragma once

#include "wfd_q8_attn.cuh"

namespace wfd {

template <int NQP>
struct Q8Cfg {
  static constexpr int N = 2 * NQP;                  // MMA columns: both pieces
  static constexpr int STAGES = NQP == 16 ? 6 : 5;   // 128-key tiles of K and V
  static constexpr int TILE_BYTES = kTcTile * 128;
  static constexpr int KV_STAGE = 2 * TILE_BYTES;
  static constexpr int Q_BYTES = N * 128;            // one of two buffers
  static constexpr int P_ROWB = N;                   // one key's row of P^T
  static constexpr int P_BYTES = 2 * kTcTile * P_ROWB;
  static constexpr int P_SWZ_BITS = NQP == 16 ? 1 : 2;     // 32- / 64-byte swizzle
  static constexpr uint64_t P_LAYOUT = NQP == 16 ? 6 : 4;
  static constexpr int P_ATOM = 8 * P_ROWB;
  static constexpr int RED_FLOATS = 2 * 4 * NQP;
  static constexpr int SMEM = STAGES * KV_STAGE + 2 * Q_BYTES + P_BYTES + 2 * RED_FLOATS * 4 + 4 * NQP * 4 + 1024;
  static constexpr int S_COL = 0;                    // S^T of tile pair buffer sb, half hf: (2 sb + hf) N
  static constexpr int O_COL = 4 * N;                // O^T, two accumulator chains
  static constexpr int TMEM_COLS = NQP == 16 ? 256 : 512;
  static constexpr int PART_FLOATS = NQP * (128 + 2);
  static_assert(O_COL + 2 * N <= TMEM_COLS, "TMEM columns");
  static_assert(SMEM + 2048 <= 232448, "shared memory per CTA (dynamic + the kernel's static arrays)");
};

__host__ __device__ constexpr int q8_slices(int na) { return na >= 16 ? 2 : 1; }  // column slices of the softmax
__host__ __device__ constexpr int q8_tc_threads(int na) { return 96 + 128 * q8_slices(na); }

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

// Two weights as two pieces: codes of (a, b) in the low 16 bits of p1 and p2.
__device__ __forceinline__ void q8_split(float a, float b, uint32_t& p1, uint32_t& p2) {
  p1 = e4m3x2(a, b);
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)p1, __NV_E4M3);
  const float2 f = __half22float2(__half2(h));
  p2 = e4m3x2((a - f.x) * 16.f, (b - f.y) * 16.f);
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
    share = (total + gridDim.x - 1) / gridDim.x;
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
struct UnitCols {
  int v0, nv1, nvec;
  __device__ __forceinline__ UnitCols(const VerifyParams& p, const Seg& S, int qg, int nqp) {
    const int gh = p.pair ? nqp / 2 : nqp;
    v0 = qg * gh;
    nv1 = min(gh, S.q_len * p.G - v0);
    nvec = p.pair ? 2 * nv1 : nv1;
    if (!p.pair) nv1 = 0x7fffffff;
  }
  __device__ __forceinline__ int head(int n) const { return n >= nv1 ? 1 : 0; }
  __device__ __forceinline__ int vec(int n) const { return v0 + (n >= nv1 ? n - nv1 : n); }
};

// NA: query columns the softmax works on (every unit has at most NA vectors).
template <int NQP, int NA>
__global__ void __launch_bounds__(q8_tc_threads(NA), 1)
    q8_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                 const __grid_constant__ TailMaps tails, const Q8AttnParams p) {
  using C = Q8Cfg<NQP>;
  constexpr int STAGES = C::STAGES;
  constexpr int N = C::N;
  constexpr int THREADS = q8_tc_threads(NA);
  constexpr int H2 = q8_slices(NA);  // column slices of the softmax (4 warps each)
  constexpr int NL = NA / H2;        // query columns per softmax thread
  constexpr int SMT = 128 * H2;
  static_assert(NL == 2 || NL == 4 || NL == 8 || NL == 16, "columns per softmax thread");
  static_assert(NA <= NQP, "active query columns");
  const float NEG_INF = -__int_as_float(0x7f800000);

  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* kvs = smem;                                // STAGES x (K tile, V tile)
  unsigned char* qs = kvs + STAGES * C::KV_STAGE;           // 2 x Q operand (K-major, 128B swizzle)
  unsigned char* ps = qs + 2 * C::Q_BYTES;                  // P^T operand of a tile pair (MN-major)
  float* red = reinterpret_cast<float*>(ps + C::P_BYTES);   // [2][4][NQP] column maxima
  float* lred = red + C::RED_FLOATS;                        // [2][4][NQP] column sums
  float* cscale = lred + C::RED_FLOATS;                     // [4][NQP] score scale of each column, per unit

  __shared__ __align__(8) uint64_t bar_full[STAGES];
  __shared__ __align__(8) uint64_t bar_empty[STAGES];
  __shared__ __align__(8) uint64_t bar_sfull[2];
  __shared__ __align__(8) uint64_t bar_sfree[2];
  __shared__ __align__(8) uint64_t bar_pfull;
  __shared__ __align__(8) uint64_t bar_ofull;
  __shared__ __align__(8) uint64_t bar_ofree;
  __shared__ __align__(8) uint64_t bar_qready[4];  // unit's Q and column scales written
  __shared__ __align__(8) uint64_t bar_qfree[2];
  __shared__ __align__(8) uint64_t bar_drain;
  __shared__ uint32_t s_tmem;
  __shared__ int s_rp[NQP];  // gapped windows: each query column's row position
  __shared__ volatile int s_abort;
  __shared__ int s_flag;
  __shared__ SelfStart s_start;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const bool self = p.items != nullptr;
  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tm_k)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tm_v)) : "memory");
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&bar_full[s], 1);
      mbar_init(&bar_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bar_sfull[s], 1);
      mbar_init(&bar_sfree[s], 4 * H2);
      mbar_init(&bar_qfree[s], 1);
    }
    for (int s = 0; s < 4; ++s) mbar_init(&bar_qready[s], 1);
    mbar_init(&bar_pfull, 1);
    mbar_init(&bar_ofull, 1);
    mbar_init(&bar_ofree, 4 * H2);
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
      share = (total + gridDim.x - 1) / gridDim.x;
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
    uint32_t n_iss = 0;  // tiles whose loads were issued (a prefix of the sequence: issue stops at an abort)
    while (itr.next(p, S, u, r_lo, r_hi, ustart)) {
      const int h = u % p.Hkv;
      const int n_sub = (r_hi - r_lo + kTcTile - 1) / kTcTile;
      const long long row0 = S.k_row0 + p.k_row_offset + r_lo;
      for (int t = 0; t < n_sub; ++t, ++it) {
        const int stage = (int)(it % STAGES);
        need_rows(itr, r_lo + (t + 1) * kTcTile);
        const bool go = (it >= (uint32_t)STAGES) ? tc_wait(&bar_empty[stage], ((it / STAGES) - 1) & 1u, &s_abort, p.err)
                                                 : !s_abort;
        if (go && lane == 0) {
          unsigned char* dst = kvs + stage * C::KV_STAGE;
          const int row = (int)(row0 + (long long)t * kTcTile);
          // a tail of at most 96 rows loads only those, in pieces of 64 / 32 / 16 / 8
          const int rows_left = r_hi - r_lo - t * kTcTile;
          const int nr = rows_left > 96 ? kTcTile : ((rows_left + 7) & ~7);
          mbar_arrive_expect_tx(&bar_full[stage], (uint32_t)(nr * 128 * 2));
          if (nr == kTcTile) {
            tma_load_3d(dst, &tm_k, 0, h, row, &bar_full[stage]);
            tma_load_3d(dst + C::TILE_BYTES, &tm_v, 0, h, row, &bar_full[stage]);
          } else {
            int off = 0;
#pragma unroll
            for (int pc = 0; pc < 4; ++pc) {
              const int pr = 64 >> pc;
              if (nr & pr) {
                tma_load_3d(dst + off * 128, &tails.k[pc], 0, h, row + off, &bar_full[stage]);
                tma_load_3d(dst + C::TILE_BYTES + off * 128, &tails.v[pc], 0, h, row + off, &bar_full[stage]);
                off += pr;
              }
            }
          }
          n_iss = it + 1;
          if (p.fail_waits && n_iss == 1) {  // test hook: give up with this tile's copies in flight
            set_error(p.err, kErrTimeout);
            s_abort = 1;
          }
        }
        __syncwarp();
      }
    }
    const uint32_t n_used = it;
    for (uint32_t j = (n_used > (uint32_t)STAGES ? n_used - STAGES : 0); j < n_used; ++j)
      tc_wait(&bar_empty[j % STAGES], (j / STAGES) & 1u, &s_abort, p.err);
    // copies in flight land before the CTA exits, also after an abort
    if (lane == 0) {
      for (uint32_t j = (n_iss > (uint32_t)STAGES ? n_iss - STAGES : 0); j < n_iss; ++j)
        if (!mbar_wait_bounded(&bar_full[j % STAGES], (j / STAGES) & 1u)) set_error(p.err, kErrTimeout);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    UnitIter itr = make_iter();
    uint32_t it = 0, tt = 0, pv = 0, units = 0;
    constexpr uint32_t IDESC_S = q8_idesc(N, false, false);
    constexpr uint32_t IDESC_PV = q8_idesc(N, true, true);
    const uint32_t q_addr = smem_u32(qs);
    const uint32_t p_addr = smem_u32(ps);
    while (itr.next(p, S, u, r_lo, r_hi, ustart)) {
      const int n_sub = (r_hi - r_lo + kTcTile - 1) / kTcTile;
      const int n_t = (n_sub + 1) >> 1;
      const int qb = (int)(units & 1u);
      const uint32_t qa = q_addr + (uint32_t)(qb * C::Q_BYTES);
      tc_wait(&bar_qready[units & 3u], (units >> 2) & 1u, &s_abort, p.err);
      tc_fence_after();
      for (int t = 0; t <= n_t; ++t) {
        if (t < n_t) {
          const uint32_t ti = tt + t;
          const int sb = (int)(ti & 1u);
          const int nh = (2 * t + 1 < n_sub) ? 2 : 1;
          const uint32_t i0 = it + 2 * t;
          bool go = true;
          for (int hf = 0; hf < nh; ++hf)
            go = tc_wait(&bar_full[(i0 + hf) % STAGES], ((i0 + hf) / STAGES) & 1u, &s_abort, p.err) && go;
          if (ti >= 2) go = tc_wait(&bar_sfree[sb], ((ti >> 1) - 1) & 1u, &s_abort, p.err) && go;
          tc_fence_after();
          if (go && lane == 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // 32 bytes of the row; the halves are independent accumulators
              for (int hf = 0; hf < nh; ++hf) {
                const uint32_t k_addr = smem_u32(kvs + (int)((i0 + hf) % STAGES) * C::KV_STAGE);
                umma_f8(tmem + (uint32_t)((2 * sb + hf) * N), umma_desc(k_addr + j * 32, 16, 1024, 2),
                        umma_desc(qa + j * 32, 16, 1024, 2), IDESC_S, j > 0 ? 1u : 0u);
              }
            }
            umma_commit(&bar_sfull[sb]);
            if (t == n_t - 1) umma_commit(&bar_qfree[qb]);  // the unit's Q buffer may be rewritten
          }
          __syncwarp();
        }
        if (t >= 1) {
          bool go = tc_wait(&bar_pfull, pv & 1u, &s_abort, p.err);
          if (pv >= 1) go = tc_wait(&bar_ofree, (pv - 1) & 1u, &s_abort, p.err) && go;
          tc_fence_after();
          const int nh = (2 * (t - 1) + 1 < n_sub) ? 2 : 1;
          const uint32_t i0 = it + 2 * (t - 1);
          if (go && lane == 0) {
            for (int hf = 0; hf < nh; ++hf) {
              const uint32_t v_addr = smem_u32(kvs + (int)((i0 + hf) % STAGES) * C::KV_STAGE + C::TILE_BYTES);
#pragma unroll
              for (int j = 0; j < 4; ++j)  // 32 keys: four 8-row groups of V and of P^T
                umma_f8(tmem + (uint32_t)(C::O_COL + (j & 1) * N), umma_desc(v_addr + j * 4096, 16, 1024, 2),
                        umma_desc(p_addr + (hf * 16 + j * 4) * C::P_ATOM, 16, C::P_ATOM, C::P_LAYOUT), IDESC_PV,
                        (hf > 0 || j >= 2) ? 1u : 0u);
            }
            umma_commit(&bar_ofull);
            for (int hf = 0; hf < nh; ++hf) umma_commit(&bar_empty[(i0 + hf) % STAGES]);
          }
          __syncwarp();
          ++pv;
        }
      }
      it += n_sub;
      tt += n_t;
      ++units;
    }
    // every MMA complete before TMEM is freed and the CTA exits, also after an abort
    if (lane == 0) {
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
      const bool go = units >= 2 ? tc_wait(&bar_qfree[qb], ((units >> 1) - 1) & 1u, &s_abort, p.err) : !s_abort;
      if (go) {
        const UnitCols uc(p, S, qg, NQP);
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
              if (p.pair) {
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
            q8_split(f[0] * sc, f[1] * sc, a1, a2);
            q8_split(f[2] * sc, f[3] * sc, b1, b2);
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
      tc_wait(&bar_qfree[k & 1u], (k >> 1) & 1u, &s_abort, p.err);
  } else {
    // ------------------------------------------------------------ softmax warps
    const int sw = warp - 3;
    const int sq = sw & 3;              // warp within its column slice
    const int col0 = (sw >> 2) * NL;    // first query column of this thread
    const int qd = warp & 3;            // TMEM lane quadrant this warp may access
    const int stid = tid - 96;
    const int my_row = qd * 32 + lane;  // key of either tile, then head dim, this thread owns
    const uint32_t tq = tmem + ((uint32_t)(qd * 32) << 16);
    UnitIter itr = make_iter();
    uint32_t it = 0, tt = 0, pv = 0, units = 0;
    // columns past the unit's vectors hold anything: an MMA column enters no other
    while (itr.next(p, S, u, r_lo, r_hi, ustart)) {
      const int h = u % p.Hkv, qg = u / p.Hkv;
      const int n_sub = (r_hi - r_lo + kTcTile - 1) / kTcTile;
      const int n_t = (n_sub + 1) >> 1;
      const UnitCols uc(p, S, qg, NQP);
      const int nvec = uc.nvec;
      if (nvec > NA && stid == 0) set_error(p.err, kErrBadRows);  // an item longer than the call's max_q
      const int c_first = (int)(ustart / share);
      const int c_last = (int)((ustart + S.k_len - 1) / share);
      const int n_contrib = p.invariant ? 1 : c_last - c_first + 1;
      int arrived = 0;
      // (the plan kernel clears the counters, so they are read after it only)
      if (n_contrib > 1 && stid == 0 && itr.waited) arrived = ld_relaxed_gpu(p.ws_cnt + c_first);

      // exponents of this thread's two keys (head pairs: of both heads), one tile
      // pair ahead; loaded past L1, since the append may write neighbouring bytes
      const long long ebase = S.k_row0 * p.c.Hkv + (long long)(p.pair ? 2 * h : h) * p.c.max_seq;
      const int estep = p.pair ? p.c.max_seq : 0;
      int ke[2][2], ve[2][2];  // [half][head of the pair]
      auto load_exps = [&](int t) {
        need_rows(itr, min(r_hi, r_lo + (t + 1) * 2 * kTcTile));
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int key = r_lo + (2 * t + hf) * kTcTile + my_row;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            ke[hf][e] = ve[hf][e] = 0;
            if (key < r_hi) {
              ke[hf][e] = __ldcg(reinterpret_cast<const signed char*>(p.c.ke) + ebase + e * estep + key);
              ve[hf][e] = __ldcg(reinterpret_cast<const signed char*>(p.c.ve) + ebase + e * estep + key);
            }
          }
        }
      };
      load_exps(0);
      if (p.row_pos != nullptr) {
        if (sq == 0 && lane < NL) {
          const int n = col0 + lane;
          s_rp[n] = n < nvec ? p.row_pos[(long long)(S.q_row0 + uc.vec(n) / p.G) * p.row_pos_stride] : -1;
        }
        softmax_bar<SMT>();
      }
      tc_wait(&bar_qready[units & 3u], (units >> 2) & 1u, &s_abort, p.err);
      float csc[NL], m[NL], lp[NL], oacc[NL];
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        csc[j] = cscale[(units & 3u) * NQP + col0 + j];
        m[j] = NEG_INF;
        lp[j] = 0.f;
        oacc[j] = 0.f;
      }
      auto add_o = [&]() {  // the last tile pair's P.V joins O
        tc_wait(&bar_ofull, pv & 1u, &s_abort, p.err);
        tc_fence_after();
        float o0[NL], o1[NL], o2[NL], o3[NL];
        tmem_cols<NL>(tq + (uint32_t)(C::O_COL + col0), o0);
        tmem_cols<NL>(tq + (uint32_t)(C::O_COL + NQP + col0), o1);
        tmem_cols<NL>(tq + (uint32_t)(C::O_COL + N + col0), o2);
        tmem_cols<NL>(tq + (uint32_t)(C::O_COL + N + NQP + col0), o3);
        tc_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_ofree);
        ++pv;
#pragma unroll
        for (int j = 0; j < NL; ++j) oacc[j] += fmaf(o1[j] + o3[j], 0.0625f, o0[j] + o2[j]);
      };
      for (int t = 0; t < n_t; ++t) {
        const uint32_t ti = tt + t;
        const int sb = (int)(ti & 1u);
        const int k0 = r_lo + t * 2 * kTcTile;
        float ksc[2][2], vex[2][2];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            ksc[hf][e] = exp2_int(ke[hf][e]);
            vex[hf][e] = (float)ve[hf][e];
          }
        if (t + 1 < n_t) load_exps(t + 1);
        tc_wait(&bar_sfull[sb], (ti >> 1) & 1u, &s_abort, p.err);
        tc_fence_after();
        float x[2][NL];
        {
          float lo[2][NL];
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            tmem_cols<NL>(tq + (uint32_t)((2 * sb + hf) * N + col0), x[hf]);
            tmem_cols<NL>(tq + (uint32_t)((2 * sb + hf) * N + NQP + col0), lo[hf]);
          }
          tc_wait_ld();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar_sfree[sb]);
#pragma unroll
          for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int j = 0; j < NL; ++j) {
              const int e = uc.head(col0 + j);
              x[hf][j] = fmaf(fmaf(lo[hf][j], 0.0625f, x[hf][j]) * ksc[hf][e], csc[j], vex[hf][e]);
            }
        }
        // masking, as K2: nothing to do on a tile pair inside the unit and below the
        // causal frontier of the window's first row
        const int tile_last = k0 + 2 * kTcTile - 1;
        const bool interior = tile_last < r_hi && col0 + NL <= nvec && p.row_pos == nullptr &&
                              tile_last <= S.k_len - S.q_len;
        if (!interior) {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const int key = k0 + hf * kTcTile + my_row;
            const int nlim = key < r_hi ? nvec : 0;
            const int thr = (key - (S.k_len - S.q_len)) * p.G;
#pragma unroll
            for (int j = 0; j < NL; ++j) {
              const int n = col0 + j;
              const bool see = n < nlim && (p.row_pos != nullptr ? key <= s_rp[n] : uc.vec(n) >= thr);
              x[hf][j] = see ? x[hf][j] : NEG_INF;
            }
          }
        }
        float* rb = red + (ti & 1u) * (4 * NQP);
        {
          float r[NL];
#pragma unroll
          for (int j = 0; j < NL; ++j) r[j] = warp_max_f32(fmaxf(x[0][j], x[1][j]));
          if (lane == 0) {
#pragma unroll
            for (int j = 0; j < NL; ++j) rb[sq * NQP + col0 + j] = r[j];
          }
        }
        softmax_bar<SMT>();
        if (t >= 1) add_o();  // relative to the maximum before this tile; also frees P^T
        // every thread keeps the running maxima of its columns
#pragma unroll
        for (int j = 0; j < NL; ++j) {
          const int c = col0 + j;
          const float mx = fmaxf(fmaxf(rb[c], rb[NQP + c]), fmaxf(rb[2 * NQP + c], rb[3 * NQP + c]));
          if (mx > m[j] + 0.75f) {
            const float al = fast_exp2(m[j] - mx);
            lp[j] *= al;
            oacc[j] *= al;
            m[j] = mx;
          }
        }
        const int n_here = (2 * t + 1 < n_sub) ? 2 : 1;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          if (hf < n_here) {
            const int key = k0 + hf * kTcTile + my_row;
            if (key >= r_hi && col0 == 0) {
              // rows past the range may hold anything: zero this key's V row
              unsigned char* vrow = kvs + (int)((it + 2 * t + hf) % STAGES) * C::KV_STAGE + C::TILE_BYTES + my_row * 128;
#pragma unroll
              for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(vrow + c * 16) = make_uint4(0, 0, 0, 0);
            }
            const float iv0 = exp2_int(-(int)vex[hf][0]), iv1 = exp2_int(-(int)vex[hf][1]);
            uint32_t w1[(NL + 3) / 4], w2[(NL + 3) / 4];
#pragma unroll
            for (int j = 0; j < NL; j += 2) {
              float w[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float mb = m[j + e] == NEG_INF ? 0.f : m[j + e] - 8.f;  // no key seen: exp2(-inf) = 0
                w[e] = fast_exp2(x[hf][j + e] - mb);
                lp[j + e] = fmaf(w[e], uc.head(col0 + j + e) ? iv1 : iv0, lp[j + e]);
              }
              uint32_t p1, p2;
              q8_split(w[0], w[1], p1, p2);
              if ((j & 2) == 0) {
                w1[j / 4] = p1;
                w2[j / 4] = p2;
              } else {
                w1[j / 4] |= p1 << 16;
                w2[j / 4] |= p2 << 16;
              }
            }
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
            put(col0, w1);
            put(NQP + col0, w2);
          }
        }
        fence_async_smem();
        softmax_bar<SMT>();
        if (stid == 0) mbar_arrive(&bar_pfull);
      }
      add_o();
      it += n_sub;
      tt += n_t;
      ++units;

      // ---- column sums of the weights over the unit's keys
      float* lb = lred + (units & 1u) * (4 * NQP);
      {
        float w[NL];
#pragma unroll
        for (int j = 0; j < NL; ++j) w[j] = lp[j];
        const float r = warp_col_sum<NL>(w, lane);
        if (lane < NL) lb[sq * NQP + col0 + reduced_col<NL>(lane)] = r;
      }
      softmax_bar<SMT>();
      auto lsum = [&](int n) { return lb[n] + lb[NQP + n] + lb[2 * NQP + n] + lb[3 * NQP + n]; };
      const int dim = my_row;
      // output element of query column n held by this thread's O^T row, or -1
      auto out_at = [&](int n) -> long long {
        const int e = uc.head(n), v = uc.vec(n);
        const long long row = (long long)(S.q_row0 + v / p.G) * p.Hq + v % p.G;
        if (p.pair) return (dim >> 6) == e ? (row + (2 * h + e) * p.G) * 64 + (dim & 63) : -1;
        return (row + h * p.G) * 128 + dim;
      };
      auto put_out = [&](int n, float O, float L) {
        const long long oi = out_at(n);
        if (oi >= 0) static_cast<__nv_bfloat16*>(p.out)[oi] = __float2bfloat16_rn(L == 0.f ? 0.f : O / L);
      };
      if (n_contrib == 1) {
#pragma unroll
        for (int j = 0; j < NL; ++j)
          if (col0 + j < nvec) put_out(col0 + j, oacc[j], lsum(col0 + j));
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
        softmax_bar<SMT>();
        if (s_flag != 2) {
          const int slot = (ustart < a) ? 2 * (int)blockIdx.x : 2 * (int)blockIdx.x + 1;
          float* pb = p.ws_part + (size_t)slot * C::PART_FLOATS;
#pragma unroll
          for (int j = 0; j < NL; ++j) {
            if (col0 + j < nvec) {
              if (dim == 0) {
                pb[col0 + j] = m[j];
                pb[NQP + col0 + j] = lsum(col0 + j);
              }
              pb[2 * NQP + (col0 + j) * 128 + dim] = oacc[j];
            }
          }
          __threadfence();
          softmax_bar<SMT>();
          if (stid == 0) {
            const int prev = atomicAdd(p.ws_cnt + c_first, 1);
            s_flag = (prev == n_contrib - 1) ? 1 : 0;
          }
          softmax_bar<SMT>();
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
                mk[j] = m[j];
                lk[j] = lsum(n);
                ok[j] = oacc[j];
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
        softmax_bar<SMT>();  // s_flag is rewritten by the next unit
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
