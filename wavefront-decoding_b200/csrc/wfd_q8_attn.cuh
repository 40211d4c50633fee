// K10 — wavefront attention over the 8-bit slot cache on the CUDA cores: fp32
// queries, and the bf16 shapes the tensor-core kernel (K11) does not take.
//
//   s_t = scale * 2^{e_k[t]} (q . codes_k[t]),  t <= the row's position
//   o   = sum_t softmax(s)_t 2^{e_v[t]} codes_v[t]
// The key scale multiplies the finished dot product and the value scale the
// weight, so the inner loops see codes only.  All arithmetic fp32; the exponent is
// taken of (s_t - m) scale log2(e), subtracted first: the rounding of a large
// score does not enter the weight.
//
// One CTA per SM works on an equal share of the flattened (segment, query group,
// kv head, key) space; units that straddle CTAs are merged by the last to arrive,
// in key order.  A head's row of Dh codes is read by Dh / 16 lanes, 16 bytes each:
// a warp takes 4 (Dh 128) or 8 (Dh 64) keys a step, U steps of K and V in flight.
// Every lane group keeps its own running (m, l, O); groups, warps and CTAs are
// merged at the end of a unit.  Up to 4 query vectors per unit: q and O take 128
// registers; more vectors are further units over the same keys.
//
// Bound by latency: 32 windows of 3 rows over 777 keys, 8 heads of 64, fp32, take
// 30 us a call (4 us of HBM time), three units a CTA of three rounds of 256 keys, each
// waiting for its loads, and a merge of 8 warps.  (Loads in branches, one round trip
// each, and 12 warps that spilled: 41 us; scalar products instead of pairs: 30.)
#pragma once

#include "wfd_q8.cuh"
#include "wfd_verify.cuh"

namespace wfd {

struct Q8AttnParams : VerifyParams {
  Q8Cache c;  // counted from the call's slot offset
};

// A CTA's share is at least this many keys of one unit, a round of its 8 to 12 warps:
// a piece of fewer takes as long, and every further piece is one more to merge.
constexpr int kQ8MinShare = 256;

// Two fp32 values in one 64-bit register: one instruction for both.
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

// Threads of a CTA, one CTA an SM: 4 vectors' queries and sums take 128 registers.
__host__ __device__ constexpr int q8_simt_threads(int nq) { return nq == 4 ? 256 : 384; }
constexpr int kQ8SimtNQ = 4;  // query vectors per unit, at most

template <typename T, int DH, int NQ>
__global__ void __launch_bounds__(q8_simt_threads(NQ), 1) q8_attn_kernel(const Q8AttnParams p) {
  constexpr int LPR = DH / 16;      // lanes per key row
  constexpr int KPW = 32 / LPR;     // keys per warp step
  constexpr int U = 4;              // steps in flight
  constexpr int THREADS = q8_simt_threads(NQ), WARPS = THREADS / 32;
  const float NEG_INF = -__int_as_float(0x7f800000);
  __shared__ float s_q[NQ][DH];
  __shared__ int s_lim[NQ];               // last key a vector sees
  __shared__ float s_o[WARPS][NQ][DH];
  __shared__ float s_m[WARPS][NQ], s_l[WARPS][NQ];
  __shared__ int s_last;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int sub = lane % LPR, grp = lane / LPR;
  griddep_wait();
  const long long total = (long long)p.Hkv * p.prefix[p.n_segs];
  long long share = 1, a = 0, b = 0;
  if (total > 0) {
    share = max((total + gridDim.x - 1) / gridDim.x, (long long)kQ8MinShare);
    a = (long long)blockIdx.x * share;
    b = (a + share < total) ? a + share : total;
  }
  if (a >= b) return;
  const CtaStart cs = p.start[blockIdx.x];
  UnitIter itr{a, b, cs.seg};
  itr.have = true;
  itr.S = cs.S;
  itr.base = cs.base;
  itr.nbase = cs.nbase;
  Seg S;
  int u, r_lo, r_hi;
  long long ustart;
  const float c2 = p.scale_log2;
  const T* q = static_cast<const T*>(p.q);
  T* out = static_cast<T*>(p.out);
  while (itr.next(p, S, u, r_lo, r_hi, ustart)) {
    const int h = u % p.Hkv, qg = u / p.Hkv;
    const int nvec = min(NQ, S.q_len * p.G - qg * NQ);
    auto q_at = [&](int n) -> long long {  // first element of query vector n of this unit
      const int v = qg * NQ + n;
      return ((long long)(S.q_row0 + v / p.G) * p.Hq + h * p.G + v % p.G) * DH;
    };
    __syncthreads();  // the previous unit's shared state is read
    for (int i = tid; i < NQ * DH; i += THREADS) {
      const int n = i / DH;
      s_q[n][i % DH] = n < nvec ? to_f<T>(q[q_at(n) + i % DH]) : 0.f;
    }
    if (tid < NQ) {
      const int row = (qg * NQ + tid) / p.G;
      s_lim[tid] = tid >= nvec ? -1
                   : p.row_pos != nullptr ? p.row_pos[(long long)(S.q_row0 + row) * p.row_pos_stride]
                                          : S.k_len - S.q_len + row;
    }
    __syncthreads();
    f32x2 qr[NQ][8], acc[NQ][8];
    float m[NQ], l[NQ];
    int lim[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        qr[n][i] = pk2(s_q[n][sub * 16 + 2 * i], s_q[n][sub * 16 + 2 * i + 1]);
        acc[n][i] = pk2(0.f, 0.f);
      }
      m[n] = NEG_INF;
      l[n] = 0.f;
      lim[n] = s_lim[n];
    }
    const long long row_codes = (long long)p.Hkv * DH;
    const long long c0 = S.k_row0 * row_codes + h * DH + sub * 16;
    const long long e0 = S.k_row0 * p.Hkv + (long long)h * p.c.max_seq;
    for (int kb = r_lo + warp * (KPW * U); kb < r_hi; kb += WARPS * KPW * U) {
      uint4 kq[U], vq[U];
      float ks[U], vs[U];
      signed char ke[U], ve[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {  // loads without branches: all in flight at once
        const int key = min(kb + j * KPW + grp, r_hi - 1);
        kq[j] = *reinterpret_cast<const uint4*>(p.c.k + c0 + key * row_codes);
        vq[j] = *reinterpret_cast<const uint4*>(p.c.v + c0 + key * row_codes);
        ke[j] = p.c.ke[e0 + key];
        ve[j] = p.c.ve[e0 + key];
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        ks[j] = exp2_int(ke[j]);
        vs[j] = exp2_int(ve[j]);
      }
      float s[U][NQ];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        f32x2 s2[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) s2[n] = pk2(0.f, 0.f);
        const uint32_t w[4] = {kq[j].x, kq[j].y, kq[j].z, kq[j].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float f[4];
          e4m3x4_to_f(w[i], f);
          const f32x2 f0 = pk2(f[0], f[1]), f1 = pk2(f[2], f[3]);
#pragma unroll
          for (int n = 0; n < NQ; ++n) s2[n] = fma2(qr[n][2 * i + 1], f1, fma2(qr[n][2 * i], f0, s2[n]));
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          float s_even, s_odd;
          up2(s2[n], s_even, s_odd);
          s[j][n] = s_even + s_odd;
#pragma unroll
          for (int o = LPR / 2; o > 0; o >>= 1) s[j][n] += __shfl_xor_sync(0xffffffffu, s[j][n], o);
          const int key = kb + j * KPW + grp;
          s[j][n] = (key < r_hi && key <= lim[n]) ? s[j][n] * ks[j] : NEG_INF;
        }
      }
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float mn = m[n];
#pragma unroll
        for (int j = 0; j < U; ++j) mn = fmaxf(mn, s[j][n]);
        const float ms = mn == NEG_INF ? 0.f : mn;  // no key seen yet: every weight below is exp2(-inf) = 0
        const float cr = fast_exp2((m[n] - ms) * c2);
        m[n] = mn;
        l[n] *= cr;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[n][i] = mul2(acc[n][i], pk2(cr, cr));
#pragma unroll
        for (int j = 0; j < U; ++j) {
          const float w = fast_exp2((s[j][n] - ms) * c2);
          l[n] += w;
          s[j][n] = w == 0.f ? 0.f : w * vs[j];
        }
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const uint32_t w[4] = {vq[j].x, vq[j].y, vq[j].z, vq[j].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float f[4];
          e4m3x4_to_f(w[i], f);
          const f32x2 f0 = pk2(f[0], f[1]), f1 = pk2(f[2], f[3]);
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            const f32x2 wn = pk2(s[j][n], s[j][n]);
            acc[n][2 * i] = fma2(wn, f0, acc[n][2 * i]);
            acc[n][2 * i + 1] = fma2(wn, f1, acc[n][2 * i + 1]);
          }
        }
      }
    }
    // merge the warp's lane groups, then publish the warp's (m, l, O)
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
      for (int o = LPR; o < 32; o <<= 1) {
        const float mo = __shfl_xor_sync(0xffffffffu, m[n], o);
        const float lo = __shfl_xor_sync(0xffffffffu, l[n], o);
        const float mn = fmaxf(m[n], mo);
        const float ms = mn == NEG_INF ? 0.f : mn;
        const float ca = fast_exp2((m[n] - ms) * c2), cb = fast_exp2((mo - ms) * c2);
        l[n] = l[n] * ca + lo * cb;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const f32x2 ao = __shfl_xor_sync(0xffffffffu, acc[n][i], o);
          acc[n][i] = fma2(ao, pk2(cb, cb), mul2(acc[n][i], pk2(ca, ca)));
        }
        m[n] = mn;
      }
      if (grp == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) up2(acc[n][i], s_o[warp][n][sub * 16 + 2 * i], s_o[warp][n][sub * 16 + 2 * i + 1]);
        if (sub == 0) {
          s_m[warp][n] = m[n];
          s_l[warp][n] = l[n];
        }
      }
    }
    __syncthreads();
    const int c_first = (int)(ustart / share);
    const int c_last = (int)((ustart + S.k_len - 1) / share);
    const int n_contrib = p.invariant ? 1 : c_last - c_first + 1;
    constexpr int PART = NQ * (DH + 2);
    for (int i = tid; i < nvec * DH; i += THREADS) {
      const int n = i / DH, d = i % DH;
      float M = NEG_INF;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) M = fmaxf(M, s_m[w][n]);
      const float ms = M == NEG_INF ? 0.f : M;
      float L = 0.f, O = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float cw = fast_exp2((s_m[w][n] - ms) * c2);
        L += s_l[w][n] * cw;
        O += s_o[w][n][d] * cw;
      }
      if (n_contrib == 1) {
        out[q_at(n) + d] = from_f<T>(L == 0.f ? 0.f : O / L);
      } else {
        const int slot = (ustart < a) ? 2 * (int)blockIdx.x : 2 * (int)blockIdx.x + 1;
        float* pb = p.ws_part + (size_t)slot * PART;
        if (d == 0) {
          pb[n] = M;
          pb[NQ + n] = L;
        }
        pb[2 * NQ + i] = O;
      }
    }
    if (n_contrib > 1) {
      __threadfence();
      __syncthreads();
      if (tid == 0) s_last = atomicAdd(p.ws_cnt + c_first, 1) == n_contrib - 1 ? 1 : 0;
      __syncthreads();
      if (s_last) {
        __threadfence();
        for (int i = tid; i < nvec * DH; i += THREADS) {
          const int n = i / DH, d = i % DH;
          float M = NEG_INF, L = 0.f, O = 0.f;
          for (int k = 0; k < n_contrib; ++k) {  // in key order, whoever arrives last
            const int cc = c_first + k;
            const float* pb = p.ws_part + (size_t)(k == 0 ? 2 * cc + 1 : 2 * cc) * PART;
            const float mk = ld_cg_f32(pb + n), lk = ld_cg_f32(pb + NQ + n), ok = ld_cg_f32(pb + 2 * NQ + i);
            const float mn = fmaxf(M, mk);
            const float ms = mn == NEG_INF ? 0.f : mn;
            const float ca = fast_exp2((M - ms) * c2), cb = fast_exp2((mk - ms) * c2);
            L = L * ca + lk * cb;
            O = O * ca + ok * cb;
            M = mn;
          }
          out[q_at(n) + d] = from_f<T>(L == 0.f ? 0.f : O / L);
        }
        if (tid == 0) p.ws_cnt[c_first] = 0;
      }
    }
  }
}

}  // namespace wfd
