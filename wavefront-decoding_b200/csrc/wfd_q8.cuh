// K9 — the 8-bit KV-slot cache: rows quantised as they are written, read back,
// and compacted.
//
// A cached row (one slot, sequence, kv head and position; Dh values of K or V)
// is Dh e4m3 codes q_i and one exponent e (int8):
//     e = clamp(smallest integer with max |x_i| <= 448 * 2^e, -32, 32)
//     q_i = e4m3(x_i * 2^-e), nearest even, saturating;   value = q_i * 2^e
// The scale is a power of two on purpose: x_i * 2^-e and q_i * 2^e are exact, so
// a row's codes are the same whatever arithmetic computes them and a value is
// exact in bf16; e4m3 keeps 4 significant bits down to 2^-6 of its scale, so a
// scale up to 2 x too large costs nothing but the subnormal floor.  The clamp
// bounds what two rows' scales can differ by (2^64), which the attention's
// running sums rely on; rows above 448 * 2^32 saturate.  A NaN is stored as 0 and
// reported (kErrNaN): a cached row is always finite, so a key that a query masks
// cannot leak into it through 0 * NaN.
//
// Layout: codes (n_slots, n_seqs, max_seq, Hkv, Dh) as the unquantised cache;
// exponents (n_slots, n_seqs, Hkv, max_seq), so the 128 keys of one attention
// tile have theirs in 128 contiguous bytes.
//
// All of these are byte movers, bound by HBM at prompt size and by the launch at
// tick size.  Eight values per thread: Dh / 8 neighbouring lanes hold a row and
// find its maximum by shuffles.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "wfd_cache.cuh"
#include "wfd_common.cuh"
#include "wfd_model.cuh"

namespace wfd {

constexpr int kQ8ExpMax = 32;
enum : int { kErrNaN = 1 << 8 };  // a NaN in a row to be quantised (stored as 0)

// smallest e with a <= 448 * 2^e (448 = 1.75 * 2^8), unclamped; a >= 0, inf -> 120
__device__ __forceinline__ int q8_exponent(float a) {
  const uint32_t b = __float_as_uint(a);
  return (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
}
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((127 + e) << 23); }  // -126 <= e <= 127

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
// 4 codes -> 4 floats (exact)
__device__ __forceinline__ void e4m3x4_to_f(uint32_t w, float (&f)[4]) {
  const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
  const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
  const float2 fa = __half22float2(__half2(a)), fb = __half22float2(__half2(b));
  f[0] = fa.x; f[1] = fa.y; f[2] = fb.x; f[3] = fb.y;
}

// Quantise the row held by this thread's group of `lanes` neighbouring lanes (a
// power of two; every lane of the warp calls), 8 values each.  The largest |x| is
// found as an integer: a NaN's bits lie above those of infinity, so the same maximum
// tells whether the row holds one.
__device__ __forceinline__ uint32_t q8_max_bits(const float (&f)[8]) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, __float_as_uint(f[i]) & 0x7fffffffu);
  return a;
}
// ... of 8 packed bf16 (a NaN comes out as one)
__device__ __forceinline__ uint32_t q8_max_bits(const uint4& w) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
  const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
  const uint32_t u = *reinterpret_cast<const uint32_t*>(&m);
  return max(u << 16, u & 0xffff0000u) & 0x7fffffffu;
}
// a: q8_max_bits of f
__device__ __forceinline__ uint2 q8_quantise(float (&f)[8], uint32_t a, int lanes, int& e, bool& nan) {
  for (int o = lanes >> 1; o > 0; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
  nan = a > 0x7f800000u;
  if (__any_sync(0xffffffffu, nan)) {
    a = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (isnan(f[i])) f[i] = 0.f;
      a = max(a, __float_as_uint(f[i]) & 0x7fffffffu);
    }
    for (int o = lanes >> 1; o > 0; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
  }
  e = max(-kQ8ExpMax, min(kQ8ExpMax, q8_exponent(__uint_as_float(a))));
  const float s = exp2_int(-e);
  uint2 q;
  q.x = e4m3x2(f[0] * s, f[1] * s) | (e4m3x2(f[2] * s, f[3] * s) << 16);
  q.y = e4m3x2(f[4] * s, f[5] * s) | (e4m3x2(f[6] * s, f[7] * s) << 16);
  return q;
}

struct Q8Cache {
  uint8_t* k;
  uint8_t* v;
  int8_t* ke;
  int8_t* ve;
  int n_slots, n_seqs, max_seq, Hkv, Dh;
  __device__ __forceinline__ long long row(int slot, int seq, int pos) const {  // codes, in elements
    return (((long long)slot * n_seqs + seq) * max_seq + pos) * (long long)Hkv * Dh;
  }
  __device__ __forceinline__ long long exps(int slot, int seq) const {  // of head 0, position 0
    return ((long long)slot * n_seqs + seq) * (long long)Hkv * max_seq;
  }
};

// Rows src_row0 .. src_row0 + n - 1 of k_new / v_new (all heads) to (slot, seq,
// pos_of(j)), by the whole block; rows with pos_of(j) < 0 are left out.
template <typename T, typename PosOf>
__device__ __forceinline__ void q8_put_rows(const T* k_new, const T* v_new, long long src_row0, int n,
                                            const Q8Cache& c, int slot, int seq, PosOf pos_of, int* err) {
  const int lanes = c.Dh >> 3;
  const int per = c.Hkv * lanes;  // threads' worth of one row of K
  const int width = c.Hkv * c.Dh;
  const long long units = (long long)n * 2 * per;
  for (long long e0 = 0; e0 < units; e0 += blockDim.x) {
    const long long e = e0 + threadIdx.x;
    const int j = (int)(e / (2 * per)), r = (int)(e % (2 * per));
    const bool isv = r >= per;
    const int x = (isv ? r - per : r) * 8;
    const int pos = e < units ? pos_of(j) : -1;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (pos >= 0) Vec8<T>::load((isv ? v_new : k_new) + (src_row0 + j) * width + x, f);
    int ex;
    bool nan;
    const uint2 q = q8_quantise(f, q8_max_bits(f), lanes, ex, nan);
    if (pos >= 0) {
      *reinterpret_cast<uint2*>((isv ? c.v : c.k) + c.row(slot, seq, pos) + x) = q;
      const int h = x / c.Dh;
      if (x == h * c.Dh) (isv ? c.ve : c.ke)[c.exps(slot, seq) + (long long)h * c.max_seq + pos] = (int8_t)ex;
      if (nan) set_error(err, kErrNaN);
    }
  }
}

// write_tokens: one block per new row.  Where several rows of a call name the
// same place the last one is stored, as a loop over the rows would have it
// (codes and exponent of one row belong together, so a race between two would
// leave neither).
template <typename T>
__global__ void q8_append_kernel(const T* k_new, const T* v_new, const Q8Cache c, int32_t* lens, const int32_t* slots,
                                 const int32_t* seqs, const int32_t* positions, int n, int slot_offset, int* err) {
  griddep_wait();
  const int i = blockIdx.x;
  const int slot0 = slots[i], seq = seqs[i], pos = positions[i];
  const long long slot = (long long)slot0 + slot_offset;
  if (slot < 0 || slot >= c.n_slots || seq < 0 || seq >= c.n_seqs) {
    if (threadIdx.x == 0) set_error(err, kErrBadSlot);
    return;
  }
  if (pos < 0 || pos >= c.max_seq) {
    if (threadIdx.x == 0) set_error(err, kErrBadPos);
    return;
  }
  int later = 0;
  for (int j = i + 1 + threadIdx.x; j < n; j += blockDim.x)
    later |= (positions[j] == pos && seqs[j] == seq && slots[j] == slot0) ? 1 : 0;
  if (__syncthreads_or(later)) return;
  q8_put_rows(k_new, v_new, i, 1, c, (int)slot, seq, [&](int) { return pos; }, err);
  if (threadIdx.x == 0 && lens != nullptr) atomicMax(lens + (long long)slot * c.n_seqs + seq, pos + 1);
}

// The prompt write and the read-back move blocks of 32 positions x up to 512 values
// of the row (8 heads of 64, 4 of 128): their exponents, one byte per head and
// position, 32 of a head contiguous, pass through shared memory, so that they are
// read and written as whole 32-byte sectors, and blocks are small enough that a
// single prompt fills the GPU.  A thread keeps its place in the row and steps through
// the positions; all its loads are in flight before the first is used.  (Prompt of
// 64 x 1024 x 24 x 64, bf16: 109 us written, 93 us read back, 92 us each of HBM
// time; whole rows a block, with divisions by the head count: 167 and 103.)
constexpr int kQ8Chunk = 32;
constexpr int kQ8Threads = 256;
constexpr int kQ8MaxHeads = 1024;  // kv heads
constexpr int kQ8Span = 512;       // values of a row per block
constexpr int kQ8Heads = kQ8Span / 16;  // heads per block, at most

// write_prefill: k, v (n_seqs, L, Hkv, Dh) -> positions [0, L) of `slot`.
// Block (chunk, sequence, part of the row of K or V).
template <typename T>
__global__ void __launch_bounds__(kQ8Threads)
    q8_prefill_kernel(const T* k, const T* v, const Q8Cache c, int32_t* lens, int slot, int L, int log2_dh, int* err) {
  griddep_wait();
  __shared__ int8_t s_exp[kQ8Heads][kQ8Chunk];
  const int p0 = blockIdx.x * kQ8Chunk, seq = blockIdx.y;
  const bool isv = (blockIdx.z & 1) != 0;
  const int width = c.Hkv * c.Dh;
  const int x0 = (blockIdx.z >> 1) * kQ8Span;
  const int np = min(kQ8Chunk, L - p0);
  const int lanes = c.Dh >> 3;
  constexpr int PER = kQ8Span / 8;                 // threads of one position
  constexpr int STEP = kQ8Threads / PER;           // positions a pass
  constexpr int U = kQ8Chunk / STEP;
  const int xi = (threadIdx.x % PER) * 8, x = x0 + xi, j0 = threadIdx.x / PER;
  const bool on = x < width;
  const T* src = (isv ? v : k) + ((long long)seq * L + p0) * width + x;
  uint8_t* dst = (isv ? c.v : c.k) + c.row(slot, seq, p0) + x;
  constexpr int NV = (int)sizeof(T) / 2;  // 16-byte vectors of 8 values
  uint4 raw[U][NV];                        // kept as loaded: unpacked, the rows would take twice the registers
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int j = j0 + u * STEP;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      raw[u][i] = make_uint4(0, 0, 0, 0);
      if (on && j < np) raw[u][i] = ld_nc_v4(reinterpret_cast<const uint4*>(src + (long long)j * width) + i);
    }
  }
  bool any_nan = false;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int j = j0 + u * STEP;
    int ex;
    bool nan;
    float f[8];
    constexpr int EV = 8 / NV;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float part[EV];
      Elem<T>::unpack(raw[u][i], part);
#pragma unroll
      for (int e = 0; e < EV; ++e) f[i * EV + e] = part[e];
    }
    uint32_t a;
    if constexpr (NV == 1)
      a = q8_max_bits(raw[u][0]);
    else
      a = q8_max_bits(f);
    const uint2 q = q8_quantise(f, a, lanes, ex, nan);
    if (on && j < np) {
      *reinterpret_cast<uint2*>(dst + (long long)j * width) = q;
      if ((xi & (c.Dh - 1)) == 0) s_exp[xi >> log2_dh][j] = (int8_t)ex;
      any_nan |= nan;
    }
  }
  if (any_nan) set_error(err, kErrNaN);
  __syncthreads();
  const int h0 = x0 >> log2_dh, nh = min(kQ8Span, width - x0) >> log2_dh;
  int8_t* edst = (isv ? c.ve : c.ke) + c.exps(slot, seq) + (long long)h0 * c.max_seq + p0;
  for (int t = threadIdx.x; t < nh * kQ8Chunk; t += kQ8Threads) {
    const int h = t / kQ8Chunk, j = t % kQ8Chunk;
    if (j < np) edst[(long long)h * c.max_seq + j] = s_exp[h][j];
  }
  if (lens != nullptr && blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0)
    atomicMax(lens + (long long)slot * c.n_seqs + seq, L);
}

// Read back: segment i dequantises positions [0, cu_k[i+1] - cu_k[i]) of
// (slots[i], seqs[i]) into rows cu_k[i].. of k_pack / v_pack (total rows each).
// Block (chunk stride, segment, part of the row of K or V).
template <typename T>
__global__ void __launch_bounds__(kQ8Threads)
    q8_gather_kernel(const Q8Cache c, T* k_pack, T* v_pack, const int32_t* slots, const int32_t* seqs,
                     const int32_t* cu_k, long long total, int log2_dh, int* err) {
  griddep_wait();
  __shared__ int8_t s_exp[kQ8Heads][kQ8Chunk];
  const int i = blockIdx.y;
  const bool isv = (blockIdx.z & 1) != 0;
  const int slot = slots[i], seq = seqs[i];
  const long long k0 = cu_k[i], len = (long long)cu_k[i + 1] - k0;
  const bool ok_slot = slot >= 0 && slot < c.n_slots && seq >= 0 && seq < c.n_seqs;
  if (!ok_slot || len < 0 || len > c.max_seq || k0 < 0 || k0 + len > total) {
    if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.z == 0) set_error(err, ok_slot ? kErrBadPos : kErrBadSlot);
    return;
  }
  const int width = c.Hkv * c.Dh;
  const int x0 = (blockIdx.z >> 1) * kQ8Span;
  constexpr int PER = kQ8Span / 8, STEP = kQ8Threads / PER, U = kQ8Chunk / STEP;
  const int xi = (threadIdx.x % PER) * 8, x = x0 + xi, j0 = threadIdx.x / PER;
  const bool on = x < width;
  const int h0 = x0 >> log2_dh, nh = min(kQ8Span, width - x0) >> log2_dh;
  const int8_t* esrc = (isv ? c.ve : c.ke) + c.exps(slot, seq) + (long long)h0 * c.max_seq;
  for (long long p0 = (long long)blockIdx.x * kQ8Chunk; p0 < len; p0 += (long long)gridDim.x * kQ8Chunk) {
    const int np = (int)min((long long)kQ8Chunk, len - p0);
    const uint8_t* src = (isv ? c.v : c.k) + c.row(slot, seq, (int)p0) + x;
    T* dst = (isv ? v_pack : k_pack) + (k0 + p0) * width + x;
    uint2 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * STEP;
      q[u] = on && j < np ? *reinterpret_cast<const uint2*>(src + (long long)j * width) : make_uint2(0, 0);
    }
    __syncthreads();  // the previous chunk's exponents are read
    for (int t = threadIdx.x; t < nh * kQ8Chunk; t += kQ8Threads) {
      const int h = t / kQ8Chunk, j = t % kQ8Chunk;
      if (j < np) s_exp[h][j] = esrc[(long long)h * c.max_seq + p0 + j];
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * STEP;
      if (on && j < np) {
        const float s = exp2_int(s_exp[xi >> log2_dh][j]);
        float a[4], b[4];
        e4m3x4_to_f(q[u].x, a);
        e4m3x4_to_f(q[u].y, b);
        const float f[8] = {a[0] * s, a[1] * s, a[2] * s, a[3] * s, b[0] * s, b[1] * s, b[2] * s, b[3] * s};
        Vec8<T>::store(dst + (long long)j * width, f);
      }
    }
  }
}

// Accept commit of verify windows, as commit_window_kernel: accepted rows move in
// order to pos0, pos0 + 1, ..., one at a time with a barrier between them (a row
// moves only to a position below its own), codes and exponents alike.
__global__ void __launch_bounds__(kCommitThreads)
    q8_commit_window_kernel(const Q8Cache c, int32_t* lens, const wfd_item* items, const int32_t* accept_len,
                            const uint8_t* accept_mask, int32_t* acc_rows, int32_t* acc_count, int n_rows,
                            int slot_offset, int* err) {
  griddep_wait();
  const wfd_item it = items[blockIdx.x];
  const long long slot = (long long)it.slot + slot_offset;
  const bool ok_slot = slot >= 0 && slot < c.n_slots && it.seq >= 0 && it.seq < c.n_seqs;
  const bool ok_pos = it.pos0 >= 0 && it.q_len >= 0 && (long long)it.pos0 + it.q_len <= c.max_seq;
  const bool ok_rows = it.q_row0 >= 0 && (long long)it.q_row0 + it.q_len <= n_rows && it.q_len <= 1024;
  if (!ok_slot || !ok_pos || !ok_rows) {
    if (threadIdx.x == 0) set_error(err, !ok_slot ? kErrBadSlot : !ok_pos ? kErrBadPos : kErrBadRows);
    return;
  }
  __shared__ int s_rank[1024];
  if (threadIdx.x == 0) {
    int n = 0;
    for (int j = 0; j < it.q_len; ++j) {
      const bool acc = accept_len != nullptr ? j < accept_len[blockIdx.x] : accept_mask[it.q_row0 + j] != 0;
      s_rank[j] = acc ? n++ : -1;
    }
    if (acc_count != nullptr) acc_count[blockIdx.x] = n;
    lens[slot * c.n_seqs + it.seq] = it.pos0 + n;
  }
  __syncthreads();
  const int rb = c.Hkv * c.Dh;
  const long long row0 = c.row((int)slot, it.seq, it.pos0), e0 = c.exps((int)slot, it.seq) + it.pos0;
  for (int j = 0; j < it.q_len; ++j) {
    const int rk = s_rank[j];
    if (rk < 0) continue;
    if (acc_rows != nullptr && threadIdx.x == 0) acc_rows[it.q_row0 + rk] = it.q_row0 + j;
    if (rk == j) continue;
    const long long src = row0 + (long long)j * rb, dst = row0 + (long long)rk * rb;
    for (int o = threadIdx.x * 16; o < rb; o += kCommitThreads * 16) {
      const uint4 kv = ld_cg_v4(c.k + src + o);
      const uint4 vv = ld_cg_v4(c.v + src + o);
      *reinterpret_cast<uint4*>(c.k + dst + o) = kv;
      *reinterpret_cast<uint4*>(c.v + dst + o) = vv;
    }
    for (int h = threadIdx.x; h < c.Hkv; h += kCommitThreads) {
      const long long eo = e0 + (long long)h * c.max_seq;
      c.ke[eo + rk] = *const_cast<volatile int8_t*>(c.ke + eo + j);
      c.ve[eo + rk] = *const_cast<volatile int8_t*>(c.ve + eo + j);
    }
    __syncthreads();
  }
}

}  // namespace wfd
