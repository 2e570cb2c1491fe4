// kv_device.cuh -- device helpers of the paged key/value kernels: which
// sequence a row belongs to, where a token lies, and the value types.
#pragma once
#include <cuda_bf16.h>
#include "kv.h"
#include "kv_ptx.cuh"

namespace iq {

// An entry of row_start, within the batch's rows whatever the caller wrote:
// counts and products of rows cannot overflow.
__device__ __forceinline__ int kv_row(const KvBatch& b, int at) { return min(max(at, 0), b.rows); }

// Sequence of `row` (warp-wide; every lane returns it), the row's index in it,
// the sequence's rows and its first position; -1 when the row lies behind the
// last sequence.  row_start ascends; each round narrows the range 32-fold, and
// the last round's loads are the answer's.
struct KvSeq {
  int seq, in_seq, rows;
  int64_t pos;
};
__device__ __forceinline__ KvSeq kv_seq_of_row(const KvBatch& b, int row, int lane) {
  if (!b.row_start) return {0, row, b.rows, b.position[0]};
  int lo = 0, n = b.seqs;  // the sequences that end at or before `row` number lo .. lo + n
  while (n > 32) {
    const int step = (n + 31) >> 5;
    const int at = lo + (lane + 1) * step;  // row_start[at] ends the lane's group
    const bool before = (lane + 1) * step <= n && b.row_start[at] <= row;
    const int full = __popc(__ballot_sync(0xffffffffu, before));
    lo += full * step;
    n = min(step, b.seqs - lo);
  }
  const int s = min(lo + lane, b.seqs - 1);
  const int begin = kv_row(b, b.row_start[s]), end = kv_row(b, b.row_start[s + 1]), pos = b.position[s];
  const uint32_t past = __ballot_sync(0xffffffffu, lane < n && end > row);
  if (!past) return {-1, 0, 0, 0};
  const int at = __ffs(past) - 1;
  const int first = __shfl_sync(0xffffffffu, begin, at);
  return {row < first ? -1 : lo + at, row - first, __shfl_sync(0xffffffffu, end, at) - first,
          __shfl_sync(0xffffffffu, pos, at)};
}

// Page that holds position `pos` (>= 0) of sequence `s`; -1 (and the pool's
// flag) where the table or the pool does not reach.
__device__ __forceinline__ int kv_page(const KvPool& p, const KvBatch& b, int s, int64_t pos) {
  const int64_t col = pos >> p.page_shift;
  if (col < b.table_cols) {
    const int page = b.table[(int64_t)s * b.table_ld + col];
    if (page >= 0 && page < p.pages) return page;
  }
  atomicOr(p.flag, kKvBadPage);
  return -1;
}

// Byte offset of 16-byte chunk c of token t inside a page's head.
template <int FMT, int HD>
__device__ __forceinline__ int kv_chunk(int t, int c, int page_tokens) {
  if constexpr (FMT == kKvI8) return t * HD + ((c ^ i8_swizzle(t, HD)) << 4);
  return ((c >> 3) * page_tokens + t) * 128 + (((c & 7) ^ (t & 7)) << 4);
}

template <class T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f(float x) { return x; }
template <>
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }

// N contiguous elements; `vec`: the address is a multiple of min(16, N * sizeof(T)).
template <class T, int N>
__device__ __forceinline__ void load_n(const T* p, bool vec, float (&x)[N]) {
  constexpr int kB = N * (int)sizeof(T), kW = kB < 16 ? kB : 16;
  if (vec) {
    alignas(16) T v[N];
#pragma unroll
    for (int i = 0; i < kB / kW; i++) {
      if constexpr (kW == 16) reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(p)[i];
      else if constexpr (kW == 8) reinterpret_cast<uint2*>(v)[i] = reinterpret_cast<const uint2*>(p)[i];
      else reinterpret_cast<uint32_t*>(v)[i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = to_f(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = to_f(p[i]);
  }
}
template <class T, int N>
__device__ __forceinline__ void store_n(T* p, bool vec, const float (&x)[N]) {
  constexpr int kB = N * (int)sizeof(T), kW = kB < 16 ? kB : 16;
  if (vec) {
    alignas(16) T v[N];
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = from_f<T>(x[i]);
#pragma unroll
    for (int i = 0; i < kB / kW; i++) {
      if constexpr (kW == 16) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(v)[i];
      else if constexpr (kW == 8) reinterpret_cast<uint2*>(p)[i] = reinterpret_cast<const uint2*>(v)[i];
      else reinterpret_cast<uint32_t*>(p)[i] = reinterpret_cast<const uint32_t*>(v)[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) p[i] = from_f<T>(x[i]);
  }
}

// B bytes as one access.
template <int B>
__device__ __forceinline__ void copy_bytes(void* dst, const void* src) {
  if constexpr (B == 16) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
  else if constexpr (B == 8) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(src);
  else if constexpr (B == 4) *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(src);
  else *reinterpret_cast<uint16_t*>(dst) = *reinterpret_cast<const uint16_t*>(src);
}

// Exponent e of the power of two that brings a vector of largest magnitude
// `amax` to [2^14, 2^15) as x / 2^e: inside f16's normal range with 28
// binades below.  0 for a non-finite maximum; at least -126, so that 2^e and
// 2^-e are f32 normals.
__device__ __forceinline__ int f16_exponent(float amax) {
  const int be = (__float_as_int(amax) >> 23) & 255;
  if (be == 255) return 0;
  return max(max(be, 1) - 127 - 14, -126);
}

}  // namespace iq
