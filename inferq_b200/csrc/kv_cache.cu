// kv_cache.cu -- the paged key/value cache: rows quantised as they are
// written, vectors read back, and the C ABI of iq_kv.
//
// Formats, per token, KV head and of keys and values each, amax = max |x|:
//   i8   code q = the integer nearest to 127 x / amax (ties to even), scale =
//        amax / 127, value q * scale
//   f16  x / 2^e as f16 (one rounding of 2^-11 relative), scale 2^e, with
//        amax / 2^e in [2^14, 2^15): f16 rows and bf16 rows within 28 binades
//        of their maximum are kept exactly, and no magnitude overflows
// A vector that holds a NaN or an infinity is stored as zeros with a NaN
// scale: it reads back as NaN, and in attention it reaches the rows that see
// it and no others (a zero weight never meets a NaN element).
//
// The code is the rounding of the real quotient, not of a float one: the f32
// product x * (127 / amax) (two roundings of 2^-24, so at most 127 * 2^-23 <
// 2^-15 off) decides except within 2^-15 of a border between two codes, where
// 64 bits decide: 127 x is exact there, and a quotient of 24-bit numbers that
// is no tie is further from one than the division rounds.  So a code depends
// on nothing but x and amax.
//
// What bounds both kernels.  The bytes, if the instructions allow: a warp's
// 32 bytes in and out a lane come with some 4 instructions an element, so the
// arithmetic is written for few of them (rounding and byte by one addition of
// 1.5 * 2^23 + 128, two f32 an operation, one test for all of a lane's
// borders), and a row's place is found by one thread, not by its warp.
// 16384 bf16 rows of 2 heads of 256 into i8: 18 us (2.8 TB/s; a call of 50 MB
// is mostly start and end); 65536 f32 rows read back: 61 us (5.5 TB/s).
#include <cmath>
#include <memory>
#include <new>
#include <type_traits>
#include "kv_device.cuh"

namespace iq {
namespace {

constexpr float kMagic = 12582912.f + 128.f;  // v + kMagic holds rint(v) + 128 in its low byte, |v| <= 127

__device__ __forceinline__ float max_nan_abs(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(fabsf(a)), "f"(fabsf(b)));
  return d;
}
// Low bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(float a, float b, float c, float d) {
  const uint32_t x = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040);
  const uint32_t y = __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040);
  return __byte_perm(x, y, 0x5410);
}

// (A call: inlined sixteen times it does not fit the instruction cache.)
__device__ __noinline__ float code_f64(float x, float amax) {
  return (float)rint(127.0 * (double)x / (double)amax) + kMagic;
}

// Biased codes of N elements; amax finite and above zero.  kShort: x and amax
// have at most 11 significant bits (f16 and bf16 rows, up to 40% of whose
// vectors meet a tie).  127 x is exact then, and a quotient that is no tie lies
// at least 2^-20 of itself from one ((254 mx 2^k - (2n + 1) ma) / 2 ma is a
// multiple of 2^k / 2 ma with ma < 2^11 and 2^k >= q / 254): a quotient
// corrected by its exact remainder is a tie where the real one is, and on the
// right side otherwise.
template <int N, bool kShort>
__device__ __forceinline__ void codes_i8(const float (&x)[N], float amax, uint8_t* out) {
  float t[N];
  if (!(amax > 0x1p-100f && amax < 0x1p100f)) {  // a factor or a product would leave f32's normals
#pragma unroll  // (an index that varies would put the arrays in local memory)
    for (int j = 0; j < N; j++) t[j] = code_f64(x[j], amax);
  } else if constexpr (kShort) {
    const float inv = __fdiv_rn(1.f, amax);
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const float2 num = kvp::mul2(make_float2(x[j], x[j + 1]), make_float2(127.f, 127.f));
      float2 q = kvp::mul2(num, make_float2(inv, inv));
      const float2 left = kvp::fma2(make_float2(-q.x, -q.y), make_float2(amax, amax), num);
      q = kvp::fma2(left, make_float2(inv, inv), q);
      q = kvp::add2(q, make_float2(kMagic, kMagic));
      t[j] = q.x;
      t[j + 1] = q.y;
    }
  } else {
    const float c = __fdiv_rn(127.f, amax);
    float far = 0.f, d[N];
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const float2 v = kvp::mul2(make_float2(x[j], x[j + 1]), make_float2(c, c));
      const float2 u = kvp::add2(v, make_float2(kMagic, kMagic));
      const float2 r = kvp::add2(u, make_float2(-kMagic, -kMagic));
      const float2 e = kvp::add2(v, make_float2(-r.x, -r.y));
      t[j] = u.x;
      t[j + 1] = u.y;
      d[j] = fabsf(e.x);
      d[j + 1] = fabsf(e.y);
      far = fmaxf(far, fmaxf(d[j], d[j + 1]));
    }
    constexpr float kNear = 0.5f - 0x1p-15f;
    if (far > kNear) {
#pragma unroll
      for (int j = 0; j < N; j++)
        if (d[j] > kNear) t[j] = code_f64(x[j], amax);
    }
  }
  if constexpr (N == 2) {
    *reinterpret_cast<uint16_t*>(out) = (uint16_t)__byte_perm(__float_as_uint(t[0]), __float_as_uint(t[1]), 0x0040);
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 4)
      reinterpret_cast<uint32_t*>(out)[j / 4] = low_bytes(t[j], t[j + 1], t[j + 2], t[j + 3]);
  }
}

// Where the CTA's items (row, KV head) lie, found by one thread each: a page
// and a token in it, kNoRow behind the last sequence, kPadding at a negative
// position, -1 outside the table or the pool.
constexpr int kNoRow = -2, kPadding = -3, kMostItems = 32;

__device__ __forceinline__ int2 place_of(const KvPool& p, const KvBatch& b, int row) {
  int s = 0, first = 0;
  if (b.row_start) {
    int hi = b.seqs;  // the first sequence that ends behind the row
    while (s < hi) {
      const int mid = (s + hi) >> 1;
      if (b.row_start[mid + 1] <= row) s = mid + 1;
      else hi = mid;
    }
    if (s == b.seqs) return make_int2(kNoRow, 0);
    first = kv_row(b, b.row_start[s]);
    if (row < first) return make_int2(kNoRow, 0);
  }
  const int64_t pos = (int64_t)b.position[s] + (row - first);
  if (pos < 0) return make_int2(kPadding, 0);
  return make_int2(kv_page(p, b, s, pos), (int)pos & (p.page_tokens - 1));
}

// A CTA takes 8 `turns` items, a warp one in turn: keys and values of a row's
// head.  Loads are hidden by the SM's other warps: at most 51 registers, five
// CTAs an SM (with 88, for the next item's loads in registers, two CTAs fitted
// and 16384 bf16 rows took 37 us).
template <class T, int HD, int FMT>
__global__ void __launch_bounds__(256, 5) kv_append_kernel(const __grid_constant__ KvPool p, const __grid_constant__ KvBatch b,
                                                        KvTensor k, KvTensor v, bool vec, int turns) {
  constexpr int N = HD / 32;
  constexpr int kB = FMT == kKvI8 ? N : 2 * N;  // bytes a lane
  __shared__ int2 places[kMostItems];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t items = (uint32_t)b.rows * p.nkv, item0 = blockIdx.x * 8 * turns;  // (below 2^31: checked by the caller)
  auto load = [&](uint32_t item, float (&x)[2][N]) {
    if (item >= items) return;
    const int64_t row = item / (uint32_t)p.nkv, head = item - (uint32_t)row * p.nkv;
    load_n<T, N>(static_cast<const T*>(k.p) + row * k.row + head * k.head + lane * N, vec, x[0]);
    load_n<T, N>(static_cast<const T*>(v.p) + row * v.row + head * v.head + lane * N, vec, x[1]);
  };
  float x[2][N];
  if (turns == 1) load(item0 + warp, x);  // (under the search)
  if (threadIdx.x < 8 * turns && item0 + threadIdx.x < items)
    places[threadIdx.x] = place_of(p, b, (int)((item0 + threadIdx.x) / (uint32_t)p.nkv));
  __syncthreads();
  for (int turn = 0; turn < turns; turn++) {
    const uint32_t item = item0 + turn * 8 + warp;
    if (item >= items) return;
    if (turns > 1) load(item, x);
    const int2 at = places[turn * 8 + warp];
    if (at.x >= 0) {
      const int64_t run = (int64_t)at.x * p.nkv + item % (uint32_t)p.nkv;
      const int64_t off = run * kv_head_bytes(FMT, HD, p.page_tokens) +
                          kv_chunk<FMT, HD>(at.y, lane * kB >> 4, p.page_tokens) + (lane * kB & 15);
#pragma unroll
      for (int w = 0; w < 2; w++) {
        float m = max_nan_abs(x[w][0], x[w][1]);
#pragma unroll
        for (int j = 2; j < N; j++) m = max_nan_abs(m, x[w][j]);
        // as bits a NaN is above every number
        const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
        const float amax = __uint_as_float(bits);
        const bool finite = bits < 0x7f800000u;
        float scale;
        alignas(16) uint8_t held[kB];
        if constexpr (FMT == kKvI8) {
          scale = finite ? __fdiv_rn(amax, 127.f) : __int_as_float(0x7fffffff);
          if (finite && bits) {
            codes_i8<N, sizeof(T) == 2>(x[w], amax, held);
          } else {
#pragma unroll
            for (int j = 0; j < N; j++) held[j] = 128;
          }
        } else {
          const int e = f16_exponent(amax);
          scale = finite ? kvp::pow2i(e) : __int_as_float(0x7fffffff);
          const float f = kvp::pow2i(-e);
#pragma unroll
          for (int j = 0; j < N; j += 2)
            reinterpret_cast<__half2*>(held)[j / 2] =
                finite ? __floats2half2_rn(x[w][j] * f, x[w][j + 1] * f) : __floats2half2_rn(0.f, 0.f);
        }
        copy_bytes<kB>((w ? p.v : p.k) + off, held);
        if (lane == 0) (w ? p.vs : p.ks)[run * p.page_tokens + at.y] = scale;
      }
    }
  }
}

// The reverse; rows at negative positions or behind the table read as zeros.
template <class T, int HD, int FMT>
__global__ void __launch_bounds__(256, 6) kv_read_kernel(const __grid_constant__ KvPool p, const __grid_constant__ KvBatch b,
                                                      KvTensor k, KvTensor v, bool vec, int turns) {
  constexpr int N = HD / 32;
  constexpr int kB = FMT == kKvI8 ? N : 2 * N;
  __shared__ int2 places[kMostItems];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t items = (uint32_t)b.rows * p.nkv, item0 = blockIdx.x * 8 * turns;
  if (threadIdx.x < 8 * turns && item0 + threadIdx.x < items)
    places[threadIdx.x] = place_of(p, b, (int)((item0 + threadIdx.x) / (uint32_t)p.nkv));
  __syncthreads();
#pragma unroll 1  // (two turns unrolled: 71 us instead of 61 for 65536 f32 rows, by their registers)
  for (int turn = 0; turn < turns; turn++) {
    const uint32_t item = item0 + turn * 8 + warp;
    if (item >= items) return;
    const int2 at = places[turn * 8 + warp];
    if (at.x == kNoRow) continue;
    const int64_t row = item / (uint32_t)p.nkv, head = item - (uint32_t)row * p.nkv, run = (int64_t)at.x * p.nkv + head;
    const int64_t off = run * kv_head_bytes(FMT, HD, p.page_tokens) +
                        kv_chunk<FMT, HD>(at.y, lane * kB >> 4, p.page_tokens) + (lane * kB & 15);
    float x[2][N];
#pragma unroll
    for (int w = 0; w < 2; w++) {
      alignas(16) uint8_t held[kB];
      float scale = 0.f;
      if (at.x >= 0) {
        copy_bytes<kB>(held, (w ? p.v : p.k) + off);
        scale = (w ? p.vs : p.ks)[run * p.page_tokens + at.y];
      }
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        float2 f;
        if constexpr (FMT == kKvI8) {
          // 2^23 + u as f32, minus 2^23 + 128: the code, exactly
          f = make_float2(__uint_as_float(0x4b000000u | held[j]), __uint_as_float(0x4b000000u | held[j + 1]));
          f = kvp::add2(f, make_float2(-8388736.f, -8388736.f));
        } else {
          f = __half22float2(reinterpret_cast<const __half2*>(held)[j / 2]);
        }
        f = kvp::mul2(f, make_float2(scale, scale));
        x[w][j] = at.x < 0 ? 0.f : f.x;
        x[w][j + 1] = at.x < 0 ? 0.f : f.y;
      }
    }
    store_n<T, N>(static_cast<T*>(k.p) + row * k.row + head * k.head + lane * N, vec, x[0]);
    store_n<T, N>(static_cast<T*>(v.p) + row * v.row + head * v.head + lane * N, vec, x[1]);
  }
}

// The flag read and cleared in one step: what another stream records meanwhile
// stays for the next reader.
__global__ void kv_take_flag_kernel(int* flag, int* out) { *out = atomicExch(flag, 0); }
constexpr int kStatusWords = 63;  // behind the flag: one for each of so many iq_kv_status calls at once

// Whether every lane's elements start on a multiple of their own size (16
// bytes at most): base and strides in bytes.
bool vector_ok(const KvTensor& t, int item, int hd) {
  const int w = std::min(16, hd / 32 * item);
  return ((uintptr_t)t.p | (uintptr_t)(t.row * item) | (uintptr_t)(t.head * item)) % w == 0;
}

template <class T>
cudaError_t launch(bool append, const KvPool& p, const KvBatch& b, const KvTensor& k, const KvTensor& v,
                   cudaStream_t st) {
  const bool vec = vector_ok(k, sizeof(T), p.hd) && vector_ok(v, sizeof(T), p.hd);
  // items a warp: one, until 64 warps an SM have four each
  const int64_t items = (int64_t)b.rows * p.nkv;
  const int turns = items >= 4 * 64 * 148 ? kMostItems / 8 : 1;
  const unsigned grid = (unsigned)ceil_div(items, 8 * turns);
  auto go = [&](auto hd, auto fmt) {
    constexpr int HD = decltype(hd)::value, FMT = decltype(fmt)::value;
    if (append) kv_append_kernel<T, HD, FMT><<<grid, 256, 0, st>>>(p, b, k, v, vec, turns);
    else kv_read_kernel<T, HD, FMT><<<grid, 256, 0, st>>>(p, b, k, v, vec, turns);
    return cudaGetLastError();
  };
  using I8 = std::integral_constant<int, kKvI8>;
  using H = std::integral_constant<int, kKvF16>;
  auto by_format = [&](auto hd) { return p.format == kKvI8 ? go(hd, I8()) : go(hd, H()); };
  switch (p.hd) {
    case 64: return by_format(std::integral_constant<int, 64>());
    case 128: return by_format(std::integral_constant<int, 128>());
    case 256: return by_format(std::integral_constant<int, 256>());
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t by_type(bool append, const KvPool& p, const KvBatch& b, int dtype, const KvTensor& k, const KvTensor& v,
                    cudaStream_t st) {
  switch (dtype) {
    case F32: return launch<float>(append, p, b, k, v, st);
    case F16: return launch<__half>(append, p, b, k, v, st);
    case BF16: return launch<__nv_bfloat16>(append, p, b, k, v, st);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

cudaError_t kv_append_launch(const KvPool& p, const KvBatch& b, int dtype, const KvTensor& k, const KvTensor& v,
                             cudaStream_t st) {
  return by_type(true, p, b, dtype, k, v, st);
}
cudaError_t kv_read_launch(const KvPool& p, const KvBatch& b, int dtype, const KvTensor& k, const KvTensor& v,
                           cudaStream_t st) {
  return by_type(false, p, b, dtype, k, v, st);
}

int kv_create(int format, int kv_heads, int head_dim, int page_tokens, int64_t pages, int* flag, iq_kv& c) {
  IQ_CUDA(cudaGetDevice(&c.device));
  // (below 2^31 * 2^8 heads * 2^17 bytes: no overflow)
  const size_t bytes = (size_t)pages * kv_heads * (size_t)kv_head_bytes(format, head_dim, page_tokens);
  const size_t sbytes = (size_t)pages * kv_heads * page_tokens * 4;
  DevBuf* bufs[] = {&c.k, &c.v, &c.ks, &c.vs, &c.flag};
  const size_t sizes[] = {bytes, bytes, sbytes, sbytes, (1 + kStatusWords) * sizeof(int)};
  const int n = flag ? 4 : 5;
  for (int i = 0; i < n; i++) {
    const cudaError_t e = bufs[i]->reserve(sizes[i]);
    if (e == cudaErrorMemoryAllocation) cudaGetLastError();  // not sticky: clear it
    IQ_CHECK(e != cudaErrorMemoryAllocation, IQ_ENOMEM, "no room for a cache of %lld pages (%zu bytes)",
             (long long)pages, 2 * (bytes + sbytes));
    IQ_CUDA(e);
  }
  // Every token of the pool is finite from the start: kernels may read
  // tokens of a page that are not written yet, with weight zero.
  for (int i = 0; i < n; i++) IQ_CUDA(cudaMemset(bufs[i]->p, 0, sizes[i]));
  IQ_CUDA(cudaStreamSynchronize(nullptr));
  KvPool& p = c.pool;
  p.k = c.k.as<uint8_t>();
  p.v = c.v.as<uint8_t>();
  p.ks = c.ks.as<float>();
  p.vs = c.vs.as<float>();
  p.flag = flag ? flag : c.flag.as<int>();
  p.pages = pages;
  p.nkv = kv_heads;
  p.hd = head_dim;
  p.page_tokens = page_tokens;
  p.page_shift = __builtin_ctz((unsigned)page_tokens);
  p.format = format;
  return IQ_OK;
}

}  // namespace iq

using namespace iq;

namespace {

// A call runs on the cache's device whatever the thread's current one is.
struct OnDevice {
  int before = -1;
  cudaError_t err;
  explicit OnDevice(int device) {
    int cur = 0;
    err = cudaGetDevice(&cur);
    if (err == cudaSuccess && cur != device) {
      err = cudaSetDevice(device);
      if (err == cudaSuccess) before = cur;
    }
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

int check_batch(const char* name, const iq_kv_batch* in, KvBatch& b) {
  IQ_CHECK(in, IQ_EINVAL, "%s: null batch", name);
  IQ_CHECK(in->rows >= 0 && in->seqs >= 0, IQ_EINVAL, "%s: %d rows of %d sequences", name, in->rows, in->seqs);
  IQ_CHECK(in->table_cols >= 0 && in->table_ld >= in->table_cols, IQ_EINVAL,
           "%s: a block table of %d columns cannot have rows %lld apart", name, in->table_cols,
           (long long)in->table_ld);
  if (in->rows && in->seqs) {
    IQ_CHECK(in->table && in->position, IQ_EINVAL, "%s: null block table or positions", name);
    IQ_CHECK(in->row_start || in->seqs == 1, IQ_EINVAL, "%s: %d sequences need row_start", name, in->seqs);
  }
  b = {};
  b.table = in->table;
  b.position = in->position;
  b.row_start = in->row_start;
  b.table_ld = in->table_ld;
  b.seqs = in->seqs;
  b.table_cols = in->table_cols;
  b.rows = in->rows;
  return IQ_OK;
}

int check_type(const char* name, int dtype) {
  IQ_CHECK(dtype == IQ_F32 || dtype == IQ_F16 || dtype == IQ_BF16, IQ_EUNSUPPORTED,
           "%s: rows of dtype %d; expected F32, F16 or BF16", name, dtype);
  return IQ_OK;
}

int check_tensor(const char* name, const char* what, const KvTensor& t, int64_t rows, int heads, int hd, int dtype,
                 bool written) {
  const void* p = t.p;
  const int64_t row = t.row, head = t.head;
  const int item = dtype == IQ_F32 ? 4 : 2;
  IQ_CHECK(p, IQ_EINVAL, "%s: null %s", name, what);
  IQ_CHECK((uintptr_t)p % item == 0, IQ_EINVAL, "%s: %s is not aligned to its element", name, what);
  IQ_CHECK(row >= 0 && head >= 0, IQ_EINVAL, "%s: negative stride of %s", name, what);
  // what is written must not lie on itself, in either order of the axes
  const bool by_row = (heads == 1 || head >= hd) && (rows == 1 || row >= (heads - 1) * head + hd);
  const bool by_head = (rows == 1 || row >= hd) && (heads == 1 || head >= (rows - 1) * row + hd);
  IQ_CHECK(!written || by_row || by_head, IQ_EINVAL, "%s: strides %lld and %lld put the heads of %s on one another",
           name, (long long)row, (long long)head, what);
  return IQ_OK;
}

int rows_call(const char* name, bool append, const iq_kv* c, const iq_kv_batch* batch, int dtype, const KvTensor& k,
              const KvTensor& v, void* stream) {
  clear_error();
  IQ_CHECK(c, IQ_EINVAL, "%s: null cache", name);
  KvBatch b;
  if (int rc = check_batch(name, batch, b)) return rc;
  if (int rc = check_type(name, dtype)) return rc;
  if (!b.rows || !b.seqs) return IQ_OK;
  const KvPool& p = c->pool;
  IQ_CHECK((int64_t)b.rows * p.nkv < (1ll << 31) - 8, IQ_EINVAL, "%s: %d rows of %d KV heads are too many", name, b.rows,
           p.nkv);
  if (int rc = check_tensor(name, "keys", k, b.rows, p.nkv, p.hd, dtype, !append)) return rc;
  if (int rc = check_tensor(name, "values", v, b.rows, p.nkv, p.hd, dtype, !append)) return rc;
  IQ_CHECK(append || k.p != v.p, IQ_EINVAL, "%s: keys and values go to one place", name);
  OnDevice on(c->device);
  IQ_CUDA(on.err);
  IQ_CUDA(by_type(append, p, b, dtype, k, v, static_cast<cudaStream_t>(stream)));
  return IQ_OK;
}

}  // namespace

extern "C" {

int iq_kv_create(int format, int kv_heads, int head_dim, int page_tokens, int64_t pages, iq_kv** out) {
  clear_error();
  IQ_CHECK(out, IQ_EINVAL, "iq_kv_create: null argument");
  IQ_CHECK(format == IQ_F16 || format == IQ_I8, IQ_EUNSUPPORTED,
           "unsupported cache format %d; expected F16 (%d) or I8 (%d)", format, IQ_F16, IQ_I8);
  IQ_CHECK(head_dim == 64 || head_dim == 128 || head_dim == 256, IQ_EUNSUPPORTED,
           "head size %d; expected 64, 128 or 256", head_dim);
  IQ_CHECK(kv_heads >= 1 && kv_heads <= 256, IQ_EINVAL, "%d KV heads; expected 1..256", kv_heads);
  IQ_CHECK(page_tokens == 16 || page_tokens == 32 || page_tokens == 64 || page_tokens == 128 || page_tokens == 256,
           IQ_EINVAL, "pages of %d tokens; expected 16, 32, 64, 128 or 256", page_tokens);
  IQ_CHECK(pages >= 1 && pages < (1ll << 31), IQ_EINVAL, "a pool of %lld pages", (long long)pages);
  std::unique_ptr<iq_kv> c(new (std::nothrow) iq_kv);
  IQ_CHECK(c, IQ_ENOMEM, "out of host memory");
  if (int rc = kv_create(format, kv_heads, head_dim, page_tokens, pages, nullptr, *c)) return rc;
  *out = c.release();
  return IQ_OK;
}

void iq_kv_destroy(iq_kv* c) {
  if (!c) return;
  OnDevice on(c->device);
  delete c;
}

int iq_kv_bytes(const iq_kv* c, int64_t* bytes) {
  clear_error();
  IQ_CHECK(c && bytes, IQ_EINVAL, "iq_kv_bytes: null argument");
  *bytes = (int64_t)(c->k.bytes + c->v.bytes + c->ks.bytes + c->vs.bytes);
  return IQ_OK;
}

int iq_kv_append(iq_kv* c, const iq_kv_batch* batch, int dtype, const void* k, int64_t k_row, int64_t k_head,
                 const void* v, int64_t v_row, int64_t v_head, void* stream) {
  return rows_call("iq_kv_append", true, c, batch, dtype, KvTensor{const_cast<void*>(k), k_row, k_head},
                   KvTensor{const_cast<void*>(v), v_row, v_head}, stream);
}

int iq_kv_read(const iq_kv* c, const iq_kv_batch* batch, int dtype, void* k, int64_t k_row, int64_t k_head, void* v,
               int64_t v_row, int64_t v_head, void* stream) {
  return rows_call("iq_kv_read", false, c, batch, dtype, KvTensor{k, k_row, k_head}, KvTensor{v, v_row, v_head},
                   stream);
}

static int attend_args(const iq_kv* c, const iq_kv_batch* batch, const iq_kv_attn* at, KvAttnArgs& a) {
  IQ_CHECK(c && at, IQ_EINVAL, "iq_kv_attend: null argument");
  if (int rc = check_batch("iq_kv_attend", batch, a.b)) return rc;
  if (int rc = check_type("iq_kv_attend", at->dtype)) return rc;
  const KvPool& p = c->pool;
  IQ_CHECK(at->heads >= 1 && at->heads % p.nkv == 0 && at->heads / p.nkv <= 128, IQ_EINVAL,
           "%d query heads over %d KV heads (a multiple of them, at most 128 to one)", at->heads, p.nkv);
  IQ_CHECK(at->scale == at->scale && at->scale - at->scale == 0.f, IQ_EINVAL, "iq_kv_attend: scale is not finite");
  IQ_CHECK(at->window >= 0 && at->sinks >= 0, IQ_EINVAL, "window %d and sinks %d cannot be negative", at->window,
           at->sinks);
  IQ_CHECK(at->chunk >= 0 && at->chunk % 64 == 0, IQ_EINVAL, "a split of %d tokens is not a multiple of 64",
           at->chunk);
  IQ_CHECK(batch->max_rows >= 0, IQ_EINVAL, "max_rows %d is negative", batch->max_rows);
  IQ_CHECK((int64_t)a.b.table_cols * p.page_tokens < (1ll << 31) - 512, IQ_EINVAL,
           "a block table of %d pages of %d tokens is too wide", a.b.table_cols, p.page_tokens);
  IQ_CHECK((int64_t)a.b.rows * at->heads < (1ll << 31), IQ_EINVAL, "%d rows of %d heads are too many", a.b.rows,
           at->heads);
  a.pool = p;
  a.dtype = at->dtype;
  a.heads = at->heads;
  a.scale_log2e = (float)((at->scale != 0.f ? (double)at->scale : 1.0 / sqrt((double)p.hd)) * 1.4426950408889634);
  IQ_CHECK(a.scale_log2e - a.scale_log2e == 0.f, IQ_EINVAL, "iq_kv_attend: a scale of %g is too large", at->scale);
  a.window = at->window;
  a.sinks = at->window ? at->sinks : 0;
  a.chunk = at->chunk;
  return IQ_OK;
}

int iq_kv_attend_workspace(const iq_kv* c, const iq_kv_batch* batch, const iq_kv_attn* at, size_t* bytes) {
  clear_error();
  IQ_CHECK(bytes, IQ_EINVAL, "iq_kv_attend_workspace: null argument");
  KvAttnArgs a = {};
  if (int rc = attend_args(c, batch, at, a)) return rc;
  *bytes = a.b.rows && a.b.seqs ? kv_attend_plan(a, batch->max_rows) : 0;
  return IQ_OK;
}

int iq_kv_attend(const iq_kv* c, const iq_kv_batch* batch, const iq_kv_attn* at, const void* q, int64_t q_row,
                 int64_t q_head, void* out, int64_t out_row, int64_t out_head, void* workspace, size_t bytes,
                 void* stream) {
  clear_error();
  KvAttnArgs a = {};
  if (int rc = attend_args(c, batch, at, a)) return rc;
  if (!a.b.rows || !a.b.seqs) return IQ_OK;
  a.q = KvTensor{const_cast<void*>(q), q_row, q_head};
  a.out = KvTensor{out, out_row, out_head};
  const int hd = c->pool.hd;
  if (int rc = check_tensor("iq_kv_attend", "queries", a.q, a.b.rows, at->heads, hd, at->dtype, false)) return rc;
  if (int rc = check_tensor("iq_kv_attend", "outputs", a.out, a.b.rows, at->heads, hd, at->dtype, true)) return rc;
  const size_t need = kv_attend_plan(a, batch->max_rows);
  IQ_CHECK(bytes >= need, IQ_EINVAL, "iq_kv_attend: the workspace holds %zu bytes, %zu are needed", bytes, need);
  IQ_CHECK(!need || (workspace && (uintptr_t)workspace % 16 == 0), IQ_EINVAL,
           "iq_kv_attend: the workspace is not aligned to 16 bytes");
  kv_attend_bind(a, workspace);
  OnDevice on(c->device);
  IQ_CUDA(on.err);
  IQ_CUDA(kv_attend_launch(a, static_cast<cudaStream_t>(stream)));
  return IQ_OK;
}

int iq_kv_status(iq_kv* c, void* stream) {
  clear_error();
  IQ_CHECK(c, IQ_EINVAL, "iq_kv_status: null cache");
  OnDevice on(c->device);
  IQ_CUDA(on.err);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int f = 0, *word = c->pool.flag + 1 + c->status_calls.fetch_add(1) % kStatusWords;
  kv_take_flag_kernel<<<1, 1, 0, st>>>(c->pool.flag, word);
  IQ_CUDA(cudaGetLastError());
  IQ_CUDA(cudaMemcpyAsync(&f, word, sizeof f, cudaMemcpyDeviceToHost, st));
  IQ_CUDA(cudaStreamSynchronize(st));
  const char* page = f & kKvBadPage
                         ? "a row or a token stood outside its block table, or the table named a page outside the pool"
                         : "";
  IQ_CHECK(!(f & kKvTimeout), IQ_ETIMEDOUT,
           "attention over the cache gave up a bounded device wait; results of that call are invalid%s%s",
           *page ? "; and " : "", page);
  IQ_CHECK(!*page, IQ_EINVAL, "%s", page);
  return IQ_OK;
}

}  // extern "C"
