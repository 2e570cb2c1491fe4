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
// quotient (three roundings of 2^-24, so at most 127 * 3 * 2^-24 < 2^-15 off)
// decides except within 2^-15 of a border between two codes, where 64 bits
// decide: 127 x is exact there, and a quotient of 24-bit numbers that is no
// tie is further from one than the division rounds.  So a code depends on
// nothing but x and amax.
#include <cmath>
#include <memory>
#include <new>
#include <type_traits>
#include "kv_device.cuh"

namespace iq {
namespace {

__device__ __forceinline__ int code_i8(float x, float inv, float amax) {
  const float v = x * 127.f * inv;
  const float r = rintf(v);
  if (0.5f - fabsf(v - r) < 0x1p-15f) return (int)rint(127.0 * (double)x / (double)amax);
  return (int)r;
}

// One warp per (row, KV head) for keys and values together: 2 x hd elements
// in, quantised in registers, out as 16-byte chunks or parts of them.  The
// work is the bytes (hd = 256, f32 rows: 2 KB in, 0.5 KB out a warp).
template <class T, int HD, int FMT>
__global__ void __launch_bounds__(256) kv_append_kernel(KvPool p, KvBatch b, KvTensor k, KvTensor v, bool vec) {
  constexpr int N = HD / 32;
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int row = (int)(item / p.nkv), head = (int)(item % p.nkv);
  if (row >= b.rows) return;
  float x[2][N];
  load_n<T, N>(static_cast<const T*>(k.p) + row * k.row + head * k.head + lane * N, vec, x[0]);
  load_n<T, N>(static_cast<const T*>(v.p) + row * v.row + head * v.head + lane * N, vec, x[1]);
  int i;
  const int s = kv_seq_of_row(b, row, lane, &i);
  if (s < 0) return;
  const int64_t pos = (int64_t)b.position[s] + i;
  if (pos < 0) return;
  const int page = kv_page(p, b, s, pos);
  if (page < 0) return;
  const int t = (int)pos & (p.page_tokens - 1);
  const int64_t run = (int64_t)page * p.nkv + head;
#pragma unroll
  for (int w = 0; w < 2; w++) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < N; j++) m = max(m, __float_as_uint(x[w][j]) & 0x7fffffffu);
    m = __reduce_max_sync(0xffffffffu, m);
    const bool finite = m < 0x7f800000u;
    const float amax = __uint_as_float(m);
    float scale;
    uint8_t* dst = (w ? p.v : p.k) + run * kv_head_bytes(FMT, HD, p.page_tokens);
    if constexpr (FMT == kKvI8) {
      // both sides of the quotient moved by 2^64, away from f32's ends (an x
      // that falls below the normals there is below amax / 2^62: code 0)
      const float f = amax >= 1.f ? 0x1p-64f : 0x1p64f;
      const float am = amax * f;
      const bool live = finite && m != 0;
      const float inv = live ? __fdiv_rn(1.f, am) : 0.f;
      scale = finite ? __fdiv_rn(amax, 127.f) : __int_as_float(0x7fffffff);
      alignas(8) uint8_t q[N];
#pragma unroll
      for (int j = 0; j < N; j++)
        q[j] = (uint8_t)((live ? code_i8(x[w][j] * f, inv, am) : 0) + 128);
      const int c = lane * N;
      dst += kv_chunk<FMT, HD>(t, c >> 4, p.page_tokens) + (c & 15);
      if constexpr (N == 8) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(q);
      else if constexpr (N == 4) *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(q);
      else *reinterpret_cast<uint16_t*>(dst) = *reinterpret_cast<const uint16_t*>(q);
    } else {
      const int e = f16_exponent(amax);
      scale = finite ? kvp::pow2i(e) : __int_as_float(0x7fffffff);
      const float f = kvp::pow2i(-e);
      alignas(16) __half h[N];
#pragma unroll
      for (int j = 0; j < N; j++) h[j] = __float2half_rn(finite ? x[w][j] * f : 0.f);
      const int c = lane * N * 2;
      dst += kv_chunk<FMT, HD>(t, c >> 4, p.page_tokens) + (c & 15);
      if constexpr (N == 8) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(h);
      else if constexpr (N == 4) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(h);
      else *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(h);
    }
    if (lane == 0) (w ? p.vs : p.ks)[run * p.page_tokens + t] = scale;
  }
}

// The reverse: one warp per (row, KV head); rows at negative positions or
// behind the table read as zeros.
template <class T, int HD, int FMT>
__global__ void __launch_bounds__(256) kv_read_kernel(KvPool p, KvBatch b, KvTensor k, KvTensor v, bool vec) {
  constexpr int N = HD / 32;
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int row = (int)(item / p.nkv), head = (int)(item % p.nkv);
  if (row >= b.rows) return;
  int i;
  const int s = kv_seq_of_row(b, row, lane, &i);
  if (s < 0) return;
  const int64_t pos = (int64_t)b.position[s] + i;
  const int page = pos < 0 ? -1 : kv_page(p, b, s, pos);
  const int t = (int)pos & (p.page_tokens - 1);
  const int64_t run = (int64_t)page * p.nkv + head;
  float x[2][N];
#pragma unroll
  for (int w = 0; w < 2; w++) {
    if (page < 0) {
#pragma unroll
      for (int j = 0; j < N; j++) x[w][j] = 0.f;
      continue;
    }
    const uint8_t* src = (w ? p.v : p.k) + run * kv_head_bytes(FMT, HD, p.page_tokens);
    const float scale = (w ? p.vs : p.ks)[run * p.page_tokens + t];
    if constexpr (FMT == kKvI8) {
      const int c = lane * N;
      src += kv_chunk<FMT, HD>(t, c >> 4, p.page_tokens) + (c & 15);
      alignas(8) uint8_t q[N];
      if constexpr (N == 8) *reinterpret_cast<uint2*>(q) = *reinterpret_cast<const uint2*>(src);
      else if constexpr (N == 4) *reinterpret_cast<uint32_t*>(q) = *reinterpret_cast<const uint32_t*>(src);
      else *reinterpret_cast<uint16_t*>(q) = *reinterpret_cast<const uint16_t*>(src);
#pragma unroll
      for (int j = 0; j < N; j++) x[w][j] = (float)((int)q[j] - 128) * scale;
    } else {
      const int c = lane * N * 2;
      src += kv_chunk<FMT, HD>(t, c >> 4, p.page_tokens) + (c & 15);
      alignas(16) __half h[N];
      if constexpr (N == 8) *reinterpret_cast<uint4*>(h) = *reinterpret_cast<const uint4*>(src);
      else if constexpr (N == 4) *reinterpret_cast<uint2*>(h) = *reinterpret_cast<const uint2*>(src);
      else *reinterpret_cast<uint32_t*>(h) = *reinterpret_cast<const uint32_t*>(src);
#pragma unroll
      for (int j = 0; j < N; j++) x[w][j] = __half2float(h[j]) * scale;
    }
  }
  store_n<T, N>(static_cast<T*>(k.p) + row * k.row + head * k.head + lane * N, vec, x[0]);
  store_n<T, N>(static_cast<T*>(v.p) + row * v.row + head * v.head + lane * N, vec, x[1]);
}

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
  const unsigned grid = (unsigned)ceil_div((int64_t)b.rows * p.nkv, 8);
  auto go = [&](auto hd, auto fmt) {
    constexpr int HD = decltype(hd)::value, FMT = decltype(fmt)::value;
    if (append) kv_append_kernel<T, HD, FMT><<<grid, 256, 0, st>>>(p, b, k, v, vec);
    else kv_read_kernel<T, HD, FMT><<<grid, 256, 0, st>>>(p, b, k, v, vec);
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
  const size_t sizes[] = {bytes, bytes, sbytes, sbytes, sizeof(int)};
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
  if (int rc = check_tensor(name, "keys", k, b.rows, p.nkv, p.hd, dtype, !append)) return rc;
  if (int rc = check_tensor(name, "values", v, b.rows, p.nkv, p.hd, dtype, !append)) return rc;
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
  IQ_CUDA(kv_attend_launch(a, batch->max_rows, static_cast<cudaStream_t>(stream)));
  return IQ_OK;
}

int iq_kv_status(iq_kv* c, void* stream) {
  clear_error();
  IQ_CHECK(c, IQ_EINVAL, "iq_kv_status: null cache");
  OnDevice on(c->device);
  IQ_CUDA(on.err);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int f = 0;
  IQ_CUDA(cudaMemcpyAsync(&f, c->pool.flag, sizeof f, cudaMemcpyDeviceToHost, st));
  IQ_CUDA(cudaStreamSynchronize(st));
  if (f) IQ_CUDA(cudaMemsetAsync(c->pool.flag, 0, sizeof f, st));
  IQ_CHECK(!(f & kKvTimeout), IQ_ETIMEDOUT,
           "attention over the cache gave up a bounded device wait; results of that call are invalid");
  IQ_CHECK(!(f & kKvBadPage), IQ_EINVAL,
           "a row or a token stood outside its block table, or the table named a page outside the pool");
  return IQ_OK;
}

}  // extern "C"
