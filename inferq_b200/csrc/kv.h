// kv.h -- the paged key/value cache behind iq_kv and its kernels' arguments.
//
// Storage.  Per layer one pool of keys and one of values, cut into pages of
// `page_tokens` tokens; the tokens of a page's KV head lie together, so a
// tile of tokens is one contiguous run per page and reaches shared memory by
// bulk copies.  Within a run the 16-byte chunks lie as the attention kernels
// read them from shared memory, so that no kernel rearranges a tile:
//   i8   [page][head][token][head_dim] bytes q + 128, the chunks of a token
//        XOR-ed with i8_swizzle(token): adjacent tokens (key fragments, one
//        16-byte word a lane) and tokens two apart (value fragments, four
//        bytes a lane) then fall on different banks
//   f16  [page][head][head_dim / 64][token][64] halves, 128 bytes a token and
//        slab, its chunks XOR-ed with token & 7: the tensor cores' 128-byte
//        swizzle, keys K-major and values MN-major
// and per token and head one f32 scale each for keys and values,
// [page][head][token].
#pragma once
#include <atomic>
#include <cstdint>
#include "api_util.h"
#include "iq_common.cuh"

namespace iq {

enum KvFormat : int { kKvF16 = 1, kKvI8 = 24 };  // GGML ids of F16 and I8

struct KvPool {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  int* flag;        // kKvBad* bits
  int64_t pages;
  int nkv, hd, page_tokens, page_shift, format;
};
constexpr int kKvBadPage = 1;      // a page id or position outside the table or the pool
constexpr int kKvTimeout = 2;      // a bounded device wait gave up

// A ragged batch of rows (iq_kv_batch).
struct KvBatch {
  const int32_t* table;
  const int32_t* position;
  const int32_t* row_start;  // NULL: one sequence of all rows
  int64_t table_ld;
  int seqs, table_cols, rows;
};

struct KvTensor {  // [row][head][hd], elements contiguous within a head
  void* p;
  int64_t row, head;  // strides in elements
};

struct KvAttnArgs {
  KvPool pool;
  KvBatch b;
  KvTensor q, out;
  int dtype;           // of q and out
  int heads;
  float scale_log2e;   // score scale times log2(e)
  int window, sinks;   // window 0: none
  int chunk;           // tokens per split, a multiple of 64
  int tq;              // query rows a tile: 8, 16, 32, 64 or the tensor-core kernel's 128
  int slots;           // splits that a tile of query rows can need
  bool narrow;         // never the tensor-core kernel (its rows' results depend on the launch)
  int wait_limit;      // tries of a device wait, up to 2 us each (kv_attend_launch sets it)
  bool test_skip;      // tests only: the first CTA's first copy is not requested
  float* part;         // slots > 1: [row][head][slot][hd] unnormalised outputs
  float2* ml;          //            [row][head][slot] {maximum, sum}, base-2 exponents
};

__host__ __device__ inline int64_t kv_head_bytes(int format, int hd, int page_tokens) {
  return (int64_t)page_tokens * hd * (format == kKvI8 ? 1 : 2);
}
__host__ __device__ inline int i8_swizzle(int token, int hd) {
  return ((((token >> 1) & 3) << 1) ^ ((token & 1) << 2)) & (hd / 16 - 1);
}

cudaError_t kv_append_launch(const KvPool& p, const KvBatch& b, int dtype, const KvTensor& k, const KvTensor& v,
                             cudaStream_t st);
cudaError_t kv_read_launch(const KvPool& p, const KvBatch& b, int dtype, const KvTensor& k, const KvTensor& v,
                           cudaStream_t st);

// The split of an attention call: fills tq, chunk and slots (chunk 0 on entry:
// chosen here) and returns the workspace bytes it needs (0 when unsplit).
size_t kv_attend_plan(KvAttnArgs& a, int max_rows);
// a.part / a.ml point into the workspace.
void kv_attend_bind(KvAttnArgs& a, void* workspace);
cudaError_t kv_attend_launch(const KvAttnArgs& a, cudaStream_t st);

}  // namespace iq

struct iq_kv;
namespace iq {
// Allocates and clears a cache on the current device (iq_kv_create's part
// behind its checks).  `flag`: where errors are recorded, NULL for a word of
// its own.
int kv_create(int format, int kv_heads, int head_dim, int page_tokens, int64_t pages, int* flag, iq_kv& c);
}  // namespace iq

struct iq_kv {
  iq::KvPool pool = {};
  iq::DevBuf k, v, ks, vs, flag;
  int device = 0;
  std::atomic<uint32_t> status_calls{0};
};
