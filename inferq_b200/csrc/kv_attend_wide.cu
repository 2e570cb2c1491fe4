// kv_attend_wide.cu -- attention of chunks of new rows over the paged cache on
// the tensor cores (tcgen05): more than 64 query rows of a sequence and KV
// head.  The mathematics is that of kv_attend.cu; the split over the tokens
// and the join of its partial results are shared with it (kv_split.cuh).
//
// Tiles.  A CTA takes 128 query rows (row x head of one KV head, so with 8
// query heads to a KV head 16 rows share every key and value it loads) and
// walks one chunk of the tokens in tiles of 64:
//     S = Q K^T      128 x 64,  A = Q from TMEM, B = K from shared memory
//     O += P V       128 x hd,  A = P from TMEM, B = V from shared memory
// Q stays in TMEM (hd / 2 columns of f16 pairs): as a shared-memory operand
// its 4 KB a step would hold the 64-column product to two thirds of the
// tensor rate (128 bytes a cycle; measured, with four score buffers in the
// room that it leaves: 2048 bf16 rows over 32768 f16 tokens of hd 256 in 1315
// us instead of 1140).  TMEM: O in hd columns, the buffers of S (64 columns
// each; P replaces S in place), Q.  Of S there is room for two buffers at hd
// 256 and four below, where scores then run three tiles ahead of the sums (two
// and four side by side, hd 128: 1035 and 930 us).  K tiles are K-major and V
// tiles MN-major in the 128-byte swizzle, in which the f16 cache already keeps
// its pages: its tiles arrive by bulk copies alone.  i8 tiles arrive as bytes in
// small stages, and eight warps expand them to f16 integers.
//
// f32 rows enter as two f16 parts: Q's second part is a shared-memory operand
// of a second product into the same S, P's second part lies beside the first.
//
// Softmax: sixteen warps in two groups that take the tiles in turn, so that one
// group's waits and exponentials lie beside the other's; a row's 64 scores lie
// with two threads, 32 each.  All share the row's maximum: the group of tile i
// decides on it (after the group of tile i - 1 has), and it moves only when a
// tile exceeds it by more than 2^8 (one barrier a tile says whether any row of
// a pair of warps needs that; the accumulator is then rescaled in TMEM).  With
// m the maximum and ev two binades above the first value scales that the row
// sees (all of a tile's, or in a masked tile its own), a row's reference is
// r = m - 7 + ev:
//     p_t = 2^(s_t log2e - r),  weight p_t b_t <= 2^8 2^7 2^-ev b_t <= 2^15,
// the weight of the largest score about 2^4, and f16 keeps 11 bits down to
// 2^-14 and 2^-25 below.  {r, l, o} are the partial result.
//
// The tensor cores cut a sum off towards zero at every instruction, eight of
// them a tile for f32 rows and four for others, while l is summed by rounding
// additions.  What O loses depends on what is added (nothing behind a first
// token that outweighs the rest, up to 5e-8 of it an instruction where equal
// values add up), so no factor on l makes up for it; the length of a chunk
// bounds it instead (kv_split.cuh), and the join adds by rounding.
//
// Warps: 0-15 softmax and results, 16 issues the MMAs (one elected lane: issued
// under a plain lane test each instruction cost four times the cycles), 17-20
// request keys and values (two warps each, tiles in turn: a tile costs one some
// 2000 cycles of dependent address arithmetic and waits), 21-28 expand i8.
// Every wait is bounded; one that runs out sets the cache's flag, and the CTA
// winds down (copies and MMAs drained, TMEM freed) without results.
//
// Bound: the chain scores -> softmax -> values of a tile, of which two are in
// flight (tensor pipe active half of the cycles, issue slots 49%).  2048 rows of
// 16 heads over 32768 tokens of 2 heads of 256: bf16 over f16 1093 us (975
// TFLOP/s, 58% of a measured GEMM's rate), over i8 1399 us; hd 128 987 and 1124.
#include <cfloat>
#include <climits>
#include <type_traits>
#include "kv_device.cuh"
#include "kv_split.cuh"
#include "kv_wide.h"

namespace iq {
namespace {

using namespace kvp;

constexpr int kM = 128, kT = 64;
constexpr int kScaleRing = 4;
// Keys' scales are taken times 2^-14 and the queries' factors times 2^14: scores
// of keys up to 2^118 stay below f32's end until a small query brings them back.
// i8 values' scales, 2^8 above f16's for the same values, are taken times 2^-8:
// p = 2^(4 - ev) then stays 20 binades above f32's beginning for values of 2^119.
constexpr float kKeyDown = 0x1p-14f, kKeyUp = 0x1p14f;
constexpr int kSoftWarps = 16, kMmaWarp = 16, kLoadWarp = 17, kExpandWarp = 21;

template <int HD, int FMT, bool F32Q>
struct Geo {
  static constexpr int kTileBytes = kT * HD * 2;  // an f16 tile of keys or values
  static constexpr int kQlo = F32Q ? kM * HD * 2 : 0;
  // Tiles of keys and of values.  f32 rows at hd 256 leave less room: with i8
  // one tile of values (it is filled again under the next scores' product).
  static constexpr bool kSmall = F32Q && HD == 256;
  static constexpr int kRing = HD < 256 ? 4 : FMT == kKvI8 || F32Q ? 2 : 3;
  static constexpr int kRingV = kSmall && FMT == kKvI8 ? 1 : kRing;
  // i8 tiles pass through stages of bytes, for keys and for values each: whole
  // tiles, or three halves
  static constexpr int kStageTokens = kSmall ? 32 : kT;
  static constexpr int kStage = FMT == kKvI8 ? kStageTokens * HD : 0;
  static constexpr int kStages = FMT != kKvI8 ? 1 : kSmall || HD < 256 ? 3 : 2;
  static constexpr int kScaleBytes = kScaleRing * (2 * kT + 4) * 4 + 6 * kM * 4;
  static constexpr int kSmem = (kRing + kRingV) * kTileBytes + kQlo + 2 * kStages * kStage + kScaleBytes + 1024;
  static constexpr int kExpandWarps = FMT == kKvI8 ? 8 : 0;
  static constexpr int kThreads = (kExpandWarp + kExpandWarps) * 32;
  static constexpr int kBufs = HD < 256 ? 4 : 2;  // of scores
  static constexpr uint32_t kTmemS = HD, kTmemQ = HD + kBufs * kT;
  static constexpr uint32_t kTmemCols = 512;
  static_assert(kTmemQ + HD / 2 <= kTmemCols, "O, S and Q fit the tensor memory");
  static_assert(kRingV * kTileBytes >= kM * HD * 2 || (FMT == kKvI8 && kRing * kTileBytes >= kM * HD * 2), "Q is staged where tiles come later");
  static_assert(kStages >= (kStageTokens == kT ? 2 : 3) || FMT != kKvI8, "see the loader's turns");
  static_assert(kSmem <= 227 * 1024, "shared memory of an SM");
};

__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// f32 D, f16 A and B, M = 128.
constexpr uint32_t idesc(int n, bool b_mn_major) {
  return (1u << 4) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kM >> 4) << 24);
}
// 128-byte swizzle, 8-row groups `stride` apart; `lead`: distance of 64-element
// blocks of an MN-major operand (unused for K-major).
__device__ __forceinline__ uint64_t sw128(uint32_t saddr, uint32_t lead) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, uint32_t accumulate) {
  asm volatile(
      "{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d),
      "r"(a), "l"(b), "r"(desc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, uint32_t accumulate) {
  asm volatile(
      "{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d),
      "l"(a), "l"(b), "r"(desc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(su32(b))
               : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t a, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(a)
      : "memory");
}
// Wait for this thread's TMEM loads; the array is an operand, so that no use
// of it moves before the wait.
__device__ __forceinline__ void tmem_wait(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]),
                 "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]),
                 "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]),
                 "+r"(v[30]), "+r"(v[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_st16(uint32_t a, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t a, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(a), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t a, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(a)
      : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Barrier of a group's two warps (64 threads) that share a quarter of the
// rows, and whether any of them sets `x`; of all softmax warps.
__device__ __forceinline__ void pair_sync(int q) { asm volatile("barrier.cta.sync %0, 64;" ::"r"(q + 1) : "memory"); }
__device__ __forceinline__ bool soft_any(bool x) {
  uint32_t r;
  asm volatile(
      "{ .reg .pred p, c; setp.ne.u32 c, %1, 0; barrier.cta.red.or.pred p, 9, %2, c; selp.u32 %0, 1, 0, p; }"
      : "=r"(r)
      : "r"((uint32_t)x), "n"(kSoftWarps * 32)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void soft_sync() { asm volatile("barrier.cta.sync 9, %0;" ::"n"(kSoftWarps * 32) : "memory"); }
__device__ __forceinline__ bool pair_any(int q, bool x) {
  uint32_t r;
  asm volatile(
      "{ .reg .pred p, c; setp.ne.u32 c, %2, 0; barrier.cta.red.or.pred p, %1, 64, c; selp.u32 %0, 1, 0, p; }"
      : "=r"(r)
      : "r"(q + 1), "r"((uint32_t)x)
      : "memory");
  return r != 0;
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

template <int HD, int FMT, bool F32Q>
__global__ void __launch_bounds__(Geo<HD, FMT, F32Q>::kThreads, 1)
    kv_attend_wide_kernel(const __grid_constant__ KvAttnArgs a, const bool vec) {
  using G_ = Geo<HD, FMT, F32Q>;
  constexpr int NB = G_::kBufs, R = G_::kRing, RV = G_::kRingV, TB = G_::kTileBytes, NS = G_::kStages, SB = G_::kStage;
  __shared__ __align__(8) uint64_t kfull[R], kempty[R], vfull[RV], vempty[RV], sfull[NB], pfull[NB], odone[NB], qfull, decided[2], drained;
  __shared__ __align__(8) uint64_t scfull[kScaleRing], scempty[kScaleRing];
  __shared__ __align__(8) uint64_t stfull[2 * NS], stempty[2 * NS];  // stages of keys, then of values
  __shared__ uint32_t tmem_s;
  __shared__ int abort_s;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (su32(smem_raw) & 1023)) & 1023);
  uint8_t* kring = smem;
  uint8_t* vring = smem + R * TB;
  uint8_t* qlo = vring + RV * TB;
  // Q's first parts pass through a ring before its tiles come: that of the
  // values, which are needed last, where it is large enough
  constexpr bool kQinV = RV * TB >= kM * HD * 2;
  uint8_t* qring = kQinV ? vring : kring;
  uint8_t* stages = qlo + G_::kQlo;                                 // [keys, values][stage]
  float* scales = reinterpret_cast<float*>(stages + 2 * NS * SB);  // [ring][keys 64, values 64, exponent, pad]
  float* tops = scales + kScaleRing * (2 * kT + 4);  // [half][row] maxima of a tile
  float* mrow = tops + 2 * kM;                       // [row] maximum
  int* erow = reinterpret_cast<int*>(mrow + kM);     // [row] exponent
  float* sums = reinterpret_cast<float*>(erow + kM); // [2][row]
  int* eshare = reinterpret_cast<int*>(sums);        // the halves' exponents, before the sums

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const KvPool& p = a.pool;
  const int group = a.heads / p.nkv;
  const int slot = blockIdx.x % a.slots;
  const int kvh = blockIdx.x / a.slots % p.nkv;
  const int tile = blockIdx.x / a.slots / p.nkv;
  // One warp finds the tile's rows and tokens (a few hundred instructions, which
  // 27 warps would issue in turn).
  __shared__ KvTileRows tr_s;
  __shared__ KvSpan sp_s;
  if (warp == 0) {
    KvTileRows t = {};
    KvSpan s = {};
    const bool any = kv_tile_rows(a.b, tile, kM, group, lane, &t);
    if (any) s = kv_span(a, t, kM, slot);
    if (lane == 0) {
      if (!any) t.seq = -1;
      if (any && s.outside) atomicOr(p.flag, kKvBadPage);
      tr_s = t;
      sp_s = s;
    }
  }
  __syncthreads();
  const KvTileRows tr = tr_s;
  const KvSpan sp = sp_s;
  if (tr.seq < 0 || (sp.first >= sp.end && a.slots > 1)) return;

  if (threadIdx.x == 0) {
    for (int s = 0; s < R; s++) {
      bar_init(&kfull[s], FMT == kKvI8 ? 4 : 1);
      bar_init(&kempty[s], 1);
    }
    for (int s = 0; s < RV; s++) {
      bar_init(&vfull[s], FMT == kKvI8 ? 4 : 1);
      bar_init(&vempty[s], 1);
    }
    for (int b = 0; b < NB; b++) {
      bar_init(&sfull[b], 1);
      bar_init(&pfull[b], 8);
      bar_init(&odone[b], 1);
    }
    for (int s = 0; s < kScaleRing; s++) {
      bar_init(&scfull[s], 2);
      bar_init(&scempty[s], 8);
    }
    for (int s = 0; s < 2 * NS; s++) {
      bar_init(&stfull[s], 1);
      bar_init(&stempty[s], 4);
    }
    bar_init(&qfull, kSoftWarps);
    bar_init(&decided[0], 8);
    bar_init(&decided[1], 8);
    bar_init(&drained, 1);
    abort_s = 0;
    bar_init_fence();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&tmem_s)),
                 "r"(G_::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = tmem_s;
  volatile int* abort_v = &abort_s;
  auto give_up = [&]() {
    atomicOr(p.flag, kKvTimeout);
    *abort_v = 1;
  };
  // a warp's wait: one outcome for all lanes
  auto wait = [&](uint64_t* b, uint32_t parity) {
    for (int i = 0; i < a.wait_limit; i++) {
      if (__all_sync(0xffffffffu, bar_try(b, parity))) return true;
      if ((i & 31) == 31 && __any_sync(0xffffffffu, *abort_v)) return false;
    }
    give_up();
    return false;
  };

  if (warp < kSoftWarps) {
    // ------------------------------------------------------- query rows
    // Row by row with the lanes along the head; first parts go through a
    // ring (chunks XOR-ed with the row) to the thread that owns the row.
    const int quarter = warp & 3, half = (warp >> 2) & 1, grp = warp >> 3, r0 = quarter * 32;
    const int pair = grp * 4 + quarter, part = warp >> 2;
    {
      constexpr int N = HD / 32, U = 4;  // rows in flight
      // where the warp's eight rows begin, one to a lane: -1 behind the last
      // (divisions once a lane, not once a row: sixteen warps share the issue)
      int64_t begin = -1;
      {
        const int rr = tr.r0 + r0 + 8 * part + (lane & 7);
        const int i = rr / group, h = kvh * group + rr - i * group;
        if (rr < tr.nr) begin = (int64_t)(tr.row0 + i) * a.q.row + (int64_t)h * a.q.head;
      }
#pragma unroll 1
      for (int rb = 8 * part; rb < 8 * part + 8; rb += U) {
        float x[U][N];
#pragma unroll
        for (int u = 0; u < U; u++) {
          const int64_t at = __shfl_sync(0xffffffffu, begin, (rb & 7) + u);
          const int64_t o = at + lane * N;
          if (at >= 0) {
            if constexpr (F32Q) load_n<float, N>(static_cast<const float*>(a.q.p) + o, vec, x[u]);
            else if (a.dtype == F16) load_n<__half, N>(static_cast<const __half*>(a.q.p) + o, vec, x[u]);
            else load_n<__nv_bfloat16, N>(static_cast<const __nv_bfloat16*>(a.q.p) + o, vec, x[u]);
          } else {
#pragma unroll
            for (int j = 0; j < N; j++) x[u][j] = 0.f;
          }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
          const int row = r0 + rb + u;
          uint32_t m = 0;
#pragma unroll
          for (int j = 0; j < N; j++) m = max(m, __float_as_uint(x[u][j]) & 0x7fffffffu);
          const int e = f16_exponent(__uint_as_float(__reduce_max_sync(0xffffffffu, m)));
          const float f = a.scale_log2e < 0.f ? -pow2i(-e) : pow2i(-e);  // a factor below zero turns the row
          alignas(16) __half hi[N], lo[N];
#pragma unroll
          for (int j = 0; j < N; j++) {
            const float y = x[u][j] * f;
            hi[j] = __float2half_rn(y);
            lo[j] = __float2half_rn(y - __half2float(hi[j]));
          }
          const int byte = lane * N * 2, c = byte >> 4;
          uint8_t* d = qring + row * HD * 2 + ((c ^ (row & 7)) << 4) + (byte & 15);
          uint8_t* dl = qlo + ((c >> 3) * kM + row) * 128 + (((c & 7) ^ (row & 7)) << 4) + (byte & 15);
          if constexpr (N == 8) {
            *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(hi);
            if constexpr (F32Q) *reinterpret_cast<uint4*>(dl) = *reinterpret_cast<const uint4*>(lo);
          } else if constexpr (N == 4) {
            *reinterpret_cast<uint2*>(d) = *reinterpret_cast<const uint2*>(hi);
            if constexpr (F32Q) *reinterpret_cast<uint2*>(dl) = *reinterpret_cast<const uint2*>(lo);
          } else {
            *reinterpret_cast<uint32_t*>(d) = *reinterpret_cast<const uint32_t*>(hi);
            if constexpr (F32Q) *reinterpret_cast<uint32_t*>(dl) = *reinterpret_cast<const uint32_t*>(lo);
          }
          // (never 0 or infinite: hidden scores stay -inf, others finite)
          if (lane == 0) tops[row] = fminf(fmaxf(pow2i(e) * fabsf(a.scale_log2e) * kKeyUp, FLT_MIN), FLT_MAX);
        }
      }
    }
    soft_sync();
    const int row = r0 + lane, rr = tr.r0 + row;
    const bool live = rr < tr.nr;
    const uint32_t lanes = tmem + ((uint32_t)r0 << 16);
    const float cq = tops[row];
    int rp = -1;
    if (live) rp = (int)max(min(tr.pos + rr / group, (int64_t)INT_MAX), (int64_t)-1);
    // the four warps of a quarter move a fourth of its Q each
    constexpr int kQC = HD / 32;  // 16-byte chunks
#pragma unroll
    for (int c = 0; c < kQC; c += 2) {
      uint32_t v[8];
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const uint4 w = *reinterpret_cast<const uint4*>(qring + row * HD * 2 + (((part * kQC + c + k) ^ (row & 7)) << 4));
        v[4 * k] = w.x, v[4 * k + 1] = w.y, v[4 * k + 2] = w.z, v[4 * k + 3] = w.w;
      }
      tmem_st8(lanes + G_::kTmemQ + 4 * (part * kQC + c), v);
    }
    if (part == 0) {
      mrow[row] = -INFINITY;
      erow[row] = -100;
    }
    tmem_wait_st();
    tc_before();
    async_fence();  // the second parts and the ring's hand-over to the copies
    __syncwarp();
    if (lane == 0) bar_arrive(&qfull);

    // ----------------------------------------------------------- softmax
    soft_sync();  // mrow and erow are set
    float m = -INFINITY;
    float2 l2 = make_float2(0.f, 0.f);
    int ev = -100;
    bool ok = true;
    int it = 0, mine = -1;  // tiles so far, the group's last
    for (int ti = sp.first; ti < sp.end; ti = sp.next(ti), it++) {
      if ((it & 1) != grp) continue;
      mine = it;
      const int b = it % NB, sr = it % kScaleRing, t0 = ti * kT + 32 * half;
      const float* sc = scales + sr * (2 * kT + 4);
      // A wait that ran out is told to the pair's other warp at its barrier,
      // so that no warp is left in one.
      ok = ok && wait(&scfull[sr], (it / kScaleRing) & 1) && wait(&sfull[b], (it / NB) & 1);
      tc_after();
      const uint32_t st = lanes + G_::kTmemS + b * kT;
      uint32_t s0[32];
      tmem_ld32(st + 32 * half, s0);
      float2 x[16];
      const float4* ks = reinterpret_cast<const float4*>(sc + 32 * half);
      int et = __float_as_int(sc[2 * kT]);
      tmem_wait(s0);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float4 k = ks[j];
        x[2 * j] = mul2(make_float2(__uint_as_float(s0[4 * j]), __uint_as_float(s0[4 * j + 1])), make_float2(k.x, k.y));
        x[2 * j + 1] = mul2(make_float2(__uint_as_float(s0[4 * j + 2]), __uint_as_float(s0[4 * j + 3])), make_float2(k.z, k.w));
      }
      const bool whole = sp.whole(ti * kT, kT);
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 16; j++) {
          if (!sp.sees(rp, t0 + 2 * j)) x[j].x = -INFINITY;
          if (!sp.sees(rp, t0 + 2 * j + 1)) x[j].y = -INFINITY;
        }
        // The exponent above the scales that the row sees: a hidden token's would
        // take bits of its weights.
        const float4* vs = reinterpret_cast<const float4*>(sc + kT + 32 * half);
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float4 v = vs[j];
          if (x[2 * j].x != -INFINITY && v.x < INFINITY) top = fmaxf(top, v.x);
          if (x[2 * j].y != -INFINITY && v.y < INFINITY) top = fmaxf(top, v.y);
          if (x[2 * j + 1].x != -INFINITY && v.z < INFINITY) top = fmaxf(top, v.z);
          if (x[2 * j + 1].y != -INFINITY && v.w < INFINITY) top = fmaxf(top, v.w);
        }
        et = max(__float_as_int(top) >> 23, 1) - 126;
      }
      float m4[4];
#pragma unroll
      for (int j = 0; j < 4; j++) m4[j] = fmaxf(x[j].x, x[j].y);
#pragma unroll
      for (int j = 4; j < 16; j++) m4[j & 3] = max3(m4[j & 3], x[j].x, x[j].y);
      float mx = fmaxf(max3(m4[0], m4[1], m4[2]), m4[3]) * cq;
      if (it > 0) {  // the other group's decision on the tile before
        // (A barrier for each group: scores lie ready for several tiles, so a warp
        // may be at its next tile before its own group is through with this one;
        // on one barrier it would meet a phase two behind.)
        ok = ok && wait(&decided[(it - 1) & 1], ((it - 1) >> 1) & 1);
        const float mo = mrow[row];
        const int eo = erow[row];
        if (mo != m || eo != ev) {
          const float f = m == -INFINITY ? 0.f : ex2(m - mo + (float)(ev - eo));
          l2 = mul2(l2, make_float2(f, f));
          m = mo;
          ev = eo;
        }
      }
      // both threads of a row have read its scores when the barrier opens
      int en = ev;
      const bool move = mx > m + 8.f || m == -INFINITY || et > ev;
      float fo = 1.f;
      if (!whole || pair_any(pair, move || !ok)) {
        tops[half * kM + row] = mx;
        eshare[half * kM + row] = ok ? et : INT_MAX;  // INT_MAX: the warp gave up
        pair_sync(pair);
        mx = fmaxf(mx, tops[(half ^ 1) * kM + row]);
        const int eo = eshare[(half ^ 1) * kM + row];
        pair_sync(pair);
        if (!__all_sync(0xffffffffu, ok && eo != INT_MAX)) {
          ok = false;
          break;
        }
        et = max(et, eo);
        if (et > ev) en = et + 2;
        const float mn = mx > m + 8.f || m == -INFINITY ? mx : m;
        // o and l by 2^(old reference - new)
        const float d = (m == -INFINITY ? 0.f : m) - (mn == -INFINITY ? 0.f : mn) + (float)(ev - en);
        fo = m == mn && en == ev ? 1.f : m == -INFINITY ? 0.f : ex2(d);
        m = mn;
        ev = en;
        l2 = mul2(l2, make_float2(fo, fo));
        if (half == 0) {
          mrow[row] = m;
          erow[row] = ev;
        }
      }
      __syncwarp();
      if (lane == 0) bar_arrive(&decided[grp]);
      const float r = (m == -INFINITY ? 0.f : m) - 7.f + (float)ev;
      const float4* vs = reinterpret_cast<const float4*>(sc + kT + 32 * half);
#pragma unroll
      for (int hh = 0; hh < 2; hh++) {
        uint32_t w[8], wl[8];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const float4 v = vs[4 * hh + j];
          const float2 x0 = x[8 * hh + 2 * j], x1 = x[8 * hh + 2 * j + 1];
          float2 a0 = fma2(x0, make_float2(cq, cq), make_float2(-r, -r)),
                 a1 = fma2(x1, make_float2(cq, cq), make_float2(-r, -r));
          a0 = make_float2(ex2(a0.x), ex2(a0.y));
          a1 = make_float2(ex2(a1.x), ex2(a1.y));
          l2 = add2(l2, add2(a0, a1));
          float2 w0 = mul2(a0, make_float2(v.x, v.y)), w1 = mul2(a1, make_float2(v.z, v.w));
          if (!whole) {  // a hidden token weighs zero whatever its scale is
            if (x0.x == -INFINITY) w0.x = 0.f;
            if (x0.y == -INFINITY) w0.y = 0.f;
            if (x1.x == -INFINITY) w1.x = 0.f;
            if (x1.y == -INFINITY) w1.y = 0.f;
          }
          w[2 * j] = pack2(w0.x, w0.y);
          w[2 * j + 1] = pack2(w1.x, w1.y);
          if constexpr (F32Q) {
            const float2 f0 = unpack2(w[2 * j]), f1 = unpack2(w[2 * j + 1]);
            wl[2 * j] = pack2(w0.x - f0.x, w0.y - f0.y);
            wl[2 * j + 1] = pack2(w1.x - f1.x, w1.y - f1.y);
          }
        }
        tmem_st8(st + 16 * half + 8 * hh, w);
        if constexpr (F32Q) tmem_st8(st + 32 + 16 * half + 8 * hh, wl);
      }
      __syncwarp();
      if (lane == 0) bar_arrive(&scempty[sr]);
      if (it > 0 && __any_sync(0xffffffffu, fo != 1.f)) {
        // The previous product has been added.  (One phase behind at most: these
        // scores came after the product of tile it - NB.)
        ok = wait(&odone[(it - 1) % NB], ((it - 1) / NB) & 1);
        tc_after();
#pragma unroll 1
        for (int c = half * (HD / 2); c < (half + 1) * (HD / 2); c += 16) {
          uint32_t o[16];
          tmem_ld16(lanes + c, o);
#pragma unroll
          for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * fo);
          tmem_st16(lanes + c, o);
        }
      }
      tmem_wait_st();
      tc_before();
      __syncwarp();
      if (lane == 0) bar_arrive(&pfull[b]);
    }
    // ----------------------------------------------------------- results
    tmem_wait_st();  // no store in flight past this point
    // Every product has been added when `drained` fires (its only phase; odone
    // may be two phases on by now, and a parity cannot tell).
    ok = ok && wait(&drained, 0);
    if (ok && it > 0 && mine != it - 1) {  // the last decision was the other group's
      const float mo = mrow[row];
      const int eo = erow[row];
      const float f = mo == m && eo == ev ? 1.f : m == -INFINITY ? 0.f : ex2(m - mo + (float)(ev - eo));
      l2 = mul2(l2, make_float2(f, f));
      m = mo;
      ev = eo;
    }
    // (a group that gave up leaves the others to their own waits: every
    // thread of the softmax warps comes here)
    soft_sync();
    float* ls = half ? sums : tops;  // [group][row]
    ls[grp * kM + row] = l2.x + l2.y;
    if (!soft_any(!ok || *abort_v)) {  // one outcome for all: barriers follow
      tc_after();
      const float l = (tops[row] + tops[kM + row]) + (sums[row] + sums[kM + row]);
      const int grow = tr.row0 + rr / group, h = kvh * group + rr % group;
      const int64_t rh = (int64_t)grow * a.heads + h;
      constexpr float kUp = FMT == kKvI8 ? 0x1p8f : 1.f;
      const float f = a.slots > 1 ? kUp : l != 0.f ? __fdiv_rn(kUp, l) : 0.f;
      if (a.slots > 1 && live && part == 0) a.ml[rh * a.slots + slot] = make_float2(m - 7.f + (float)ev, l);
      // A row's elements lie with one thread: they go to shared memory, a row
      // of hd elements and 16 bytes apart (so that eight lanes' stores meet
      // eight bank groups), and from there to memory as whole rows.
      auto put = [&](auto* base, int64_t at, bool whole_rows) {
        using T = std::remove_reference_t<decltype(*base)>;
        constexpr int kRow = HD * (int)sizeof(T) + 16;
        static_assert(kM * kRow <= (R + RV) * TB + G_::kQlo + 2 * NS * SB, "the rings hold the results");
        T* mine = reinterpret_cast<T*>(smem + row * kRow);
#pragma unroll 1
        for (int c = part * (HD / 4); c < (part + 1) * (HD / 4); c += 16) {
          uint32_t o[16];
          if (it > 0) {
            tmem_ld16(lanes + c, o);
          } else {
#pragma unroll
            for (int j = 0; j < 16; j++) o[j] = 0;
          }
#pragma unroll
          for (int j = 0; j < 16; j += 8) {
            float y[8];
#pragma unroll
            for (int k = 0; k < 8; k++) y[k] = __uint_as_float(o[j + k]) * f;
            store_n<T, 8>(mine + c + j, true, y);
          }
        }
        if (whole_rows) async_fence();
        // the quarter's four warps hold parts of its rows
        asm volatile("barrier.cta.sync %0, 128;" ::"r"(10 + quarter) : "memory");
        if (whole_rows) {
          if (part == 0 && live)
            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(base + at), "r"(su32(mine)),
                         "r"(HD * (int)sizeof(T))
                         : "memory");
          asm volatile("cp.async.bulk.commit_group;\ncp.async.bulk.wait_group.read 0;" ::: "memory");
        } else {
          for (int i = 8 * part; i < 8 * part + 8; i++) {
            const int64_t to = __shfl_sync(0xffffffffu, at, i);
            if (tr.r0 + r0 + i >= tr.nr) continue;
            const T* src = reinterpret_cast<const T*>(smem + (r0 + i) * kRow);
            for (int c = lane; c < HD; c += 32) base[to + c] = src[c];
          }
        }
      };
      const int64_t at = (int64_t)grow * a.out.row + (int64_t)h * a.out.head;
      if (a.slots > 1) put(a.part, (rh * a.slots + slot) * HD, true);
      else if constexpr (F32Q) put(static_cast<float*>(a.out.p), at, vec);
      else if (a.dtype == F16) put(static_cast<__half*>(a.out.p), at, vec);
      else put(static_cast<__nv_bfloat16*>(a.out.p), at, vec);
    }
  } else if (warp == kMmaWarp) {
    // --------------------------------------------------------- products
    // The whole warp waits, one lane issues.
    constexpr uint32_t dS = idesc(kT, false), dO = idesc(HD, true);
    const uint32_t k0 = su32(kring), v0 = su32(vring), ql = su32(qlo);
    uint32_t leader;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(leader));
    bool ok = wait(&qfull, 0);
    tc_after();
    auto score = [&](int i) {
      const int s = i % R;
      if (!wait(&kfull[s], (i / R) & 1)) return false;
      tc_after();
      if (leader) {
        const uint32_t d = tmem + G_::kTmemS + (i % NB) * kT, kb = k0 + s * TB;
        if constexpr (F32Q) {  // the small parts first: fewer cuts of the whole sum
#pragma unroll
          for (int st = 0; st < HD / 16; st++)
            mma_ss(d, sw128(ql + (st >> 2) * (kM * 128) + (st & 3) * 32, 16),
                   sw128(kb + (st >> 2) * (kT * 128) + (st & 3) * 32, 16), dS, st > 0);
        }
#pragma unroll
        for (int st = 0; st < HD / 16; st++)
          mma_ts(d, tmem + G_::kTmemQ + 8 * st, sw128(kb + (st >> 2) * (kT * 128) + (st & 3) * 32, 16), dS, F32Q || st > 0);
        commit(&sfull[i % NB]);
        commit(&kempty[s]);
      }
      __syncwarp();
      return true;
    };
    // Scores run NB - 1 tiles ahead of the sums: product it - 1, issued before,
    // has read the buffer that the scores of tile it + NB - 1 fill.
    int ns = 0, ts = sp.first;
#pragma unroll 1
    for (; ok && ts < sp.end && ns < NB - 1; ts = sp.next(ts)) ok = score(ns++);
    for (int it = 0; ok && it < ns; it++) {
      if (ts < sp.end) {
        ts = sp.next(ts);
        if (!(ok = score(ns++))) break;
      }
      const int s = it % RV;
      ok = wait(&pfull[it % NB], (it / NB) & 1) && wait(&vfull[s], (it / RV) & 1);
      if (!ok) break;
      tc_after();
      if (leader) {
        const uint32_t pa = tmem + G_::kTmemS + (it % NB) * kT, vb = v0 + s * TB;
#pragma unroll
        for (int part = 0; part < (F32Q ? 2 : 1); part++)
#pragma unroll
          for (int kk = 0; kk < kT / 16; kk++)
            mma_ts(tmem, pa + part * 32 + 8 * kk, sw128(vb + kk * 2048, kT * 128), dO, it > 0 || kk > 0 || part > 0);
        commit(&vempty[s]);
        commit(&odone[it % NB]);
      }
      __syncwarp();
    }
    if (leader) commit(&drained);  // every product issued above has completed when this fires
    __syncwarp();
    bar_wait(&drained, 0, 4 * a.wait_limit);
  } else if (warp < kExpandWarp) {
    // ----------------------------------------------------- bulk copies
    // A warp takes every other tile of keys or values.  The page ids of its
    // next tile are read a turn ahead, that tile's scales likewise, and neither
    // is looked at before then, so that no load is waited for.
    const bool isv = (warp - kLoadWarp) & 1;
    const int turn = (warp - kLoadWarp) >> 1;
    uint8_t* ring = isv ? vring : kring;
    uint64_t* full = isv ? vfull : kfull;
    uint64_t* empty = isv ? vempty : kempty;
    const uint8_t* pool = isv ? p.v : p.k;
    const float* spool = isv ? p.vs : p.ks;
    const int rs = min(p.page_shift, 6), rt = 1 << rs, runs = kT >> rs;  // tokens of a page's run in a tile
    const int64_t hb = kv_head_bytes(FMT, HD, p.page_tokens);
    auto holds = [&](int ti) {  // whether the lane's run of tile ti begins with a token of the sequence
      return ti < sp.end && lane < runs && ti * kT + lane * rt < sp.tokens;
    };
    auto ask = [&](int ti) {
      const int col = (ti * kT + lane * rt) >> p.page_shift;  // inside the table: below sp.tokens
      return holds(ti) ? __ldg(a.b.table + (int64_t)tr.seq * a.b.table_ld + col) : -1;
    };
    auto page_of = [&](int ti, int id) {
      if (holds(ti) && (id < 0 || id >= p.pages)) {
        atomicOr(p.flag, kKvBadPage);
        id = 0;
      }
      // runs behind the last token are filled from the tile's first page
      const int first = __shfl_sync(0xffffffffu, id, 0);
      return holds(ti) ? id : max(first, 0);
    };
    float sv[2] = {0.f, 0.f};
    auto load_scales = [&](int ti, int page) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int t = lane + 32 * h;
        const int64_t at = (int64_t)__shfl_sync(0xffffffffu, page, t >> rs) * p.nkv + kvh;
        sv[h] = spool[at * p.page_tokens + ((ti * kT + t) & (p.page_tokens - 1))];
      }
    };
    // A parity tells two phases apart only while the barrier is known to be at
    // most one behind.  Fill n waits for the emptying of fill n - NS, so fill
    // n - 2 NS has to be known as emptied from the warp's fill before: with
    // whole tiles n - 2 (behind n - 2 - NS), with halves n - 3 (behind n - 3 -
    // NS), and the rings are emptied in order: NS >= 2, and >= 3 for halves.
    auto after = [&](int ti) { return sp.next(sp.next(ti)); };
    int it = turn, ti = turn ? sp.next(sp.first) : sp.first, t1 = after(ti);
    bool ok = true;
    const bool skip_first = a.test_skip && blockIdx.x == 0 && !isv && turn == 0 && lane == 0;
    int page = page_of(ti, ask(ti)), id1 = ask(t1);
    if (ti < sp.end) load_scales(ti, page);
    if (FMT == kKvF16 && isv && ti < sp.end) ok = wait(&qfull, 0);  // the V ring holds the query rows first
    int requested = 0;  // one past the last fill of the ring (f16) or of the stages (i8)
    for (; ok && ti < sp.end; it += 2) {
      // the tile's scales and the exponent above the values'
      const int sr = it % kScaleRing;
      if (it >= kScaleRing && !(ok = wait(&scempty[sr], ((it / kScaleRing) + 1) & 1))) break;
      float* sc = scales + sr * (2 * kT + 4);
      uint32_t top = 0;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int t = lane + 32 * h;
        const float s = sv[h] * (!isv ? kKeyDown : FMT == kKvI8 ? 0x1p-8f : 1.f);
        sc[isv * kT + t] = s;
        const uint32_t bits = __float_as_uint(s);
        if (bits < 0x7f800000u && ti * kT + t < sp.tokens) top = max(top, bits);
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if (isv && lane == 0) sc[2 * kT] = __int_as_float(max((int)(top >> 23), 1) - 126);
      __syncwarp();
      if (lane == 0) bar_arrive(&scfull[sr]);
      const int page1 = page_of(t1, id1), t2 = after(t1);
      if (t1 < sp.end) load_scales(t1, page1);
      id1 = ask(t2);
      const int tp = (ti * kT) & (p.page_tokens - 1);
      if constexpr (FMT == kKvF16) {
        constexpr int kParts = HD / 64;
        const int s = it % R;
        if (it >= R && !(ok = wait(&empty[s], ((it / R) + 1) & 1))) break;
        if (lane == 0) bar_expect(&full[s], TB);
        __syncwarp();
        requested = it + 1;
#pragma unroll 1
        for (int c0 = 0; c0 < runs * kParts; c0 += 32) {
          const int c = c0 + lane, run = min(c / kParts, runs - 1), part = c % kParts;
          const int64_t at = (int64_t)__shfl_sync(0xffffffffu, page, run) * p.nkv + kvh;
          if (c < runs * kParts && !(skip_first && it + c0 == 0))
            bulk_load(su32(ring + s * TB + (part * kT + run * rt) * 128),
                      pool + at * hb + ((int64_t)part * p.page_tokens + tp) * 128, rt * 128, &full[s]);
        }
        __syncwarp();
      } else {
        constexpr int kPer = kT / G_::kStageTokens;  // stages of a tile
        const int cs = min(rs, G_::kSmall ? 5 : 6), ct = 1 << cs, copies = G_::kStageTokens >> cs;
#pragma unroll 1
        for (int q = 0; q < kPer; q++) {
          const int n = it * kPer + q, s = n % NS;
          if (n >= NS && !(ok = wait(&stempty[isv * NS + s], ((n / NS) + 1) & 1))) break;
          uint64_t* bar = &stfull[isv * NS + s];
          if (lane == 0) bar_expect(bar, SB);
          __syncwarp();
          requested = n + 1;
          const int t = q * G_::kStageTokens + min(lane, copies - 1) * ct;
          const int64_t at = (int64_t)__shfl_sync(0xffffffffu, page, t >> rs) * p.nkv + kvh;
          if (lane < copies && !(skip_first && n == 0))
            bulk_load(su32(stages + (isv * NS + s) * SB + lane * ct * HD),
                      pool + at * hb + (int64_t)((ti * kT + t) & (p.page_tokens - 1)) * HD, ct * HD, bar);
          __syncwarp();
        }
        if (!ok) break;
      }
      ti = t1;
      t1 = t2;
      page = page1;
    }
    // Where every tile is used, its copy has landed.  Otherwise no copy may
    // outlive the CTA: the last fills are waited for (again bounded).
    if (!ok || __any_sync(0xffffffffu, *abort_v)) {
      uint64_t* bars = FMT == kKvF16 ? full : stfull + isv * NS;
      constexpr int kRound = FMT == kKvF16 ? R : NS;
      for (int n = max(requested - 2 * kRound, 0); n < requested; n++) bar_wait(&bars[n % kRound], (n / kRound) & 1, 1 << 10);
    }
  } else {
    // ------------------------------------------- expansion to f16 (i8)
    // Four warps for keys, four for values; a thread takes 16-byte chunks.
    const int isv = (warp - kExpandWarp) >> 2, tid = threadIdx.x - (kExpandWarp + 4 * isv) * 32;
    uint8_t* ring = isv ? vring : kring;
    uint64_t* full = isv ? vfull : kfull;
    uint64_t* empty = isv ? vempty : kempty;
    const int rn = isv ? RV : R;
    constexpr int C = HD / 16, TP = 128 / C;         // chunks a token, tokens a pass
    constexpr int kPer = kT / G_::kStageTokens, NP = G_::kStageTokens / TP;  // stages a tile, passes a stage
    const int ch = tid % C, tk = tid / C;
    bool ok = true;
    if (isv == kQinV && sp.first < sp.end) ok = wait(&qfull, 0);  // the ring holds the query rows first
    int it = 0;
    for (int ti = sp.first; ok && ti < sp.end; ti = sp.next(ti), it++) {
      const int s = it % rn;
      if (it >= rn && !(ok = wait(&empty[s], ((it / rn) + 1) & 1))) break;
      uint8_t* dst = ring + s * TB;
#pragma unroll
      for (int q = 0; q < kPer; q++) {
        const int n = it * kPer + q, sn = n % NS;
        if (!(ok = wait(&stfull[isv * NS + sn], (n / NS) & 1))) break;
        const uint8_t* src = stages + (isv * NS + sn) * SB + tid * 16;
#pragma unroll
        for (int i = 0; i < NP; i++) {
          const uint4 raw = *reinterpret_cast<const uint4*>(src + 2048 * i);
          const int t = (NP * q + i) * TP + tk, c = ch ^ i8_swizzle(t, HD);  // 16 elements: chunks 2c, 2c + 1 of the f16 row
          const uint2 y0 = biased4_to_f16(raw.x), y1 = biased4_to_f16(raw.y), y2 = biased4_to_f16(raw.z),
                      y3 = biased4_to_f16(raw.w);
          const uint4 lo = make_uint4(y0.x, y0.y, y1.x, y1.y), hi = make_uint4(y2.x, y2.y, y3.x, y3.y);
          uint8_t* rowp = dst + ((c >> 2) * kT + t) * 128;
          // the two 64-element blocks that a quarter warp meets take their
          // halves in turn, so that its eight stores fall on different banks
          const int turn = (c >> 2) & 1, c8 = (c & 3) * 2;
          *reinterpret_cast<uint4*>(rowp + (((c8 + turn) ^ (t & 7)) << 4)) = turn ? hi : lo;
          *reinterpret_cast<uint4*>(rowp + (((c8 + 1 - turn) ^ (t & 7)) << 4)) = turn ? lo : hi;
        }
        __syncwarp();
        if (lane == 0) bar_arrive(&stempty[isv * NS + sn]);
      }
      if (!ok) break;
      async_fence();
      __syncwarp();
      if (lane == 0) bar_arrive(&full[s]);
    }
  }
  __syncwarp();
  tc_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G_::kTmemCols) : "memory");
  }
}

template <int HD, int FMT, bool F32Q>
cudaError_t launch(const KvAttnArgs& a, int64_t ctas, bool vec, cudaStream_t st) {
  using G_ = Geo<HD, FMT, F32Q>;
  static bool configured[64] = {};
  static std::mutex mu;
  const cudaError_t e = once_per_device(configured, mu, [] {
    return cudaFuncSetAttribute(kv_attend_wide_kernel<HD, FMT, F32Q>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                G_::kSmem);
  });
  if (e != cudaSuccess) return e;
  kv_attend_wide_kernel<HD, FMT, F32Q><<<(unsigned)ctas, G_::kThreads, G_::kSmem, st>>>(a, vec);
  return cudaGetLastError();
}

}  // namespace

cudaError_t kv_attend_wide_launch(const KvAttnArgs& a, int64_t ctas, bool vec, cudaStream_t st) {
  auto by_type = [&](auto hd, auto fmt) {
    constexpr int HD = decltype(hd)::value, FMT = decltype(fmt)::value;
    return a.dtype == F32 ? launch<HD, FMT, true>(a, ctas, vec, st) : launch<HD, FMT, false>(a, ctas, vec, st);
  };
  auto by_format = [&](auto hd) {
    return a.pool.format == kKvI8 ? by_type(hd, std::integral_constant<int, kKvI8>())
                                  : by_type(hd, std::integral_constant<int, kKvF16>());
  };
  switch (a.pool.hd) {
    case 64: return by_format(std::integral_constant<int, 64>());
    case 128: return by_format(std::integral_constant<int, 128>());
    case 256: return by_format(std::integral_constant<int, 256>());
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace iq
