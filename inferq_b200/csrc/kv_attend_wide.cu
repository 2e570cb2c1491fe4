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
// tensor rate (128 bytes a cycle).  TMEM: O in hd columns, two buffers of S
// (64 columns each; P replaces S in place), Q.  K tiles are K-major and V
// tiles MN-major in the 128-byte swizzle, in which the f16 cache already
// keeps its pages: its tiles arrive by bulk copies alone.  i8 tiles are
// expanded to f16 integers on the way (two groups of four warps, one for keys
// and one for values, global loads in flight while the other tile is written).
//
// f32 rows enter as two f16 parts: Q's second part is a shared-memory operand
// of a second product into the same S, P's second part lies beside the first.
//
// Softmax: four warps, one row a thread, so that no maximum crosses a lane.
// The running maximum moves only when a tile exceeds it by more than 2^8 (the
// accumulator is rescaled in TMEM then); weights are at most
// 2^8 * 2^(7 - 2): ev keeps two binades of room above the first value scales.
// The weight of the largest score is at least 2^-3 * 2^5, and f16 keeps 11
// bits down to 2^-14, i.e. to 2^-16 of it, and absolute 2^-25 below.
//
// Warps: 0-3 softmax and results, 4 issues the MMAs, 5.. load (one warp of
// bulk copies for f16, eight warps for i8).  Every wait is bounded; one that
// runs out sets the cache's flag, and the CTA winds down (copies and MMAs
// drained, TMEM freed) without results.
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
constexpr int kWaitLimit = 1 << 20;
constexpr int kDrainLimit = 1 << 24;
constexpr int kScaleRing = 4;
constexpr int kMmaWarp = 4, kLoadWarp = 5;

template <int HD, int FMT, bool F32Q>
struct Geo {
  static constexpr int kTileBytes = kT * HD * 2;  // an f16 tile of keys or values
  static constexpr int kQlo = F32Q ? kM * HD * 2 : 0;
  // f32 rows at hd 256: 64 KB of Q parts and two tiles each; three otherwise
  static constexpr int kRing = F32Q && HD == 256 ? 2 : HD == 256 ? 3 : 4;
  static constexpr int kScaleBytes = kScaleRing * (2 * kT + 4) * 4;
  static constexpr int kSmem = 2 * kRing * kTileBytes + kQlo + kScaleBytes + 1024;
  static constexpr int kLoadWarps = FMT == kKvI8 ? 8 : 1;
  static constexpr int kThreads = (kLoadWarp + kLoadWarps) * 32;
  static constexpr uint32_t kTmemS = HD, kTmemQ = HD + 2 * kT;
  static constexpr uint32_t kTmemCols = HD + 2 * kT + HD / 2 > 256 ? 512 : 256;
  static_assert(HD + 2 * kT + HD / 2 <= 512, "O, S and Q fit the tensor memory");
  static_assert(kRing * kTileBytes >= kM * HD * 2, "Q is staged where V tiles come later");
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
__device__ __forceinline__ void tmem_st32(uint32_t a, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(a),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

template <int HD, int FMT, bool F32Q>
__global__ void __launch_bounds__(Geo<HD, FMT, F32Q>::kThreads, 1)
    kv_attend_wide_kernel(const __grid_constant__ KvAttnArgs a, const bool vec) {
  using G_ = Geo<HD, FMT, F32Q>;
  constexpr int R = G_::kRing, TB = G_::kTileBytes;
  __shared__ __align__(8) uint64_t kfull[R], kempty[R], vfull[R], vempty[R], sfull[2], pfull[2], odone, qfull, drained;
  __shared__ __align__(8) uint64_t scfull[kScaleRing], scempty[kScaleRing];
  __shared__ uint32_t tmem_s;
  __shared__ int abort_s;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (su32(smem_raw) & 1023)) & 1023);
  uint8_t* kring = smem;
  uint8_t* vring = smem + R * TB;
  uint8_t* qlo = vring + R * TB;
  float* scales = reinterpret_cast<float*>(qlo + G_::kQlo);  // [ring][keys 64, values 64, exponent, pad]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const KvPool& p = a.pool;
  const int group = a.heads / p.nkv;
  const int slot = blockIdx.x % a.slots;
  const int kvh = blockIdx.x / a.slots % p.nkv;
  const int tile = blockIdx.x / a.slots / p.nkv;
  KvTileRows tr;
  if (!kv_tile_rows(a.b, tile, kM, group, lane, &tr)) return;
  const KvSpan sp = kv_span(a, tr, kM, slot);
  if (sp.outside && threadIdx.x == 0) atomicOr(p.flag, kKvBadPage);
  if (sp.first >= sp.end && a.slots > 1) return;

  if (threadIdx.x == 0) {
    for (int s = 0; s < R; s++) {
      bar_init(&kfull[s], FMT == kKvI8 ? 4 : 1);
      bar_init(&kempty[s], 1);
      bar_init(&vfull[s], FMT == kKvI8 ? 4 : 1);
      bar_init(&vempty[s], 1);
    }
    for (int b = 0; b < 2; b++) {
      bar_init(&sfull[b], 1);
      bar_init(&pfull[b], 4);
    }
    for (int s = 0; s < kScaleRing; s++) {
      bar_init(&scfull[s], FMT == kKvI8 ? 2 : 1);
      bar_init(&scempty[s], 4);
    }
    bar_init(&odone, 1);
    bar_init(&qfull, 4);
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
    if (__any_sync(0xffffffffu, *abort_v)) return false;
    const bool ok = __all_sync(0xffffffffu, bar_wait(b, parity, kWaitLimit));
    if (!ok) give_up();
    return ok;
  };

  if (warp < 4) {
    // ------------------------------------------------------- query rows
    // Row by row with the lanes along the head; first parts go through the V
    // ring (chunks XOR-ed with the row) to the thread that owns the row.
    const int r0 = warp * 32;
    float cq = 0.f;
    int rp = -1;
    {
      constexpr int N = HD / 32, U = 8;  // U rows in flight
      for (int rb = 0; rb < 32; rb += U) {
        float x[U][N];
#pragma unroll
        for (int u = 0; u < U; u++) {
          const int rr = tr.r0 + r0 + rb + u;
          const bool live = rr < tr.nr;
          const int i = rr / group, h = kvh * group + rr % group;
          const int64_t o = (int64_t)(tr.row0 + i) * a.q.row + (int64_t)h * a.q.head + lane * N;
          if (live) {
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
          const int row = r0 + rb + u, rr = tr.r0 + row;
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
          uint8_t* d = vring + row * HD * 2 + ((c ^ (row & 7)) << 4) + (byte & 15);
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
          if (lane == rb + u) {
            cq = fmaxf(pow2i(e) * fabsf(a.scale_log2e), FLT_MIN);  // never 0: hidden scores stay -inf
            if (rr < tr.nr) rp = (int)max(min(tr.pos + rr / group, (int64_t)INT_MAX), (int64_t)-1);
          }
        }
      }
    }
    __syncwarp();
    const int row = r0 + lane;
    const uint32_t lanes = tmem + ((uint32_t)r0 << 16);
#pragma unroll
    for (int b = 0; b < HD / 64; b++) {
      uint32_t v[32];
#pragma unroll
      for (int c = 0; c < 8; c++) {
        const uint4 w = *reinterpret_cast<const uint4*>(vring + row * HD * 2 + (((b * 8 + c) ^ (row & 7)) << 4));
        v[4 * c] = w.x, v[4 * c + 1] = w.y, v[4 * c + 2] = w.z, v[4 * c + 3] = w.w;
      }
      tmem_st32(lanes + G_::kTmemQ + 32 * b, v);
    }
    tmem_wait_st();
    tc_before();
    async_fence();  // the second parts and the ring's hand-over to the copies
    __syncwarp();
    if (lane == 0) bar_arrive(&qfull);

    // ----------------------------------------------------------- softmax
    float m = -INFINITY, l = 0.f;
    int ev = -100;
    bool ok = true;
    int it = 0;
    for (int ti = sp.first; ti < sp.end; ti = sp.next(ti), it++) {
      const int b = it & 1, sr = it % kScaleRing, t0 = ti * kT;
      const float* sc = scales + sr * (2 * kT + 4);
      ok = wait(&scfull[sr], (it / kScaleRing) & 1) && wait(&sfull[b], (it >> 1) & 1);
      if (!ok) break;
      tc_after();
      const uint32_t st = lanes + G_::kTmemS + b * kT;
      uint32_t s0[32], s1[32];
      tmem_ld32(st, s0);
      tmem_ld32(st + 32, s1);
      tmem_wait(s0);
      tmem_wait(s1);
      float x[kT];
#pragma unroll
      for (int j = 0; j < 32; j += 4) {
        const float4 k0 = *reinterpret_cast<const float4*>(sc + j), k1 = *reinterpret_cast<const float4*>(sc + 32 + j);
        x[j] = __uint_as_float(s0[j]) * k0.x, x[j + 1] = __uint_as_float(s0[j + 1]) * k0.y;
        x[j + 2] = __uint_as_float(s0[j + 2]) * k0.z, x[j + 3] = __uint_as_float(s0[j + 3]) * k0.w;
        x[32 + j] = __uint_as_float(s1[j]) * k1.x, x[33 + j] = __uint_as_float(s1[j + 1]) * k1.y;
        x[34 + j] = __uint_as_float(s1[j + 2]) * k1.z, x[35 + j] = __uint_as_float(s1[j + 3]) * k1.w;
      }
      const bool whole = sp.whole(t0, kT);
      uint64_t hidden = 0;
      if (!whole) {
#pragma unroll
        for (int j = 0; j < kT; j++)
          if (!sp.sees(rp, t0 + j)) {
            x[j] = -INFINITY;
            hidden |= 1ull << j;
          }
      }
      float mt[8];
#pragma unroll
      for (int j = 0; j < 8; j++) mt[j] = x[j];
#pragma unroll
      for (int j = 8; j < kT; j++) mt[j & 7] = fmaxf(mt[j & 7], x[j]);
      const float mx = fmaxf(fmaxf(fmaxf(mt[0], mt[1]), fmaxf(mt[2], mt[3])), fmaxf(fmaxf(mt[4], mt[5]), fmaxf(mt[6], mt[7]))) * cq;
      // the maximum and the exponent move only when weights could overflow
      const float mn = mx > m + 8.f || m == -INFINITY ? mx : m;
      const float ms = mn == -INFINITY ? 0.f : mn;
      const int et = __float_as_int(sc[2 * kT]);
      const int en = et > ev ? et + 2 : ev;
      const float alpha = m == mn ? 1.f : ex2(m - ms);
      const float fo = alpha * (ev - en < -126 ? 0.f : pow2i(max(ev - en, -126)));
      m = mn;
      ev = en;
      l *= alpha;
      const float up = pow2i(-en) * 128.f;
      uint32_t w[32];
      uint32_t wl[F32Q ? 32 : 1];
      float la[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < kT; j += 4) {
        const float4 vs = *reinterpret_cast<const float4*>(sc + kT + j);
        const float p0 = ex2(fmaf(x[j], cq, -ms)), p1 = ex2(fmaf(x[j + 1], cq, -ms)), p2 = ex2(fmaf(x[j + 2], cq, -ms)),
                    p3 = ex2(fmaf(x[j + 3], cq, -ms));
        la[0] += p0, la[1] += p1, la[2] += p2, la[3] += p3;
        float w0 = p0 * (vs.x * up), w1 = p1 * (vs.y * up), w2 = p2 * (vs.z * up), w3 = p3 * (vs.w * up);
        if (!whole) {  // a hidden token weighs zero whatever its scale is
          if (hidden >> j & 1) w0 = 0.f;
          if (hidden >> (j + 1) & 1) w1 = 0.f;
          if (hidden >> (j + 2) & 1) w2 = 0.f;
          if (hidden >> (j + 3) & 1) w3 = 0.f;
        }
        w[j / 2] = pack2(w0, w1);
        w[j / 2 + 1] = pack2(w2, w3);
        if constexpr (F32Q) {
          const float2 f0 = unpack2(w[j / 2]), f1 = unpack2(w[j / 2 + 1]);
          wl[j / 2] = pack2(w0 - f0.x, w1 - f0.y);
          wl[j / 2 + 1] = pack2(w2 - f1.x, w3 - f1.y);
        }
      }
      l += (la[0] + la[1]) + (la[2] + la[3]);
      __syncwarp();
      if (lane == 0) bar_arrive(&scempty[sr]);
      tmem_st32(st, w);
      if constexpr (F32Q) tmem_st32(st + 32, wl);
      if (it > 0 && __any_sync(0xffffffffu, fo != 1.f)) {
        ok = wait(&odone, (it - 1) & 1);  // the previous product has been added
        if (!ok) break;
        tc_after();
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
          uint32_t o[32];
          tmem_ld32(lanes + c, o);
          tmem_wait(o);
#pragma unroll
          for (int j = 0; j < 32; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * fo);
          tmem_st32(lanes + c, o);
        }
      }
      tmem_wait_st();
      tc_before();
      __syncwarp();
      if (lane == 0) bar_arrive(&pfull[b]);
    }
    // ----------------------------------------------------------- results
    tmem_wait_st();  // no store in flight past this point
    // The last tile's scores say that the product two tiles back was added, so
    // the two after it are waited for in turn: a parity names a phase only
    // while no other of its kind is outstanding.
    if (ok && it > 1) ok = wait(&odone, it & 1);
    if (ok && it > 0) ok = wait(&odone, (it - 1) & 1);
    if (ok && !__any_sync(0xffffffffu, *abort_v)) {
      tc_after();
      const int rr = tr.r0 + row;
      const int grow = tr.row0 + rr / group, h = kvh * group + rr % group;
      const int64_t rh = (int64_t)grow * a.heads + h;
      const bool live = rr < tr.nr;
      const float f = a.slots > 1 ? 0x1p-7f : l != 0.f ? __fdiv_rn(0x1p-7f, l) : 0.f;
      const float back = pow2i(ev);
      if (a.slots > 1 && live) a.ml[rh * a.slots + slot] = make_float2(m, l);
      auto put = [&](auto* dst, bool v16) {
        using T = std::remove_reference_t<decltype(*dst)>;
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
          uint32_t o[32];
          if (it > 0) {
            tmem_ld32(lanes + c, o);
            tmem_wait(o);
          } else {
#pragma unroll
            for (int j = 0; j < 32; j++) o[j] = 0;
          }
          if (!live) continue;
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            float y[8];
#pragma unroll
            for (int k = 0; k < 8; k++) y[k] = __uint_as_float(o[j + k]) * back * f;
            store_n<T, 8>(dst + c + j, v16, y);
          }
        }
      };
      const int64_t at = (int64_t)grow * a.out.row + (int64_t)h * a.out.head;
      if (a.slots > 1) put(a.part + (rh * a.slots + slot) * HD, true);
      else if constexpr (F32Q) put(static_cast<float*>(a.out.p) + at, vec);
      else if (a.dtype == F16) put(static_cast<__half*>(a.out.p) + at, vec);
      else put(static_cast<__nv_bfloat16*>(a.out.p) + at, vec);
    }
  } else if (warp == kMmaWarp) {
    // --------------------------------------------------------- products
    // The whole warp waits, one lane issues.
    constexpr uint32_t dS = idesc(kT, false), dO = idesc(HD, true);
    const uint32_t k0 = su32(kring), v0 = su32(vring), ql = su32(qlo);
    bool ok = wait(&qfull, 0);
    tc_after();
    auto score = [&](int i) {
      const int s = i % R;
      if (!wait(&kfull[s], (i / R) & 1)) return false;
      tc_after();
      if (lane == 0) {
        const uint32_t d = tmem + G_::kTmemS + (i & 1) * kT, kb = k0 + s * TB;
#pragma unroll
        for (int st = 0; st < HD / 16; st++)
          mma_ts(d, tmem + G_::kTmemQ + 8 * st, sw128(kb + (st >> 2) * (kT * 128) + (st & 3) * 32, 16), dS, st > 0);
        if constexpr (F32Q) {
#pragma unroll
          for (int st = 0; st < HD / 16; st++)
            mma_ss(d, sw128(ql + (st >> 2) * (kM * 128) + (st & 3) * 32, 16),
                   sw128(kb + (st >> 2) * (kT * 128) + (st & 3) * 32, 16), dS, 1);
        }
        commit(&sfull[i & 1]);
        commit(&kempty[s]);
      }
      __syncwarp();
      return true;
    };
    int it = 0, ti = sp.first;
    if (ok && ti < sp.end) ok = score(0);
    for (; ok && ti < sp.end; it++) {
      ti = sp.next(ti);
      if (ti < sp.end && !(ok = score(it + 1))) break;
      const int s = it % R;
      ok = wait(&pfull[it & 1], (it >> 1) & 1) && wait(&vfull[s], (it / R) & 1);
      if (!ok) break;
      tc_after();
      if (lane == 0) {
        const uint32_t pa = tmem + G_::kTmemS + (it & 1) * kT, vb = v0 + s * TB;
#pragma unroll
        for (int part = 0; part < (F32Q ? 2 : 1); part++)
#pragma unroll
          for (int kk = 0; kk < kT / 16; kk++)
            mma_ts(tmem, pa + part * 32 + 8 * kk, sw128(vb + kk * 2048, kT * 128), dO, it > 0 || kk > 0 || part > 0);
        commit(&vempty[s]);
        commit(&odone);
      }
      __syncwarp();
    }
    if (lane == 0) commit(&drained);  // every product issued above has completed when this fires
    __syncwarp();
    bar_wait(&drained, 0, kDrainLimit);
  } else if constexpr (FMT == kKvF16) {
    // ------------------------------------------------ bulk copies (f16)
    const int rt = min(p.page_tokens, kT), runs = kT / rt;
    const int64_t hb = kv_head_bytes(FMT, HD, p.page_tokens);
    constexpr int kParts = HD / 64;
    auto page_of = [&](int ti) {
      const int64_t pos = (int64_t)ti * kT + (int64_t)lane * rt;
      const bool in = lane < runs && pos < sp.tokens;
      int page = in ? kv_page(p, a.b, tr.seq, pos) : -1;
      const int first = __shfl_sync(0xffffffffu, page, 0);
      if (!in) page = first;
      return max(page, 0);
    };
    auto copy = [&](int ti, int page, const uint8_t* pool, uint8_t* dst, uint64_t* full) {
      const int tp = (ti * kT) & (p.page_tokens - 1);
      if (lane == 0) bar_expect(full, TB);
      __syncwarp();
      for (int c0 = 0; c0 < runs * kParts; c0 += 32) {
        const int c = c0 + lane, run = min(c / kParts, runs - 1), part = c % kParts;
        const int64_t at = (int64_t)__shfl_sync(0xffffffffu, page, run) * p.nkv + kvh;
        if (c < runs * kParts)
          bulk_load(su32(dst + (part * kT + run * rt) * 128), pool + at * hb + ((int64_t)part * p.page_tokens + tp) * 128,
                    rt * 128, full);
      }
      __syncwarp();
    };
    // scales of two tokens a lane, and the exponent above the values'
    auto put_scales = [&](int i, int ti, int page) {
      const int sr = i % kScaleRing;
      if (i >= kScaleRing && !wait(&scempty[sr], ((i / kScaleRing) + 1) & 1)) return false;
      float* sc = scales + sr * (2 * kT + 4);
      uint32_t top = 0;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int t = lane + 32 * h;
        const int64_t at = ((int64_t)__shfl_sync(0xffffffffu, page, t / rt) * p.nkv + kvh) * p.page_tokens +
                           ((ti * kT + t) & (p.page_tokens - 1));
        const float v = p.vs[at];
        sc[t] = p.ks[at];
        sc[kT + t] = v;
        const uint32_t bits = __float_as_uint(v);
        if (bits < 0x7f800000u && ti * kT + t < sp.tokens) top = max(top, bits);
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0) sc[2 * kT] = __int_as_float(max((int)(top >> 23), 1) - 126);
      __syncwarp();
      if (lane == 0) bar_arrive(&scfull[sr]);
      return true;
    };
    int it = 0, ti = sp.first, kn = 0, vn = 0;  // tiles of keys and values requested
    bool ok = true;
    if (ti < sp.end) {
      int page = page_of(ti);
      copy(ti, page, p.k, kring, &kfull[0]);
      kn = 1;
      ok = put_scales(0, ti, page);
      for (; ok && ti < sp.end; it++) {
        const int nt = sp.next(ti);
        int npage = 0;
        if (nt < sp.end) {
          npage = page_of(nt);
          const int s = (it + 1) % R;
          if (it + 1 >= R && !(ok = wait(&kempty[s], (((it + 1) / R) + 1) & 1))) break;
          copy(nt, npage, p.k, kring + s * TB, &kfull[s]);
          kn = it + 2;
          if (!(ok = put_scales(it + 1, nt, npage))) break;
        }
        const int s = it % R;
        // the V ring holds the query rows first
        if (it == 0 && !(ok = wait(&qfull, 0))) break;
        if (it >= R && !(ok = wait(&vempty[s], ((it / R) + 1) & 1))) break;
        copy(ti, page, p.v, vring + s * TB, &vfull[s]);
        vn = it + 1;
        ti = nt;
        page = npage;
      }
    }
    for (int s = 0; s < R; s++) {  // no copy outlives the CTA
      if (kn > s) bar_wait(&kfull[(kn - 1 - s) % R], ((kn - 1 - s) / R) & 1, kDrainLimit);
      if (vn > s) bar_wait(&vfull[(vn - 1 - s) % R], ((vn - 1 - s) / R) & 1, kDrainLimit);
    }
  } else {
    // ------------------------------------------- expansion to f16 (i8)
    // Warps 5-8 keys, 9-12 values; a thread takes HD / 32 16-byte chunks of a
    // tile, all loaded before the ring's slot is waited for.
    const int isv = (warp - kLoadWarp) >> 2, tid = threadIdx.x - (kLoadWarp + 4 * isv) * 32;
    const bool first_warp = tid < 32;
    uint8_t* ring = isv ? vring : kring;
    uint64_t* full = isv ? vfull : kfull;
    uint64_t* empty = isv ? vempty : kempty;
    const uint8_t* pool = isv ? p.v : p.k;
    const float* spool = isv ? p.vs : p.ks;
    const int64_t hb = kv_head_bytes(FMT, HD, p.page_tokens);
    const int rt = min(p.page_tokens, kT), runs = kT / rt;
    constexpr int C = HD / 16, TP = 128 / C, NP = kT / TP;  // chunks a token, tokens a pass, passes
    const int ch = tid % C, tk = tid / C;
    auto page_of = [&](int ti) {
      const int64_t pos = (int64_t)ti * kT + (int64_t)lane * rt;
      const bool in = ti < sp.end && lane < runs && pos < sp.tokens;
      int page = in ? kv_page(p, a.b, tr.seq, pos) : -1;
      const int f = __shfl_sync(0xffffffffu, page, 0);
      if (!in) page = f;
      return max(page, 0);
    };
    uint4 raw[NP];
    float sv[2] = {0.f, 0.f};
    auto load = [&](int ti, int page) {
#pragma unroll
      for (int i = 0; i < NP; i++) {
        const int t = i * TP + tk;  // physical chunk ch of token t
        const int64_t at = (int64_t)__shfl_sync(0xffffffffu, page, t / rt) * p.nkv + kvh;
        raw[i] = __ldg(reinterpret_cast<const uint4*>(pool + at * hb + (int64_t)((ti * kT + t) & (p.page_tokens - 1)) * HD + 16 * ch));
      }
      if (first_warp) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int t = lane + 32 * h;
          const int64_t at = (int64_t)__shfl_sync(0xffffffffu, page, t / rt) * p.nkv + kvh;
          sv[h] = spool[at * p.page_tokens + ((ti * kT + t) & (p.page_tokens - 1))];
        }
      }
    };
    bool ok = true;
    if (isv && sp.first < sp.end) ok = wait(&qfull, 0);  // the V ring holds the query rows first
    int ti = sp.first, nt = sp.next(ti);
    int page = ok && ti < sp.end ? page_of(ti) : 0;
    if (ok && ti < sp.end) load(ti, page);
    page = page_of(nt);
    for (int it = 0; ok && ti < sp.end; it++) {
      const int s = it % R, sr = it % kScaleRing;
      const int nn = sp.next(nt), npage = page_of(nn);
      if (first_warp) {
        if (it >= kScaleRing && !(ok = wait(&scempty[sr], ((it / kScaleRing) + 1) & 1))) break;
        float* sc = scales + sr * (2 * kT + 4);
        uint32_t top = 0;
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int t = lane + 32 * h;
          sc[isv * kT + t] = sv[h];
          const uint32_t bits = __float_as_uint(sv[h]);
          if (bits < 0x7f800000u && ti * kT + t < sp.tokens) top = max(top, bits);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if (isv && lane == 0) sc[2 * kT] = __int_as_float(max((int)(top >> 23), 1) - 126);
        __syncwarp();
        if (lane == 0) bar_arrive(&scfull[sr]);
      }
      if (it >= R && !(ok = wait(&empty[s], ((it / R) + 1) & 1))) break;
      uint8_t* dst = ring + s * TB;
#pragma unroll
      for (int i = 0; i < NP; i++) {
        const int t = i * TP + tk, c = ch ^ i8_swizzle(t, HD);  // its 16 elements are chunks 2c and 2c + 1 of the f16 row
        const uint2 x0 = biased4_to_f16(raw[i].x), x1 = biased4_to_f16(raw[i].y), x2 = biased4_to_f16(raw[i].z),
                    x3 = biased4_to_f16(raw[i].w);
        const uint4 lo = make_uint4(x0.x, x0.y, x1.x, x1.y), hi = make_uint4(x2.x, x2.y, x3.x, x3.y);
        uint8_t* rowp = dst + ((c >> 2) * kT + t) * 128;
        // the two 64-element blocks that a quarter warp meets take their halves
        // in turn, so that its eight stores fall on different banks
        const int turn = (c >> 2) & 1, c8 = (c & 3) * 2;
        *reinterpret_cast<uint4*>(rowp + (((c8 + turn) ^ (t & 7)) << 4)) = turn ? hi : lo;
        *reinterpret_cast<uint4*>(rowp + (((c8 + 1 - turn) ^ (t & 7)) << 4)) = turn ? lo : hi;
      }
      async_fence();
      __syncwarp();
      if (lane == 0) bar_arrive(&full[s]);
      if (nt < sp.end) load(nt, page);
      ti = nt;
      nt = nn;
      page = npage;
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
