// kv_attend.cu -- attention of few query rows over the paged cache (single
// tokens, verify passes, any batch of short row groups), split over the
// tokens, and the join of the splits.
//
// Mathematics.  For a query row at position p with scale c,
//     s_t = c q . k_t,  o = sum_t 2^(s_t log2e - m) v_t / sum_t 2^(s_t log2e - m)
// over the visible t, in one pass with the running maximum m and sum l.  Keys
// and values are kept as k_t = a_t K_t, v_t = b_t V_t (K, V integers of 8
// bits or f16, a and b f32), so the matrix instructions multiply K and V as
// they are stored, a_t scales the score and b_t the weight:
//     s_t = a_t (q . K_t),  o = sum_t (p_t b_t) V_t / l.
// Weights enter as f16: p_t b_t 2^(14 - e), with 2^e above every b that the row
// has seen so far (e grows like m, a row's own; the accumulators follow by
// powers of two), so the largest weights are at most 2^14 and weights down to
// 2^-28 of them keep 11 bits.
// f32 rows split queries and weights into two f16 parts each (22 bits).  A
// query row is divided by a power of two first, which joins its scale.
//
// Work split.  A CTA takes 8 NT query rows (rows x heads of one KV head) and
// one chunk of the tokens; partial results {m, l, o} go to the workspace and
// a second kernel joins a row's chunks.  Keys are the M side of the first
// product (S^T = K Q^T) and value elements that of the second (O^T = V^T
// P^T), so 8 rows fill an instruction: with 8 query heads to a KV head a
// single token needs no padding.  Four warps: a warp scores 16 of the tile's
// 64 tokens for all rows, then sums a quarter of the head's elements over all
// 64 tokens; so each stored byte is expanded to f16 once.  A fifth warp keeps
// the next tiles' bulk copies in flight.  All rows' arithmetic is their own
// and does not depend on NT: a row's result is the same in any batch.
//
// Bound: the cache's bytes for 8 query rows (one f16 token over 262144 positions
// of 2 heads of 256: 87 us, 6.2 TB/s with its join; bf16 over i8: 54 us, 5.1
// TB/s, f32 59, where the chain of a tile and a CTA's start and end weigh twice
// as much; 64 bf16 tokens over 6000 i8 positions each: 79 us, 5.1 TB/s); the
// tensor pipe and shared memory from about 64 query rows on (spills too: 64 f32
// rows of hd 256 want some 90 registers more than there are).  One token over
// 4096 positions takes 9.5 us: start, one pass of loads, and the join, each
// bound by latency.
#include <cfloat>
#include <climits>
#include <cstdlib>
#include <type_traits>
#include "kv_device.cuh"
#include "kv_split.cuh"
#include "kv_wide.h"
#include "model_kernels.cuh"

namespace iq {
namespace {

using namespace kvp;

constexpr int kTile = kKvTile;
constexpr int kWarps = 4;
constexpr int kWaitLimit = 1 << 19;   // of 2 us each: a second

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// Transpose of an 8 x 8 matrix of f16 held as fragments.
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void consumers_sync() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }
// The same, and whether any thread's `bad` is set.
__device__ __forceinline__ bool consumers_any(bool bad) {
  uint32_t r;
  asm volatile(
      "{ .reg .pred p, q; setp.ne.u32 q, %1, 0; barrier.cta.red.or.pred p, 1, 128, q; selp.u32 %0, 1, 0, p; }"
      : "=r"(r)
      : "r"((uint32_t)bad)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

template <int HD, int FMT, int NT, bool F32Q>
struct Geo {
  static constexpr KvNarrow kGeo = kv_narrow(FMT, HD, NT, F32Q);
  static constexpr int kTileBytes = kTile * HD * (FMT == kKvI8 ? 1 : 2);  // of keys, and of values
  static constexpr int kTQ = 8 * NT;
  static constexpr int kQld = HD * 2 + 16;                                // bytes of a staged query row
  static constexpr int kQBytes = kTQ * kQld * (F32Q ? 2 : 1);
  static constexpr int kPBytes = NT * 4 * 32 * 8 * (F32Q ? 2 : 1);
  static_assert(kGeo.fixed == kQBytes + kPBytes + 12 * kTQ * 4 + 64, "queries, weights, maxima, factors, positions, exponents");
  static constexpr int kStages = kGeo.stages, kSmem = kGeo.smem;
  static_assert(kStages >= 2, "two stages keep a copy in flight");
};

// CTAs an SM that registers must allow: those for which they suffice without
// spills (five warps of up to 168 registers: two).
template <int HD, int FMT, int NT, bool F32Q>
constexpr int kMinCtas = NT == 1 ? 3 : (HD == 64 && NT == 4) || (HD == 256 && NT == 2 && FMT == kKvI8 && !F32Q) ? 2 : 1;

template <int HD, int FMT, int NT, bool F32Q>
__global__ void __launch_bounds__(160, kMinCtas<HD, FMT, NT, F32Q>) kv_attend_kernel(const __grid_constant__ KvAttnArgs a, const bool vec) {
  using G_ = Geo<HD, FMT, NT, F32Q>;
  constexpr int TQ = G_::kTQ, ST = G_::kStages, QLD = G_::kQld;
  __shared__ __align__(8) uint64_t full[ST], empty[ST];
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (su32(smem_raw) & 1023)) & 1023);
  float* scales = reinterpret_cast<float*>(smem + ST * 2 * G_::kTileBytes);  // [stage][keys, values][64]
  uint8_t* qs = reinterpret_cast<uint8_t*>(scales + ST * 128);               // [part][TQ][QLD]
  uint2* ps = reinterpret_cast<uint2*>(qs + G_::kQBytes);                    // [part][NT][4][32]
  float* mx = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(ps) + G_::kPBytes);  // [4][TQ]
  float* cq = mx + 4 * TQ;                                                   // [TQ] row factor
  int* rpos = reinterpret_cast<int*>(cq + TQ);                               // [TQ] row position, -1: none
  int* evr = rpos + TQ;                                                      // [4][TQ] exponents of a masked tile
  float2* esc = reinterpret_cast<float2*>(evr + 4 * TQ);                     // [TQ] {factor of the sums, of the scales}
  int* evw = reinterpret_cast<int*>(esc + TQ);                               // [4] exponent of a tile

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const KvPool& p = a.pool;
  const int group = a.heads / p.nkv;
  const int slot = blockIdx.x % a.slots;
  const int kvh = blockIdx.x / a.slots % p.nkv;
  const int tile = blockIdx.x / a.slots / p.nkv;
  KvTileRows tr;
  if (!kv_tile_rows(a.b, tile, TQ, group, lane, &tr)) return;
  const KvSpan sp = kv_span(a, tr, TQ, slot);
  if (sp.outside && threadIdx.x == 0) atomicOr(p.flag, kKvBadPage);
  // splits that no row of the tile sees are not read by the join
  if (sp.first >= sp.end && a.slots > 1) return;

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; s++) {
      bar_init(&full[s], 1);
      bar_init(&empty[s], kWarps);
    }
    bar_init_fence();
  }
  __syncthreads();

  if (warp == kWarps) {
    // ------------------------------------------------------ copies in flight
    const int rt = min(p.page_tokens, kTile), runs = kTile / rt;
    const int64_t hb = kv_head_bytes(FMT, HD, p.page_tokens);
    constexpr int kParts = FMT == kKvI8 ? 1 : HD / 64;  // contiguous pieces of a run
    const int per = 2 * kParts + 2, copies = runs * per;
    auto page_of = [&](int ti) {
      // runs behind the last token are filled from the tile's first page
      const int64_t pos = (int64_t)ti * kTile + (int64_t)lane * rt;
      const bool in = lane < runs && pos < sp.tokens;
      int page = in ? kv_page(p, a.b, tr.seq, pos) : -1;
      const int first = __shfl_sync(0xffffffffu, page, 0);
      if (!in) page = first;
      return max(page, 0);
    };
    int it = 0, page = sp.first < sp.end ? page_of(sp.first) : 0;
    bool ok = true;
    for (int ti = sp.first; ti < sp.end; it++) {
      const int s = it % ST;
      if (it >= ST && !__all_sync(0xffffffffu, bar_wait(&empty[s], ((it / ST) + 1) & 1, a.wait_limit))) {
        ok = false;
        break;
      }
      if (lane == 0) bar_expect(&full[s], 2 * G_::kTileBytes + 2 * kTile * 4);
      __syncwarp();
      const int tp = (ti * kTile) & (p.page_tokens - 1);
      uint8_t* kt = smem + s * 2 * G_::kTileBytes;
      for (int c0 = 0; c0 < copies; c0 += 32) {
        const int c = c0 + lane, run = min(c / per, runs - 1), what = c % per;
        const int64_t at = (int64_t)__shfl_sync(0xffffffffu, page, run) * p.nkv + kvh;
        if (c >= copies || (a.test_skip && blockIdx.x == 0 && it == 0 && c == 0)) continue;
        if (what < 2 * kParts) {
          const int part = what % kParts, isv = what / kParts;
          const uint8_t* src = (isv ? p.v : p.k) + at * hb;
          uint8_t* dst = kt + isv * G_::kTileBytes;
          if constexpr (FMT == kKvI8)
            bulk_load(su32(dst + run * rt * HD), src + (int64_t)tp * HD, rt * HD, &full[s]);
          else
            bulk_load(su32(dst + (part * kTile + run * rt) * 128), src + ((int64_t)part * p.page_tokens + tp) * 128,
                      rt * 128, &full[s]);
        } else {
          const int isv = what - 2 * kParts;
          bulk_load(su32(scales + s * 128 + isv * 64 + run * rt), (isv ? p.vs : p.ks) + at * p.page_tokens + tp, rt * 4,
                    &full[s]);
        }
      }
      ti = sp.next(ti);
      if (ti < sp.end) page = page_of(ti);
    }
    if (!ok && lane == 0) atomicOr(p.flag, kKvTimeout);
    // no copy outlives the CTA, also when the readers gave up
    for (int s = 0; s < ST; s++)
      if (it > s) bar_wait(&full[s], ((it - 1 - s) / ST) & 1, 4 * a.wait_limit);
    return;
  }

  // ---------------------------------------------------------- query rows
  // Elements are stored in the order in which a lane's fragments take them:
  // 16 contiguous halves serve four instructions.
  for (int r = warp; r < TQ; r += kWarps) {
    const int rr = tr.r0 + r;
    const bool live = rr < tr.nr;
    const int i = rr / group, h = kvh * group + rr % group;
    constexpr int N = HD / 32;
    float x[N];
    if (live) {
      const int64_t o = (int64_t)(tr.row0 + i) * a.q.row + (int64_t)h * a.q.head + lane * N;
      if constexpr (F32Q) load_n<float, N>(static_cast<const float*>(a.q.p) + o, vec, x);
      else if (a.dtype == F16) load_n<__half, N>(static_cast<const __half*>(a.q.p) + o, vec, x);
      else load_n<__nv_bfloat16, N>(static_cast<const __nv_bfloat16*>(a.q.p) + o, vec, x);
    } else {
#pragma unroll
      for (int j = 0; j < N; j++) x[j] = 0.f;
    }
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < N; j++) m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);
    const int e = f16_exponent(__uint_as_float(__reduce_max_sync(0xffffffffu, m)));
    const float f = pow2i(-e);
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int d = lane * N + j;
      const int o = FMT == kKvI8 ? d
                                 : (d & ~63) + 16 * ((d & 7) >> 1) + 4 * ((d & 63) >> 4) + 2 * ((d >> 3) & 1) + (d & 1);
      const float y = x[j] * f;
      const __half hi = __float2half_rn(y);
      *reinterpret_cast<__half*>(qs + r * QLD + 2 * o) = hi;
      if constexpr (F32Q)
        *reinterpret_cast<__half*>(qs + (TQ + r) * QLD + 2 * o) = __float2half_rn(y - __half2float(hi));
    }
    if (lane == 0) {
      cq[r] = pow2i(e) * a.scale_log2e;
      rpos[r] = live ? (int)max(min(tr.pos + i, (int64_t)INT_MAX), (int64_t)-1) : -1;
    }
  }
  consumers_sync();

  const int g = lane >> 2, t = lane & 3;
  constexpr int kBlocks = HD / 32;                       // 32-element blocks of the head
  constexpr int kMine = kBlocks >= kWarps ? kBlocks / kWarps : 1;
  const bool sums = kBlocks >= kWarps || warp < kBlocks;  // hd 64: two warps sum
  float o[kMine][2][NT][4];
#pragma unroll
  for (int b = 0; b < kMine; b++)
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int c = 0; c < 4; c++) o[b][m][n][c] = 0.f;
  float mrow[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; n++) mrow[n][0] = mrow[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
  // Rows have one exponent, evu, until a masked tile: then each has its own,
  // which esc keeps as 2^(14 - e), at most evu, until a whole tile reaches evu.
  // (Every row's in every thread's registers: spills, and 25% more time for 64
  // f32 rows of hd 256.)
  int evu = -100;  // so that 2^(14 - e) is finite
  bool one = true;
  bool failed = false;

  int it = 0;
  for (int ti = sp.first; ti < sp.end; ti = sp.next(ti), it++) {
    const int s = it % ST, t0 = ti * kTile;
    const uint32_t kt = su32(smem + s * 2 * G_::kTileBytes), vt = kt + G_::kTileBytes;
    const float* sc = scales + s * 128;
    const bool ok = __all_sync(0xffffffffu, bar_wait(&full[s], (it / ST) & 1, a.wait_limit));
    float sa[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++) sa[n][0] = sa[n][1] = sa[n][2] = sa[n][3] = 0.f;
    if (ok) {
      // ------------------------------------------------ S^T = K Q^T
      const uint32_t qa = su32(qs) + g * QLD + 32 * t;
#pragma unroll
      for (int j = 0; j < HD / 64; j++) {
        uint32_t ka[4][4];  // fragments of the group's four instructions
        if constexpr (FMT == kKvI8) {
          const uint32_t at = kt + (16 * warp + g) * HD + (((4 * j + t) ^ i8_swizzle(g, HD)) << 4);
          const uint4 w0 = lds128(at), w1 = lds128(at + 8 * HD);
          const uint32_t u0[4] = {w0.x, w0.y, w0.z, w0.w}, u1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint2 x = biased4_to_f16(u0[i]), y = biased4_to_f16(u1[i]);
            ka[i][0] = x.x, ka[i][1] = y.x, ka[i][2] = x.y, ka[i][3] = y.y;
          }
        } else {
          const int m = lane >> 3, row = 16 * warp + (lane & 7) + (m & 1) * 8;
#pragma unroll
          for (int i = 0; i < 4; i++)
            ldsm4(ka[i], kt + (j * kTile + row) * 128 + (((2 * i + (m >> 1)) ^ (row & 7)) << 4));
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
          float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int part = F32Q ? 1 : 0; part >= 0; part--) {  // the small parts first
            const uint32_t at = qa + (part * TQ + n * 8) * QLD + 128 * j;
            const uint4 q0 = lds128(at), q1 = lds128(at + 16);
            mma16816(x, ka[0][0], ka[0][1], ka[0][2], ka[0][3], q0.x, q0.y);
            mma16816(x, ka[1][0], ka[1][1], ka[1][2], ka[1][3], q0.z, q0.w);
            mma16816(x, ka[2][0], ka[2][1], ka[2][2], ka[2][3], q1.x, q1.y);
            mma16816(x, ka[3][0], ka[3][1], ka[3][2], ka[3][3], q1.z, q1.w);
          }
#pragma unroll
          for (int c = 0; c < 4; c++) sa[n][c] += x[c];
        }
      }
      // ------------------------------------- scores, masks, tile maxima
      const int ta = t0 + 16 * warp + g;
      const float k0 = sc[16 * warp + g], k1 = sc[16 * warp + g + 8];
      const bool whole = sp.whole(t0, kTile);
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int q = n * 8 + 2 * t + e;
          const float f = cq[q];
          float s0 = sa[n][e] * (k0 * f), s1 = sa[n][2 + e] * (k1 * f);
          if (!whole) {
            const int rp = rpos[q];
            if (!sp.sees(rp, ta)) s0 = -INFINITY;
            if (!sp.sees(rp, ta + 8)) s1 = -INFINITY;
          }
          sa[n][e] = s0;
          sa[n][2 + e] = s1;
          float m = fmaxf(s0, s1);
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
          if (lane < 4) mx[warp * TQ + q] = m;
        }
      // Exponent above the tile's value scales, and in a masked tile above those
      // that a row sees: a hidden token's would take bits of the row's weights.
      uint32_t vb = 0;
      if (lane < 16 && t0 + 16 * warp + lane < sp.tokens) vb = __float_as_uint(sc[64 + 16 * warp + lane]);
      if (vb >= 0x7f800000u) vb = 0;  // a NaN scale's rows are NaN whatever the exponent
      vb = __reduce_max_sync(0xffffffffu, vb);
      if (lane == 0) evw[warp] = max((int)(vb >> 23), 1) - 126;
      if (!whole) {
        uint32_t e0 = __float_as_uint(sc[64 + 16 * warp + g]) >> 23, e1 = __float_as_uint(sc[64 + 16 * warp + g + 8]) >> 23;
        if (e0 >= 255) e0 = 0;
        if (e1 >= 255) e1 = 0;
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const int q = n * 8 + 2 * t;
          uint32_t x = 0;  // the two rows' in halves of a word
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const int rp = rpos[q + e];
            x |= max(sp.sees(rp, ta) ? e0 : 0, sp.sees(rp, ta + 8) ? e1 : 0) << (16 * e);
          }
          x = __vmaxu2(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = __vmaxu2(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = __vmaxu2(x, __shfl_xor_sync(0xffffffffu, x, 16));
          if (lane < 4) {
            evr[warp * TQ + q] = max((int)(x & 0xffff), 1) - 126;
            evr[warp * TQ + q + 1] = max((int)(x >> 16), 1) - 126;
          }
        }
      }
    }
    if (consumers_any(!ok)) {
      failed = true;
      break;
    }
    // -------------------------------------------------- weights and sums
    const int evt = max(max(evw[0], evw[1]), max(evw[2], evw[3]));
    const float b0 = sc[64 + 16 * warp + g], b1 = sc[64 + 16 * warp + g + 8];
    const bool whole = sp.whole(t0, kTile), own = !(whole && one);
    auto shrink_of = [](int from, int to) { return from - to < -126 ? 0.f : pow2i(from - to); };
    float shrink = 0.f, up = 0.f;  // of all rows
    if (own) {
      if (threadIdx.x < TQ) {
        const int r = threadIdx.x, from = one ? evu : 14 - ((__float_as_int(esc[r].y) >> 23) - 127);
        const int to = max(from, whole ? evt : max(max(evr[r], evr[TQ + r]), max(evr[2 * TQ + r], evr[3 * TQ + r])));
        esc[r] = make_float2(shrink_of(from, to), pow2i(14 - to));
      }
      consumers_sync();
      one = whole && evt >= evu;
      evu = max(evu, evt);
    } else {
      const int to = max(evu, evt);
      shrink = shrink_of(evu, to);
      up = pow2i(14 - to);
      evu = to;
    }
    float fo[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      float w[4];
      float4 f = make_float4(shrink, up, shrink, up);
      if (own) f = *reinterpret_cast<const float4*>(esc + n * 8 + 2 * t);  // of both rows
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int q = n * 8 + 2 * t + e;
        const float m = fmaxf(fmaxf(mrow[n][e], fmaxf(mx[q], mx[TQ + q])), fmaxf(mx[2 * TQ + q], mx[3 * TQ + q]));
        const float ms = m == -INFINITY ? 0.f : m;
        const float alpha = ex2(mrow[n][e] - ms);
        mrow[n][e] = m;
        const float p0 = ex2(sa[n][e] - ms), p1 = ex2(sa[n][2 + e] - ms);
        l[n][e] = l[n][e] * alpha + (p0 + p1);
        fo[n][e] = alpha * (e ? f.z : f.x);
        // a hidden token weighs zero whatever its scale is
        w[e] = sa[n][e] == -INFINITY ? 0.f : p0 * (b0 * (e ? f.w : f.y));
        w[2 + e] = sa[n][2 + e] == -INFINITY ? 0.f : p1 * (b1 * (e ? f.w : f.y));
      }
      const uint32_t h0 = pack2(w[0], w[1]), h1 = pack2(w[2], w[3]);
      ps[(n * 4 + warp) * 32 + lane] = make_uint2(transpose8(h0), transpose8(h1));
      if constexpr (F32Q) {
        const float2 f0 = unpack2(h0), f1 = unpack2(h1);
        ps[((NT + n) * 4 + warp) * 32 + lane] =
            make_uint2(transpose8(pack2(w[0] - f0.x, w[1] - f0.y)), transpose8(pack2(w[2] - f1.x, w[3] - f1.y)));
      }
    }
    consumers_sync();
    // --------------------------------------------------- O^T += V^T P^T
    if (sums) {
#pragma unroll
      for (int b = 0; b < kMine; b++) {
        const int blk = warp * kMine + b;
        float x[2][NT][4];
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int c = 0; c < 4; c++) x[m][n][c] = 0.f;
#pragma unroll
        for (int kk = 0; kk < 4; kk++) {
          uint32_t va[2][4];
          if constexpr (FMT == kKvI8) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const int tok = 16 * kk + 2 * t + (i & 1) + 8 * (i >> 1);
              w[i] = lds32(vt + tok * HD + (((2 * blk + (g >> 2)) ^ i8_swizzle(tok, HD)) << 4) + ((4 * g) & 15));
            }
            // bytes of two tokens side by side, element by element
            const uint2 x0 = biased4_to_f16(__byte_perm(w[0], w[1], 0x5140)),
                        x1 = biased4_to_f16(__byte_perm(w[0], w[1], 0x7362)),
                        y0 = biased4_to_f16(__byte_perm(w[2], w[3], 0x5140)),
                        y1 = biased4_to_f16(__byte_perm(w[2], w[3], 0x7362));
            va[0][0] = x0.x, va[0][1] = x0.y, va[0][2] = y0.x, va[0][3] = y0.y;
            va[1][0] = x1.x, va[1][1] = x1.y, va[1][2] = y1.x, va[1][3] = y1.y;
          } else {
            const int m = lane >> 3, tok = 16 * kk + (lane & 7) + (m >> 1) * 8;
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
              const int c = blk * 4 + mt * 2 + (m & 1);
              ldsm4t(va[mt], vt + ((c >> 3) * kTile + tok) * 128 + (((c & 7) ^ (tok & 7)) << 4));
            }
          }
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int part = F32Q ? 1 : 0; part >= 0; part--) {
              const uint2 w = ps[((part * NT + n) * 4 + kk) * 32 + lane];
#pragma unroll
              for (int mt = 0; mt < 2; mt++) mma16816(x[mt][n], va[mt][0], va[mt][1], va[mt][2], va[mt][3], w.x, w.y);
            }
        }
        // The tensor cores cut a sum off (2^-25 of it a step on average, always
        // towards zero); a tile's sums are added to the rest by rounding
        // additions, so that no cut accumulates over the tokens.
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int c = 0; c < 4; c++) o[b][m][n][c] = fmaf(o[b][m][n][c], fo[n][c & 1], x[m][n][c]);
      }
    }
    __syncwarp();
    if (lane == 0) bar_arrive(&empty[s]);
  }
  if (failed) {
    if (threadIdx.x == 0) atomicOr(p.flag, kKvTimeout);
    return;
  }
  // ------------------------------------------------------------- results
  consumers_sync();  // mx and esc are read no more
  if (threadIdx.x < TQ) esc[threadIdx.x].x = one ? pow2i(evu) : __fdiv_rn(16384.f, esc[threadIdx.x].y);
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      float v = l[n][e];
      v += __shfl_xor_sync(0xffffffffu, v, 4);
      v += __shfl_xor_sync(0xffffffffu, v, 8);
      v += __shfl_xor_sync(0xffffffffu, v, 16);
      if (lane < 4) mx[warp * TQ + n * 8 + 2 * t + e] = v;
    }
  consumers_sync();
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int q = n * 8 + 2 * t + e, rr = tr.r0 + q;
      if (rr >= tr.nr) continue;
      const float sum = (mx[q] + mx[TQ + q]) + (mx[2 * TQ + q] + mx[3 * TQ + q]);
      const int row = tr.row0 + rr / group, h = kvh * group + rr % group;
      const int64_t rh = (int64_t)row * a.heads + h;
      const float back = esc[q].x;
      const float f = a.slots > 1 ? 0x1p-14f : sum != 0.f ? __fdiv_rn(0x1p-14f, sum) : 0.f;
      if (a.slots > 1 && warp == 0 && g == 0) a.ml[rh * a.slots + slot] = make_float2(mrow[n][e], sum);
      if (!sums) continue;
#pragma unroll
      for (int b = 0; b < kMine; b++) {
        const int blk = warp * kMine + b;
        // i8: elements 4g .. 4g+3 of the block; f16: g, g+8, g+16, g+24
        // (back last: before the division by the sum a value near f32's end would pass it)
        const float x[4] = {o[b][0][n][e] * f * back, o[b][0][n][2 + e] * f * back, o[b][1][n][e] * f * back,
                            o[b][1][n][2 + e] * f * back};
        auto put = [&](auto* dst, bool v4) {
          using T = std::remove_reference_t<decltype(*dst)>;
          if constexpr (FMT == kKvI8) {
            store_n<T, 4>(dst + blk * 32 + 4 * g, v4, x);
          } else {
#pragma unroll
            for (int c = 0; c < 4; c++) dst[blk * 32 + g + 8 * c] = from_f<T>(x[c]);
          }
        };
        if (a.slots > 1) {
          put(a.part + (rh * a.slots + slot) * HD, true);
        } else {
          const int64_t at = (int64_t)row * a.out.row + (int64_t)h * a.out.head;
          if constexpr (F32Q) put(static_cast<float*>(a.out.p) + at, vec);
          else if (a.dtype == F16) put(static_cast<__half*>(a.out.p) + at, vec);
          else put(static_cast<__nv_bfloat16*>(a.out.p) + at, vec);
        }
      }
    }
}

// A row's splits joined: out = sum_c 2^(m_c - M) o_c / sum_c 2^(m_c - M) l_c
// over the chunks c that the row sees.  Chunk c belongs to group c mod 8; a
// group's chunks are summed in order, then the groups in order, whichever
// kernel does it: the result depends on the row's own chunks only.
constexpr int kGroups = 8;

struct JoinRow {
  KvChunks ch;
  KvRowChunks rc;
  int64_t rh;
};
// False for a row behind the last sequence.  Warp-wide.
__device__ __forceinline__ bool join_row(const KvAttnArgs& a, int row, int h, int tq, int lane, JoinRow* j) {
  const KvSeq q = kv_seq_of_row(a.b, row, lane);
  if (q.seq < 0) return false;
  const int group = a.heads / a.pool.nkv;
  const int tile0 = (q.in_seq * group + h % group) / tq * tq;  // the row's tile begins here
  j->ch = kv_chunks(a, q.pos + tile0 / group);
  j->rc = kv_row_chunks(a, j->ch, q.pos + q.in_seq);
  j->rh = (int64_t)row * a.heads + h;
  return true;
}
// Chunks [b, e) are a run of one of the row's two lists (first tokens, window).
struct JoinRun {
  int b, e;
};
__device__ __forceinline__ JoinRun join_run(const JoinRow& j, int r) {
  if (r == 0) return {0, j.rc.firsts};
  return {j.rc.window0, j.rc.window0 + j.rc.count - j.rc.firsts};
}

// Up to eight slots: one warp per (row, head).  A group has at most one chunk
// of either list then, so groups are summed as they come, the loads of four of
// them in flight.
template <class T, int HD>
__global__ void __launch_bounds__(128) kv_join_few_kernel(const __grid_constant__ KvAttnArgs a, const int tq,
                                                          const bool vec) {
  constexpr int N = HD / 32;
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const uint32_t item = blockIdx.x * 4 + (threadIdx.x >> 5);  // (rows x heads below 2^31)
  const int row = (int)(item / (uint32_t)a.heads), h = (int)(item - (uint32_t)row * a.heads);
  if (row >= a.b.rows) return;
  JoinRow j;
  if (!join_row(a, row, h, tq, lane, &j)) return;
  const float2* ml = a.ml + j.rh * a.slots;
  const float* part = a.part + j.rh * a.slots * HD + lane * N;
  const float2 mine = lane < j.rc.count ? ml[j.ch.slot(j.rc.chunk(lane))] : make_float2(-INFINITY, 0.f);
  float M = mine.x;
#pragma unroll
  for (int w = 4; w; w >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, w));
  M = __shfl_sync(0xffffffffu, M, 0);
  const float wt = kvp::ex2(mine.x - (M == -INFINITY ? 0.f : M));
  float o[N], sum = 0.f;
#pragma unroll
  for (int k = 0; k < N; k++) o[k] = 0.f;
  const JoinRun first = join_run(j, 0), second = join_run(j, 1);
  const int at = j.rc.firsts - second.b;  // a chunk's place among the row's
#pragma unroll 4
  for (int g = 0; g < kGroups; g++) {
    const int c0 = first.b + ((g - first.b) & (kGroups - 1)), c1 = second.b + ((g - second.b) & (kGroups - 1));
    const bool in0 = c0 < first.e, in1 = c1 < second.e;
    const float w0 = __shfl_sync(0xffffffffu, wt, c0 & 31), l0 = __shfl_sync(0xffffffffu, mine.y, c0 & 31);
    const float w1 = __shfl_sync(0xffffffffu, wt, (c1 + at) & 31), l1 = __shfl_sync(0xffffffffu, mine.y, (c1 + at) & 31);
    float t[N], x[N], s = 0.f;
#pragma unroll
    for (int k = 0; k < N; k++) t[k] = 0.f;
    if (in0) {
      load_n<float, N>(part + (int64_t)j.ch.slot(c0) * HD, true, x);
#pragma unroll
      for (int k = 0; k < N; k++) t[k] = fmaf(w0, x[k], t[k]);
      s = fmaf(w0, l0, s);
    }
    if (in1) {
      load_n<float, N>(part + (int64_t)j.ch.slot(c1) * HD, true, x);
#pragma unroll
      for (int k = 0; k < N; k++) t[k] = fmaf(w1, x[k], t[k]);
      s = fmaf(w1, l1, s);
    }
#pragma unroll
    for (int k = 0; k < N; k++) o[k] += t[k];
    sum += s;
  }
  const float f = sum != 0.f ? __fdiv_rn(1.f, sum) : 0.f;
#pragma unroll
  for (int k = 0; k < N; k++) o[k] *= f;
  store_n<T, N>(static_cast<T*>(a.out.p) + (int64_t)row * a.out.row + (int64_t)h * a.out.head + lane * N, vec, o);
}

// One CTA per (row, head), a warp per group, any number of slots.
template <class T, int HD>
__global__ void __launch_bounds__(256) kv_join_kernel(const __grid_constant__ KvAttnArgs a, const int tq,
                                                      const bool vec) {
  constexpr int N = HD / 32, kWeights = 1024, U = 8;
  __shared__ float2 wt[kWeights];  // {weight, sum}
  __shared__ float red[8], sums[kGroups], os[kGroups][HD];
  pdl_wait();
  const int row = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
  JoinRow j;
  if (!join_row(a, row, h, tq, lane, &j)) return;
  const float2* ml = a.ml + j.rh * a.slots;
  const float* part = a.part + j.rh * a.slots * HD + lane * N;
  float mxv = -INFINITY;
  float2 held[kWeights / 256];
#pragma unroll
  for (int i = 0; i < kWeights / 256; i++) {
    const int c = threadIdx.x + 256 * i;
    held[i] = c < j.rc.count ? ml[j.ch.slot(j.rc.chunk(c))] : make_float2(-INFINITY, 0.f);
    mxv = fmaxf(mxv, held[i].x);
  }
  for (int c = kWeights + threadIdx.x; c < j.rc.count; c += 256) mxv = fmaxf(mxv, ml[j.ch.slot(j.rc.chunk(c))].x);
#pragma unroll
  for (int w = 16; w; w >>= 1) mxv = fmaxf(mxv, __shfl_xor_sync(0xffffffffu, mxv, w));
  if (lane == 0) red[grp] = mxv;
  __syncthreads();
  float M = red[0];
#pragma unroll
  for (int w = 1; w < 8; w++) M = fmaxf(M, red[w]);
  const float ms = M == -INFINITY ? 0.f : M;
  float acc[N], sum = 0.f;
#pragma unroll
  for (int k = 0; k < N; k++) acc[k] = 0.f;
  for (int p0 = 0; p0 < j.rc.count; p0 += kWeights) {  // places p0 .. p0 + 1023 of the row's chunks
    const int p1 = min(p0 + kWeights, j.rc.count);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWeights / 256; i++) {
      const int c = p0 + threadIdx.x + 256 * i;
      if (c >= p1) continue;
      const float2 v = p0 ? ml[j.ch.slot(j.rc.chunk(c))] : held[i];
      wt[c - p0] = make_float2(kvp::ex2(v.x - ms), v.y);
    }
    __syncthreads();
    for (int r = 0; r < 2; r++) {
      JoinRun run = join_run(j, r);
      const int at = (r ? j.rc.firsts : 0) - run.b;
      run.b = max(run.b, p0 - at);
      run.e = min(run.e, p1 - at);
      // the group's chunks of the run, eight loads in flight
      for (int c0 = run.b + ((grp - run.b) & (kGroups - 1)); c0 < run.e; c0 += U * kGroups) {
        float x[U][N];
#pragma unroll
        for (int u = 0; u < U; u++)
          if (c0 + u * kGroups < run.e) load_n<float, N>(part + (int64_t)j.ch.slot(c0 + u * kGroups) * HD, true, x[u]);
#pragma unroll
        for (int u = 0; u < U; u++) {
          if (c0 + u * kGroups >= run.e) continue;
          const float2 w = wt[c0 + u * kGroups + at - p0];
#pragma unroll
          for (int k = 0; k < N; k++) acc[k] = fmaf(w.x, x[u][k], acc[k]);
          sum = fmaf(w.x, w.y, sum);
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < N; k++) os[grp][lane * N + k] = acc[k];
  if (lane == 0) sums[grp] = sum;
  __syncthreads();
  if (grp) return;
  sum = 0.f;
#pragma unroll
  for (int k = 0; k < N; k++) acc[k] = 0.f;
  for (int g = 0; g < kGroups; g++) {
#pragma unroll
    for (int k = 0; k < N; k++) acc[k] += os[g][lane * N + k];
    sum += sums[g];
  }
  const float f = sum != 0.f ? __fdiv_rn(1.f, sum) : 0.f;
#pragma unroll
  for (int k = 0; k < N; k++) acc[k] *= f;
  store_n<T, N>(static_cast<T*>(a.out.p) + (int64_t)row * a.out.row + (int64_t)h * a.out.head + lane * N, vec, acc);
}

template <int HD, int FMT, int NT, bool F32Q>
cudaError_t launch_split(const KvAttnArgs& a, int64_t ctas, bool vec, cudaStream_t st) {
  using G_ = Geo<HD, FMT, NT, F32Q>;
  static bool configured[64] = {};
  static std::mutex mu;
  const cudaError_t e = once_per_device(configured, mu, [] {
    return cudaFuncSetAttribute(kv_attend_kernel<HD, FMT, NT, F32Q>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                G_::kSmem);
  });
  if (e != cudaSuccess) return e;
  kv_attend_kernel<HD, FMT, NT, F32Q><<<(unsigned)ctas, 160, G_::kSmem, st>>>(a, vec);
  return cudaGetLastError();
}

bool strides_ok(const KvTensor& t, int item, int bytes) {
  return ((uintptr_t)t.p | (uintptr_t)(t.row * item) | (uintptr_t)(t.head * item)) % bytes == 0;
}

template <class T, int HD>
cudaError_t launch_join(const KvAttnArgs& a, int tq, cudaStream_t st) {
  const int64_t items = (int64_t)a.b.rows * a.heads;
  const bool vec = strides_ok(a.out, sizeof(T), 16);
  if (a.slots <= kGroups)
    return launch_pdl(kv_join_few_kernel<T, HD>, dim3((unsigned)ceil_div(items, 4)), dim3(128), 0, st, true, a, tq, vec);
  return launch_pdl(kv_join_kernel<T, HD>, dim3((unsigned)items), dim3(256), 0, st, true, a, tq, vec);
}

}  // namespace

size_t kv_attend_plan(KvAttnArgs& a, int max_rows) { return kv_plan(a, max_rows); }

void kv_attend_bind(KvAttnArgs& a, void* workspace) {
  if (a.slots == 1) return;
  a.part = static_cast<float*>(workspace);
  a.ml = reinterpret_cast<float2*>(a.part + (int64_t)a.b.rows * a.heads * a.slots * a.pool.hd);
}

cudaError_t kv_attend_launch(const KvAttnArgs& args, cudaStream_t st) {
  KvAttnArgs a = args;
  // tests only, looked up at every launch: a copy that never comes, and waits of
  // a millisecond for it (every copy that is requested lands long before)
  a.test_skip = getenv("IQ_KV_TEST_TIMEOUT") != nullptr;
  a.wait_limit = a.test_skip ? 1 << 9 : kWaitLimit;
  const int tq = a.tq;
  const int64_t ctas = kv_tiles_bound(a, tq) * a.pool.nkv * a.slots;
  if (ctas >= (1ll << 31)) return cudaErrorInvalidValue;
  const int item = a.dtype == F32 ? 4 : 2;
  // one flag for reading queries (hd / 32 elements a lane) and writing four
  // elements: both are whole words of up to 16 bytes
  const bool vec = strides_ok(a.q, item, 16) && strides_ok(a.out, item, 16);
  auto by_rows = [&](auto hd, auto fmt, auto f32) {
    constexpr int HD = decltype(hd)::value, FMT = decltype(fmt)::value;
    constexpr bool F = decltype(f32)::value;
    switch (tq) {
      case 8: return launch_split<HD, FMT, 1, F>(a, ctas, vec, st);
      case 16: return launch_split<HD, FMT, 2, F>(a, ctas, vec, st);
      case 32: return launch_split<HD, FMT, 4, F>(a, ctas, vec, st);
      default: return launch_split<HD, FMT, 8, F>(a, ctas, vec, st);
    }
  };
  auto by_type = [&](auto hd, auto fmt) {
    return a.dtype == F32 ? by_rows(hd, fmt, std::true_type()) : by_rows(hd, fmt, std::false_type());
  };
  auto by_format = [&](auto hd) {
    return a.pool.format == kKvI8 ? by_type(hd, std::integral_constant<int, kKvI8>())
                                  : by_type(hd, std::integral_constant<int, kKvF16>());
  };
  auto join = [&](auto hd) {
    constexpr int HD = decltype(hd)::value;
    return a.dtype == F32   ? launch_join<float, HD>(a, tq, st)
           : a.dtype == F16 ? launch_join<__half, HD>(a, tq, st)
                            : launch_join<__nv_bfloat16, HD>(a, tq, st);
  };
  auto go = [&](auto hd) {
    const cudaError_t e = tq > 64 ? kv_attend_wide_launch(a, ctas, vec, st) : by_format(hd);
    return e != cudaSuccess || a.slots == 1 ? e : join(hd);
  };
  switch (a.pool.hd) {
    case 64: return go(std::integral_constant<int, 64>());
    case 128: return go(std::integral_constant<int, 128>());
    case 256: return go(std::integral_constant<int, 256>());
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace iq
