// kv_split.cuh -- which query rows a CTA takes, which tokens they see, and
// how the tokens are split into chunks.  The attention kernels and the join
// of their partial results go by the same functions.
//
// Chunk c holds the positions [c * chunk, (c + 1) * chunk) of a sequence.  A
// tile of query rows at positions pa..pb has partial results for the slots
// 0 .. slots - 1: the chunks of the always-visible first tokens, then those
// from the first token that the row at pa sees.
#pragma once
#include <algorithm>
#include "kv_device.cuh"

namespace iq {

__host__ __device__ inline int64_t kv_min(int64_t a, int64_t b) { return a < b ? a : b; }
__host__ __device__ inline int64_t kv_max(int64_t a, int64_t b) { return a > b ? a : b; }

// A position inside 0 .. 2^31 - 1 (divisions stay in 32 bits).
__host__ __device__ inline int kv_clip(int64_t a) { return (int)kv_min(kv_max(a, 0), 0x7fffffff); }

struct KvTileRows {
  int seq, row0;  // the sequence and its first row
  int r0, nr;     // first query row of the tile and query rows (row x head of the KV head) of the sequence
  int64_t pos;    // position of the sequence's first row
};

// Tile `tile` of `tq` query rows, counted through the sequences; false when
// the batch has fewer.  Warp-wide; every lane gets the result.
__device__ __forceinline__ bool kv_tile_rows(const KvBatch& b, int tile, int tq, int group, int lane, KvTileRows* t) {
  int n;
  if (!b.row_start) {
    t->seq = t->row0 = 0;
    n = b.rows;
    t->r0 = tile * tq;
    t->pos = b.position[0];
  } else if (group % tq == 0) {  // no tile crosses a row: no sum over sequences
    const int per = group / tq, row = tile / per;
    if (row >= b.rows) return false;
    const KvSeq q = kv_seq_of_row(b, row, lane);
    if (q.seq < 0) return false;
    t->seq = q.seq;
    t->row0 = row - q.in_seq;
    t->pos = q.pos;
    n = q.rows;
    t->r0 = q.in_seq * group + tile % per * tq;
  } else {
    int before = 0;  // tiles of the sequences up to s0
    t->seq = -1;
    for (int s0 = 0; s0 < b.seqs; s0 += 32) {
      const int s = min(s0 + lane, b.seqs - 1);
      const int begin = kv_row(b, b.row_start[s]), end = kv_row(b, b.row_start[s + 1]), pos = b.position[s];
      const int rows = s0 + lane < b.seqs ? max(end - begin, 0) : 0;
      const int tiles = (int)(((int64_t)rows * group + tq - 1) / tq);
      int sum = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += x;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, before + sum > tile);
      if (past) {
        const int at = __ffs(past) - 1;
        t->seq = s0 + at;
        t->r0 = (tile - before - __shfl_sync(0xffffffffu, sum - tiles, at)) * tq;
        t->row0 = __shfl_sync(0xffffffffu, begin, at);
        t->pos = __shfl_sync(0xffffffffu, pos, at);
        n = __shfl_sync(0xffffffffu, rows, at);
        break;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (t->seq < 0) return false;
  }
  if (t->r0 < 0) return false;  // (a row_start so wrong that the tiles' number overflows)
  t->nr = min(n, b.rows - t->row0) * group;
  return t->r0 < t->nr;
}

struct KvChunks {
  int first_chunks;  // chunks of the always-visible first tokens
  int window0;       // first chunk of the window part
  __host__ __device__ int slot(int c) const { return c < first_chunks ? c : first_chunks + c - window0; }
  __host__ __device__ int chunk(int s) const { return s < first_chunks ? s : window0 + s - first_chunks; }
};
// pa: position of the tile's first row.
__host__ __device__ inline KvChunks kv_chunks(const KvAttnArgs& a, int64_t pa) {
  KvChunks c = {0, 0};
  if (a.window) {
    c.first_chunks = a.sinks ? (a.sinks - 1) / a.chunk + 1 : 0;  // (no sum that passes 31 bits)
    c.window0 = (int)kv_max(c.first_chunks, kv_clip(pa - a.window + 1) / a.chunk);
  }
  return c;
}

// The chunks that hold a visible token of the row at `pos`, ascending.
struct KvRowChunks {
  int firsts, window0, count;
  __host__ __device__ int chunk(int j) const { return j < firsts ? j : window0 + j - firsts; }
};
__host__ __device__ inline KvRowChunks kv_row_chunks(const KvAttnArgs& a, const KvChunks& ch, int64_t pos) {
  const int64_t cap = (int64_t)a.b.table_cols << a.pool.page_shift;
  const int64_t top = kv_min(pos, cap - 1);
  if (top < 0) return {0, 0, 0};
  KvRowChunks r;
  const int last = kv_clip(top) / a.chunk;
  r.firsts = (int)kv_min(ch.first_chunks, last + 1);
  r.window0 = a.window ? (int)kv_max(ch.first_chunks, kv_clip(pos - a.window + 1) / a.chunk) : 0;
  r.count = r.firsts + (int)kv_max(last - r.window0 + 1, 0);
  return r;
}

// The tokens of one chunk that a tile of rows sees, in tiles of 64.
struct KvSpan {
  int first, end;       // tiles first, next(first), ... below end
  int tokens;           // tokens up to the last row's, as far as the table reaches
  int pa, pb;           // first and last row's position
  int window, sinks;
  bool outside;         // a row stands behind the table
  __host__ __device__ int skip(int ti) const {
    if (window && ti * 64 >= sinks && ti * 64 + 63 <= pa - window) return (pa - window + 1) >> 6;
    return ti;
  }
  __host__ __device__ int next(int ti) const { return skip(ti + 1); }
  // Whether every row sees all tokens [t0, t0 + n).
  __host__ __device__ bool whole(int t0, int n) const {
    return t0 + n - 1 <= pa && t0 + n <= tokens && (!window || t0 > pb - window || t0 + n <= sinks);
  }
  // Whether the row at position rp (-1: none) sees token t.
  __host__ __device__ bool sees(int rp, int t) const {
    return t <= rp && t < tokens && (!window || t > rp - window || t < sinks);
  }
};
__host__ __device__ inline KvSpan kv_span(const KvAttnArgs& a, const KvTileRows& t, int tq, int slot) {
  const int group = a.heads / a.pool.nkv;
  const int64_t cap = (int64_t)a.b.table_cols << a.pool.page_shift;
  const int64_t pa = t.pos + t.r0 / group, pb = t.pos + ((int)kv_min(t.r0 + tq, t.nr) - 1) / group;
  const int64_t top = (1ll << 31) - 1;
  KvSpan s;
  s.pa = (int)kv_max(kv_min(pa, top), -1);  // (any negative position is padding; less a window it stays in 32 bits)
  s.pb = (int)kv_max(kv_min(pb, top), -1);
  s.outside = pb >= cap;
  s.tokens = (int)kv_max(kv_min(pb + 1, cap), 0);
  s.window = a.window;
  s.sinks = a.sinks;
  const int64_t c0 = (int64_t)kv_chunks(a, pa).chunk(slot) * a.chunk;
  const int64_t c1 = kv_min(c0 + a.chunk, s.tokens);
  s.first = s.skip((int)kv_min(c0 >> 6, 1 << 26));
  s.end = (int)((c1 + 63) >> 6);
  return s;
}

// ------------------------------------------------------------ host side
constexpr int kKvTile = 64;  // tokens a tile

// Shared memory of the split kernel (kv_attend.cu): 8 nt query rows, tiles of
// 64 tokens, two to four stages; three CTAs an SM where two stages and the rest
// take a third of it, else two, else one.
struct KvNarrow {
  int fixed, stages, smem, ctas;
};
constexpr KvNarrow kv_narrow(int format, int hd, int nt, bool f32) {
  const int tile = kKvTile * hd * (format == kKvI8 ? 1 : 2), per = 2 * tile + 512, parts = f32 ? 2 : 1;
  KvNarrow g = {};
  g.fixed = 8 * nt * (hd * 2 + 16) * parts + nt * 1024 * parts + 12 * 8 * nt * 4 + 64;
  const int limit = 2 * tile > 32768 ? 226 : g.fixed <= 10 * 1024 ? 78 : g.fixed <= 48 * 1024 ? 112 : 226;
  const int room = limit * 1024 - 2048 - g.fixed;
  g.stages = room / per > 4 ? 4 : room / per;
  g.smem = g.stages * per + g.fixed + 1024;
  g.ctas = (227 * 1024) / (g.smem + 1280);  // (static shared memory and 1 KB a CTA)
  return g;
}

// Query rows of a tile: the fewest of 8, 16, 32, 64 that take a sequence's
// rows of one KV head at once, or the tensor-core kernel's 128: above 64 rows
// unless the call keeps to the other, and above 16 where the split is free
// too.  us for f32 and bf16 rows, i8, tiles of 128 and of up to 64 (as few as
// take a sequence's rows):
//   8 heads of 256  16 x 4 rows over 4127    69, 57     85, 74
//                   16 x 8 over 4127         71, 59    180, 161
//                   16 x 8 over 700          24, 22     42, 36
//                   1 x 4 over 4096          22, 20     20, 18
//                   1 x 8 over 32768         33, 28     72, 58
//   4 of 128        16 x 8 over 4127        159, 104   196, 160
//                   1 x 8 over 32768         74, 48     83, 70
//   4 of 64         16 x 8 over 4127         47, 45     50, 47
//                   64 x 8 over 2000         81, 60     75, 66
// One short sequence, and many of small heads in f32, would take the smaller
// tiles by a tenth.
inline int kv_tile_query_rows(const KvAttnArgs& a, int max_rows) {
  const int64_t r = (int64_t)(max_rows ? std::min(max_rows, a.b.rows) : a.b.rows) * (a.heads / a.pool.nkv);
  if (!a.narrow && r > (a.chunk ? 64 : 16)) return 128;
  return r <= 8 ? 8 : r <= 16 ? 16 : r <= 32 ? 32 : 64;
}
inline int64_t kv_tiles_bound(const KvAttnArgs& a, int tq) {
  const int64_t r = (int64_t)a.b.rows * (a.heads / a.pool.nkv);
  if (!a.b.row_start) return ceil_div(r, tq);
  if ((a.heads / a.pool.nkv) % tq == 0) return r / tq;
  return r / tq + std::min(a.b.seqs, a.b.rows);
}

// The most tokens that one accumulator of the tensor-core kernel sums, for the
// cuts that its steps make (kv_attend_wide.cu).  f32 rows over 640 tokens:
// 4.0e-6 where equal values add up, 2.0e-6 of the outputs' size for values of
// both signs (over 1536: 1.0e-5 and 4.0e-6; 32-bit torch operations 1.4e-6);
// 512 of them over 2560 tokens take 78 us instead of 63, 2048 over 32768 3300
// instead of 2584.  16-bit rows over 16384 tokens: 5.5e-5, an eighth of f16's
// half step; 2048 over 131072 i8 tokens 5690 us instead of 5470.
constexpr int kWideChunkF32 = 640, kWideChunk = 16384;

// Fills tq, chunk (where it is 0) and slots; the workspace bytes.
inline size_t kv_plan(KvAttnArgs& a, int max_rows) {
  const int group = a.heads / a.pool.nkv, tq = kv_tile_query_rows(a, max_rows);
  a.tq = tq;
  const int64_t cap = (int64_t)a.b.table_cols * a.pool.page_tokens;
  // what reaches past the table says no more than the table's end
  const int end = (int)align_up(cap + 1, kKvTile);
  a.window = std::min(a.window, end);
  a.sinks = std::min(a.sinks, end);
  a.chunk = std::min(a.chunk, end);
  const int tile_tokens = (tq - 1) / group + 1;
  const int64_t span = a.window ? std::min<int64_t>(cap, (int64_t)a.window + a.sinks + tile_tokens + kKvTile) : cap;
  // what one accumulator may sum; a window's rows see no more than `span` tokens of any chunk
  const int64_t limit = tq != 128 ? span : a.dtype == F32 ? kWideChunkF32 : kWideChunk;
  if (!a.chunk) {
    // The split n with the least estimated time, in us: CTAs run in waves of
    // `ctas` an SM; a wave costs its tiles, at the SM's share of what bounds
    // them, and a start and an end that nothing hides; n > 1 adds partial
    // results that cross HBM twice and the join.  Tiles: the cache's bytes at
    // 44 KB a us and SM; in the split kernel at least 0.4 us for 8 rows (twice
    // that for f32 rows) at hd 256, in the tensor-core kernel 1.1 us (1.8).
    // Several sequences are taken to be of mixed lengths, two thirds of the
    // table on average: an SM that got long ones only sets the time (64 bf16
    // sequences of up to 8209 tokens, i8, hd 256: chunks of 8256 take 144 us,
    // of 4160 101, of 2048 70, of 1024 79, of 256 93, of 128 118; the rule's
    // 1408 takes 87, and 64 sequences of 6000 tokens 79 of at best 72).
    const bool wide = tq == 128, f32 = a.dtype == F32;
    const int elt = a.pool.format == kKvI8 ? 1 : 2;
    const double read = (2.0 * kKvTile * a.pool.hd * elt + 512) / 43.9e3;
    const double work = (wide ? 0.7 * (f32 ? 2 : 1) * a.pool.hd / 256 + 0.4
                              : 0.4 * (tq / 8) * (f32 ? 2 : 1) * a.pool.hd / 256);
    const double tile = std::max(read, work), fixed = wide ? 14 : 6;
    const int64_t sms = 148, ctas = wide ? 1 : kv_narrow(a.pool.format, a.pool.hd, tq / 8, f32).ctas;
    // (the tiles there will be, as far as max_rows tells, not the most possible)
    const int64_t rows = max_rows ? std::min(max_rows, a.b.rows) : a.b.rows;
    const int64_t items = std::min(kv_tiles_bound(a, tq), a.b.seqs * ceil_div(rows * group, tq)) * a.pool.nkv;
    const double result = (double)a.b.rows * a.heads * a.pool.hd * 8 / 5e6;
    const int64_t most = std::min<int64_t>(512, std::max<int64_t>(span / (2 * kKvTile), 1));
    double best = 0;
    for (int64_t n = 1; n <= most; n += 1 + n / 16) {
      // (unsplit, a chunk holds all of the table: first tokens and window in one)
      const int64_t chunk = align_up(n == 1 ? std::max<int64_t>(cap, 1) : ceil_div(span, n), kKvTile);
      if (std::min(chunk, span) > limit && n < most) continue;
      const int64_t slots = n == 1 ? 1 : ceil_div(span, chunk) + (a.window && a.sinks ? 1 : 0);
      const int64_t all = items * slots, full = all / (sms * ctas), rest = all % (sms * ctas);
      const double tiles = (double)ceil_div(ceil_div(span, n), kKvTile);
      double cost;
      if (a.b.seqs > 1) {
        cost = std::max(1.0, 0.65 * all / (sms * ctas)) * (tiles * tile * ctas + fixed);
      } else {
        cost = full * (tiles * tile * ctas + fixed);
        if (rest) cost += tiles * std::max(tile * ceil_div(rest, sms), 1.0) + fixed;
      }
      if (n > 1) cost += 3 + slots * result;
      if (!a.chunk || cost < best) best = cost, a.chunk = (int)chunk;
    }
    // (the steps of n may pass over `most`, every split before it too long for one accumulator)
    if (!a.chunk) a.chunk = (int)limit;
  }
  if (span > limit) a.chunk = (int)std::min<int64_t>(a.chunk, limit);
  const int64_t all = std::max<int64_t>(ceil_div(cap, a.chunk), 1);
  a.slots = (int)all;
  if (a.window)
    a.slots = (int)std::min<int64_t>(all, ceil_div(a.sinks, a.chunk) + ((int64_t)a.window + tile_tokens) / a.chunk + 2);
  if (a.slots == 1) return 0;
  const int64_t parts = (int64_t)a.b.rows * a.heads * a.slots;
  return (size_t)(parts * a.pool.hd * 4 + parts * 8);
}

}  // namespace iq
