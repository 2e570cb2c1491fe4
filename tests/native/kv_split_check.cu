// Host check of the paged attention's split (inferq_b200/csrc/kv_split.cuh):
// for one sequence given on the command line, every visible (row, token) is
// met exactly once by the tiles of the chunks that the join reads, nothing
// hidden is, and every slot lies inside the planned ones.
//   kv_split_check heads kv_heads page cols rows position window sinks chunk max_rows
#include <cstdio>
#include <cstdlib>
#include <map>
#include <set>
#include <vector>
#include "kv_split.cuh"

using namespace iq;

int main(int argc, char** argv) {
  if (argc != 11) return 2;
  auto arg = [&](int i) { return atoi(argv[i]); };
  KvAttnArgs a = {};
  a.heads = arg(1);
  a.pool.nkv = arg(2);
  a.pool.hd = 64;
  a.pool.format = kKvI8;
  a.pool.page_tokens = arg(3);
  a.pool.page_shift = __builtin_ctz(arg(3));
  a.b.table_cols = arg(4);
  a.b.rows = arg(5);
  a.b.seqs = 1;
  const int position = arg(6);
  a.window = arg(7);
  a.sinks = a.window ? arg(8) : 0;
  a.chunk = arg(9);
  const size_t need = kv_plan(a, arg(10));
  const int group = a.heads / a.pool.nkv, tq = a.tq;
  const int64_t cap = (int64_t)a.b.table_cols * a.pool.page_tokens;
  if ((need == 0) != (a.slots == 1)) return printf("workspace %zu for %d slots\n", need, a.slots), 1;
  const int tiles = (int)kv_tiles_bound(a, tq);
  for (int tile = 0; tile < tiles; tile++) {
    KvTileRows tr = {0, 0, tile * tq, a.b.rows * group, position};
    if (tr.r0 >= tr.nr) return printf("tile %d has no row\n", tile), 1;
    std::map<int, KvSpan> spans;
    for (int slot = 0; slot < a.slots; slot++) {
      const KvSpan sp = kv_span(a, tr, tq, slot);
      if (sp.first < sp.end || a.slots == 1) spans[slot] = sp;
    }
    const int first = tr.r0, last = (int)kv_min(tr.r0 + tq, tr.nr);
    for (int r = first; r < last; r += 1) {
      const int64_t pos = position + r / group;
      const int rp = pos < 0 ? -1 : (int)pos;
      std::vector<char> met(cap > 0 ? cap : 1, 0);
      std::set<int> slots;
      if (a.slots == 1) {
        slots.insert(0);
      } else {
        const KvChunks ch = kv_chunks(a, position + tr.r0 / group);
        const KvRowChunks rc = kv_row_chunks(a, ch, pos);
        int before = -1;
        for (int j = 0; j < rc.count; j++) {
          const int c = rc.chunk(j), s = ch.slot(c);
          if (c <= before) return printf("chunks do not ascend\n"), 1;
          before = c;
          if (s < 0 || s >= a.slots || ch.chunk(s) != c) return printf("row %d chunk %d slot %d of %d\n", r, c, s, a.slots), 1;
          if (!spans.count(s)) return printf("row %d reads slot %d, which is not written\n", r, s), 1;
          slots.insert(s);
        }
      }
      for (int s : slots) {
        const KvSpan& sp = spans[s];
        int before = -1;
        for (int ti = sp.first; ti < sp.end; ti = sp.next(ti)) {
          if (ti <= before || ti < 0) return printf("tiles do not ascend\n"), 1;
          before = ti;
          if ((int64_t)ti * 64 >= cap) return printf("tile %d begins behind the table\n", ti), 1;
          const bool whole = sp.whole(ti * 64, 64);
          for (int t = ti * 64; t < ti * 64 + 64; t++) {
            const bool sees = sp.sees(rp, t);
            if (whole && !sees) return printf("tile %d is not whole for row %d\n", ti, r), 1;
            if (sees && t >= cap) return printf("token %d behind the table\n", t), 1;
            if (sees && met[t]++) return printf("row %d meets token %d twice\n", r, t), 1;
          }
        }
      }
      for (int64_t t = 0; t < cap; t++) {
        const bool want = t <= pos && (!a.window || t > pos - a.window || t < a.sinks);
        if (want != (bool)met[t]) return printf("row %d token %d: %d\n", r, (int)t, met[t]), 1;
      }
    }
  }
  printf("ok tq %d chunk %d slots %d\n", tq, a.chunk, a.slots);
  return 0;
}
