// Host check of the paged attention's plan (inferq_b200/csrc/kv_split.cuh)
// over tables of up to 2^31 tokens: every call gets a split that is a multiple
// of 64, an accumulator of the tensor-core kernel never sums more than its
// bound, and slots and workspace follow from the split.
#include <cstdio>
#include "kv_split.cuh"

using namespace iq;

int main() {
  const int64_t most = (1ll << 31) - 512;
  long calls = 0;
  for (int dtype : {F32, F16, BF16})
    for (int group : {1, 7, 8, 128})
      for (int page : {16, 256})
        for (int64_t tokens = 0; tokens < most; tokens = tokens < 64 ? tokens + 16 : tokens + tokens / 3 + 16)
          for (int rows : {1, 3, 20, 512})
            for (int seqs : {1, 5})
              for (int window : {0, 1, 1000, 100000, 2147483647})
                for (int sinks : {0, 5, 70000})
                  for (int chunk : {0, 64, 4096, 2147483584}) {
                    KvAttnArgs a = {};
                    a.dtype = dtype;
                    a.pool.nkv = 2;
                    a.heads = 2 * group;
                    a.pool.hd = 256;
                    a.pool.format = kKvI8;
                    a.pool.page_tokens = page;
                    a.pool.page_shift = __builtin_ctz(page);
                    a.b.table_cols = (int)(tokens / page);
                    a.b.rows = rows;
                    a.b.seqs = seqs;
                    a.window = window;
                    a.sinks = window ? sinks : 0;
                    a.chunk = chunk;
                    int32_t starts = 0;
                    a.b.row_start = seqs > 1 ? &starts : nullptr;  // (whether it is there is all that counts)
                    const size_t need = kv_plan(a, rows);
                    calls++;
                    const int64_t cap = (int64_t)a.b.table_cols * page;
                    const int64_t seen = a.window ? kv_min(cap, (int64_t)a.window + a.sinks + (a.tq - 1) / group + 65) : cap;
                    const int64_t limit = dtype == F32 ? kWideChunkF32 : kWideChunk;
                    const size_t part = a.slots == 1 ? 0 : (size_t)rows * a.heads * a.slots * (a.pool.hd * 4 + 8);
                    if (a.chunk <= 0 || a.chunk % 64 || a.slots < 1 || need != part ||
                        (a.slots == 1 && !window && a.chunk < cap) || (a.tq == 128 && kv_min(a.chunk, seen) > limit)) {
                      printf("dtype %d group %d tokens %lld rows %d seqs %d window %d sinks %d chunk %d: tq %d chunk %d "
                             "slots %d workspace %zu\n", dtype, group, (long long)cap, rows, seqs, window, sinks, chunk,
                             a.tq, a.chunk, a.slots, need);
                      return 1;
                    }
                  }
  printf("ok %ld\n", calls);
  return 0;
}
