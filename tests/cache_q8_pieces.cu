// Host program of test_cache_q8_pieces_cpu.py: which states of a shared prefix a CTA leaves that gives up in its k-th part, against those
// that the joins read. Arguments: requests, query heads, KV heads, prefix tokens, CTA budget.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "attn_q8.cuh"

int main(int, char** a) {
  nfk_attn_q8_params p = {};
  p.req_count = std::atoi(a[1]);
  p.q_heads = std::atoi(a[2]);
  p.kv_heads = std::atoi(a[3]);
  p.prefix_len = std::atoi(a[4]);
  p.num_ctas = std::atoi(a[5]);
  p.head_dim = 128;
  const nf::PrefixPlan f = nf::prefix_plan(p);
  const int items = p.kv_heads * f.blocks, span = f.lead + f.tiles;
  std::vector<int> read(items + f.ctas, 0);
  for (int item = 0; item < items; ++item)                       // (as attn_join_rows_q8_kernel has it)
    for (int c = f.cut.of(item * span + f.lead); c <= f.cut.of((item + 1) * span - 1); ++c) ++read[item + c];
  std::vector<int> parts(f.ctas, 0);
  for (int c = 0; c < f.ctas; ++c)
    for (nf::Share s(f, c); s.next();) ++parts[c];
  int most = 0;
  for (int n : parts) most = n > most ? n : most;
  for (int k = 0; k <= most; ++k) {                              // every CTA gives up in its k-th part
    std::vector<int> written(items + f.ctas, 0);
    for (int c = 0; c < f.ctas; ++c) {
      nf::Share now(f, c);
      int done = 0;
      bool ok = true;
      while (ok && now.next()) {
        if (done == k) { ok = false; break; }
        ++written[now.item + c];
        ++done;
      }
      if (!ok) now.rest([&](int item) { ++written[item + c]; });
    }
    if (written != read) {
      std::printf("given up in part %d: other states than are read\n", k);
      return 1;
    }
  }
  std::printf("%d items, %d CTAs, %d parts at most\n", items, f.ctas, most);
  return 0;
}
