// Trees of drafted tokens: who descends from whom, the branch that the model agrees with, and that branch's keys and values moved to
// the front of the tree's places in the cache. Small work, bound by latency; the moves, by the cache's bandwidth where there are many.
// All three in a graph: 1 request of 26 tokens, 32 layers 5.3 us; 48 of up to 60, 32 layers 12.4 (moved bytes 7.7 at the copy rate).
#include "common.cuh"
#include "kernels.h"

namespace nf {
namespace {

constexpr int kPage = 16;

// Tokens [begin, begin + n) of request r; lists that are none hold none.
__device__ __forceinline__ int2 tokens_of(const int* qo_indptr, int r, int num_tokens, unsigned int* status) {
  const int a = qo_indptr[r], b = qo_indptr[r + 1];
  if (a < 0 || b < a || b > num_tokens) {
    if (threadIdx.x == 0) report_status(status, NF_ST_BAD_INDEX);
    return make_int2(0, 0);
  }
  return make_int2(a, b - a);
}

// mask(i) = bit i or mask(parent(i)), by doubling: with masks that reach up 2^k steps and the ancestor after so many, one step more
// joins the two halves of 2^(k+1). A CTA per request, a thread per token; W: words of a mask, or the next power of two.
template <int W>
__global__ void __launch_bounds__(W * 64) tree_masks_kernel(nfk_tree_masks_params p) {
  constexpr int N = W * 64;
  __shared__ unsigned long long mask[N][W];
  __shared__ int up[N], depth[N];
  const int i = threadIdx.x;
  let_next_start();
  await_previous();
  const int2 own = tokens_of(p.qo_indptr, blockIdx.x, p.num_tokens, p.status);
  const int bits = p.words * 64, n = min(own.y, bits);
  if (own.y > bits) {                            // tokens behind the last that a mask has bits for see the context only
    if (i == 0) report_status(p.status, NF_ST_BAD_INDEX);
    for (int t = n + i; t < own.y; t += N) {
      for (int w = 0; w < p.words; ++w) p.mask[static_cast<long long>(own.x + t) * p.words + w] = 0ull;
      if (p.positions != nullptr) p.positions[own.x + t] = p.positions[own.x];
    }
  }
  int at = -1, d = 0, first = 0;
  unsigned long long m[W];
#pragma unroll
  for (int w = 0; w < W; ++w) m[w] = 0ull;
  if (i < n) {
    at = p.parents[own.x + i];
    if (at < -1 || at >= i) {                    // no parent in front of it
      report_status(p.status, NF_ST_BAD_INDEX);
      at = -1;
    }
    if (p.positions != nullptr) first = p.positions[own.x];
    d = at >= 0 ? 1 : 0;
#pragma unroll
    for (int w = 0; w < W; ++w) m[w] = (i >> 6) == w ? 1ull << (i & 63) : 0ull;
  }
  while (__syncthreads_or(at >= 0)) {
#pragma unroll
    for (int w = 0; w < W; ++w) mask[i][w] = m[w];
    up[i] = at;
    depth[i] = d;
    __syncthreads();
    if (at >= 0) {
#pragma unroll
      for (int w = 0; w < W; ++w) m[w] |= mask[at][w];
      d += depth[at];
      at = up[at];
    }
  }
  if (i < n) {
    for (int w = 0; w < p.words; ++w) {
      unsigned long long v = 0ull;
#pragma unroll
      for (int k = 0; k < W; ++k)
        if (k == w) v = m[k];
      p.mask[static_cast<long long>(own.x + i) * p.words + w] = v;
    }
    if (p.positions != nullptr) p.positions[own.x + i] = first + d;
  }
}

// A warp per request: from token 0 on, the first of the next tokens (32 at a time) whose parent is the last one taken and that holds what
// the model says behind it. Children lie behind their parents, so the search goes on from there.
constexpr int kAcceptWarps = 4;
__global__ void __launch_bounds__(kAcceptWarps * 32) tree_accept_kernel(nfk_tree_accept_params p) {
  __shared__ int parent_s[kAcceptWarps][NFK_TREE_NODES], token_s[kAcceptWarps][NFK_TREE_NODES];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = blockIdx.x * kAcceptWarps + warp;
  let_next_start();
  await_previous();
  if (r >= p.requests) return;
  const int a = p.qo_indptr[r], b = p.qo_indptr[r + 1];
  const bool bad = a < 0 || b < a || b > p.num_tokens;
  int n = bad ? 0 : b - a;
  const int all = n;
  if (n > NFK_TREE_NODES) n = NFK_TREE_NODES;
  if ((bad || all > n) && lane == 0) report_status(p.status, NF_ST_BAD_INDEX);
  for (int i = lane; i < n; i += 32) {
    parent_s[warp][i] = p.parents[a + i];
    token_s[warp][i] = p.tokens[a + i];
  }
  __syncwarp();
  int* path = p.path + static_cast<long long>(r) * p.max_path;
  int count = 0, said = -1;
  for (int at = n > 0 && p.max_path > 0 ? 0 : -1; at >= 0;) {
    if (lane == 0) path[count] = at;
    ++count;
    said = p.targets[a + at];
    int next = -1;
    for (int i0 = at + 1; count < p.max_path && i0 < n; i0 += 32) {
      const int i = i0 + lane;
      const unsigned int hit = __ballot_sync(0xffffffffu, i < n && parent_s[warp][min(i, n - 1)] == at && token_s[warp][min(i, n - 1)] == said);
      if (hit != 0u) {
        next = i0 + __ffs(static_cast<int>(hit)) - 1;
        break;
      }
    }
    at = next;
  }
  for (int k = count + lane; k < p.max_path; k += 32) path[k] = -1;
  if (lane == 0) {
    p.counts[r] = count;
    p.next_tokens[r] = said;
    if (p.dropped != nullptr) p.dropped[r] = all - count;
  }
}

// A CTA per (request, pool). A thread moves the same 16 bytes of the same head of every token, in the order of the path: token path[k] never
// lies in front of place k, so that what a move overwrites has been moved before; four moves' loads are on their way at once. A chain of
// loads (lists and path, slots, vectors) takes most of a CTA's time, which other CTAs fill: registers for six to an SM (48 requests of up
// to 60 tokens, 32 pools: with eight loads and four CTAs 2 us longer, with two pools to a CTA 4).
constexpr int kKeepThreads = 256, kAhead = 4;
__global__ void __launch_bounds__(kKeepThreads, 6) kv_keep_kernel(const __grid_constant__ nfk_kv_keep_params p) {
  __shared__ int from_s[NFK_TREE_NODES], to_s[NFK_TREE_NODES], moves_s;
  const int r = blockIdx.x / p.num_pools, pool = blockIdx.x - r * p.num_pools;
  let_next_start();
  await_previous();
  const int a = p.qo_indptr[r], b = p.qo_indptr[r + 1];
  const int* path = p.path + static_cast<long long>(r) * p.max_path;
  const int first = threadIdx.x < static_cast<unsigned int>(p.max_path) ? path[threadIdx.x] : -1;      // (with the lists, not behind them)
  int count = p.counts[r];
  bool bad = a < 0 || b < a || b > p.num_tokens || count < 0 || count > p.max_path || count > b - a || count > NFK_TREE_NODES;
  if (bad) count = 0;
  // moves that change something, in their order; by one warp
  if (threadIdx.x < 32) {
    int moves = 0;
    for (int k0 = 0; k0 < count; k0 += 32) {
      const int k = k0 + threadIdx.x;
      int from = -1, to = -1;
      if (k < count) {
        const int i = k0 == 0 ? first : path[k];
        const bool ok = i >= k && i < b - a;
        if (ok && i != k) {
          from = p.slots[a + i];
          to = p.slots[a + k];
          if (from < 0 || from >= p.num_pages * kPage || to < 0 || to >= p.num_pages * kPage) {
            bad = true;
            from = -1;
          }
        }
        bad = bad || !ok;
      }
      const unsigned int on = __ballot_sync(0xffffffffu, from >= 0);
      if (from >= 0) {
        const int at = moves + __popc(on & ((1u << threadIdx.x) - 1u));
        from_s[at] = from;
        to_s[at] = to;
      }
      moves += __popc(on);
    }
    if (threadIdx.x == 0) moves_s = moves;
    if (bad) report_status(p.status, NF_ST_BAD_INDEX);
  }
  __syncthreads();
  const int moves = moves_s;
  if (moves == 0) return;
  const int per_vec = p.head_dim / 8, chunks = 2 * p.kv_heads * per_vec;         // 16 bytes each, of a token
  uint4* base = static_cast<uint4*>(p.pools[pool]);
  auto place = [&](int slot, int chunk) {
    const int vec = chunk / per_vec;             // side and head
    return base + ((static_cast<long long>(slot / kPage) * 2 * p.kv_heads + vec) * kPage + slot % kPage) * per_vec + (chunk - vec * per_vec);
  };
  for (int chunk = threadIdx.x; chunk < chunks; chunk += kKeepThreads) {
    for (int k0 = 0; k0 < moves; k0 += kAhead) {
      uint4 v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (k0 + k < moves) v[k] = *place(from_s[k0 + k], chunk);
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (k0 + k < moves) *place(to_s[k0 + k], chunk) = v[k];
    }
  }
}

bool fits(int entries) { return entries >= 0 && entries <= NFK_DRAFT_ENTRIES; }
int started(cudaError_t e) {
  if (e == cudaSuccess) return NF_OK;
  (void)cudaGetLastError();
  return NF_ERR_CUDA;
}

}  // namespace
}  // namespace nf

extern "C" int nfk_tree_masks(const nfk_tree_masks_params* p, cudaStream_t stream) {
  using namespace nf;
  if (p == nullptr || !fits(p->requests) || !fits(p->num_tokens) || p->words < 1 || p->words > NFK_TREE_NODES / 64) return NF_ERR_BAD_ARG;
  if (p->requests == 0 || p->num_tokens == 0) return NF_OK;
  if (!p->parents || !p->qo_indptr || !p->mask || (reinterpret_cast<uintptr_t>(p->mask) & 7) != 0) return NF_ERR_BAD_ARG;
  const auto run = [&](auto kernel, int words) { return started(launch_kernel(early_first(p->early_start), kernel, p->requests, words * 64, 0, stream, 1, *p)); };
  if (p->words == 1) return run(tree_masks_kernel<1>, 1);
  if (p->words == 2) return run(tree_masks_kernel<2>, 2);
  if (p->words <= 4) return run(tree_masks_kernel<4>, 4);
  return run(tree_masks_kernel<8>, 8);
}

extern "C" int nfk_tree_accept(const nfk_tree_accept_params* p, cudaStream_t stream) {
  using namespace nf;
  if (p == nullptr || !fits(p->requests) || !fits(p->num_tokens) || !fits(p->max_path)) return NF_ERR_BAD_ARG;
  if (p->requests == 0) return NF_OK;
  if (!p->qo_indptr || !p->counts || !p->next_tokens || (p->max_path > 0 && !p->path) ||
      (p->num_tokens > 0 && (!p->tokens || !p->parents || !p->targets)))
    return NF_ERR_BAD_ARG;
  return started(launch_kernel(early_first(p->early_start), tree_accept_kernel, (p->requests + kAcceptWarps - 1) / kAcceptWarps, kAcceptWarps * 32, 0,
                               stream, 1, *p));
}

extern "C" int nfk_kv_keep(const nfk_kv_keep_params* p, cudaStream_t stream) {
  using namespace nf;
  if (p == nullptr || !fits(p->requests) || !fits(p->num_tokens) || !fits(p->max_path) || p->num_pools < 0 || p->num_pools > NFK_KEEP_POOLS)
    return NF_ERR_BAD_ARG;
  if (p->head_dim < 8 || p->head_dim % 8 != 0 || p->head_dim > 1024) return NF_ERR_UNSUPPORTED;
  if (p->requests == 0 || p->num_pools == 0 || p->max_path == 0 || p->num_tokens == 0) return NF_OK;
  if (!p->slots || !p->path || !p->counts || !p->qo_indptr || p->num_pages <= 0 || p->num_pages > 0x7fffffff / kPage || p->kv_heads <= 0 ||
      p->kv_heads > 65536)
    return NF_ERR_BAD_ARG;
  for (int i = 0; i < p->num_pools; ++i)
    if (!p->pools[i] || (reinterpret_cast<uintptr_t>(p->pools[i]) & 15) != 0) return NF_ERR_BAD_ARG;
  const long long ctas = static_cast<long long>(p->requests) * p->num_pools;
  if (ctas > 0x7fffffffll) return NF_ERR_BAD_ARG;
  return started(launch_kernel(early_first(p->early_start), kv_keep_kernel, static_cast<int>(ctas), kKeepThreads, 0, stream, 1, *p));
}
