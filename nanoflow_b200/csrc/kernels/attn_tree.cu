// Attention of drafted tokens (trees or chains, one to some hundred tokens a request) over the paged bf16 cache, on the 5th-generation
// tensor cores:  o = sum_j e^(s_j) v_j / sum_j e^(s_j),  s_j = sm_scale q.k_j  over the tokens j that the query's token sees.
//
// The rows of an item are those query rows of a request that share a KV head (tokens x group), in blocks of up to 256. Every key and
// value is read once per block, 4 head_dim operations a row for 4 head_dim bytes: the cache's bytes bound it below some 250 rows, the
// products (and 2^x, 16 a clock and SM, which takes as long as both products of a tile) above.
//
// A CTA has an SM to itself and two slots of 128 rows, each with scores and sums of its own in tensor memory, so that one slot's softmax
// runs under the other's products. Up to 128 rows, both slots hold the same rows and take turns at the tiles of 128 tokens, and their
// states are joined at the end; up to 256, each has its own rows and both take every tile.
//
//   8 warps     softmax, a thread per row: a tile's 128 scores to registers, running maximum and sum, weights as bf16 pairs back over
//               the scores' columns, the A operand of the second product
//   1 warp      copies (TMA, no multicast): queries, and keys and values page by page into a ring; walks the work
//   1 warp      tcgen05.mma
//
// Work is a row of pages of all requests, KV heads and blocks, cut evenly over the CTAs whatever the requests' lengths; an item that is
// cut leaves a state (maximum, sum, sums of values) per piece, which a second kernel joins, in the order of the pieces: results do not
// depend on the order in which anything runs.
//
// Weights are rounded to bf16 (2^-9 of each on average), the type of the values that they meet in the product. Scores, maxima, sums and
// states are fp32. The reference that weights are relative to moves (and sums are rescaled) where a row's maximum outgrows it by 2^8.
//
// Only tiles with drafted tokens or the end of a piece need care: masks of 128 bits a row; and values that a row does not see must not
// reach it as 0 * inf, so rows of values behind the end become zeros, as do infinities and NaN of drafted tokens, which the rows that do
// see them get back at the end (restore_odd).
#include "attn_mma.cuh"
#include "cache_q8.cuh"
#include "common.cuh"
#include "kernels.h"

namespace nf {
namespace {

constexpr int kTile = 128;            // cached tokens per tile
constexpr int kTilePages = kTile / kPage;
constexpr int kThreads = 320;         // warps 0-3 slot 0, 4-7 slot 1, 8 copies, 9 products
constexpr int kLoadWarp = 8, kMmaWarp = 9;
constexpr float kGap = 8.f;           // log2 of how far a row's maximum may outgrow its reference
// What an item's beginning and end cost, in pages: where the work is cut, the ends count too.
constexpr int kLead = 8;
// Pages that a CTA takes at least, so that the states of short requests do not outweigh their pages.
constexpr int kLeast = 8;

template <int HD>
struct Cfg {
  static constexpr int NH = HD / 64;
  static constexpr int kHalf = kTile * 128;                    // [128 tokens or rows][64 elements]
  static constexpr int kStage = NH * kHalf;                    // a tile of keys or of values; a slot's queries
  static constexpr int kStages = HD == 128 ? 5 : 10;
  static constexpr int kRing = 2 * kStage;                     // (queries of both slots in front)
  static constexpr int kMl = kRing + kStages * kStage;         // [2 slots][128] float2
  static constexpr int kBars = kMl + 2 * 128 * 8;
  static constexpr int kBytes = kBars + 512;
  enum Bar : int {
    FULL = 0, EMPTY = FULL + kStages, Q_FULL = EMPTY + kStages, Q_EMPTY, READ, O_FREE, LAST, S_FULL, P_FULL = S_FULL + 2, PV_DONE = P_FULL + 2,
    MERGE = PV_DONE + 2, kNum = MERGE + 4
  };
  static_assert(kNum * 8 + 8 + 64 + 16 + 64 <= 512 && kBytes <= 227 * 1024, "shared memory");
};

// What the roles need to know of a piece.
struct Piece {
  int tok;           // first query token of the block
  int node;          // its place among the request's tokens
  int nodes;         // tokens of the block
  int all;           // tokens of the request
  int kvh;
  int len;           // cached tokens of the request (0: nothing is known of it, or there are none)
  int list;          // the request's page list
  int page0, pages;  // of it
  int to;            // piece number, -1: the whole item
  int two;           // blocks of more than 128 rows: each slot its own
};
// What a CTA leaves for the kernel that joins states: the item that begins with it and goes on behind it, if there is one.
struct Record {
  int pieces, tok, nodes, kvh;
};

struct Workspace {
  Record* records;   // [CTAs]
  float2* ml;        // [2 CTAs][256]: reference (of exponents to base 2) and sum
  float* o;          // [2 CTAs][256][head_dim], not divided by the sum
};
long long workspace_bytes(int head_dim, Workspace* w = nullptr, void* base = nullptr) {
  const long long n = device_sm_count(), records = (n * static_cast<long long>(sizeof(Record)) + 255) / 256 * 256, ml = 2 * n * 256 * 8;
  if (w != nullptr) {
    char* at = static_cast<char*>(base);
    w->records = reinterpret_cast<Record*>(at);
    w->ml = reinterpret_cast<float2*>(at + records);
    w->o = reinterpret_cast<float*>(at + records + ml);
  }
  return records + ml + 2 * n * 256 * head_dim * 4;
}

// A request as the lists have it. Lists that are none: no query tokens, or no cached ones.
struct Request {
  int tok, n, list, pages, len;
  long long blocks;
};
__device__ __forceinline__ Request read_request(const nfk_attn_tree_params& p, int r, int nodes_per_block, bool report) {
  const int req = p.req_begin + r;
  Request q;
  q.tok = p.qo_indptr[req];
  q.n = p.qo_indptr[req + 1];
  q.list = p.kv_indptr[req];
  q.pages = p.kv_indptr[req + 1];
  const int last = p.kv_last_page_len[req];
  const bool q_bad = q.tok < 0 || q.n < q.tok || q.n > p.num_tokens;
  q.n = q_bad ? 0 : q.n - q.tok;
  bool kv_bad = q.list < 0 || q.pages < q.list || q.pages > p.num_indices || q.pages - q.list > 0x7fffff0 || (q.pages > q.list && (last < 1 || last > kPage));
  q.pages = kv_bad ? 0 : q.pages - q.list;
  q.len = q.pages > 0 ? (q.pages - 1) * kPage + last : 0;
  if (!kv_bad && q.len < q.n && q.n > 0) kv_bad = true;       // drafted tokens that are not cached
  if (kv_bad) q.pages = q.len = 0;
  if (report && (q_bad || kv_bad)) report_status(p.status, NF_ST_BAD_INDEX);
  q.blocks = (q.n + nodes_per_block - 1) / nodes_per_block;
  return q;
}
// Units of a request, for one KV head.
__device__ __forceinline__ long long units_of(const Request& q) { return q.blocks * (kLead + q.pages); }

// How `total` units are cut over `w` CTAs.
struct Cut {
  long long total;
  int w;
  __device__ __forceinline__ Cut(long long t, int ctas) : total(t) {
    const long long most = (t + kLead + kLeast - 1) / (kLead + kLeast);
    w = static_cast<int>(most < ctas ? (most > 0 ? most : 1) : ctas);
  }
  __device__ __forceinline__ long long begin(int c) const { return total * c / w; }
  __device__ __forceinline__ int of(long long u) const { return static_cast<int>(((u + 1) * w - 1) / total); }
};

// Bits of the 32 tokens from `off` on (counted from the first drafted token, negative: context) that the token `node` sees.
__device__ __forceinline__ uint32_t seen_bits(const uint32_t* row, int words32, int node, int all, int off) {
  if (off <= -32) return ~0u;
  uint32_t bits;
  if (row == nullptr) {
    const int n = node + 1 - max(off, 0);                      // that it sees from there on
    bits = n >= 32 ? ~0u : n > 0 ? (1u << n) - 1u : 0u;
  } else {
    const int o = max(off, 0), k = o >> 5;
    const uint32_t lo = k < words32 ? row[k] : 0u, hi = k + 1 < words32 ? row[k + 1] : 0u;
    bits = __funnelshift_r(lo, hi, o & 31);
  }
  const int left = all - max(off, 0);
  if (left < 32) bits &= left > 0 ? (1u << left) - 1u : 0u;
  if (off < 0) bits = (bits << -off) | ((1u << -off) - 1u);
  return bits;
}

__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* tm, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// bf16 pairs with an infinity or NaN in them
__device__ __forceinline__ bool odd_pair(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }
__device__ __forceinline__ uint32_t without_odd(uint32_t w) {
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
  return w;
}

// Infinities and NaN of the drafted tokens [from, end) that the row sees, in 16 columns: as terms of its sums they are what they are,
// whatever their weights. (Only where there are some.)
template <int HD>
__device__ __forceinline__ void restore_odd(const nfk_attn_tree_params& p, const Piece& f, const uint32_t* tree, int node, int from, int end, int c,
                                         float (&o)[16]) {
  for (int t = from; t < end; ++t) {
    if ((seen_bits(tree, 2 * p.words, node, f.all, t - (f.len - f.all)) & 1u) == 0u) continue;
    int page = p.kv_indices[f.list + t / kPage];
    if (page < 0 || page >= p.num_pages) page = 0;               // (as it was read)
    const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(p.kv_pool) + (((static_cast<long long>(page) * 2 + 1) * p.kv_heads + f.kvh) * kPage + t % kPage) * HD + c;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float x = __bfloat162float(v[j]);
      if (!isfinite(x)) o[j] += x;
    }
  }
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
attn_tree_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmKV, nfk_attn_tree_params p, Workspace ws) {
  using C = Cfg<HD>;
  constexpr int NH = C::NH, NST = C::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sb = smem_u32(smem);
  float2* ml_s = reinterpret_cast<float2*>(smem + C::kMl);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kNum);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* odd_item = reinterpret_cast<volatile int*>(tmem_slot + 2);         // [2]: numbers of items with odd values
  Piece* piece_s = reinterpret_cast<Piece*>(tmem_slot + 4);
  // (before the roles begin) sums of the warps' units, units in front of the CTA's first request, its number
  long long* scan_s = reinterpret_cast<long long*>(smem + C::kMl);
  long long* start_off_s = scan_s + kThreads / 32;
  int* start_req_s = reinterpret_cast<int*>(start_off_s + 1);
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int group = p.q_heads / p.kv_heads, per_slot = 128 / group;                // tokens of a slot
  if ((sb & 1023u) != 0u) {                      // the operands' layouts need it; report instead of computing garbage
    await_previous();
    if (threadIdx.x == 0) {
      report_status(p.status, NF_ST_BAD_INDEX);
      ws.records[blockIdx.x] = Record{0, 0, 0, 0};
    }
    return;
  }
  if (threadIdx.x == 0) {
    for (int b = 0; b < C::kNum; ++b) {
      const int n = b == C::READ ? 9 : b == C::O_FREE ? 8 : (b >= C::P_FULL && b < C::PV_DONE) ? 4 : b >= C::MERGE ? 2 : 1;
      mbar_init(&bars[b], n);
    }
    *abort_flag = 0;
    odd_item[0] = odd_item[1] = -1;
    mbar_fence_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmKV);
  }
  await_previous();                              // (before tensor memory is taken, which the kernel before may need)
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, 512);                  // of each slot (256 columns): scores in [0, 128), sums in [128, 128 + HD)
    tmem_relinquish();
  }
  // ---- where this CTA's share of the units begins: units of every thread's requests, scanned ----
  const int per_thread = (p.req_count + kThreads - 1) / kThreads;
  const int r0 = min(p.req_count, static_cast<int>(threadIdx.x) * per_thread), r1 = min(p.req_count, r0 + per_thread);
  long long mine = 0;
  for (int r = r0; r < r1; ++r) mine += units_of(read_request(p, r, 2 * per_slot, blockIdx.x == 0)) * p.kv_heads;
  long long sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += v;
  }
  if (lane == 31) scan_s[warp] = sum;
  if (threadIdx.x == 0) *start_req_s = -1;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  long long before = sum - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    const long long v = scan_s[w];
    if (w < warp) before += v;
    total += v;
  }
  const Cut cut(total, gridDim.x);
  const bool works = total > 0 && static_cast<int>(blockIdx.x) < cut.w;
  const long long u0 = works ? cut.begin(blockIdx.x) : 0, u1 = works ? cut.begin(blockIdx.x + 1) : 0;
  if (works && u0 >= before && u0 < before + mine) {           // one thread
    long long at = before;
    for (int r = r0; r < r1; ++r) {
      const long long n = units_of(read_request(p, r, 2 * per_slot, false)) * p.kv_heads;
      if (u0 < at + n) {
        *start_req_s = r;
        *start_off_s = at;
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  const uint32_t tmem = *tmem_slot;
  const int start_req = *start_req_s;
  const long long start_off = *start_off_s;
  __syncthreads();
  let_next_start();

  auto fail = [&](unsigned int code) {
    if (lane == 0) report_status(p.status, code);
    *abort_flag = 1;
  };
  auto passed = [&](int bar, uint32_t parity) { return __all_sync(0xffffffffu, wait_or_abort(&bars[bar], parity, abort_flag)) != 0; };
  // ring positions of an item's tiles, in the order of their use: K0, K1, V0, K2, V1, ... , V(n-1)
  auto k_at = [](int t) { return t == 0 ? 0 : 2 * t - 1; };
  auto v_at = [](int t, int n) { return t == n - 1 ? 2 * n - 1 : 2 * t + 2; };

  if (!works || start_req < 0) {
    if (threadIdx.x == 0) ws.records[blockIdx.x] = Record{0, 0, 0, 0};
  } else if (warp == kLoadWarp) {
    // ------------------------------------------------------------------ copies (the warp walks, an elected lane issues)
    Record record{0, 0, 0, 0};
    uint32_t ring = 0, n_item = 0;               // tiles so far (keys and values each), items so far
    const int no_row = static_cast<int>(min(static_cast<long long>(p.num_pages) * 2 * p.kv_heads * kPage, 0x7fffff00ll));   // behind the pool: zeros
    bool ok = true;
    long long at = start_off;                    // units in front of request r
    for (int r = start_req; ok && r < p.req_count && at < u1; ++r) {
      const Request q = read_request(p, r, 2 * per_slot, false);
      const long long span = kLead + q.pages, n_items = q.blocks * p.kv_heads;
      for (long long i = max(0ll, (u0 - at) / (span > 0 ? span : 1)); ok && i < n_items; ++i) {
        const long long s = at + i * span;       // the item's first unit
        if (s >= u1) break;
        if (s + span <= u0) continue;
        Piece f;
        f.kvh = static_cast<int>(i / q.blocks);
        f.node = static_cast<int>(i - f.kvh * q.blocks) * 2 * per_slot;
        f.tok = q.tok + f.node;
        f.nodes = min(2 * per_slot, q.n - f.node);
        f.all = q.n;
        f.list = q.list;
        f.len = q.len;
        f.two = f.nodes > per_slot;
        const long long first = s + kLead, lo = max(u0, first), hi = min(u1, s + span);
        f.page0 = static_cast<int>(lo - first);
        f.pages = static_cast<int>(max(0ll, hi - lo));
        f.to = -1;
        if (q.pages == 0) {
          if (s < u0) continue;                  // rows of zeros: by the CTA that the item begins with
        } else {
          if (f.pages == 0) continue;
          const int c0 = cut.of(first), c1 = cut.of(s + span - 1);
          if (c0 != c1) {
            f.to = 2 * blockIdx.x + (c0 == static_cast<int>(blockIdx.x) ? 1 : 0);
            if (c0 == static_cast<int>(blockIdx.x)) record = Record{c1 - c0 + 1, f.tok, f.nodes, f.kvh};
          }
        }
        const int tiles = (f.pages + kTilePages - 1) / kTilePages;
        const int* list = p.kv_indices + q.list + f.page0;
        // Page numbers of 32 pages (four tiles) at a time, a lane each; keys are a tile ahead of values, so that of the next 32 come first
        // when there is one tile of the others left.
        auto fetch = [&](int group_of_32) {
          const int j = group_of_32 * 32 + lane;
          int page = -1;
          if (j < f.pages) {
            page = list[j];
            if (page < 0 || page >= p.num_pages) {
              report_status(p.status, NF_ST_BAD_INDEX);
              page = 0;
            }
          }
          return page;
        };
        int held[2] = {-1, -1};
        auto issue = [&](int pos, int tile, int part) {
          if (part == 0 && (tile & 3) == 0) {
            if ((tile >> 2 & 1) != 0) held[1] = fetch(tile >> 2);
            else held[0] = fetch(tile >> 2);
          }
          const int pages = (tile >> 2 & 1) != 0 ? held[1] : held[0];
          const uint32_t at_ring = ring + pos, stage = at_ring % NST;
          if (!passed(C::EMPTY + stage, (at_ring / NST & 1) ^ 1)) return false;
          uint8_t* to = smem + C::kRing + stage * C::kStage;
          int rows[kTilePages];
#pragma unroll
          for (int j = 0; j < kTilePages; ++j) {
            const int page = __shfl_sync(0xffffffffu, pages, (tile & 3) * kTilePages + j);
            rows[j] = page < 0 ? no_row : ((page * 2 + part) * p.kv_heads + f.kvh) * kPage;
          }
          if (elect_one()) {
            mbar_expect_tx(&bars[C::FULL + stage], C::kStage);
#pragma unroll
            for (int j = 0; j < kTilePages; ++j)
#pragma unroll
              for (int h = 0; h < NH; ++h)
                tma_load_2d(to + h * C::kHalf + j * (kPage * 128), &tmKV, &bars[C::FULL + stage], h * 64, rows[j]);
          }
          __syncwarp();
          return true;
        };
        // the first tiles are on their way before the queries, which wait for the item before
        const int ahead = min(2 * tiles, 3);
        auto issue_at = [&](int pos) {           // the inverse of k_at, v_at
          const bool key = pos == 0 || ((pos & 1) != 0 && pos != 2 * tiles - 1);
          return issue(pos, key ? (pos + 1) / 2 : pos == 2 * tiles - 1 ? tiles - 1 : pos / 2 - 1, key ? 0 : 1);
        };
        int pos = 0;
        for (; ok && pos < ahead; ++pos) ok = issue_at(pos);
        if (!ok || !passed(C::READ, (n_item & 1) ^ 1) || !passed(C::Q_EMPTY, (n_item & 1) ^ 1)) {
          ring += pos;
          ok = false;
          break;
        }
        if (elect_one()) {
          *piece_s = f;
          const int slots = f.two ? 2 : 1;
          mbar_expect_tx(&bars[C::Q_FULL], slots * NH * per_slot * group * 128);
          for (int slot = 0; slot < slots; ++slot)
#pragma unroll
            for (int h = 0; h < NH; ++h)
              tma_load_3d(smem + slot * C::kStage + h * C::kHalf, &tmQ, &bars[C::Q_FULL], h * 64, f.kvh * group, f.tok + slot * per_slot);
        }
        __syncwarp();
        ++n_item;
        for (; ok && pos < 2 * tiles; ++pos) ok = issue_at(pos);
        ring += pos;
      }
      at += n_items * span;
    }
    if (!ok) fail(NF_ST_TIMEOUT_SMEM_EMPTY);
    if (lane == 0) ws.records[blockIdx.x] = record;
    if (ok && passed(C::READ, (n_item & 1) ^ 1) && passed(C::Q_EMPTY, (n_item & 1) ^ 1)) {
      if (elect_one()) {                         // no more pieces
        piece_s->nodes = 0;
        mbar_arrive(&bars[C::Q_FULL]);
      }
      __syncwarp();
    } else if (n_item > 0) {
      (void)mbar_wait(&bars[C::Q_FULL], (n_item - 1) & 1);
    }
    // copies still in flight must have landed before the CTA gives its shared memory back
    for (uint32_t k = ring > NST ? ring - NST : 0; k < ring; ++k) (void)mbar_wait(&bars[C::FULL + k % NST], k / NST & 1);
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------------ products (the warp walks, an elected lane issues)
    const uint32_t idesc_s = umma_idesc_bf16(128, kTile), idesc_o = umma_idesc_bf16(128, HD) | kIdescBMnMajor;
    const uint64_t q_desc = umma_desc_k_sw128(sb), k_desc = umma_desc_k_sw128(sb + C::kRing);
    const uint64_t v_desc = umma_desc_mn_sw128(sb + C::kRing, C::kHalf, 1024);
    uint32_t ring = 0, n_item = 0, done[2] = {0, 0};           // second products issued, of each slot
    bool ok = true;
    for (;;) {
      if (!passed(C::Q_FULL, n_item & 1)) { ok = false; break; }
      const int nodes = piece_s->nodes, pages = piece_s->pages, two = piece_s->two;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[C::READ]);
      if (nodes == 0) break;
      const int tiles = (pages + kTilePages - 1) / kTilePages;
      const int n0 = two ? tiles : (tiles + 1) / 2, n1 = two ? tiles : tiles / 2;
      int left = n0 + n1;                        // scores to issue
      // S(slot) of its i-th tile goes over the weights of the one before, which that one's second product reads: it must have ended
      auto scores = [&](int slot, int i) {
        const int tile = two ? i : 2 * i + slot;
        const uint32_t k = ring + k_at(tile);
        if (done[slot] > 0 && !passed(C::PV_DONE + slot, (done[slot] - 1) & 1)) return false;
        if (!passed(C::FULL + k % NST, k / NST & 1)) return false;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t qd = q_desc + static_cast<uint64_t>((two ? slot : 0) * (C::kStage >> 4)), kd = k_desc + static_cast<uint64_t>(k % NST * (C::kStage >> 4));
#pragma unroll
          for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int s = 0; s < 4; ++s)
              umma_bf16_ss(tmem + slot * 256, qd + ((h * C::kHalf + s * 32) >> 4), kd + ((h * C::kHalf + s * 32) >> 4), idesc_s, (h | s) ? 1u : 0u);
          umma_commit(&bars[C::S_FULL + slot]);
          if (!two || slot == 1) umma_commit(&bars[C::EMPTY + k % NST]);
          if (left == 1) umma_commit(&bars[C::Q_EMPTY]);
        }
        __syncwarp();
        --left;
        return true;
      };
      auto sums = [&](int slot, int i) {
        const int tile = two ? i : 2 * i + slot;
        const uint32_t v = ring + v_at(tile, tiles);
        // the item before must have been read out of both slots' sums
        if (i == 0 && !passed(C::O_FREE, (n_item & 1) ^ 1)) return false;
        if (!passed(C::FULL + v % NST, v / NST & 1) || !passed(C::P_FULL + slot, done[slot] & 1)) return false;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t vd = v_desc + static_cast<uint64_t>(v % NST * (C::kStage >> 4));
#pragma unroll
          for (int s = 0; s < kTile / 16; ++s)
            umma_bf16_ts(tmem + slot * 256 + kTile, tmem + slot * 256 + s * 8, vd + ((s * 2048) >> 4), idesc_o, (i | s) ? 1u : 0u);
          umma_commit(&bars[C::PV_DONE + slot]);
          if (!two || slot == 1) umma_commit(&bars[C::EMPTY + v % NST]);
        }
        __syncwarp();
        ++done[slot];
        return true;
      };
      if (tiles == 0) {                          // (phases are not skipped: a parity stands for every other one)
        ok = passed(C::O_FREE, (n_item & 1) ^ 1);
        if (elect_one()) mbar_arrive(&bars[C::Q_EMPTY]);
        __syncwarp();
      }
      ok = ok && (n0 == 0 || scores(0, 0)) && (n1 == 0 || scores(1, 0));
      for (int i = 0; ok && i < n0; ++i) {
        // (with two row blocks slot 0 has made the tile's values fit to be multiplied before slot 1 comes to them)
        ok = sums(0, i) && (i + 1 >= n0 || scores(0, i + 1)) && (i >= n1 || sums(1, i)) && (i + 1 >= n1 || scores(1, i + 1));
      }
      if (!ok) break;
      ring += 2 * tiles;
      ++n_item;
    }
    if (!ok) {                                   // products in flight get a bounded chance to end before their memory is given back
      fail(NF_ST_TIMEOUT_SMEM_FULL);
      if (elect_one()) umma_commit(&bars[C::LAST]);
      __syncwarp();
      (void)mbar_wait(&bars[C::LAST], 0);
    }
  } else {
    // ------------------------------------------------------------------ softmax (a thread per query row)
    const int slot = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t t_s = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + slot * 256, t_o = t_s + kTile;
    const int in_slot = row / group, hh = row - in_slot * group;
    const float scale = p.sm_scale * kLog2e;
    uint32_t ring = 0, n_item = 0, n_done = 0, n_merge = 0;
    // States that will not be formed are NaN, and not what an earlier call left in the workspace.
#pragma unroll
    for (int k = 0; k < 2; ++k) __stcg(ws.ml + (2 * blockIdx.x + k) * 256 + slot * 128 + row, make_float2(0.f, __uint_as_float(0x7fc00000u)));
    for (;;) {
      if (!passed(C::Q_FULL, n_item & 1)) { fail(NF_ST_TIMEOUT_SMEM_FULL); break; }
      const Piece f = *piece_s;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[C::READ]);
      if (f.nodes == 0) break;
      const int tiles = (f.pages + kTilePages - 1) / kTilePages;
      const int n_mine = f.two ? tiles : (tiles + 1 - slot) / 2;
      const int node_in = in_slot + (f.two ? slot * per_slot : 0);       // of the block
      const bool on = in_slot < per_slot && node_in < f.nodes;
      const bool warp_on = __any_sync(0xffffffffu, on);
      const int node = f.node + node_in, ctx = f.len - f.all;
      const uint32_t* tree = p.tree == nullptr ? nullptr : reinterpret_cast<const uint32_t*>(p.tree + static_cast<long long>(f.tok + (on ? node_in : 0)) * p.words);
      const int end = min(f.len, (f.page0 + f.pages) * kPage);           // of the piece's tokens
      float ref = -INFINITY, l = 0.f;
      bool sees = false, ok = true;
      for (int i = 0; i < n_mine; ++i) {
        const int tile = f.two ? i : 2 * i + slot;
        const int at = f.page0 * kPage + tile * kTile;                   // the tile's first token
        const bool care = at + kTile > min(ctx, end);
        uint32_t bits[4] = {~0u, ~0u, ~0u, ~0u};
        if (care) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int left = end - (at + k * 32);
            bits[k] = on ? seen_bits(tree, 2 * p.words, node, f.all, at + k * 32 - ctx) & (left >= 32 ? ~0u : left > 0 ? (1u << left) - 1u : 0u) : 0u;
          }
        }
        if (!passed(C::S_FULL + slot, n_done & 1)) { ok = false; break; }
        if (care && (!f.two || slot == 0)) {
          // ---- values of the tile: a thread per token ----
          // (Behind the wait for the scores: a parity tells only neighbouring phases apart, and where the scores have been issued, what
          // was in the ring's place before these values has come and been used.)
          const uint32_t v = ring + v_at(tile, tiles);
          if (!passed(C::FULL + v % NST, v / NST & 1)) { ok = false; break; }
          const int token = at + row;
          if (token >= ctx) {
            const uint32_t v_row = sb + C::kRing + v % NST * C::kStage + row * 128;
            bool odd = false;
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) {
              const uint32_t a = v_row + (c >> 3) * C::kHalf + (((c & 7) ^ (row & 7)) << 4);
              if (token >= end) {
                st_shared_v4(a, make_uint4(0u, 0u, 0u, 0u));
              } else {
                uint4 w = ld_shared_v4(a);
                if (odd_pair(w.x) || odd_pair(w.y) || odd_pair(w.z) || odd_pair(w.w)) {
                  odd = true;
                  w = make_uint4(without_odd(w.x), without_odd(w.y), without_odd(w.z), without_odd(w.w));
                  st_shared_v4(a, w);
                }
              }
            }
            if (odd) odd_item[n_item & 1] = static_cast<int>(n_item);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (warp_on) {
          tc_fence_after();
          uint32_t x[4][32];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(t_s + c * 32, x[c]);
          tmem_ld_wait();
          if (care) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              sees = sees || bits[c] != 0u;
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if ((bits[c] >> j & 1u) == 0u) x[c][j] = 0xff800000u;    // -inf
            }
          } else {
            sees = true;
          }
          float mq[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int j = 0; j < 32; j += 2) mq[c] = max3(mq[c], __uint_as_float(x[c][j]), __uint_as_float(x[c][j + 1]));
          const float mx = fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3])) * scale;
          const bool grow = mx > ref + kGap || (ref == -INFINITY && mx > -INFINITY);
          if (i == 0) {
            ref = mx;
          } else if (__any_sync(0xffffffffu, grow)) {
            // The second product before this tile's is the last one issued, and it has ended: the tile's scores were issued after that.
            if (!passed(C::PV_DONE + slot, (n_done - 1) & 1)) { ok = false; break; }
            tc_fence_after();
            const float alpha = grow ? (ref == -INFINITY ? 0.f : fast_exp2(ref - mx)) : 1.f;
#pragma unroll 1
            for (int c = 0; c < HD / 16; ++c) {
              uint32_t o[16];
              tmem_ld_32x32b_x16n(t_o + c * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
              asm volatile(
                  "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(t_o + c * 16),
                  "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7]), "r"(o[8]), "r"(o[9]), "r"(o[10]),
                  "r"(o[11]), "r"(o[12]), "r"(o[13]), "r"(o[14]), "r"(o[15])
                  : "memory");
            }
            tmem_st_wait();
            l *= alpha;
            if (grow) ref = mx;
          }
          const float ms = ref == -INFINITY ? 0.f : ref;
          const f32x2 scale2 = pair(scale, scale), ms2 = pair(-ms, -ms);
          f32x2 rs[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[32];                     // column j: tokens 2j, 2j + 1
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float2 y = halves(fma2(pair(__uint_as_float(x[2 * c + (j >> 4)][2 * (j & 15)]), __uint_as_float(x[2 * c + (j >> 4)][2 * (j & 15) + 1])), scale2, ms2));
              const float e0 = fast_exp2(y.x), e1 = fast_exp2(y.y);
              rs[j & 1] = add2(rs[j & 1], pair(e0, e1));
              pk[j] = pack_bf16x2(e0, e1);
            }
            tmem_st_32x32b_x32(t_s + c * 32, pk);
          }
          const float2 t = halves(add2(rs[0], rs[1]));
          l += t.x + t.y;
          tmem_st_wait();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[C::P_FULL + slot]);
        ++n_done;
      }
      if (!ok) { fail(NF_ST_TIMEOUT_TMEM_FULL); break; }
      ring += 2 * tiles;
      if (n_mine > 0 && !passed(C::PV_DONE + slot, (n_done - 1) & 1)) { fail(NF_ST_TIMEOUT_TMEM_FULL); break; }
      tc_fence_after();
      if (sees && l == 0.f) l = __uint_as_float(0x7fc00000u);            // all that it sees has a score of minus infinity
      // ---- sums of the row: columns [from, to), a0 times those of slot 0 and a1 times those of slot 1 ----
      float a_mine = 1.f, a_other = 0.f;
      int from = 0, to = HD;
      if (!f.two) {
        // (one without tiles does not write, it may be an item ahead of the other's reads)
        if (n_mine > 0) ml_s[slot * 128 + row] = make_float2(ref, l);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[C::MERGE + (warp & 3)]);
        if (!passed(C::MERGE + (warp & 3), n_merge & 1)) { fail(NF_ST_TIMEOUT_TMEM_FULL); break; }
        ++n_merge;
        tc_fence_after();
        const bool alone = tiles < (slot == 0 ? 2 : 1);
        const float2 other = alone ? make_float2(-INFINITY, 0.f) : ml_s[(slot ^ 1) * 128 + row];
        const float top = fmaxf(ref, other.x);
        if (top == -INFINITY) {
          a_mine = 0.f;
          l += other.y;
        } else {                                 // (NaN where a score is infinite)
          a_mine = ref == -INFINITY ? 0.f : fast_exp2(ref - top);
          a_other = other.x == -INFINITY ? 0.f : fast_exp2(other.x - top);
          l = (a_mine != 0.f ? a_mine * l : 0.f) + (a_other != 0.f ? a_other * other.y : 0.f);
        }
        ref = top;
        from = slot * (HD / 2);
        to = from + HD / 2;
      } else if (ref == -INFINITY) {
        a_mine = 0.f;
      }
      const bool odd = odd_item[n_item & 1] == static_cast<int>(n_item);
      // a row without weights: zeros, or NaN (l) where it sees something
      const float by = f.to < 0 ? (l > 0.f ? 1.f / l : l) : 1.f;
      const long long out_row = static_cast<long long>(f.tok + node_in) * p.ld_out + (f.kvh * group + hh) * HD;
      const long long o_row = (static_cast<long long>(f.to) * 256 + (f.two ? slot * 128 : 0) + row) * HD;
      if (warp_on) {
        const bool use_mine = a_mine != 0.f, use_other = a_other != 0.f;
#pragma unroll 1
        for (int c = from; c < to; c += 16) {
          uint32_t a[16], b[16];
          float o[16];
          tmem_ld_32x32b_x16n(t_o + c, a);
          if (!f.two) tmem_ld_32x32b_x16n((t_o ^ 256u) + c, b);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) o[j] = (use_mine ? a_mine * __uint_as_float(a[j]) : 0.f) + (use_other ? a_other * __uint_as_float(b[j]) : 0.f);
          if (on) {
            if (odd) restore_odd<HD>(p, f, tree, node, max(f.page0 * kPage, ctx), end, c, o);
            if (f.to < 0) {
              __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.out) + out_row + c;
#pragma unroll
              for (int k = 0; k < 2; ++k)
                *reinterpret_cast<uint4*>(dst + k * 8) =
                    make_uint4(pack_bf16x2(o[8 * k] * by, o[8 * k + 1] * by), pack_bf16x2(o[8 * k + 2] * by, o[8 * k + 3] * by),
                               pack_bf16x2(o[8 * k + 4] * by, o[8 * k + 5] * by), pack_bf16x2(o[8 * k + 6] * by, o[8 * k + 7] * by));
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                __stcg(reinterpret_cast<float4*>(ws.o + o_row + c) + k, make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]));
            }
          }
          __syncwarp();
        }
        if (on && f.to >= 0 && (f.two || slot == 0)) __stcg(ws.ml + static_cast<long long>(f.to) * 256 + (f.two ? slot * 128 : 0) + row, make_float2(ref, l));
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[C::O_FREE]);
      ++n_item;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Rows of items that were cut: a warp per row, lanes over its pieces for the weights and over head_dim for the sums.
constexpr int kJoinWarps = 8, kJoinParts = 8;
template <int HD>
__global__ void __launch_bounds__(kJoinWarps * 32) attn_tree_join_kernel(nfk_attn_tree_params p, Workspace ws, int ctas) {
  constexpr int V = HD / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = p.q_heads / p.kv_heads, per_slot = 128 / group;
  await_previous();
  let_next_start();
  for (int work = blockIdx.x; work < ctas * kJoinParts; work += gridDim.x) {
    const int c = work / kJoinParts, part = work - c * kJoinParts;
    const int4 rec = __ldcg(reinterpret_cast<const int4*>(ws.records + c));
    const int pieces = rec.x, tok = rec.y, nodes = rec.z, kvh = rec.w;
    for (int b = part * kJoinWarps + warp; pieces > 0 && b < nodes * group; b += kJoinParts * kJoinWarps) {
      const int node = b / group, hh = b - node * group, slot = node / per_slot;
      const int row = slot * 128 + (node - slot * per_slot) * group + hh;
      auto number = [&](int k) { return static_cast<long long>(k == 0 ? 2 * c + 1 : 2 * (c + k)) * 256 + row; };
      float top = -INFINITY, odd = 0.f;
      for (int k = lane; k < pieces; k += 32) {
        const float2 ml = __ldcg(ws.ml + number(k));
        top = fmaxf(top, ml.x);
        if (ml.y != ml.y) odd = ml.y;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      float sum = 0.f, acc[V];
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] = 0.f;
      for (int k0 = 0; k0 < pieces; k0 += 32) {
        float w = 0.f, l = 0.f;
        if (k0 + lane < pieces) {
          const float2 ml = __ldcg(ws.ml + number(k0 + lane));
          w = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - top);
          l = ml.y;
        }
        sum += w != 0.f ? w * l : 0.f;
        const int here = min(32, pieces - k0);
#pragma unroll 4
        for (int k = 0; k < here; ++k) {
          const float by = __shfl_sync(0xffffffffu, w, k);
          const float* from = ws.o + number(k0 + k) * HD + lane * V;
          float x[V];
          if (V == 4) {
            const float4 y = __ldcg(reinterpret_cast<const float4*>(from));
            x[0] = y.x; x[1] = y.y; x[V - 2] = y.z; x[V - 1] = y.w;
          } else {
            const float2 y = __ldcg(reinterpret_cast<const float2*>(from));
            x[0] = y.x; x[1] = y.y;
          }
#pragma unroll
          for (int v = 0; v < V; ++v) acc[v] += by != 0.f ? by * x[v] : 0.f;
        }
      }
      sum = warp_sum(sum);
      // without weights: zeros, or NaN where the row sees something
      odd = top == -INFINITY ? warp_sum(odd) : 0.f;
      const float by = sum > 0.f ? 1.f / sum : sum + odd;
      uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(p.out) + static_cast<long long>(tok + node) * p.ld_out + (kvh * group + hh) * HD + lane * V);
#pragma unroll
      for (int v = 0; v < V; v += 2) dst[v / 2] = pack_bf16x2(acc[v] * by, acc[v + 1] * by);
    }
  }
}

int encode(CUtensorMap* out, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
  const nf_encode_tiled_fn enc = get_encode_tiled();
  if (enc == nullptr) return NF_ERR_CUDA;
  const cuuint32_t ones[3] = {1, 1, 1};
  return enc(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? NF_OK : NF_ERR_CUDA;
}

template <int HD>
int launch(const nfk_attn_tree_params& p, cudaStream_t stream) {
  using C = Cfg<HD>;
  static bool attr_dev[kMaxDevices] = {false};
  bool& attr = attr_dev[device_slot()];
  if (!attr) {
    if (cudaFuncSetAttribute(attn_tree_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kBytes) != cudaSuccess) {
      (void)cudaGetLastError();
      return NF_ERR_CUDA;
    }
    attr = true;
  }
  const int group = p.q_heads / p.kv_heads;
  CUtensorMap tm_q, tm_kv;
  const cuuint64_t q_dims[3] = {HD, static_cast<cuuint64_t>(p.q_heads), static_cast<cuuint64_t>(p.num_tokens)};
  const cuuint64_t q_strides[2] = {HD * 2, static_cast<cuuint64_t>(p.ld_q) * 2};
  const cuuint32_t q_box[3] = {64, static_cast<cuuint32_t>(group), static_cast<cuuint32_t>(128 / group)};
  int rc = encode(&tm_q, 3, p.q, q_dims, q_strides, q_box);
  if (rc != NF_OK) return rc;
  const cuuint64_t kv_dims[2] = {HD, static_cast<cuuint64_t>(p.num_pages) * 2 * p.kv_heads * kPage}, kv_strides[1] = {HD * 2};
  const cuuint32_t kv_box[2] = {64, kPage};
  rc = encode(&tm_kv, 2, p.kv_pool, kv_dims, kv_strides, kv_box);
  if (rc != NF_OK) return rc;
  Workspace ws;
  workspace_bytes(HD, &ws, p.workspace);
  const int sms = device_sm_count(), ctas = p.num_ctas > 0 && p.num_ctas < sms ? p.num_ctas : sms;
  int joins = ctas * kJoinParts;
  if (p.num_ctas > 0 && p.num_ctas < joins) joins = p.num_ctas;
  if (launch_kernel(early_first(p.early_start), attn_tree_kernel<HD>, ctas, kThreads, C::kBytes, stream, 1, tm_q, tm_kv, p, ws) != cudaSuccess ||
      launch_kernel(early_further(p.early_start), attn_tree_join_kernel<HD>, joins, kJoinWarps * 32, 0, stream, 1, p, ws, ctas) != cudaSuccess) {
    (void)cudaGetLastError();
    return NF_ERR_CUDA;
  }
  return NF_OK;
}

}  // namespace
}  // namespace nf

extern "C" long long nfk_attn_tree_workspace(const nfk_attn_tree_params* p) {
  return p != nullptr && (p->head_dim == 64 || p->head_dim == 128) ? nf::workspace_bytes(p->head_dim) : 0;
}

extern "C" int nfk_attn_tree(const nfk_attn_tree_params* p, cudaStream_t stream) {
  using namespace nf;
  if (p == nullptr || p->req_count < 0 || p->req_begin < 0 || p->num_ctas < 0) return NF_ERR_BAD_ARG;
  if ((p->head_dim != 64 && p->head_dim != 128) || p->kv_heads <= 0 || p->q_heads <= 0 || p->q_heads % p->kv_heads != 0 || p->q_heads / p->kv_heads > 128)
    return NF_ERR_UNSUPPORTED;
  if (p->req_count == 0 || p->num_tokens == 0) return NF_OK;
  const auto off = [](const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) != 0; };
  const long long row = static_cast<long long>(p->q_heads) * p->head_dim;
  if (!p->q || !p->out || !p->kv_pool || !p->qo_indptr || !p->kv_indptr || !p->kv_indices || !p->kv_last_page_len || !p->workspace || off(p->q) ||
      off(p->out) || off(p->kv_pool) || (reinterpret_cast<uintptr_t>(p->workspace) & 255) != 0 || (reinterpret_cast<uintptr_t>(p->tree) & 7) != 0)
    return NF_ERR_BAD_ARG;
  if (p->num_tokens < 0 || p->num_pages <= 0 || p->num_indices < 0 || p->ld_q % 8 != 0 || p->ld_out % 8 != 0 || p->ld_q < row || p->ld_out < row ||
      p->req_begin > 0x7fffffff - p->req_count || !(p->sm_scale > 0.f) || p->sm_scale > 3e38f || p->workspace_bytes < workspace_bytes(p->head_dim) ||
      (p->tree != nullptr && (p->words < 1 || p->words > NFK_TREE_NODES / 64)) ||
      static_cast<long long>(p->num_pages) * 2 * p->kv_heads * kPage > 0x7fff0000ll)
    return NF_ERR_BAD_ARG;
  return p->head_dim == 128 ? launch<128>(*p, stream) : launch<64>(*p, stream);
}
