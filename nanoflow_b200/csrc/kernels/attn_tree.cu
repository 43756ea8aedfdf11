// Attention of drafted tokens (trees or chains, one to some hundred tokens a request) over the paged bf16 cache, on the 5th-generation
// tensor cores:  o = sum_j e^(s_j) v_j / sum_j e^(s_j),  s_j = sm_scale q.k_j  over the tokens j that the query's token sees.
//
// The rows of an item are those query rows of a request that share a KV head (tokens x group), in blocks of 128 (one slot) or of up to 256
// (two). Every key and value is read once per block, 4 head_dim operations a row for 4 head_dim bytes: the cache's bytes bound it below some
// 250 rows, the products above. In between and beyond, what a tile waits for is what counts: scores, their 2^x (16 a clock and SM: 1024
// clocks for a tile of 256 rows, where both products take 1430 at the measured rate), weights, sums follow one another, and no stage of it
// is ever the only one.
//
// Tiles are of 64 tokens, and a slot has two buffers of scores in tensor memory: the next tile's scores are formed while the softmax goes
// through this one's. Weights (bf16 pairs) go over the scores that they come from and are the second product's A operand from there.
//   One slot:   two CTAs to an SM, of 7 warps: four of softmax (a thread per row), one that copies keys (TMA, page by page into a ring),
//               one that copies values, one of products. A CTA's softmax runs under the other's products.
//   Two slots:  a CTA to an SM, of 12 warps: eight of softmax, the two of copies, one of products for each slot. Up to 128 rows both
//               slots hold the same rows and take turns at the tiles, and their states are joined at the end; up to 256 each has its own
//               rows and both take every tile.
// A product of 128 x 64 x 16 takes as long as one of 128 x 128 x 16 (63 clocks), so that scores run at half the tensor cores' rate; tiles
// of 128 tokens leave room for one buffer of scores only, and cost more than they gain: with the weights over the scores 32 x 64 tokens
// of 512 rows take 470 us against 279, with the weights by way of shared memory 339 (with rings of a tile and a half). Tiles of 64 tokens
// with the weights by way of shared memory, so that nothing has to wait for the place of the scores: 325, since both products then read all
// operands from there. Two threads to a row, 375. What is left is the softmax's own chain, some 2200 clocks a tile for the two warps of a
// scheduler, 1040 of them 2^x: without 2^x the same case takes 12 us less, with half of the scores' products 13, with the cache in the L2
// 10; letting the two warps take turns at 2^x makes it 302.
//
// Work is a row of pages of all requests, KV heads and blocks, cut evenly over the CTAs whatever the requests' lengths; an item that is
// cut leaves a state (reference, sum, sums of values) per piece, which a second kernel joins, in the order of the pieces: results do not
// depend on the order in which anything runs.
//
// Weights are rounded to bf16 (at most 2^-8 of each), the type of the values that they meet in the product. Scores, references, sums and
// states are fp32. Weights are relative to a reference, at first the first tile's largest score (and 2^32, kSpare). The largest score of a
// further tile is looked for only where its weights' sum reaches 2^14 of the first one's largest, and the reference moves (sums are rescaled,
// the tile's weights formed anew) where that score is above it by 2^8 or more: 286 us instead of 296 with a search in every tile.
//
// Measured (32 query and 8 KV heads of 128, a launch of both kernels in a graph): 64 requests of 5 tokens behind up to 4000 68 us (5.3 TB/s),
// 256 single tokens behind up to 2000 146 us (5.9 TB/s), one of 60 behind 100000 116 to 122 us; with 64 query heads 32 of 64 tokens behind
// up to 8000 281 us (0.89 PFLOP/s; for seconds 333, at the power cap and 1590 MHz); one of 26 behind 2000 14.4 us, which is two launches, the
// scan of the lists and a few tiles' way through all of it.
//
// Only tiles with drafted tokens or the end of a piece need care: masks of 64 bits a row; and values that a row does not see must not
// reach it as 0 * inf, so rows of values behind the end become zeros, as do infinities and NaN of drafted tokens, which the rows that do
// see them get back at the end (restore_odd).
#include "attn_mma.cuh"
#include "cache_q8.cuh"
#include "common.cuh"
#include "kernels.h"

namespace nf {
namespace {

constexpr int kTile = 64;             // cached tokens per tile
constexpr int kTilePages = kTile / kPage;
constexpr float kGap = 8.f;           // log2 of how far a row's largest score may outgrow its reference where it is looked for,
// Weights are 2^-kSpare of what they would be: sums of many tokens with values next to bf16's largest stay finite, and a weight is lost
// only where it is 2^-94 of the largest.
constexpr float kSpare = 32.f;
constexpr float kMostWeight = 16384.f / 4294967296.f;        // the sum of a tile's weights from which on it is: 64 weights of 2^kGap
// What an item's beginning and end cost, in pages: where the work is cut, the ends count too. (64 requests of 5 tokens 69.8 us, with 8 pages
// 72.1, with 4 76.7; 24 cost single tokens 1 % and give batches of short contexts 2 to 5.) It is also the least share of a CTA: 1 x 26
// tokens behind 2000 take 14.9 us, with shares of 24 15.9; fewer make more pieces than they save tiles.
constexpr int kLead = 16;

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
template <int HD, int SLOTS>
struct Cfg {
  // warps: four of softmax a slot, one that copies keys, one of products a slot, one that copies values
  static constexpr int kSoftWarps = 4 * SLOTS, kKeyWarp = kSoftWarps, kMmaWarp = kKeyWarp + 1, kValueWarp = kMmaWarp + SLOTS, kThreads = 32 * (kValueWarp + 1);
  static constexpr int NH = HD / 64;
  static constexpr int kQHalf = 128 * 128, kHalf = kTile * 128;        // [128 rows or 64 tokens][64 elements]
  static constexpr int kQ = NH * kQHalf, kStage = NH * kHalf;  // a slot's queries; a tile of keys or of values
  static constexpr int kStages = (HD == 128 ? 2 : 4) * SLOTS;  // tiles of keys, and as many of values (a power of two)
  static constexpr int kRing = SLOTS * kQ;
  static constexpr int kOut = kRing + 2 * kStages * kStage;    // of each softmax warp [32 rows][32 columns] fp32: rows on their way out
  static constexpr int kMl = kOut + kSoftWarps * 4096;         // [2 slots][128] float2; before that, where the CTA begins
  static constexpr int kBars = kMl + (SLOTS == 2 ? 2 * 128 * 8 : 256);
  static constexpr int kBytes = kBars + 640;
  enum Bar : int {
    K_FULL = 0, K_EMPTY = K_FULL + kStages, V_FULL = K_EMPTY + kStages, V_EMPTY = V_FULL + kStages, Q_FULL = V_EMPTY + kStages, Q_EMPTY, READ, O_FREE, LAST,
    CARE = LAST + 2, S_FULL = CARE + 2, P_FULL = S_FULL + 4, PV_DONE = P_FULL + 4, MERGE = PV_DONE + 4, kNum = MERGE + 4   // (S_FULL to PV_DONE: two to a slot, which its tiles use in turn)
  };
  static_assert(kNum * 8 + 20 + sizeof(Piece) <= 640 && SLOTS * kBytes <= SLOTS * 227 * 1024 && (3 - SLOTS) * (kBytes + 1024) <= 228 * 1024, "shared memory");
};

// What a CTA leaves for the kernel that joins states: the item that begins with it and goes on behind it, if there is one.
struct Record {
  int pieces, tok, nodes, kvh;
};

struct Workspace {
  Record* records;   // [CTAs]
  float2* ml;        // [2 CTAs][rows of a block]: reference (of exponents to base 2) and sum
  float* o;          // [2 CTAs][rows of a block][head_dim], not divided by the sum
};
// CTAs at most: two to an SM.
int most_ctas() {
  const int n = 2 * device_sm_count();
  return n < 512 ? n : 512;
}
long long workspace_bytes(int head_dim, Workspace* w = nullptr, void* base = nullptr) {
  const long long n = most_ctas(), records = (n * static_cast<long long>(sizeof(Record)) + 255) / 256 * 256, ml = 2 * n * 128 * 8;
  if (w != nullptr) {
    char* at = static_cast<char*>(base);
    w->records = reinterpret_cast<Record*>(at);
    w->ml = reinterpret_cast<float2*>(at + records);
    w->o = reinterpret_cast<float*>(at + records + ml);
  }
  return records + ml + 2 * n * 128 * head_dim * 4;
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
    const long long most = (t + kLead - 1) / kLead;
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
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* tm, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __noinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, wait_or_abort(bar, parity, abort_flag)) != 0;
}
// bf16 pairs with an infinity or NaN in them
__device__ __forceinline__ bool odd_pair(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }
__device__ __forceinline__ uint32_t without_odd(uint32_t w) {
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
  return w;
}

// fp32 numbers from 2^28 on are 32 and more apart, so that there is nothing but weights of the largest score and none. The exponent of the
// exact product against a rounded reference would be as far off, which 2^x has no room for from 2^31 on: rows with such a reference take
// all at the power of two that brings it to [2^27, 2^28). There it is off by 8, and products q.k that differ in their last bit by 8 or more.
// (What differs less is what fp32 does not tell apart as a score.) One for references below 2^28.
__device__ __forceinline__ float shrink(float ref) {
  const uint32_t e = __float_as_uint(ref) >> 23 & 255u;        // 127 + exponent
  return __uint_as_float((127u - (max(e, 154u) - 154u)) << 23);
}

// Waits, for a while, until *count is `goal`; for a whole warp.
__device__ __forceinline__ bool reached(volatile int* count, int goal, volatile int* abort_flag) {
  bool ok = false;
  for (int it = 0; it < (1 << 22) && !ok && *abort_flag == 0; ++it) ok = *count >= goal;
  __threadfence_block();
  return __all_sync(0xffffffffu, ok) != 0;
}
// Quotients of what fits 32 bits without the long way of 64.
__device__ __forceinline__ long long divide(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<unsigned int>(a) / static_cast<unsigned int>(b);
  return a / b;
}

// Infinities and NaN of the drafted tokens [first, end) that the row sees, in its columns [from, to): as terms of its sums they are what
// they are, whatever their weights, and are added to the row where it has been written. (Only where there are some.)
template <int HD>
__device__ __noinline__ void restore_odd(const nfk_attn_tree_params& p, const int* list, int kvh, const uint32_t* tree, int node, int all, int ctx, int first, int end,
                                         int from, int to, float* sums, __nv_bfloat16* out) {
  for (int t = first; t < end; ++t) {
    if ((seen_bits(tree, 2 * p.words, node, all, t - ctx) & 1u) == 0u) continue;
    int page = list[t / kPage];
    if (page < 0 || page >= p.num_pages) page = 0;               // (as it was read)
    const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(p.kv_pool) + (((static_cast<long long>(page) * 2 + 1) * p.kv_heads + kvh) * kPage + t % kPage) * HD;
    for (int c = from; c < to; ++c) {
      const float x = __bfloat162float(v[c]);
      if (isfinite(x)) continue;
      if (sums != nullptr) __stcg(sums + c, __ldcg(sums + c) + x);
      else out[c] = __float2bfloat16(__bfloat162float(*const_cast<volatile __nv_bfloat16*>(out + c)) + x);
    }
  }
}

template <int HD, int SLOTS>
__global__ void __launch_bounds__(Cfg<HD, SLOTS>::kThreads, 3 - SLOTS)
attn_tree_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmKV,
                 const __grid_constant__ nfk_attn_tree_params p, Workspace ws) {
  using C = Cfg<HD, SLOTS>;
  // Exponents by two to an instruction or by one: the one needs pairs of registers, which cost moves; the same values. (One slot: 128
  // requests of 64 rows 59.6 us by two, 62 by one. Two slots: 32 requests of 512 rows 290 and 279.)
  constexpr bool kInPairs = SLOTS == 1;
  constexpr int NH = C::NH, NST = C::kStages, kKeyWarp = C::kKeyWarp, kMmaWarp = C::kMmaWarp, kValueWarp = C::kValueWarp, kThreads = C::kThreads;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sb = smem_u32(smem);
  float2* ml_s = reinterpret_cast<float2*>(smem + C::kMl);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kNum);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* odd_item = reinterpret_cast<volatile int*>(tmem_slot + 2);         // [2]: numbers of items with odd values
  int* cleared = reinterpret_cast<int*>(tmem_slot + 4);                            // warps of slot 0 that have been through a tile's values
  Piece* piece_s = reinterpret_cast<Piece*>(tmem_slot + 5);
  // (before the roles begin) sums of the warps' units, units in front of the CTA's first request, its number
  long long* scan_s = reinterpret_cast<long long*>(smem + C::kMl);
  long long* start_off_s = scan_s + kThreads / 32;
  Request* start_s = reinterpret_cast<Request*>(start_off_s + 1);
  int* start_req_s = reinterpret_cast<int*>(start_s + 1);
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int group = p.q_heads / p.kv_heads, per_slot = 128 / group, per_block = SLOTS * per_slot;     // tokens of a slot, of a block of rows
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
      const int n = b == C::READ ? C::kSoftWarps + SLOTS : b == C::O_FREE ? C::kSoftWarps : (b >= C::P_FULL && b < C::PV_DONE) ? 4 : b >= C::MERGE ? 2
                    : b == C::Q_EMPTY || (b >= C::K_EMPTY && b < C::V_FULL) || (b >= C::V_EMPTY && b < C::Q_FULL) ? SLOTS : 1;
      mbar_init(&bars[b], n);
    }
    *abort_flag = 0;
    odd_item[0] = odd_item[1] = -1;
    *cleared = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmKV);
  }
  await_previous();                              // (before tensor memory is taken, which the kernel before may need)
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, 256 * SLOTS);                  // of each slot (256 columns): scores in [0, 64) and [64, 128), sums in [128, 128 + HD)
    tmem_relinquish();
  }
  // ---- where this CTA's share of the units begins: units of every thread's requests, scanned ----
  const int per_thread = (p.req_count + kThreads - 1) / kThreads;
  const int r0 = min(p.req_count, static_cast<int>(threadIdx.x) * per_thread), r1 = r0 + min(per_thread, p.req_count - r0);
  long long mine = 0;
  for (int r = r0; r < r1; ++r) mine += units_of(read_request(p, r, per_block, blockIdx.x == 0)) * p.kv_heads;
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
      const Request q = read_request(p, r, per_block, false);
      const long long n = units_of(q) * p.kv_heads;
      if (u0 < at + n) {
        *start_s = q;
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
  Request start = *start_s;
  __syncthreads();
  let_next_start();

  auto fail = [&](unsigned int code) {
    if (lane == 0) report_status(p.status, code);
    *abort_flag = 1;
  };
  const uint32_t bars_at = smem_u32(bars);
  // for a whole warp; most barriers have been passed long before
  auto passed = [&](int bar, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_test(bars_at + bar * 8, parity)) != 0 || wait_for(&bars[bar], parity, abort_flag);
  };
  if (!works || start_req < 0) {
    if (threadIdx.x == 0) ws.records[blockIdx.x] = Record{0, 0, 0, 0};
  } else if (warp == kKeyWarp || warp == kValueWarp) {
    // ------------------------------------------------------------------ copies (a warp walks, an elected lane issues)
    // Keys and values have a warp each, since a tile's eight copies and the wait for its place take most of the time that its bytes do.
    const int part = warp == kKeyWarp ? 0 : 1, full = part == 0 ? C::K_FULL : C::V_FULL, empty = part == 0 ? C::K_EMPTY : C::V_EMPTY;
    uint8_t* const tiles_at = smem + C::kRing + part * (NST * C::kStage);
    Record record{0, 0, 0, 0};
    uint32_t ring = 0, n_item = 0;               // tiles and items so far
    const int no_row = static_cast<int>(min(static_cast<long long>(p.num_pages) * 2 * p.kv_heads * kPage, 0x7fffff00ll));   // behind the pool: zeros
    bool ok = true;
    long long at = start_off;                    // units in front of request r
    for (int r = start_req; ok && r < p.req_count && at < u1; ++r) {
      const Request q = r == start_req ? start : read_request(p, r, per_block, false);
      const long long span = kLead + q.pages, n_items = q.blocks * p.kv_heads;
      for (long long i = u0 > at ? divide(u0 - at, span) : 0; ok && i < n_items; ++i) {
        const long long s = at + i * span;       // the item's first unit
        if (s >= u1) break;
        if (s + span <= u0) continue;
        Piece f;
        f.kvh = static_cast<int>(divide(i, q.blocks));
        f.node = static_cast<int>(i - f.kvh * q.blocks) * per_block;
        f.tok = q.tok + f.node;
        f.nodes = min(per_block, q.n - f.node);
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
          const bool begins = first >= u0, ends = s + span <= u1;
          if (!begins || !ends) f.to = 2 * blockIdx.x + (begins ? 1 : 0);
          if (begins && !ends) record = Record{cut.of(s + span - 1) - static_cast<int>(blockIdx.x) + 1, f.tok, f.nodes, f.kvh};
        }
        const int tiles = (f.pages + kTilePages - 1) / kTilePages;
        const int* list = p.kv_indices + q.list + f.page0;
        // Page numbers of 32 pages (eight tiles) at a time, a lane each.
        int pages = 0;
        auto fetch = [&](int tile) {
          const int j = tile * kTilePages + lane;
          pages = -1;
          if (j < f.pages) {
            pages = list[j];
            if (pages < 0 || pages >= p.num_pages) {
              report_status(p.status, NF_ST_BAD_INDEX);
              pages = 0;
            }
          }
        };
        fetch(0);
        auto issue = [&](int tile) {
          if (tile > 0 && (tile & 7) == 0) fetch(tile);
          const uint32_t at_ring = ring + tile, stage = at_ring % NST;
          int rows[kTilePages];
#pragma unroll
          for (int j = 0; j < kTilePages; ++j) {
            const int page = __shfl_sync(0xffffffffu, pages, (tile & 7) * kTilePages + j);
            rows[j] = page < 0 ? no_row : ((page * 2 + part) * p.kv_heads + f.kvh) * kPage;
          }
          if (!passed(empty + stage, (at_ring / NST & 1) ^ 1)) return false;
          uint8_t* to = tiles_at + stage * C::kStage;
          if (elect_one()) {
            uint64_t* bar = &bars[full + stage];
            mbar_expect_tx(bar, C::kStage);
#pragma unroll
            for (int j = 0; j < kTilePages; ++j)
#pragma unroll
              for (int h = 0; h < NH; ++h) tma_load_2d(to + h * C::kHalf + j * (kPage * 128), &tmKV, bar, h * 64, rows[j]);
          }
          __syncwarp();
          return true;
        };
        int tile = 0;
        if (part == 0) {
          // the first tiles are on their way before the queries, which wait for the item before
          if (n_item > 0)
            for (; ok && tile < min(tiles, NST); ++tile) ok = issue(tile);
          ok = ok && passed(C::READ, (n_item & 1) ^ 1) && passed(C::Q_EMPTY, (n_item & 1) ^ 1);
          if (ok) {
            if (elect_one()) {
              *piece_s = f;
              const int slots = f.two ? 2 : 1;
              mbar_expect_tx(&bars[C::Q_FULL], slots * NH * per_slot * group * 128);
              for (int slot = 0; slot < slots; ++slot)
#pragma unroll
                for (int h = 0; h < NH; ++h)
                  tma_load_3d(smem + slot * C::kQ + h * C::kQHalf, &tmQ, &bars[C::Q_FULL], h * 64, f.kvh * group, f.tok + slot * per_slot);
            }
            __syncwarp();
            ++n_item;
          }
        }
        for (; ok && tile < tiles; ++tile) ok = issue(tile);
        ring += tile;
      }
      at += n_items * span;
    }
    if (!ok) fail(NF_ST_TIMEOUT_SMEM_EMPTY);
    if (part == 0 && lane == 0) ws.records[blockIdx.x] = record;
    if (part == 0 && ok && passed(C::READ, (n_item & 1) ^ 1) && passed(C::Q_EMPTY, (n_item & 1) ^ 1)) {
      if (elect_one()) {                         // no more pieces
        piece_s->nodes = 0;
        mbar_arrive(&bars[C::Q_FULL]);
      }
      __syncwarp();
    } else if (part == 0 && n_item > 0) {
      (void)mbar_wait(&bars[C::Q_FULL], (n_item - 1) & 1);
    }
    // copies still in flight must have landed before the CTA gives its shared memory back
    for (uint32_t k = ring > NST ? ring - NST : 0; k < ring; ++k) (void)mbar_wait(&bars[full + k % NST], k / NST & 1);
  } else if (warp >= kMmaWarp && warp < kValueWarp) {
    // ------------------------------------------------------------------ products (the warp walks, an elected lane issues)
    const uint32_t idesc_s = umma_idesc_bf16(128, kTile), idesc_o = umma_idesc_bf16(128, HD) | kIdescBMnMajor;
    const uint64_t q_desc = umma_desc_k_sw128(sb), k_desc = umma_desc_k_sw128(sb + C::kRing);
    const uint64_t v_desc = umma_desc_mn_sw128(sb + C::kRing + NST * C::kStage, C::kHalf, 1024);
    // A warp per slot: what it spends is not the products but the waits in front of them (some 100 cycles each, also where the barrier has
    // long been passed), and one warp for both took 2600 cycles for a tile of both.
    const int slot = warp - kMmaWarp;
    const uint32_t t_s = tmem + slot * 256, t_o = t_s + 2 * kTile;
    uint32_t ring = 0, n_item = 0, n_tile = 0;   // (tiles of this slot in front of this item)
    int n_cleared = 0;
    bool ok = true;
    for (;;) {
      if (!passed(C::Q_FULL, n_item & 1)) { ok = false; break; }
      const int nodes = piece_s->nodes, pages = piece_s->pages, page0 = piece_s->page0;
      const bool two = SLOTS == 2 && piece_s->two != 0, every = SLOTS == 1 || two;      // whether the slot takes every tile
      const int care_from = min(piece_s->len - piece_s->all, min(piece_s->len, (page0 + pages) * kPage));
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[C::READ]);
      if (nodes == 0) break;
      const int tiles = (pages + kTilePages - 1) / kTilePages;
      const int n = every ? tiles : (tiles + 1 - slot) / 2;
      const uint64_t qd = q_desc + static_cast<uint64_t>((two ? slot : 0) * (C::kQ >> 4));
      // The other slot's tiles pass by: both warps wait for all of a ring's places in their order, since a parity tells only neighbouring
      // phases apart.
      auto pass_by = [&](int full, int empty, int tile) {
        if (every || tile >= tiles) return true;
        const uint32_t at = ring + tile;
        if (!passed(full + at % NST, at / NST & 1)) return false;
        if (lane == 0) mbar_arrive(&bars[empty + at % NST]);
        return true;
      };
      auto other_keys = [&](int i) { return pass_by(C::K_FULL, C::K_EMPTY, 2 * i + (slot ^ 1)); };
      auto other_values = [&](int i) { return pass_by(C::V_FULL, C::V_EMPTY, 2 * i + (slot ^ 1)); };
      // S(i) goes over the weights of the slot's tile before the last one, which that one's second product reads: it must have ended
      auto scores = [&](int i) {
        const uint32_t k = ring + (every ? i : 2 * i + slot), g = n_tile + i, at = slot * 2 + (g & 1);
        if (g >= 2 && !passed(C::PV_DONE + at, ((g >> 1) - 1) & 1)) return false;
        if (!passed(C::K_FULL + k % NST, k / NST & 1)) return false;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t kd = k_desc + static_cast<uint64_t>(k % NST * (C::kStage >> 4));
#pragma unroll
          for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int s = 0; s < 4; ++s)
              umma_bf16_ss(t_s + (g & 1) * kTile, qd + ((h * C::kQHalf + s * 32) >> 4), kd + ((h * C::kHalf + s * 32) >> 4), idesc_s, (h | s) ? 1u : 0u);
          umma_commit(&bars[C::S_FULL + at]);
          umma_commit(&bars[C::K_EMPTY + k % NST]);
          if (i == n - 1) umma_commit(&bars[C::Q_EMPTY]);
        }
        __syncwarp();
        return true;
      };
      auto sums = [&](int i) {
        const int tile = every ? i : 2 * i + slot;
        const uint32_t v = ring + tile, g = n_tile + i, at = slot * 2 + (g & 1);
        // the item before must have been read out of both slots' sums
        if (i == 0 && !passed(C::O_FREE, (n_item & 1) ^ 1)) return false;
        if (!passed(C::V_FULL + v % NST, v / NST & 1)) return false;
        if (page0 * kPage + (tile + 1) * kTile > care_from) {    // the values are gone through first, by slot 0 for both if both have them
          if (!two || slot == 0) {
            if (lane == 0) mbar_arrive(&bars[C::CARE + slot]);
          } else if (!reached(cleared, n_cleared += 4, abort_flag)) {
            return false;
          }
        }
        if (!passed(C::P_FULL + at, g >> 1 & 1)) return false;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t vd = v_desc + static_cast<uint64_t>(v % NST * (C::kStage >> 4));
#pragma unroll
          for (int s = 0; s < kTile / 16; ++s)
            umma_bf16_ts(t_o, t_s + (g & 1) * kTile + s * 8, vd + ((s * 2048) >> 4), idesc_o, (i | s) ? 1u : 0u);
          umma_commit(&bars[C::PV_DONE + at]);
          umma_commit(&bars[C::V_EMPTY + v % NST]);
        }
        __syncwarp();
        return true;
      };
      if (n == 0) {                              // (phases are not skipped: a parity stands for every other one)
        if (lane == 0) mbar_arrive(&bars[C::Q_EMPTY]);
        ok = passed(C::O_FREE, (n_item & 1) ^ 1);
      } else {
        ok = scores(0);
      }
      ok = ok && other_keys(0);
      for (int i = 0; ok && i < (every ? tiles : (tiles + 1) / 2); ++i)
        ok = (i + 1 >= n || scores(i + 1)) && other_keys(i + 1) && (i >= n || sums(i)) && other_values(i);
      if (!ok) break;
      ring += tiles;
      n_tile += n;
      ++n_item;
    }
    if (!ok) {                                   // products in flight get a bounded chance to end before their memory is given back
      fail(NF_ST_TIMEOUT_SMEM_FULL);
      if (elect_one()) umma_commit(&bars[C::LAST + slot]);
      __syncwarp();
      (void)mbar_wait(&bars[C::LAST + slot], 0);
    }
  } else {
    // ------------------------------------------------------------------ softmax (a thread per query row)
    const int slot = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t t_slot = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + slot * 256, t_o = t_slot + 2 * kTile;
    const int in_slot = row / group, hh = row - in_slot * group;
    const float scale = p.sm_scale * kLog2e;
    uint32_t ring = 0, n_item = 0, n_done = 0, n_merge = 0, n_care = 0;
    // States that will not be formed are NaN, and not what an earlier call left in the workspace.
#pragma unroll
    for (int k = 0; k < 2; ++k) __stcg(ws.ml + ((2 * blockIdx.x + k) * SLOTS + slot) * 128 + row, make_float2(0.f, __uint_as_float(0x7fc00000u)));
    for (;;) {
      if (!passed(C::Q_FULL, n_item & 1)) { fail(NF_ST_TIMEOUT_SMEM_FULL); break; }
      const Piece f = *piece_s;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[C::READ]);
      if (f.nodes == 0) break;
      const int tiles = (f.pages + kTilePages - 1) / kTilePages;
      const bool two = SLOTS == 2 && f.two != 0, every = SLOTS == 1 || two;
      const int n_mine = every ? tiles : (tiles + 1 - slot) / 2;
      const int node_in = in_slot + (two ? slot * per_slot : 0);       // of the block
      const bool on = in_slot < per_slot && node_in < f.nodes;
      const bool warp_on = __any_sync(0xffffffffu, on);
      const int node = f.node + node_in, ctx = f.len - f.all;
      const uint32_t* tree = p.tree == nullptr ? nullptr : reinterpret_cast<const uint32_t*>(p.tree + static_cast<long long>(f.tok + (on ? node_in : 0)) * p.words);
      const int end = min(f.len, (f.page0 + f.pages) * kPage);           // of the piece's tokens
      // The exponent of a weight is product * row_scale + less, which are formed where the reference moves (32 x 64 tokens: 3 % more than with
      // one scale for all rows, that is without shrink; with both formed in every tile 4 %, with the difference of two products taken first
      // and the scale behind it 5 %).
      float ref = -INFINITY, l = 0.f, row_scale = scale, less = 0.f;
      auto refer = [&](float to) {
        ref = to;
        const float f = shrink(ref);
        row_scale = scale * f;
        less = ref == -INFINITY ? 0.f : fmaf(-ref, f, kSpare * f - kSpare);
      };
      bool sees = false, ok = true;
      for (int i = 0; i < n_mine; ++i) {
        const int tile = every ? i : 2 * i + slot;
        const int at = f.page0 * kPage + tile * kTile;                   // the tile's first token
        const bool care = at + kTile > min(ctx, end);
        uint32_t bits[2] = {~0u, ~0u};
        if (care) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int left = end - (at + k * 32);
            bits[k] = on ? seen_bits(tree, 2 * p.words, node, f.all, at + k * 32 - ctx) & (left >= 32 ? ~0u : left > 0 ? (1u << left) - 1u : 0u) : 0u;
          }
        }
        const int b = slot * 2 + (n_done & 1);
        const uint32_t t_s = t_slot + (n_done & 1) * kTile;
        if (!passed(C::S_FULL + b, n_done >> 1 & 1)) { ok = false; break; }
        if (care && (!two || slot == 0)) {
          // ---- values of the tile: two threads per token ----
          // (by way of the warp that waits for all of the ring's places in their order)
          const uint32_t v = ring + tile;
          if (!passed(C::CARE + slot, n_care & 1) || !passed(C::V_FULL + v % NST, v / NST & 1)) { ok = false; break; }
          ++n_care;
          const int in_tile = row & (kTile - 1), token = at + in_tile;
          if (token >= ctx) {
            const uint32_t v_row = sb + C::kRing + NST * C::kStage + v % NST * C::kStage + in_tile * 128;
            bool odd = false;
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
              const int c = (row / kTile) * (HD / 16) + k;
              const uint32_t a = v_row + (c >> 3) * C::kHalf + (((c & 7) ^ (in_tile & 7)) << 4);
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
          if (two && lane == 0) {
            __threadfence_block();
            atomicAdd(cleared, 1);
          }
        }
        if (warp_on) {
          tc_fence_after();
          uint32_t x[2][32];
          tmem_ld_32x32b_x32(t_s, x[0]);
          tmem_ld_32x32b_x32(t_s + 32, x[1]);
          tmem_ld_wait();
          if (care) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              sees = sees || bits[c] != 0u;
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if ((bits[c] >> j & 1u) == 0u) x[c][j] = 0xff800000u;    // -inf
            }
          } else {
            sees = true;
          }
          auto largest = [&]() {                 // as a reference
            float mq[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // (NaN where there is one)
#pragma unroll
            for (int j = 0; j < 32; ++j)
              mq[j & 3] = max3_nan(mq[j & 3], __uint_as_float(x[j >> 4][2 * (j & 15)]), __uint_as_float(x[j >> 4][2 * (j & 15) + 1]));
            const float mx = max3_nan(max3_nan(mq[0], mq[1], mq[2]), mq[3], mq[3]) * scale;
            if (mx < INFINITY) return mx + kSpare;
            l = __uint_as_float(0x7fc00000u);    // a score of infinity, or none
            return 0.f;
          };
          if (i == 0) refer(largest());
          // Weights relative to the reference as it is. Only where their sum says that it has been left far behind (or that there is none
          // yet, or a NaN) is the largest score looked for, and the weights are formed once more.
          float sum;
          for (bool again = false;; again = true) {
            const f32x2 by2 = pair(row_scale, row_scale), ms2 = pair(less, less);
            f32x2 rs[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t pk[16];                   // column j: tokens 2j, 2j + 1
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const float x0 = __uint_as_float(x[h][2 * j]), x1 = __uint_as_float(x[h][2 * j + 1]);
                const float2 y = kInPairs ? halves(fma2(pair(x0, x1), by2, ms2)) : make_float2(fmaf(x0, row_scale, less), fmaf(x1, row_scale, less));
                const float e0 = fast_exp2(y.x), e1 = fast_exp2(y.y);
                rs[j & 1] = add2(rs[j & 1], pair(e0, e1));
                pk[j] = pack_bf16x2(e0, e1);
              }
              tmem_st_32x32b_x16(t_s + 16 * h, pk);
            }
            const float2 both = halves(add2(rs[0], rs[1]));
            sum = both.x + both.y;
            const bool look = on && (!(sum < kMostWeight) || ref == -INFINITY);
            if (again || !__any_sync(0xffffffffu, look)) break;
            const float mx = largest();
            const bool grow = mx > ref + kGap || (ref == -INFINITY && mx > -INFINITY);
            if (i == 0 || !__any_sync(0xffffffffu, grow)) break;
            // Sums may be touched between two products only: that of the tile before is the last one issued (this tile's needs its weights)
            if (!passed(C::PV_DONE + slot * 2 + ((n_done - 1) & 1), (n_done - 1) >> 1 & 1)) { ok = false; break; }
            tc_fence_after();
            const float alpha = grow ? (ref == -INFINITY ? 0.f : fast_exp2(ref - mx)) : 1.f;
#pragma unroll 1
            for (int c = 0; c < HD / 16; ++c) {
              uint32_t o[16];
              tmem_ld_32x32b_x16n(t_o + c * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
              tmem_st_32x32b_x16(t_o + c * 16, o);
            }
            l *= alpha;
            if (grow) refer(mx);
            tmem_st_wait();                      // (the weights go over those of the first pass: two stores have no order of their own)
          }
          if (!ok) break;
          l += sum;
          tmem_st_wait();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[C::P_FULL + b]);
        ++n_done;
      }
      if (!ok) { fail(NF_ST_TIMEOUT_TMEM_FULL); break; }
      ring += tiles;
      if (n_mine > 0 && !passed(C::PV_DONE + slot * 2 + ((n_done - 1) & 1), (n_done - 1) >> 1 & 1)) { fail(NF_ST_TIMEOUT_TMEM_FULL); break; }
      tc_fence_after();
      if (sees && l == 0.f) l = __uint_as_float(0x7fc00000u);            // all that it sees has a score of minus infinity
      // ---- sums of the row: columns [from, to), a0 times those of slot 0 and a1 times those of slot 1 ----
      float a_mine = 1.f, a_other = 0.f;
      int from = 0, to = HD;
      if (!every) {
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
        } else {                                 // (a sum of NaN counts whatever its weight, but for a slot without weights)
          a_mine = ref == -INFINITY ? 0.f : fast_exp2(ref - top);
          a_other = other.x == -INFINITY ? 0.f : fast_exp2(other.x - top);
          l = (ref == -INFINITY ? 0.f : a_mine * l) + (other.x == -INFINITY ? 0.f : a_other * other.y);
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
      // (in steps of eight elements: row strides are multiples of that)
      const int out_row = static_cast<int>((static_cast<long long>(f.tok + node_in) * p.ld_out + (f.kvh * group + hh) * HD) >> 3);
      if (warp_on) {
        const bool use_mine = a_mine != 0.f, use_other = a_other != 0.f;
        const int rows_on = min(per_slot, f.nodes - (two ? slot * per_slot : 0)) * group - (warp & 3) * 32;   // of this warp
        float* o_rows = ws.o + ((static_cast<long long>(f.to) * SLOTS + (two ? slot : 0)) * 128 + (warp & 3) * 32) * HD;
        // A thread has its own row; by way of shared memory, so that a store is of 128 (or, in bf16, 64) bytes of some rows at once. In few
        // instructions, which an item meets for the first time.
        const float times = f.to < 0 ? by : 1.f;
        const uint32_t via = sb + C::kOut + warp * 4096;
#pragma unroll 1
        for (int c = from; c < to; c += 32) {
          uint32_t a[32], other[32];
          tmem_ld_32x32b_x32(t_o + c, a);
          if (!every) tmem_ld_32x32b_x32((t_o ^ 256u) + c, other);
          tmem_ld_wait();
          __syncwarp();                          // (the columns before have been read)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
              o[j] = __float_as_uint(((use_mine ? a_mine * __uint_as_float(a[4 * k + j]) : 0.f) + (use_other ? a_other * __uint_as_float(other[4 * k + j]) : 0.f)) * times);
            st_shared_v4(via + lane * 128 + ((k ^ (lane & 7)) << 4), make_uint4(o[0], o[1], o[2], o[3]));
          }
          __syncwarp();
          if (f.to < 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = i * 8 + (lane >> 2), j = 2 * (lane & 3);
              const int at = __shfl_sync(0xffffffffu, out_row, r);
              const uint4 lo = ld_shared_v4(via + r * 128 + ((j ^ (r & 7)) << 4)), hi = ld_shared_v4(via + r * 128 + (((j + 1) ^ (r & 7)) << 4));
              if (r < rows_on)
                static_cast<uint4*>(p.out)[static_cast<long long>(static_cast<unsigned int>(at)) + c / 8 + j / 2] =
                    make_uint4(pack_bf16x2(__uint_as_float(lo.x), __uint_as_float(lo.y)), pack_bf16x2(__uint_as_float(lo.z), __uint_as_float(lo.w)),
                               pack_bf16x2(__uint_as_float(hi.x), __uint_as_float(hi.y)), pack_bf16x2(__uint_as_float(hi.z), __uint_as_float(hi.w)));
            }
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = i * 4 + (lane >> 3), j = lane & 7;
              const uint4 w = ld_shared_v4(via + r * 128 + ((j ^ (r & 7)) << 4));
              if (r < rows_on) __stcg(reinterpret_cast<uint4*>(o_rows + r * HD + c) + j, w);
            }
          }
        }
        if (__any_sync(0xffffffffu, odd)) {
          __syncwarp();
          if (on)
            restore_odd<HD>(p, p.kv_indices + f.list, f.kvh, tree, node, f.all, ctx, max(f.page0 * kPage, ctx), end, from, to,
                            f.to < 0 ? nullptr : o_rows + lane * HD,
                            static_cast<__nv_bfloat16*>(p.out) + static_cast<long long>(static_cast<unsigned int>(out_row)) * 8);
        }
        if (on && f.to >= 0 && (every || slot == 0)) __stcg(ws.ml + (static_cast<long long>(f.to) * SLOTS + (two ? slot : 0)) * 128 + row, make_float2(ref, l));
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
    tmem_dealloc(tmem, 256 * SLOTS);
  }
}

// Rows of items that were cut: LANES lanes each, over its pieces for the weights and over head_dim, a float4 or two a lane, for the sums.
// Three CTAs to an SM: with four, at 64 registers, rows on their way spill (1 request of 26 tokens behind 2000 15.4 us and 16.0, 32 x 64 281 and
// 284, 64 x 128 rows 84.7 and 86.4).
constexpr int kJoinWarps = 8, kJoinPerSm = 3, kMostCtas = 2 * kJoinWarps * 32;
template <int HD, int SLOTS, int LANES, int AHEAD>         // AHEAD: pieces on their way at once
__device__ __forceinline__ void join_rows(const nfk_attn_tree_params& p, const Workspace& ws, const int4* record_s, const int* rows_s, int total, int warp, int lane) {
  constexpr int V = HD / 4 / LANES, ROWS = 32 / LANES;
  const int sub = lane & (LANES - 1), group = p.q_heads / p.kv_heads, per_slot = 128 / group;
  for (int first = (blockIdx.x * kJoinWarps + warp) * ROWS; first < total; first += gridDim.x * kJoinWarps * ROWS) {
    const int work = min(first + lane / LANES, total - 1);       // (the last row again, where there are no others beside it)
    int c = 0;                                   // the last record with rows_s <= work
#pragma unroll
    for (int step = kMostCtas / 2; step > 0; step >>= 1)
      if (rows_s[c + step] <= work) c += step;
    const int pieces = record_s[c].x, tok = record_s[c].y, kvh = record_s[c].w;
    int most = pieces;
#pragma unroll
    for (int o = 16; o >= LANES; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    const int b = work - rows_s[c], node = b / group, hh = b - node * group, slot = node / per_slot;
    const int row = slot * 128 + (node - slot * per_slot) * group + hh;
    auto number = [&](int k) { return static_cast<long long>(k == 0 ? 2 * c + 1 : 2 * (c + k)) * (128 * SLOTS) + row; };
    float4 x[AHEAD][V];
    auto load = [&](int k0) {
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (k0 + k < pieces)
#pragma unroll
          for (int v = 0; v < V; ++v) x[k][v] = __ldcg(reinterpret_cast<const float4*>(ws.o + number(k0 + k) * HD) + v * LANES + sub);
    };
    load(0);
    float2 ml = make_float2(-INFINITY, 0.f);     // the first pieces', one a lane
    if (sub < pieces) ml = __ldcg(ws.ml + number(sub));
    float top = ml.x, odd = ml.y != ml.y ? ml.y : 0.f;
    for (int k = LANES + sub; k < pieces; k += LANES) {
      const float2 far = __ldcg(ws.ml + number(k));
      top = fmaxf(top, far.x);
      if (far.y != far.y) odd = far.y;
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float total_l = 0.f;
    float4 acc[V];
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = 0; k0 < most; k0 += LANES) {
      if (k0 > 0) ml = k0 + sub < pieces ? __ldcg(ws.ml + number(k0 + sub)) : make_float2(-INFINITY, 0.f);
      const float w = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - top);
      total_l += ml.x == -INFINITY ? 0.f : w * ml.y;             // (a sum of NaN counts whatever its weight)
      for (int k1 = k0; k1 < min(k0 + LANES, most); k1 += AHEAD) {
        if (k1 > 0) load(k1);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          const float by = __shfl_sync(0xffffffffu, w, (lane & ~(LANES - 1)) | ((k1 + k) & (LANES - 1)));
          if (by != 0.f)                         // (zero behind the last piece)
#pragma unroll
            for (int v = 0; v < V; ++v) {
              acc[v].x += by * x[k][v].x;
              acc[v].y += by * x[k][v].y;
              acc[v].z += by * x[k][v].z;
              acc[v].w += by * x[k][v].w;
            }
        }
      }
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
      total_l += __shfl_xor_sync(0xffffffffu, total_l, o);
      odd += __shfl_xor_sync(0xffffffffu, odd, o);
    }
    // without weights: zeros, or NaN where the row sees something
    const float by = total_l > 0.f ? 1.f / total_l : total_l + (top == -INFINITY ? odd : 0.f);
    uint2* dst = reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + static_cast<long long>(tok + node) * p.ld_out + (kvh * group + hh) * HD);
#pragma unroll
    for (int v = 0; v < V; ++v)
      dst[v * LANES + sub] = make_uint2(pack_bf16x2(acc[v].x * by, acc[v].y * by), pack_bf16x2(acc[v].z * by, acc[v].w * by));
  }
}
// Every CTA works out from all records which rows there are.
template <int HD, int SLOTS>
__global__ void __launch_bounds__(kJoinWarps * 32, kJoinPerSm) attn_tree_join_kernel(const __grid_constant__ nfk_attn_tree_params p, Workspace ws, int ctas) {
  __shared__ int4 record_s[kMostCtas];
  __shared__ int rows_s[kMostCtas], warp_s[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = p.q_heads / p.kv_heads;
  await_previous();
  let_next_start();
  // ---- rows in front of each record ----
  int4 rec[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int c = 2 * threadIdx.x + k;
    rec[k] = c < ctas ? __ldcg(reinterpret_cast<const int4*>(ws.records + c)) : make_int4(0, 0, 0, 0);
  }
  const int mine0 = rec[0].x > 0 ? rec[0].z * group : 0, mine = mine0 + (rec[1].x > 0 ? rec[1].z * group : 0);
  int sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += v;
  }
  if (lane == 31) warp_s[warp] = sum;
  __syncthreads();
  int before = sum - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) {
    if (w < warp) before += warp_s[w];
    total += warp_s[w];
  }
  record_s[2 * threadIdx.x] = rec[0];
  record_s[2 * threadIdx.x + 1] = rec[1];
  rows_s[2 * threadIdx.x] = before;
  rows_s[2 * threadIdx.x + 1] = before + mine0;
  __syncthreads();
  // few rows of many pieces, or many of few: a lane's loads are latency's in the one case, throughput's in the other
  if (total <= static_cast<int>(gridDim.x) * kJoinWarps) join_rows<HD, SLOTS, HD / 4, 8>(p, ws, record_s, rows_s, total, warp, lane);
  else join_rows<HD, SLOTS, HD / 8, 4>(p, ws, record_s, rows_s, total, warp, lane);
}

int encode(CUtensorMap* out, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
  const nf_encode_tiled_fn enc = get_encode_tiled();
  if (enc == nullptr) return NF_ERR_CUDA;
  const cuuint32_t ones[3] = {1, 1, 1};
  return enc(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? NF_OK : NF_ERR_CUDA;
}

template <int HD, int SLOTS>
int launch(const nfk_attn_tree_params& p, cudaStream_t stream) {
  using C = Cfg<HD, SLOTS>;
  const auto kernel = attn_tree_kernel<HD, SLOTS>;
  static bool attr_dev[kMaxDevices] = {false};
  bool& attr = attr_dev[device_slot()];
  if (!attr) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kBytes) != cudaSuccess) {
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
  const int sms = most_ctas() / 2, most = sms * (3 - SLOTS), ctas = p.num_ctas > 0 && p.num_ctas < most ? p.num_ctas : most;
  int joins = sms * kJoinPerSm;
  if (p.num_ctas > 0 && p.num_ctas < joins) joins = p.num_ctas;
  if (launch_kernel(early_first(p.early_start), kernel, ctas, C::kThreads, C::kBytes, stream, 1, tm_q, tm_kv, p, ws) != cudaSuccess ||
      launch_kernel(early_further(p.early_start), attn_tree_join_kernel<HD, SLOTS>, joins, kJoinWarps * 32, 0, stream, 1, p, ws, ctas) != cudaSuccess) {
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
  if (p == nullptr || p->req_count < 0 || p->req_count > NFK_DRAFT_ENTRIES || p->num_tokens > NFK_DRAFT_ENTRIES || p->req_begin < 0 || p->num_ctas < 0)
    return NF_ERR_BAD_ARG;
  if ((p->head_dim != 64 && p->head_dim != 128) || p->kv_heads <= 0 || p->q_heads <= 0 || p->q_heads % p->kv_heads != 0 || p->q_heads / p->kv_heads > 128)
    return NF_ERR_UNSUPPORTED;
  if (p->req_count == 0 || p->num_tokens == 0) return NF_OK;
  const auto off = [](const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) != 0; };
  const long long row = static_cast<long long>(p->q_heads) * p->head_dim;
  if (!p->q || !p->out || !p->kv_pool || !p->qo_indptr || !p->kv_indptr || !p->kv_indices || !p->kv_last_page_len || !p->workspace || off(p->q) ||
      off(p->out) || off(p->kv_pool) || (reinterpret_cast<uintptr_t>(p->workspace) & 255) != 0 || (reinterpret_cast<uintptr_t>(p->tree) & 7) != 0)
    return NF_ERR_BAD_ARG;
  if (p->num_tokens < 0 || p->request_tokens < 0 || p->listed < 0 || p->num_pages <= 0 || p->num_indices < 0 || p->ld_q % 8 != 0 ||
      p->ld_out % 8 != 0 || p->ld_q < row || p->ld_out < row ||
      p->req_begin > 0x7fffffff - p->req_count || !(p->sm_scale > 0.f) || p->sm_scale > 2e38f ||
      p->ld_q > (1ll << 38) || p->ld_out / 8 > 0xffffffffll / p->num_tokens ||             // (places of output rows: 16 bytes each, in 32 bits)
      p->workspace_bytes < workspace_bytes(p->head_dim) ||
      (p->tree != nullptr && (p->words < 1 || p->words > NFK_TREE_NODES / 64)) ||
      static_cast<long long>(p->num_pages) * 2 * p->kv_heads * kPage > 0x7fff0000ll)
    return NF_ERR_BAD_ARG;
  // 128 elements a head: two slots to a CTA where requests have more than 128 rows (by request_tokens; without it on average, in which rows of
  // q that are no request's count as well), since both take every tile that has been read: 32 requests of 64 tokens, 512 rows each, 279 us, by
  // two CTAs of a slot 317; one of 240 rows behind 100000 tokens 115 and 143; 8 of 160 rows behind 6000 64.5 and 67.5. Short contexts are the
  // other way, 128 of 200 rows behind 350 118 and 114, and so are few rows, 128 requests of 20 rows behind 500 77 and 61, 256 of four behind
  // 1000 190 and 175. 64 elements: always one slot, as its tiles are half as much to read and two CTAs wait less for one another than two
  // slots (64 requests of 256 rows: 119 us against 135; 32 of 512: 211 and 243; one of 240 behind 100000: 92 and 107).
  const long long tokens = p->request_tokens > 0 ? p->request_tokens : p->num_tokens;
  const long long requests = p->request_tokens > 0 ? 1 : p->listed > 0 ? p->listed : p->req_count;
  const bool wide = tokens * (p->q_heads / p->kv_heads) > 128 * requests;
  if (p->head_dim == 64) return launch<64, 1>(*p, stream);
  return wide ? launch<128, 2>(*p, stream) : launch<128, 1>(*p, stream);
}
