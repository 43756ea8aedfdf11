// What the two kernels of attention over the 8-bit cache share: how work is cut, and where partial results lie.
//
// Both walk a row of equal units (pages, or tiles of the shared prefix) that is cut into ranges of equal length, give or take a unit
// (Ranges), without regard to where a request ends. What a range holds of a request (or of a block of query rows) is a piece, and
// pieces are joined by their softmax states.
#pragma once
#include "cache_q8.cuh"

namespace nf {

constexpr int kQ8Page = 16;
constexpr float kQ8Log2e = 1.4426950408889634f;
// States hold their sums of values times this, 2^-32: up to 2^32 weights of 1 on the largest values of bf16 stay finite, and values from
// 2^-80 on (smaller ones are not cached) keep their bits.
constexpr float kStateUnit = 2.3283064365386963e-10f;

// A row of n units in w ranges (w <= n): the first n % w ranges have one more than the others.
struct Ranges {
  int per, extra;
  Ranges() = default;
  __host__ __device__ __forceinline__ Ranges(int n, int w) : per(w > 0 ? n / w : 0), extra(n - per * w) {}
  __host__ __device__ __forceinline__ int begin(int w) const { return w * per + (w < extra ? w : extra); }
  __host__ __device__ __forceinline__ int of(int u) const {             // the range that holds unit u
    const unsigned int longer = static_cast<unsigned int>(extra) * (per + 1u), v = u;
    const bool in_longer = v < longer;
    return static_cast<int>((in_longer ? v : v - longer) / (in_longer ? per + 1u : static_cast<unsigned int>(per)) + (in_longer ? 0u : extra));
  }
};

// The shared prefix: the query rows of a KV head (requests x group) are cut into blocks of at most `rows` (128 or 256) rows, whole
// requests each. An item is (KV head, block), its units `lead` units for its beginning and then the prefix's tiles of 64 tokens. The
// piece of item i by CTA c has number i + c: along the row of units every new piece raises one of the two.
constexpr int kPrefixTile = 64;
struct PrefixPlan {
  int rows, reqs_per_block, blocks, tiles, lead, ctas;
  int most_ctas;             // that this prefix or a part of it is cut over
  Ranges cut;                // of the units
  float* ml;                 // states, [pieces][rows]: reference (of exponents to base 2) and sum,
  float* o;                  // [pieces][rows][head_dim], times kStateUnit, not divided by the sum
};

// A CTA's share of the units, one item after the other.
struct Share {
  int u, end, lead, tiles, blocks;
  int item, kvh, block, t0, n;         // the current part: tiles t0 .. t0 + n - 1 of item (kvh, block)
  __host__ __device__ __forceinline__ Share(const PrefixPlan& f, int cta) : lead(f.lead), tiles(f.tiles), blocks(f.blocks) {
    u = f.cut.begin(cta);
    end = f.cut.begin(cta + 1);
  }
  __host__ __device__ __forceinline__ bool next() {
    while (u < end) {
      const int span = lead + tiles, from = (item = u / span) * span, to = end - from < span ? end - from : span;
      t0 = u - from > lead ? u - from - lead : 0;
      n = to - lead - t0;
      u = from + to;
      if (n <= 0) continue;                                      // no more than the item's beginning
      kvh = item / blocks;
      block = item - kvh * blocks;
      return true;
    }
    return false;
  }
  // f(item) for the current part and those that would follow
  template <class F>
  __host__ __device__ __forceinline__ void rest(F f) {
    do f(item);
    while (next());
  }
};

// The row of pages of the decode kernel is cut into a range for each of its warps, of two pages at least.
constexpr int kDecodeCtasPerSm = 4, kDecodeWarps = 4;      // at most, of so many warps
__host__ __device__ __forceinline__ int decode_ranges(int units, int ctas) {
  const int most = ctas * kDecodeWarps, useful = (units + 1) / 2;
  return useful < most ? useful : most;
}
// What a range leaves for the kernel that joins states: the request that begins in it and goes on behind it, if there is one.
struct DecodeRecord {
  int kvh, r, tok, n;        // n: ranges that hold parts of it; 0: no such request
};

// Where things lie in the workspace: a word that says whether the page lists are none, a record for each range, states of the
// decode kernel's pieces (two a range), of whole requests that wait for the prefix's share, and the prefix's.
struct Q8Workspace {
  long long records, ml, o, whole_ml, whole_o, prefix_ml, prefix_o, bytes;
};
inline Q8Workspace q8_workspace(const nfk_attn_q8_params& p, const PrefixPlan& f) {
  Q8Workspace w;
  const int group = p.q_heads / p.kv_heads;
  const long long ranges = static_cast<long long>(kDecodeCtasPerSm) * kDecodeWarps * device_sm_count(), pieces = 2 * ranges * group;
  const long long whole = p.prefix_len > 0 ? static_cast<long long>(p.req_count) * p.q_heads : 0;
  const long long prefix = (static_cast<long long>(p.kv_heads) * f.blocks + f.ctas) * f.rows;
  const auto up = [](long long x) { return (x + 255) / 256 * 256; };
  w.records = 256;
  w.ml = w.records + up(ranges * static_cast<long long>(sizeof(DecodeRecord)));
  w.o = w.ml + up(pieces * 8);
  w.whole_ml = w.o + up(pieces * p.head_dim * 4);
  w.whole_o = w.whole_ml + up(whole * 8);
  w.prefix_ml = w.whole_o + up(whole * p.head_dim * 4);
  w.prefix_o = w.prefix_ml + up(prefix * 8);
  w.bytes = w.prefix_o + prefix * p.head_dim * 4;
  return w;
}
PrefixPlan prefix_plan(const nfk_attn_q8_params& p);
int launch_prefix_q8(const nfk_attn_q8_params& p, const PrefixPlan& f, cudaStream_t stream);

#ifdef __CUDACC__
__device__ __forceinline__ float q8_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
#endif

}  // namespace nf
