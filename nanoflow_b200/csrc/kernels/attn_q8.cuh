// What the two kernels of attention over the 8-bit cache share: how work is cut, and where partial results lie.
//
// Both walk a row of equal units (pages, or tiles of the shared prefix) that is cut into equal ranges without regard to where a
// request ends: worker w of W takes units [w U / W, (w + 1) U / W). What a range holds of a request (or of a block of query rows)
// is a piece, and pieces are joined by their softmax states.
#pragma once
#include "cache_q8.cuh"

namespace nf {

constexpr int kQ8Page = 16;
constexpr float kQ8Log2e = 1.4426950408889634f;

// A row of n units in w ranges (w <= n): the first n % w ranges have one more than the others.
struct Ranges {
  int per, extra;
  __host__ __device__ __forceinline__ Ranges(int n, int w) : per(w > 0 ? n / w : 0), extra(n - per * w) {}
  __host__ __device__ __forceinline__ int begin(int w) const { return w * per + (w < extra ? w : extra); }
  __host__ __device__ __forceinline__ int of(int u) const {             // the range that holds unit u
    const int longer = extra * (per + 1);
    return u < longer ? u / (per + 1) : extra + (u - longer) / per;
  }
};

// The shared prefix: the query rows of a KV head (requests x group) are cut into blocks of at most 128 rows, whole requests each.
// An item is (KV head, block), its units the prefix's tiles of 64 tokens. The piece of item i by CTA c has number i + c: along
// the row of units every new piece raises one of the two.
constexpr int kPrefixTile = 64, kPrefixRows = 128;
struct PrefixPlan {
  int reqs_per_block, blocks, tiles, ctas;
  const float* o;            // [pieces][128 rows][head_dim], not divided by the sum
  const float* ml;           // [pieces][128 rows][2]: reference (of exponents to base 2), sum
};
__host__ __device__ __forceinline__ int prefix_units(const PrefixPlan& f, int kv_heads) { return kv_heads * f.blocks * f.tiles; }

constexpr int kDecodeCtasPerSm = 4, kDecodeWarps = 4;      // of the decode kernel: at most, of so many warps

// Where things lie in the workspace, in this order: counts of pieces that have been left, partial rows of the decode kernel's CTAs
// (two requests each), rows that its warps keep (two requests each), the prefix's pieces.
struct Q8Workspace {
  long long counts, ml, o, kept, prefix_ml, prefix_o, bytes;
};
inline Q8Workspace q8_workspace(int group, int head_dim, long long prefix_pieces) {
  Q8Workspace w;
  const long long ctas = static_cast<long long>(kDecodeCtasPerSm) * device_sm_count();
  const auto up = [](long long x) { return (x + 255) / 256 * 256; };
  w.counts = 0;
  w.ml = up(ctas * 4);
  w.o = w.ml + up(ctas * 2 * group * 8);
  w.kept = w.o + up(ctas * 2 * group * head_dim * 4ll);
  w.prefix_ml = w.kept + up(2 * ctas * kDecodeWarps * group * (head_dim + 2) * 4ll);
  w.prefix_o = w.prefix_ml + up(prefix_pieces * kPrefixRows * 8);
  w.bytes = w.prefix_o + prefix_pieces * kPrefixRows * head_dim * 4;
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
