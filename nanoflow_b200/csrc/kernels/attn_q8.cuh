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

__host__ __device__ __forceinline__ long long range_begin(long long w, long long units, long long workers) { return w * units / workers; }
// The worker whose range holds unit u (each has at least one: workers <= units).
__host__ __device__ __forceinline__ long long range_of(long long u, long long units, long long workers) {
  return ((u + 1) * workers + units - 1) / units - 1;
}

// The shared prefix: the query rows of a KV head (requests x group) are cut into blocks of at most 128 rows, whole requests each.
// An item is (KV head, block), its units the prefix's tiles of 64 tokens. The piece of item i by CTA c has number i + c: along
// the row of units every new piece raises one of the two.
constexpr int kPrefixTile = 64, kPrefixRows = 128;
struct PrefixPlan {
  int reqs_per_block, blocks, tiles, ctas;
  const float* o;            // [pieces][128 rows][head_dim], not divided by the sum
  const float* ml;           // [pieces][128 rows][2]: reference (of exponents to base 2), sum
};
__host__ __device__ __forceinline__ long long prefix_units(const PrefixPlan& f, int kv_heads) {
  return static_cast<long long>(kv_heads) * f.blocks * f.tiles;
}

// Where things lie in the workspace, in this order: counts and partial rows of the decode kernel's CTAs, then the prefix's.
constexpr int kDecodeCtasPerSm = 4;      // at most
struct Q8Workspace {
  long long counts, ml, o, prefix_ml, prefix_o, bytes;
};
inline Q8Workspace q8_workspace(int group, int head_dim, long long prefix_pieces) {
  Q8Workspace w;
  const long long ctas = static_cast<long long>(kDecodeCtasPerSm) * device_sm_count();
  const auto up = [](long long x) { return (x + 255) / 256 * 256; };
  w.counts = 0;
  w.ml = up(ctas * 4);
  w.o = w.ml + up(ctas * 2 * group * 8);
  w.prefix_ml = w.o + up(ctas * 2 * group * head_dim * 4ll);
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
