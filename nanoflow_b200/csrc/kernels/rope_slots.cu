// Rotary positions in all their layouts, and the write of keys and values into the tokens' slots of the paged cache.
//
//   (x, y) -> f (x c - y s, y c + x s),  c, s = cos, sin(pos w_i),  (x, y) = (x_i, x_(i + pairs)) or (x_2i, x_(2i+1)),  i < pairs;
// what lies behind the first 2 pairs elements of a head stays as it is, as do values. All in fp32 from the bf16 inputs, rounded once.
// Memory-bound: every element is read once and written once. In a graph, heads of 128: 8192 tokens of 32 query and 8 KV heads 36.2 us
// (201 MB, 5.6 TB/s; floor 30.8), any number of pairs 54, by way of shared memory for each element's partner; 1215 tokens of 64 and 8 heads
// 12.3 (floor 7.6: a token's CTA has a chain of position, angles and two batches of heads to itself, and 1215 of them are 31 more than fit
// the SMs at once); 26 tokens 2.7.
#include "cache_q8.cuh"
#include "common.cuh"
#include "kernels.h"

namespace nf {
namespace {

constexpr int kPage = 16;
constexpr int kThreads = 128;

// cos and sin of pos * w. The product is formed in 64 bits and brought to one turn there: in fp32 the angle of position 100000
// would be off by 0.004.
__device__ __forceinline__ float2 turn(int pos, float w, float factor) {
  const double t = static_cast<double>(pos) * static_cast<double>(w) * 0.15915494309189533577;
  float s, c;
  sincospif(2.f * static_cast<float>(t - rint(t)), &s, &c);
  return make_float2(c * factor, s * factor);
}
// Two neighbouring elements of a word, and back.
__device__ __forceinline__ float2 elements(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

// Which elements a thread's two vectors of eight hold: HALVES the two of its eight pairs (pairs a multiple of eight), NEIGHBOURS and
// SCATTERED 16 elements in a row; SCATTERED (half layout, any number of pairs) finds each element's partner in shared memory.
enum { HALVES, NEIGHBOURS, SCATTERED };

// A CTA per token, HD / 16 threads per head, the same elements of each head that they take, so that their cosines and sines stay in
// registers. Three heads a thread are requested before the token's angles are worked out; what hides their latency beyond that is the
// number of CTAs, of which 64 registers let eight share an SM.
template <int HD, int LAYOUT>
__global__ void __launch_bounds__(kThreads, 8) rope_slots_kernel(const __grid_constant__ nfk_rope_slots_params p) {
  constexpr int LPH = HD / 16, AT_ONCE = kThreads / LPH, BATCH = 3;
  __shared__ __align__(16) float cosines[HD / 2], sines[HD / 2];
  __shared__ __align__(16) __nv_bfloat16 raw[LAYOUT == SCATTERED ? AT_ONCE : 1][HD];     // of the heads at hand
  const int l = threadIdx.x % LPH, h0 = threadIdx.x / LPH, t = blockIdx.x, rot = 2 * p.pairs;
  const int heads = p.q_heads + 2 * p.kv_heads;
  const bool apart = LAYOUT == HALVES && 16 * l < rot;
  const int ea = apart ? 8 * l : 16 * l, eb = apart ? 8 * l + p.pairs : 16 * l + 8;
  const __nv_bfloat16* row = static_cast<const __nv_bfloat16*>(p.qkv) + t * p.ld_qkv;
  auto source = [&](int h) {
    return row + (h < p.q_heads ? p.q_off + h * HD : h < p.q_heads + p.kv_heads ? p.k_off + (h - p.q_heads) * HD
                                                                               : p.v_off + (h - p.q_heads - p.kv_heads) * HD);
  };
  uint4 a[BATCH], b[BATCH];
  auto load = [&](int first) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int h = first + i * AT_ONCE + h0;
      if (h >= heads) continue;
      a[i] = __ldcs(reinterpret_cast<const uint4*>(source(h) + ea));
      b[i] = __ldcs(reinterpret_cast<const uint4*>(source(h) + eb));
    }
  };
  let_next_start();
  await_previous();
  load(0);
  const int pos = p.positions[t], slot = p.slots[t];
  for (int i = threadIdx.x; i < p.pairs; i += kThreads) {
    const float2 cs = turn(pos, p.inv_freq[i], p.factor);
    cosines[i] = cs.x;
    sines[i] = cs.y;
  }
  __syncthreads();
  const bool cached = slot >= 0 && slot < p.num_pages * kPage;
  if (slot >= p.num_pages * kPage && threadIdx.x == 0) report_status(p.status, NF_ST_BAD_INDEX);
  // of the thread's eight pairs; of those that do not turn, what leaves them as they are is not (0 times infinity), so there is a bit each
  float c[8], s[8];
  uint32_t turning = 0;
  if (LAYOUT == SCATTERED) {
    turning = 16 * l < rot ? 1u : 0u;            // (its cosines and sines stay in shared memory)
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = 8 * l + j;
      const bool turns = i < p.pairs;
      c[j] = turns ? cosines[i] : 0.f;
      s[j] = turns ? sines[i] : 0.f;
      turning |= turns ? 1u << j : 0u;
    }
  }
  for (int first = 0; first < heads; first += BATCH * AT_ONCE) {
    if (first > 0) load(first);
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      if (first + i * AT_ONCE >= heads) break;   // (the same for all threads)
      const int h = first + i * AT_ONCE + h0;
      const bool on = h < heads, is_q = h < p.q_heads, is_v = h >= p.q_heads + p.kv_heads;
      uint32_t va[4] = {a[i].x, a[i].y, a[i].z, a[i].w}, vb[4] = {b[i].x, b[i].y, b[i].z, b[i].w};
      if (LAYOUT == SCATTERED) {
        __syncwarp();                            // (a head's threads are of one warp)
        if (on) {
          *reinterpret_cast<uint4*>(&raw[h0][ea]) = a[i];
          *reinterpret_cast<uint4*>(&raw[h0][eb]) = b[i];
        }
        __syncwarp();
      }
      if (!on || (!is_q && !cached)) continue;
      if (!is_v && turning != 0u) {
        if constexpr (LAYOUT == HALVES) {        // (all eight pairs turn or none does)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 x = elements(va[k]), y = elements(vb[k]);
            va[k] = pack_bf16x2(fmaf(y.x, -s[2 * k], x.x * c[2 * k]), fmaf(y.y, -s[2 * k + 1], x.y * c[2 * k + 1]));
            vb[k] = pack_bf16x2(fmaf(x.x, s[2 * k], y.x * c[2 * k]), fmaf(x.y, s[2 * k + 1], y.y * c[2 * k + 1]));
          }
        } else if constexpr (LAYOUT == NEIGHBOURS) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            uint32_t& w = k < 4 ? va[k & 3] : vb[k & 3];
            const float2 x = elements(w);
            if ((turning >> k & 1u) != 0u) w = pack_bf16x2(fmaf(x.y, -s[k], x.x * c[k]), fmaf(x.x, s[k], x.y * c[k]));
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            uint32_t& w = k < 4 ? va[k & 3] : vb[k & 3];
            const int e0 = 16 * l + 2 * k;
            if (e0 >= rot) continue;
            float2 x = elements(w);
            auto turned = [&](int e, float own) {
              const int i = e < p.pairs ? e : e - p.pairs;
              const float other = __bfloat162float(raw[h0][e < p.pairs ? e + p.pairs : i]);
              return fmaf(other, e < p.pairs ? -sines[i] : sines[i], own * cosines[i]);
            };
            w = pack_bf16x2(turned(e0, x.x), turned(e0 + 1, x.y));       // (rot is even)
          }
        }
      }
      __nv_bfloat16* dst;
      if (is_q) {
        dst = static_cast<__nv_bfloat16*>(p.q_out) + (static_cast<long long>(t) * p.q_heads + h) * HD;
      } else {
        const int hh = h - p.q_heads - (is_v ? p.kv_heads : 0);
        dst = static_cast<__nv_bfloat16*>(p.kv_pool) + (((static_cast<long long>(slot / kPage) * 2 + (is_v ? 1 : 0)) * p.kv_heads + hh) * kPage + slot % kPage) * HD;
      }
      *reinterpret_cast<uint4*>(dst + ea) = make_uint4(va[0], va[1], va[2], va[3]);
      *reinterpret_cast<uint4*>(dst + eb) = make_uint4(vb[0], vb[1], vb[2], vb[3]);
    }
  }
}

}  // namespace
}  // namespace nf

extern "C" int nfk_rope_slots(const nfk_rope_slots_params* p, cudaStream_t stream) {
  using namespace nf;
  if (p == nullptr || p->T < 0) return NF_ERR_BAD_ARG;
  if (p->head_dim != 64 && p->head_dim != 128) return NF_ERR_UNSUPPORTED;
  if (p->T == 0) return NF_OK;
  const auto off = [](const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) != 0; };
  if (!p->qkv || !p->q_out || !p->kv_pool || !p->inv_freq || !p->positions || !p->slots || off(p->qkv) || off(p->q_out) || off(p->kv_pool))
    return NF_ERR_BAD_ARG;
  if (p->q_heads <= 0 || p->kv_heads <= 0 || p->num_pages <= 0 || p->num_pages > 0x7fffffff / kPage || p->pairs < 1 || 2 * p->pairs > p->head_dim ||
      p->ld_qkv % 8 != 0 || p->q_off < 0 || p->k_off < 0 || p->v_off < 0 || p->q_off % 8 != 0 || p->k_off % 8 != 0 || p->v_off % 8 != 0)
    return NF_ERR_BAD_ARG;
  const auto run = [&](auto kernel) {
    if (launch_kernel(early_first(p->early_start), kernel, p->T, kThreads, 0, stream, 1, *p) == cudaSuccess) return static_cast<int>(NF_OK);
    (void)cudaGetLastError();
    return static_cast<int>(NF_ERR_CUDA);
  };
  const int layout = p->interleaved != 0 ? NEIGHBOURS : p->pairs % 8 == 0 ? HALVES : SCATTERED;
  if (p->head_dim == 128)
    return run(layout == HALVES ? rope_slots_kernel<128, HALVES> : layout == NEIGHBOURS ? rope_slots_kernel<128, NEIGHBOURS> : rope_slots_kernel<128, SCATTERED>);
  return run(layout == HALVES ? rope_slots_kernel<64, HALVES> : layout == NEIGHBOURS ? rope_slots_kernel<64, NEIGHBOURS> : rope_slots_kernel<64, SCATTERED>);
}
