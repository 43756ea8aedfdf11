// Rotary positions in all their layouts, and the write of keys and values into the tokens' slots of the paged cache.
//
//   (x, y) -> f (x c - y s, y c + x s),  c, s = cos, sin(pos w_i),  (x, y) = (x_i, x_(i + pairs)) or (x_2i, x_(2i+1)),  i < pairs;
// what lies behind the first 2 pairs elements of a head stays as it is, as do values. All in fp32 from the bf16 inputs, rounded once.
// Memory-bound: every element is read once and written once.
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
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[2 * j] = __uint_as_float(w[j] << 16);
    f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}

// Which elements a thread's two vectors of eight hold: HALVES the two of its eight pairs (pairs a multiple of eight), NEIGHBOURS and
// SCATTERED 16 elements in a row; SCATTERED (half layout, any number of pairs) fetches each element's partner by itself.
enum { HALVES, NEIGHBOURS, SCATTERED };

// A CTA per token, HD / 16 threads per head, the same elements of each head that they take, so that their cosines and sines stay in
// registers. Three heads a thread are requested before the token's angles are worked out.
template <int HD, int LAYOUT>
__global__ void __launch_bounds__(kThreads) rope_slots_kernel(nfk_rope_slots_params p) {
  constexpr int LPH = HD / 16, AT_ONCE = kThreads / LPH, BATCH = 3;
  __shared__ __align__(16) float cosines[HD / 2], sines[HD / 2];
  const int l = threadIdx.x % LPH, h0 = threadIdx.x / LPH, t = blockIdx.x, rot = 2 * p.pairs;
  const int heads = p.q_heads + 2 * p.kv_heads;
  int ea = 16 * l, eb = 16 * l + 8;
  if (LAYOUT == HALVES && 16 * l < rot) {
    ea = 8 * l;
    eb = 8 * l + p.pairs;
  }
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
      a[i] = *reinterpret_cast<const uint4*>(source(h) + ea);
      b[i] = *reinterpret_cast<const uint4*>(source(h) + eb);
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
  // element e turns with its partner: f e' = e c + partner s, s negative for the first one of a pair
  float c[16], s[16];
  uint32_t turning = 0;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int e = j < 8 ? ea + j : eb + j - 8;
    const bool turns = e < rot;
    const int i = LAYOUT == NEIGHBOURS ? e >> 1 : e < p.pairs ? e : e - p.pairs;
    const bool second = LAYOUT == NEIGHBOURS ? (e & 1) != 0 : e >= p.pairs;
    c[j] = turns ? cosines[i] : 1.f;
    s[j] = turns ? (second ? sines[i] : -sines[i]) : 0.f;
    turning |= turns ? 1u << j : 0u;
  }
  for (int first = 0; first < heads; first += BATCH * AT_ONCE) {
    if (first > 0) load(first);
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int h = first + i * AT_ONCE + h0;
      if (h >= heads) continue;
      const bool is_q = h < p.q_heads, is_v = h >= p.q_heads + p.kv_heads;
      if (!is_q && !cached) continue;
      __nv_bfloat16* dst;
      if (is_q) {
        dst = static_cast<__nv_bfloat16*>(p.q_out) + (static_cast<long long>(t) * p.q_heads + h) * HD;
      } else {
        const int hh = h - p.q_heads - (is_v ? p.kv_heads : 0);
        dst = static_cast<__nv_bfloat16*>(p.kv_pool) + (((static_cast<long long>(slot / kPage) * 2 + (is_v ? 1 : 0)) * p.kv_heads + hh) * kPage + slot % kPage) * HD;
      }
      uint4 va = a[i], vb = b[i];
      if (!is_v) {
        float x[8], y[8], u[8], v[8];
        unpack8(va, x);
        unpack8(vb, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float px, py;                          // partners
          if (LAYOUT == HALVES) {
            px = y[j];
            py = x[j];
          } else if (LAYOUT == NEIGHBOURS) {
            px = x[j ^ 1];
            py = y[j ^ 1];
          } else {
            const int e0 = ea + j, e1 = eb + j;
            px = e0 < rot ? __bfloat162float(source(h)[e0 < p.pairs ? e0 + p.pairs : e0 - p.pairs]) : 0.f;
            py = e1 < rot ? __bfloat162float(source(h)[e1 < p.pairs ? e1 + p.pairs : e1 - p.pairs]) : 0.f;
          }
          u[j] = (turning >> j & 1u) != 0u ? fmaf(px, s[j], x[j] * c[j]) : x[j];
          v[j] = (turning >> (8 + j) & 1u) != 0u ? fmaf(py, s[8 + j], y[j] * c[8 + j]) : y[j];
        }
        va = pack8(u);
        vb = pack8(v);
      }
      *reinterpret_cast<uint4*>(dst + ea) = va;
      *reinterpret_cast<uint4*>(dst + eb) = vb;
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
