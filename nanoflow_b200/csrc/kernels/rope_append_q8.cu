// Write into and read from the 8-bit paged KV cache, memory-bound passes.
//
//   nfk_rope_append_q8  q_out[t, h] = rot(norm(q[t, h]), pos[t]);  k[t, h], v[t, h] -> numbers and a scale in their page slot,
//                       k normed and rotated like q. rot pairs element i with i + head_dim / 2:
//                       (y_i c_i - y_{i+half} s_i, y_{i+half} c_i + y_i s_i), c_i, s_i = cos, sin(pos f_i);
//                       norm(x) = x / sqrt(mean(x^2) + eps) * w. All in fp32 from the bf16 inputs, rounded once.
//   nfk_kv_read_q8      pages as bf16 pages: number * scale, for the attention of prompts, which reads bf16.
#include "cache_q8.cuh"
#include "kernels.h"

namespace nf {
namespace {

constexpr int kQ8Page = 16;
constexpr int kAppendThreads = 256;

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 x = unpack_bf16x2(w[j]);
    f[2 * j] = x.x;
    f[2 * j + 1] = x.y;
  }
}

// cos and sin of pos * f. The product is formed in 64 bits and brought to one turn there: in fp32 the angle of position 100000
// would be off by 0.004.
__device__ __forceinline__ float2 turn(int pos, float f) {
  const double t = static_cast<double>(pos) * static_cast<double>(f) * 0.15915494309189533577;
  float s, c;
  sincospif(2.f * static_cast<float>(t - rint(t)), &s, &c);
  return make_float2(c, s);
}

// A CTA per token (grid-stride); HD / 16 threads per head, each with eight elements of either half, so that a thread holds both
// elements of its eight pairs, and the same pairs for every head that it takes: its cosines and sines stay in registers.
template <int HD, int KIND>
__global__ void __launch_bounds__(kAppendThreads) rope_append_q8_kernel(nfk_rope_append_q8_params p) {
  constexpr int HALF = HD / 2, LPH = HD / 16, HEADS_AT_ONCE = kAppendThreads / LPH;
  __shared__ float2 table[HALF];
  const int l = threadIdx.x % LPH, h0 = threadIdx.x / LPH;
  const int heads = p.q_heads + 2 * p.kv_heads;
  for (int t = blockIdx.x; t < p.T; t += gridDim.x) {
    const int pos = p.positions[t];
    __syncthreads();                                          // the previous token's table is no longer in use
    if (threadIdx.x < HALF)
      table[threadIdx.x] = p.cos_sin != nullptr ? reinterpret_cast<const float2*>(p.cos_sin)[static_cast<long long>(t) * HALF + threadIdx.x]
                                                : turn(pos, p.inv_freq[threadIdx.x]);
    const int req = p.token_req[t];
    int page = -1;
    if (req >= 0 && req < p.num_reqs && pos >= 0) {
      const int entry = p.kv_indptr[req] + pos / kQ8Page;
      if (entry >= 0 && entry < p.kv_indptr[req + 1] && entry < p.num_indices) page = p.kv_indices[entry];
    }
    const bool page_ok = page >= 0 && page < p.num_pages;
    if (!page_ok && threadIdx.x == 0) report_status(p.status, NF_ST_BAD_INDEX);
    __syncthreads();
    float2 cs[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) cs[j] = table[8 * l + j];
    const __nv_bfloat16* row = reinterpret_cast<const __nv_bfloat16*>(p.qkv) + t * p.ld_qkv;
    for (int hb = 0; hb < heads; hb += HEADS_AT_ONCE) {
      const int h = hb + h0;
      const bool on = h < heads;
      const bool is_q = h < p.q_heads, is_k = !is_q && h < p.q_heads + p.kv_heads;
      const int hh = is_q ? h : is_k ? h - p.q_heads : h - p.q_heads - p.kv_heads;
      const __nv_bfloat16* src = row + (is_q ? p.q_off : is_k ? p.k_off : p.v_off) + hh * HD + 8 * l;
      float a[8] = {}, b[8] = {};
      if (on) {
        unpack8(*reinterpret_cast<const uint4*>(src), a);
        unpack8(*reinterpret_cast<const uint4*>(src + HALF), b);
      }
      const void* norm = is_q ? p.q_norm : is_k ? p.k_norm : nullptr;
      if (p.q_norm != nullptr || p.k_norm != nullptr) {       // (the same for all threads: the sum crosses lanes)
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += a[j] * a[j] + b[j] * b[j];
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (on && norm != nullptr) {
          const float inv = rsqrtf(ss / HD + p.eps);
          float wa[8], wb[8];
          unpack8(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(norm) + 8 * l), wa);
          unpack8(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(norm) + HALF + 8 * l), wb);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            a[j] *= inv * wa[j];
            b[j] *= inv * wb[j];
          }
        }
      }
      if (is_q || is_k) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = a[j], y = b[j];
          a[j] = x * cs[j].x - y * cs[j].y;
          b[j] = y * cs[j].x + x * cs[j].y;
        }
      }
      if (on && is_q) {
        __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(p.q_out) + (static_cast<long long>(t) * p.q_heads + hh) * HD + 8 * l;
        *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(a[4], a[5]), pack_bf16x2(a[6], a[7]));
        *reinterpret_cast<uint4*>(dst + HALF) = make_uint4(pack_bf16x2(b[0], b[1]), pack_bf16x2(b[2], b[3]), pack_bf16x2(b[4], b[5]), pack_bf16x2(b[6], b[7]));
      }
      // Largest magnitude; as bits, so that infinities and NaN come out on top.
      uint32_t most = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        most = max(most, max(__float_as_uint(a[j]) & 0x7fffffffu, __float_as_uint(b[j]) & 0x7fffffffu));
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      if (on && !is_q && page_ok) {
        float scale = __uint_as_float(most) / q8_largest<KIND>(), inv = 1.f / scale;
        if (most >= 0x7f800000u) scale = __uint_as_float(0x7fc00000u), inv = 0.f;
        else if (__uint_as_float(most) < kQ8Smallest) scale = 0.f, inv = 0.f;
        if (inv == 0.f) {
#pragma unroll
          for (int j = 0; j < 8; ++j) a[j] = b[j] = 0.f;
        }
        const long long vec = ((static_cast<long long>(page) * 2 + (is_k ? 0 : 1)) * p.kv_heads + hh) * kQ8Page + pos % kQ8Page;
        uint8_t* dst = reinterpret_cast<uint8_t*>(p.kv_pool) + vec * HD + 8 * l;
        *reinterpret_cast<uint2*>(dst) = make_uint2(q8_from_f32<KIND>(a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv),
                                                    q8_from_f32<KIND>(a[4] * inv, a[5] * inv, a[6] * inv, a[7] * inv));
        *reinterpret_cast<uint2*>(dst + HALF) = make_uint2(q8_from_f32<KIND>(b[0] * inv, b[1] * inv, b[2] * inv, b[3] * inv),
                                                           q8_from_f32<KIND>(b[4] * inv, b[5] * inv, b[6] * inv, b[7] * inv));
        if (l == 0) p.kv_scale[vec] = scale;
      }
    }
  }
}

// 16 numbers per thread and step: a 16-byte load, their vector's scale, two 16-byte stores.
template <int KIND>
__global__ void __launch_bounds__(256) kv_read_q8_kernel(nfk_kv_read_q8_params p) {
  constexpr int STEPS = 4;
  const int per_page = 2 * p.kv_heads * kQ8Page * p.head_dim / 16, per_vec = p.head_dim / 16;
  const long long total = static_cast<long long>(p.n_pages) * per_page;
  const long long first = static_cast<long long>(blockIdx.x) * (256 * STEPS) + threadIdx.x;
  uint4 raw[STEPS];
  float scale[STEPS];
  bool on[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const long long i = first + s * 256;
    on[s] = i < total;
    if (!on[s]) continue;
    const int which = static_cast<int>(i / per_page), at = static_cast<int>(i - static_cast<long long>(which) * per_page);
    const int page = p.page_ids[which];
    if (page < 0 || page >= p.num_pages) {
      if (at == 0) report_status(p.status, NF_ST_BAD_INDEX);
      on[s] = false;
      continue;
    }
    raw[s] = __ldcs(reinterpret_cast<const uint4*>(p.kv_pool) + static_cast<long long>(page) * per_page + at);
    scale[s] = p.kv_scale[static_cast<long long>(page) * (2 * p.kv_heads * kQ8Page) + at / per_vec];
  }
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    if (!on[s]) continue;
    const uint32_t w[4] = {raw[s].x, raw[s].y, raw[s].z, raw[s].w};
    uint32_t o[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t lo, hi;
      q8_to_f16<KIND>(w[j], lo, hi);
      const float2 x = unpack_f16x2(lo), y = unpack_f16x2(hi);
      o[2 * j] = pack_bf16x2(x.x * scale[s], x.y * scale[s]);
      o[2 * j + 1] = pack_bf16x2(y.x * scale[s], y.y * scale[s]);
    }
    uint4* dst = reinterpret_cast<uint4*>(p.out) + (first + s * 256) * 2;
    dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

bool aligned16(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) == 0; }
int launched() { return cudaGetLastError() == cudaSuccess ? NF_OK : NF_ERR_CUDA; }

}  // namespace
}  // namespace nf

extern "C" int nfk_rope_append_q8(const nfk_rope_append_q8_params* p, cudaStream_t stream) {
  using namespace nf;
  if (p == nullptr || p->T < 0) return NF_ERR_BAD_ARG;
  if (p->head_dim != 64 && p->head_dim != 128) return NF_ERR_UNSUPPORTED;
  if (p->kind != NFK_Q8_E4M3 && p->kind != NFK_Q8_INT8) return NF_ERR_UNSUPPORTED;
  if (p->T == 0) return NF_OK;
  if (!p->qkv || !p->q_out || !p->kv_pool || !p->kv_scale || (!p->inv_freq && !p->cos_sin) || !p->positions || !p->token_req ||
      !p->kv_indptr || !p->kv_indices)
    return NF_ERR_BAD_ARG;
  if (p->q_heads <= 0 || p->kv_heads <= 0 || p->num_pages <= 0 || p->num_reqs <= 0 || p->num_indices < 0 || p->ld_qkv % 8 != 0 ||
      p->q_off < 0 || p->k_off < 0 || p->v_off < 0 || p->q_off % 8 != 0 || p->k_off % 8 != 0 || p->v_off % 8 != 0 ||
      !aligned16(p->qkv) || !aligned16(p->q_out) || !aligned16(p->kv_pool) || !aligned16(p->q_norm) || !aligned16(p->k_norm) ||
      (reinterpret_cast<uintptr_t>(p->cos_sin) & 7) != 0)
    return NF_ERR_BAD_ARG;
  const int most = device_sm_count() * 8, blocks = p->T < most ? p->T : most;
  if (p->head_dim == 128)
    (p->kind == NFK_Q8_E4M3 ? rope_append_q8_kernel<128, NFK_Q8_E4M3> : rope_append_q8_kernel<128, NFK_Q8_INT8>)<<<blocks, kAppendThreads, 0, stream>>>(*p);
  else
    (p->kind == NFK_Q8_E4M3 ? rope_append_q8_kernel<64, NFK_Q8_E4M3> : rope_append_q8_kernel<64, NFK_Q8_INT8>)<<<blocks, kAppendThreads, 0, stream>>>(*p);
  return launched();
}

extern "C" int nfk_kv_read_q8(const nfk_kv_read_q8_params* p, cudaStream_t stream) {
  using namespace nf;
  if (p == nullptr || p->n_pages < 0) return NF_ERR_BAD_ARG;
  if (p->head_dim != 64 && p->head_dim != 128) return NF_ERR_UNSUPPORTED;
  if (p->kind != NFK_Q8_E4M3 && p->kind != NFK_Q8_INT8) return NF_ERR_UNSUPPORTED;
  if (p->n_pages == 0) return NF_OK;
  if (!p->kv_pool || !p->kv_scale || !p->out || !p->page_ids || p->kv_heads <= 0 || p->num_pages <= 0 || !aligned16(p->kv_pool) ||
      !aligned16(p->out))
    return NF_ERR_BAD_ARG;
  const long long total = static_cast<long long>(p->n_pages) * (2 * p->kv_heads * kQ8Page * p->head_dim / 16);
  const long long blocks = (total + 1023) / 1024;
  if (blocks > 0x7fffffffll) return NF_ERR_BAD_ARG;
  (p->kind == NFK_Q8_E4M3 ? kv_read_q8_kernel<NFK_Q8_E4M3> : kv_read_q8_kernel<NFK_Q8_INT8>)<<<static_cast<int>(blocks), 256, 0, stream>>>(*p);
  return launched();
}
