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
constexpr int kAppendThreads = 128;

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

// A CTA per token; HD / 16 threads per head, each with eight elements of either half, so that a thread holds both elements of its
// eight pairs, and the same pairs for every head that it takes: its cosines and sines stay in registers. What bounds it is latency:
// a thread requests its elements of BATCH heads before the CTA works out the token's angles and page.
template <int HD, int KIND>
__global__ void __launch_bounds__(kAppendThreads, 5) rope_append_q8_kernel(nfk_rope_append_q8_params p) {
  constexpr int HALF = HD / 2, LPH = HD / 16, AT_ONCE = kAppendThreads / LPH, BATCH = 3;
  __shared__ float2 table[HALF];
  const int l = threadIdx.x % LPH, h0 = threadIdx.x / LPH, t = blockIdx.x;
  const int heads = p.q_heads + 2 * p.kv_heads;
  const __nv_bfloat16* row = reinterpret_cast<const __nv_bfloat16*>(p.qkv) + t * p.ld_qkv + 8 * l;
  uint4 lo[BATCH], hi[BATCH];
  auto load = [&](int first) {
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int h = first + b * AT_ONCE + h0;
      if (h >= heads) continue;
      const __nv_bfloat16* src = row + (h < p.q_heads ? p.q_off + h * HD : h < p.q_heads + p.kv_heads ? p.k_off + (h - p.q_heads) * HD
                                                                                            : p.v_off + (h - p.q_heads - p.kv_heads) * HD);
      lo[b] = __ldcs(reinterpret_cast<const uint4*>(src));
      hi[b] = __ldcs(reinterpret_cast<const uint4*>(src + HALF));
    }
  };
  load(0);
  const int pos = p.positions[t], req = p.token_req[t];
  const bool req_ok = req >= 0 && req < p.num_reqs && pos >= 0;
  const int begin = p.kv_indptr[req_ok ? req : 0], end = p.kv_indptr[req_ok ? req + 1 : 0];        // (not looked at before they are needed)
  if (threadIdx.x < HALF)
    table[threadIdx.x] = p.cos_sin != nullptr ? reinterpret_cast<const float2*>(p.cos_sin)[static_cast<long long>(t) * HALF + threadIdx.x]
                                              : turn(pos, p.inv_freq[threadIdx.x]);
  __syncthreads();
  const long long entry = static_cast<long long>(begin) + pos / kQ8Page;
  const bool entry_ok = req_ok && begin >= 0 && entry < end && entry < p.num_indices;
  const int page = entry_ok ? p.kv_indices[entry] : -1;
  float2 cs[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) cs[j] = table[8 * l + j];
  const bool norms = p.q_norm != nullptr || p.k_norm != nullptr;
  for (int first = 0; first < heads; first += BATCH * AT_ONCE) {
    if (first > 0) load(first);
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      if (first + i * AT_ONCE >= heads) break;                // (the same for all threads: sums cross lanes)
      const int h = first + i * AT_ONCE + h0;
      const bool on = h < heads, is_q = h < p.q_heads, is_k = !is_q && h < p.q_heads + p.kv_heads;
      const int hh = is_q ? h : is_k ? h - p.q_heads : h - p.q_heads - p.kv_heads;
      float a[8] = {}, b[8] = {};
      if (on) {
        unpack8(lo[i], a);
        unpack8(hi[i], b);
      }
      const void* norm = is_q ? p.q_norm : is_k ? p.k_norm : nullptr;
      if (norms) {
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
      if (__all_sync(0xffffffffu, is_q)) continue;
      uint32_t most = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        most = max(most, max(__float_as_uint(a[j]) & 0x7fffffffu, __float_as_uint(b[j]) & 0x7fffffffu));
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      const bool page_ok = page >= 0 && page < p.num_pages;
      if (on && !is_q && !page_ok && l == 0) report_status(p.status, NF_ST_BAD_INDEX);
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

// A thread has eight numbers per step: an 8-byte load, their vector's scale, a 16-byte store, so that a warp's loads and its stores
// are of whole rows (16 numbers and two stores 32 bytes apart: 4096 pages 77 us instead of 69). All loads of a CTA's STEPS steps are
// on their way before the first store.
constexpr int kReadSteps = 8;
template <int HD, int KIND>
__global__ void __launch_bounds__(256) kv_read_q8_kernel(nfk_kv_read_q8_params p, int parts) {
  constexpr int PER_VEC = HD / 8;
  const int which = blockIdx.x / parts, part = blockIdx.x - which * parts, per_page = 2 * p.kv_heads * kQ8Page * PER_VEC;
  const int page = p.page_ids[which];
  if (page < 0 || page >= p.num_pages) {
    if (threadIdx.x == 0) report_status(p.status, NF_ST_BAD_INDEX);
    return;
  }
  const uint2* from = reinterpret_cast<const uint2*>(p.kv_pool) + static_cast<long long>(page) * per_page;
  const float* scales = p.kv_scale + static_cast<long long>(page) * (per_page / PER_VEC);
  uint4* to = reinterpret_cast<uint4*>(p.out) + static_cast<long long>(which) * per_page;
  const int first = part * (256 * kReadSteps) + threadIdx.x;
  uint2 raw[kReadSteps];
  float scale[kReadSteps];
#pragma unroll
  for (int s = 0; s < kReadSteps; ++s) {
    const int i = first + s * 256;
    if (i >= per_page) break;
    raw[s] = __ldcs(from + i);
    scale[s] = scales[i / PER_VEC];
  }
#pragma unroll
  for (int s = 0; s < kReadSteps; ++s) {
    const int i = first + s * 256;
    if (i >= per_page) break;
    uint32_t a, b, c, d;
    q8_to_f16<KIND>(raw[s].x, a, b);
    q8_to_f16<KIND>(raw[s].y, c, d);
    const float2 w = unpack_f16x2(a), x = unpack_f16x2(b), y = unpack_f16x2(c), z = unpack_f16x2(d);
    to[i] = make_uint4(pack_bf16x2(w.x * scale[s], w.y * scale[s]), pack_bf16x2(x.x * scale[s], x.y * scale[s]),
                       pack_bf16x2(y.x * scale[s], y.y * scale[s]), pack_bf16x2(z.x * scale[s], z.y * scale[s]));
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
  if (p->head_dim == 128)
    (p->kind == NFK_Q8_E4M3 ? rope_append_q8_kernel<128, NFK_Q8_E4M3> : rope_append_q8_kernel<128, NFK_Q8_INT8>)<<<p->T, kAppendThreads, 0, stream>>>(*p);
  else
    (p->kind == NFK_Q8_E4M3 ? rope_append_q8_kernel<64, NFK_Q8_E4M3> : rope_append_q8_kernel<64, NFK_Q8_INT8>)<<<p->T, kAppendThreads, 0, stream>>>(*p);
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
  const int parts = (2 * p->kv_heads * kQ8Page * p->head_dim / 8 + 256 * kReadSteps - 1) / (256 * kReadSteps);
  const long long blocks = static_cast<long long>(p->n_pages) * parts;
  if (blocks > 0x7fffffffll) return NF_ERR_BAD_ARG;
  const auto run = [&](auto kernel) { kernel<<<static_cast<int>(blocks), 256, 0, stream>>>(*p, parts); };
  if (p->head_dim == 128) run(p->kind == NFK_Q8_E4M3 ? kv_read_q8_kernel<128, NFK_Q8_E4M3> : kv_read_q8_kernel<128, NFK_Q8_INT8>);
  else run(p->kind == NFK_Q8_E4M3 ? kv_read_q8_kernel<64, NFK_Q8_E4M3> : kv_read_q8_kernel<64, NFK_Q8_INT8>);
  return launched();
}
