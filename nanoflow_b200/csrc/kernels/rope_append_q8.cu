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

__device__ __forceinline__ void unpack8(const uint4& v, f32x2 (&f)[4]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = pair(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
}
__device__ __forceinline__ uint4 pack8(const f32x2 (&f)[4]) {
  const float2 a = halves(f[0]), b = halves(f[1]), c = halves(f[2]), d = halves(f[3]);
  return make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(b.x, b.y), pack_bf16x2(c.x, c.y), pack_bf16x2(d.x, d.y));
}

// cos and sin of pos * f. The product is formed in 64 bits and brought to one turn there: in fp32 the angle of position 100000
// would be off by 0.004.
__device__ __forceinline__ float2 turn(int pos, float f) {
  const double t = static_cast<double>(pos) * static_cast<double>(f) * 0.15915494309189533577;
  float s, c;
  sincospif(2.f * static_cast<float>(t - rint(t)), &s, &c);
  return make_float2(c, s);
}

// Mean squares (and eps) that a norm takes as fp32 sums them: nothing that counts is lost below, and the sum of 128 squares is finite.
constexpr float kLeastSquare = 7.8886091e-31f, kMostSquare = 1.329228e36f;      // 2^-100, 2^120

// A CTA per token; HD / 16 threads per head, each with eight elements of either half, so that a thread holds both elements of its
// eight pairs, and the same pairs for every head that it takes: its cosines and sines stay in registers. What bounds it is the issue
// of instructions, and latency (2048 tokens, 32 / 8 heads, norms: 13 us for 46 MB; 683 tokens of 64 / 8 heads 6.4): arithmetic is two elements at a time,
// and a thread requests its elements of BATCH heads before the CTA works out the token's angles and page. It does not let the next
// kernel start: CTAs that wait beside its last ones cost more than their launch (2048 tokens and a kv_read_q8 behind them 17.7 us,
// without 15.9).
template <int HD, int KIND>
__global__ void __launch_bounds__(kAppendThreads, 5) rope_append_q8_kernel(nfk_rope_append_q8_params p) {
  constexpr int HALF = HD / 2, LPH = HD / 16, AT_ONCE = kAppendThreads / LPH, BATCH = 3;
  __shared__ __align__(16) float cosines[HALF], sines[HALF], weights[2][HD];        // weights of the norms of queries and of keys
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
  await_previous();
  load(0);
  const int pos = p.positions[t], req = p.token_req[t];
  const bool req_ok = req >= 0 && req < p.num_reqs && pos >= 0;
  const int begin = p.kv_indptr[req_ok ? req : 0], end = p.kv_indptr[req_ok ? req + 1 : 0];        // (not looked at before they are needed)
  if (threadIdx.x < HALF) {
    const float2 cs = p.cos_sin != nullptr ? reinterpret_cast<const float2*>(p.cos_sin)[static_cast<long long>(t) * HALF + threadIdx.x]
                                           : turn(pos, p.inv_freq[threadIdx.x]);
    cosines[threadIdx.x] = cs.x;
    sines[threadIdx.x] = cs.y;
  }
  if (threadIdx.x < HD) {
    if (p.q_norm != nullptr) weights[0][threadIdx.x] = __bfloat162float(static_cast<const __nv_bfloat16*>(p.q_norm)[threadIdx.x]);
    if (p.k_norm != nullptr) weights[1][threadIdx.x] = __bfloat162float(static_cast<const __nv_bfloat16*>(p.k_norm)[threadIdx.x]);
  }
  __syncthreads();
  const long long entry = static_cast<long long>(begin) + pos / kQ8Page;
  const bool entry_ok = req_ok && begin >= 0 && entry < end && entry < p.num_indices;
  const int page = entry_ok ? p.kv_indices[entry] : -1;
  const bool page_ok = page >= 0 && page < p.num_pages;
  f32x2 co[4], si[4], minus_si[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    co[j] = reinterpret_cast<const f32x2*>(cosines + 8 * l)[j];
    si[j] = reinterpret_cast<const f32x2*>(sines + 8 * l)[j];
    minus_si[j] = si[j] ^ 0x8000000080000000ull;
  }
  // the head's largest magnitude, NaN where there is one
  const auto largest = [](const f32x2 (&x)[4], const f32x2 (&y)[4]) {
    float most = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      most = max3_magnitude(most, halves(x[j]).x, halves(x[j]).y);
      most = max3_magnitude(most, halves(y[j]).x, halves(y[j]).y);
    }
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) most = max3_magnitude(most, __shfl_xor_sync(0xffffffffu, most, o), 0.f);
    return most;
  };
  for (int first = 0; first < heads; first += BATCH * AT_ONCE) {
    if (first > 0) load(first);
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      if (first + i * AT_ONCE >= heads) break;                // (the same for all threads: sums cross lanes)
      const int h = first + i * AT_ONCE + h0;
      const bool on = h < heads, is_q = h < p.q_heads, is_k = !is_q && h < p.q_heads + p.kv_heads;
      f32x2 a[4], b[4];
      unpack8(on ? lo[i] : make_uint4(0, 0, 0, 0), a);
      unpack8(on ? hi[i] : make_uint4(0, 0, 0, 0), b);
      const bool norm = is_q ? p.q_norm != nullptr : is_k && p.k_norm != nullptr;
      if (__any_sync(0xffffffffu, norm)) {
        const auto mean = [&]() {
          f32x2 ss = mul2(a[0], a[0]);
#pragma unroll
          for (int j = 1; j < 4; ++j) ss = fma2(a[j], a[j], ss);
#pragma unroll
          for (int j = 0; j < 4; ++j) ss = fma2(b[j], b[j], ss);
          float sum = halves(ss).x + halves(ss).y;
#pragma unroll
          for (int o = LPH / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          return sum * (1.f / HD);
        };
        float square = mean() + p.eps;
        const bool far = norm && !(square >= kLeastSquare && square <= kMostSquare);
        if (__any_sync(0xffffffffu, far)) {                    // such a head once more, brought to [1, 2) by a power of two
          const float top = largest(a, b);
          const float by = far ? __uint_as_float((254u - min(max(__float_as_uint(top) >> 23 & 255u, 47u), 253u)) << 23) : 1.f;      // (up to 2^80)
          const f32x2 by2 = pair(by, by);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            a[j] = mul2(a[j], by2);
            b[j] = mul2(b[j], by2);
          }
          square = mean() + p.eps * by * by;
        }
        if (norm) {
          const float inv = rsqrtf(square);
          const f32x2 inv2 = pair(inv, inv);
          const f32x2* w = reinterpret_cast<const f32x2*>(weights[is_q ? 0 : 1] + 8 * l);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            a[j] = mul2(a[j], mul2(inv2, w[j]));
            b[j] = mul2(b[j], mul2(inv2, w[HALF / 2 + j]));
          }
        }
      }
      if (is_q || is_k) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x2 x = a[j], y = b[j];
          a[j] = fma2(y, minus_si[j], mul2(x, co[j]));
          b[j] = fma2(x, si[j], mul2(y, co[j]));
        }
      }
      if (is_q) {
        __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(p.q_out) + (static_cast<long long>(t) * p.q_heads + h) * HD + 8 * l;
        *reinterpret_cast<uint4*>(dst) = pack8(a);
        *reinterpret_cast<uint4*>(dst + HALF) = pack8(b);
      }
      if (__all_sync(0xffffffffu, is_q)) continue;
      const float most = largest(a, b);
      if (on && !is_q) {
        const int hh = is_k ? h - p.q_heads : h - p.q_heads - p.kv_heads;
        // (a quarter of both: __fdividef gives 0 for a divisor above 2^126)
        float scale = most * (1.f / q8_largest<KIND>()), inv = __fdividef(0.25f * q8_largest<KIND>(), 0.25f * most);
        if (!(most >= kQ8Smallest && most <= 3.402823466e38f)) {       // nothing to speak of, or not finite
          scale = most < kQ8Smallest ? 0.f : __uint_as_float(0x7fc00000u);
          inv = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) a[j] = b[j] = 0ull;
        }
        if (!page_ok) {
          if (l == 0) report_status(p.status, NF_ST_BAD_INDEX);
          continue;
        }
        const long long vec = ((static_cast<long long>(page) * 2 + (is_k ? 0 : 1)) * p.kv_heads + hh) * kQ8Page + pos % kQ8Page;
        uint8_t* dst = reinterpret_cast<uint8_t*>(p.kv_pool) + vec * HD + 8 * l;
        const f32x2 inv2 = pair(inv, inv);
        const auto numbers = [&](const f32x2 (&x)[4]) {
          const float2 u = halves(mul2(x[0], inv2)), v = halves(mul2(x[1], inv2)), y = halves(mul2(x[2], inv2)), z = halves(mul2(x[3], inv2));
          return make_uint2(q8_from_f32<KIND>(u.x, u.y, v.x, v.y), q8_from_f32<KIND>(y.x, y.y, z.x, z.y));
        };
        *reinterpret_cast<uint2*>(dst) = numbers(a);
        *reinterpret_cast<uint2*>(dst + HALF) = numbers(b);
        if (l == 0) p.kv_scale[vec] = scale;
      }
    }
  }
}

// A thread has eight numbers per step: an 8-byte load, their vector's scale, a 16-byte store, so that a warp's loads and its stores
// are of whole rows (16 numbers and two stores 32 bytes apart: 4096 pages 77 us instead of 69). All loads of a CTA's steps are on
// their way before the first store: 4096 pages of 8 heads 66 us, 6.2 TB/s, 0.94 of a copy's rate.
constexpr int kReadSteps = 8;
template <int HD, int KIND>
__global__ void __launch_bounds__(256) kv_read_q8_kernel(nfk_kv_read_q8_params p, int parts) {
  constexpr int PER_VEC = HD / 8;
  const int which = blockIdx.x / parts, part = blockIdx.x - which * parts, per_page = 2 * p.kv_heads * kQ8Page * PER_VEC;
  let_next_start();
  await_previous();
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
int started(cudaError_t e) {
  if (e == cudaSuccess) return NF_OK;
  (void)cudaGetLastError();
  return NF_ERR_CUDA;
}

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
  const auto run = [&](auto kernel) { return started(launch_kernel(early_first(p->early_start), kernel, p->T, kAppendThreads, 0, stream, 1, *p)); };
  if (p->head_dim == 128) return run(p->kind == NFK_Q8_E4M3 ? rope_append_q8_kernel<128, NFK_Q8_E4M3> : rope_append_q8_kernel<128, NFK_Q8_INT8>);
  return run(p->kind == NFK_Q8_E4M3 ? rope_append_q8_kernel<64, NFK_Q8_E4M3> : rope_append_q8_kernel<64, NFK_Q8_INT8>);
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
  const auto run = [&](auto kernel) { return started(launch_kernel(early_first(p->early_start), kernel, static_cast<int>(blocks), 256, 0, stream, 1, *p, parts)); };
  if (p->head_dim == 128) return run(p->kind == NFK_Q8_E4M3 ? kv_read_q8_kernel<128, NFK_Q8_E4M3> : kv_read_q8_kernel<128, NFK_Q8_INT8>);
  return run(p->kind == NFK_Q8_E4M3 ? kv_read_q8_kernel<64, NFK_Q8_E4M3> : kv_read_q8_kernel<64, NFK_Q8_INT8>);
}
