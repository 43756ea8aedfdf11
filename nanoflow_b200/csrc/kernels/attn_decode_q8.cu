// Attention of one query token per request over the 8-bit paged cache.
//
//   o_h = sum_j e^(s_hj) v_j / sum_j e^(s_hj),   s_hj = sm_scale (q_h . k_j),   k_j = number_j * kscale_j, v_j likewise
//
// Bound by the cache's bytes. A warp reads pages straight into the layout that the tensor cores take: with S^T = K Q^T the keys
// are the 16-row operand (a page's 16 tokens) and the up to 8 query heads of a KV head the 8 columns (16 heads: two such
// products), and which elements of head_dim form a step of the product is free, so a lane's bytes of a key are 16 neighbours, its
// f16 pairs the operand's registers, and no lane needs what another one loaded. O^T = V^T P^T works the same way: V^T is the
// 16-row operand, two of its rows are two neighbouring elements, and a lane reads 16 neighbours of the four tokens whose weights
// it multiplies. P^T gets into its layout by one transposing move per 8 tokens.
// Numbers are exact in f16. Queries are, too, up to a power of two per head (their small elements may be rounded at 2^-25 of the
// largest). The keys' scales join the scores in fp32; the values' scales join the weights, which are rounded to f16 (2^-12)
// relative to the largest value scale so far, `v_ref`, with 2^7 of headroom: values up to 2^20 smaller keep full precision.
//
// A warp keeps a reference per head instead of a running maximum: it moves only where a score exceeds it by 8 (in exponents to
// base 2), so that the common page has one vote and no reduction across lanes; sums stay per lane until a request ends.
#include "attn_q8.cuh"
#include "attn_mma.cuh"

namespace nf {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kStages = 3;
constexpr float kGap = 8.f, kHeadroom = 128.f;      // weights are below 2^8 * 2^7, f16 ends at 65504

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void cp_async8(uint32_t smem_addr, const void* g) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_addr), "l"(g) : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 ld_shared_v2(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ float ld_shared_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}

// Lanes are (g, t) = (lane / 4, lane % 4), as the products' layouts have it.
template <int HD>
struct Dec {
  static constexpr int kKeyBytes = 16 * HD, kStageBytes = 2 * kKeyBytes + 128;    // keys, values, 16 scales of each
  static constexpr int kWarpBytes = kStages * kStageBytes;
};

// fn(row of the partial results) for each of the shared prefix's pieces, for head `h` of KV head `kvh` of request `r`.
template <class F>
__device__ __forceinline__ void for_prefix_pieces(const PrefixPlan& f, int kv_heads, int group, int kvh, int r, int h, F fn) {
  const long long units = prefix_units(f, kv_heads), item = static_cast<long long>(kvh) * f.blocks + r / f.reqs_per_block;
  const int row = r % f.reqs_per_block * group + h;
  const long long c0 = range_of(item * f.tiles, units, f.ctas), c1 = range_of((item + 1) * f.tiles - 1, units, f.ctas);
#pragma unroll 4
  for (long long c = c0; c <= c1; ++c) fn((item + c) * kPrefixRows + row);
}

// A piece's softmax state for one head, spread over the lanes of a warp: HD / 32 elements each.
template <int HD>
struct Row {
  float m = -INFINITY, l = 0.f, o[HD / 32] = {};
  __device__ __forceinline__ void add(float m2, float l2, const float (&x)[HD / 32]) {
    const float top = fmaxf(m, m2), safe = top == -INFINITY ? 0.f : top;
    const float a = q8_exp2(m - safe), b = q8_exp2(m2 - safe);
    l = l * a + l2 * b;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) o[i] = o[i] * a + x[i] * b;
    m = top;
  }
  __device__ __forceinline__ void add_from(const float* ml, const float* row) {
    const float2 s = __ldcg(reinterpret_cast<const float2*>(ml));
    float x[HD / 32];
    load(row, x);
    add(s.x, s.y, x);
  }
  static __device__ __forceinline__ void load(const float* row, float (&x)[HD / 32]) {
    const int lane = threadIdx.x & 31;
    if constexpr (HD == 128) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(row) + lane);
      x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(row) + lane);
      x[0] = v.x; x[1] = v.y;
    }
  }
  __device__ __forceinline__ void store(float* row) const {
    const int lane = threadIdx.x & 31;
    if constexpr (HD == 128) __stcg(reinterpret_cast<float4*>(row) + lane, make_float4(o[0], o[1], o[2], o[3]));
    else __stcg(reinterpret_cast<float2*>(row) + lane, make_float2(o[0], o[1]));
  }
  __device__ __forceinline__ void finish(__nv_bfloat16* out) const {
    const int lane = threadIdx.x & 31;
    const float inv = l == 0.f ? 0.f : 1.f / l;                // (a sum that is NaN stays visible)
    if constexpr (HD == 128)
      reinterpret_cast<uint2*>(out)[lane] = make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
    else
      reinterpret_cast<uint32_t*>(out)[lane] = pack_bf16x2(o[0] * inv, o[1] * inv);
  }
  __device__ __forceinline__ void add_prefix(const PrefixPlan& f, int kv_heads, int group, int kvh, int r, int h) {
    for_prefix_pieces(f, kv_heads, group, kvh, r, h, [&](long long piece) { add_from(f.ml + piece * 2, f.o + piece * HD); });
  }
};

// A piece that a warp leaves for its CTA.
struct Piece {
  int kvh, r, flags;         // flags: 1 there is one, 2 the request starts in it, 4 ends in it
};

template <int HD, int NT, int KIND, bool SHARED>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 3 : 2)
attn_decode_q8_kernel(nfk_attn_q8_params p, PrefixPlan f, unsigned int* counts, float* part_ml, float* part_o) {
  using D = Dec<HD>;
  constexpr int KS = HD / 16, MT = HD / 16, VB = HD / 8;      // steps of Q K^T, row tiles of V^T, bytes of a token's values per lane
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Piece pieces[2 * kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int group = p.q_heads / p.kv_heads;
  const int* indptr = p.kv_indptr + p.req_begin;
  const int base = indptr[0];
  long long pages_all = static_cast<long long>(indptr[p.req_count]) - base;
  if (base < 0 || pages_all < 0 || base + pages_all > p.num_indices) {       // lists that are none: nothing is read
    if (threadIdx.x == 0) report_status(p.status, NF_ST_BAD_INDEX);
    pages_all = 0;
  }
  int seen = 0;
  for (int r = threadIdx.x; r < p.req_count; r += kThreads) {
    const int pages = indptr[r + 1] - indptr[r];
    seen |= pages < 0 ? 1 : pages == 0 ? 2 : 0;
  }
  if (__syncthreads_or(seen & 1) != 0 && pages_all > 0) {
    if (threadIdx.x == 0) report_status(p.status, NF_ST_BAD_INDEX);
    pages_all = 0;
  }
  const bool some_empty = __syncthreads_or(seen & 2) != 0 || pages_all == 0;
  const long long units = pages_all * p.kv_heads;
  const long long most_workers = static_cast<long long>(gridDim.x) * kWarps;
  const long long workers = units < most_workers ? units : most_workers;
  const float scale = p.sm_scale * kQ8Log2e;
  __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(p.out);
  const int vec = HD / 32;

  auto row_of = [&](int r) {                                   // the request's row of q and out
    const int tok = p.qo_indptr[p.req_begin + r];
    if (tok >= 0 && tok < p.num_tokens) return tok;
    if (lane == 0) report_status(p.status, NF_ST_BAD_INDEX);
    return -1;
  };

  const long long w = static_cast<long long>(blockIdx.x) * kWarps + warp;
  const bool working = w < workers;
  // this warp's own slots for pieces: the first behind the pipelines, the second over its own pipeline when that is done
  const int slot_floats = group * (HD + 2);
  const uint32_t pipe = smem_u32(smem) + warp * D::kWarpBytes;
  if (lane < 2) pieces[warp * 2 + lane].flags = 0;
  __syncwarp();

  if (working) {
    const long long u0 = range_begin(w, units, workers), u1 = range_begin(w + 1, units, workers);
    const int n = static_cast<int>(u1 - u0);
    // ---- loads: unit i of the range is page (u0 + i) % pages_all of KV head (u0 + i) / pages_all ----
    int i_kvh = static_cast<int>(u0 / pages_all), i_page = static_cast<int>(u0 - i_kvh * pages_all);
    int ids = 0, ids_left = 0;                                 // page numbers, one per lane, fetched 32 at a time
    const uint8_t* pool = reinterpret_cast<const uint8_t*>(p.kv_pool);
    auto issue = [&](int i) {
      if (i < n) {
        if (ids_left == 0) {
          ids_left = min(32, static_cast<int>(pages_all) - i_page);
          ids = lane < ids_left ? p.kv_indices[base + i_page + lane] : 0;
          if (ids < 0 || ids >= p.num_pages) {
            report_status(p.status, NF_ST_BAD_INDEX);
            ids = 0;
          }
          // lane 0 holds the next one
        }
        const int page = __shfl_sync(0xffffffffu, ids, 0);
        ids = __shfl_down_sync(0xffffffffu, ids, 1);
        --ids_left;
        const long long head = static_cast<long long>(page) * 2 * p.kv_heads + i_kvh;
        const uint8_t* k = pool + head * D::kKeyBytes;
        const uint8_t* v = k + static_cast<long long>(p.kv_heads) * D::kKeyBytes;
        const uint32_t st = pipe + (i % kStages) * D::kStageBytes;
#pragma unroll
        for (int x = 0; x < HD / 64; ++x)
#pragma unroll
          for (int hi = 0; hi < 2; ++hi) cp_async16(st + (x * 2 + hi) * 512 + lane * 16, k + (g + 8 * hi) * HD + x * 64 + t * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint8_t* from = v + (2 * t + (j & 1) + 8 * (j >> 1)) * HD + g * VB;
          const uint32_t to = st + D::kKeyBytes + j * 32 * VB + lane * VB;
          if constexpr (HD == 128) cp_async16(to, from);
          else cp_async8(to, from);
        }
        if (lane < 8) cp_async16(st + 2 * D::kKeyBytes + lane * 16, p.kv_scale + (head + (lane >> 2) * p.kv_heads) * kQ8Page + (lane & 3) * 4);
        if (++i_page == pages_all) {
          i_page = 0;
          ++i_kvh;
          ids_left = 0;
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) issue(s);

    // ---- the request that the first unit belongs to: the last whose pages start at or before it, 32 candidates at a time ----
    int kvh = static_cast<int>(u0 / pages_all);
    int at = static_cast<int>(u0 - kvh * pages_all);           // place in the row of pages
    auto find = [&](int place) {
      int lo = 0, hi = p.req_count;                            // it is in [lo, hi)
      while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int r = lo + lane * step;
        const unsigned int before = __ballot_sync(0xffffffffu, r < hi && indptr[r] - base <= place);
        const int last = 31 - __clz(before);                   // (lane 0's is one: lo starts at or before the place)
        lo += last * step;
        hi = min(hi, lo + step);
      }
      return lo;
    };
    int r = find(at);

    int i = 0;
    while (i < n) {
      // ---- a request's run of pages in this range ----
      const int r_begin = indptr[r] - base, r_end = indptr[r + 1] - base;
      const int count = min(n - i, r_end - at);
      const bool starts = at == r_begin, ends = at + count == r_end;
      const int last_len = p.kv_last_page_len[p.req_begin + r];
      const int tok = row_of(r);
      uint32_t qb[NT][KS][2];
      float q_up[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int h = nt * 8 + g;
        const bool on = tok >= 0 && h < group;
        const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(p.q) +
                                                          (static_cast<long long>(on ? tok : 0) * p.q_heads + kvh * group + (on ? h : 0)) * HD) + t * 2;
        uint4 raw[KS / 2];
        uint32_t most = 0;
#pragma unroll
        for (int x = 0; x < KS / 2; ++x) {
          raw[x] = on ? src[(x >> 1) * 8 + (x & 1)] : make_uint4(0, 0, 0, 0);
          const uint32_t q4[4] = {raw[x].x, raw[x].y, raw[x].z, raw[x].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) most = max(most, max(q4[e] << 16 & 0x7fffffffu, q4[e] & 0x7fff0000u));
        }
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        float down, up;
        q_powers(__uint_as_float(most), down, up);
#pragma unroll
        for (int x = 0; x < KS / 2; ++x) {
          const uint32_t q4[4] = {raw[x].x, raw[x].y, raw[x].z, raw[x].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 q2 = unpack_bf16x2(q4[e]);
            qb[nt][x * 2 + (e >> 1)][e & 1] = pack_f16x2(q2.x * down, q2.y * down);
          }
        }
        up *= scale;
        q_up[nt][0] = __shfl_sync(0xffffffffu, up, 8 * t);     // of the columns that this lane's scores are in
        q_up[nt][1] = __shfl_sync(0xffffffffu, up, 8 * t + 4);
      }
      float o[NT][MT][4], ref[NT][2], l[NT][2], v_ref = 7.8886091e-31f, v_unit = kHeadroom / 7.8886091e-31f;      // 2^-100
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        ref[nt][0] = ref[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int j = 0; j < MT; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
      }

      for (int c = 0; c < count; ++c, ++i) {
        cp_async_wait<kStages - 2>();
        __syncwarp();
        const uint32_t st = pipe + (i % kStages) * D::kStageBytes;
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
        for (int x = 0; x < HD / 64; ++x) {
          const uint4 a = ld_shared_v4(st + x * 1024 + lane * 16), b = ld_shared_v4(st + x * 1024 + 512 + lane * 16);
          const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t a0, a1, a2, a3;
            q8_to_f16<KIND>(aw[e], a0, a2);
            q8_to_f16<KIND>(bw[e], a1, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(s[nt], a0, a1, a2, a3, qb[nt][x * 4 + e][0], qb[nt][x * 4 + e][1]);
          }
        }
        const uint32_t sc = st + 2 * D::kKeyBytes;
        const int valid = ends && c == count - 1 ? last_len : kQ8Page;
        const bool on0 = g < valid, on1 = g + 8 < valid;
        const float k0 = ld_shared_f32(sc + g * 4), k1 = ld_shared_f32(sc + g * 4 + 32);
        const float v0 = on0 ? ld_shared_f32(sc + 64 + g * 4) : 0.f, v1 = on1 ? ld_shared_f32(sc + 96 + g * 4) : 0.f;
        bool grow = v0 > v_ref || v1 > v_ref;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            s[nt][e] = on0 ? s[nt][e] * k0 * q_up[nt][e] : -INFINITY;
            s[nt][2 + e] = on1 ? s[nt][2 + e] * k1 * q_up[nt][e] : -INFINITY;
            grow = grow || fmaxf(s[nt][e], s[nt][2 + e]) > ref[nt][e] + kGap;
          }
        }
        if (__any_sync(0xffffffffu, grow)) {
          float most = fmaxf(v_ref, fmaxf(v0, v1));
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
          most = __uint_as_float((__float_as_uint(most) + 0x7fffffu) & 0xff800000u);          // the next power of two
          const float shrink = v_ref / most;
          v_ref = most;
          v_unit = kHeadroom / most;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float by[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mx = fmaxf(s[nt][e], s[nt][2 + e]);
#pragma unroll
              for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
              const float top = mx > ref[nt][e] + kGap ? mx : ref[nt][e];
              const float alpha = top == ref[nt][e] ? 1.f : q8_exp2(ref[nt][e] - top);
              ref[nt][e] = top;
              l[nt][e] *= alpha;
              by[e] = alpha * shrink;
            }
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              o[nt][j][0] *= by[0]; o[nt][j][1] *= by[1]; o[nt][j][2] *= by[0]; o[nt][j][3] *= by[1];
            }
          }
        }
        const float w0 = v0 * v_unit, w1 = v1 * v_unit;
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float e0[2], e1[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float safe = ref[nt][e] == -INFINITY ? 0.f : ref[nt][e];
            e0[e] = q8_exp2(s[nt][e] - safe);
            e1[e] = q8_exp2(s[nt][2 + e] - safe);
            l[nt][e] += e0[e] + e1[e];
          }
          pb[nt][0] = transpose_8x8(pack_f16x2(e0[0] * w0, e0[1] * w0));
          pb[nt][1] = transpose_8x8(pack_f16x2(e1[0] * w1, e1[1] * w1));
        }
        uint32_t vw[4][VB / 4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t from = st + D::kKeyBytes + j * 32 * VB + lane * VB;
          if constexpr (HD == 128) {
            const uint4 v = ld_shared_v4(from);
            vw[j][0] = v.x; vw[j][1] = v.y; vw[j][2] = v.z; vw[j][3] = v.w;
          } else {
            const uint2 v = ld_shared_v2(from);
            vw[j][0] = v.x; vw[j][1] = v.y;
          }
        }
        if (valid < kQ8Page)                                   // what lies behind the last token may be anything, NaN among it
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < VB / 4; ++e) vw[j][e] = 2 * t + (j & 1) + 8 * (j >> 1) < valid ? vw[j][e] : 0u;
#pragma unroll
        for (int j = 0; j < MT; ++j) {                         // elements 2j (rows g) and 2j + 1 (rows g + 8) of the lane's
          const uint32_t sel = (j & 1) ? 0x7362u : 0x5140u;
          uint32_t a0, a1, a2, a3;
          q8_to_f16<KIND>(__byte_perm(vw[0][j >> 1], vw[1][j >> 1], sel), a0, a1);
          q8_to_f16<KIND>(__byte_perm(vw[2][j >> 1], vw[3][j >> 1], sel), a2, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][j], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
        }
        __syncwarp();
        issue(i + kStages - 1);
      }

      // ---- the run's end: the final row where it is the whole request, else a piece ----
      const bool whole = starts && ends, last_run = i == n;
      const float v_back = v_ref / kHeadroom;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], off);
      if (whole) {
        if (SHARED) await_previous();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int h = nt * 8 + 2 * t + e;
            if (h >= group || tok < 0) continue;
            float x[VB], sum = l[nt][e], m = ref[nt][e];
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              x[2 * j] = o[nt][j][e] * v_back;
              x[2 * j + 1] = o[nt][j][2 + e] * v_back;
            }
            if (SHARED)
              for_prefix_pieces(f, p.kv_heads, group, kvh, r, h, [&](long long piece) {
                const float2 s2 = __ldcg(reinterpret_cast<const float2*>(f.ml) + piece);
                const float4* from = reinterpret_cast<const float4*>(f.o + piece * HD + g * VB);
                const float top = fmaxf(m, s2.x), safe = top == -INFINITY ? 0.f : top;
                const float a = q8_exp2(m - safe), b = q8_exp2(s2.x - safe);
                sum = sum * a + s2.y * b;
                m = top;
#pragma unroll
                for (int j = 0; j < VB / 4; ++j) {
                  const float4 y = __ldcg(from + j);
                  x[4 * j] = x[4 * j] * a + y.x * b;
                  x[4 * j + 1] = x[4 * j + 1] * a + y.y * b;
                  x[4 * j + 2] = x[4 * j + 2] * a + y.z * b;
                  x[4 * j + 3] = x[4 * j + 3] * a + y.w * b;
                }
              });
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            uint4* dst = reinterpret_cast<uint4*>(out + (static_cast<long long>(tok) * p.q_heads + kvh * group + h) * HD + g * VB);
#pragma unroll
            for (int j = 0; j < VB / 8; ++j)
              dst[j] = make_uint4(pack_bf16x2(x[8 * j] * inv, x[8 * j + 1] * inv), pack_bf16x2(x[8 * j + 2] * inv, x[8 * j + 3] * inv),
                                  pack_bf16x2(x[8 * j + 4] * inv, x[8 * j + 5] * inv), pack_bf16x2(x[8 * j + 6] * inv, x[8 * j + 7] * inv));
          }
      } else {
        const int which = last_run ? 1 : 0;                    // a run that is neither whole nor the last is the first
        if (last_run) {
          cp_async_wait<0>();
          __syncwarp();
        }
        float* po = last_run ? reinterpret_cast<float*>(smem + warp * D::kWarpBytes)
                             : reinterpret_cast<float*>(smem + kWarps * D::kWarpBytes) + warp * slot_floats;
        float* pml = po + group * HD;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int h = nt * 8 + 2 * t + e;
            if (h >= group) continue;
            if (g == 0) {
              pml[h * 2] = ref[nt][e];
              pml[h * 2 + 1] = l[nt][e];
            }
#pragma unroll
            for (int j = 0; j < MT; ++j)
              *reinterpret_cast<float2*>(po + h * HD + g * VB + 2 * j) = make_float2(o[nt][j][e] * v_back, o[nt][j][2 + e] * v_back);
          }
        if (lane == 0) pieces[warp * 2 + which] = Piece{kvh, r, 1 | (starts ? 2 : 0) | (ends ? 4 : 0)};
      }

      // ---- the next request that has pages ----
      at += count;
      if (i < n) {
        if (at == pages_all) {
          at = 0;
          ++kvh;
        }
        r = r + 1 < p.req_count && at > 0 && indptr[r + 1] - base <= at && indptr[r + 2] - base > at ? r + 1 : find(at);
      }
    }
    cp_async_wait<0>();
  }
  if (SHARED) await_previous();
  __syncthreads();

  // ---- requests without pages of their own: zeros, or the prefix alone ----
  if (some_empty)
    for (long long i = w; i < static_cast<long long>(p.req_count) * p.q_heads; i += most_workers) {
      const int r = static_cast<int>(i / p.q_heads), head = static_cast<int>(i % p.q_heads);
      if (pages_all > 0 && indptr[r + 1] > indptr[r]) continue;
      const int tok = row_of(r);
      Row<HD> row;
      if (SHARED) row.add_prefix(f, p.kv_heads, group, head / group, r, head % group);
      if (tok >= 0) row.finish(out + (static_cast<long long>(tok) * p.q_heads + head) * HD);
    }

  // ---- pieces of the CTA's warps, joined request by request; what the CTA holds only a part of goes to the workspace ----
  for (int first = 0; first < 2 * kWarps; ++first) {
    if (pieces[first].flags == 0) continue;
    int last = first;
    for (int k = first + 1; k < 2 * kWarps; ++k)
      if (pieces[k].flags != 0) {
        if (pieces[k].kvh != pieces[first].kvh || pieces[k].r != pieces[first].r) break;
        last = k;
      }
    const int kvh = pieces[first].kvh, r = pieces[first].r;
    const bool starts = (pieces[first].flags & 2) != 0, ends = (pieces[last].flags & 4) != 0;
    const int tok = row_of(r);
    const int side = starts ? 1 : 0;                           // a request that goes on behind this CTA, or one from before it
    const long long mine = (static_cast<long long>(blockIdx.x) * 2 + side) * group;
    for (int h = warp; h < group; h += kWarps) {
      Row<HD> row;
      for (int k = first; k <= last; ++k) {
        if (pieces[k].flags == 0) continue;
        const float* po = (k & 1) ? reinterpret_cast<const float*>(smem + (k >> 1) * D::kWarpBytes)
                                  : reinterpret_cast<const float*>(smem + kWarps * D::kWarpBytes) + (k >> 1) * slot_floats;
        float x[HD / 32];
#pragma unroll
        for (int d = 0; d < vec; ++d) x[d] = po[h * HD + lane * vec + d];
        row.add(po[group * HD + h * 2], po[group * HD + h * 2 + 1], x);
      }
      if (starts && ends) {
        if (SHARED) row.add_prefix(f, p.kv_heads, group, kvh, r, h);
        if (tok >= 0) row.finish(out + (static_cast<long long>(tok) * p.q_heads + kvh * group + h) * HD);
      } else {
        row.store(part_o + (mine + h) * HD);
        if (lane == 0) __stcg(reinterpret_cast<float2*>(part_ml) + mine + h, make_float2(row.m, row.l));
      }
    }
    if (!(starts && ends)) {
      // The CTAs that hold parts of the request follow from the ranges. The last of them to arrive joins all parts, in their order.
      const long long begin = kvh * pages_all + indptr[r] - base, end = kvh * pages_all + indptr[r + 1] - base;
      const int c0 = static_cast<int>(range_of(begin, units, workers) / kWarps), c1 = static_cast<int>(range_of(end - 1, units, workers) / kWarps);
      __syncthreads();
      int done = 0;
      if (threadIdx.x == 0) {
        __threadfence();
        done = atomicAdd(counts + c0, 1u) == static_cast<unsigned int>(c1 - c0) ? 1 : 0;
        if (done != 0) {
          counts[c0] = 0u;
          __threadfence();
        }
      }
      if (__syncthreads_or(done) != 0)
        for (int h = warp; h < group; h += kWarps) {
          Row<HD> row;
#pragma unroll 4
          for (int c = c0; c <= c1; ++c) {
            const long long from = (static_cast<long long>(c) * 2 + (c == c0 ? 1 : 0)) * group + h;
            row.add_from(part_ml + from * 2, part_o + from * HD);
          }
          if (SHARED) row.add_prefix(f, p.kv_heads, group, kvh, r, h);
          if (tok >= 0) row.finish(out + (static_cast<long long>(tok) * p.q_heads + kvh * group + h) * HD);
        }
    }
    first = last;
  }
}

template <int HD, int NT, int KIND, bool SHARED>
int launch_decode(const nfk_attn_q8_params& p, const PrefixPlan& f, const Q8Workspace& ws, cudaStream_t stream) {
  const int group = p.q_heads / p.kv_heads;
  const int bytes = kWarps * (Dec<HD>::kWarpBytes + group * (HD + 2) * 4);
  // CTAs that fit an SM, by the largest group of this instantiation
  static int fit_dev[kMaxDevices] = {0};
  int& fit = fit_dev[device_slot()];
  const auto kernel = attn_decode_q8_kernel<HD, NT, KIND, SHARED>;
  if (fit == 0) {
    const int most = kWarps * (Dec<HD>::kWarpBytes + NT * 8 * (HD + 2) * 4);
    int per_sm = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kThreads, most) != cudaSuccess || per_sm < 1) {
      (void)cudaGetLastError();
      return NF_ERR_CUDA;
    }
    fit = per_sm < kDecodeCtasPerSm ? per_sm : kDecodeCtasPerSm;
  }
  const long long room = static_cast<long long>(fit) * device_sm_count();
  long long ctas = p.num_ctas > 0 && p.num_ctas < room ? p.num_ctas : room;
  const long long work = static_cast<long long>(p.num_indices) * p.kv_heads + static_cast<long long>(p.req_count) * p.q_heads;
  const long long useful = (work + kWarps - 1) / kWarps;
  if (ctas > useful) ctas = useful;
  char* base = static_cast<char*>(p.workspace);
  if (launch_kernel(SHARED, kernel, static_cast<int>(ctas), kThreads, bytes, stream, 1, p, f, reinterpret_cast<unsigned int*>(base + ws.counts),
                    reinterpret_cast<float*>(base + ws.ml), reinterpret_cast<float*>(base + ws.o)) == cudaSuccess)
    return NF_OK;
  (void)cudaGetLastError();
  return NF_ERR_CUDA;
}

template <int HD, int NT, int KIND>
int launch_decode(const nfk_attn_q8_params& p, const PrefixPlan& f, const Q8Workspace& ws, cudaStream_t stream) {
  return p.prefix_len > 0 ? launch_decode<HD, NT, KIND, true>(p, f, ws, stream) : launch_decode<HD, NT, KIND, false>(p, f, ws, stream);
}
template <int HD>
int launch_decode(const nfk_attn_q8_params& p, const PrefixPlan& f, const Q8Workspace& ws, cudaStream_t stream) {
  const bool wide = p.q_heads / p.kv_heads > 8;
  if (p.kind == NFK_Q8_E4M3) return wide ? launch_decode<HD, 2, NFK_Q8_E4M3>(p, f, ws, stream) : launch_decode<HD, 1, NFK_Q8_E4M3>(p, f, ws, stream);
  return wide ? launch_decode<HD, 2, NFK_Q8_INT8>(p, f, ws, stream) : launch_decode<HD, 1, NFK_Q8_INT8>(p, f, ws, stream);
}

bool sizes_built(const nfk_attn_q8_params& p) {
  return (p.head_dim == 64 || p.head_dim == 128) && p.kv_heads > 0 && p.q_heads > 0 && p.q_heads % p.kv_heads == 0 &&
         p.q_heads / p.kv_heads <= 16;
}
bool aligned16(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) == 0; }

}  // namespace
}  // namespace nf

extern "C" long long nfk_attn_q8_workspace(const nfk_attn_q8_params* p) {
  using namespace nf;
  if (p == nullptr || !sizes_built(*p) || p->req_count < 0 || p->prefix_len < 0) return 0;
  const PrefixPlan f = prefix_plan(*p);
  return q8_workspace(p->q_heads / p->kv_heads, p->head_dim, static_cast<long long>(p->kv_heads) * f.blocks + f.ctas).bytes;
}

extern "C" int nfk_attn_decode_q8(const nfk_attn_q8_params* p, cudaStream_t stream) {
  using namespace nf;
  if (p == nullptr || p->req_count < 0 || p->req_begin < 0 || p->prefix_len < 0) return NF_ERR_BAD_ARG;
  if (!sizes_built(*p) || (p->kind != NFK_Q8_E4M3 && p->kind != NFK_Q8_INT8)) return NF_ERR_UNSUPPORTED;
  if (p->req_count == 0) return NF_OK;
  if (!p->q || !p->out || !p->kv_pool || !p->kv_scale || !p->qo_indptr || !p->kv_indptr || !p->kv_last_page_len || !p->workspace ||
      (p->num_indices > 0 && !p->kv_indices) || (p->prefix_len > 0 && !p->prefix_pages) || p->num_pages <= 0 || p->num_tokens <= 0 ||
      p->num_indices < 0 || p->num_ctas < 0 || !aligned16(p->q) || !aligned16(p->out) || !aligned16(p->kv_pool) ||
      !aligned16(p->kv_scale) || (reinterpret_cast<uintptr_t>(p->workspace) & 255) != 0)
    return NF_ERR_BAD_ARG;
  PrefixPlan f = prefix_plan(*p);
  const Q8Workspace ws = q8_workspace(p->q_heads / p->kv_heads, p->head_dim, static_cast<long long>(p->kv_heads) * f.blocks + f.ctas);
  if (p->workspace_bytes < ws.bytes) return NF_ERR_BAD_ARG;
  f.ml = reinterpret_cast<const float*>(static_cast<const char*>(p->workspace) + ws.prefix_ml);
  f.o = reinterpret_cast<const float*>(static_cast<const char*>(p->workspace) + ws.prefix_o);
  if (p->prefix_len > 0) {
    const int rc = launch_prefix_q8(*p, f, stream);
    if (rc != NF_OK) return rc;
  }
  return p->head_dim == 128 ? launch_decode<128>(*p, f, ws, stream) : launch_decode<64>(*p, f, ws, stream);
}
