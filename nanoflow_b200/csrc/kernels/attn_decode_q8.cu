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

constexpr int kWarps = kDecodeWarps, kThreads = 32 * kWarps;
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
  static constexpr int kStages = HD == 128 ? 3 : 5;            // pages of a warp: the one it works on and those on their way
  static constexpr int kWarpBytes = kStages * kStageBytes;
  // Where a page's 16-byte pieces lie, so that neither copies nor reads meet on a bank: piece c of a token's key; of the values of
  // token 2t + (j & 1) + 8 (j >> 1).
  static __device__ __forceinline__ uint32_t key_at(int tok, int c) { return tok * HD + ((HD == 128 ? c ^ ((tok & 1) << 2) : c) << 4); }
  static __device__ __forceinline__ uint32_t value_at(int j, int t, int c) {
    return (j * 4 + t) * HD + ((HD == 128 ? c ^ (t << 1) : c ^ (t & 2)) << 4);
  }
};

// A softmax state for one head, spread over the lanes of a warp: HD / 32 elements each.
template <int HD>
struct Row {
  static constexpr int N = HD / 32;
  float m = -INFINITY, l = 0.f, o[N] = {};
  __device__ __forceinline__ void add(const Row& y) {
    const float top = fmaxf(m, y.m), safe = top == -INFINITY ? 0.f : top;
    const float a = q8_exp2(m - safe), b = q8_exp2(y.m - safe);
    l = l * a + y.l * b;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * a + y.o[i] * b;
    m = top;
  }
  // A piece as the warps write it: rows of HD, behind them a (reference, sum) for each.
  __device__ __forceinline__ void read(const float* piece, int group, int h) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 v = *reinterpret_cast<const float2*>(piece + h * HD + lane * N + i);
      o[i] = v.x;
      o[i + 1] = v.y;
    }
    const float2 s = *reinterpret_cast<const float2*>(piece + group * HD + 2 * h);
    m = s.x;
    l = s.y;
  }
  __device__ __forceinline__ void store(float* ml, float* row) const {
    const int lane = threadIdx.x & 31;
    if constexpr (HD == 128) __stcg(reinterpret_cast<float4*>(row) + lane, make_float4(o[0], o[1], o[2], o[3]));
    else __stcg(reinterpret_cast<float2*>(row) + lane, make_float2(o[0], o[1]));
    if (lane == 0) __stcg(reinterpret_cast<float2*>(ml), make_float2(m, l));
  }
  __device__ __forceinline__ void finish(__nv_bfloat16* out) const {
    const int lane = threadIdx.x & 31;
    const float inv = l == 0.f ? 0.f : 1.f / l;                // (a sum that is NaN stays visible)
    if constexpr (HD == 128)
      reinterpret_cast<uint2*>(out)[lane] = make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
    else
      reinterpret_cast<uint32_t*>(out)[lane] = pack_bf16x2(o[0] * inv, o[1] * inv);
  }
};

// Sum of n states in the workspace, the i-th in row at(i), in their order. Lanes fetch 32 references and sums at a time, so that
// the rows are requested without waiting for one another.
template <int HD, class At>
__device__ __forceinline__ Row<HD> sum_rows(const float* ml, const float* o, int n, At at) {
  const int lane = threadIdx.x & 31;
  Row<HD> all;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int here = min(32, n - i0);
    const long long mine = at(i0 + min(lane, here - 1));
    const float2 s = __ldcg(reinterpret_cast<const float2*>(ml) + mine);
    Row<HD> part;
    part.m = s.x;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) part.m = fmaxf(part.m, __shfl_xor_sync(0xffffffffu, part.m, off));
    const float w = lane < here ? q8_exp2(s.x - (part.m == -INFINITY ? 0.f : part.m)) : 0.f;
    part.l = lane < here ? s.y * w : 0.f;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) part.l += __shfl_xor_sync(0xffffffffu, part.l, off);
    for (int i = 0; i < here; i += 8) {
      float x[8][Row<HD>::N];
#pragma unroll
      for (int k = 0; k < 8; ++k) {                            // (rows behind the last: that one again, times zero)
        const float* row = o + __shfl_sync(0xffffffffu, mine, min(i + k, here - 1)) * HD;
        if constexpr (HD == 128) {
          const float4 v = __ldcg(reinterpret_cast<const float4*>(row) + lane);
          x[k][0] = v.x; x[k][1] = v.y; x[k][2] = v.z; x[k][3] = v.w;
        } else {
          const float2 v = __ldcg(reinterpret_cast<const float2*>(row) + lane);
          x[k][0] = v.x; x[k][1] = v.y;
        }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float by = i + k < here ? __shfl_sync(0xffffffffu, w, i + k) : 0.f;
        if (i + k < here)
#pragma unroll
          for (int e = 0; e < Row<HD>::N; ++e) part.o[e] += by * x[k][e];
      }
    }
    if (i0 == 0) all = part;
    else all.add(part);
  }
  return all;
}

// What the shared prefix gives for head `h` of KV head `kvh` of request `r`.
template <int HD>
__device__ __forceinline__ Row<HD> prefix_row(const PrefixPlan& f, int kv_heads, int group, int kvh, int r, int h) {
  const Ranges ranges(prefix_units(f, kv_heads), f.ctas);
  const int item = kvh * f.blocks + r / f.reqs_per_block, row = r % f.reqs_per_block * group + h;
  const int c0 = ranges.of(item * f.tiles), c1 = ranges.of((item + 1) * f.tiles - 1);
  return sum_rows<HD>(f.ml, f.o, c1 - c0 + 1, [&](int i) { return static_cast<long long>(item + c0 + i) * kPrefixRows + row; });
}

// A piece that a warp leaves for its CTA: what its range holds of a request for a KV head.
struct Piece {
  int kvh, r, tok, begin, end;     // request (from req_begin), its row of q, its pages in the row of pages
  int flags;                       // 1 there is one, 2 the request starts in it, 4 ends in it
};
// A request of which a CTA holds a part only: the first of the CTAs that do and their number; `last`: the others' parts are left.
struct Part {
  int kvh, r, tok, first, n, last;
};

template <int HD, int NT, int KIND, bool SHARED>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 4 : 3)
attn_decode_q8_kernel(nfk_attn_q8_params p, PrefixPlan f, unsigned int* counts, float* part_ml, float* part_o, float* kept) {
  using D = Dec<HD>;
  constexpr int KS = HD / 16, MT = HD / 16, VB = HD / 8;      // steps of Q K^T, row tiles of V^T, bytes of a token's values per lane
  constexpr int ST = D::kStages;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Piece pieces[2 * kWarps];
  __shared__ Part parts[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int group = p.q_heads / p.kv_heads, ctas = gridDim.x;
  const int* indptr = p.kv_indptr + p.req_begin;
  const int base = indptr[0];
  const long long listed = static_cast<long long>(indptr[p.req_count]) - base;
  bool listed_well = base >= 0 && listed >= 0 && base + listed <= p.num_indices;       // else nothing is read
  const int pages_all = listed_well ? static_cast<int>(listed) : 0;
  const int units = pages_all * p.kv_heads, workers = min(units, ctas * kWarps);
  const Ranges ranges(units, workers);
  const float scale = p.sm_scale * kQ8Log2e;
  __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(p.out);

  auto row_of = [&](int r) {                                   // the request's row of q and out
    const int tok = p.qo_indptr[p.req_begin + r];
    if (tok >= 0 && tok < p.num_tokens) return tok;
    if (lane == 0) report_status(p.status, NF_ST_BAD_INDEX);
    return -1;
  };

  // A warp's places for pieces: of its range's last run over its pipeline, which is done by then; of the first run in the workspace,
  // and behind those of all warps that of a request which lies within the range and waits for the prefix's share.
  static_assert(D::kWarpBytes >= 8 * NT * (HD + 2) * 4, "a piece lies over its warp's pipeline");
  const int piece_floats = group * (HD + 2);
  const uint32_t pipe = smem_u32(smem) + warp * D::kWarpBytes;
  auto piece_at = [&](int k) {                                 // warp k / 2, its first (0) or last (1) run
    return (k & 1) ? reinterpret_cast<float*>(smem + (k >> 1) * D::kWarpBytes)
                   : kept + (static_cast<long long>(blockIdx.x) * kWarps + (k >> 1)) * piece_floats;
  };

  // ---- loads: unit i of the range is page (u0 + i) % pages_all of KV head (u0 + i) / pages_all ----
  int n = 0, kvh = 0, at = 0;                                  // units of the range; KV head and place in the row of pages of the next one
  int i_kvh = 0, i_page = 0, ids = 0, ids_left = 0;            // of the next one to load; page numbers, one per lane, 32 at a time
  const uint8_t* pool = reinterpret_cast<const uint8_t*>(p.kv_pool);
  auto issue = [&](int i) {
    if (i < n) {
      if (ids_left == 0) {
        ids_left = min(32, pages_all - i_page);
        ids = lane < ids_left ? p.kv_indices[base + i_page + lane] : 0;
        if (ids < 0 || ids >= p.num_pages) {
          report_status(p.status, NF_ST_BAD_INDEX);
          ids = 0;
        }
      }
      const int page = __shfl_sync(0xffffffffu, ids, 0);       // lane 0 holds the next one
      ids = __shfl_down_sync(0xffffffffu, ids, 1);
      --ids_left;
      const long long head = static_cast<long long>(page) * 2 * p.kv_heads + i_kvh;
      const uint8_t* k = pool + head * D::kKeyBytes;
      const uint8_t* v = k + static_cast<long long>(p.kv_heads) * D::kKeyBytes;
      const uint32_t st = pipe + i % ST * D::kStageBytes;
      // eight (head_dim 64: four) neighbouring lanes take a token's row: a sector asked for by itself comes at half the rate
#pragma unroll
      for (int y = 0; y < HD / 32; ++y) {
        const int tok = y * (512 / HD) + lane / (HD / 16), c = lane % (HD / 16);
        cp_async16(st + D::key_at(tok, c), k + tok * HD + c * 16);
        cp_async16(st + D::kKeyBytes + D::value_at((tok & 1) + (tok >> 3) * 2, (tok >> 1) & 3, c), v + tok * HD + c * 16);
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
  // The request that a place in the row of pages belongs to: the last whose pages start at or before it, 32 candidates at a time.
  auto find = [&](int place) {
    int lo = 0, hi = p.req_count;                              // it is in [lo, hi)
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32;
      const int r = lo + lane * step;
      const unsigned int before = __ballot_sync(0xffffffffu, r < hi && indptr[r] - base <= place);
      lo += (31 - __clz(before)) * step;                       // (lane 0's is one: lo starts at or before the place)
      hi = min(hi, lo + step);
    }
    return lo;
  };

  const int w = blockIdx.x * kWarps + warp;
  if (w < workers) {
    const int u0 = ranges.begin(w);
    n = ranges.begin(w + 1) - u0;
    i_kvh = kvh = u0 / pages_all;
    i_page = at = u0 - kvh * pages_all;
#pragma unroll
    for (int s = 0; s < ST - 1; ++s) issue(s);
  }
  // (while the first pages are on their way)
  int seen = 0;
  for (int r = threadIdx.x; r < p.req_count; r += kThreads) {
    const int own = indptr[r + 1] - indptr[r];
    seen |= own < 0 ? 1 : own == 0 ? 2 : 0;
  }
  if (lane < 2) pieces[warp * 2 + lane].flags = 0;
  if (threadIdx.x < 2) parts[threadIdx.x].n = 0;
  listed_well = __syncthreads_or(seen & 1) == 0 && listed_well;
  const bool some_empty = __syncthreads_or(seen & 2) != 0 || pages_all == 0 || !listed_well;
  if (!listed_well) {
    if (threadIdx.x == 0) report_status(p.status, NF_ST_BAD_INDEX);
    n = 0;
  }

  int r = n > 0 ? find(at) : 0;
  for (int i = 0; i < n;) {
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
      cp_async_wait<ST - 2>();
      __syncwarp();                                          // the page is there, and no lane looks at the one before any more
      issue(i + ST - 1);
      const uint32_t st = pipe + i % ST * D::kStageBytes;
      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int x = 0; x < HD / 64; ++x) {
        const uint4 a = ld_shared_v4(st + D::key_at(g, x * 4 + t)), b = ld_shared_v4(st + D::key_at(g + 8, x * 4 + t));
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
        const uint32_t from = st + D::kKeyBytes + (HD == 128 ? D::value_at(j, t, g) : D::value_at(j, t, g >> 1) + (g & 1) * 8);
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
    auto leave = [&](float* piece) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int h = nt * 8 + 2 * t + e;
          if (h >= group) continue;
          if (g == 0) *reinterpret_cast<float2*>(piece + group * HD + 2 * h) = make_float2(ref[nt][e], l[nt][e]);
#pragma unroll
          for (int j = 0; j < MT; ++j)
            *reinterpret_cast<float2*>(piece + h * HD + g * VB + 2 * j) = make_float2(o[nt][j][e] * v_back, o[nt][j][2 + e] * v_back);
        }
    };
    if (whole && !SHARED) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int h = nt * 8 + 2 * t + e;
          if (h >= group || tok < 0) continue;
          const float inv = l[nt][e] == 0.f ? 0.f : v_back / l[nt][e];
          uint4* dst = reinterpret_cast<uint4*>(out + (static_cast<long long>(tok) * p.q_heads + kvh * group + h) * HD + g * VB);
#pragma unroll
          for (int j = 0; j < MT; j += 4)
            dst[j / 4] = make_uint4(pack_bf16x2(o[nt][j][e] * inv, o[nt][j][2 + e] * inv), pack_bf16x2(o[nt][j + 1][e] * inv, o[nt][j + 1][2 + e] * inv),
                                    pack_bf16x2(o[nt][j + 2][e] * inv, o[nt][j + 2][2 + e] * inv), pack_bf16x2(o[nt][j + 3][e] * inv, o[nt][j + 3][2 + e] * inv));
        }
    } else if (whole && !last_run) {                         // the warp joins it with the prefix itself
      float* piece = kept + (static_cast<long long>(ctas + blockIdx.x) * kWarps + warp) * piece_floats;
      leave(piece);
      await_previous();
      __syncwarp();
      for (int h = 0; h < group; ++h) {
        Row<HD> row;
        row.read(piece, group, h);
        row.add(prefix_row<HD>(f, p.kv_heads, group, kvh, r, h));
        if (tok >= 0) row.finish(out + (static_cast<long long>(tok) * p.q_heads + kvh * group + h) * HD);
      }
      __syncwarp();
    } else {                                                 // a run that is neither whole nor the last is the first
      const int k = warp * 2 + (last_run ? 1 : 0);
      if (last_run) __syncwarp();                            // no lane looks at its last page any more
      leave(piece_at(k));
      if (lane == 0) pieces[k] = Piece{kvh, r, tok, r_begin, r_end, 1 | (starts ? 2 : 0) | (ends ? 4 : 0)};
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
  if (SHARED) await_previous();
  __syncthreads();

  // ---- requests without pages of their own: zeros, or the prefix alone ----
  if (some_empty)
    for (int e = blockIdx.x * kWarps + warp; e < p.req_count * p.q_heads; e += ctas * kWarps) {
      const int er = e / p.q_heads, head = e - er * p.q_heads;
      if (listed_well && indptr[er + 1] > indptr[er]) continue;
      const int tok = row_of(er);
      Row<HD> row;
      if (SHARED) row = prefix_row<HD>(f, p.kv_heads, group, head / group, er, head % group);
      if (tok >= 0) row.finish(out + (static_cast<long long>(tok) * p.q_heads + head) * HD);
    }

  // ---- pieces of the CTA's warps, joined request by request. Of a request that goes on in another CTA a part is left in the
  // workspace: at most one that began before this CTA's pages (side 0) and one that begins in them (side 1). ----
  bool left = false;
  for (int first = 0; first < 2 * kWarps; ++first) {
    const Piece piece = pieces[first];
    if (piece.flags == 0) continue;
    int last = first;
    for (int k = first + 1; k < 2 * kWarps; ++k)
      if (pieces[k].flags != 0) {
        if (pieces[k].kvh != piece.kvh || pieces[k].r != piece.r) break;
        last = k;
      }
    const bool starts = (piece.flags & 2) != 0, ends = (pieces[last].flags & 4) != 0, inside = starts && ends;
    if (!inside && threadIdx.x == kThreads - 1) {            // the CTAs that hold parts of the request follow from the ranges
      const int c0 = ranges.of(piece.kvh * pages_all + piece.begin) / kWarps, c1 = ranges.of(piece.kvh * pages_all + piece.end - 1) / kWarps;
      parts[starts ? 1 : 0] = Part{piece.kvh, piece.r, piece.tok, c0, c1 - c0 + 1, 0};
    }
    left = left || !inside;
    for (int h = warp; h < group; h += kWarps) {
      Row<HD> row;
      for (int k = first; k <= last; ++k) {
        if (pieces[k].flags == 0) continue;
        Row<HD> one;
        one.read(piece_at(k), group, h);
        row.add(one);
      }
      if (inside) {
        if (SHARED) row.add(prefix_row<HD>(f, p.kv_heads, group, piece.kvh, piece.r, h));
        if (piece.tok >= 0) row.finish(out + (static_cast<long long>(piece.tok) * p.q_heads + piece.kvh * group + h) * HD);
      } else {
        const long long to = (static_cast<long long>(blockIdx.x) * 2 + (starts ? 1 : 0)) * group + h;
        row.store(part_ml + to * 2, part_o + to * HD);
      }
    }
    first = last;
  }
  if (left) {
    __syncthreads();
    if (threadIdx.x < 2 && parts[threadIdx.x].n > 0) {
      Part& part = parts[threadIdx.x];
      __threadfence();
      if (atomicAdd(counts + part.first, 1u) == static_cast<unsigned int>(part.n - 1)) {
        counts[part.first] = 0u;
        part.last = 1;
        __threadfence();
      }
    }
    __syncthreads();
    // the last of a request's parts to be left: all of them, in their order
    for (int side = 0; side < 2; ++side) {
      const Part part = parts[side];
      if (part.n == 0 || part.last == 0) continue;
      for (int h = warp; h < group; h += kWarps) {
        Row<HD> row = sum_rows<HD>(part_ml, part_o, part.n,
                                   [&](int i) { return (static_cast<long long>(part.first + i) * 2 + (i == 0 ? 1 : 0)) * group + h; });
        if (SHARED) row.add(prefix_row<HD>(f, p.kv_heads, group, part.kvh, part.r, h));
        if (part.tok >= 0) row.finish(out + (static_cast<long long>(part.tok) * p.q_heads + part.kvh * group + h) * HD);
      }
    }
  }
}

template <int HD, int NT, int KIND, bool SHARED>
int launch_decode(const nfk_attn_q8_params& p, const PrefixPlan& f, const Q8Workspace& ws, cudaStream_t stream) {
  constexpr int bytes = kWarps * Dec<HD>::kWarpBytes;
  static int fit_dev[kMaxDevices] = {0};                       // CTAs that fit an SM
  int& fit = fit_dev[device_slot()];
  const auto kernel = attn_decode_q8_kernel<HD, NT, KIND, SHARED>;
  if (fit == 0) {
    int per_sm = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kThreads, bytes) != cudaSuccess || per_sm < 1) {
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
                    reinterpret_cast<float*>(base + ws.ml), reinterpret_cast<float*>(base + ws.o), reinterpret_cast<float*>(base + ws.kept)) == cudaSuccess)
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
      p->num_indices < 0 || static_cast<long long>(p->num_indices) * p->kv_heads > 0x7fffffffll ||
      static_cast<long long>(p->req_count) * p->q_heads > 0x7fffffffll || p->num_ctas < 0 || !aligned16(p->q) || !aligned16(p->out) || !aligned16(p->kv_pool) ||
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
