// Attention of one query token per request over the 8-bit paged cache.
//
//   o_h = sum_j e^(s_hj) v_j / sum_j e^(s_hj),   s_hj = sm_scale (q_h . k_j),   k_j = number_j * kscale_j, v_j likewise
//
// Bound by the cache's bytes: 683 requests of 1024 to 1536 tokens, 32 / 8 heads, 316 us, 5.8 TB/s, 0.89 of a copy's rate; 256
// requests of 200 to 2000, 64 / 8 heads, 93 us, 0.74 (83 without the join). A warp reads pages straight into the layout that the
// tensor cores take: with S^T = K Q^T the keys are the 16-row operand (a page's 16 tokens) and the up to 8 query heads of a KV head
// the 8 columns (16 heads: two such products), and which elements of head_dim form a step of the product is free, so a lane's bytes
// of a key are 16 neighbours, its f16 pairs the operand's registers, and no lane needs what another one loaded. O^T = V^T P^T works
// the same way: V^T is the 16-row operand, two of its rows are two neighbouring elements, and a lane reads 16 neighbours of the
// four tokens whose weights it multiplies. P^T gets into its layout by one transposing move per 8 tokens.
// Numbers are exact in f16. Queries are, too, up to a power of two per head (their small elements may be rounded at 2^-25 of the
// largest). The keys' scales join the scores in fp32; the values' scales join the weights, which are rounded to f16 (2^-11)
// relative to the largest value scale so far, `v_ref`, with 2^7 of headroom: values up to 2^20 smaller keep full precision.
//
// A warp keeps a reference per head instead of a running maximum: it moves only where a score exceeds it by 8 (in exponents to
// base 2), so that the common page has one vote and no reduction across lanes; sums stay per lane until a request ends.
//
// All pages of all requests, one KV head after the other, are a row that is cut into ranges for single warps, without regard to where
// a request ends (attn_q8.cuh). A warp writes the rows of requests that lie within one of its ranges; of others it leaves states in
// the workspace, and a second kernel joins them, and the shared prefix's where there is one. Warps wait for nothing but their pages.
#include "attn_q8.cuh"
#include "attn_mma.cuh"

namespace nf {
namespace {

constexpr int kWarps = kDecodeWarps, kThreads = 32 * kWarps;
constexpr int kListed = 1000;
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

// Who writes rows of requests: the first kernel those in one range, the second one the others (PLAIN); the second one all, with the
// prefix's share (SHARED_PREFIX); the first one all (FEW, for small batches).
enum { PLAIN = 0, SHARED_PREFIX = 1, FEW = 2 };

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

// A softmax state for one head, spread over the lanes of a warp: HD / 32 elements each (see kStateUnit).
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
  __device__ __forceinline__ void finish(__nv_bfloat16* out) const {
    const int lane = threadIdx.x & 31;
    const float inv = l == 0.f ? 0.f : 1.f / (kStateUnit * l);                // (a sum that is NaN stays visible)
    if constexpr (HD == 128)
      reinterpret_cast<uint2*>(out)[lane] = make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
    else
      reinterpret_cast<uint32_t*>(out)[lane] = pack_bf16x2(o[0] * inv, o[1] * inv);
  }
};

// States in the workspace, [..][group or heads]: (reference, sum) and rows of head_dim.
struct States {
  float* ml;
  float* o;
};
// One of them: its reference and sum, and the place of its row, counted in 16 bytes from the workspace's begin.
struct State {
  float2 ml;
  unsigned int row;
};
template <int HD>
__device__ __forceinline__ State state_at(const void* workspace, const float* ml, const float* o, unsigned int i) {
  return State{__ldcg(reinterpret_cast<const float2*>(ml) + i),
               static_cast<unsigned int>((reinterpret_cast<const char*>(o) - static_cast<const char*>(workspace)) >> 4) + i * (HD / 4)};
}
// Sums of n states for H neighbouring heads, the i-th of head k being at(i, k), in their order. Lanes fetch 32 references and sums at
// a time and AHEAD rows of each head are requested without waiting for one another.
template <int HD, int AHEAD, int H, class At>
__device__ __forceinline__ void sum_states(const void* workspace, int n, At at, Row<HD> (&all)[H]) {
  constexpr int N = Row<HD>::N;
  const int lane = threadIdx.x & 31;
  const char* base = static_cast<const char*>(workspace) + lane * (N * 4);
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int here = min(32, n - i0);
    State mine[H];
#pragma unroll
    for (int k = 0; k < H; ++k) mine[k] = at(i0 + min(lane, here - 1), k);
    Row<HD> part[H];
    float w[H] = {};
    for (int i = 0; i < here; i += AHEAD) {
      float x[AHEAD][H][N];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        if (i + j >= here) break;
        const char* row = base + (static_cast<unsigned long long>(__shfl_sync(0xffffffffu, mine[0].row, i + j)) << 4);
#pragma unroll
        for (int k = 0; k < H; ++k)
          if constexpr (HD == 128) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(row + k * (HD * 4)));
            x[j][k][0] = v.x; x[j][k][1] = v.y; x[j][k][2] = v.z; x[j][k][3] = v.w;
          } else {
            const float2 v = __ldcg(reinterpret_cast<const float2*>(row + k * (HD * 4)));
            x[j][k][0] = v.x; x[j][k][1] = v.y;
          }
      }
      if (i == 0)                                              // (while the first rows are on their way)
#pragma unroll
        for (int k = 0; k < H; ++k) {
          part[k].m = mine[k].ml.x;
#pragma unroll
          for (int off = 16; off > 0; off >>= 1) part[k].m = fmaxf(part[k].m, __shfl_xor_sync(0xffffffffu, part[k].m, off));
          w[k] = lane < here ? q8_exp2(mine[k].ml.x - (part[k].m == -INFINITY ? 0.f : part[k].m)) : 0.f;
          part[k].l = mine[k].ml.y * w[k];
#pragma unroll
          for (int off = 16; off > 0; off >>= 1) part[k].l += __shfl_xor_sync(0xffffffffu, part[k].l, off);
        }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        if (i + j >= here) break;
#pragma unroll
        for (int k = 0; k < H; ++k) {
          const float by = __shfl_sync(0xffffffffu, w[k], i + j);
#pragma unroll
          for (int e = 0; e < N; ++e) part[k].o[e] += by * x[j][k][e];
        }
      }
    }
#pragma unroll
    for (int k = 0; k < H; ++k) {
      if (i0 == 0) all[k] = part[k];
      else all[k].add(part[k]);
    }
  }
}

__device__ __forceinline__ float2 ld_cluster_f32x2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}

// FEW: the warps of a cluster take equal shares of one request's pages for one KV head, and join in distributed shared memory.
template <int HD, int NT, int KIND, int MODE>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 4 : HD == 64 ? 3 : 2)
attn_decode_q8_kernel(nfk_attn_q8_params p, int* bad_lists, DecodeRecord* records, States parts, States wholes) {
  using D = Dec<HD>;
  constexpr int KS = HD / 16, MT = HD / 16, VB = HD / 8;      // steps of Q K^T, row tiles of V^T, bytes of a token's values per lane
  constexpr int ST = D::kStages;
  constexpr bool SHARED = MODE == SHARED_PREFIX;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int starts[kListed + 1];                          // places of the requests' first pages in the row, for up to kListed requests
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int group = p.q_heads / p.kv_heads;
  // (A prefix's kernel lets this one read without a wait, see let_next_read.)
  const Early<int, SHARED> indptr{p.kv_indptr + p.req_begin}, indices{p.kv_indices}, rows{p.qo_indptr + p.req_begin},
      last_lens{p.kv_last_page_len + p.req_begin};
  if (!SHARED) await_previous();
  if (MODE != PLAIN) let_next_start();
  else if (warp == kWarps - 1) let_next_read();                // for the kernel that joins states
  const int base = indptr[0];
  const bool in_shared = p.req_count <= kListed;
  auto start_of = [&](int r) { return in_shared ? starts[r] : indptr[r] - base; };
  const long long listed = static_cast<long long>(indptr[p.req_count]) - base;
  bool listed_well = base >= 0 && listed >= 0 && base + listed <= p.num_indices;       // else nothing is read
  const int pages_all = listed_well ? static_cast<int>(listed) : 0;
  const int n_ranges = decode_ranges(pages_all * p.kv_heads, gridDim.x);
  const Ranges ranges(pages_all * p.kv_heads, n_ranges);
  const float scale = p.sm_scale * kQ8Log2e;
  __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(p.out);

  // ---- loads: the pages of this warp's range ----
  const int range = blockIdx.x * kWarps + warp;
  int n = 0, kvh = 0, at = 0, r = 0;                           // pages; of the next one to work on: KV head, place in the row, request
  if (MODE == FEW) {
    const int size = gridDim.x / (p.req_count * p.kv_heads), which = blockIdx.x / size;
    r = which / p.kv_heads;
    kvh = which - r * p.kv_heads;
    const int begin = indptr[r] - base, own = indptr[r + 1] - base - begin, share = static_cast<int>(cluster_ctarank()) * kWarps + warp;
    if (begin >= 0 && own > 0 && begin + own <= pages_all) {
      const Ranges shares(own, size * kWarps);
      at = begin + shares.begin(share);
      n = begin + shares.begin(share + 1) - at;
    }
  } else if (range < n_ranges) {
    const int u0 = ranges.begin(range);
    n = ranges.begin(range + 1) - u0;
    kvh = u0 / pages_all;
    at = u0 - kvh * pages_all;
  }
  const uint32_t pipe = smem_u32(smem) + warp * D::kWarpBytes;
  const uint8_t* pool = reinterpret_cast<const uint8_t*>(p.kv_pool);
  int i_left = n, i_kvh = kvh, i_page = at;                    // of the next one to load; pages that are left
  int ids = 0, ids_left = 0;                                   // page numbers, one per lane, 32 at a time
  uint32_t to = pipe;                                          // the stage that is loaded next
  const States own_states = {reinterpret_cast<float*>(smem + warp * D::kWarpBytes) + group * HD, reinterpret_cast<float*>(smem + warp * D::kWarpBytes)};
  static_assert(D::kWarpBytes >= 8 * NT * (HD + 2) * 4, "a state of all heads lies over the pipeline");
  auto issue = [&]() {
    if (i_left > 0) {
      if (ids_left == 0) {
        ids_left = min(32, pages_all - i_page);
        ids = lane < ids_left ? indices[base + i_page + lane] : 0;
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
      // Eight (head_dim 64: four) neighbouring lanes take a token's row. With a sector to each quarter of the warp L2 had twice as
      // many requests to answer: 683 requests of 1024 to 1536 tokens, 378 us instead of 318.
#pragma unroll
      for (int y = 0; y < HD / 32; ++y) {
        const int tok = y * (512 / HD) + lane / (HD / 16), c = lane % (HD / 16);
        cp_async16(to + D::key_at(tok, c), k + tok * HD + c * 16);
        cp_async16(to + D::kKeyBytes + D::value_at((tok & 1) + (tok >> 3) * 2, (tok >> 1) & 3, c), v + tok * HD + c * 16);
      }
      if (lane < 8) cp_async16(to + 2 * D::kKeyBytes + lane * 16, p.kv_scale + (head + (lane >> 2) * p.kv_heads) * kQ8Page + (lane & 3) * 4);
      --i_left;
      if (++i_page == pages_all) {
        i_page = 0;
        ++i_kvh;
        ids_left = 0;
      }
    }
    to = to + D::kStageBytes == pipe + D::kWarpBytes ? pipe : to + D::kStageBytes;
    cp_async_commit();
  };
  // The request that a place in the row of pages belongs to: the last whose pages start at or before it, 32 candidates at a time.
  auto find = [&](int place) {
    int lo = 0, hi = p.req_count;                              // it is in [lo, hi)
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32;
      const int r = lo + lane * step;
      const unsigned int before = __ballot_sync(0xffffffffu, r < hi && start_of(r) <= place);
      lo += (31 - __clz(before)) * step;                       // (lane 0's is one: lo starts at or before the place)
      hi = min(hi, lo + step);
    }
    return lo;
  };

  auto row_of = [&](int r) {                                   // the request's row of q and out
    const int tok = rows[r];
    if (tok >= 0 && tok < p.num_tokens) return tok;
    if (lane == 0) report_status(p.status, NF_ST_BAD_INDEX);
    return -1;
  };

#pragma unroll
  for (int s = 0; s < ST - 1; ++s) issue();
  // (while the first pages are on their way: the lists must go up, or runs of pages would have no end)
  bool falls = false, none = false;
  for (int r = threadIdx.x; r < p.req_count; r += kThreads) {
    const int start = indptr[r], own = indptr[r + 1] - start;
    if (in_shared) starts[r] = start - base;
    falls = falls || own < 0;
    none = none || own == 0;
  }
  if (in_shared && threadIdx.x == 0) starts[p.req_count] = pages_all;
  listed_well = __syncthreads_or(falls ? 1 : 0) == 0 && listed_well;
  // requests without pages: zeros (with a prefix the other kernel's)
  if (MODE == PLAIN && (__syncthreads_or(none ? 1 : 0) != 0 || !listed_well))
    for (int e = range; e < p.req_count * p.q_heads; e += gridDim.x * kWarps) {
      const int er = e / p.q_heads, tok = !listed_well || start_of(er + 1) == start_of(er) ? row_of(er) : -1;
      if (tok >= 0) Row<HD>().finish(out + (static_cast<long long>(tok) * p.q_heads + e - er * p.q_heads) * HD);
    }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    if (MODE != FEW) *bad_lists = listed_well ? 0 : 1;
    if (!listed_well) report_status(p.status, NF_ST_BAD_INDEX);
  }

  DecodeRecord record = {0, 0, 0, 0};
  if (listed_well && n > 0) {
    uint32_t st = pipe;                                        // the stage that is worked on
    if (MODE != FEW) r = find(at);
    for (int i = 0; i < n;) {
      // ---- a request's run of pages in this range ----
      const int last_len = last_lens[r];
      const int tok = row_of(r);
      const int r_begin = start_of(r), r_end = start_of(r + 1);
      const int count = min(n - i, r_end - at);
      const bool begins = at == r_begin, ends = at + count == r_end;
      uint32_t qb[NT][KS][2];
      float q_up[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int h = nt * 8 + g;
        const bool on = tok >= 0 && h < group;
        const Early<uint4, SHARED> src{reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(p.q) +
                                                                      (static_cast<long long>(on ? tok : 0) * p.q_heads + kvh * group + (on ? h : 0)) * HD) + t * 2};
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
        issue();
        float s[NT][4], s_odd[NT][4];                          // sums of even and of odd steps: half as long a chain of products
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][e] = s_odd[nt][e] = 0.f;
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
            for (int nt = 0; nt < NT; ++nt) mma_f16((e & 1) ? s_odd[nt] : s[nt], a0, a1, a2, a3, qb[nt][x * 4 + e][0], qb[nt][x * 4 + e][1]);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][e] += s_odd[nt][e];
        const uint32_t sc = st + 2 * D::kKeyBytes;
        const int valid = ends && c == count - 1 ? last_len : kQ8Page;
        const bool on0 = g < valid, on1 = g + 8 < valid;
        const float k0 = ld_shared_f32(sc + g * 4), k1 = ld_shared_f32(sc + g * 4 + 32);
        const float v0 = on0 ? ld_shared_f32(sc + 64 + g * 4) : 0.f, v1 = on1 ? ld_shared_f32(sc + 96 + g * 4) : 0.f;
        bool grow = fabsf(v0) > v_ref || fabsf(v1) > v_ref;
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
          float most = fmaxf(v_ref, fmaxf(fabsf(v0), fabsf(v1)));
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
        st = st + D::kStageBytes == pipe + D::kWarpBytes ? pipe : st + D::kStageBytes;
      }

      // ---- the run's end: the final row where it is the whole request and no prefix joins it, else its state ----
      const float v_back = v_ref / kHeadroom, s_back = v_back * kStateUnit;
      const bool final = begins && ends && MODE == PLAIN;
      // states of this run's heads: of a whole request by its number; of a piece by the range's, those of a request that began before
      // it first; in a cluster over the warp's own pipeline, which is done
      States states = begins && ends ? wholes : parts;
      long long first = begins && ends ? static_cast<long long>(r) * p.q_heads + kvh * group
                                       : (static_cast<long long>(range) * 2 + (begins ? 1 : 0)) * group;
      if (MODE == FEW) {
        states = own_states;
        first = 0;
        __syncwarp();
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], off);
          const int h = nt * 8 + 2 * t + e;
          if (h >= group) continue;
          if (final) {
            if (tok < 0) continue;
            const float inv = l[nt][e] == 0.f ? 0.f : v_back / l[nt][e];
            uint4* dst = reinterpret_cast<uint4*>(out + (static_cast<long long>(tok) * p.q_heads + kvh * group + h) * HD + g * VB);
#pragma unroll
            for (int j = 0; j < MT; j += 4)
              dst[j / 4] = make_uint4(pack_bf16x2(o[nt][j][e] * inv, o[nt][j][2 + e] * inv), pack_bf16x2(o[nt][j + 1][e] * inv, o[nt][j + 1][2 + e] * inv),
                                      pack_bf16x2(o[nt][j + 2][e] * inv, o[nt][j + 2][2 + e] * inv), pack_bf16x2(o[nt][j + 3][e] * inv, o[nt][j + 3][2 + e] * inv));
          } else {
            if (g == 0) *reinterpret_cast<float2*>(states.ml + (first + h) * 2) = make_float2(ref[nt][e], l[nt][e]);
            float4* dst = reinterpret_cast<float4*>(states.o + (first + h) * HD + g * VB);
#pragma unroll
            for (int j = 0; j < MT; j += 2)
              dst[j / 2] = make_float4(o[nt][j][e] * s_back, o[nt][j][2 + e] * s_back, o[nt][j + 1][e] * s_back, o[nt][j + 1][2 + e] * s_back);
          }
        }

      if (begins && !ends) record = DecodeRecord{kvh, r, tok, ranges.of(kvh * pages_all + r_end - 1) - range + 1};

      // ---- the next request that has pages ----
      at += count;
      if (i < n) {
        if (at == pages_all) {
          at = 0;
          ++kvh;
        }
        r = r + 1 < p.req_count && at > 0 && start_of(r + 2) > at ? r + 1 : find(at);
      }
    }
  }
  if (MODE == FEW) {
    cp_async_wait<0>();
    __syncwarp();
    if (!listed_well || n == 0)                                // no share of the pages: an empty state
      for (int e = lane; e < group * (HD + 2); e += 32) own_states.o[e] = e >= group * HD && (e & 1) == 0 ? -INFINITY : 0.f;
    cluster_sync_all();
    const int size = gridDim.x / (p.req_count * p.kv_heads), states = size * kWarps, tok = row_of(r);
    for (int h = static_cast<int>(cluster_ctarank()) * kWarps + warp; h < group; h += states) {
      // state i: of warp i % kWarps in CTA i / kWarps
      const auto state = [&](int i) { return mapa_shared(smem_u32(smem) + i % kWarps * D::kWarpBytes, i / kWarps); };
      const float2 s = ld_cluster_f32x2(state(min(lane, states - 1)) + (group * HD + 2 * h) * 4);
      float m = s.x;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
      const float w = lane < states ? q8_exp2(s.x - (m == -INFINITY ? 0.f : m)) : 0.f;
      Row<HD> row;
      row.m = m;
      row.l = lane < states ? s.y * w : 0.f;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) row.l += __shfl_xor_sync(0xffffffffu, row.l, off);
      for (int i = 0; i < states; i += kWarps)
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
          const float by = __shfl_sync(0xffffffffu, w, i + k);
          const uint32_t from = state(i + k) + (h * HD + lane * Row<HD>::N) * 4;
#pragma unroll
          for (int e = 0; e < Row<HD>::N; e += 2) {
            const float2 x = ld_cluster_f32x2(from + e * 4);
            row.o[e] += by * x.x;
            row.o[e + 1] += by * x.y;
          }
        }
      if (tok >= 0) row.finish(out + (static_cast<long long>(tok) * p.q_heads + kvh * group + h) * HD);
    }
    cluster_sync_all();                                        // no CTA's shared memory goes before all have read it
  } else {
    if (lane == 0) records[range] = record;
    cp_async_wait<0>();
    // One CTA stays until the prefix's kernel is complete, so that this one is not complete before it. With all of them
    // 64 requests behind 32768 tokens took 115 us instead of 110: SMs that have ended their share of the prefix would hold this kernel's
    // first CTAs.
    if (SHARED && blockIdx.x == gridDim.x - 1) await_previous();
  }
}

// Joins the states of requests that lie in more than one range, a warp to each (range that one begins in, H heads). Bound by latency:
// record, then states, in some waves; 8 us for 256 requests of 64 heads. Fewer CTAs that walk over the records were slower by 2 to 4 us.
template <int HD, int H>
__global__ void __launch_bounds__(128)
attn_join_parts_q8_kernel(nfk_attn_q8_params p, const DecodeRecord* records, States parts, unsigned int group, unsigned int n_ranges) {
  await_previous();
  for (unsigned int e = blockIdx.x * 4 + (threadIdx.x >> 5); e < n_ranges * (group / H); e += gridDim.x * 4) {
    const unsigned int range = e / (group / H), h = (e - range * (group / H)) * H;
    const int4 raw = __ldcg(reinterpret_cast<const int4*>(records) + range);
    const DecodeRecord rec = {raw.x, raw.y, raw.z, raw.w};
    if (rec.n == 0) continue;
    Row<HD> rows[H];
    sum_states<HD, H == 2 ? 2 : 6>(p.workspace, rec.n, [&](int i, int k) {
      return state_at<HD>(p.workspace, parts.ml, parts.o, ((range + i) * 2 + (i == 0 ? 1 : 0)) * group + h + k);
    }, rows);
    if (rec.tok < 0) continue;
#pragma unroll
    for (int k = 0; k < H; ++k)
      rows[k].finish(reinterpret_cast<__nv_bfloat16*>(p.out) + (static_cast<long long>(rec.tok) * p.q_heads + rec.kvh * group + h + k) * HD);
  }
}

// The same row by row, with the shared prefix's states where there is one, and WARPS warps to a row: a context of 900 tokens is 29
// pieces for each of 32 heads, one of 100000 tokens 296.
template <int HD, int WARPS>
__global__ void __launch_bounds__(128)
attn_join_rows_q8_kernel(nfk_attn_q8_params p, PrefixPlan f, const int* bad_lists, States parts, States wholes, unsigned int group, int decode_ctas) {
  __shared__ float shared_ml[4][2];
  __shared__ float shared_o[4][HD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, which = warp % WARPS;
  // lists and their cut while the kernels before this one still run (let_next_read)
  const Early<int> indptr{p.kv_indptr + p.req_begin}, toks{p.qo_indptr + p.req_begin};
  const unsigned int q_heads = p.q_heads, n_rows = p.req_count * q_heads;
  const int base = indptr[0], pages_all = indptr[p.req_count] - base;
  const Ranges ranges(pages_all * p.kv_heads, decode_ranges(pages_all * p.kv_heads, decode_ctas));
  for (unsigned int first = blockIdx.x * (4 / WARPS); first < n_rows; first += gridDim.x * (4 / WARPS)) {
    const unsigned int e = first + warp / WARPS;                 // the row, r * q_heads + head
    const bool on = e < n_rows;
    const unsigned int r = on ? e / q_heads : 0, head = on ? e - r * q_heads : 0, kvh = head / group, h = head - kvh * group;
    const int begin = indptr[r] - base, end = indptr[r + 1] - base;
    int tok = toks[r];
    const bool tok_ok = tok >= 0 && tok < p.num_tokens;
    if (!on || !tok_ok) tok = -1;                              // (a warp behind the last row has looked at row 0)
    int k0 = 0, n_own = 0, n_prefix = 0;
    unsigned int front = 0;                                      // the prefix's first state of this row
    if (on && end > begin) {
      k0 = ranges.of(kvh * pages_all + begin);
      n_own = ranges.of(kvh * pages_all + end - 1) - k0 + 1;
    }
    if (on && p.prefix_len > 0) {
      const unsigned int in = r / static_cast<unsigned int>(f.reqs_per_block), item = kvh * f.blocks + in;
      const int span = f.lead + f.tiles, c0 = f.cut.of(item * span + f.lead);
      n_prefix = f.cut.of((item + 1) * span - 1) - c0 + 1;
      front = (item + c0) * f.rows + (r - in * f.reqs_per_block) * group + h;
    }
    await_previous();
    if (on && !tok_ok && lane == 0) report_status(p.status, NF_ST_BAD_INDEX);
    if (*bad_lists != 0) n_own = 0;
    int n_all = n_own + n_prefix;
    if (p.prefix_len == 0 && n_own <= 1) tok = -1, n_all = 0;    // the row has been written
    // all states of the row, WARPS shares of them one after the other
    const int a = n_all * which / WARPS, b = n_all * (which + 1) / WARPS;
    Row<HD> rows[1];
    Row<HD>& row = rows[0];
    sum_states<HD, WARPS == 1 ? 6 : 16>(p.workspace, b - a, [&](int i, int) {
      const int k = a + i;
      const bool is_front = k >= n_own, whole = n_own == 1;
      const unsigned int at = is_front ? front + (k - n_own) * f.rows : whole ? e : ((k0 + k) * 2 + (k == 0 ? 1 : 0)) * group + h;
      return state_at<HD>(p.workspace, is_front ? f.ml : whole ? wholes.ml : parts.ml, is_front ? f.o : whole ? wholes.o : parts.o, at);
    }, rows);
    if (WARPS > 1) {
#pragma unroll
      for (int i = 0; i < Row<HD>::N; ++i) shared_o[warp][lane * Row<HD>::N + i] = row.o[i];
      if (lane == 0) {
        shared_ml[warp][0] = row.m;
        shared_ml[warp][1] = row.l;
      }
      __syncthreads();
      if (which == 0)
        for (int k = 1; k < WARPS; ++k) {
          Row<HD> other;
          other.m = shared_ml[warp + k][0];
          other.l = shared_ml[warp + k][1];
#pragma unroll
          for (int i = 0; i < Row<HD>::N; ++i) other.o[i] = shared_o[warp + k][lane * Row<HD>::N + i];
          row.add(other);
        }
    }
    if (which == 0 && tok >= 0) row.finish(reinterpret_cast<__nv_bfloat16*>(p.out) + (static_cast<long long>(tok) * q_heads + head) * HD);
    if (WARPS > 1) __syncthreads();                            // (before the next rows' states go there)
  }
}

// CTAs that share a request's pages for one KV head in a small batch, 0 where the general form is at least as fast: one launch instead
// of two, but as slow as the request with the most pages makes it, which the host does not know (0.5 us for each page of a warp). One
// token 4.6 us instead of 7.2, 100 tokens 5.1 instead of 7.9, nine requests of 10 to 100 6.0 (with clusters of four 8.1) instead of
// 8.3; one of 900 8.4 with four CTAs (with one 11.9, two 9.6, eight 8.7), 8.3 in the general form, whose call costs the host 2 us more.
int few_cluster(const nfk_attn_q8_params& p) {
  const int pages = p.num_indices, likely = p.req_count == 1 ? pages : pages < 2 * (pages / p.req_count + 1) ? pages : 2 * (pages / p.req_count + 1);
  const int size = likely <= 5 * kWarps ? 1 : 4;
  const long long ctas = static_cast<long long>(p.req_count) * p.kv_heads * size;
  const bool fits = ctas <= 4ll * device_sm_count() && (p.num_ctas == 0 || ctas <= p.num_ctas);
  return fits && p.prefix_len == 0 && likely <= size * kWarps * 5 && pages <= size * kWarps * 10 ? size : 0;
}

// CTAs of an SM that fit, for a kernel with `bytes` of shared memory; 0: an error.
int fitting(const void* kernel, int threads, int bytes) {
  int per_sm = 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess ||
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, bytes) != cudaSuccess) {
    (void)cudaGetLastError();
    return 0;
  }
  return per_sm;
}

template <int HD, int NT, int KIND, int MODE>
int launch(const nfk_attn_q8_params& p, const PrefixPlan& f, int* bad_lists, DecodeRecord* records, const States& parts, const States& wholes,
           cudaStream_t stream) {
  constexpr int bytes = kWarps * Dec<HD>::kWarpBytes;
  constexpr bool SHARED = MODE == SHARED_PREFIX;
  const auto kernel = attn_decode_q8_kernel<HD, NT, KIND, MODE>;
  static int fit_dev[kMaxDevices] = {0};
  int& fit = fit_dev[device_slot()];
  if (fit == 0) fit = fitting(reinterpret_cast<const void*>(kernel), kThreads, bytes);
  if (fit == 0) return NF_ERR_CUDA;
  const auto done = [](cudaError_t e) {
    if (e == cudaSuccess) return true;
    (void)cudaGetLastError();
    return false;
  };
  if (MODE == FEW) {
    const int size = few_cluster(p);
    return done(launch_kernel(early_first(p.early_start), kernel, p.req_count * p.kv_heads * size, kThreads, bytes, stream, size, p, bad_lists, records, parts, wholes))
               ? NF_OK : NF_ERR_CUDA;
  }
  const int sms = device_sm_count(), room = (fit < kDecodeCtasPerSm ? fit : kDecodeCtasPerSm) * sms;
  const int useful = decode_ranges(p.num_indices * p.kv_heads, room);
  int ctas = (useful + kWarps - 1) / kWarps;
  if (ctas < 1) ctas = 1;
  if (p.num_ctas > 0 && p.num_ctas < ctas) ctas = p.num_ctas;
  if (!done(launch_kernel(SHARED ? early_further(p.early_start) : early_first(p.early_start), kernel, ctas, kThreads, bytes, stream, 1, p, bad_lists, records, parts, wholes))) return NF_ERR_CUDA;
  // Few rows: four warps to each, since there are many pieces to a row then. With a prefix every row has states to join. Else the
  // pieces lead to the rows, of which most lie in one range.
  const int rows = p.req_count * p.q_heads, group = p.q_heads / p.kv_heads;
  const auto join = [&](auto kernel, int grid, auto... args) {
    if (p.num_ctas > 0 && p.num_ctas < grid) grid = p.num_ctas;
    return done(launch_kernel(early_further(p.early_start), kernel, grid, 128, 0, stream, 1, args...)) ? NF_OK : NF_ERR_CUDA;
  };
  if (rows <= 8 * sms) return join(attn_join_rows_q8_kernel<HD, 4>, rows, p, f, bad_lists, parts, wholes, group, ctas);
  if (SHARED) return join(attn_join_rows_q8_kernel<HD, 1>, (rows + 3) / 4, p, f, bad_lists, parts, wholes, group, ctas);
  // Two heads to a warp where a KV head has many (groups of 8: 256 requests 94.1 us instead of 95.5; of 16: 31.8 instead of 32.5; of 4:
  // 88 instead of 87.4).
  if (group >= 8 && group % 2 == 0) return join(attn_join_parts_q8_kernel<HD, 2>, ctas * (group / 2), p, records, parts, group, ctas * kWarps);
  return join(attn_join_parts_q8_kernel<HD, 1>, ctas * group, p, records, parts, group, ctas * kWarps);
}

template <int HD, int NT, int KIND, class... A>
int launch(const nfk_attn_q8_params& p, const A&... a) {
  return p.prefix_len > 0 ? launch<HD, NT, KIND, SHARED_PREFIX>(p, a...) : few_cluster(p) > 0 ? launch<HD, NT, KIND, FEW>(p, a...)
                                                                         : launch<HD, NT, KIND, PLAIN>(p, a...);
}
template <int HD, class... A>
int launch(const nfk_attn_q8_params& p, const A&... a) {
  const bool wide = p.q_heads / p.kv_heads > 8;
  if (p.kind == NFK_Q8_E4M3) return wide ? launch<HD, 2, NFK_Q8_E4M3>(p, a...) : launch<HD, 1, NFK_Q8_E4M3>(p, a...);
  return wide ? launch<HD, 2, NFK_Q8_INT8>(p, a...) : launch<HD, 1, NFK_Q8_INT8>(p, a...);
}

bool sizes_built(const nfk_attn_q8_params& p) {
  return (p.head_dim == 64 || p.head_dim == 128) && p.kv_heads > 0 && p.q_heads > 0 && p.q_heads % p.kv_heads == 0 &&
         p.q_heads / p.kv_heads <= 16;
}
// All units, and all places in their rows, are counted in 32 bits, with room for a step of all warps behind the last one.
bool counts_fit(const nfk_attn_q8_params& p, const PrefixPlan& f) {
  const long long most = 0x7fff0000ll;
  return static_cast<long long>(p.num_indices) * p.kv_heads <= most && static_cast<long long>(p.req_count) * p.q_heads <= most &&
         static_cast<long long>(p.kv_heads) * f.blocks <= most / (f.tiles > 0 ? f.lead + f.tiles : 1) &&
         static_cast<long long>(p.req_begin) + p.req_count <= most;
}
bool aligned16(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) == 0; }

}  // namespace
}  // namespace nf

extern "C" long long nfk_attn_q8_workspace(const nfk_attn_q8_params* p) {
  using namespace nf;
  if (p == nullptr || !sizes_built(*p) || p->req_count < 0 || p->prefix_len < 0) return 0;
  PrefixPlan f = prefix_plan(*p);
  f.ctas = f.most_ctas;                                        // a shorter prefix may be cut finer
  const long long bytes = counts_fit(*p, f) ? q8_workspace(*p, f).bytes : 0;
  return bytes <= (1ll << 35) ? bytes : 0;                     // (rows of the workspace are counted in 16 bytes, in 32 bits)
}

extern "C" int nfk_attn_decode_q8(const nfk_attn_q8_params* p, cudaStream_t stream) {
  using namespace nf;
  if (p == nullptr || p->req_count < 0 || p->req_begin < 0 || p->prefix_len < 0) return NF_ERR_BAD_ARG;
  if (!sizes_built(*p) || (p->kind != NFK_Q8_E4M3 && p->kind != NFK_Q8_INT8)) return NF_ERR_UNSUPPORTED;
  if (p->req_count == 0) return NF_OK;
  if (!p->q || !p->out || !p->kv_pool || !p->kv_scale || !p->qo_indptr || !p->kv_indptr || !p->kv_last_page_len || !p->workspace ||
      (p->num_indices > 0 && !p->kv_indices) || (p->prefix_len > 0 && !p->prefix_pages) || p->num_pages <= 0 || p->num_tokens <= 0 ||
      p->num_indices < 0 || p->num_ctas < 0 || !aligned16(p->q) || !aligned16(p->out) || !aligned16(p->kv_pool) || !aligned16(p->kv_scale) || (reinterpret_cast<uintptr_t>(p->workspace) & 255) != 0)
    return NF_ERR_BAD_ARG;
  PrefixPlan f = prefix_plan(*p);
  if (!counts_fit(*p, f)) return NF_ERR_BAD_ARG;
  const Q8Workspace ws = q8_workspace(*p, f);
  if (p->workspace_bytes < ws.bytes || ws.bytes > (1ll << 35)) return NF_ERR_BAD_ARG;
  char* base = static_cast<char*>(p->workspace);
  const auto at = [&](long long offset) { return reinterpret_cast<float*>(base + offset); };
  f.ml = at(ws.prefix_ml);
  f.o = at(ws.prefix_o);
  if (p->prefix_len > 0) {
    const int rc = launch_prefix_q8(*p, f, stream);
    if (rc != NF_OK) return rc;
  }
  int* bad_lists = reinterpret_cast<int*>(base);
  DecodeRecord* records = reinterpret_cast<DecodeRecord*>(base + ws.records);
  const States parts = {at(ws.ml), at(ws.o)}, wholes = {at(ws.whole_ml), at(ws.whole_o)};
  return p->head_dim == 128 ? launch<128>(*p, f, bad_lists, records, parts, wholes, stream)
                            : launch<64>(*p, f, bad_lists, records, parts, wholes, stream);
}
