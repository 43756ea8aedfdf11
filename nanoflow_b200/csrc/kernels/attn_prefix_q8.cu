// Attention of a batch's query tokens over a prefix that all of them see, in the 8-bit paged cache, on the 5th-generation tensor
// cores: partial softmax states for attn_decode_q8.cu to join with each request's own tokens.
//
// The query rows of a KV head (requests x group, 128 or 256 to a block) are one operand for every key, so the prefix is read once per
// block instead of once per request, and the work is bound by the products (4 rows tokens head_dim operations) as soon as there
// are some ten requests: 256 requests behind 8192 tokens, 32 / 8 heads, 52 us, 660 TFLOP/s, 0.40 of the measured rate; 64 of 64 / 8
// heads behind 32768 91 us, 0.45. A tile of two slots takes 2200 cycles: 1024 of 2^x, 1280 of products (scores read Q from shared
// memory for 64 columns at a time), 900 of instruction issue, which overlap in part. Items (KV head, block) times tiles of 64 tokens
// are a row of units that is cut evenly over the CTAs (two to an SM, or one); each leaves a piece per item.
//
// A block has one or two slots of 128 rows: with two, which share the tiles, a CTA has the SM, with one there are two CTAs.
//
//   4 warps a slot  softmax: a thread per query row. They also bring their rows of Q into shared memory, as f16 with a power of two
//                   per row (see attn_decode_q8.cu).
//   1 warp          tcgen05.mma: S(t+1) = Q K(t+1)^T is issued before P(t) is waited for; O += P(t) V(t) takes P from tensor memory
//   2 + 2 warps     keys and values, half a tile each: 8-bit numbers from their pages, a tile ahead in registers, to exact f16 in
//                   shared memory (128-byte swizzle; V stays token-major, an MN-major operand), and the tile's scales beside them
//
// Scores are S times the key's scale, in fp32. Weights are rounded to f16 times the value's scale relative to the largest one so
// far, as in attn_decode_q8.cu; O is brought to a new reference where a row's maximum grows by 2^8 or that largest scale grows.
#include "attn_q8.cuh"

namespace nf {
namespace {

constexpr int kTile = kPrefixTile;
constexpr float kGap = 8.f, kHeadroom = 128.f;
constexpr int kHalfBytes = kTile * 128;          // [64 tokens][64 elements]

template <int HD, int SLOTS>
struct Pre {
  static constexpr int NH = HD / 64;
  static constexpr int kThreads = SLOTS * 128 + 160;
  static constexpr int kStages = SLOTS == 2 ? 4 : 2, kRing = 2 * kStages;       // tiles of K and of V; of their scales (see there)
  static constexpr int kQ = 0, kSlot = NH * 16384;               // SLOTS x NH x [128 rows][64 elements]
  static constexpr int kStage = NH * kHalfBytes;                 // a tile of K or V
  static constexpr int kK = SLOTS * kSlot, kV = kK + kStages * kStage;
  static constexpr int kScales = kV + kStages * kStage;          // [kRing][64] of keys, the same of values, [kRing] v_ref
  static constexpr int kBars = kScales + kRing * (kTile * 8 + 4);
  static constexpr int kBytes = kBars + 256;
  // barriers
  static constexpr int Q_FULL = 0, O_FREE = 1, K_FULL = 2, K_EMPTY = K_FULL + kStages, V_FULL = K_EMPTY + kStages, V_EMPTY = V_FULL + kStages,
                       S_FULL = V_EMPTY + kStages, P_FULL = S_FULL + 2 * SLOTS, PV_DONE = P_FULL + 2 * SLOTS, LAST = PV_DONE + 2 * SLOTS, kNumBars = LAST + 1;
  static_assert(kBars % 8 == 0 && kNumBars * 8 + 8 <= 256, "room for the barriers");
};

// f16 x f16 -> fp32
constexpr uint32_t idesc_f16(int m, int n) { return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24); }

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ float4 ld_shared_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Keys (PART 0) or values (PART 1) of the CTA's tiles: tokens 32 half .. 32 half + 31 of each, by one warp.
template <int HD, int SLOTS, int KIND, int PART>
__device__ __forceinline__ void bring_tiles(const nfk_attn_q8_params& p, const PrefixPlan& f, int half, uint32_t sb, float* scales, float* v_refs,
                                            uint64_t* bars, volatile int* abort_flag) {
  using C = Pre<HD, SLOTS>;
  constexpr int LANES = HD / 16, AT_ONCE = 32 / LANES, NI = 32 / AT_ONCE;       // lanes of a token, tokens of a load, loads
  const int lane = threadIdx.x & 31, c = lane % LANES;
  // head_dim 128: the lanes of the row's second half take the neighbouring token's, so that the two halves (which lie 8 KB apart)
  // are stored to different banks
  const int row = (lane / LANES) ^ (c >> 2);
  const int n_pages = (p.prefix_len + kQ8Page - 1) / kQ8Page;
  const uint8_t* pool = static_cast<const uint8_t*>(p.kv_pool) + row * HD + c * 16;
  uint64_t* full = bars + (PART == 0 ? C::K_FULL : C::V_FULL);
  uint64_t* empty = bars + (PART == 0 ? C::K_EMPTY : C::V_EMPTY);
  uint4 raw[NI];
  float sc[2];
  // lane j < 4: the vectors of page j of the tile, -1 where there is none
  auto page_of = [&](int tile) {
    int at = -1;
    const int slot = tile * (kTile / kQ8Page) + lane;
    if (lane < kTile / kQ8Page && slot < n_pages) {
      int page = p.prefix_pages[slot];
      if (page < 0 || page >= p.num_pages) {
        report_status(p.status, NF_ST_BAD_INDEX);
        page = 0;
      }
      at = page;
    }
    return at;
  };
  // numbers of the warp's two pages, and the tile's scales
  auto load = [&](int at, int kvh) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int page = __shfl_sync(0xffffffffu, at, half * 2 + j);
      const uint8_t* from = pool + ((static_cast<long long>(page) * 2 + PART) * p.kv_heads + kvh) * (kQ8Page * HD);
#pragma unroll
      for (int n = 0; n < NI / 2; ++n)
        raw[j * (NI / 2) + n] = page < 0 ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4*>(from + n * AT_ONCE * HD);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int page = __shfl_sync(0xffffffffu, at, 2 * k + lane / kQ8Page);
      sc[k] = page < 0 ? 0.f : p.kv_scale[((static_cast<long long>(page) * 2 + PART) * p.kv_heads + kvh) * kQ8Page + lane % kQ8Page];
    }
  };
  Share now(f, blockIdx.x), ahead = now;
  int left = 0, tile_ahead = 0;                                  // the tile that is loaded next
  auto advance = [&]() {                                         // false: none
    if (left == 0) {
      if (!ahead.next()) return false;
      left = ahead.n;
      tile_ahead = ahead.t0;
    } else {
      ++tile_ahead;
    }
    --left;
    return true;
  };
  // numbers are requested a tile ahead, page numbers two
  if (advance()) load(page_of(tile_ahead), ahead.kvh);
  bool more = advance();
  int at = more ? page_of(tile_ahead) : -1, kvh = ahead.kvh;
  uint32_t g = 0;
  while (now.next()) {
    float v_ref = 7.8886091e-31f;                                // 2^-100
    for (int t = 0; t < now.n; ++t, ++g) {
      const int s = g % C::kStages, ring = g % C::kRing;
      const int valid = p.prefix_len - (now.t0 + t) * kTile;     // tokens of the tile
      const bool more_then = more && advance();
      const int kvh_then = ahead.kvh, at_then = more_then ? page_of(tile_ahead) : -1;
      if (!__all_sync(0xffffffffu, wait_or_abort(&empty[s], (g / C::kStages & 1) ^ 1, abort_flag))) {
        if (lane == 0) report_status(p.status, NF_ST_TIMEOUT_SMEM_EMPTY);
        *abort_flag = 1;
        return;
      }
      // what lies behind the prefix may be anything: as values it would spoil every row (as keys it is masked)
      if (PART == 1 && valid < kTile)
#pragma unroll
        for (int n = 0; n < NI; ++n)
          if (half * 32 + n * AT_ONCE + row >= valid) raw[n] = make_uint4(0, 0, 0, 0);
      const uint32_t stage = sb + (PART == 0 ? C::kK : C::kV) + s * C::kStage + (c >> 2) * kHalfBytes + (half * 32 + row) * 128;
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        uint32_t o[8];
        q8_to_f16<KIND>(raw[n].x, o[0], o[1]);
        q8_to_f16<KIND>(raw[n].y, o[2], o[3]);
        q8_to_f16<KIND>(raw[n].z, o[4], o[5]);
        q8_to_f16<KIND>(raw[n].w, o[6], o[7]);
        const uint32_t to = stage + n * AT_ONCE * 128, c0 = (2 * (c & 3)) ^ ((n * AT_ONCE + row) & 7);
        st_shared_v4(to + (c0 << 4), o[0], o[1], o[2], o[3]);
        st_shared_v4(to + ((c0 ^ 1) << 4), o[4], o[5], o[6], o[7]);
      }
      float* dst = scales + (PART * C::kRing + ring) * kTile + half * 32;
      if (PART == 0) {
        dst[lane] = sc[half] * (p.sm_scale * kQ8Log2e);
      } else {
        const float a = lane < valid ? sc[0] : 0.f, b = lane + 32 < valid ? sc[1] : 0.f;
        float most = fmaxf(fabsf(a), fabsf(b));
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
        if (most > v_ref) v_ref = __uint_as_float((__float_as_uint(most) + 0x7fffffu) & 0xff800000u);   // the next power of two
        dst[lane] = (half == 0 ? a : b) * (kHeadroom / v_ref);
        if (lane == 0 && half == 0) v_refs[ring] = v_ref;
      }
      if (more) load(at, kvh);
      more = more_then;
      at = at_then;
      kvh = kvh_then;
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[s]);
    }
  }
}

template <int HD, int SLOTS, int KIND>
__global__ void __launch_bounds__(SLOTS * 128 + 160, SLOTS == 2 ? 1 : 2)
attn_prefix_q8_kernel(nfk_attn_q8_params p, PrefixPlan f) {
  using C = Pre<HD, SLOTS>;
  constexpr int NH = C::NH, ST = C::kStages, MMA_WARP = 4 * SLOTS;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sb = smem_u32(smem);
  float* scales = reinterpret_cast<float*>(smem + C::kScales);
  float* v_refs = scales + 2 * C::kRing * kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  await_previous();                              // (before tensor memory is taken, which the kernel before may need)
  // a piece that will not be computed: its rows come out as NaN, and not as what an earlier call left in the workspace
  auto spoil = [&](int item) {
    if (threadIdx.x < 128 * SLOTS)
      __stcg(reinterpret_cast<float2*>(f.ml) + static_cast<long long>(item + blockIdx.x) * (128 * SLOTS) + threadIdx.x, make_float2(0.f, __uint_as_float(0x7fc00000u)));
  };
  if ((sb & 1023u) != 0u) {                      // the operands' layouts need it; report instead of computing garbage
    if (threadIdx.x == 0) report_status(p.status, NF_ST_BAD_INDEX);
    Share all(f, blockIdx.x);
    if (all.next()) all.rest(spoil);
    return;
  }
  if (threadIdx.x == 0) {
    for (int b = 0; b < C::kNumBars; ++b) {
      const bool bring = (b >= C::K_FULL && b < C::K_EMPTY) || (b >= C::V_FULL && b < C::V_EMPTY), weights = b >= C::P_FULL && b < C::PV_DONE;
      mbar_init(&bars[b], b <= C::O_FREE ? 4 * SLOTS : weights ? 4 : bring ? 2 : 1);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == MMA_WARP) {
    tmem_alloc(tmem_slot, 256 * SLOTS);          // of each slot: S0 in columns [0, 64), S1 in [64, 128), O in [128, 128 + HD)
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The requests' own tokens begin where SMs are done with the prefix. (Beside it, with three stages and 96 registers so that a CTA of
  // either fits an SM, both were slower: 256 requests behind 8192 tokens 104 us instead of 81.)
  if (warp == MMA_WARP) let_next_read();         // (the warp that has time for it)
  const int group = p.q_heads / p.kv_heads;
  auto fail = [&](unsigned int code) {
    if (lane == 0) report_status(p.status, code);
    *abort_flag = 1;
  };
  auto passed = [&](int bar, uint32_t parity) {
    return __all_sync(0xffffffffu, wait_or_abort(&bars[bar], parity, abort_flag)) != 0;
  };

  if (warp > MMA_WARP && warp <= MMA_WARP + 2) {
    bring_tiles<HD, SLOTS, KIND, 0>(p, f, warp - MMA_WARP - 1, sb, scales, v_refs, bars, abort_flag);
  } else if (warp > MMA_WARP + 2) {
    bring_tiles<HD, SLOTS, KIND, 1>(p, f, warp - MMA_WARP - 3, sb, scales, v_refs, bars, abort_flag);
  } else if (warp == MMA_WARP) {
    // ------------------------------------------------------------------ products (the warp walks, an elected lane issues)
    const uint32_t idesc_s = idesc_f16(128, kTile), idesc_o = idesc_f16(128, HD) | kIdescBMnMajor;
    const uint64_t q_desc = umma_desc_k_sw128(sb + C::kQ), k_desc = umma_desc_k_sw128(sb + C::kK);
    const uint64_t v_desc = umma_desc_mn_sw128(sb + C::kV, kHalfBytes, 1024);
    uint32_t g = 0, parts = 0;
    // S(gt) goes over P(gt - 2), which PV(gt - 2) reads: the latest PV issued must have completed
    auto issue_s = [&](uint32_t gt, uint32_t pv_issued) {
      if (!passed(C::K_FULL + gt % ST, gt / ST & 1)) return false;
      const uint64_t kd = k_desc + static_cast<uint64_t>(gt % ST * (C::kStage >> 4));
#pragma unroll
      for (int slot = 0; slot < SLOTS; ++slot) {
        if (pv_issued > 0 && !passed(C::PV_DONE + slot * 2 + ((pv_issued - 1) & 1), ((pv_issued - 1) >> 1) & 1)) return false;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_bf16_ss(tmem + slot * 256 + (gt & 1) * kTile, q_desc + ((slot * C::kSlot + h * 16384 + k * 32) >> 4),
                           kd + ((h * kHalfBytes + k * 32) >> 4), idesc_s, (h | k) ? 1u : 0u);
          umma_commit(&bars[C::S_FULL + slot * 2 + (gt & 1)]);
          if (slot == SLOTS - 1) umma_commit(&bars[C::K_EMPTY + gt % ST]);
        }
        __syncwarp();
      }
      return true;
    };
    bool ok = true;
    Share now(f, blockIdx.x);
    while (ok && now.next()) {
      if (!passed(C::Q_FULL, parts & 1) || !issue_s(g, g)) { fail(NF_ST_TIMEOUT_SMEM_FULL); ok = false; break; }
      for (int t = 0; ok && t < now.n; ++t) {
        const uint32_t gt = g + t;
        if (t + 1 < now.n && !issue_s(gt + 1, gt)) { fail(NF_ST_TIMEOUT_SMEM_FULL); ok = false; break; }
        // the item before must have been read out of O
        if (t == 0 && !passed(C::O_FREE, (parts & 1) ^ 1)) { fail(NF_ST_TIMEOUT_TMEM_EMPTY); ok = false; break; }
        if (!passed(C::V_FULL + gt % ST, gt / ST & 1)) { fail(NF_ST_TIMEOUT_SMEM_FULL); ok = false; break; }
        const uint64_t vd = v_desc + static_cast<uint64_t>(gt % ST * (C::kStage >> 4));
#pragma unroll
        for (int slot = 0; slot < SLOTS; ++slot) {
          if (!passed(C::P_FULL + slot * 2 + (gt & 1), (gt >> 1) & 1)) { fail(NF_ST_TIMEOUT_SMEM_FULL); ok = false; break; }
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_bf16_ts(tmem + slot * 256 + 2 * kTile, tmem + slot * 256 + (gt & 1) * kTile + k * 8, vd + ((k * 2048) >> 4), idesc_o,
                           (t | k) ? 1u : 0u);
            umma_commit(&bars[C::PV_DONE + slot * 2 + (gt & 1)]);
            if (slot == SLOTS - 1) umma_commit(&bars[C::V_EMPTY + gt % ST]);
          }
          __syncwarp();
        }
      }
      g += now.n;
      ++parts;
    }
    if (!ok) {                                   // products in flight get a bounded chance to end before their memory is given back
      if (elect_one()) umma_commit(&bars[C::LAST]);
      __syncwarp();
      (void)mbar_wait(&bars[C::LAST], 0);
    }
  } else {
    // ------------------------------------------------------------------ softmax (a thread per query row)
    const int row = warp * 32 + lane, slot = warp >> 2;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + slot * 256;
    const uint32_t q_row = sb + C::kQ + slot * C::kSlot + (row & 127) * 128;
    const uint32_t t_o = t_lane + 2 * kTile;
    const int in_block = row / group, hh = row - in_block * group;
    uint32_t g = 0;
    bool ok = true;
    Share now(f, blockIdx.x);
    while (ok && now.next()) {
      // ---- this thread's row of Q. The products of the item before have all been formed: its last scores have been read. ----
      const int r = now.block * f.reqs_per_block + in_block;
      int tok = -1;
      if (in_block < f.reqs_per_block && r < p.req_count) {
        tok = p.qo_indptr[p.req_begin + r];
        if (tok < 0 || tok >= p.num_tokens) tok = -1;            // (reported where the row would be written)
      }
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.q) +
                                                        (static_cast<long long>(tok < 0 ? 0 : tok) * p.q_heads + now.kvh * group + (tok < 0 ? 0 : hh)) * HD);
      uint4 raw[HD / 8];
#pragma unroll
      for (int c = 0; c < HD / 8; ++c) raw[c] = tok < 0 ? make_uint4(0, 0, 0, 0) : src[c];
      uint32_t most = 0;
#pragma unroll
      for (int c = 0; c < HD / 8; ++c) {
        const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) most = max(most, max(w[e] << 16 & 0x7fffffffu, w[e] & 0x7fff0000u));
      }
      float down, up;
      q_powers(__uint_as_float(most), down, up);
#pragma unroll
      for (int c = 0; c < HD / 8; ++c) {
        const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 x = unpack_bf16x2(w[e]);
          o[e] = pack_f16x2(x.x * down, x.y * down);
        }
        st_shared_v4(q_row + (c >> 3) * 16384 + (((c & 7) ^ (row & 7)) << 4), o[0], o[1], o[2], o[3]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[C::Q_FULL]);

      float ref = -INFINITY, l = 0.f, v_ref = 0.f;
      for (int t = 0; t < now.n; ++t) {
        const uint32_t gt = g + t;
        const int s = gt & 1;
        if (!passed(C::S_FULL + slot * 2 + s, (gt >> 1) & 1) || !passed(C::V_FULL + gt % ST, gt / ST & 1)) { fail(NF_ST_TIMEOUT_TMEM_FULL); ok = false; break; }
        tc_fence_after();
        const ulonglong2* k4 = reinterpret_cast<const ulonglong2*>(scales + gt % C::kRing * kTile);
        const ulonglong2* v4 = reinterpret_cast<const ulonglong2*>(scales + (C::kRing + gt % C::kRing) * kTile);
        f32x2 x0[16], x1[16];                                    // scores of tokens 2j, 2j + 1 (and of 32 tokens further)
        {
          uint32_t r0[32], r1[32];
          tmem_ld_32x32b_x32(t_lane + s * kTile, r0);
          tmem_ld_32x32b_x32(t_lane + s * kTile + 32, r1);
          tmem_ld_wait();
          const int valid = p.prefix_len - (now.t0 + t) * kTile;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const ulonglong2 a = k4[j], b = k4[8 + j];
            x0[2 * j] = mul2(pair(__uint_as_float(r0[4 * j]), __uint_as_float(r0[4 * j + 1])), a.x);
            x0[2 * j + 1] = mul2(pair(__uint_as_float(r0[4 * j + 2]), __uint_as_float(r0[4 * j + 3])), a.y);
            x1[2 * j] = mul2(pair(__uint_as_float(r1[4 * j]), __uint_as_float(r1[4 * j + 1])), b.x);
            x1[2 * j + 1] = mul2(pair(__uint_as_float(r1[4 * j + 2]), __uint_as_float(r1[4 * j + 3])), b.y);
          }
          if (valid < kTile) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float2 a = halves(x0[j]), b = halves(x1[j]);
              x0[j] = pair(2 * j >= valid ? -INFINITY : a.x, 2 * j + 1 >= valid ? -INFINITY : a.y);
              x1[j] = pair(32 + 2 * j >= valid ? -INFINITY : b.x, 33 + 2 * j >= valid ? -INFINITY : b.y);
            }
          }
        }
        float mq[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float2 a = halves(x0[j]), b = halves(x1[j]);
          mq[j & 1] = max3(mq[j & 1], a.x, a.y);
          mq[2 + (j & 1)] = max3(mq[2 + (j & 1)], b.x, b.y);
        }
        const float mx = fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3])) * up;
        const float v_new = v_refs[gt % C::kRing];
        if (t == 0) {
          ref = mx;
          v_ref = v_new;
        } else {
          const bool grow = mx > ref + kGap;
          if (__any_sync(0xffffffffu, grow || v_new != v_ref)) {
            // O may be touched between two products only: PV(t - 1) is the last one issued (PV(t) needs this tile's P)
            if (!passed(C::PV_DONE + slot * 2 + ((gt - 1) & 1), ((gt - 1) >> 1) & 1)) { fail(NF_ST_TIMEOUT_TMEM_FULL); ok = false; break; }
            tc_fence_after();
            const float alpha = grow ? q8_exp2(ref - mx) : 1.f, by = alpha * (v_ref / v_new);
#pragma unroll 1
            for (int c = 0; c < HD / 16; ++c) {
              uint32_t ov[16];
              tmem_ld_32x32b_x16n(t_o + c * 16, ov);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) ov[j] = __float_as_uint(__uint_as_float(ov[j]) * by);
              tmem_st_32x32b_x16(t_o + c * 16, ov);
            }
            tmem_st_wait();
            l *= alpha;
            if (grow) ref = mx;
            v_ref = v_new;
          }
        }
        const float ms = ref == -INFINITY ? 0.f : ref;
        const f32x2 up2 = pair(up, up), ms2 = pair(-ms, -ms);
        f32x2 rs = pair(0.f, 0.f);
        auto weights = [&](const f32x2 (&x)[16], const ulonglong2* v, uint32_t to) {
          uint32_t pk[16];                                       // column j: tokens 2j, 2j + 1
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float2 y = halves(fma2(x[j], up2, ms2));
            const f32x2 e = pair(q8_exp2(y.x), q8_exp2(y.y));
            rs = add2(rs, e);
            const float2 w = halves(mul2(e, (j & 1) ? v[j >> 1].y : v[j >> 1].x));
            pk[j] = pack_f16x2(w.x, w.y);
          }
          tmem_st_32x32b_x16(to, pk);
        };
        weights(x0, v4, t_lane + s * kTile);
        weights(x1, v4 + 8, t_lane + s * kTile + 16);
        l += halves(rs).x + halves(rs).y;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[C::P_FULL + slot * 2 + s]);
      }
      if (!ok) break;
      g += now.n;
      if (!passed(C::PV_DONE + slot * 2 + ((g - 1) & 1), ((g - 1) >> 1) & 1)) { fail(NF_ST_TIMEOUT_TMEM_FULL); ok = false; break; }
      tc_fence_after();
      const long long at = static_cast<long long>(now.item + blockIdx.x) * (128 * SLOTS) + row;
      const float back = v_ref / kHeadroom * kStateUnit;
      // by way of the warp's own rows of Q, which no product reads any more, so that stores are of whole rows (a thread's own row by
      // itself took 5300 cycles, as long as two tiles; now 4000)
      float* const rows_o = f.o + (at - lane) * HD;
      const uint32_t own = q_row - lane * 128;
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t v[32];
        tmem_ld_32x32b_x32(t_o + c * 32, v);
        tmem_ld_wait();
        const uint32_t via = own + c % NH * 16384;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j)
          st_shared_v4(via + lane * 128 + ((j ^ (lane & 7)) << 4), __float_as_uint(__uint_as_float(v[4 * j]) * back),
                       __float_as_uint(__uint_as_float(v[4 * j + 1]) * back), __float_as_uint(__uint_as_float(v[4 * j + 2]) * back),
                       __float_as_uint(__uint_as_float(v[4 * j + 3]) * back));
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = i * 4 + (lane >> 3), j = lane & 7;
          const float4 x = ld_shared_f32x4(via + r * 128 + ((j ^ (r & 7)) << 4));
          __stcg(reinterpret_cast<float4*>(rows_o + r * HD + c * 32 + j * 4), x);
        }
      }
      __syncwarp();
      __stcg(reinterpret_cast<float2*>(f.ml) + at, make_float2(ref, l));
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[C::O_FREE]);
    }
    if (!ok) now.rest(spoil);                    // (the current one, whose state is written last, among them)
  }

  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem, 256 * SLOTS);
  }
}

template <int HD, int SLOTS, int KIND>
int launch(const nfk_attn_q8_params& p, const PrefixPlan& f, cudaStream_t stream) {
  using C = Pre<HD, SLOTS>;
  const auto kernel = attn_prefix_q8_kernel<HD, SLOTS, KIND>;
  static bool attr_dev[kMaxDevices] = {false};
  bool& attr = attr_dev[device_slot()];
  if (!attr) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kBytes) != cudaSuccess) return NF_ERR_CUDA;
    attr = true;
  }
  if (launch_kernel(early_first(p.early_start), kernel, f.ctas, C::kThreads, C::kBytes, stream, 1, p, f) == cudaSuccess) return NF_OK;
  (void)cudaGetLastError();
  return NF_ERR_CUDA;
}
template <int HD, int SLOTS>
int launch(const nfk_attn_q8_params& p, const PrefixPlan& f, cudaStream_t stream) {
  return p.kind == NFK_Q8_E4M3 ? launch<HD, SLOTS, NFK_Q8_E4M3>(p, f, stream) : launch<HD, SLOTS, NFK_Q8_INT8>(p, f, stream);
}

}  // namespace

PrefixPlan prefix_plan(const nfk_attn_q8_params& p) {
  PrefixPlan f = {};
  if (p.prefix_len <= 0) return f;
  const int group = p.q_heads / p.kv_heads, slots = static_cast<long long>(p.req_count) * group > 128 ? 2 : 1;
  f.rows = 128 * slots;
  f.reqs_per_block = f.rows / group;
  f.blocks = static_cast<int>((static_cast<long long>(p.req_count) + f.reqs_per_block - 1) / f.reqs_per_block);
  f.tiles = static_cast<int>((static_cast<long long>(p.prefix_len) + kPrefixTile - 1) / kPrefixTile);
  const long long units = static_cast<long long>(p.kv_heads) * f.blocks * f.tiles;         // (whether they fit 32 bits is asked afterwards)
  int ctas = (slots == 2 ? 1 : 2) * device_sm_count();
  if (p.num_ctas > 0 && p.num_ctas < ctas) ctas = p.num_ctas;
  f.most_ctas = units < ctas ? static_cast<int>(units) : ctas;
  // Some tiles to a CTA where the prefix is long: every CTA leaves a piece of each row, and the rows' joins are bound by their number (8
  // requests of one KV head behind 30000 tokens: 31 us with a tile or two, 19 with four, 22 with eight; 16 of 8 behind 2000: 16.0 with
  // one, 14.4 with two, 14.8 with four; behind 500 12.5 with one, 12.9 with two).
  const int least = f.tiles >= 128 ? 4 : f.tiles >= 32 ? 2 : 1;
  if (ctas > (units + least - 1) / least) ctas = static_cast<int>((units + least - 1) / least);
  f.ctas = ctas;
  // An item's beginning and end (Q, O) take as long as some tiles: where CTAs have some tiles, one with the ends of two items gets fewer
  // (256 requests behind 8192 tokens 76.1 us instead of 79.8, 15 behind 12342 33.1 instead of 34.0; 2, 4, 8 and 10 units 79.1, 77.7,
  // 76.8 and 76.1). With fewer tiles to a CTA ranges rather end with the items.
  f.lead = units >= 4ll * ctas ? 6 : 0;
  const long long all = units + static_cast<long long>(p.kv_heads) * f.blocks * f.lead;
  if (all <= 0x7fffffff) f.cut = Ranges(static_cast<int>(all), ctas);
  return f;
}

int launch_prefix_q8(const nfk_attn_q8_params& p, const PrefixPlan& f, cudaStream_t stream) {
  if (p.head_dim == 128) return f.rows == 256 ? launch<128, 2>(p, f, stream) : launch<128, 1>(p, f, stream);
  return f.rows == 256 ? launch<64, 2>(p, f, stream) : launch<64, 1>(p, f, stream);
}

}  // namespace nf
