// Page tables on the GPU: growth by a step's tokens, with the lists that the step's kernels read, and the way back.
//
//   nfk_tables_grow  pages(r) = ceil((lengths + tokens) / 16), places of requests in the lists by sums over the requests in front
//   nfk_tables_trim  pages of dropped tokens back onto the stack of free ones
//
// One launch each, bound by latency (a chain of three loads, a scan) for all but the largest batches: every CTA works out all sums by
// itself, in shared memory, and then writes its share of the lists, an entry's request found by bisection. What the call changes
// is written by the CTA that is the last to have read it, known by a ticket.
//
// A step's growth and the way back together, in a graph: 1 request 7.1 us, 512 of up to 6000 tokens 11.7, 2048 of up to 4000 17.9, of which
// bytes need 0.3: loads of rows, lengths and pages behind one another, the barriers of the scan, eleven steps of bisection.
#include "common.cuh"
#include "kernels.h"

namespace nf {
namespace {

constexpr int kPage = 16;
constexpr int kMostThreads = 1024, kMine = NFK_TABLES_REQUESTS / kMostThreads;   // requests of a thread at most
// Threads of a CTA: barriers of many take longer, and up to three requests a thread cost less (growth and the way back: 256 requests 11.1 us,
// with 1024 threads 13.0; 512 11.7 and 13.0; 768 13.1 and 13.6; with a fourth it is the other way: 800 13.8, with 256 threads 14.5).
constexpr int kFewThreads = 256, kFewRequests = 3 * kFewThreads;
// entries of the lists that a thread writes before there are further CTAs
constexpr int kPerThread = 2;

__device__ __forceinline__ int pages_of(int tokens) { return (tokens + kPage - 1) / kPage; }

// Sums over the requests in front of each, of up to three things.
struct Sums {
  int* row;         // [requests] row of the tables
  int* old;         // [requests] length before the call
  int* at[3];       // [requests + 1]
  unsigned int* taken;   // rows, a bit each
};
__device__ __forceinline__ Sums sums_in(uint8_t* smem, int requests) {
  Sums s;
  int* a = reinterpret_cast<int*>(smem);
  s.row = a;
  s.old = a + requests;
  for (int k = 0; k < 3; ++k) s.at[k] = a + 2 * requests + k * (requests + 1);
  s.taken = reinterpret_cast<unsigned int*>(s.at[2] + requests + 1);
  return s;
}
int smem_bytes(int requests, int max_requests) { return (5 * requests + 3 + (max_requests + 31) / 32) * 4; }

// at[k][r] = sum of what[k] of the requests in front of r, `total` of all; entries hold `what` before, none negative. Sums end at the
// largest int: a total of that says that they do not fit, and nothing else then means anything.
constexpr unsigned int kFull = 0x7fffffffu;
__device__ __forceinline__ unsigned int add(unsigned int a, unsigned int b) { return min(a + b, kFull); }
__device__ __forceinline__ void scan(const Sums& s, int requests, int (&total)[3]) {
  __shared__ unsigned int warp_sum[3][kMostThreads / 32];
  const int threads = blockDim.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = (requests + threads - 1) / threads, r0 = min(requests, static_cast<int>(threadIdx.x) * per), r1 = min(requests, r0 + per);
  unsigned int mine[3] = {0, 0, 0}, sum[3];
  for (int r = r0; r < r1; ++r)
#pragma unroll
    for (int k = 0; k < 3; ++k) mine[k] = add(mine[k], s.at[k][r]);
#pragma unroll
  for (int k = 0; k < 3; ++k) sum[k] = mine[k];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const unsigned int v = __shfl_up_sync(0xffffffffu, sum[k], o);
      if (lane >= o) sum[k] = add(sum[k], v);
    }
#pragma unroll
  for (int k = 0; k < 3; ++k)
    if (lane == 31) warp_sum[k][warp] = sum[k];
  __syncthreads();
  unsigned int own[3], up[3];                    // the warps' sums, by every warp for itself
#pragma unroll
  for (int k = 0; k < 3; ++k) own[k] = up[k] = lane < threads / 32 ? warp_sum[k][lane] : 0u;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const unsigned int v = __shfl_up_sync(0xffffffffu, up[k], o);
      if (lane >= o) up[k] = add(up[k], v);
    }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    total[k] = static_cast<int>(__shfl_sync(0xffffffffu, up[k], 31));
    unsigned int a = __shfl_sync(0xffffffffu, up[k] - own[k], warp) + sum[k] - mine[k];
    for (int r = r0; r < r1; ++r) {
      const unsigned int n = s.at[k][r];
      s.at[k][r] = static_cast<int>(a);
      a += n;
    }
    if (threadIdx.x == 0) s.at[k][requests] = total[k];
  }
  __syncthreads();
}
// The request that entry e belongs to: the last one with at[r] <= e.
__device__ __forceinline__ int holder(const int* at, int requests, int e) {
  int r = 0, n = requests;
  while (n > 1) {
    const int half = n >> 1;
    if (at[r + half] <= e) {
      r += half;
      n -= half;
    } else {
      n = half;
    }
  }
  return r;
}
// Requests as they come, into row, old and at[0] (tokens); false, for all threads, where one is none.
__device__ __forceinline__ bool read_requests(const nfk_tables_params& p, const Sums& s) {
  const int words = (p.max_requests + 31) / 32, threads = blockDim.x;
  for (int w = threadIdx.x; w < words; w += threads) s.taken[w] = 0;
  int row[kMine], n[kMine], old[kMine];          // all of a thread's loads on their way at once
#pragma unroll
  for (int k = 0; k < kMine; ++k) {
    const int r = threadIdx.x + k * threads;
    row[k] = r < p.requests ? p.rows[r] : -1;
    n[k] = r < p.requests ? p.tokens[r] : 0;
  }
#pragma unroll
  for (int k = 0; k < kMine; ++k) old[k] = row[k] >= 0 && row[k] < p.max_requests ? p.lengths[row[k]] : -1;
  __syncthreads();
  bool bad = false;
#pragma unroll
  for (int k = 0; k < kMine; ++k) {
    const int r = threadIdx.x + k * threads;
    if (r >= p.requests) continue;
    bool ok = old[k] >= 0 && old[k] <= p.max_pages * kPage && n[k] >= 0;
    if (ok) ok = (atomicOr(&s.taken[row[k] >> 5], 1u << (row[k] & 31)) >> (row[k] & 31) & 1u) == 0u;
    s.row[r] = row[k];
    s.old[r] = ok ? old[k] : 0;
    s.at[0][r] = n[k];
    bad = bad || !ok;
  }
  return __syncthreads_or(bad) == 0;
}
// How many CTAs before this one have read what the call changes: asked behind a barrier of the block, by thread 0, and looked at in the end.
__device__ __forceinline__ unsigned int take_ticket(unsigned int* ticket) {
  if (threadIdx.x != 0 || gridDim.x == 1) return 0;
  __threadfence();
  return atomicAdd(ticket, 1u);
}
// Whether this CTA was the last of them; for all threads.
__device__ __forceinline__ bool last_reader(unsigned int* ticket, unsigned int mine) {
  const bool last = __syncthreads_or(threadIdx.x == 0 && mine == gridDim.x - 1) != 0;
  if (last && threadIdx.x == 0 && gridDim.x > 1) {
    *ticket = 0;
    __threadfence();
  }
  return last;
}

__global__ void __launch_bounds__(kMostThreads) tables_grow_kernel(const __grid_constant__ nfk_tables_params p) {
  extern __shared__ __align__(16) uint8_t smem[];
  const Sums s = sums_in(smem, p.requests);
  const int R = p.requests;
  let_next_start();
  await_previous();
  const int free_count = *p.free_count;
  bool ok = read_requests(p, s) && free_count >= 0 && free_count <= p.num_pages;
  int total[3] = {0, 0, 0};                      // tokens, pages, pages taken
  if (ok) {
    bool bad = false;
    for (int r = threadIdx.x; r < R; r += blockDim.x) {
      const int old = s.old[r], n = s.at[0][r];
      if (n > p.max_pages * kPage - old) {
        bad = true;
        continue;
      }
      s.at[1][r] = pages_of(old + n);
      s.at[2][r] = pages_of(old + n) - pages_of(old);
    }
    ok = __syncthreads_or(bad) == 0;
  }
  if (ok) {
    scan(s, R, total);
    const int most = static_cast<int>(kFull) - 1;
    ok = total[0] <= min(p.num_tokens, most) && total[1] <= min(p.num_indices, most) && total[2] <= free_count;
  }
  const unsigned int ticket = take_ticket(p.ticket);
  if (!ok) {
    total[0] = total[1] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) report_status(p.status, NF_ST_BAD_INDEX);
  }
  const int at = blockIdx.x * blockDim.x + threadIdx.x, step = gridDim.x * blockDim.x;
  // requests, and requests of nothing behind the last one, to the lists' ends
  for (int r = at; r <= max(R, max(max(p.num_qo, p.num_kv) - 1, p.num_last)); r += step) {
    if (r <= R || r < p.num_qo) p.qo_indptr[r] = ok ? s.at[0][min(r, R)] : 0;
    if (r <= R || r < p.num_kv) p.kv_indptr[r] = ok ? s.at[1][min(r, R)] : 0;
    if (r < R || r < p.num_last) {
      const int length = ok && r < R ? s.old[r] + s.at[0][r + 1] - s.at[0][r] : 0;
      p.kv_last_page_len[r] = length - max(pages_of(length) - 1, 0) * kPage;
    }
  }
  // page i of request r: the table's, or a new one
  auto page = [&](int r, int i) {
    const int had = pages_of(s.old[r]);
    return i < had ? p.table[static_cast<long long>(s.row[r]) * p.max_pages + i] : p.free_pages[free_count - 1 - (s.at[2][r] + i - had)];
  };
  for (int e = at; e < total[1]; e += step) {
    const int r = holder(s.at[1], R, e), i = e - s.at[1][r], id = page(r, i);
    p.kv_indices[e] = id;
    if (i >= pages_of(s.old[r])) p.table[static_cast<long long>(s.row[r]) * p.max_pages + i] = id;
  }
  for (int t = at; t < p.num_tokens; t += step) {
    int pos = 0, req = -1, slot = -1;
    if (t < total[0]) {
      req = holder(s.at[0], R, t);
      pos = s.old[req] + t - s.at[0][req];
      slot = page(req, pos / kPage) * kPage + pos % kPage;
    }
    p.positions[t] = pos;
    p.token_req[t] = req;
    p.slots[t] = slot;
  }
  if (last_reader(p.ticket, ticket) && ok) {
    for (int r = threadIdx.x; r < R; r += blockDim.x) p.lengths[s.row[r]] = s.old[r] + s.at[0][r + 1] - s.at[0][r];
    if (threadIdx.x == 0) *p.free_count = free_count - total[2];
  }
}

__global__ void __launch_bounds__(kMostThreads) tables_trim_kernel(const __grid_constant__ nfk_tables_params p) {
  extern __shared__ __align__(16) uint8_t smem[];
  const Sums s = sums_in(smem, p.requests);
  const int R = p.requests;
  let_next_start();
  await_previous();
  const int free_count = *p.free_count;
  bool ok = read_requests(p, s) && free_count >= 0 && free_count <= p.num_pages;
  int total[3] = {0, 0, 0};                      // new lengths (their sums are not looked at), unused, pages that come free
  if (ok) {
    for (int r = threadIdx.x; r < R; r += blockDim.x) {
      const int old = s.old[r], length = old - min(s.at[0][r], old);
      s.at[0][r] = length;
      s.at[1][r] = 0;
      s.at[2][r] = pages_of(old) - pages_of(length);
      s.old[r] = length;
    }
    __syncthreads();
    scan(s, R, total);
    ok = total[2] <= p.num_pages - free_count;
  }
  const unsigned int ticket = take_ticket(p.ticket);
  if (!ok && blockIdx.x == 0 && threadIdx.x == 0) report_status(p.status, NF_ST_BAD_INDEX);
  const int n = ok ? total[2] : 0;
  for (int e = blockIdx.x * blockDim.x + threadIdx.x; e < n; e += gridDim.x * blockDim.x) {
    const int r = holder(s.at[2], R, e);
    p.free_pages[free_count + n - 1 - e] = p.table[static_cast<long long>(s.row[r]) * p.max_pages + pages_of(s.old[r]) + e - s.at[2][r]];
  }
  if (last_reader(p.ticket, ticket) && ok) {
    for (int r = threadIdx.x; r < R; r += blockDim.x) p.lengths[s.row[r]] = s.old[r];
    if (threadIdx.x == 0) *p.free_count = free_count + n;
  }
}

template <bool GROW>
int launch(const nfk_tables_params& p, long long entries, cudaStream_t stream) {
  const auto kernel = GROW ? tables_grow_kernel : tables_trim_kernel;
  const int bytes = smem_bytes(p.requests, p.max_requests);
  static bool attr_dev[kMaxDevices] = {false};   // the attribute is per device
  bool& attr = attr_dev[device_slot()];
  if (!attr) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(NFK_TABLES_REQUESTS, NFK_TABLES_ROWS)) != cudaSuccess) {
      (void)cudaGetLastError();
      return NF_ERR_CUDA;
    }
    attr = true;
  }
  const int threads = p.requests <= kFewRequests ? kFewThreads : kMostThreads;
  long long ctas = (entries + threads * kPerThread - 1) / (threads * kPerThread);
  if (ctas > device_sm_count()) ctas = device_sm_count();
  if (ctas < 1) ctas = 1;
  if (launch_kernel(early_first(p.early_start), kernel, static_cast<int>(ctas), threads, bytes, stream, 1, p) == cudaSuccess) return NF_OK;
  (void)cudaGetLastError();
  return NF_ERR_CUDA;
}
int check(const nfk_tables_params* p) {
  if (p == nullptr || p->requests < 0 || p->requests > NFK_TABLES_REQUESTS || p->max_requests < 1 || p->max_requests > NFK_TABLES_ROWS ||
      p->max_pages < 1 || p->max_pages > 0x7fffffff / kPage || p->num_pages < 1 || p->num_pages > 0x7fffffff / kPage)
    return NF_ERR_BAD_ARG;
  return p->table && p->lengths && p->free_pages && p->free_count && p->ticket && p->rows && p->tokens ? NF_OK : NF_ERR_BAD_ARG;
}

}  // namespace
}  // namespace nf

extern "C" int nfk_tables_grow(const nfk_tables_params* p, cudaStream_t stream) {
  using namespace nf;
  const int rc = check(p);
  if (rc != NF_OK) return rc;
  if (!p->qo_indptr || !p->kv_indptr || !p->kv_indices || !p->kv_last_page_len || !p->positions || !p->token_req || !p->slots ||
      p->num_indices < 0 || p->num_indices > NFK_DRAFT_ENTRIES || p->num_tokens < 0 || p->num_tokens > NFK_DRAFT_ENTRIES ||
      p->num_qo > NFK_DRAFT_ENTRIES || p->num_kv > NFK_DRAFT_ENTRIES || p->num_last > NFK_DRAFT_ENTRIES)
    return NF_ERR_BAD_ARG;
  // (lists of a captured graph may be far longer than what a step fills, so that both count)
  return launch<true>(*p, static_cast<long long>(p->num_indices) + p->num_tokens, stream);
}

extern "C" int nfk_tables_trim(const nfk_tables_params* p, cudaStream_t stream) {
  using namespace nf;
  const int rc = check(p);
  if (rc != NF_OK) return rc;
  if (p->requests == 0) return NF_OK;
  return launch<false>(*p, static_cast<long long>(p->requests) * 16, stream);
}
