// Calls of the drafted tokens' kernels from Python (module nanoflow_b200.ops._draft): the checks of arguments that the C ABI cannot
// make, the parameter block, and the launch on the tensors' device and its current stream.
//
// Functions take positional arguments only; nanoflow_b200/ops/draft.py gives them names, defaults and documentation. The kernel
// library is loaded there, too, and hands over its entry points' addresses.
#include "checks.h"

#include <vector>

namespace {

struct Entries {
  int (*grow)(const nfk_tables_params*, cudaStream_t) = nullptr;
  int (*trim)(const nfk_tables_params*, cudaStream_t) = nullptr;
  int (*rope)(const nfk_rope_slots_params*, cudaStream_t) = nullptr;
  int (*attend)(const nfk_attn_tree_params*, cudaStream_t) = nullptr;
  int (*masks)(const nfk_tree_masks_params*, cudaStream_t) = nullptr;
  int (*accept)(const nfk_tree_accept_params*, cudaStream_t) = nullptr;
  int (*keep)(const nfk_kv_keep_params*, cudaStream_t) = nullptr;
} entries;

constexpr int kPage = 16;

c10::Device cuda_of(const char* what, const char* name, const Tensor& t) {
  if (!t.is_cuda()) refuse(what, std::string(name) + " must be a CUDA tensor");
  return t.device();
}
int* ints(const Tensor& t) { return static_cast<int*>(t.data_ptr()); }
const Tensor& int32(const char* what, const char* name, PyObject* o, c10::Device device) { return checked(what, name, o, at::kInt, device); }

struct Pool {
  const Tensor& pool;
  int pages, kv_heads, head_dim;
};
Pool bf16_pool(const char* what, PyObject* o, bool any_head = false) {
  const Tensor& pool = tensor(what, "kv_pool", o);
  if (pool.scalar_type() != at::kBFloat16 || pool.dim() != 5 || !pool.is_contiguous() || !pool.is_cuda())
    refuse(what, "kv_pool must be a contiguous CUDA bfloat16 [pages, 2, kv_heads, 16, head_dim]");
  if (pool.size(1) != 2 || pool.size(3) != kPage || (!any_head && pool.size(4) != 64 && pool.size(4) != 128) || pool.size(0) < 1 || pool.size(2) < 1 ||
      pool.size(0) > INT32_MAX / kPage || pool.size(2) > 65536 || pool.size(4) > 1024)
    refuse(what, "pages hold 16 tokens of keys and of values, head_dim is 64 or 128");
  return Pool{pool, static_cast<int>(pool.size(0)), static_cast<int>(pool.size(2)), static_cast<int>(pool.size(4))};
}
// Rows of bf16 with unit inner stride; their distance (of a single row: any that is aligned).
long long rows_of(const char* what, const char* name, const Tensor& t, c10::Device device, int64_t columns) {
  if (t.scalar_type() != at::kBFloat16 || t.dim() != 2 || t.device() != device || (columns >= 0 && t.size(1) != columns) ||
      (t.size(1) > 1 && t.stride(1) != 1) || t.size(0) > INT32_MAX || t.size(1) > INT32_MAX)
    refuse(what, std::string(name) + " must be bfloat16 rows" + (columns >= 0 ? " of " + std::to_string(columns) : std::string()) +
                     " with unit inner stride on " + device.str());
  return t.size(0) > 1 ? t.stride(0) : (t.size(1) + 7) / 8 * 8;
}

struct Tables {
  nfk_tables_params p = {};
  const Tensor *table, *lengths, *free_pages, *free_count, *ticket, *rows, *tokens;
  c10::Device device;
};
// table, lengths, free_pages, free_count, ticket, rows, tokens
Tables tables_of(const char* what, PyObject* const* a) {
  const Tensor& table = tensor(what, "table", a[0]);
  Tables t{{}, &table, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, cuda_of(what, "table", table)};
  if (table.scalar_type() != at::kInt || table.dim() != 2 || !table.is_contiguous()) refuse(what, "table must be a contiguous int32 [rows, pages]");
  t.lengths = &int32(what, "lengths", a[1], t.device);
  t.free_pages = &int32(what, "free_pages", a[2], t.device);
  t.free_count = &int32(what, "free_count", a[3], t.device);
  t.ticket = &int32(what, "ticket", a[4], t.device);
  t.rows = &int32(what, "rows", a[5], t.device);
  t.tokens = &int32(what, "tokens", a[6], t.device);
  if (table.size(0) < 1 || table.size(0) > NFK_TABLES_ROWS || table.size(1) < 1 || table.size(1) > INT32_MAX / kPage)
    refuse(what, "table has 1 to " + std::to_string(NFK_TABLES_ROWS) + " rows of one page or more");
  if (t.lengths->numel() != table.size(0)) refuse(what, "lengths have an entry per row of the table");
  if (t.free_pages->numel() < 1 || t.free_pages->numel() > INT32_MAX / kPage || t.free_count->numel() != 1 || t.ticket->numel() != 1)
    refuse(what, "free_pages have an entry per page of the cache, free_count and ticket are a word each");
  if (t.tokens->numel() != t.rows->numel() || t.rows->numel() > NFK_TABLES_REQUESTS)
    refuse(what, "rows and tokens have an entry per request, of which there are up to " + std::to_string(NFK_TABLES_REQUESTS));
  nfk_tables_params& p = t.p;
  p.table = ints(table);
  p.lengths = ints(*t.lengths);
  p.free_pages = ints(*t.free_pages);
  p.free_count = ints(*t.free_count);
  p.ticket = word(t.ticket);
  p.rows = ints(*t.rows);
  p.tokens = ints(*t.tokens);
  p.requests = static_cast<int>(t.rows->numel());
  p.max_requests = static_cast<int>(table.size(0));
  p.max_pages = static_cast<int>(table.size(1));
  p.num_pages = static_cast<int>(t.free_pages->numel());
  return t;
}

// tables_of's, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, positions, token_req, slots, status, early_start
PyObject* grow(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 16, [&] {
    const char* what = "tables_grow";
    Tables t = tables_of(what, a);
    const Tensor& qo = int32(what, "qo_indptr", a[7], t.device);
    const Tensor& kv = int32(what, "kv_indptr", a[8], t.device);
    const Tensor& indices = int32(what, "kv_indices", a[9], t.device);
    const Tensor& last = int32(what, "kv_last_page_len", a[10], t.device);
    const Tensor& positions = int32(what, "positions", a[11], t.device);
    const Tensor& token_req = int32(what, "token_req", a[12], t.device);
    const Tensor& slots = int32(what, "slots", a[13], t.device);
    const int64_t R = t.p.requests;
    if (qo.numel() < R + 1 || kv.numel() < R + 1 || last.numel() < R) refuse(what, "the lists have an entry per request, qo_indptr and kv_indptr one more");
    if (positions.numel() != slots.numel() || token_req.numel() != slots.numel()) refuse(what, "positions, token_req and slots have an entry per token");
    const Tensor* status = status_word(what, a[14], t.device);
    apart(what, {t.table, t.lengths, t.free_count, t.ticket, &qo, &kv, &indices, &last, &positions, &token_req, &slots, status}, {t.free_pages, t.rows, t.tokens});
    t.p.qo_indptr = ints(qo);
    t.p.kv_indptr = ints(kv);
    t.p.kv_indices = ints(indices);
    t.p.kv_last_page_len = ints(last);
    t.p.positions = ints(positions);
    t.p.token_req = ints(token_req);
    t.p.slots = ints(slots);
    t.p.num_qo = count(what, qo, "qo_indptr");
    t.p.num_kv = count(what, kv, "kv_indptr");
    t.p.num_last = count(what, last, "kv_last_page_len");
    t.p.num_indices = count(what, indices, "kv_indices");
    t.p.num_tokens = count(what, slots, "slots");
    t.p.status = word(status);
    t.p.early_start = whole(a[15], what, "early_start");
    // (a list without entries has no memory, and none of it is touched)
    static int none[1];
    for (const int** at : {const_cast<const int**>(&t.p.kv_indices), const_cast<const int**>(&t.p.positions), const_cast<const int**>(&t.p.token_req),
                           const_cast<const int**>(&t.p.slots), const_cast<const int**>(&t.p.kv_last_page_len), &t.p.rows, &t.p.tokens})
      if (*at == nullptr) *at = none;
    launch("nfk_tables_grow", entries.grow, t.p, t.device);
  });
}

// tables_of's, status, early_start
PyObject* trim(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 9, [&] {
    const char* what = "tables_trim";
    Tables t = tables_of(what, a);
    const Tensor* status = status_word(what, a[7], t.device);
    apart(what, {t.lengths, t.free_pages, t.free_count, t.ticket, status}, {t.table, t.rows, t.tokens});
    t.p.status = word(status);
    t.p.early_start = whole(a[8], what, "early_start");
    if (t.p.requests > 0) launch("nfk_tables_trim", entries.trim, t.p, t.device);
  });
}

// qkv, q_out, kv_pool, inv_freq, positions, slots, q_heads, kv_heads, head_dim, q_off, k_off, v_off, interleaved, factor, status, early_start
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 16, [&] {
    const char* what = "rope_append_slots";
    const Pool c = bf16_pool(what, a[2]);
    const c10::Device device = c.pool.device();
    const Tensor& qkv = tensor(what, "qkv", a[0]);
    nfk_rope_slots_params p = {};
    p.ld_qkv = rows_of(what, "qkv", qkv, device, -1);
    p.q_heads = whole(a[6], what, "q_heads");
    p.kv_heads = whole(a[7], what, "kv_heads");
    p.head_dim = whole(a[8], what, "head_dim");
    p.q_off = whole(a[9], what, "q_off");
    p.k_off = whole(a[10], what, "k_off");
    p.v_off = whole(a[11], what, "v_off");
    const int interleaved = PyObject_IsTrue(a[12]);
    if (interleaved < 0) {
      PyErr_Clear();
      refuse(what, "interleaved must be a truth value");
    }
    p.interleaved = interleaved;
    p.factor = real(a[13], what, "factor");
    if (c.kv_heads != p.kv_heads || c.head_dim != p.head_dim || p.q_heads < 1 || p.q_heads > 65536) refuse(what, "kv_pool does not have these heads");
    const int64_t T = qkv.size(0), columns = qkv.size(1), hd = p.head_dim;
    if (p.q_off < 0 || p.q_off + p.q_heads * hd > columns || p.k_off < 0 || p.k_off + p.kv_heads * hd > columns || p.v_off < 0 ||
        p.v_off + p.kv_heads * hd > columns)
      refuse(what, "heads lie outside qkv's columns");
    const Tensor& q_out = checked(what, "q_out", a[1], at::kBFloat16, device);
    if (q_out.numel() != T * p.q_heads * hd) refuse(what, "q_out must be [T, q_heads * head_dim]");
    const Tensor& inv_freq = checked(what, "inv_freq", a[3], at::kFloat, device);
    const Tensor& positions = int32(what, "positions", a[4], device);
    const Tensor& slots = int32(what, "slots", a[5], device);
    if (positions.numel() != T || slots.numel() != T) refuse(what, "positions and slots have an entry per token");
    if (inv_freq.numel() < 1 || 2 * inv_freq.numel() > hd) refuse(what, "inv_freq has an entry for each pair that turns, up to head_dim / 2");
    const Tensor* status = status_word(what, a[14], device);
    apart(what, {&q_out, &c.pool, status}, {&qkv, &inv_freq, &positions, &slots});
    p.qkv = qkv.data_ptr();
    p.q_out = q_out.data_ptr();
    p.kv_pool = c.pool.data_ptr();
    p.inv_freq = static_cast<const float*>(inv_freq.data_ptr());
    p.positions = ints(positions);
    p.slots = ints(slots);
    p.T = static_cast<int>(T);
    p.pairs = static_cast<int>(inv_freq.numel());
    p.num_pages = c.pages;
    p.status = word(status);
    p.early_start = whole(a[15], what, "early_start");
    if (T > 0) launch("nfk_rope_slots", entries.rope, p, device);
  });
}

// q, out, kv_pool, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, tree, q_heads, req_begin, req_count, sm_scale, num_ctas, workspace,
// status, early_start, request_tokens
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 17, [&] {
    const char* what = "attn_tree";
    const Pool c = bf16_pool(what, a[2]);
    const c10::Device device = c.pool.device();
    const Tensor& q = tensor(what, "q", a[0]);
    const Tensor& out = tensor(what, "out", a[1]);
    nfk_attn_tree_params p = {};
    p.q_heads = whole(a[8], what, "q_heads");
    p.kv_heads = c.kv_heads;
    p.head_dim = c.head_dim;
    if (p.q_heads < 1 || p.q_heads % p.kv_heads != 0 || p.q_heads / p.kv_heads > 128)
      refuse(what, "up to 128 query heads share a KV head, all KV heads the same number");
    const int64_t row = static_cast<int64_t>(p.q_heads) * p.head_dim;
    p.ld_q = rows_of(what, "q", q, device, row);
    p.ld_out = rows_of(what, "out", out, device, row);
    if (out.size(0) != q.size(0)) refuse(what, "out has a row for each of q");
    if (q.size(0) > 1 && (p.ld_q < row || p.ld_out < row)) refuse(what, "rows of q and of out must not overlap");
    const Tensor& qo = int32(what, "qo_indptr", a[3], device);
    const Tensor& kv = int32(what, "kv_indptr", a[4], device);
    const Tensor& indices = int32(what, "kv_indices", a[5], device);
    const Tensor& last = int32(what, "kv_last_page_len", a[6], device);
    p.req_begin = whole(a[9], what, "req_begin");
    p.req_count = a[10] == Py_None ? static_cast<int>(std::min<int64_t>(last.numel() - p.req_begin, INT32_MAX)) : whole(a[10], what, "req_count");
    const int64_t end = static_cast<int64_t>(p.req_begin) + p.req_count;
    if (p.req_begin < 0 || p.req_count < 0 || qo.numel() < end + 1 || kv.numel() < end + 1 || last.numel() < end)
      refuse(what, "requests " + std::to_string(p.req_begin) + " to " + std::to_string(end) + " are not all listed");
    const Tensor* tree = nullptr;
    if (a[7] != Py_None) {
      tree = &checked(what, "tree", a[7], at::kLong, device);
      if (tree->dim() != 2 || tree->size(0) < q.size(0) || tree->size(1) < 1 || tree->size(1) > NFK_TREE_NODES / 64)
        refuse(what, "tree must be [tokens, words] of bits, up to " + std::to_string(NFK_TREE_NODES / 64) + " words");
      p.tree = static_cast<const unsigned long long*>(tree->data_ptr());
      p.words = static_cast<int>(tree->size(1));
    }
    p.sm_scale = a[11] == Py_None ? (c.head_dim == 128 ? 0.08838834764831845f : 0.125f) : real(a[11], what, "sm_scale");
    if (!(p.sm_scale > 0.f) || p.sm_scale > 2e38f) refuse(what, "sm_scale must be positive, up to 2e38");
    if (q.size(0) > 0 && p.ld_out / 8 > 0xffffffffll / q.size(0)) refuse(what, "rows of out reach over more than 64 GB");
    p.num_ctas = whole(a[12], what, "num_ctas");
    if (a[13] == Py_None) refuse(what, "needs a workspace (tree_workspace)");
    const Tensor& workspace = checked(what, "workspace", a[13], at::kByte, device);
    const Tensor* status = status_word(what, a[14], device);
    apart(what, {&out, &workspace, status}, {&q, &c.pool, &qo, &kv, &indices, &last, tree});
    p.q = q.data_ptr();
    p.out = out.data_ptr();
    p.kv_pool = c.pool.data_ptr();
    p.qo_indptr = ints(qo);
    p.kv_indptr = ints(kv);
    p.kv_indices = ints(indices);
    p.kv_last_page_len = ints(last);
    p.num_pages = c.pages;
    p.num_tokens = static_cast<int>(q.size(0));
    p.num_indices = count(what, indices, "kv_indices");
    static int none[1];
    if (p.kv_indices == nullptr) p.kv_indices = none;            // (a list without entries, none of which is read)
    p.workspace = workspace.data_ptr();
    p.workspace_bytes = workspace.numel();
    p.status = word(status);
    p.early_start = whole(a[15], what, "early_start");
    p.request_tokens = whole(a[16], what, "request_tokens");
    p.listed = count(what, last, "kv_last_page_len");
    if (p.req_count > 0 && p.num_tokens > 0) launch("nfk_attn_tree", entries.attend, p, device);
  });
}

// parents, qo_indptr, mask, positions, status, early_start
PyObject* masks(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 6, [&] {
    const char* what = "tree_masks";
    const Tensor& mask = tensor(what, "mask", a[2]);
    const c10::Device device = cuda_of(what, "mask", mask);
    const Tensor& parents = int32(what, "parents", a[0], device);
    const Tensor& qo = int32(what, "qo_indptr", a[1], device);
    if (mask.scalar_type() != at::kLong || mask.dim() != 2 || !mask.is_contiguous() || mask.size(0) != parents.numel() || mask.size(1) < 1 ||
        mask.size(1) > NFK_TREE_NODES / 64)
      refuse(what, "mask must be a contiguous int64 [tokens, words] of up to " + std::to_string(NFK_TREE_NODES / 64) + " words");
    const Tensor* positions = optional(what, "positions", a[3], at::kInt, device);
    if (positions != nullptr && positions->numel() < parents.numel()) refuse(what, "positions have an entry per token");
    if (qo.numel() < 1) refuse(what, "qo_indptr has an entry per request and one more");
    const Tensor* status = status_word(what, a[4], device);
    apart(what, {&mask, positions, status}, {&parents, &qo});
    nfk_tree_masks_params p = {};
    p.parents = ints(parents);
    p.qo_indptr = ints(qo);
    p.mask = static_cast<unsigned long long*>(mask.data_ptr());
    p.positions = positions != nullptr ? ints(*positions) : nullptr;
    p.requests = count(what, qo, "qo_indptr") - 1;
    p.num_tokens = count(what, parents, "parents");
    p.words = static_cast<int>(mask.size(1));
    p.status = word(status);
    p.early_start = whole(a[5], what, "early_start");
    if (p.requests > 0 && p.num_tokens > 0) launch("nfk_tree_masks", entries.masks, p, device);
  });
}

// tokens, parents, targets, qo_indptr, path, counts, next_tokens, dropped, status, early_start
PyObject* accept(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 10, [&] {
    const char* what = "tree_accept";
    const Tensor& tokens = tensor(what, "tokens", a[0]);
    const c10::Device device = cuda_of(what, "tokens", tokens);
    (void)int32(what, "tokens", a[0], device);
    const Tensor& parents = int32(what, "parents", a[1], device);
    const Tensor& targets = int32(what, "targets", a[2], device);
    const Tensor& qo = int32(what, "qo_indptr", a[3], device);
    const Tensor& path = int32(what, "path", a[4], device);
    const Tensor& counts = int32(what, "counts", a[5], device);
    const Tensor& next = int32(what, "next_tokens", a[6], device);
    const Tensor* dropped = optional(what, "dropped", a[7], at::kInt, device);
    if (parents.numel() != tokens.numel() || targets.numel() != tokens.numel()) refuse(what, "tokens, parents and targets have an entry per token");
    if (qo.numel() < 1 || path.dim() != 2 || path.size(0) != qo.numel() - 1 || counts.numel() != qo.numel() - 1 || next.numel() != qo.numel() - 1 ||
        (dropped != nullptr && dropped->numel() != qo.numel() - 1))
      refuse(what, "path is [requests, places], counts, next_tokens and dropped have an entry per request, qo_indptr one more");
    const Tensor* status = status_word(what, a[8], device);
    apart(what, {&path, &counts, &next, dropped, status}, {&tokens, &parents, &targets, &qo});
    nfk_tree_accept_params p = {};
    p.tokens = ints(tokens);
    p.parents = ints(parents);
    p.targets = ints(targets);
    p.qo_indptr = ints(qo);
    p.path = ints(path);
    p.counts = ints(counts);
    p.next_tokens = ints(next);
    p.dropped = dropped != nullptr ? ints(*dropped) : nullptr;
    p.requests = count(what, qo, "qo_indptr") - 1;
    p.num_tokens = count(what, tokens, "tokens");
    if (path.size(1) > INT32_MAX) refuse(what, "path has too many entries");
    p.max_path = static_cast<int>(path.size(1));
    p.status = word(status);
    p.early_start = whole(a[9], what, "early_start");
    if (p.requests > 0) launch("nfk_tree_accept", entries.accept, p, device);
  });
}

// kv_pools (a list or tuple), slots, path, counts, qo_indptr, status, early_start
PyObject* keep(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 7, [&] {
    const char* what = "kv_keep";
    if (!PyList_Check(a[0]) && !PyTuple_Check(a[0])) refuse(what, "kv_pools must be a list of pools");
    const Py_ssize_t pools = PySequence_Fast_GET_SIZE(a[0]);
    PyObject** items = PySequence_Fast_ITEMS(a[0]);
    if (pools == 0) return;
    const Pool c = bf16_pool(what, items[0], true);
    const c10::Device device = c.pool.device();
    std::vector<std::pair<const char*, const char*>> spans;      // of all pools
    for (Py_ssize_t i = 0; i < pools; ++i) {
      const Pool d = bf16_pool(what, items[i], true);
      if (d.pool.sizes() != c.pool.sizes() || d.pool.device() != device) refuse(what, "pools must be of one size, on one device");
      const char* at = static_cast<const char*>(d.pool.data_ptr());
      if ((reinterpret_cast<uintptr_t>(at) & 15) != 0) refuse(what, "pools must begin at 16 bytes");       // (before the first launch)
      spans.emplace_back(at, at + d.pool.nbytes());
    }
    const Tensor& slots = int32(what, "slots", a[1], device);
    const Tensor& path = int32(what, "path", a[2], device);
    const Tensor& counts = int32(what, "counts", a[3], device);
    const Tensor& qo = int32(what, "qo_indptr", a[4], device);
    if (qo.numel() < 1 || path.dim() != 2 || path.size(0) != qo.numel() - 1 || counts.numel() != qo.numel() - 1 || path.size(1) > INT32_MAX)
      refuse(what, "path is [requests, places], counts have an entry per request, qo_indptr one more");
    const Tensor* status = status_word(what, a[5], device);
    apart(what, {status}, {&slots, &path, &counts, &qo});
    for (const Tensor* t : {&slots, &path, &counts, &qo, status}) {
      if (t == nullptr || t->numel() == 0) continue;
      const char* at = static_cast<const char*>(t->data_ptr());
      spans.emplace_back(at, at + t->nbytes());
    }
    for (Py_ssize_t i = 0; i < pools; ++i)
      for (size_t j = i + 1; j < spans.size(); ++j)
        if (spans[i].first < spans[j].second && spans[j].first < spans[i].second) refuse(what, "tensors overlap, and one of them is written");
    nfk_kv_keep_params p = {};
    p.slots = ints(slots);
    p.path = ints(path);
    p.counts = ints(counts);
    p.qo_indptr = ints(qo);
    p.requests = count(what, qo, "qo_indptr") - 1;
    p.num_tokens = count(what, slots, "slots");
    p.max_path = static_cast<int>(path.size(1));
    p.num_pages = c.pages;
    p.kv_heads = c.kv_heads;
    p.head_dim = c.head_dim;
    p.status = word(status);
    p.early_start = whole(a[6], what, "early_start");
    if (p.requests == 0 || p.max_path == 0 || p.num_tokens == 0) return;
    for (Py_ssize_t first = 0; first < pools; first += NFK_KEEP_POOLS) {
      p.num_pools = static_cast<int>(std::min<Py_ssize_t>(pools - first, NFK_KEEP_POOLS));
      for (int i = 0; i < p.num_pools; ++i) p.pools[i] = THPVariable_Unpack(items[first + i]).data_ptr();
      launch("nfk_kv_keep", entries.keep, p, device);
    }
  });
}

// addresses of nfk_tables_grow, nfk_tables_trim, nfk_rope_slots, nfk_attn_tree, nfk_tree_masks, nfk_tree_accept, nfk_kv_keep
PyObject* connect(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 7, [&] {
    void* at[7];
    for (int i = 0; i < 7; ++i) {
      at[i] = PyLong_AsVoidPtr(a[i]);
      if (at[i] == nullptr) {
        PyErr_Clear();
        refuse("connect", "addresses expected");
      }
    }
    entries.grow = reinterpret_cast<decltype(entries.grow)>(at[0]);
    entries.trim = reinterpret_cast<decltype(entries.trim)>(at[1]);
    entries.rope = reinterpret_cast<decltype(entries.rope)>(at[2]);
    entries.attend = reinterpret_cast<decltype(entries.attend)>(at[3]);
    entries.masks = reinterpret_cast<decltype(entries.masks)>(at[4]);
    entries.accept = reinterpret_cast<decltype(entries.accept)>(at[5]);
    entries.keep = reinterpret_cast<decltype(entries.keep)>(at[6]);
  });
}

PyMethodDef methods[] = {method<connect>("connect"), method<grow>("grow"), method<trim>("trim"), method<rope>("rope"), method<attend>("attend"),
                         method<masks>("masks"), method<accept>("accept"), method<keep>("keep"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_draft", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__draft() { return PyModule_Create(&module); }
