// The torch side of the paged cache's calls: argument checks, outputs, workspace and stream (a call of a few microseconds of kernel has no
// time for the interpreter to do it).  Python (cache.py) documents them and keeps the status word.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "../../include/htree_b200.h"

namespace {

using OptTensor = c10::optional<at::Tensor>;

int dtype_code(at::ScalarType t) { return t == at::kFloat ? HTREE_F32 : t == at::kBFloat16 ? HTREE_BF16 : t == at::kHalf ? HTREE_F16 : -1; }

void check(int64_t rc, const char* what) {
    TORCH_CHECK(rc == 0, "htree_b200 ", what, " failed with code ", rc, ": ", htree_b200_error_string((int)rc));
}

cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }

void want(const at::Tensor& t, const char* name, int64_t dim, at::ScalarType type, const at::Tensor& like) {
    TORCH_CHECK_VALUE(t.dim() == dim, name, " must have ", dim, " dimensions, not ", t.dim());
    TORCH_CHECK_VALUE(t.scalar_type() == type, name, " must be ", type, ", not ", t.scalar_type());
    TORCH_CHECK_VALUE(t.device() == like.device(), name, " is on ", t.device(), " and others on ", like.device());
}
void want_int32(const at::Tensor& t, const char* name, int64_t dim, const at::Tensor& like) { want(t, name, dim, at::kInt, like); }

// (torch.no_grad() turns gradients off, but not tangents)
void no_grad(std::initializer_list<const at::Tensor*> ts, const char* what) {
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode())
        for (const at::Tensor* t : ts) TORCH_CHECK(!t->_fw_grad(/*level=*/0).defined(), what, " has no forward-mode derivative: pass it the primal tensors");
    if (!at::GradMode::is_enabled()) return;
    for (const at::Tensor* t : ts)
        TORCH_CHECK(!t->requires_grad(), what, " has no backward: call it under torch.no_grad(), or detach its inputs");
}

bool aligned16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0; }

// Strides of the three leading dimensions; those of dimensions of one element do not matter.
bool rows_ok(const at::Tensor& t, int64_t (&s)[3]) {
    if (t.size(3) > 1 && t.stride(3) != 1) return false;
    bool ok = aligned16(t);
    for (int i = 0; i < 3; ++i) {
        s[i] = t.size(i) > 1 ? t.stride(i) : 0;
        ok = ok && (s[i] * t.element_size()) % 16 == 0;
    }
    return ok;
}
// ... of a tensor that is read: copied where its rows are not dense and 16-byte aligned
at::Tensor readable(const at::Tensor& t, int64_t (&s)[3]) {
    if (rows_ok(t, s)) return t;
    at::Tensor c = t.is_contiguous() ? t.clone() : t.contiguous();
    TORCH_CHECK(rows_ok(c, s), "htree_b200: row widths must be multiples of 8");
    return c;
}

void check_tables(const at::Tensor& table, const at::Tensor& lengths, int64_t B) {
    want_int32(table, "block_table", 2, table);
    want_int32(lengths, "lengths", 1, table);
    TORCH_CHECK_VALUE(table.size(0) == B && lengths.size(0) == B, "block_table and lengths must have one row per request (", B, "), not ", table.size(0),
                      " and ", lengths.size(0));
    TORCH_CHECK_VALUE(table.size(1) > 0, "block_table must have at least one column");
    TORCH_CHECK_VALUE(lengths.is_contiguous() && (table.size(1) == 1 || table.stride(1) == 1) && (B <= 1 || table.stride(0) >= table.size(1)),
                      "lengths must be contiguous, and the rows of block_table dense and apart");
}
int64_t table_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

HtreeCache make_cache(const at::Tensor& k, const at::Tensor& v, bool written) {
    TORCH_CHECK(k.is_cuda() && v.is_cuda(), "htree_b200 runs on CUDA tensors only; there is no CPU implementation");
    TORCH_CHECK_VALUE(k.dim() == 4 && v.dim() == 4, "k_cache and v_cache must be [pages, page_size, H_kv, width]");
    TORCH_CHECK_VALUE(k.scalar_type() == v.scalar_type() && dtype_code(k.scalar_type()) >= 0, "k_cache and v_cache must share one of fp32/bf16/fp16");
    TORCH_CHECK_VALUE(k.device() == v.device(), "k_cache and v_cache must be on one device");
    TORCH_CHECK_VALUE(k.size(0) == v.size(0) && k.size(1) == v.size(1) && k.size(2) == v.size(2), "k_cache and v_cache must have the same pages and heads");
    TORCH_CHECK_VALUE(k.numel() > 0 && v.numel() > 0, "the cache is empty");
    TORCH_CHECK_VALUE(k.size(3) % 8 == 0 && v.size(3) % 8 == 0, "row widths must be multiples of 8, not ", k.size(3), " and ", v.size(3));
    TORCH_CHECK_VALUE(k.size(0) <= INT32_MAX && k.size(1) <= (1 << 20) && k.size(2) <= INT32_MAX, "cache too large: page_size up to 2^20");
    int64_t ks[3], vs[3];
    TORCH_CHECK_VALUE(rows_ok(k, ks) && rows_ok(v, vs), "rows of k_cache and v_cache must be dense and start on 16-byte boundaries");
    if (written)
        for (int i = 0; i < 3; ++i)
            TORCH_CHECK_VALUE((k.size(i) == 1 || ks[i] != 0) && (v.size(i) == 1 || vs[i] != 0), "k_cache and v_cache must not be expanded: they are written");
    HtreeCache c{};
    c.k = k.data_ptr(); c.v = v.data_ptr();
    c.k_page = ks[0]; c.k_row = ks[1]; c.k_head = ks[2];
    c.v_page = vs[0]; c.v_row = vs[1]; c.v_head = vs[2];
    c.pages = (int32_t)k.size(0); c.page_size = (int32_t)k.size(1); c.H_kv = (int32_t)k.size(2);
    c.K = (int32_t)k.size(3); c.V = (int32_t)v.size(3); c.dtype = dtype_code(k.scalar_type());
    return c;
}

void check_new(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache, const at::Tensor& v_cache) {
    want(k, "k", 4, k_cache.scalar_type(), k_cache);
    want(v, "v", 4, k_cache.scalar_type(), k_cache);
    TORCH_CHECK_VALUE(k.size(0) == v.size(0) && k.size(1) == v.size(1), "k and v must have the same requests and tokens");
    TORCH_CHECK_VALUE(k.size(2) == k_cache.size(2) && v.size(2) == k_cache.size(2) && k.size(3) == k_cache.size(3) && v.size(3) == v_cache.size(3),
                      "k and v must have the heads and row widths of the cache");
    TORCH_CHECK_VALUE(k.size(0) <= INT32_MAX && k.size(1) <= INT32_MAX, "too many tokens");
}

// What a call has written: saved for somebody's backward, it has changed since.
void written(std::initializer_list<const at::Tensor*> ts) {
    for (const at::Tensor* t : ts)
        if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

// A new tensor without a way through the dispatcher (which takes as long as the allocation).
at::Tensor fresh(at::IntArrayRef size, at::ScalarType type, const at::Tensor& like) { return at::Tensor(at::detail::empty_cuda(size, type, like.device(), c10::nullopt)); }

int32_t* status_of(const at::Tensor& status) { return status.data_ptr<int32_t>(); }

std::tuple<at::Tensor, at::Tensor> cache_plan(const at::Tensor& lengths, const at::Tensor& counts, const at::Tensor& table, const at::Tensor& pool,
                                              const at::Tensor& top, int64_t page_size, int64_t n, const at::Tensor& status) {
    TORCH_CHECK_VALUE(lengths.dim() == 1, "lengths must have 1 dimension, not ", lengths.dim());
    const int64_t B = lengths.size(0);
    check_tables(table, lengths, B);
    want_int32(counts, "counts", 1, table);
    want_int32(pool, "pool", 1, table);
    TORCH_CHECK_VALUE(top.numel() == 1 && top.scalar_type() == at::kInt && top.device() == table.device(), "top must be one int32 on the tables' device");
    TORCH_CHECK_VALUE(counts.size(0) == B, "counts must have one entry per request");
    TORCH_CHECK_VALUE(pool.size(0) > 0 && pool.is_contiguous(), "pool must be contiguous and hold at least one page");
    TORCH_CHECK_VALUE(page_size > 0 && page_size <= (1 << 20), "page_size must be between 1 and 2^20, not ", page_size);
    TORCH_CHECK_VALUE(n > 0 && n <= INT32_MAX, "n must be positive, not ", n);
    TORCH_CHECK_VALUE(B <= 65535 && table.size(1) <= INT32_MAX && pool.size(0) <= INT32_MAX, "at most 65535 requests");
    c10::cuda::CUDAGuard guard(table.device());
    at::Tensor slots = fresh({B, n}, at::kLong, table), taken = fresh({B}, at::kInt, table);
    if (B == 0) return {slots, taken};
    const at::Tensor c = counts.contiguous();
    check(htree_b200_cache_plan((int32_t)B, (int32_t)table.size(1), (int32_t)page_size, (int32_t)n, lengths.data_ptr<int32_t>(), c.data_ptr<int32_t>(),
                                table.data_ptr<int32_t>(), table_stride(table), pool.data_ptr<int32_t>(), (int32_t)pool.size(0), top.data_ptr<int32_t>(),
                                slots.data_ptr<int64_t>(), taken.data_ptr<int32_t>(), status_of(status), stream()),
          "cache_plan");
    written({&lengths, &table, &pool, &top});
    return {slots, taken};
}

void cache_append(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& slots,
                  const OptTensor& index, const at::Tensor& status) {
    const HtreeCache cache = make_cache(k_cache, v_cache, true);
    check_new(k, v, k_cache, v_cache);
    no_grad({&k, &v, &k_cache, &v_cache}, "cache_append");
    want(slots, "slots", 2, at::kLong, k_cache);
    const int64_t B = k.size(0), N = k.size(1), n = slots.size(1);
    TORCH_CHECK_VALUE(slots.size(0) == B, "slots must have one row per request");
    at::Tensor idx;
    if (index.has_value()) {
        want_int32(*index, "index", 2, k_cache);
        TORCH_CHECK_VALUE(index->sizes() == slots.sizes(), "index must have the shape of slots");
        idx = index->contiguous();
    } else {
        TORCH_CHECK_VALUE(n <= N, "slots has more columns (", n, ") than k has tokens (", N, "): pass index");
    }
    TORCH_CHECK_VALUE(B * n < INT32_MAX, "too many slots");
    if (B == 0 || n == 0) return;
    TORCH_CHECK_VALUE(N > 0, "k has no tokens");
    c10::cuda::CUDAGuard guard(k_cache.device());
    int64_t ks[3], vs[3];
    const at::Tensor kk = readable(k, ks), vv = readable(v, vs), s = slots.contiguous();
    check(htree_b200_cache_append(&cache, (int32_t)B, (int32_t)N, (int32_t)n, kk.data_ptr(), ks, vv.data_ptr(), vs, s.data_ptr<int64_t>(),
                                  idx.defined() ? idx.data_ptr<int32_t>() : nullptr, status_of(status), stream()),
          "cache_append");
    written({&k_cache, &v_cache});
}

std::tuple<at::Tensor, at::Tensor> cache_gather(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& table, const at::Tensor& lengths,
                                                int64_t T, const at::Tensor& status) {
    const HtreeCache cache = make_cache(k_cache, v_cache, false);
    no_grad({&k_cache, &v_cache}, "cache_gather");
    TORCH_CHECK_VALUE(lengths.dim() == 1, "lengths must have 1 dimension, not ", lengths.dim());
    const int64_t B = lengths.size(0);
    check_tables(table, lengths, B);
    TORCH_CHECK_VALUE(table.device() == k_cache.device(), "block_table and the cache must be on one device");
    TORCH_CHECK_VALUE(T >= 0 && T <= INT32_MAX && B <= 65535 && table.size(1) <= INT32_MAX, "T must not be negative; at most 65535 requests");
    c10::cuda::CUDAGuard guard(k_cache.device());
    at::Tensor k = fresh({B, T, k_cache.size(2), k_cache.size(3)}, k_cache.scalar_type(), k_cache);
    at::Tensor v = fresh({B, T, k_cache.size(2), v_cache.size(3)}, k_cache.scalar_type(), k_cache);
    if (B == 0 || T == 0) return {k, v};
    check(htree_b200_cache_gather(&cache, (int32_t)B, (int32_t)table.size(1), (int32_t)T, table.data_ptr<int32_t>(), table_stride(table),
                                  lengths.data_ptr<int32_t>(), k.data_ptr(), v.data_ptr(), status_of(status), stream()),
          "cache_gather");
    return {k, v};
}

std::tuple<at::Tensor, OptTensor> draft_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache,
                                                  const at::Tensor& v_cache, const at::Tensor& table, const at::Tensor& lengths, const OptTensor& parents,
                                                  double scale, bool want_lse, const at::Tensor& status) {
    const HtreeCache cache = make_cache(k_cache, v_cache, false);
    check_new(k, v, k_cache, v_cache);
    want(q, "q", 4, k_cache.scalar_type(), k_cache);
    no_grad({&q, &k, &v, &k_cache, &v_cache}, "draft_attention");
    const int64_t B = q.size(0), N = q.size(1), H = q.size(2);
    TORCH_CHECK_VALUE(k.size(0) == B && k.size(1) == N, "q, k and v must have the same requests and drafts");
    TORCH_CHECK_VALUE(q.size(3) == cache.K, "q and k must have the same row width");
    TORCH_CHECK_VALUE(H > 0 && H % cache.H_kv == 0, "H (", H, ") must be divisible by H_kv (", cache.H_kv, ")");
    TORCH_CHECK_VALUE(cache.K <= 256 && cache.V <= 256, "rows of up to 256 elements, not ", cache.K, " and ", cache.V);
    check_tables(table, lengths, B);
    TORCH_CHECK_VALUE(table.device() == k_cache.device(), "block_table and the cache must be on one device");
    TORCH_CHECK_VALUE(B * N * H < INT32_MAX && table.size(1) <= INT32_MAX, "too many drafts");
    at::Tensor par;
    if (parents.has_value()) {
        want_int32(*parents, "parents", 2, k_cache);
        TORCH_CHECK_VALUE(parents->size(0) == B && parents->size(1) == N, "parents must have one entry per draft");
        TORCH_CHECK_VALUE(N <= 1024, "trees of up to 1024 drafts, not ", N);
        par = parents->contiguous();
    }
    c10::cuda::CUDAGuard guard(k_cache.device());
    at::Tensor out = fresh({B, N, H, (int64_t)cache.V}, q.scalar_type(), q);
    OptTensor lse;
    if (want_lse) lse = fresh({B, N, H}, at::kFloat, q);
    if (B == 0 || N == 0) return {out, lse};
    HtreeDrafts d{};
    const at::Tensor qq = readable(q, d.q_stride), kk = readable(k, d.k_stride), vv = readable(v, d.v_stride);
    d.q = qq.data_ptr(); d.k = kk.data_ptr(); d.v = vv.data_ptr();
    d.table = table.data_ptr<int32_t>(); d.lengths = lengths.data_ptr<int32_t>(); d.parents = par.defined() ? par.data_ptr<int32_t>() : nullptr;
    d.out = out.data_ptr(); d.lse = want_lse ? lse->data_ptr<float>() : nullptr;
    d.table_stride = table_stride(table);
    d.B = (int32_t)B; d.N = (int32_t)N; d.H = (int32_t)H; d.M = (int32_t)table.size(1);
    d.scale = (float)scale;
    const int64_t bytes = htree_b200_draft_workspace(&cache, &d);
    if (bytes < 0) check(bytes, "draft_attention");
    const c10::DataPtr ws = c10::cuda::CUDACachingAllocator::get()->allocate((size_t)bytes);       // (of the current stream, as the tensors)
    check(htree_b200_draft_attention(&cache, &d, ws.get(), bytes, status_of(status), stream()), "draft_attention");
    return {out, lse};
}

}  // namespace

void bind_cache(py::module& m) {
    m.def("cache_plan", &cache_plan, py::call_guard<py::gil_scoped_release>());
    m.def("cache_append", &cache_append, py::call_guard<py::gil_scoped_release>());
    m.def("cache_gather", &cache_gather, py::call_guard<py::gil_scoped_release>());
    m.def("draft_attention", &draft_attention, py::call_guard<py::gil_scoped_release>());
}
