// tvq_torch.cpp -- the decoding operators on torch CUDA tensors: checks, output
// and scratch tensors, the current stream, and the call of libtvq's C ABI
// (include/tvq.h).  A decoding loop makes these calls once a layer and step,
// and a step of a small model is a few microseconds on the GPU: checked in
// Python and passed through ctypes, a call took the host 15-20 us, here 6-12.
#include <torch/extension.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <string>
#include <tuple>

#include "tvq.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

void need(bool ok, const char* msg) {
    if (!ok) throw py::value_error(msg);
}

// The library's error as the package raises it (ValueError for sizes, TvqError else).
void check(int rc) {
    if (rc == TVQ_OK) return;
    py::gil_scoped_acquire gil;
    py::module_::import("tokenvector.inference_b200._native").attr("check")(rc);
}

int type_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return TVQ_TYPE_F32;
        case at::kHalf: return TVQ_TYPE_F16;
        case at::kBFloat16: return TVQ_TYPE_BF16;
        default: return -1;
    }
}

void same_device(const Tensor& t, at::Device dev, const char* name) {
    if (t.device() != dev) throw py::value_error(std::string(name) + " is on " + t.device().str() + ", not on " + dev.str());
}
void same_device(const OptTensor& t, at::Device dev, const char* name) {
    if (t) same_device(*t, dev, name);
}

const int32_t* i32_of(const Tensor& t, int ndim, const char* name) {
    if (t.scalar_type() != at::kInt || t.dim() != ndim)
        throw py::value_error(std::string(name) + " must be an int32 tensor of " + std::to_string(ndim) + " dimension(s)");
    if (t.size(ndim - 1) > 1 && t.stride(ndim - 1) != 1)
        throw py::value_error(std::string(name) + " must be contiguous in its last dimension");
    return static_cast<const int32_t*>(t.data_ptr());
}

// Elements from row to row (a row alone may have any stride; 0: an expanded tensor, all rows are the first).
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : std::max(t.stride(0), t.size(1)); }

void* ptr(const Tensor& t) { return t.data_ptr(); }
void* ptr(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }

// The operators have no backward pass: an output that a gradient is expected of would silently have none.
void no_grad(const Tensor& t, const char* name) {
    if (t.requires_grad() && at::GradMode::is_enabled())
        throw py::value_error(std::string(name) + " requires a gradient, which this operator does not have: detach it, or "
                                                  "call under torch.no_grad()");
}
void no_grad(const OptTensor& t, const char* name) {
    if (t) no_grad(*t, name);
}

// Scratch of one call (stream-ordered memory of torch's allocator).
Tensor workspace(at::Device dev, int64_t bytes) {
    return at::empty({bytes}, at::TensorOptions().dtype(at::kByte).device(dev));
}

// One layer's cache and the sequences in it, checked, as the C ABI takes them.
struct Cache {
    int type;
    int64_t shape[4], strides[6];
    const int32_t *table, *ctx, *cu;
    int64_t table_stride, cols, seqs;
};
Cache cache_of(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& ctx, const OptTensor& cu, int64_t n_rows) {
    no_grad(k, "k_pages");
    no_grad(v, "v_pages");
    need(k.is_cuda(), "the cache must be on a CUDA device");
    Cache c;
    c.type = type_of(k);
    need((c.type == TVQ_TYPE_F16 || c.type == TVQ_TYPE_BF16) && v.scalar_type() == k.scalar_type(),
         "k_pages and v_pages must both be float16 or both bfloat16");
    need(k.dim() == 4 && v.sizes() == k.sizes(), "k_pages and v_pages must be [pages, page, kv_heads, head_dim], alike");
    need(k.stride(3) == 1 && v.stride(3) == 1, "the cache's last dimension must be contiguous");
    c.table = i32_of(table, 2, "table");
    c.ctx = i32_of(ctx, 1, "ctx_len");
    c.seqs = ctx.size(0);
    need(table.size(0) == c.seqs, "table must have one row for each sequence");
    c.cu = nullptr;
    if (cu) {
        c.cu = i32_of(*cu, 1, "cu");
        need(cu->size(0) == c.seqs + 1, "cu must hold one entry more than there are sequences");
    } else {
        need(n_rows == c.seqs, "without cu every sequence has one row");
    }
    const at::Device dev = k.device();
    same_device(v, dev, "v_pages");
    same_device(table, dev, "table");
    same_device(ctx, dev, "ctx_len");
    same_device(cu, dev, "cu");
    for (int i = 0; i < 4; i++) c.shape[i] = k.size(i);
    for (int i = 0; i < 3; i++) {
        c.strides[i] = k.stride(i);
        c.strides[3 + i] = v.stride(i);
    }
    c.table_stride = row_stride(table);
    c.cols = table.size(1);
    return c;
}

void rows_of(const Tensor& t, int64_t heads, int64_t dim, const char* name) {
    if (t.dim() != 3 || (heads >= 0 && t.size(1) != heads) || t.size(2) != dim)
        throw py::value_error(std::string(name) + " must be [rows, heads, head_dim] like the cache");
    if (t.stride(2) != 1) throw py::value_error(std::string(name) + " must be contiguous in its last dimension");
}

OptTensor paged_append(const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table,
                       const Tensor& ctx_len, const OptTensor& cu, const OptTensor& q) {
    no_grad(k, "k");
    no_grad(v, "v");
    no_grad(q, "q");
    need(k.dim() == 3, "k must be [rows, heads, head_dim] like the cache");
    const Cache c = cache_of(k_pages, v_pages, table, ctx_len, cu, k.size(0));
    rows_of(k, c.shape[2], c.shape[3], "k");
    rows_of(v, c.shape[2], c.shape[3], "v");
    need(type_of(k) >= 0 && v.scalar_type() == k.scalar_type() && v.size(0) == k.size(0),
         "k and v must be float32, float16 or bfloat16 rows, alike");
    int64_t strides[6] = {k.stride(0), k.stride(1), v.stride(0), v.stride(1), 0, 0}, q_heads = 0;
    const at::Device dev = k_pages.device();
    same_device(k, dev, "k");
    same_device(v, dev, "v");
    OptTensor out;
    c10::cuda::CUDAGuard guard(dev);
    if (q) {
        rows_of(*q, -1, c.shape[3], "q");
        need(q->scalar_type() == k.scalar_type() && q->size(0) == k.size(0), "q must have k's type and rows");
        same_device(q, dev, "q");
        q_heads = q->size(1);
        strides[4] = q->stride(0);
        strides[5] = q->stride(1);
        out = at::empty(q->sizes(), k_pages.options());
    }
    check(tvq_dev_paged_append(c.type, type_of(k), ptr(k), ptr(v), ptr(q), strides, q_heads, ptr(out), ptr(k_pages),
                               ptr(v_pages), c.shape, c.strides, c.table, c.table_stride, c.cols, c.ctx, c.cu, c.seqs,
                               k.size(0), c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
    return out;
}

std::tuple<Tensor, OptTensor> paged_attention(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table,
                                              const Tensor& ctx_len, const OptTensor& cu, std::optional<int64_t> max_q,
                                              std::optional<double> scale, int64_t window, const OptTensor& given,
                                              bool return_lse) {
    no_grad(q, "q");
    need(q.dim() == 3, "q must be [rows, heads, head_dim] like the cache");
    const int64_t n_rows = q.size(0), heads = q.size(1);
    const Cache c = cache_of(k_pages, v_pages, table, ctx_len, cu, n_rows);
    rows_of(q, -1, c.shape[3], "q");
    need(q.scalar_type() == k_pages.scalar_type(), "q must have the cache's type");
    need(heads > 0 && c.shape[2] > 0 && heads % c.shape[2] == 0, "q's heads must be a multiple of the cache's");
    need(window >= 0, "window must not be negative");
    const at::Device dev = k_pages.device();
    same_device(q, dev, "q");
    c10::cuda::CUDAGuard guard(dev);
    Tensor out;
    if (given) {
        need(given->sizes() == q.sizes() && given->scalar_type() == q.scalar_type() && given->is_contiguous(),
             "out must be contiguous, with q's shape and type");
        same_device(given, dev, "out");
        out = *given;
    } else {
        out = at::empty(q.sizes(), k_pages.options());
    }
    OptTensor lse;
    if (return_lse) lse = at::empty({n_rows, heads}, at::TensorOptions().dtype(at::kFloat).device(dev));
    const int64_t most = max_q ? *max_q : cu ? n_rows : 1, strides[2] = {q.stride(0), q.stride(1)};
    const cudaStream_t st = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    int64_t bytes = 0;
    check(tvq_paged_attention_workspace(heads, c.shape[2], c.shape[3], c.seqs, n_rows, most, &bytes));
    const Tensor ws = workspace(dev, bytes);
    check(tvq_dev_paged_attention(c.type, ptr(q), strides, heads, ptr(k_pages), ptr(v_pages), c.shape, c.strides, c.table,
                                  c.table_stride, c.cols, c.ctx, c.cu, c.seqs, n_rows, most,
                                  static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(c.shape[3]))), window,
                                  ptr(out), static_cast<float*>(ptr(lse)), ptr(ws), bytes, st));
    return {out, lse};
}

std::tuple<Tensor, Tensor, Tensor> beam_select(const Tensor& logits, const Tensor& scores, int64_t beams, int64_t keep,
                                               const OptTensor& finished, std::optional<int64_t> eos) {
    no_grad(logits, "logits");
    no_grad(scores, "scores");
    need(logits.dim() == 2 && type_of(logits) >= 0 && logits.is_cuda(),
         "logits must be a [rows, vocab] tensor of floats on a CUDA device");
    const int64_t rows = logits.size(0), vocab = logits.size(1);
    need(beams >= 1 && rows % beams == 0, "logits must have batch * beams rows");
    need(vocab <= 1 || logits.stride(1) == 1, "logits must be contiguous in the vocabulary");
    need(scores.scalar_type() == at::kFloat && scores.dim() == 1 && scores.size(0) == rows && scores.is_contiguous(),
         "scores must be float32, one for each row of logits");
    need(keep <= vocab, "keep larger than the vocabulary");
    const at::Device dev = logits.device();
    if (finished) {
        need(finished->scalar_type() == at::kBool && finished->dim() == 1 && finished->size(0) == rows && finished->is_contiguous(),
             "finished must be bool, one for each row of logits");
        need(eos.has_value(), "finished beams need eos");
    }
    same_device(scores, dev, "scores");
    same_device(finished, dev, "finished");
    c10::cuda::CUDAGuard guard(dev);
    const int64_t batch = rows / beams;
    const auto opts = at::TensorOptions().device(dev);
    const Tensor out = at::empty({batch, std::max<int64_t>(keep, 0)}, opts.dtype(at::kFloat));
    const Tensor tokens = at::empty(out.sizes(), opts.dtype(at::kLong)), parents = at::empty(out.sizes(), opts.dtype(at::kInt));
    const cudaStream_t st = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    int64_t bytes = 0;
    check(tvq_beam_select_workspace(batch, beams, keep, vocab, &bytes));
    const Tensor ws = workspace(dev, bytes);
    check(tvq_dev_beam_select(type_of(logits), ptr(logits), row_stride(logits), static_cast<const float*>(ptr(scores)),
                              static_cast<const uint8_t*>(ptr(finished)), batch, beams, keep, vocab, eos ? *eos : -1,
                              static_cast<float*>(ptr(out)), static_cast<int64_t*>(ptr(tokens)),
                              static_cast<int32_t*>(ptr(parents)), ptr(ws), bytes, st));
    return {out, tokens, parents};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> beam_reorder(const Tensor& table, const Tensor& lens, const Tensor& parents,
                                                        const Tensor& refs, const Tensor& k, const Tensor& v) {
    no_grad(k, "k_pages");
    no_grad(v, "v_pages");
    const int32_t* table_p = i32_of(table, 2, "table");
    const int32_t* lens_p = i32_of(lens, 1, "lens");
    const int32_t* parents_p = i32_of(parents, 1, "parents");
    const int32_t* refs_p = i32_of(refs, 1, "refs");
    need(table.is_cuda(), "the tables must be on a CUDA device");
    need(lens.size(0) == table.size(0), "lens must have one entry for each row of the table");
    need(k.dim() == 5 && v.sizes() == k.sizes() && (k.scalar_type() == at::kHalf || k.scalar_type() == at::kBFloat16) &&
             v.scalar_type() == k.scalar_type(),
         "k_pages and v_pages must be [layers, pages, page, kv_heads, head_dim], both float16 or both bfloat16");
    need(k.stride(4) == 1 && v.stride(4) == 1, "the cache's last dimension must be contiguous");
    need(refs.size(0) == k.size(1), "refs must have one entry for each page");
    const at::Device dev = table.device();
    same_device(lens, dev, "lens");
    same_device(parents, dev, "parents");
    same_device(refs, dev, "refs");
    same_device(k, dev, "k_pages");
    same_device(v, dev, "v_pages");
    c10::cuda::CUDAGuard guard(dev);
    const int64_t rows = table.size(0), cols = table.size(1), new_rows = parents.size(0), pages = refs.size(0);
    const auto opts = at::TensorOptions().dtype(at::kInt).device(dev);
    const Tensor new_table = at::empty({new_rows, cols}, opts), new_lens = at::empty({new_rows}, opts);
    const Tensor new_refs = at::empty({pages}, opts), status = at::empty({2}, opts);
    const int64_t shape[5] = {pages, k.size(2), k.size(3), k.size(4), k.size(0)};
    int64_t strides[8];
    for (int i = 0; i < 4; i++) {
        strides[i] = k.stride(i);
        strides[4 + i] = v.stride(i);
    }
    const cudaStream_t st = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    int64_t bytes = 0;
    check(tvq_beam_reorder_workspace(pages, rows, new_rows, &bytes));
    const Tensor ws = workspace(dev, bytes);
    auto i32 = [](const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); };
    check(tvq_dev_beam_reorder(table_p, row_stride(table), lens_p, rows, cols, parents_p, new_rows, refs_p, ptr(k),
                               ptr(v), shape, strides, i32(new_table), i32(new_lens), i32(new_refs), i32(status), ptr(ws), bytes,
                               st));
    return {new_table, new_lens, new_refs, status};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    using NoGil = py::call_guard<py::gil_scoped_release>;  // a launch may wait for room in the queue
    m.def("paged_append", &paged_append, NoGil());
    m.def("paged_attention", &paged_attention, NoGil());
    m.def("beam_select", &beam_select, NoGil());
    m.def("beam_reorder", &beam_reorder, NoGil());
}
