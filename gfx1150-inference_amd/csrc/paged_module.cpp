// paged_module: the paged-cache and beam-search entry points of include/qmm.h for torch tensors.
//
// Checks a call's tensors, fills the C structures and launches on torch's current stream.  Host code only; paged.py
// and beam.py hold the documented functions.  A decoding step makes these calls once per layer and waits for
// each: the same checks in Python cost 13 us a call, more than most of the kernels; here 6 us.
//
// Refusals are ValueError, other failures of the library RuntimeError, as in qmm.py.
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <optional>
#include <sstream>
#include <string>

#include "qmm.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

void require(bool ok, const char* msg) {
    if (!ok) throw py::value_error(msg);
}

void check(int rc) {
    if (rc == QMM_OK) return;
    if (rc == QMM_ERR_INVALID_ARGUMENT) throw py::value_error(qmm_last_error());
    throw std::runtime_error(qmm_last_error());
}

int code_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return QMM_DTYPE_F32;
        case at::kHalf: return QMM_DTYPE_F16;
        case at::kBFloat16: return QMM_DTYPE_BF16;
        case at::kFloat8_e4m3fn: return QMM_DTYPE_E4M3;
        default: return -1;
    }
}

int32_t int_of(int64_t x, const char* what) {
    if (x < INT32_MIN || x > INT32_MAX) throw py::value_error(std::string(what) + " is out of range");
    return static_cast<int32_t>(x);
}

std::string shape_of(const Tensor& t) {
    std::ostringstream s;
    s << t.sizes();
    return s.str();
}

// An int32 index tensor, its last dimension contiguous (one entry always is); sizes of -1 are free.
void check_ints(const Tensor& t, const char* name, std::initializer_list<int64_t> sizes, c10::Device device) {
    if (t.scalar_type() != at::kInt || t.device() != device || t.dim() != static_cast<int64_t>(sizes.size()) || (t.numel() > 0 && t.size(-1) > 1 && t.stride(-1) != 1))
        throw py::value_error(std::string(name) + " must be an int32 tensor of " + std::to_string(sizes.size()) +
                              " dimension(s) on the cache's device, its last one contiguous");
    int64_t d = 0;
    for (int64_t want : sizes) {
        if (want >= 0 && t.size(d) != want) throw py::value_error(std::string(name) + " has shape " + shape_of(t) + ", which does not fit the call");
        ++d;
    }
}

// The cache of checked arguments.
qmm_paged_kv cache_of(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor* cu, const Tensor& ctx, double k_scale,
                      double v_scale, bool layered) {
    const int64_t dims = layered ? 5 : 4;
    require(k.dim() == dims && v.sizes() == k.sizes(), layered ? "k_cache and v_cache must be alike: [layers, pages, kv_heads, page_size, head_dim]"
                                                               : "k_cache and v_cache must be alike: [pages, kv_heads, page_size, head_dim]");
    const int code = code_of(k.scalar_type());
    require(code >= 0 && code != QMM_DTYPE_F32 && v.scalar_type() == k.scalar_type(), "k_cache and v_cache must both be float16, bfloat16 or float8_e4m3fn");
    const c10::Device device = k.device();
    require(device.is_cuda() && v.device() == device, "k_cache and v_cache must be on one GPU");
    require(k.stride(-1) == 1 && v.stride(-1) == 1, "head_dim must be contiguous in k_cache and v_cache");
    check_ints(ctx, "ctx", {-1}, device);
    const int64_t batch = ctx.size(0);
    check_ints(table, "table", {batch, -1}, device);
    if (cu) check_ints(*cu, "cu", {batch + 1}, device);
    const int64_t at = layered ? 1 : 0;
    qmm_paged_kv c{};
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    c.table = static_cast<const int32_t*>(table.data_ptr());
    c.cu = cu ? static_cast<const int32_t*>(cu->data_ptr()) : nullptr;
    c.ctx = static_cast<const int32_t*>(ctx.data_ptr());
    c.table_stride = table.stride(0);
    c.k_layer = layered ? k.stride(0) : 0;
    c.k_page = k.stride(at);
    c.k_head = k.stride(at + 1);
    c.k_slot = k.stride(at + 2);
    c.v_layer = layered ? v.stride(0) : 0;
    c.v_page = v.stride(at);
    c.v_head = v.stride(at + 1);
    c.v_slot = v.stride(at + 2);
    c.table_width = int_of(table.size(1), "table's width");
    c.batch = int_of(batch, "batch");
    c.dtype = code;
    c.num_layers = layered ? int_of(k.size(0), "the count of layers") : 1;
    c.num_pages = int_of(k.size(at), "the count of pages");
    c.kv_heads = int_of(k.size(at + 1), "kv_heads");
    c.page_size = int_of(k.size(at + 2), "page_size");
    c.head_dim = int_of(k.size(at + 3), "head_dim");
    c.k_scale = static_cast<float>(k_scale);
    c.v_scale = static_cast<float>(v_scale);
    return c;
}

// New tokens [tokens, heads, head_dim]; heads and tokens of -1 are free.
void check_rows(const Tensor& x, const char* name, int64_t tokens, int64_t heads, const Tensor& cache, at::ScalarType dtype) {
    if (x.dim() != 3 || x.size(2) != cache.size(-1) || (heads >= 0 && x.size(1) != heads) || (tokens >= 0 && x.size(0) != tokens))
        throw py::value_error(std::string(name) + " must be [tokens, heads, head_dim] of the call, got " + shape_of(x));
    if (x.scalar_type() != dtype || x.device() != cache.device())
        throw py::value_error(std::string(name) + " must be of the call's type and on the cache's device");
    if (x.stride(2) != 1) throw py::value_error(std::string("head_dim must be contiguous in ") + name);
}

// The current stream; the caller's current device must be the tensors'.
void* stream_of(c10::Device device) {
    const auto current = c10::hip::current_device();
    if (device.index() != current)
        throw py::value_error("the tensors are on cuda:" + std::to_string(device.index()) + ", the current device is cuda:" + std::to_string(current));
    return c10::hip::getCurrentHIPStream(device.index()).stream();
}

Tensor ints(at::IntArrayRef sizes, c10::Device device) { return at::empty(sizes, at::TensorOptions().dtype(at::kInt).device(device)); }

OptTensor append(const Tensor& k, const Tensor& v, const Tensor& k_cache, const Tensor& v_cache, const Tensor& table, const Tensor& cu,
                 const Tensor& ctx, const OptTensor& q, OptTensor q_out, const OptTensor& positions, double freq_base,
                 std::optional<int64_t> rotary_dim, bool neox, double k_scale, double v_scale) {
    require(k.is_cuda(), "k must be on a GPU");
    const qmm_paged_kv kv = cache_of(k_cache, v_cache, table, &cu, ctx, k_scale, v_scale, false);
    const auto dtype = k.scalar_type();
    require(dtype == at::kHalf || dtype == at::kBFloat16, "k, v and q must be float16 or bfloat16");
    require(k.dim() == 3, "k must be [tokens, kv_heads, head_dim]");
    const int64_t tokens = k.size(0);
    check_rows(k, "k", tokens, kv.kv_heads, k_cache, dtype);
    check_rows(v, "v", tokens, kv.kv_heads, k_cache, dtype);
    qmm_paged_new in{};
    in.k = k.data_ptr();
    in.v = v.data_ptr();
    in.k_token = k.stride(0);
    in.k_head = k.stride(1);
    in.v_token = v.stride(0);
    in.v_head = v.stride(1);
    if (positions) {
        check_ints(*positions, "positions", {tokens}, k_cache.device());
        in.positions = static_cast<const int32_t*>(positions->data_ptr());
    }
    if (q) {
        check_rows(*q, "q", tokens, -1, k_cache, dtype);
        if (!q_out) q_out = at::empty(q->sizes(), at::TensorOptions().dtype(dtype).device(q->device()));
        check_rows(*q_out, "q_out", tokens, q->size(1), k_cache, dtype);
        in.q = q->data_ptr();
        in.q_out = q_out->data_ptr();
        in.heads = int_of(q->size(1), "heads");
        in.q_token = q->stride(0);
        in.q_head = q->stride(1);
        in.qo_token = q_out->stride(0);
        in.qo_head = q_out->stride(1);
    } else {
        require(!q_out, "q_out needs q");
    }
    in.tokens = int_of(tokens, "the count of tokens");
    in.dtype = code_of(dtype);
    in.rotary_dim = int_of(rotary_dim.value_or(kv.head_dim), "rotary_dim");
    in.neox = neox ? 1 : 0;
    in.freq_base = static_cast<float>(freq_base);
    check(qmm_paged_append(&kv, &in, stream_of(k_cache.device())));
    return q_out;
}

Tensor tree_attention(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& table, const Tensor& cu, const Tensor& ctx,
                      const OptTensor& mask, std::optional<int64_t> max_new, std::optional<double> scale, double k_scale, double v_scale,
                      OptTensor out) {
    require(q.is_cuda(), "q must be on a GPU");
    const qmm_paged_kv kv = cache_of(k_cache, v_cache, table, &cu, ctx, k_scale, v_scale, false);
    const auto dtype = q.scalar_type();
    require(dtype == at::kHalf || dtype == at::kBFloat16, "q must be float16 or bfloat16");
    check_rows(q, "q", -1, -1, k_cache, dtype);
    const int64_t tokens = q.size(0);
    if (!out) out = at::empty(q.sizes(), at::TensorOptions().dtype(dtype).device(q.device()));
    check_rows(*out, "out", tokens, q.size(1), k_cache, dtype);
    qmm_paged_query in{};
    in.q = q.data_ptr();
    in.out = out->data_ptr();
    in.q_token = q.stride(0);
    in.q_head = q.stride(1);
    in.out_token = out->stride(0);
    in.out_head = out->stride(1);
    if (mask) {
        check_ints(*mask, "mask", {tokens, -1}, k_cache.device());
        require(mask->size(1) > 0 || tokens == 0, "mask has no words");
        in.mask = static_cast<const int32_t*>(mask->data_ptr());
        in.mask_stride = mask->stride(0);
        in.mask_words = int_of(mask->size(1), "the count of mask words");
    }
    in.tokens = int_of(tokens, "the count of tokens");
    in.max_new = int_of(max_new.value_or(tokens), "max_new");
    in.heads = int_of(q.size(1), "heads");
    in.dtype = code_of(dtype);
    in.scale = static_cast<float>(scale.value_or(0.0));  // 0: the default
    require(!scale || in.scale != 0.0f, "scale must not be 0 in 32 bits");
    void* stream = stream_of(k_cache.device());
    const size_t need = qmm_paged_attention_workspace(&kv, &in);
    Tensor space;  // the allocator's: safe to capture
    if (need) space = at::empty({static_cast<int64_t>(need)}, at::TensorOptions().dtype(at::kByte).device(q.device()));
    check(qmm_paged_tree_attention(&kv, &in, need ? space.data_ptr() : nullptr, need, stream));
    return *out;
}

Tensor commit_path(const Tensor& k_cache, const Tensor& v_cache, const Tensor& table, const Tensor& cu, const Tensor& ctx, const Tensor& path) {
    require(path.is_cuda(), "path must be on a GPU");
    const qmm_paged_kv kv = cache_of(k_cache, v_cache, table, &cu, ctx, 1.0, 1.0, true);
    check_ints(path, "path", {kv.batch, -1}, k_cache.device());
    Tensor lens = ints({kv.batch}, k_cache.device());
    check(qmm_paged_commit_path(&kv, static_cast<const int32_t*>(path.data_ptr()), path.stride(0), int_of(path.size(1), "the path's length"),
                                static_cast<int32_t*>(lens.data_ptr()), stream_of(k_cache.device())));
    return lens;
}

std::tuple<Tensor, Tensor, Tensor> beam_select(const Tensor& logits, const Tensor& scores) {
    require(logits.is_cuda() && logits.dim() == 3, "logits must be a [sentences, beams, vocab] tensor on a GPU");
    const int code = code_of(logits.scalar_type());
    require(code >= 0 && code != QMM_DTYPE_E4M3, "logits must be float32, float16 or bfloat16");
    const int64_t S = logits.size(0), W = logits.size(1), V = logits.size(2);
    require(logits.stride(2) == 1 || V <= 1, "vocab must be contiguous in logits");
    const c10::Device device = logits.device();
    require(scores.scalar_type() == at::kFloat && scores.device() == device && scores.dim() == 2 && scores.size(0) == S && scores.size(1) == W &&
                scores.is_contiguous(),
            "scores must be a contiguous float32 [sentences, beams] tensor on the logits' device");
    const int s = int_of(S, "the count of sentences"), w = int_of(W, "beams"), vocab = int_of(V, "vocab");
    Tensor best = at::empty({S, W}, scores.options()), both = ints({2, S, W}, device);
    Tensor parents = both.select(0, 0), tokens = both.select(0, 1);
    void* stream = stream_of(device);
    const size_t need = qmm_beam_select_workspace(code, s, w, vocab);
    Tensor space = at::empty({static_cast<int64_t>(need)}, at::TensorOptions().dtype(at::kByte).device(device));
    check(qmm_beam_select(logits.data_ptr(), code, logits.stride(0), logits.stride(1), static_cast<const float*>(scores.data_ptr()), s, w, vocab,
                          static_cast<float*>(best.data_ptr()), static_cast<int32_t*>(parents.data_ptr()),
                          static_cast<int32_t*>(tokens.data_ptr()), space.data_ptr(), need, stream));
    return {best, parents, tokens};
}

std::tuple<Tensor, Tensor> beam_reorder(const Tensor& k_cache, const Tensor& v_cache, const Tensor& table, const Tensor& lens,
                                        const Tensor& parents, const Tensor& fresh) {
    require(parents.is_cuda(), "parents must be on a GPU");
    const qmm_paged_kv kv = cache_of(k_cache, v_cache, table, nullptr, lens, 1.0, 1.0, true);
    const c10::Device device = k_cache.device();
    check_ints(parents, "parents", {-1, -1}, device);
    check_ints(fresh, "fresh", {parents.size(0), parents.size(1)}, device);
    require(parents.numel() == kv.batch && parents.is_contiguous() && fresh.is_contiguous(),
            "parents and fresh must be contiguous and hold one entry per sequence");
    Tensor new_table = ints(table.sizes(), device), new_lens = ints(lens.sizes(), device);
    check(qmm_beam_reorder(&kv, static_cast<const int32_t*>(parents.data_ptr()), static_cast<const int32_t*>(fresh.data_ptr()),
                           int_of(parents.size(1), "beams"), static_cast<int32_t*>(new_table.data_ptr()),
                           static_cast<int32_t*>(new_lens.data_ptr()), stream_of(device)));
    return {new_table, new_lens};
}

}  // namespace

PYBIND11_MODULE(paged_module, m) {
    m.doc() = "Paged key/value cache and beam search on torch tensors (see paged.py and beam.py)";
    m.def("append", &append);
    m.def("tree_attention", &tree_attention);
    m.def("commit_path", &commit_path);
    m.def("beam_select", &beam_select);
    m.def("beam_reorder", &beam_reorder);
}
