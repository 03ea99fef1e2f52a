// Bindings of the answering path: paged key/value cache, attention over it, drawing of tokens.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cmath>
#include <string>

#include "ext_api.h"
#include "paged_kv.h"
#include "sampling.h"

namespace {
using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }
int sms() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }
bool given(const OptTensor& t) { return t.has_value() && t->defined(); }
// Numbers in messages go in as text: with some tool chains a stream's number formatting crashes inside an extension.
std::string num(int64_t v) { return std::to_string(v); }
bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int kv_type(const Tensor& t, const char* what) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return sg::kKvBf16;
        case at::kHalf: return sg::kKvFp16;
        case at::kFloat8_e4m3fn: return sg::kKvE4m3;
        case at::kFloat: return sg::kKvFp32;
        default: TORCH_CHECK(false, what, " must be bf16, fp16, fp32 or float8_e4m3fn, not ", c10::toString(t.scalar_type()));
    }
}
const int* index_ptr(const Tensor& t, const Tensor& like, int64_t n, const char* what) {
    TORCH_CHECK(t.device() == like.device() && t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && (n < 2 || t.stride(0) == 1), what, " must be int32 [", num(n),
                "], contiguous, on the cache's device");
    return t.data_ptr<int>();
}

// `t` where its last dimension is contiguous and all before it 16-byte aligned, else a copy that is
Tensor rows16(const Tensor& t) {
    bool ok = aligned(t.data_ptr(), 16) && (t.size(-1) < 2 || t.stride(-1) == 1);
    for (int64_t d = 0; ok && d + 1 < t.dim(); ++d) ok = t.size(d) < 2 || t.stride(d) * t.element_size() % 16 == 0;
    return ok || t.numel() == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
}

// One layer's pages [pages, 2, heads, page size, dim]
sg::KvPages pages_of(const Tensor& kv, const OptTensor& scales) {
    TORCH_CHECK(kv.is_cuda() && kv.dim() == 5 && kv.size(1) == 2, "kv must be a CUDA tensor [pages, 2, kv heads, page size, head size]");
    sg::KvPages k{};
    k.type = kv_type(kv, "kv");
    const int64_t es = kv.element_size();
    TORCH_CHECK(kv.size(0) > 0 && kv.size(2) > 0 && kv.size(3) > 0 && kv.size(4) > 0, "kv must not be empty");
    TORCH_CHECK(kv.size(0) < (int64_t{1} << 31) && kv.size(2) <= 65535, "kv: too many pages or heads");
    TORCH_CHECK(kv.size(3) % 16 == 0 && kv.size(3) <= 65536, "kv: the page size must be a multiple of 16, not ", num(kv.size(3)));
    TORCH_CHECK(kv.size(4) % 8 == 0 && kv.size(4) <= 256 && kv.size(4) * es % 16 == 0, "kv: the head size must fill 16-byte vectors and be at most 256, not ", num(kv.size(4)));
    TORCH_CHECK(kv.stride(4) == 1 && aligned(kv.data_ptr(), 16), "kv: the elements of a head must be contiguous, and 16-byte aligned");
    for (int i = 0; i < 4; ++i) TORCH_CHECK(kv.size(i) == 1 || (kv.stride(i) > 0 && kv.stride(i) * es % 16 == 0), "kv: strides must be positive multiples of 16 bytes");
    k.data = kv.data_ptr();
    k.page_stride = kv.stride(0);
    k.kv_stride = kv.stride(1);
    k.head_stride = kv.stride(2);
    k.tok_stride = kv.stride(3);
    k.num_pages = static_cast<int>(kv.size(0));
    k.heads = static_cast<int>(kv.size(2));
    k.page_size = static_cast<int>(kv.size(3));
    k.dim = static_cast<int>(kv.size(4));
    TORCH_CHECK(given(scales) == (k.type == sg::kKvE4m3), "scales go with a float8_e4m3fn cache, and only with one");
    if (given(scales)) {
        const Tensor& s = *scales;
        TORCH_CHECK(s.device() == kv.device() && s.scalar_type() == at::kFloat && s.dim() == 4 && s.size(0) == kv.size(0) && s.size(1) == 2 && s.size(2) == kv.size(2) &&
                        s.size(3) == kv.size(3),
                    "scales must be fp32 [pages, 2, kv heads, page size] on the cache's device");
        TORCH_CHECK(s.stride(3) == 1 && aligned(s.data_ptr(), 16) && s.stride(0) % 4 == 0 && s.stride(1) % 4 == 0 && s.stride(2) % 4 == 0,
                    "scales: the places of a page must be contiguous and 16-byte aligned");
        k.scales = s.data_ptr<float>();
        k.s_page_stride = s.stride(0);
        k.s_kv_stride = s.stride(1);
        k.s_head_stride = s.stride(2);
    }
    return k;
}
void table_of(const Tensor& table, const Tensor& kv, int64_t B, const int*& ptr, int64_t& stride, int& width) {
    TORCH_CHECK(table.device() == kv.device() && table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == B && (table.size(1) < 2 || table.stride(1) == 1),
                "page_table must be int32 [", num(B), ", pages of a row], rows contiguous, on the cache's device");
    TORCH_CHECK(table.size(1) > 0 && table.size(1) * kv.size(3) <= (int64_t{1} << 30), "page_table: rows must hold 1 to 2^30 tokens");
    ptr = table.data_ptr<int>();
    stride = table.stride(0);
    width = static_cast<int>(table.size(1));
}

void kv_append(const Tensor& kv, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& start, const OptTensor& count, const OptTensor& scales) {
    sg::KvAppend p{};
    p.kv = pages_of(kv, scales);
    TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() && k.device() == kv.device() && v.device() == kv.device() && k.size(2) == p.kv.heads &&
                    k.size(3) == p.kv.dim,
                "k and v must be [rows, tokens, ", num(p.kv.heads), ", ", num(p.kv.dim), "] of one type on the cache's device");
    p.src_type = kv_type(k, "k and v");
    TORCH_CHECK(p.kv.type == sg::kKvE4m3 ? p.src_type != sg::kKvE4m3 : p.src_type == p.kv.type, "k and v must have the cache's type (with an e4m3 cache: bf16, fp16 or fp32)");
    const c10::cuda::CUDAGuard guard(kv.device());
    const Tensor src[2] = {rows16(k), rows16(v)};
    for (int i = 0; i < 2; ++i) {
        const Tensor& t = src[i];
        p.src[i] = t.data_ptr();
        p.b_stride[i] = t.stride(0);
        p.t_stride[i] = t.stride(1);
        p.h_stride[i] = t.stride(2);
    }
    const int64_t B = k.size(0), T = k.size(1);
    TORCH_CHECK(B <= 65535 && T < (int64_t{1} << 30) && B * T * 2 * p.kv.heads < (int64_t{1} << 33), "k and v: at most 65535 rows, and 2^33 heads of tokens, in one call");
    if (B == 0 || T == 0) return;
    table_of(table, kv, B, p.table, p.table_stride, p.table_width);
    p.start = index_ptr(start, kv, B, "start");
    if (given(count)) p.count = index_ptr(*count, kv, B, "count");
    p.B = static_cast<int>(B);
    p.T = static_cast<int>(T);
    p.error_flag = sg_error_flag();
    sg_count_launch(1);
    sg::kv_append(p, cur_stream());
    C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void kv_copy_pages(const Tensor& kv, const Tensor& src, const Tensor& dst, const OptTensor& scales) {
    TORCH_CHECK(kv.is_cuda() && kv.dim() == 6 && kv.size(2) == 2, "kv must be a CUDA tensor [layers, pages, 2, kv heads, page size, head size]");
    TORCH_CHECK(kv.scalar_type() != at::kFloat8_e4m3fn || given(scales), "the scales of a float8_e4m3fn cache are copied with its pages");
    sg::KvCopy p{};
    const Tensor* part[2] = {&kv, given(scales) ? &*scales : nullptr};
    for (int i = 0; i < 2 && part[i]; ++i) {
        const Tensor& t = *part[i];
        if (i) TORCH_CHECK(t.device() == kv.device() && t.scalar_type() == at::kFloat && t.sizes() == kv.sizes().slice(0, 5), "scales must be fp32 [layers, pages, 2, kv heads, page size] on the cache's device");
        const int64_t es = t.element_size(), bytes = t.numel() ? t.numel() / (t.size(0) * t.size(1)) * es : 0;
        int64_t inner = 1;
        bool whole = true;
        for (int64_t d = t.dim() - 1; d >= 2; inner *= t.size(d--)) whole = whole && (t.size(d) < 2 || t.stride(d) == inner);
        TORCH_CHECK(t.numel() == 0 || whole, i ? "scales" : "kv", ": each page must be contiguous");
        TORCH_CHECK(bytes % 16 == 0 && aligned(t.data_ptr(), 16) && t.stride(0) * es % 16 == 0 && t.stride(1) * es % 16 == 0 && t.stride(0) >= 0 && t.stride(1) >= 0,
                    i ? "scales" : "kv", ": pages must be 16-byte aligned");
        p.base[i] = static_cast<uint8_t*>(t.data_ptr());
        p.layer_bytes[i] = t.stride(0) * es;
        p.page_stride_bytes[i] = t.stride(1) * es;
        p.page_bytes[i] = bytes;
    }
    const int64_t n = src.numel();
    TORCH_CHECK(n <= 65535 && kv.size(0) <= 65535 && kv.size(1) < (int64_t{1} << 31), "kv_copy_pages: at most 65535 pairs and layers in one call");
    p.src = index_ptr(src, kv, n, "src");
    p.dst = index_ptr(dst, kv, n, "dst");
    if (n == 0 || kv.numel() == 0) return;
    p.n = static_cast<int>(n);
    p.layers = static_cast<int>(kv.size(0));
    p.num_pages = static_cast<int>(kv.size(1));
    const c10::cuda::CUDAGuard guard(kv.device());
    p.error_flag = sg_error_flag();
    sg_count_launch(1);
    sg::kv_copy_pages(p, sms(), cur_stream());
    C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// -> (output [B, Hq, dim], log-sum-exp fp32 [B, Hq] or undefined)
std::tuple<Tensor, Tensor> paged_attention(const Tensor& q_given, const Tensor& kv, const Tensor& table, const Tensor& lengths, const c10::optional<double>& given_scale, int64_t window, double softcap,
                                    const OptTensor& sinks, const OptTensor& scales, bool want_lse) {
    sg::PagedAttention p{};
    p.kv = pages_of(kv, scales);
    TORCH_CHECK(p.kv.type != sg::kKvFp32, "paged_attention reads bf16, fp16 and float8_e4m3fn caches");
    TORCH_CHECK(p.kv.dim == 64 || p.kv.dim == 128 || p.kv.dim == 256, "paged_attention takes head sizes 64, 128 and 256, not ", num(p.kv.dim));
    TORCH_CHECK(q_given.device() == kv.device() && q_given.dim() == 3 && q_given.size(2) == p.kv.dim, "q must be [rows, query heads, ", num(p.kv.dim), "] on the cache's device");
    const c10::cuda::CUDAGuard guard(kv.device());
    const Tensor q = rows16(q_given);
    p.q_type = kv_type(q, "q");
    TORCH_CHECK(p.kv.type == sg::kKvE4m3 ? p.q_type == sg::kKvBf16 || p.q_type == sg::kKvFp16 : p.q_type == p.kv.type, "q must have the cache's type (with an e4m3 cache: bf16 or fp16)");
    TORCH_CHECK(q.size(1) > 0 && q.size(1) <= 65535 && q.size(1) % p.kv.heads == 0, "the query heads must be a multiple of the ", num(p.kv.heads), " key heads");
    const int64_t B = q.size(0);
    TORCH_CHECK(B <= 65535 && B * q.size(1) < (int64_t{1} << 31), "paged_attention: at most 65535 rows, and 2^31 heads of them, in one call");
    const double scale = given_scale.has_value() ? *given_scale : 1. / std::sqrt(static_cast<double>(p.kv.dim));
    // (fp32 holds the cap, its multiple by log2 e and its inverse)
    TORCH_CHECK(window >= 0 && (softcap == 0 || (softcap >= 0x1p-64 && softcap <= 0x1p64)) && std::isfinite(static_cast<float>(scale)),
                "window must not be negative, softcap 0 or within 2^-64 and 2^64, the scale finite in fp32");
    Tensor out = torch::empty({B, q.size(1), q.size(2)}, q.options()), lse;
    if (want_lse) lse = torch::empty({B, q.size(1)}, q.options().dtype(at::kFloat));
    if (B == 0) return {out, lse};
    table_of(table, kv, B, p.table, p.table_stride, p.table_width);
    p.lengths = index_ptr(lengths, kv, B, "lengths");
    if (given(sinks)) {
        TORCH_CHECK(sinks->device() == kv.device() && sinks->scalar_type() == at::kFloat && sinks->is_contiguous() && sinks->numel() == q.size(1), "sinks must be fp32 [query heads]");
        p.sinks = sinks->data_ptr<float>();
    }
    p.q = q.data_ptr();
    p.q_b_stride = q.stride(0);
    p.q_h_stride = q.stride(1);
    p.out = out.data_ptr();
    p.lse = want_lse ? lse.data_ptr<float>() : nullptr;
    p.B = static_cast<int>(B);
    p.Hq = static_cast<int>(q.size(1));
    const int64_t room = static_cast<int64_t>(p.table_width) * p.kv.page_size;
    p.window = static_cast<int>(window >= room ? 0 : window);
    p.scale = static_cast<float>(scale);
    p.softcap = static_cast<float>(softcap);
    p.error_flag = sg_error_flag();
    const sg::PagedAttentionPlan plan = sg::paged_attention_plan(p.B, p.Hq, p.kv.heads, p.kv.dim, p.kv.type, p.window ? std::min<int64_t>(room, p.window + 64) : room, sms());
    Tensor ws;      // from the caching allocator, on the stream that uses it
    if (plan.workspace_floats) ws = torch::empty({plan.workspace_floats}, q.options().dtype(at::kFloat));
    sg_count_launch(plan.whole ? 1 : 2);
    const char* err = sg::paged_attention(p, plan, plan.workspace_floats ? ws.data_ptr<float>() : nullptr, cur_stream());
    TORCH_CHECK(err == nullptr, err ? err : "");
    return {out, lse};
}

std::tuple<Tensor, Tensor> sample_tokens(const Tensor& logits_given, const Tensor& u, const OptTensor& temperature, const OptTensor& top_k, const OptTensor& top_p, const OptTensor& min_p,
                                         double temperature_all, int64_t top_k_all, double top_p_all, double min_p_all) {
    TORCH_CHECK(logits_given.is_cuda() && logits_given.dim() == 2, "logits must be a CUDA tensor [rows, vocabulary]");
    const c10::cuda::CUDAGuard guard(logits_given.device());
    const Tensor logits = logits_given.size(1) < 2 || logits_given.stride(1) == 1 ? logits_given : logits_given.contiguous();
    sg::SampleTokens p{};
    p.type = kv_type(logits, "logits");
    TORCH_CHECK(p.type != sg::kKvE4m3, "logits must be bf16, fp16 or fp32");
    const int64_t B = logits.size(0), V = logits.size(1);
    // (a million weights of at most 2^44 each: their sum fits 64 bits)
    TORCH_CHECK(V > 0 && V < (int64_t{1} << 20) && B < (int64_t{1} << 27), "logits: the vocabulary must have 1 to 2^20 - 1 tokens, and there may be 2^27 rows");
    auto floats = [&](const OptTensor& t, const char* what) -> const float* {
        if (!given(t)) return nullptr;
        TORCH_CHECK(t->device() == logits.device() && t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == B && (B < 2 || t->stride(0) == 1), what, " must be fp32 [", num(B),
                    "], contiguous, on the logits' device");
        return t->data_ptr<float>();
    };
    p.u = floats(u, "u");
    p.temperature = floats(temperature, "temperature");
    p.top_p = floats(top_p, "top_p");
    p.min_p = floats(min_p, "min_p");
    if (given(top_k)) {
        TORCH_CHECK(top_k->device() == logits.device() && top_k->scalar_type() == at::kInt && top_k->dim() == 1 && top_k->size(0) == B && (B < 2 || top_k->stride(0) == 1),
                    "top_k must be int32 [", num(B), "], contiguous, on the logits' device");
        p.top_k = top_k->data_ptr<int>();
    }
    p.temperature_all = static_cast<float>(temperature_all);
    p.top_k_all = static_cast<int>(std::min<int64_t>(std::max<int64_t>(top_k_all, 0), V));
    p.top_p_all = static_cast<float>(top_p_all);
    p.min_p_all = static_cast<float>(min_p_all);
    Tensor token = torch::empty({B}, logits.options().dtype(at::kInt)), logprob = torch::empty({B}, logits.options().dtype(at::kFloat));
    if (B == 0) return {token, logprob};
    p.logits = logits.data_ptr();
    p.row_stride = logits.stride(0);
    p.B = static_cast<int>(B);
    p.V = static_cast<int>(V);
    p.token = token.data_ptr<int>();
    p.logprob = logprob.data_ptr<float>();
    sg_count_launch(1);
    const char* err = sg::sample_tokens(p, sms(), cur_stream());
    TORCH_CHECK(err == nullptr, err ? err : "");
    return {token, logprob};
}

}  // namespace

void sg_register_decode(pybind11::module_& m) {
    namespace py = pybind11;
    m.def("kv_append", &kv_append, py::arg("kv"), py::arg("k"), py::arg("v"), py::arg("page_table"), py::arg("start"), py::arg("count") = OptTensor(), py::arg("scales") = OptTensor());
    m.def("kv_copy_pages", &kv_copy_pages, py::arg("kv"), py::arg("src"), py::arg("dst"), py::arg("scales") = OptTensor());
    m.def("paged_attention", &paged_attention, py::arg("q"), py::arg("kv"), py::arg("page_table"), py::arg("lengths"), py::arg("scale") = c10::optional<double>(), py::arg("window") = 0,
          py::arg("softcap") = 0.0, py::arg("sinks") = OptTensor(), py::arg("scales") = OptTensor(), py::arg("want_lse") = false);
    m.def("sample_tokens", &sample_tokens, py::arg("logits"), py::arg("u"), py::arg("temperature") = OptTensor(), py::arg("top_k") = OptTensor(), py::arg("top_p") = OptTensor(),
          py::arg("min_p") = OptTensor(), py::arg("temperature_all") = 1.0, py::arg("top_k_all") = 0, py::arg("top_p_all") = 1.0, py::arg("min_p_all") = 0.0);
}
