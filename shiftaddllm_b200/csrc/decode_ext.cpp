// The 4-bit cache and the sampler for torch tensors, in the compiled `lutgemm` extension module: the argument checks of
// shiftaddllm_b200/decode_ops.py and the call of the C ABI (include/sal_decode_ops.h).  A call of one token is a few microseconds of GPU work;
// the same steps in Python cost 12 to 15.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cmath>
#include <string>
#include <vector>

#include "sal_decode_ops.h"
#include "sal_lutgemm.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

void check_status(int rc, const char *what) {
    if (rc == SAL_OK) return;
    std::string msg = std::string(what) + " failed: " + sal_status_string(rc) + " (status " + std::to_string(rc) + ")";
    if (rc == SAL_E_LAUNCH) msg += std::string("; CUDA: ") + sal_last_cuda_error();
    TORCH_CHECK(false, msg);
}

// A contiguous tensor of this dtype on this device: so many numbers in all, so many in its last dimension.
void want(const char *what, const char *name, const Tensor &t, c10::ScalarType dtype, int64_t numel, int64_t last, c10::Device device) {
    TORCH_CHECK(t.device() == device && t.scalar_type() == dtype && t.is_contiguous() && t.numel() == numel && (t.dim() == 0 || t.size(-1) == last), what, ": ",
                name, " must be a contiguous ", c10::toString(dtype), " tensor of ", numel, " numbers, ", last, " in its last dimension, on ", device, ", got ",
                t.sizes(), " ", c10::toString(t.scalar_type()), " on ", t.device());
}

struct Cache {
    c10::Device device;
    int64_t batch, max_pages, pages;
};
Cache check_cache(const char *what, const Tensor &pool, const Tensor &table, const Tensor &pos, const OptTensor &rows, int64_t kv_heads, int64_t hd) {
    TORCH_CHECK(pool.is_cuda(), what, ": pool must be a CUDA tensor (there is no CPU path)");
    TORCH_CHECK(hd == 64 || hd == 128 || hd == 256, "the 4-bit cache takes heads of 64, 128 or 256 numbers, got ", hd);
    const int64_t record = SAL_KV4_PAGE * (hd + hd / 8), batch = pos.numel();
    TORCH_CHECK(pool.dim() == 3 && pool.size(1) == kv_heads && pool.size(2) == record && pool.scalar_type() == torch::kUInt8 && pool.is_contiguous(), what,
                ": pool must be a contiguous uint8 tensor [pages, ", kv_heads, ", ", record, "], got ", pool.sizes(), " ", c10::toString(pool.scalar_type()));
    want(what, "pos", pos, torch::kInt64, batch, batch, pool.device());
    TORCH_CHECK(table.dim() == 2 && table.size(0) == batch && table.size(1) >= 1, what, ": table must be an int32 tensor [", batch, ", pages of a sequence]");
    want(what, "table", table, torch::kInt32, table.numel(), table.size(1), pool.device());
    if (rows.has_value()) want(what, "rows", *rows, torch::kInt32, batch, batch, pool.device());
    return {pool.device(), batch, table.size(1), pool.size(0)};
}
int64_t rows_per_sequence(const char *what, const char *name, const Tensor &t, int64_t batch, int64_t width) {
    TORCH_CHECK(batch >= 1 && width >= 1 && t.numel() > 0 && t.numel() % (batch * width) == 0, what, ": ", name, " must hold the same number of rows of ", width,
                " numbers for each of ", batch, " sequences");
    return t.numel() / (batch * width);
}
int whole(const char *what, int64_t v) {
    TORCH_CHECK(v >= -0x7fffffff && v <= 0x7fffffff, what, ": ", v, " is too large");
    return (int)v;
}
void *stream_of(c10::Device device) { return at::cuda::getCurrentCUDAStream(device.index()).stream(); }

void rope_kv4_write(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &cos, const Tensor &sin, const Tensor &pos, const Tensor &table,
                    const Tensor &pool, const Tensor &q_out, int64_t heads, int64_t kv_heads, int64_t hd, const OptTensor &rows) {
    const char *what = "rope_kv4_write";
    const Cache c = check_cache(what, pool, table, pos, rows, kv_heads, hd);
    const int64_t m = rows_per_sequence(what, "q", q, c.batch, heads * hd), nq = c.batch * m * heads * hd, nk = c.batch * m * kv_heads * hd;
    want(what, "q", q, torch::kFloat16, nq, heads * hd, c.device);
    want(what, "q_out", q_out, torch::kFloat16, nq, heads * hd, c.device);
    want(what, "k", k, torch::kFloat16, nk, kv_heads * hd, c.device);
    want(what, "v", v, torch::kFloat16, nk, kv_heads * hd, c.device);
    const int64_t angles = cos.numel() / (hd / 2);
    want(what, "cos", cos, torch::kFloat32, angles * (hd / 2), hd / 2, c.device);
    want(what, "sin", sin, torch::kFloat32, angles * (hd / 2), hd / 2, c.device);
    c10::cuda::CUDAGuard guard(c.device);
    check_status(sal_rope_kv4_write_f16(q.data_ptr(), k.data_ptr(), v.data_ptr(), cos.data_ptr(), sin.data_ptr(), pos.data_ptr<int64_t>(),
                                        rows.has_value() ? rows->data_ptr<int32_t>() : nullptr, table.data_ptr<int32_t>(), pool.data_ptr(), q_out.data_ptr(),
                                        whole(what, c.batch), whole(what, m), whole(what, heads), whole(what, kv_heads), (int)hd, whole(what, angles),
                                        whole(what, c.max_pages), whole(what, c.pages), stream_of(c.device)),
                 "sal_rope_kv4_write_f16");
}

void read_kv4(const Tensor &pool, const Tensor &table, const Tensor &pos, const Tensor &k_out, const Tensor &v_out, int64_t kv_heads, int64_t hd) {
    const char *what = "read_kv4";
    const Cache c = check_cache(what, pool, table, pos, c10::nullopt, kv_heads, hd);
    const int64_t m = rows_per_sequence(what, "k_out", k_out, c.batch, kv_heads * hd);
    const auto dtype = k_out.scalar_type();
    TORCH_CHECK(dtype == torch::kFloat32 || dtype == torch::kFloat16, what, ": k_out must be float32 or float16, got ", c10::toString(dtype));
    want(what, "k_out", k_out, dtype, c.batch * m * kv_heads * hd, hd, c.device);
    want(what, "v_out", v_out, dtype, c.batch * m * kv_heads * hd, hd, c.device);
    c10::cuda::CUDAGuard guard(c.device);
    check_status(sal_read_kv4(pool.data_ptr(), table.data_ptr<int32_t>(), pos.data_ptr<int64_t>(), k_out.data_ptr(), v_out.data_ptr(), dtype == torch::kFloat32,
                              whole(what, c.batch), whole(what, m), whole(what, kv_heads), (int)hd, whole(what, c.max_pages), whole(what, c.pages),
                              stream_of(c.device)),
                 "sal_read_kv4");
}

void attention_kv4(const Tensor &q, const Tensor &pool, const Tensor &table, const Tensor &pos, const Tensor &out, int64_t heads, int64_t kv_heads, int64_t hd,
                   double scale, const Tensor &workspace, const OptTensor &rows) {
    const char *what = "attention_kv4";
    const Cache c = check_cache(what, pool, table, pos, rows, kv_heads, hd);
    const int64_t m = rows_per_sequence(what, "q", q, c.batch, heads * hd);
    want(what, "q", q, torch::kFloat16, c.batch * m * heads * hd, heads * hd, c.device);
    want(what, "out", out, torch::kFloat16, c.batch * m * heads * hd, heads * hd, c.device);
    want(what, "workspace", workspace, torch::kUInt8, workspace.numel(), workspace.dim() ? workspace.size(-1) : 0, c.device);
    c10::cuda::CUDAGuard guard(c.device);
    check_status(sal_attention_kv4_f16(q.data_ptr(), pool.data_ptr(), table.data_ptr<int32_t>(), pos.data_ptr<int64_t>(),
                                       rows.has_value() ? rows->data_ptr<int32_t>() : nullptr, out.data_ptr(), whole(what, c.batch), whole(what, m),
                                       whole(what, heads), whole(what, kv_heads), (int)hd, whole(what, c.max_pages), whole(what, c.pages), (float)scale,
                                       workspace.data_ptr(), (size_t)workspace.numel(), stream_of(c.device)),
                 "sal_attention_kv4_f16");
}

void copy_kv4_pages(const Tensor &pool, const std::vector<int64_t> &src, const std::vector<int64_t> &dst) {
    const char *what = "copy_kv4_pages";
    TORCH_CHECK(pool.is_cuda() && pool.scalar_type() == torch::kUInt8 && pool.dim() >= 3 && pool.is_contiguous(), what,
                ": pool must be a contiguous uint8 CUDA tensor [layers, pages, ..]");
    TORCH_CHECK(src.size() == dst.size(), what, ": ", src.size(), " pages to copy, ", dst.size(), " places");
    if (src.empty()) return;
    TORCH_CHECK(pool.numel() > 0, what, ": pool has no pages");
    std::vector<int32_t> pages;
    pages.reserve(2 * src.size());
    for (int64_t p : src) pages.push_back(whole(what, p));
    for (int64_t p : dst) pages.push_back(whole(what, p));
    c10::cuda::CUDAGuard guard(pool.device());
    check_status(sal_copy_kv4_pages(pool.data_ptr(), pages.data(), pages.data() + src.size(), whole(what, (int64_t)src.size()), whole(what, pool.size(0)),
                                    whole(what, pool.size(1)), (size_t)(pool.numel() / (pool.size(0) * pool.size(1))), stream_of(pool.device())),
                 "sal_copy_kv4_pages (no page twice, none both read and written)");
}

// A filter's setting: a tensor of one number per row, or one number for all.
struct Setting {
    const void *ptr = nullptr;
    double all = 0;
    Setting(const char *name, const py::object &v, c10::ScalarType dtype, int64_t rows, c10::Device device) {
        if (THPVariable_Check(v.ptr())) {
            const Tensor &t = THPVariable_Unpack(v.ptr());
            want("sample_token", name, t, dtype, rows, rows, device);
            ptr = t.data_ptr();
        } else {
            all = v.cast<double>();
            TORCH_CHECK(dtype != torch::kInt32 || std::fabs(all) <= 0x7fffffff, "sample_token: ", name, " must be a 32-bit number, got ", all);
        }
    }
};

void sample_token(const Tensor &logits, const Tensor &u, const Tensor &token, const py::object &temperature, const py::object &top_k, const py::object &top_p,
                  const py::object &min_p) {
    const char *what = "sample_token";
    const auto dtype = logits.scalar_type();
    TORCH_CHECK(logits.is_cuda() && (dtype == torch::kFloat16 || dtype == torch::kFloat32) && logits.is_contiguous() && logits.numel() > 0 && logits.dim() > 0, what,
                ": logits must be a contiguous float16 or float32 CUDA tensor [rows, vocab]");
    const auto device = logits.device();
    const int64_t vocab = logits.size(-1), rows = logits.numel() / vocab;
    want(what, "u", u, torch::kFloat32, rows, rows, device);
    want(what, "token", token, torch::kInt64, rows, rows, device);
    const Setting t("temperature", temperature, torch::kFloat32, rows, device), k("top_k", top_k, torch::kInt32, rows, device),
        p("top_p", top_p, torch::kFloat32, rows, device), least("min_p", min_p, torch::kFloat32, rows, device);
    py::gil_scoped_release release;
    c10::cuda::CUDAGuard guard(device);
    check_status(sal_sample_token(logits.data_ptr(), dtype == torch::kFloat32, whole(what, rows), whole(what, vocab), u.data_ptr(), t.ptr,
                                  static_cast<const int32_t *>(k.ptr), p.ptr, least.ptr, (float)t.all, (int)k.all, (float)p.all, (float)least.all,
                                  token.data_ptr<int64_t>(), stream_of(device)),
                 "sal_sample_token");
}

}  // namespace

void register_decode_ops(py::module_ &m) {
    using release = py::call_guard<py::gil_scoped_release>;
    m.def("rope_kv4_write", &rope_kv4_write, "rotary step of new rows, and their keys and values into a 4-bit cache", release());
    m.def("read_kv4", &read_kv4, "values of a 4-bit cache", release());
    m.def("attention_kv4", &attention_kv4, "attention over a 4-bit cache", release());
    m.def("copy_kv4_pages", &copy_kv4_pages, "copies pages of a 4-bit cache in all layers", release());
    m.def("sample_token", &sample_token, "the next token of each row of logits");
}
