// PyTorch C++ extension over the tb200 C ABI.  It owns no kernels: each function checks the
// tensors (device, dtype, contiguity), unwraps data_ptr() and the current CUDA stream, and calls
// the matching extern "C" entry point of libtb200.so.  A nonzero return code becomes a Python
// exception carrying tb200_last_error(), which the benchmark engine records as `cuda_err`.
// Nothing here synchronises or allocates, so every call may run under CUDA-graph capture;
// outputs and workspaces are allocated by the Python caller with torch.empty.  The layer operators, which have up to
// five outputs and run on small inputs too, also have forms (*_new) that make the outputs here, from the same allocator:
// a torch.empty from Python costs 2.4 us of host time, more than the smallest kernels take.
#include <torch/extension.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <stdexcept>
#include <string>

#include "tb200.h"

namespace {

void check_rc(int rc, const char* what) {
    if (rc == TB200_OK) return;
    std::string msg = std::string(what) + " failed (code " + std::to_string(rc) + "): " + tb200_last_error();
    if (rc == TB200_ERR_UNSUPPORTED) throw py::type_error(msg);
    if (rc == TB200_ERR_ARG || rc == TB200_ERR_ALIGN || rc == TB200_ERR_WORKSPACE) throw py::value_error(msg);
    throw std::runtime_error(msg);
}

void check_cuda(const torch::Tensor& t, const char* name, c10::ScalarType dt) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
    TORCH_CHECK(t.scalar_type() == dt, name, " has dtype ", t.scalar_type(), ", expected ", dt);
}

void* stream_of(const torch::Tensor& t) {
    return static_cast<void*>(c10::cuda::getCurrentCUDAStream(t.get_device()).stream());
}

int dt_code(c10::ScalarType t) {
    switch (t) {
        case torch::kFloat32: return TB200_DT_F32;
        case torch::kFloat16: return TB200_DT_F16;
        case torch::kBFloat16: return TB200_DT_BF16;
        default: throw py::type_error("tb200: unsupported dtype");
    }
}

void dequant_int4_group(const torch::Tensor& wp, const torch::Tensor& scales, torch::Tensor& out, int64_t group,
                        int64_t zero_point) {
    check_cuda(wp, "wp", torch::kUInt8);
    check_cuda(scales, "scales", torch::kFloat16);
    check_cuda(out, "out", torch::kFloat16);
    TORCH_CHECK(wp.dim() == 2 && scales.dim() == 2 && out.dim() == 2, "dequant_int4_group: 2-D tensors expected");
    const int64_t n = wp.size(0), k = wp.size(1) * 2;
    TORCH_CHECK(out.size(0) == n && out.size(1) == k, "out must be [n, k]");
    TORCH_CHECK(group > 0 && scales.size(0) == n && scales.size(1) * group == k, "scales must be [n, k/group]");
    c10::cuda::CUDAGuard guard(wp.device());
    check_rc(tb200_dequant_int4_group(wp.data_ptr(), scales.data_ptr(), out.data_ptr(), n, k, group,
                                      static_cast<int>(zero_point), out.stride(0), stream_of(wp)),
             "tb200_dequant_int4_group");
}

void dequant_int8_rowwise(const torch::Tensor& w, const torch::Tensor& scale, torch::Tensor& out, bool use_post,
                          double post) {
    check_cuda(w, "w", torch::kInt8);
    check_cuda(scale, "scale", torch::kFloat32);
    TORCH_CHECK(out.is_cuda() && out.is_contiguous(), "out must be a contiguous CUDA tensor");
    TORCH_CHECK(w.dim() == 2 && scale.dim() == 1 && scale.size(0) == w.size(0), "w [rows, cols], scale [rows]");
    TORCH_CHECK(out.sizes() == w.sizes(), "out must match w's shape");
    const int dt = dt_code(out.scalar_type());
    c10::cuda::CUDAGuard guard(w.device());
    check_rc(tb200_dequant_int8_rowwise(w.data_ptr(), scale.data_ptr<float>(), out.data_ptr(), w.size(0), w.size(1), dt,
                                        use_post ? 1 : 0, static_cast<float>(post), stream_of(w)),
             "tb200_dequant_int8_rowwise");
}

void weight_dequant_block(const torch::Tensor& x, const torch::Tensor& s, torch::Tensor& y, int64_t m, int64_t n,
                          int64_t tile) {
    TORCH_CHECK(x.is_cuda() && s.is_cuda() && y.is_cuda(), "CUDA tensors expected");
    TORCH_CHECK(x.is_contiguous() && s.is_contiguous() && y.is_contiguous(), "contiguous tensors expected");
    TORCH_CHECK(x.scalar_type() == s.scalar_type() && x.scalar_type() == y.scalar_type(), "x, s, y must share a dtype");
    TORCH_CHECK(x.numel() == m * n && y.numel() == m * n, "x and y must hold m*n elements");
    TORCH_CHECK(tile > 0 && s.numel() == ((m + tile - 1) / tile) * ((n + tile - 1) / tile), "s must be [ceil(m/T), ceil(n/T)]");
    const int dt = dt_code(x.scalar_type());
    c10::cuda::CUDAGuard guard(x.device());
    check_rc(tb200_weight_dequant_block(x.data_ptr(), s.data_ptr(), y.data_ptr(), m, n, tile, dt, stream_of(x)),
             "tb200_weight_dequant_block");
}

void gemm_fp8_blockscaled(const torch::Tensor& a, const torch::Tensor& sa, const torch::Tensor& b,
                          const torch::Tensor& sb, torch::Tensor& out) {
    check_cuda(a, "a", torch::kFloat8_e4m3fn);
    check_cuda(b, "b", torch::kFloat8_e4m3fn);
    check_cuda(sa, "sa", torch::kFloat32);
    check_cuda(sb, "sb", torch::kFloat32);
    check_cuda(out, "out", torch::kBFloat16);
    TORCH_CHECK(a.dim() == 2 && b.dim() == 2 && a.size(1) == b.size(1), "a [m,k], b [n,k]");
    const int64_t m = a.size(0), n = b.size(0), k = a.size(1);
    TORCH_CHECK(k % 128 == 0 && n % 128 == 0, "k and n must be multiples of 128");
    TORCH_CHECK(sa.dim() == 2 && sa.size(0) == m && sa.size(1) == k / 128, "sa must be [m, k/128]");
    TORCH_CHECK(sb.dim() == 2 && sb.size(0) == n / 128 && sb.size(1) == k / 128, "sb must be [n/128, k/128]");
    TORCH_CHECK(out.dim() == 2 && out.size(0) == m && out.size(1) == n, "out must be [m, n]");
    c10::cuda::CUDAGuard guard(a.device());
    check_rc(tb200_gemm_fp8_blockscaled(a.data_ptr(), sa.data_ptr<float>(), b.data_ptr(), sb.data_ptr<float>(),
                                        out.data_ptr(), m, n, k, out.stride(0), stream_of(a)),
             "tb200_gemm_fp8_blockscaled");
}

int64_t gemm_w4a16_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    return static_cast<int64_t>(tb200_gemm_w4a16_workspace_bytes(m, n, k));
}

// out is the full [m, ldo] result; this call fills columns [col_offset, col_offset + n).
void gemm_w4a16(const torch::Tensor& a, const torch::Tensor& wp, const torch::Tensor& scales, torch::Tensor& out,
                int64_t group, int64_t zero_point, int64_t col_offset, const c10::optional<torch::Tensor>& workspace) {
    check_cuda(a, "a", torch::kFloat16);
    check_cuda(wp, "wp", torch::kUInt8);
    check_cuda(scales, "scales", torch::kFloat16);
    TORCH_CHECK(out.is_cuda() && out.scalar_type() == torch::kFloat16 && out.dim() == 2 && out.stride(1) == 1,
                "out must be a CUDA fp16 matrix with unit column stride");
    TORCH_CHECK(a.dim() == 2 && wp.dim() == 2 && a.size(1) == wp.size(1) * 2, "a [m,k], wp [n,k/2]");
    const int64_t m = a.size(0), k = a.size(1), n = wp.size(0);
    TORCH_CHECK(group > 0 && scales.dim() == 2 && scales.size(0) == n && scales.size(1) * group == k, "scales must be [n, k/group]");
    TORCH_CHECK(out.size(0) == m && col_offset >= 0 && out.size(1) >= col_offset + n, "out must be [m, >= col_offset + n]");
    void* ws = nullptr;
    size_t ws_bytes = 0;
    if (workspace.has_value() && workspace->defined() && workspace->numel() > 0) {
        TORCH_CHECK(workspace->is_cuda() && workspace->is_contiguous(), "workspace must be a contiguous CUDA tensor");
        ws = workspace->data_ptr();
        ws_bytes = static_cast<size_t>(workspace->numel()) * workspace->element_size();
    }
    c10::cuda::CUDAGuard guard(a.device());
    check_rc(tb200_gemm_w4a16(a.data_ptr(), wp.data_ptr(), scales.data_ptr(), out.data_ptr(), m, n, k, group,
                              static_cast<int>(zero_point), out.stride(0), col_offset, ws, ws_bytes, stream_of(a)),
             "tb200_gemm_w4a16");
}

// Fused GEMM + all-gather: out_ptrs[r] is the address of rank r's full [m, ldo] fp16 output (peer-mapped).
void gemm_w4a16_gather(const torch::Tensor& a, const torch::Tensor& wp, const torch::Tensor& scales,
                       const std::vector<int64_t>& out_ptrs, int64_t rank, int64_t ldo, int64_t group,
                       int64_t zero_point) {
    check_cuda(a, "a", torch::kFloat16);
    check_cuda(wp, "wp", torch::kUInt8);
    check_cuda(scales, "scales", torch::kFloat16);
    TORCH_CHECK(a.dim() == 2 && wp.dim() == 2 && a.size(1) == wp.size(1) * 2, "a [m,k], wp [n_local,k/2]");
    const int64_t m = a.size(0), k = a.size(1), n_local = wp.size(0);
    TORCH_CHECK(group > 0 && scales.dim() == 2 && scales.size(0) == n_local && scales.size(1) * group == k, "scales must be [n_local, k/group]");
    std::vector<void*> ptrs;
    for (int64_t p : out_ptrs) ptrs.push_back(reinterpret_cast<void*>(static_cast<uintptr_t>(p)));
    c10::cuda::CUDAGuard guard(a.device());
    check_rc(tb200_gemm_w4a16_gather(a.data_ptr(), wp.data_ptr(), scales.data_ptr(), ptrs.data(), static_cast<int>(ptrs.size()),
                                     static_cast<int>(rank), m, n_local, k, group, static_cast<int>(zero_point), ldo, stream_of(a)),
             "tb200_gemm_w4a16_gather");
}

// Pushes `local` [m, n_local] into columns [rank * n_local, ...) of every rank's full [m, ldo] buffer.
void allgather_cols(const torch::Tensor& local, const std::vector<int64_t>& out_ptrs, int64_t rank, int64_t ldo) {
    TORCH_CHECK(local.is_cuda() && local.dim() == 2 && local.stride(1) == 1, "local must be a CUDA matrix with unit column stride");
    std::vector<void*> ptrs;
    for (int64_t p : out_ptrs) ptrs.push_back(reinterpret_cast<void*>(static_cast<uintptr_t>(p)));
    c10::cuda::CUDAGuard guard(local.device());
    check_rc(tb200_allgather_cols(local.data_ptr(), local.stride(0), ptrs.data(), static_cast<int>(ptrs.size()), static_cast<int>(rank),
                                  local.size(0), local.size(1), local.element_size(), ldo, stream_of(local)),
             "tb200_allgather_cols");
}

void selftest_bounded_wait(int64_t limit_cycles) {
    check_rc(tb200_selftest_bounded_wait(limit_cycles, at::cuda::getCurrentCUDAStream().stream()), "tb200_selftest_bounded_wait");
}

void quantize_fp8_block(const torch::Tensor& x, torch::Tensor& q, torch::Tensor& scales, int64_t block_rows) {
    check_cuda(x, "x", torch::kFloat32);
    check_cuda(q, "q", torch::kFloat8_e4m3fn);
    check_cuda(scales, "scales", torch::kFloat32);
    TORCH_CHECK(x.dim() == 2 && q.sizes() == x.sizes(), "x and q must be [rows, cols]");
    TORCH_CHECK(block_rows > 0 && scales.numel() == (x.size(0) / block_rows) * (x.size(1) / 128), "scales must be [rows/block_rows, cols/128]");
    c10::cuda::CUDAGuard guard(x.device());
    check_rc(tb200_quantize_fp8_block(x.data_ptr<float>(), q.data_ptr(), scales.data_ptr<float>(), x.size(0), x.size(1),
                                      static_cast<int>(block_rows), stream_of(x)),
             "tb200_quantize_fp8_block");
}

void matmul_int8_packed2(const torch::Tensor& a, const torch::Tensor& b, torch::Tensor& out) {
    check_cuda(a, "a", torch::kInt8);
    check_cuda(b, "b", torch::kUInt8);
    check_cuda(out, "out", torch::kInt32);
    TORCH_CHECK(a.dim() == 2 && b.dim() == 2 && a.size(1) == 4 * b.size(0), "a [m,k], b [k/4,n]");
    TORCH_CHECK(out.dim() == 2 && out.size(0) == a.size(0) && out.size(1) == b.size(1) && out.stride(1) == 1, "out must be [m,n]");
    c10::cuda::CUDAGuard guard(a.device());
    check_rc(tb200_matmul_int8_packed2(a.data_ptr(), b.data_ptr(), out.data_ptr(), a.size(0), b.size(1), a.size(1),
                                       out.stride(0), stream_of(a)),
             "tb200_matmul_int8_packed2");
}

void matmul_plain(const torch::Tensor& a, const torch::Tensor& b, torch::Tensor& out) {
    TORCH_CHECK(a.is_cuda() && b.is_cuda() && out.is_cuda(), "matmul_plain: tensors must be on a CUDA device");
    TORCH_CHECK(a.is_contiguous() && b.is_contiguous(), "matmul_plain: a and b must be contiguous");
    TORCH_CHECK(a.scalar_type() == b.scalar_type() && a.scalar_type() == out.scalar_type(), "matmul_plain: a, b, out must share a dtype");
    int dt = -1;
    if (a.scalar_type() == torch::kFloat32) dt = TB200_DT_F32;
    else if (a.scalar_type() == torch::kFloat16) dt = TB200_DT_F16;
    else if (a.scalar_type() == torch::kBFloat16) dt = TB200_DT_BF16;
    else if (a.scalar_type() == torch::kFloat8_e4m3fn) dt = TB200_DT_F8E4M3;
    if (dt < 0) throw py::type_error("matmul_plain: dtype must be float32, float16, bfloat16 or float8_e4m3fn");
    TORCH_CHECK(a.dim() == 2 && b.dim() == 2 && a.size(1) == b.size(0), "a [m,k], b [k,n]");
    TORCH_CHECK(out.dim() == 2 && out.size(0) == a.size(0) && out.size(1) == b.size(1) && out.stride(1) == 1, "out must be [m,n]");
    c10::cuda::CUDAGuard guard(a.device());
    check_rc(tb200_matmul_plain(a.data_ptr(), b.data_ptr(), out.data_ptr(), a.size(0), b.size(1), a.size(1), dt,
                                out.stride(0), stream_of(a)),
             "tb200_matmul_plain");
}

void quantize_int4_group(const torch::Tensor& x, torch::Tensor& wp, torch::Tensor& scales, int64_t group, int64_t zero_point) {
    check_cuda(x, "x", torch::kFloat32);
    check_cuda(wp, "wp", torch::kUInt8);
    check_cuda(scales, "scales", torch::kFloat16);
    TORCH_CHECK(x.dim() == 2 && wp.dim() == 2 && wp.size(0) == x.size(0) && wp.size(1) * 2 == x.size(1), "x [n,k], wp [n,k/2]");
    TORCH_CHECK(group > 0 && scales.dim() == 2 && scales.size(0) == x.size(0) && scales.size(1) * group == x.size(1), "scales must be [n, k/group]");
    c10::cuda::CUDAGuard guard(x.device());
    check_rc(tb200_quantize_int4_group(x.data_ptr<float>(), wp.data_ptr(), scales.data_ptr(), x.size(0), x.size(1), group,
                                       static_cast<int>(zero_point), stream_of(x)),
             "tb200_quantize_int4_group");
}

// ---- gated feed-forward block with 8-bit activation checkpoints ----
void check_same_device(const torch::Tensor& t, const char* name, const torch::Tensor& first) {
    TORCH_CHECK(t.is_cuda() && t.device() == first.device(), name, " must be on ", first.device().str(), ", is on ", t.device().str());
}
// codes [rows, cols] and scales [rows, ceil(cols / 128)] of one activation
void check_codes(const torch::Tensor& q, const torch::Tensor& s, const char* name, int64_t rows, int64_t cols, const torch::Tensor& first) {
    check_cuda(q, name, torch::kFloat8_e4m3fn);
    check_cuda(s, "scales", torch::kFloat32);
    check_same_device(q, name, first);
    check_same_device(s, "scales", first);
    // numbers go through to_string: this object and libstdc++ each hold the stream's number formatting, and mixing them crashes
    TORCH_CHECK(q.dim() == 2 && q.size(0) == rows && q.size(1) == cols, name, " must be [", std::to_string(rows), ", ", std::to_string(cols), "]");
    TORCH_CHECK(s.dim() == 2 && s.size(0) == rows && s.size(1) == (cols + 127) / 128, "the scales of ", name, " must be [", std::to_string(rows),
                ", ", std::to_string((cols + 127) / 128), "]");
}
void check_rows(const torch::Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda() && t.dim() == 2, name, " must be a CUDA matrix");
    TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, name, " must have unit column stride");
}

void act_checkpoint_fp8(const torch::Tensor& x, torch::Tensor& q, torch::Tensor& scales) {
    check_rows(x, "x");
    check_codes(q, scales, "q", x.size(0), x.size(1), x);
    c10::cuda::CUDAGuard guard(x.device());
    check_rc(tb200_act_checkpoint_fp8(x.data_ptr(), q.data_ptr(), scales.data_ptr<float>(), x.size(0), x.size(1), x.stride(0),
                                      dt_code(x.scalar_type()), stream_of(x)),
             "tb200_act_checkpoint_fp8");
}

void act_restore_fp8(const torch::Tensor& q, const torch::Tensor& scales, torch::Tensor& out) {
    TORCH_CHECK(q.is_cuda() && q.dim() == 2, "q must be a CUDA matrix");
    check_codes(q, scales, "q", q.size(0), q.size(1), q);
    check_same_device(out, "out", q);
    TORCH_CHECK(out.is_contiguous() && out.sizes() == q.sizes(), "out must be contiguous and match q's shape");
    c10::cuda::CUDAGuard guard(q.device());
    check_rc(tb200_act_restore_fp8(q.data_ptr(), scales.data_ptr<float>(), out.data_ptr(), q.size(0), q.size(1), dt_code(out.scalar_type()),
                                   stream_of(q)),
             "tb200_act_restore_fp8");
}

// x [m, k], wg and wu [f, k]; returns the dtype code
int check_block(const torch::Tensor& first, const torch::Tensor& wg, const torch::Tensor& wu) {
    const auto dt = wg.scalar_type();
    check_cuda(wg, "wg", dt);
    check_cuda(wu, "wu", dt);
    check_same_device(wg, "wg", first);
    check_same_device(wu, "wu", first);
    TORCH_CHECK(wg.dim() == 2 && wu.sizes() == wg.sizes(), "wg and wu must be [f, k]");
    return dt_code(dt);
}

void ffn_gated(const torch::Tensor& x, const torch::Tensor& wg, const torch::Tensor& wu, torch::Tensor& h, int64_t act,
               const c10::optional<torch::Tensor>& gq, const c10::optional<torch::Tensor>& gs, const c10::optional<torch::Tensor>& uq,
               const c10::optional<torch::Tensor>& us) {
    check_rows(x, "x");
    const int dt = check_block(x, wg, wu);
    TORCH_CHECK(x.scalar_type() == wg.scalar_type(), "x has dtype ", x.scalar_type(), ", expected the weights' ", wg.scalar_type());
    const int64_t m = x.size(0), k = x.size(1), f = wg.size(0);
    TORCH_CHECK(wg.size(1) == k, "x [m,k], wg [f,k]");
    check_cuda(h, "h", wg.scalar_type());
    check_same_device(h, "h", x);
    TORCH_CHECK(h.dim() == 2 && h.size(0) == m && h.size(1) == f, "h must be [m, f]");
    const int given = gq.has_value() + gs.has_value() + uq.has_value() + us.has_value();
    TORCH_CHECK(given == 0 || given == 4, "gq, gs, uq, us are given together or not at all");
    if (given) {
        check_codes(*gq, *gs, "gq", m, f, x);
        check_codes(*uq, *us, "uq", m, f, x);
    }
    c10::cuda::CUDAGuard guard(x.device());
    check_rc(tb200_ffn_gated(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), h.data_ptr(), given ? gq->data_ptr() : nullptr,
                             given ? gs->data_ptr<float>() : nullptr, given ? uq->data_ptr() : nullptr, given ? us->data_ptr<float>() : nullptr,
                             m, f, k, x.stride(0), static_cast<int>(act), dt, stream_of(x)),
             "tb200_ffn_gated");
}

int64_t ffn_gated_bwd_workspace_bytes(int64_t m, int64_t f, int64_t k, bool x_codes) {
    return static_cast<int64_t>(tb200_ffn_gated_bwd_workspace_bytes(m, f, k, x_codes ? 1 : 0));
}

void ffn_gated_bwd(const torch::Tensor& dh, const torch::Tensor& wg, const torch::Tensor& wu, const torch::Tensor& x,
                   const c10::optional<torch::Tensor>& xs, const torch::Tensor& gq, const torch::Tensor& gs, const torch::Tensor& uq,
                   const torch::Tensor& us, torch::Tensor& dx, torch::Tensor& dwg, torch::Tensor& dwu, int64_t act, torch::Tensor& workspace) {
    TORCH_CHECK(dh.is_cuda() && dh.dim() == 2, "dh must be a CUDA matrix");
    const int dt = check_block(dh, wg, wu);
    const int64_t m = dh.size(0), f = wg.size(0), k = wg.size(1);
    check_cuda(dh, "dh", wg.scalar_type());
    TORCH_CHECK(dh.size(1) == f, "dh [m,f], wg [f,k]");
    check_codes(gq, gs, "gq", m, f, dh);
    check_codes(uq, us, "uq", m, f, dh);
    if (xs.has_value()) {
        check_codes(x, *xs, "x", m, k, dh);
    } else {
        check_rows(x, "x");
        check_same_device(x, "x", dh);
        TORCH_CHECK(x.scalar_type() == wg.scalar_type(), "x has dtype ", x.scalar_type(), ", expected the weights' ", wg.scalar_type(), ", or e4m3 codes with scales");
        TORCH_CHECK(x.size(0) == m && x.size(1) == k, "x must be [m, k]");
    }
    for (const torch::Tensor* t : {&dx, &dwg, &dwu, &workspace}) check_same_device(*t, "outputs and workspace", dh);
    check_cuda(dx, "dx", wg.scalar_type());
    check_cuda(dwg, "dwg", wg.scalar_type());
    check_cuda(dwu, "dwu", wg.scalar_type());
    TORCH_CHECK(dx.dim() == 2 && dx.size(0) == m && dx.size(1) == k, "dx must be [m, k]");
    TORCH_CHECK(dwg.sizes() == wg.sizes() && dwu.sizes() == wg.sizes(), "dwg and dwu must be [f, k]");
    TORCH_CHECK(workspace.is_contiguous(), "workspace must be contiguous");
    c10::cuda::CUDAGuard guard(dh.device());
    check_rc(tb200_ffn_gated_bwd(dh.data_ptr(), wg.data_ptr(), wu.data_ptr(), x.data_ptr(), xs.has_value() ? xs->data_ptr<float>() : nullptr,
                                 gq.data_ptr(), gs.data_ptr<float>(), uq.data_ptr(), us.data_ptr<float>(), dx.data_ptr(), dwg.data_ptr(),
                                 dwu.data_ptr(), m, f, k, x.stride(0), static_cast<int>(act), dt, workspace.data_ptr(),
                                 static_cast<size_t>(workspace.numel()) * workspace.element_size(), stream_of(dh)),
             "tb200_ffn_gated_bwd");
}

// The forms that make their outputs: x may be anything, the functions above check it.
torch::Tensor empty_on(const torch::Tensor& like, at::IntArrayRef sizes, c10::ScalarType dt) {
    return at::empty(sizes, at::TensorOptions().dtype(dt).device(like.device()));
}
int64_t blocks_of(int64_t cols) { return (cols + 127) / 128; }

std::tuple<torch::Tensor, torch::Tensor> act_checkpoint_fp8_new(const torch::Tensor& x) {
    check_rows(x, "x");
    torch::Tensor q = empty_on(x, x.sizes(), torch::kFloat8_e4m3fn), s = empty_on(x, {x.size(0), blocks_of(x.size(1))}, torch::kFloat32);
    act_checkpoint_fp8(x, q, s);
    return {q, s};
}

torch::Tensor act_restore_fp8_new(const torch::Tensor& q, const torch::Tensor& scales, c10::ScalarType dtype) {
    torch::Tensor out = empty_on(q, q.sizes(), dtype);
    act_restore_fp8(q, scales, out);
    return out;
}

torch::Tensor ffn_gated_new(const torch::Tensor& x, const torch::Tensor& wg, const torch::Tensor& wu, int64_t act) {
    check_rows(x, "x");
    TORCH_CHECK(wg.dim() == 2, "wg must be [f, k]");
    torch::Tensor h = empty_on(x, {x.size(0), wg.size(0)}, x.scalar_type());
    ffn_gated(x, wg, wu, h, act, c10::nullopt, c10::nullopt, c10::nullopt, c10::nullopt);
    return h;
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> ffn_gated_checkpoint_new(
    const torch::Tensor& x, const torch::Tensor& wg, const torch::Tensor& wu, int64_t act) {
    check_rows(x, "x");
    TORCH_CHECK(wg.dim() == 2, "wg must be [f, k]");
    const int64_t m = x.size(0), f = wg.size(0);
    torch::Tensor h = empty_on(x, {m, f}, x.scalar_type());
    torch::Tensor gq = empty_on(x, {m, f}, torch::kFloat8_e4m3fn), gs = empty_on(x, {m, blocks_of(f)}, torch::kFloat32);
    torch::Tensor uq = empty_on(x, {m, f}, torch::kFloat8_e4m3fn), us = empty_on(x, {m, blocks_of(f)}, torch::kFloat32);
    ffn_gated(x, wg, wu, h, act, gq, gs, uq, us);
    return {h, gq, gs, uq, us};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> ffn_gated_bwd_new(
    const torch::Tensor& dh, const torch::Tensor& wg, const torch::Tensor& wu, const torch::Tensor& x, const c10::optional<torch::Tensor>& xs,
    const torch::Tensor& gq, const torch::Tensor& gs, const torch::Tensor& uq, const torch::Tensor& us, int64_t act) {
    TORCH_CHECK(dh.is_cuda() && dh.dim() == 2 && wg.dim() == 2, "dh [m,f], wg [f,k] must be CUDA matrices");
    const int64_t m = dh.size(0), f = wg.size(0), k = wg.size(1);
    c10::cuda::CUDAGuard guard(dh.device());                    // the workspace depends on the device's SMs
    torch::Tensor dx = empty_on(dh, {m, k}, wg.scalar_type()), dwg = empty_on(dh, {f, k}, wg.scalar_type()), dwu = empty_on(dh, {f, k}, wg.scalar_type());
    torch::Tensor ws = empty_on(dh, {ffn_gated_bwd_workspace_bytes(m, f, k, xs.has_value())}, torch::kUInt8);
    ffn_gated_bwd(dh, wg, wu, x, xs, gq, gs, uq, us, dx, dwg, dwu, act, ws);
    return {dx, dwg, dwu};
}

py::tuple device_status() {
    int code = 0, detail = 0;
    check_rc(tb200_device_status(&code, &detail), "tb200_device_status");
    return py::make_tuple(code, detail);
}

void clear_device_status() { check_rc(tb200_clear_device_status(), "tb200_clear_device_status"); }
void check_device() { check_rc(tb200_check_device(), "tb200_check_device"); }

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "PyTorch binding of the tb200 C ABI (B200 quantized-inference kernels)";
    m.def("abi_version", &tb200_abi_version);
    m.def("check_device", &check_device);
    m.def("dequant_int4_group", &dequant_int4_group);
    m.def("dequant_int8_rowwise", &dequant_int8_rowwise);
    m.def("weight_dequant_block", &weight_dequant_block);
    m.def("gemm_fp8_blockscaled", &gemm_fp8_blockscaled);
    m.def("gemm_w4a16_workspace_bytes", &gemm_w4a16_workspace_bytes);
    m.def("gemm_w4a16", &gemm_w4a16);
    m.def("gemm_w4a16_gather", &gemm_w4a16_gather);
    m.def("allgather_cols", &allgather_cols);
    m.def("selftest_bounded_wait", &selftest_bounded_wait);
    m.def("quantize_fp8_block", &quantize_fp8_block);
    m.def("matmul_int8_packed2", &matmul_int8_packed2);
    m.def("matmul_plain", &matmul_plain);
    m.def("quantize_int4_group", &quantize_int4_group);
    m.def("act_checkpoint_fp8", &act_checkpoint_fp8);
    m.def("act_restore_fp8", &act_restore_fp8);
    m.def("ffn_gated", &ffn_gated);
    m.def("ffn_gated_bwd_workspace_bytes", &ffn_gated_bwd_workspace_bytes);
    m.def("ffn_gated_bwd", &ffn_gated_bwd);
    m.def("act_checkpoint_fp8_new", &act_checkpoint_fp8_new);
    m.def("act_restore_fp8_new", &act_restore_fp8_new);
    m.def("ffn_gated_new", &ffn_gated_new);
    m.def("ffn_gated_checkpoint_new", &ffn_gated_checkpoint_new);
    m.def("ffn_gated_bwd_new", &ffn_gated_bwd_new);
    m.def("device_status", &device_status);
    m.def("clear_device_status", &clear_device_status);
}
