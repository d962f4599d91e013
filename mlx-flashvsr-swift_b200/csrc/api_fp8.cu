// api_fp8.cu — the C ABI of the 8-bit tensors, the linear layers on them and LayerNorm's training passes
// (include/fvsr_lcsa.h): host-side validation and workspace layout.
#include <stdarg.h>
#include <stdio.h>

#include "../../include/fvsr_lcsa.h"
#include "common.cuh"
#include "fp8.cuh"

namespace fvsr {
void set_last_error(const char* msg);
int current_device_is_sm100(int* dev);
}

using namespace fvsr;

namespace {

fvsr_status refuse(fvsr_status s, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    set_last_error(buf);
    return s;
}

fvsr_status launched(cudaError_t e, const char* what) {
    return e == cudaSuccess ? FVSR_OK : refuse(FVSR_ECUDA, "%s: %s", what, cudaGetErrorString(e));
}

fvsr_status check_device() {
    int dev = 0;
    if (current_device_is_sm100(&dev)) return FVSR_OK;
    return refuse(FVSR_EUNSUPPORTED, "device %d is not sm_100, the kernels need sm_100a", dev);
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

constexpr int64_t kMaxSide = 1ll << 30, kMaxElements = 1ll << 40;
constexpr int kMaxLinearSide = 1 << 22;

fvsr_status check_held_shape(int64_t rows, int64_t cols) {
    if (rows < 0 || cols < 1) return refuse(FVSR_EINVAL, "rows must be >= 0 and cols >= 1, got %lld x %lld", (long long)rows, (long long)cols);
    if (rows > kMaxSide || cols > kMaxSide || rows * cols > kMaxElements)
        return refuse(FVSR_EUNSUPPORTED, "a tensor of %lld x %lld is too large", (long long)rows, (long long)cols);
    return FVSR_OK;
}

fvsr_status check_dtype(int32_t dtype) {
    return dtype == FVSR_F32 || dtype == FVSR_BF16 ? FVSR_OK : refuse(FVSR_EINVAL, "dtype must be FVSR_F32 or FVSR_BF16, got %d", dtype);
}

fvsr_status check_linear_shape(int32_t m, int32_t n, int32_t k) {
    if (m < 0 || n < 1 || k < 1) return refuse(FVSR_EINVAL, "linear shape (%d, %d, %d): m must be >= 0, n and k >= 1", m, n, k);
    const int64_t lk = fp8_ld(k);
    if (m > kMaxLinearSide || n > kMaxLinearSide || k > kMaxLinearSide || m * lk * 2 > kMaxElements ||
        n * lk > kMaxElements || (int64_t)m * n * 4 > kMaxElements)
        return refuse(FVSR_EUNSUPPORTED, "linear shape (%d, %d, %d) is too large", m, n, k);
    return FVSR_OK;
}

// The workspace of a linear layer: the 8-bit form of a bf16 x, then the partial products of a sum over K in parts.
struct LinearWorkspace {
    size_t scale, partial, bytes;
    Fp8GemmPlan plan;
};
LinearWorkspace linear_workspace(int m, int n, int k, bool x_is_fp8) {
    LinearWorkspace w;
    w.plan = plan_gemm_fp8(m, n, k);
    w.scale = x_is_fp8 ? 0 : up256((size_t)(m * fp8_ld(k)));
    w.partial = x_is_fp8 ? 0 : w.scale + up256((size_t)fp8_scale_bytes(m, k));
    w.bytes = w.partial + up256(w.plan.partial_bytes);
    return w;
}

fvsr_status check_norm(int64_t m, int32_t c, int32_t dtype) {
    if (m < 0 || c < 1) return refuse(FVSR_EINVAL, "layernorm: m must be >= 0 and c >= 1, got %lld and %d", (long long)m, c);
    if (c > kNormTrainMaxC) return refuse(FVSR_EUNSUPPORTED, "layernorm: c must be at most %d, got %d", kNormTrainMaxC, c);
    if (m > kMaxSide) return refuse(FVSR_EUNSUPPORTED, "layernorm: m = %lld is too large", (long long)m);
    return check_dtype(dtype);
}

}  // namespace

extern "C" {

fvsr_status fvsr_fp8_bytes(int64_t rows, int64_t cols, size_t* value_bytes, size_t* scale_bytes) {
    fvsr_status s = check_held_shape(rows, cols);
    if (s != FVSR_OK) return s;
    if (value_bytes) *value_bytes = (size_t)(rows * fp8_ld(cols));
    if (scale_bytes) *scale_bytes = (size_t)fp8_scale_bytes(rows, cols);
    return FVSR_OK;
}

fvsr_status fvsr_fp8_codes(int64_t rows, int64_t cols, const void* scale, void* out, fvsr_stream_t stream) {
    fvsr_status s = check_held_shape(rows, cols);
    if (s != FVSR_OK) return s;
    if (rows == 0) return FVSR_OK;
    if (!scale || !out) return refuse(FVSR_EINVAL, "scale and out are required");
    if (!aligned(scale, 16)) return refuse(FVSR_EINVAL, "scale must be 16-byte aligned");
    if ((s = check_device()) != FVSR_OK) return s;
    return launched(launch_fp8_codes(rows, cols, static_cast<const uint8_t*>(scale), static_cast<uint8_t*>(out),
                                     reinterpret_cast<cudaStream_t>(stream)), "codes launch");
}

fvsr_status fvsr_quantize_fp8(int64_t rows, int64_t cols, const void* x, int32_t dtype, int32_t square, void* q,
                              void* scale, void* qt, void* scale_t, fvsr_stream_t stream) {
    fvsr_status s = check_held_shape(rows, cols);
    if (s != FVSR_OK || (s = check_dtype(dtype)) != FVSR_OK) return s;
    if ((q == nullptr) != (scale == nullptr) || (qt == nullptr) != (scale_t == nullptr))
        return refuse(FVSR_EINVAL, "values and scales go together");
    if (rows == 0) return FVSR_OK;
    if (!x || (!q && !qt)) return refuse(FVSR_EINVAL, "x and q or qt are required");
    if (!aligned(x, 16) || !aligned(q, 16) || !aligned(scale, 16) || !aligned(qt, 16) || !aligned(scale_t, 16))
        return refuse(FVSR_EINVAL, "x, q, qt and the scales must be 16-byte aligned");
    if ((s = check_device()) != FVSR_OK) return s;
    return launched(launch_quantize_fp8(rows, cols, x, dtype, square != 0, static_cast<uint8_t*>(q),
                                        static_cast<uint8_t*>(scale), static_cast<uint8_t*>(qt),
                                        static_cast<uint8_t*>(scale_t), reinterpret_cast<cudaStream_t>(stream)),
                    "quantize launch");
}

fvsr_status fvsr_dequantize_fp8(int64_t rows, int64_t cols, const void* q, const void* scale, void* out, int32_t dtype,
                                fvsr_stream_t stream) {
    fvsr_status s = check_held_shape(rows, cols);
    if (s != FVSR_OK || (s = check_dtype(dtype)) != FVSR_OK) return s;
    if (rows == 0) return FVSR_OK;
    if (!q || !scale || !out) return refuse(FVSR_EINVAL, "q, scale and out are required");
    if (!aligned(q, 16) || !aligned(scale, 16) || !aligned(out, 4))
        return refuse(FVSR_EINVAL, "q and scale must be 16-byte aligned, out 4-byte aligned");
    if ((s = check_device()) != FVSR_OK) return s;
    return launched(launch_dequantize_fp8(rows, cols, static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(scale),
                                          out, dtype, reinterpret_cast<cudaStream_t>(stream)),
                    "dequantize launch");
}

fvsr_status fvsr_linear_fp8_workspace_size(int32_t m, int32_t n, int32_t k, int32_t x_is_fp8, size_t* bytes) {
    fvsr_status s = check_linear_shape(m, n, k);
    if (s != FVSR_OK) return s;
    if (!bytes) return refuse(FVSR_EINVAL, "bytes is NULL");
    *bytes = m <= kFewTokens ? 0 : linear_workspace(m, n, k, x_is_fp8 != 0).bytes;
    return FVSR_OK;
}

fvsr_status fvsr_linear_fp8(int32_t m, int32_t n, int32_t k, const void* x, const void* x_scale, const void* w,
                            const void* w_scale, const void* bias, int32_t epilogue, const void* gate,
                            const void* resid, void* out, int32_t out_dtype, void* workspace, size_t workspace_bytes,
                            fvsr_stream_t stream) {
    fvsr_status s = check_linear_shape(m, n, k);
    if (s != FVSR_OK || (s = check_dtype(out_dtype)) != FVSR_OK) return s;
    if (epilogue < FVSR_LINEAR || epilogue > FVSR_LINEAR_GATED_RESIDUAL)
        return refuse(FVSR_EINVAL, "unknown epilogue %d", epilogue);
    if (m == 0) return FVSR_OK;
    if (!x || !w || !w_scale || !out) return refuse(FVSR_EINVAL, "x, w, w_scale and out are required");
    if (epilogue == FVSR_LINEAR_GATED_RESIDUAL && (!gate || !resid))
        return refuse(FVSR_EINVAL, "the gated residual needs gate and resid");
    if (!aligned(x, 16) || !aligned(x_scale, 16) || !aligned(w, 16) || !aligned(w_scale, 16) || !aligned(out, 4) ||
        !aligned(resid, 4) || !aligned(bias, 2) || !aligned(gate, 2))
        return refuse(FVSR_EINVAL, "x, w and the scales must be 16-byte aligned, out and resid 4-byte, bias and gate 2-byte aligned");
    const bool few = m <= kFewTokens;
    const LinearWorkspace ws = few ? LinearWorkspace{} : linear_workspace(m, n, k, x_scale != nullptr);
    const size_t need = ws.bytes;
    if (need > 0 && !workspace) return refuse(FVSR_EINVAL, "the workspace is required");
    if (workspace_bytes < need)
        return refuse(FVSR_ENOMEM, "workspace of %zu bytes is smaller than the %zu required", workspace_bytes, need);
    if (!aligned(workspace, 16)) return refuse(FVSR_EINVAL, "workspace must be 16-byte aligned");
    if ((s = check_device()) != FVSR_OK) return s;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    Fp8GemmArgs a{};
    a.M = m, a.N = n, a.K = k;
    a.x = static_cast<const uint8_t*>(x);
    a.x_scale = static_cast<const uint8_t*>(x_scale);
    if (!x_scale && !few) {
        uint8_t* q = static_cast<uint8_t*>(workspace);
        uint8_t* scale = q + ws.scale;
        s = launched(launch_quantize_fp8(m, k, x, FVSR_BF16, false, q, scale, nullptr, nullptr, st), "quantize launch");
        if (s != FVSR_OK) return s;
        a.x = q, a.x_scale = scale;
    }
    a.w = static_cast<const uint8_t*>(w);
    a.w_scale = static_cast<const uint8_t*>(w_scale);
    a.bias = static_cast<const __nv_bfloat16*>(bias);
    a.gate = static_cast<const __nv_bfloat16*>(gate);
    a.resid = resid;
    a.out = out;
    a.mode = epilogue;
    a.out_dtype = out_dtype;
    if (few)
        return launched(launch_gemv_fp8(a, x_scale ? nullptr : static_cast<const __nv_bfloat16*>(x), st), "linear launch");
    return launched(launch_gemm_fp8(a, ws.plan, reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + ws.partial),
                                    st), "linear launch");
}

fvsr_status fvsr_layernorm_train(int64_t m, int32_t c, const void* x, int32_t dtype, const void* weight,
                                 const void* bias, const void* shift, const void* scale, float eps, void* out,
                                 float* mean, float* rstd, fvsr_stream_t stream) {
    fvsr_status s = check_norm(m, c, dtype);
    if (s != FVSR_OK) return s;
    if ((shift == nullptr) != (scale == nullptr)) return refuse(FVSR_EINVAL, "shift and scale go together");
    if ((bias == nullptr) != (weight == nullptr)) return refuse(FVSR_EINVAL, "weight and bias go together");
    if (!(eps >= 0.0f && eps < 1e30f)) return refuse(FVSR_EINVAL, "eps must be finite and >= 0");
    if (m == 0) return FVSR_OK;
    if (!x || !out || !mean || !rstd) return refuse(FVSR_EINVAL, "x, out, mean and rstd are required");
    const uintptr_t e = dtype == FVSR_BF16 ? 2 : 4;
    if (!aligned(x, e) || !aligned(out, e) || !aligned(weight, e) || !aligned(bias, e) || !aligned(shift, e) ||
        !aligned(scale, e) || !aligned(mean, 4) || !aligned(rstd, 4))
        return refuse(FVSR_EINVAL, "tensors must be aligned to their elements");
    if ((s = check_device()) != FVSR_OK) return s;
    NormTrainArgs a{};
    a.m = m, a.c = c, a.dtype = dtype;
    a.x = x, a.weight = weight, a.bias = bias, a.shift = shift, a.scale = scale;
    a.eps = eps, a.out = out, a.mean = mean, a.rstd = rstd;
    return launched(launch_layernorm_train(a, reinterpret_cast<cudaStream_t>(stream)), "layernorm launch");
}

fvsr_status fvsr_layernorm_backward_workspace_size(int64_t m, int32_t c, size_t* bytes) {
    fvsr_status s = check_norm(m, c, FVSR_F32);
    if (s != FVSR_OK) return s;
    if (!bytes) return refuse(FVSR_EINVAL, "bytes is NULL");
    *bytes = (size_t)norm_backward_ctas(m, c) * 2 * (size_t)c * sizeof(float);
    return FVSR_OK;
}

fvsr_status fvsr_layernorm_backward(int64_t m, int32_t c, const void* dy, int32_t dtype, const void* x,
                                    const void* x_scale, const float* mean, const float* rstd, const void* weight,
                                    const void* bias, const void* scale, void* dx, float* dweight, float* dbias,
                                    float* dscale, float* dshift, void* workspace, size_t workspace_bytes,
                                    fvsr_stream_t stream) {
    fvsr_status s = check_norm(m, c, dtype);
    if (s != FVSR_OK) return s;
    if ((bias == nullptr) != (weight == nullptr)) return refuse(FVSR_EINVAL, "weight and bias go together");
    if (m > 0 && (!dy || !x || !mean || !rstd || !dx)) return refuse(FVSR_EINVAL, "dy, x, mean, rstd and dx are required");
    const uintptr_t e = dtype == FVSR_BF16 ? 2 : 4;
    if (!aligned(dy, e) || !aligned(dx, e) || !aligned(weight, e) || !aligned(bias, e) || !aligned(scale, e) ||
        !aligned(mean, 4) || !aligned(rstd, 4) || !aligned(dweight, 4) || !aligned(dbias, 4) || !aligned(dscale, 4) ||
        !aligned(dshift, 4))
        return refuse(FVSR_EINVAL, "tensors must be aligned to their elements");
    if (!aligned(x, x_scale ? 16 : e) || !aligned(x_scale, 16))
        return refuse(FVSR_EINVAL, "an 8-bit x and its scales must be 16-byte aligned");
    size_t need = 0;
    if ((s = fvsr_layernorm_backward_workspace_size(m, c, &need)) != FVSR_OK) return s;
    if (need > 0 && !workspace) return refuse(FVSR_EINVAL, "the workspace is required");
    if (workspace_bytes < need)
        return refuse(FVSR_ENOMEM, "workspace of %zu bytes is smaller than the %zu required", workspace_bytes, need);
    if (!aligned(workspace, 16)) return refuse(FVSR_EINVAL, "workspace must be 16-byte aligned");
    if ((s = check_device()) != FVSR_OK) return s;
    NormTrainArgs a{};
    a.m = m, a.c = c, a.dtype = dtype;
    a.x = x, a.x_scale = static_cast<const uint8_t*>(x_scale);
    a.weight = weight, a.bias = bias, a.scale = scale;
    a.out = dx, a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd), a.dy = dy;
    a.dweight = dweight, a.dbias = dbias, a.dscale = dscale, a.dshift = dshift;
    a.partial = static_cast<float*>(workspace);
    return launched(launch_layernorm_backward(a, reinterpret_cast<cudaStream_t>(stream)), "layernorm backward launch");
}

}  // extern "C"
