// C entry points of the 8-bit floating point blocks (include/axq.h):
// argument checks and dispatch.  Nothing here allocates device memory.
#include <algorithm>
#include <cstdint>
#include <string>

#include "axq_f8.cuh"
#include "axq_internal.h"

namespace axq {
namespace {

constexpr size_t kStatusBytes = 256;  // status words at the front of a workspace

int fail(int code, const std::string& msg) {
    set_last_error(msg);
    return code;
}

int status(cudaError_t e, const char* fn) {
    if (e == cudaSuccess) return AXQ_OK;
    return fail(AXQ_ERR_CUDA, std::string(fn) + ": " + cudaGetErrorString(e));
}

size_t up256(size_t v) { return (v + 255) / 256 * 256; }
int64_t ld_of(int64_t cols) { return (cols + 15) / 16 * 16; }
int64_t nkb_of(int64_t cols) { return (cols + kF8Block - 1) / kF8Block; }

bool float_dtype(int dtype) { return host_dtype_size(dtype) != 0; }

// Row stride, then codes and scales, of a [rows x cols] matrix.
int check_ld(int64_t ld, int64_t cols, const char* what, const char* fn) {
    if (ld >= cols && ld % 16 == 0) return AXQ_OK;
    return fail(AXQ_ERR_INVALID, std::string(fn) + ": the row stride of " + what + " must be a multiple of 16 of at least " +
                                     std::to_string(cols) + " (got " + std::to_string(ld) + ")");
}

int check_codes(const void* codes, int64_t ld, const float* scales, int64_t cols, const char* what, const char* fn) {
    if (int r = check_ld(ld, cols, what, fn)) return r;
    if (int r = check_device_ptr(codes, what, fn)) return r;
    if (int r = check_device_ptr(scales, (std::string("the scales of ") + what).c_str(), fn)) return r;
    if (reinterpret_cast<uintptr_t>(codes) % 16 || reinterpret_cast<uintptr_t>(scales) % 4)
        return fail(AXQ_ERR_INVALID, std::string(fn) + ": " + what + " must be 16-byte aligned and its scales 4-byte aligned");
    return AXQ_OK;
}

int check_blocks(int64_t rows, int64_t cols, int block_rows, const char* fn) {
    if (rows < 0 || cols < 0) return fail(AXQ_ERR_INVALID, std::string(fn) + ": negative shape");
    if (block_rows != 1 && block_rows != kF8Block)
        return fail(AXQ_ERR_INVALID, std::string(fn) + ": block_rows must be 1 or 128");
    if (cols > (int64_t(1) << 30) || rows > (int64_t(1) << 31) ||
        (rows + block_rows - 1) / block_rows * nkb_of(cols) >= (int64_t(1) << 30))
        return fail(AXQ_ERR_INVALID, std::string(fn) + ": shape too large");
    return AXQ_OK;
}

int64_t codes_span(int64_t rows, int64_t cols, int64_t ld) { return (rows - 1) * ld + cols; }
int64_t scales_span(int64_t rows, int64_t cols, int block_rows) {
    return (rows + block_rows - 1) / block_rows * nkb_of(cols) * 4;
}

}  // namespace
}  // namespace axq

using namespace axq;

extern "C" {

int axq_quantize_f8(int dtype, const void* src, void* codes, int64_t ld, float* scales, int64_t rows, int64_t cols,
                    int block_rows, axq_stream_t stream) {
    const char* fn = "axq_quantize_f8";
    if (!float_dtype(dtype)) return fail(AXQ_ERR_UNSUPPORTED, std::string(fn) + ": unsupported dtype " + std::to_string(dtype));
    if (int r = check_blocks(rows, cols, block_rows, fn)) return r;
    if (rows == 0 || cols == 0) return AXQ_OK;
    if (int r = check_ld(ld, cols, "codes", fn)) return r;
    // the zeros behind the last row's codes are written too
    const int64_t codes_bytes = (rows - 1) * ld + std::min(ld, nkb_of(cols) * kF8Block);
    if (int r = check_apart({{codes, codes_bytes, "codes"}, {scales, scales_span(rows, cols, block_rows), "the scales"}},
                            {{src, rows * cols * host_dtype_size(dtype), "src"}}, fn))
        return r;
    if (int r = check_device_ptr(src, "src", fn)) return r;
    if (reinterpret_cast<uintptr_t>(src) % host_dtype_size(dtype))
        return fail(AXQ_ERR_INVALID, std::string(fn) + ": src is not aligned to its element type");
    if (int r = check_codes(codes, ld, scales, cols, "codes", fn)) return r;
    return status(f8_pack_dispatch(dtype, src, codes, ld, scales, rows, cols, block_rows, nullptr,
                                   reinterpret_cast<cudaStream_t>(stream)), fn);
}

int axq_dequantize_f8(const void* codes, int64_t ld, const float* scales, int block_rows, float* dst, int64_t rows,
                      int64_t cols, axq_stream_t stream) {
    const char* fn = "axq_dequantize_f8";
    if (int r = check_blocks(rows, cols, block_rows, fn)) return r;
    if (rows == 0 || cols == 0) return AXQ_OK;
    if (int r = check_codes(codes, ld, scales, cols, "codes", fn)) return r;
    if (int r = check_device_ptr(dst, "dst", fn)) return r;
    if (reinterpret_cast<uintptr_t>(dst) % 4) return fail(AXQ_ERR_INVALID, std::string(fn) + ": dst must be 4-byte aligned");
    if (overlap(dst, rows * cols * 4, codes, codes_span(rows, cols, ld)) ||
        overlap(dst, rows * cols * 4, scales, scales_span(rows, cols, block_rows)))
        return fail(AXQ_ERR_INVALID, std::string(fn) + ": dst must not overlap the codes or their scales");
    return status(f8_dequant_dispatch(codes, ld, scales, block_rows, dst, rows, cols, reinterpret_cast<cudaStream_t>(stream)),
                  fn);
}

size_t axq_linear_f8_workspace_size(int x_dtype, int64_t in_features, int64_t tokens) {
    if (in_features < 0 || tokens < 0) return 0;
    if (x_dtype == AXQ_DT_F8) return kStatusBytes;
    return kStatusBytes + up256(static_cast<size_t>(tokens) * ld_of(in_features)) +
           up256(static_cast<size_t>(tokens) * nkb_of(in_features) * 4);
}

int axq_linear_f8(const void* w_codes, int64_t w_ld, const float* w_scales, int x_dtype, const void* x, int64_t x_ld,
                  const float* x_scales, const float* bias, int y_dtype, void* y, int64_t out_features,
                  int64_t in_features, int64_t tokens, void* workspace, size_t workspace_bytes, axq_stream_t stream) {
    const char* fn = "axq_linear_f8";
    const int64_t M = out_features, K = in_features, N = tokens;
    const bool packed = x_dtype == AXQ_DT_F8;
    if (!packed && !float_dtype(x_dtype))
        return fail(AXQ_ERR_UNSUPPORTED, std::string(fn) + ": unsupported dtype of x " + std::to_string(x_dtype));
    if (!float_dtype(y_dtype))
        return fail(AXQ_ERR_UNSUPPORTED, std::string(fn) + ": unsupported dtype of y " + std::to_string(y_dtype));
    if (M < 0 || K < 0 || N < 0) return fail(AXQ_ERR_INVALID, std::string(fn) + ": negative shape");
    if (M == 0 || N == 0) return AXQ_OK;
    if (N > (int64_t(1) << 24) || M > (int64_t(1) << 30) || K > (int64_t(1) << 30) || N * nkb_of(K) >= (int64_t(1) << 30))
        return fail(AXQ_ERR_INVALID, std::string(fn) + ": shape too large");
    const size_t need = axq_linear_f8_workspace_size(x_dtype, K, N);
    if (!workspace || workspace_bytes < need)
        return fail(AXQ_ERR_WORKSPACE, std::string(fn) + ": workspace of " + std::to_string(need) + " bytes required");
    // without features neither w nor x is read
    if (int r = K ? check_ld(w_ld, K, "w", fn) : AXQ_OK) return r;
    if (int r = K && packed ? check_ld(x_ld, K, "x", fn) : AXQ_OK) return r;
    const int64_t x_span = packed ? codes_span(N, K, x_ld) : N * K * host_dtype_size(x_dtype);
    if (int r = check_apart({{y, N * M * host_dtype_size(y_dtype), "y"}, {workspace, static_cast<int64_t>(need), "the workspace"}},
                            {{bias, M * 4, "the bias"},
                             {w_codes, K ? codes_span(M, K, w_ld) : 0, "w"},
                             {w_scales, scales_span(M, K, kF8Block), "the scales of w"},
                             {x, K ? x_span : 0, "x"},
                             {packed ? x_scales : nullptr, scales_span(N, K, 1), "the scales of x"}},
                            fn))
        return r;
    if (int r = check_device_ptr(y, "y", fn)) return r;
    if (reinterpret_cast<uintptr_t>(y) % host_dtype_size(y_dtype))
        return fail(AXQ_ERR_INVALID, std::string(fn) + ": y is not aligned to its element type");
    if (bias) {
        if (int r = check_device_ptr(bias, "bias", fn)) return r;
        if (reinterpret_cast<uintptr_t>(bias) % 4) return fail(AXQ_ERR_INVALID, std::string(fn) + ": bias must be 4-byte aligned");
    }
    if (int r = check_device_ptr(workspace, "workspace", fn)) return r;
    if (reinterpret_cast<uintptr_t>(workspace) % 256)
        return fail(AXQ_ERR_INVALID, std::string(fn) + ": workspace must be 256-byte aligned");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    auto* ws = static_cast<uint8_t*>(workspace);
    int* err = reinterpret_cast<int*>(ws);
    if (K == 0) return status(f8_fill_bias_dispatch(y_dtype, y, bias, M, N, err, s), fn);
    if (int r = check_codes(w_codes, w_ld, w_scales, K, "w", fn)) return r;
    F8Linear l{};
    l.w = w_codes;
    l.w_scales = w_scales;
    l.w_ld = w_ld;
    l.bias = bias;
    l.y = y;
    l.y_dtype = y_dtype;
    l.M = M;
    l.K = K;
    l.N = N;
    l.err = err;
    if (packed) {
        if (int r = check_codes(x, x_ld, x_scales, K, "x", fn)) return r;
        l.x = x;
        l.x_scales = x_scales;
        l.x_ld = x_ld;
        if (int r = status(cudaMemsetAsync(err, 0, sizeof(int), s), fn)) return r;
    } else {
        if (x_ld != K) return fail(AXQ_ERR_INVALID, std::string(fn) + ": x must be contiguous (x_ld = in_features)");
        if (int r = check_device_ptr(x, "x", fn)) return r;
        if (reinterpret_cast<uintptr_t>(x) % host_dtype_size(x_dtype))
            return fail(AXQ_ERR_INVALID, std::string(fn) + ": x is not aligned to its element type");
        if (f8_gemm_packs(M, K, N)) {
            l.x = x;
            return status(f8_gemm_unpacked_dispatch(l, x_dtype, s), fn);
        }
        l.x_ld = ld_of(K);
        uint8_t* codes = ws + kStatusBytes;
        float* scales = reinterpret_cast<float*>(codes + up256(static_cast<size_t>(N) * l.x_ld));
        l.x = codes;
        l.x_scales = scales;
        if (int r = status(f8_pack_dispatch(x_dtype, x, codes, l.x_ld, scales, N, K, 1, err, s), fn)) return r;
    }
    return status(f8_gemm_dispatch(l, s), fn);
}

}  // extern "C"
