// C entry points of the mixture-of-experts layer (include/axq.h): argument
// checks and dispatch.  Nothing here allocates device memory.
#include <cstdint>
#include <string>

#include "axq_common.cuh"
#include "axq_f8.cuh"
#include "axq_internal.h"

namespace axq {
namespace {

constexpr int64_t kMaxDim = int64_t(1) << 20;

int fail(int code, const std::string& msg) {
    set_last_error(msg);
    return code;
}

int status(cudaError_t e, const char* fn) {
    if (e == cudaSuccess) return AXQ_OK;
    return fail(AXQ_ERR_CUDA, std::string(fn) + ": " + cudaGetErrorString(e));
}

int check_aligned(const void* p, const char* what, int align, const char* fn) {
    if (int r = check_device_ptr(p, what, fn)) return r;
    if (reinterpret_cast<uintptr_t>(p) % align)
        return fail(AXQ_ERR_INVALID, std::string(fn) + ": " + what + " must be " + std::to_string(align) + "-byte aligned");
    return AXQ_OK;
}

int check_sizes(int64_t tokens, int64_t experts, int64_t top_k, int64_t hidden, int64_t ffn, const char* fn) {
    if (tokens < 0 || experts < 0 || top_k < 0 || hidden < 0 || ffn < 0)
        return fail(AXQ_ERR_INVALID, std::string(fn) + ": negative shape");
    if (experts < 1 || experts > AXQ_MOE_MAX_EXPERTS)
        return fail(AXQ_ERR_UNSUPPORTED, std::string(fn) + ": experts must be 1 .. " + std::to_string(AXQ_MOE_MAX_EXPERTS));
    if (top_k < 1 || top_k > AXQ_MOE_MAX_TOP_K)
        return fail(AXQ_ERR_UNSUPPORTED, std::string(fn) + ": top_k must be 1 .. " + std::to_string(AXQ_MOE_MAX_TOP_K));
    if (tokens > kMaxDim || hidden > kMaxDim || ffn > kMaxDim)
        return fail(AXQ_ERR_INVALID, std::string(fn) + ": shape too large");
    return AXQ_OK;
}

int check_weights(int fmt, const void* w, const float* scales, const char* what, const char* fn) {
    if (int r = check_aligned(w, what, 16, fn)) return r;
    if (fmt == AXQ_F8_E4M3) return check_aligned(scales, (std::string("the scales of ") + what).c_str(), 4, fn);
    if (scales) return fail(AXQ_ERR_INVALID, std::string(fn) + ": " + what + " is not e4m3 and has no scales");
    return AXQ_OK;
}

// Bytes of rows packed rows of cols elements; -1 past the largest allocation there can be.
int64_t packed_bytes(int fmt, int64_t rows, int64_t cols) {
    const int64_t be = fmt == AXQ_F8_E4M3 ? 1 : host_block_elems(fmt), bb = fmt == AXQ_F8_E4M3 ? 1 : host_block_bytes(fmt);
    const int64_t row = (cols + be - 1) / be * bb;
    return rows > (int64_t(1) << 45) / row ? -1 : rows * row;
}

}  // namespace
}  // namespace axq

using namespace axq;

extern "C" {

int axq_moe_route(int dtype, const void* x, const float* w_router, int32_t* ids, float* weights, int64_t tokens,
                  int64_t experts, int64_t top_k, int64_t hidden, int normalize, axq_stream_t stream) {
    const char* fn = "axq_moe_route";
    if (!host_dtype_size(dtype)) return fail(AXQ_ERR_UNSUPPORTED, std::string(fn) + ": unsupported dtype " + std::to_string(dtype));
    if (int r = check_sizes(tokens, experts, top_k, hidden, 0, fn)) return r;
    if (top_k > experts) return fail(AXQ_ERR_INVALID, std::string(fn) + ": top_k is larger than the number of experts");
    if (tokens == 0) return AXQ_OK;
    if (hidden == 0) return fail(AXQ_ERR_INVALID, std::string(fn) + ": hidden must be positive");
    // a token's choices are written while other blocks still read x and the router
    const int64_t choices = tokens * top_k * 4;
    if (int r = check_apart({{ids, choices, "ids"}, {weights, choices, "weights"}},
                            {{x, tokens * hidden * host_dtype_size(dtype), "x"}, {w_router, experts * hidden * 4, "w_router"}}, fn))
        return r;
    if (int r = check_aligned(x, "x", host_dtype_size(dtype), fn)) return r;
    if (int r = check_aligned(w_router, "w_router", 4, fn)) return r;
    if (int r = check_aligned(ids, "ids", 4, fn)) return r;
    if (int r = check_aligned(weights, "weights", 4, fn)) return r;
    return status(moe_route_dispatch(dtype, x, w_router, ids, weights, tokens, static_cast<int>(experts),
                                     static_cast<int>(top_k), hidden, normalize, reinterpret_cast<cudaStream_t>(stream)),
                  fn);
}

size_t axq_moe_workspace_size(int64_t tokens, int64_t top_k, int64_t hidden, int64_t ffn) {
    if (tokens < 0 || top_k < 1 || top_k > AXQ_MOE_MAX_TOP_K || hidden < 0 || ffn < 0) return 0;
    return moe_workspace_bytes(tokens, static_cast<int>(top_k), hidden, ffn);
}

static int moe_call(const char* fn, int fmt, const void* w_gate, const float* gate_scales, const void* w_up,
                    const float* up_scales, int fmt_down, const void* w_down, const float* down_scales, int dtype,
                    const void* x, const float* w_router, int normalize, int32_t* ids, float* weights, void* y,
                    int64_t tokens, int64_t experts, int64_t top_k, int64_t hidden, int64_t ffn, void* workspace,
                    size_t workspace_bytes, axq_stream_t stream) {
    for (int f : {fmt, fmt_down})
        if (f != AXQ_F8_E4M3 && !host_block_elems(f))
            return fail(AXQ_ERR_UNSUPPORTED, std::string(fn) + ": unsupported format " + std::to_string(f));
    if (!host_dtype_size(dtype)) return fail(AXQ_ERR_UNSUPPORTED, std::string(fn) + ": unsupported dtype " + std::to_string(dtype));
    if (int r = check_sizes(tokens, experts, top_k, hidden, ffn, fn)) return r;
    if (w_router && top_k > experts)
        return fail(AXQ_ERR_INVALID, std::string(fn) + ": top_k is larger than the number of experts");
    if (tokens == 0 || hidden == 0) return AXQ_OK;
    if ((fmt == AXQ_F8_E4M3 || fmt_down == AXQ_F8_E4M3) && (hidden % kF8Block || ffn % kF8Block))
        return fail(AXQ_ERR_UNSUPPORTED, std::string(fn) + ": e4m3 experts need hidden and ffn to be multiples of 128");
    // without hidden features (ffn 0) neither the experts' weights nor the workspace are looked at
    const size_t need = ffn ? axq_moe_workspace_size(tokens, top_k, hidden, ffn) : 0;
    if (ffn && (!workspace || workspace_bytes < need))
        return fail(AXQ_ERR_WORKSPACE, std::string(fn) + ": workspace of " + std::to_string(need) + " bytes required");
    const int64_t gate_bytes = ffn ? packed_bytes(fmt, experts * ffn, hidden) : 0;
    const int64_t down_bytes = ffn ? packed_bytes(fmt_down, experts * hidden, ffn) : 0;
    if (gate_bytes < 0 || down_bytes < 0) return fail(AXQ_ERR_INVALID, std::string(fn) + ": shape too large");
    const int64_t row = hidden * host_dtype_size(dtype), choices = tokens * top_k * 4;
    const int64_t scales = experts * (ffn / kF8Block) * (hidden / kF8Block) * 4;  // of an e4m3 matrix
    // ids and weights are written where there is a router, else read
    if (int r = check_apart({{y, tokens * row, "y"},
                             {workspace, static_cast<int64_t>(need), "the workspace"},
                             {w_router ? ids : nullptr, choices, "ids"},
                             {w_router ? weights : nullptr, choices, "weights"}},
                            {{x, tokens * row, "x"},
                             {w_router, experts * hidden * 4, "w_router"},
                             {w_router ? nullptr : ids, choices, "ids"},
                             {w_router ? nullptr : weights, choices, "weights"},
                             {w_gate, gate_bytes, "w_gate"},
                             {w_up, gate_bytes, "w_up"},
                             {w_down, down_bytes, "w_down"},
                             {gate_scales, scales, "the scales of w_gate"},
                             {up_scales, scales, "the scales of w_up"},
                             {down_scales, scales, "the scales of w_down"}},
                            fn))
        return r;
    if (int r = check_aligned(y, "y", host_dtype_size(dtype), fn)) return r;
    if (int r = check_aligned(x, "x", host_dtype_size(dtype), fn)) return r;
    if (int r = check_aligned(ids, "ids", 4, fn)) return r;
    if (int r = check_aligned(weights, "weights", 4, fn)) return r;
    if (w_router)
        if (int r = check_aligned(w_router, "w_router", 4, fn)) return r;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (ffn == 0) {
        if (w_router) {
            cudaError_t e = moe_route_dispatch(dtype, x, w_router, ids, weights, tokens, static_cast<int>(experts),
                                               static_cast<int>(top_k), hidden, normalize, s);
            if (e != cudaSuccess) return status(e, fn);
        }
        return status(cudaMemsetAsync(y, 0, static_cast<size_t>(tokens * hidden) * host_dtype_size(dtype), s), fn);
    }
    if (int r = check_weights(fmt, w_gate, gate_scales, "w_gate", fn)) return r;
    if (int r = check_weights(fmt, w_up, up_scales, "w_up", fn)) return r;
    if (int r = check_weights(fmt_down, w_down, down_scales, "w_down", fn)) return r;
    if (int r = check_aligned(workspace, "workspace", 256, fn)) return r;
    MoeMlp m{};
    m.fmt = fmt;
    m.fmt_down = fmt_down;
    m.w_gate = w_gate;
    m.w_up = w_up;
    m.w_down = w_down;
    m.s_gate = gate_scales;
    m.s_up = up_scales;
    m.s_down = down_scales;
    m.gate_bytes = gate_bytes;
    m.down_bytes = down_bytes;
    m.dtype = dtype;
    m.x = x;
    m.w_router = w_router;
    m.normalize = normalize;
    m.ids = ids;
    m.weights = weights;
    m.y = y;
    m.tokens = tokens;
    m.hidden = hidden;
    m.ffn = ffn;
    m.experts = static_cast<int>(experts);
    m.top_k = static_cast<int>(top_k);
    return status(moe_mlp_dispatch(m, workspace, reinterpret_cast<int*>(workspace), s), fn);
}

int axq_moe_mlp(int fmt, const void* w_gate, const float* gate_scales, const void* w_up, const float* up_scales,
                int fmt_down, const void* w_down, const float* down_scales, int dtype, const void* x, const int32_t* ids,
                const float* weights, void* y, int64_t tokens, int64_t experts, int64_t top_k, int64_t hidden,
                int64_t ffn, void* workspace, size_t workspace_bytes, axq_stream_t stream) {
    // without a router ids and weights are only read
    return moe_call("axq_moe_mlp", fmt, w_gate, gate_scales, w_up, up_scales, fmt_down, w_down, down_scales, dtype, x, nullptr,
                    0, const_cast<int32_t*>(ids), const_cast<float*>(weights), y, tokens, experts, top_k, hidden, ffn,
                    workspace, workspace_bytes, stream);
}

int axq_moe(int fmt, const void* w_gate, const float* gate_scales, const void* w_up, const float* up_scales, int fmt_down,
            const void* w_down, const float* down_scales, int dtype, const void* x, const float* w_router, int normalize,
            int32_t* ids, float* weights, void* y, int64_t tokens, int64_t experts, int64_t top_k, int64_t hidden,
            int64_t ffn, void* workspace, size_t workspace_bytes, axq_stream_t stream) {
    if (hidden == 0 && tokens > 0) return fail(AXQ_ERR_INVALID, "axq_moe: hidden must be positive");  // as the router
    if (!w_router && tokens > 0) return fail(AXQ_ERR_INVALID, "axq_moe: w_router is NULL");
    return moe_call("axq_moe", fmt, w_gate, gate_scales, w_up, up_scales, fmt_down, w_down, down_scales, dtype, x, w_router,
                    normalize, ids, weights, y, tokens, experts, top_k, hidden, ffn, workspace, workspace_bytes, stream);
}

}  // extern "C"
