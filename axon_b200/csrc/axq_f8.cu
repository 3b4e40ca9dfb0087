// e4m3 packing: src[rows x cols] (fp32, fp16 or bf16) -> codes and one fp32
// scale per block of R rows x 128 columns, R = 1 (activations) or 128
// (weights):
//   scale = RN(max|x| / 448),  code = e4m3(RN(x / scale)),
// both roundings to nearest even, codes saturating; a block whose scale is 0
// has codes 0.  NaN elements keep NaN codes and do not enter the maximum; an
// infinity makes its block's scale infinite, so the block decodes to NaN.
//
// HBM-bound: every element is read once (the block stays in registers between
// the maximum and the rounding) and one byte written.  Weights 28672 x 8192 fp32
// take 234 us, 4.9 TB/s; activations 2500 x 8200 fp16 16 us, issue-bound: 18
// instructions for an element, 3.5 of them the exact division and the conversion
// to e4m3, the others conversions of the source, maxima, shuffles and addresses;
// one row of 4096 2.4 us, a launch.
#include <algorithm>

#include "axq_common.cuh"
#include "axq_f8.cuh"
#include "axq_internal.h"
#include "axq_ptx.cuh"

namespace axq {
namespace {

// 1 x 128 blocks: 16 lanes hold a block, 8 elements each; a half warp takes
// kPackUnroll blocks at once so that their loads are in flight together.  A
// block's row and place in it are walked, not divided out; 48 registers let
// five blocks of threads share an SM (with 72 and three the loads' latency
// showed: 34 us at 2500 x 8200 fp16).
constexpr int kPackUnroll = 2;

template <typename T, bool VEC>
__global__ void __launch_bounds__(256, 5) f8_pack_rows_kernel(const T* __restrict__ src, uint8_t* __restrict__ codes,
                                                              int64_t ld, float* __restrict__ scales, int64_t rows,
                                                              int64_t cols, int nkb, int* __restrict__ err) {
    pdl_wait();
    pdl_launch_dependents();
    if (err && blockIdx.x == 0 && threadIdx.x == 0) *err = 0;  // status word of the call this packing opens
    const uint32_t halves = gridDim.x * blockDim.x >> 4, half = (blockIdx.x * blockDim.x + threadIdx.x) >> 4;
    const uint32_t n = static_cast<uint32_t>(nkb);
    const uint32_t step_r = halves / n, step_k = halves - step_r * n;
    uint32_t r = half / n, kb = half - r * n;
    const uint32_t nr = static_cast<uint32_t>(rows);
    const int l = threadIdx.x & 15;
    // both halves of a warp stay in the loop together (the shuffles are warp-wide)
    while (__any_sync(0xFFFFFFFFu, r < nr)) {
        float v[kPackUnroll][8];
        uint32_t ur[kPackUnroll], uk[kPackUnroll];
#pragma unroll
        for (int u = 0; u < kPackUnroll; ++u) {
            ur[u] = r;
            uk[u] = kb;
            if (r < nr) {
                load_row8<T, VEC>(src + static_cast<int64_t>(r) * cols, static_cast<int64_t>(kb) * kF8Block + 8 * l, cols, v[u]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[u][i] = 0.0f;
            }
            r += step_r;
            kb += step_k;
            if (kb >= n) {
                kb -= n;
                ++r;
            }
        }
#pragma unroll
        for (int u = 0; u < kPackUnroll; ++u) {
            uint32_t w[2];
            const float s = pack_block16(v[u], w);
            if (ur[u] < nr) {
                const int64_t c0 = static_cast<int64_t>(uk[u]) * kF8Block + 8 * l;
                if (c0 < ld) *reinterpret_cast<uint2*>(codes + static_cast<int64_t>(ur[u]) * ld + c0) = make_uint2(w[0], w[1]);
                if (l == 0) scales[static_cast<int64_t>(ur[u]) * n + uk[u]] = s;
            }
        }
    }
}

// 128 x 128 blocks: one CTA per block, 16 rows per warp, 4 elements per lane
// and row, all 64 values of a thread in registers.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) f8_pack_blocks_kernel(const T* __restrict__ src, uint8_t* __restrict__ codes,
                                                             int64_t ld, float* __restrict__ scales, int64_t rows,
                                                             int64_t cols, int nkb) {
    __shared__ float red[8];
    pdl_wait();
    pdl_launch_dependents();
    const int64_t rb = blockIdx.x / static_cast<uint32_t>(nkb);
    const int kb = static_cast<int>(blockIdx.x - static_cast<uint32_t>(rb) * nkb);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t r0 = rb * kF8Block + 16 * warp, c0 = static_cast<int64_t>(kb) * kF8Block + 4 * lane;
    float v[16][4];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const int64_t r = r0 + j;
        const T* p = src + r * cols + c0;
        if (VEC && r < rows && c0 + 4 <= cols) {
            if constexpr (sizeof(T) == 4) {
                const float4 a = *reinterpret_cast<const float4*>(p);
                v[j][0] = a.x; v[j][1] = a.y; v[j][2] = a.z; v[j][3] = a.w;
            } else {
                const uint2 a = *reinterpret_cast<const uint2*>(p);
                T h[4];
                memcpy(h, &a, 8);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[j][i] = Elem<T>::get(h[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[j][i] = (r < rows && c0 + i < cols) ? Elem<T>::get(p[i]) : 0.0f;
        }
    }
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) m = fmaxf(m, fabsf(v[j][i]));
#pragma unroll
    for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
    if (lane == 0) red[warp] = m;
    __syncthreads();
    m = red[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) m = fmaxf(m, red[i]);
    const float s = f8_scale(m);
    if (threadIdx.x == 0) scales[blockIdx.x] = s;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const int64_t r = r0 + j;
        uint32_t w[1];
        f8_codes(v[j], s, w);
        if (r < rows && c0 < ld) *reinterpret_cast<uint32_t*>(codes + r * ld + c0) = w[0];
    }
}

// dst = code * scale, one rounding; 4 elements per thread.
__global__ void __launch_bounds__(256) f8_dequant_kernel(const uint8_t* __restrict__ codes, int64_t ld,
                                                         const float* __restrict__ scales, int block_rows,
                                                         float* __restrict__ dst, int64_t rows, int64_t cols, int nkb) {
    pdl_wait();
    pdl_launch_dependents();
    const int64_t quads = (cols + 3) / 4, n = rows * quads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t r = i / quads, c = 4 * (i - r * quads);
        const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + r * ld + c);
        const float s = scales[r / block_rows * nkb + c / kF8Block];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (c + u >= cols) break;
            __nv_fp8_e4m3 q;
            q.__x = static_cast<__nv_fp8_storage_t>(w >> (8 * u));
            dst[r * cols + c + u] = __fmul_rn(static_cast<float>(q), s);
        }
    }
}

// y = bias (or 0) on every row: a product over no columns.
template <typename TY>
__global__ void f8_fill_bias_kernel(TY* __restrict__ y, const float* __restrict__ bias, int64_t M, int64_t n,
                                    int* __restrict__ err) {
    pdl_wait();
    pdl_launch_dependents();
    if (blockIdx.x == 0 && threadIdx.x == 0) *err = 0;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x)
        y[i] = Elem<TY>::put(bias ? bias[i % M] : 0.0f);
}

}  // namespace

cudaError_t f8_fill_bias_dispatch(int dtype, void* y, const float* bias, int64_t M, int64_t N, int* err, cudaStream_t s) {
    return with_dtype(dtype, [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        const int64_t grid = std::min<int64_t>((M * N + 255) / 256, int64_t(device_sm_count()) * 8);
        cudaError_t e = launch_pdl(f8_fill_bias_kernel<T>, dim3(static_cast<unsigned>(grid)), dim3(256), 0, s,
                                   static_cast<T*>(y), bias, M, M * N, err);
        return e == cudaSuccess ? cudaGetLastError() : e;
    });
}

cudaError_t f8_pack_dispatch(int dtype, const void* src, void* codes, int64_t ld, float* scales, int64_t rows,
                             int64_t cols, int block_rows, int* err, cudaStream_t s) {
    const int nkb = static_cast<int>((cols + kF8Block - 1) / kF8Block);
    auto* out = static_cast<uint8_t*>(codes);
    return with_dtype(dtype, [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        const T* p = static_cast<const T*>(src);
        // 16-byte loads (8 of a 16-bit type, 4 of fp32 in the block kernel's 8-byte ones) need every row aligned
        const bool vec = reinterpret_cast<uintptr_t>(src) % 16 == 0 && (cols * sizeof(T)) % 16 == 0;
        if (block_rows == 1) {
            // a half warp for each block up to a full GPU: small matrices are bound by the latency of one round
            const int64_t grid = std::min<int64_t>((rows * nkb + 15) / 16, int64_t(device_sm_count()) * 5);
            auto k = vec ? f8_pack_rows_kernel<T, true> : f8_pack_rows_kernel<T, false>;
            cudaError_t e = launch_pdl(k, dim3(static_cast<unsigned>(grid)), dim3(256), 0, s, p, out, ld, scales, rows,
                                       cols, nkb, err);
            return e == cudaSuccess ? cudaGetLastError() : e;
        }
        const int64_t grid = (rows + kF8Block - 1) / kF8Block * nkb;
        auto k = vec ? f8_pack_blocks_kernel<T, true> : f8_pack_blocks_kernel<T, false>;
        cudaError_t e = launch_pdl(k, dim3(static_cast<unsigned>(grid)), dim3(256), 0, s, p, out, ld, scales, rows, cols,
                                   nkb);
        return e == cudaSuccess ? cudaGetLastError() : e;
    });
}

cudaError_t f8_dequant_dispatch(const void* codes, int64_t ld, const float* scales, int block_rows, float* dst,
                                int64_t rows, int64_t cols, cudaStream_t s) {
    const int nkb = static_cast<int>((cols + kF8Block - 1) / kF8Block);
    const int64_t n = rows * ((cols + 3) / 4);
    const int64_t grid = std::min<int64_t>((n + 255) / 256, int64_t(device_sm_count()) * 16);
    cudaError_t e = launch_pdl(f8_dequant_kernel, dim3(static_cast<unsigned>(grid)), dim3(256), 0, s,
                               static_cast<const uint8_t*>(codes), ld, scales, block_rows, dst, rows, cols, nkb);
    return e == cudaSuccess ? cudaGetLastError() : e;
}

}  // namespace axq
