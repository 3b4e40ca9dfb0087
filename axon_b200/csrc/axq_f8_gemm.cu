// y[N x M] = X . W^T (+ bias) on e4m3 operands with one fp32 scale per 1 x 128
// block of X and per 128 x 128 block of W:
//   y[t][m] = sum_kb sx[t][kb] * sw[m/128][kb] * P_kb[t][m],
//   P_kb[t][m] = sum over the 128 k of block kb of x[t][k] * w[m][k].
//
// P_kb is four tcgen05 MMAs of K = 32 into TMEM (fp32); the scales change
// every 128 k, so each P_kb leaves TMEM and is added with its scale to fp32
// registers while the tensor core works on the next block in another TMEM
// buffer.  Tiles come by tensor-map copies in the 128-byte swizzle; copies
// past the edges read zeros, so any M, N and K need no other masking than
// that of the stores.
//
// Two forms:
//  * f8_pair_kernel (many tokens): a CTA pair computes 256 tokens x BN
//    weight rows with one cta_group::2 MMA; each CTA holds 128 tokens (TMEM
//    lanes) and loads half of the weight rows, so the weights cross from L2
//    once per pair.  A thread owns a token's row, so its scale is one product
//    per 128 k.  Every accumulator leaves TMEM once per 128 k, which bounds it:
//    4096 tokens x 28672 x 8192 take 900 us (2.1 PFLOP/s, the tensor pipe half
//    busy).  Clocks counted in the issuing warps: 69 % of their time they wait
//    for an empty accumulator, 10 % for operands; tiles of 128 columns, with four
//    accumulators instead of two, wait 50 % and are slower (1137 against 948 us,
//    both with the counting).  So the waits cost most: two issuing
//    warps, one commit per block and relaxed arrivals from the other CTA (a
//    release there is a memory barrier: 1.2 ms) are what they led to.  16
//    epilogue warps and accumulators as 64-bit pairs were no faster.
//  * f8_skinny_kernel (few tokens): 128 weight rows are the MMA's M side, NT
//    >= N tokens its N side, and a cluster splits K; its CTAs' sums are joined
//    through distributed shared memory in rank order.  HBM-bound on W: 28672 x
//    8192 for 16 tokens in 46 us, 5.1 TB/s; a 4096 x 4096 matrix (6.4 us) by
//    launch and latency.
#include <algorithm>
#include <type_traits>
#include <cuda.h>

#include "axq_common.cuh"
#include "axq_f8.cuh"
#include "axq_internal.h"
#include "axq_ptx.cuh"
#include "axq_tc.cuh"

namespace axq {
namespace {

constexpr int kMaxF8Stages = 8;

struct F8Args {
    const float* sx;
    const float* sw;
    const float* bias;
    void* y;
    int64_t M, N;
    int nkb;
    int nbuf;    // TMEM buffers
    int stages;
    int tiles_n, tiles_m;  // pair kernel: token tiles, weight-row tiles
    const void* x;         // unpacked X (skinny kernel that packs it itself)
    int64_t K;
    int xvec;              // its rows start on 16-byte boundaries
    int* err;
};

// One commit per K block serves both who waits for it: done[s] says that the
// MMAs on stage s have finished, so the stage may be filled again and the
// accumulator of that block be read.
struct F8Bars {
    uint64_t full[kMaxF8Stages], done[kMaxF8Stages];
    uint64_t acc_empty[4];
    uint32_t tmem;
    int abort;
};

// Bounded wait of a whole warp; on giving up sets the CTA's abort flag and the
// status word.
__device__ __forceinline__ bool f8_wait(uint64_t* bar, uint32_t parity, F8Bars* b, int* err) {
    bool ok = mbar_try_wait(bar, parity);
#pragma unroll 1
    for (int i = 0; i < 16 && !ok; ++i) ok = mbar_try_wait(bar, parity);  // before the slower timer is read
    if (__builtin_expect(!ok, 0)) ok = mbar_wait_bounded(bar, parity, &b->abort);
    ok = __all_sync(0xFFFFFFFFu, ok);
    if (__builtin_expect(!ok, 0)) {
        *const_cast<volatile int*>(&b->abort) = 1;
        if (err) atomicExch(err, 1);
    }
    return ok;
}

// Eight values to y in its type (one or two 16-byte stores).
template <typename TY>
__device__ __forceinline__ void store8(TY* p, const float* v) {
    if constexpr (sizeof(TY) == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        TY h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = Elem<TY>::put(v[i]);
        uint4 w;
        memcpy(&w, h, 16);
        *reinterpret_cast<uint4*>(p) = w;
    }
}

// Warp 0 copies, warps 1 and 2 issue MMAs (3 only pads their warpgroup), 4 to
// 11 are the epilogue.  Registers move from the first warpgroup to the two of
// the epilogue: 128 * (56 + 2 * 224) is what 384 threads are launched with (168
// each).
constexpr int kPairThreads = 384;
constexpr int kPairRegsLow = 56, kPairRegsHigh = 224;

// Output staging of an epilogue warp: 32 rows of 128 bytes, 16 bytes apart.
constexpr int kOutRow = 144, kOutWarpBytes = 32 * kOutRow;

template <int BN, typename TY>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    f8_pair_kernel(const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap mw, F8Args a) {
    constexpr int kXBytes = 128 * 128;       // this CTA's 128 tokens x 128 k
    constexpr int kWBytes = (BN / 2) * 128;  // this CTA's half of the weight rows
    constexpr int kStage = kXBytes + kWBytes;
    constexpr int kCols = BN / 2;            // accumulator columns of a thread
    constexpr uint32_t kIdesc = idesc_e4m3_f32(BN, 256);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* stage0 = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    uint8_t* out_stage = stage0 + a.stages * kStage;
    __shared__ F8Bars bars;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    if (threadIdx.x == 0) {
        for (int i = 0; i < kMaxF8Stages; ++i) {
            mbar_init(&bars.full[i], 1);
            mbar_init(&bars.done[i], 1);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&bars.acc_empty[i], 16);  // eight epilogue warps of each CTA
        bars.abort = 0;
        fence_mbar_init();
        prefetch_tensormap(&mx);
        prefetch_tensormap(&mw);
    }
    if (warp == 1) tmem_alloc_cg<2>(&bars.tmem, 512);
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = bars.tmem;
    const int ntiles = a.tiles_n * a.tiles_m;
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

    if (warp < 4) regs_dec<kPairRegsLow>();
    if (warp == 0) {
        pdl_wait();
        int s = 0;
        uint32_t par = 0;
        bool ok = true;
        int64_t issued = 0;
        for (int tile = pair; tile < ntiles && ok; tile += npairs) {
            // token tiles run fastest: the pairs at work share few weight tiles
            const int tn = tile % a.tiles_n, tm = tile / a.tiles_n;
            const int xr = tn * 256 + static_cast<int>(rank) * 128;
            const int wr = tm * BN + static_cast<int>(rank) * (BN / 2);
            for (int kb = 0; kb < a.nkb; ++kb) {
                ok = f8_wait(&bars.done[s], par ^ 1, &bars, a.err);
                if (!ok) break;
                if (elect_one()) {
                    if (rank == 0) mbar_arrive_expect_tx(&bars.full[s], 2 * kStage);
                    const uint32_t fb = cluster_addr(&bars.full[s], 0);
                    uint8_t* st = stage0 + s * kStage;
                    tma_load_2d_pair(st, &mx, kb * 128, xr, fb);
                    tma_load_2d_pair(st + kXBytes, &mw, kb * 128, wr, fb);
                }
                __syncwarp();
                ++issued;
                if (++s == a.stages) {
                    s = 0;
                    par ^= 1;
                }
            }
        }
        if (!ok && rank == 0) {
            // copies still in flight land before the pair's shared memory goes away
            const int64_t from = issued > a.stages ? issued - a.stages : 0;
            for (int64_t i = from; i < issued; ++i)
                mbar_wait_bounded(&bars.full[i % a.stages], static_cast<uint32_t>((i / a.stages) & 1));
        }
        __syncwarp();
    } else if (warp == 1 || warp == 2) {
        if (rank == 0) {
            // Two issuing warps take K blocks in turn, each block in its own
            // accumulator, so that the waits and the commit of one run beside
            // the MMAs of the other.
            const int mytiles = (ntiles - pair + npairs - 1) / npairs;
            const int64_t blocks = static_cast<int64_t>(mytiles) * a.nkb;
            int s = (warp - 1) % a.stages, b = warp - 1;
            uint32_t par = 0, bpar = 0;
            for (int64_t it = warp - 1; it < blocks; it += 2) {
                if (!f8_wait(&bars.full[s], par, &bars, a.err) || !f8_wait(&bars.acc_empty[b], bpar ^ 1, &bars, a.err))
                    break;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t xs = smem_u32(stage0 + s * kStage);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_e4m3<2>(tmem + b * BN, smem_desc_sw128(xs + 32 * k), smem_desc_sw128(xs + kXBytes + 32 * k),
                                    kIdesc, k > 0);
                    mma_commit_pair(&bars.done[s]);
                }
                __syncwarp();
                if ((s += 2) >= a.stages) {
                    s -= a.stages;
                    par ^= 1;
                }
                if ((b += 2) >= a.nbuf) {
                    b -= a.nbuf;
                    bpar ^= 1;
                }
            }
        }
    } else if (warp >= 4) {
        regs_inc<kPairRegsHigh>();
        const int q = warp & 3, g = (warp - 4) >> 2;
        pdl_wait();
        int b = 0, s = 0;
        uint32_t par = 0;
        bool ok = true;
        TY* const y = static_cast<TY*>(a.y);
        const bool vec = (a.M * sizeof(TY)) % 16 == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0;
        const uint32_t ta = tmem + (static_cast<uint32_t>(32 * q) << 16) + g * kCols;
        const uint32_t empty0 = cluster_addr(&bars.acc_empty[0], 0);
        for (int tile = pair; tile < ntiles && ok; tile += npairs) {
            const int tn = tile % a.tiles_n, tm = tile / a.tiles_n;
            const int64_t t = static_cast<int64_t>(tn) * 256 + rank * 128 + 32 * q + lane;
            const int64_t m0 = static_cast<int64_t>(tm) * BN + g * kCols;
            const float* sx = a.sx + (t < a.N ? t : 0) * a.nkb;
            const float* sw = a.sw + (m0 < a.M ? m0 / 128 : 0) * a.nkb;
            float acc[kCols];
#pragma unroll
            for (int i = 0; i < kCols; ++i) acc[i] = 0.0f;
            float nx = __ldg(sx), nw = __ldg(sw);
            // Two chunks of 32 columns in turn: the load of one runs under the
            // FMAs of the other, across K blocks too.
            float v[2][32];
            ok = f8_wait(&bars.done[s], par, &bars, a.err);
            if (ok) {
                tc_fence_after();
                tmem_ld32_issue(ta + b * BN, v[0]);
            }
            for (int kb = 0; kb < a.nkb && ok; ++kb) {
                const float sc = nx * nw;
                if (kb + 1 < a.nkb) {
                    nx = __ldg(sx + kb + 1);
                    nw = __ldg(sw + kb + 1);
                }
#pragma unroll
                for (int c = 0; c < kCols / 32; ++c) {
                    tmem_ld_wait(v[c & 1]);
                    if (c + 1 < kCols / 32) {
                        tmem_ld32_issue(ta + b * BN + 32 * (c + 1), v[(c + 1) & 1]);
                    } else {
                        tc_fence_before();
                        __syncwarp();
                        if (elect_one()) mbar_arrive_cluster_relaxed(empty0 + 8 * b);
                        if (++b == a.nbuf) b = 0;
                        if (++s == a.stages) {
                            s = 0;
                            par ^= 1;
                        }
                        if (kb + 1 < a.nkb) {
                            ok = f8_wait(&bars.done[s], par, &bars, a.err);
                            tc_fence_after();
                            if (ok) tmem_ld32_issue(ta + b * BN, v[0]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 2)
                        fma2(acc[32 * c + i], acc[32 * c + i + 1], v[c & 1][i], v[c & 1][i + 1], sc, sc);
                }
            }
            if (!ok) break;
            // Through shared memory, so that a store covers 128 bytes of four
            // rows and not 16 bytes of 32 (the MMAs wait meanwhile: 5.5 us a
            // tile before): kOutCols columns of the warp's 32 rows at a time.
            constexpr int kOutCols = 128 / static_cast<int>(sizeof(TY));
            uint8_t* const own = out_stage + (warp - 4) * kOutWarpBytes;
            const int64_t t0 = t - lane;
            const int rows = static_cast<int>(min64(32, a.N - t0));
#pragma unroll
            for (int c0 = 0; c0 < kCols; c0 += kOutCols) {
                if (m0 + c0 >= a.M) break;
                if (a.bias) {
#pragma unroll
                    for (int i = 0; i < kOutCols; ++i)
                        if (m0 + c0 + i < a.M) acc[c0 + i] += __ldg(a.bias + m0 + c0 + i);
                }
#pragma unroll
                for (int i = 0; i < kOutCols; i += 8)
                    store8(reinterpret_cast<TY*>(own + lane * kOutRow) + i, acc + c0 + i);
                __syncwarp();
                if (vec && m0 + c0 + kOutCols <= a.M) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int r = 4 * j + (lane >> 3);
                        if (r < rows)
                            *reinterpret_cast<uint4*>(y + (t0 + r) * a.M + m0 + c0 + (lane & 7) * (kOutCols / 8)) =
                                *reinterpret_cast<const uint4*>(own + r * kOutRow + (lane & 7) * 16);
                    }
                } else {
                    for (int r = 0; r < rows; ++r)
                        for (int c = lane; c < kOutCols && m0 + c0 + c < a.M; c += 32)
                            y[(t0 + r) * a.M + m0 + c0 + c] = reinterpret_cast<const TY*>(own + r * kOutRow)[c];
                }
                __syncwarp();
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // neither CTA's barriers, shared memory or TMEM goes away under the other
    pdl_launch_dependents();
    if (warp == 1) tmem_dealloc_cg<2>(tmem, 512);
}

// ---- few tokens ---------------------------------------------------------------

constexpr int kSkinnyThreads = 192;  // producer warp, MMA warp, four epilogue warps

// TX: type of an X that the kernel packs itself (every CTA its K range of all
// tokens, while the first weight tiles arrive); void: X is packed already.
template <int NT, typename TY, typename TX>
__global__ void __launch_bounds__(kSkinnyThreads)
    f8_skinny_kernel(const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap mw, F8Args a, int splits) {
    constexpr int kEpi = 4;  // epilogue warps: a TMEM lane quarter each
    constexpr int kCols = NT;
    constexpr bool kPack = !std::is_void_v<TX>;
    constexpr int kWBytes = 128 * 128, kXBytes = NT * 128, kStage = kWBytes + (kPack ? 0 : kXBytes);
    constexpr int kBuf = 2;
    constexpr uint32_t kTmem = kBuf * NT <= 32 ? 32 : kBuf * NT;
    constexpr uint32_t kIdesc = idesc_e4m3_f32(NT, 128);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* stage0 = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    uint8_t* xs = stage0 + a.stages * kStage;  // the packed X of every K block, if the kernel packs it
    const int most = (a.nkb + splits - 1) / splits;
    float* sxs = reinterpret_cast<float*>(xs + (kPack ? most * kXBytes : 0));  // [kb][NT] scales of X
    float* red = reinterpret_cast<float*>(stage0);                      // [NT][128] sums, after the last MMA
    __shared__ F8Bars bars;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int mt = blockIdx.x / splits, rank = blockIdx.x - mt * splits;
    const int kb0 = static_cast<int>(static_cast<int64_t>(a.nkb) * rank / splits);
    const int nk = static_cast<int>(static_cast<int64_t>(a.nkb) * (rank + 1) / splits) - kb0;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kMaxF8Stages; ++i) {
            mbar_init(&bars.full[i], 1);
            mbar_init(&bars.done[i], 1);
        }
        for (int i = 0; i < kBuf; ++i) mbar_init(&bars.acc_empty[i], kEpi);
        bars.abort = 0;
        fence_mbar_init();
        prefetch_tensormap(&mx);
        prefetch_tensormap(&mw);
    }
    if (warp == 1) tmem_alloc(&bars.tmem, kTmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars.tmem;

    if (warp == 0) {
        // The packing of X, launched before this kernel, let it start only
        // after everything before the packing had finished, so W is there; X
        // is waited for.  Without a packing kernel W is waited for too.
        const int first = min(nk, a.stages);
        if (kPack) pdl_wait();
        if (elect_one()) {
            for (int i = 0; i < first; ++i) {
                mbar_arrive_expect_tx(&bars.full[i], kStage);
                tma_load_2d(stage0 + i * kStage, &mw, (kb0 + i) * 128, mt * 128, &bars.full[i]);
            }
        }
        __syncwarp();
        if constexpr (!kPack) {
            pdl_wait();
            if (elect_one()) {
                for (int i = 0; i < first; ++i)
                    tma_load_2d(stage0 + i * kStage + kWBytes, &mx, (kb0 + i) * 128, 0, &bars.full[i]);
            }
            __syncwarp();
        }
        int s = 0;
        uint32_t par = 0;
        bool ok = true;
        int issued = first;
        for (int i = first; i < nk; ++i) {
            ok = f8_wait(&bars.done[s], par, &bars, a.err);
            if (!ok) break;
            if (elect_one()) {
                mbar_arrive_expect_tx(&bars.full[s], kStage);
                tma_load_2d(stage0 + s * kStage, &mw, (kb0 + i) * 128, mt * 128, &bars.full[s]);
                if constexpr (!kPack)
                    tma_load_2d(stage0 + s * kStage + kWBytes, &mx, (kb0 + i) * 128, 0, &bars.full[s]);
            }
            __syncwarp();
            ++issued;
            if (++s == a.stages) {
                s = 0;
                par ^= 1;
            }
        }
        if (!ok)  // copies still in flight land before the shared memory goes away
            for (int i = max(0, issued - a.stages); i < issued; ++i)
                mbar_wait_bounded(&bars.full[i % a.stages], static_cast<uint32_t>((i / a.stages) & 1));
        __syncwarp();
    } else if (warp == 1) {
        int s = 0, b = 0;
        uint32_t par = 0, bpar = 0;
        if constexpr (kPack) {
            asm volatile("bar.sync 2, %0;" ::"n"(32 * kEpi + 32) : "memory");  // X is packed
            tc_fence_after();
        }
        for (int i = 0; i < nk; ++i) {
            if (!f8_wait(&bars.acc_empty[b], bpar ^ 1, &bars, a.err) || !f8_wait(&bars.full[s], par, &bars, a.err)) break;
            tc_fence_after();
            if (elect_one()) {
                const uint32_t ws = smem_u32(stage0 + s * kStage);
                const uint32_t xa = kPack ? smem_u32(xs + i * kXBytes) : ws + kWBytes;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    mma_e4m3<1>(tmem + b * NT, smem_desc_sw128(ws + 32 * k), smem_desc_sw128(xa + 32 * k), kIdesc, k > 0);
                mma_commit(&bars.done[s]);
            }
            __syncwarp();
            if (++s == a.stages) {
                s = 0;
                par ^= 1;
            }
            if (++b == kBuf) {
                b = 0;
                bpar ^= 1;
            }
        }
    } else {
        const int q = warp & 3;
        const int et = threadIdx.x - 64;
        pdl_wait();
        if constexpr (kPack) {
            // A wait that gives up does so after two seconds: long after this.
            if (a.err && blockIdx.x == 0 && et == 0) *a.err = 0;
            // 16 lanes to a block of 128; rows past N keep what the memory holds: their columns are never read
            const TX* x = static_cast<const TX*>(a.x);
            const int l = lane & 15;
            constexpr int U = 4;  // blocks whose loads are in flight together
            const int items = nk * static_cast<int>(a.N);
            for (int i0 = (et >> 5) * 2; i0 < items; i0 += 2 * kEpi * U) {
                float v[U][8];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (i0 + u * 2 * kEpi >= items) break;
                    const int i = i0 + u * 2 * kEpi + (lane >> 4), n = i / nk;
                    const int64_t c0 = static_cast<int64_t>(kb0 + i - n * nk) * kF8Block + 8 * l;
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[u][j] = 0.0f;
                    if (n < a.N) {
                        if (a.xvec)
                            load_row8<TX, true>(x + n * a.K, c0, a.K, v[u]);
                        else
                            load_row8<TX, false>(x + n * a.K, c0, a.K, v[u]);
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (i0 + u * 2 * kEpi >= items) break;
                    const int i = i0 + u * 2 * kEpi + (lane >> 4), n = i / nk, k = i - n * nk;
                    uint32_t w[2];
                    const float sc = pack_block16(v[u], w);
                    if (n < a.N) {
                        // the 128-byte swizzle: 16-byte chunk c of row n is at chunk c ^ (n % 8)
                        *reinterpret_cast<uint2*>(xs + k * kXBytes + n * 128 + (((l >> 1) ^ (n & 7)) << 4) + (l & 1) * 8) =
                            make_uint2(w[0], w[1]);
                        if (l == 0) sxs[k * NT + n] = sc;
                    }
                }
            }
            for (int i = et; i < nk * NT; i += 32 * kEpi)
                if (i % NT >= a.N) sxs[i] = 0.0f;
            fence_proxy_async_smem();
            tc_fence_before();
            asm volatile("bar.sync 2, %0;" ::"n"(32 * kEpi + 32) : "memory");
        } else {
            for (int i = et; i < nk * NT; i += 32 * kEpi) {
                const int n = i / nk, k = i - n * nk;
                sxs[k * NT + n] = n < a.N ? __ldg(a.sx + static_cast<int64_t>(n) * a.nkb + kb0 + k) : 0.0f;
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpi) : "memory");
        float acc[kCols];
#pragma unroll
        for (int i = 0; i < kCols; ++i) acc[i] = 0.0f;
        const float* sw = a.sw + static_cast<int64_t>(mt) * a.nkb + kb0;
        int b = 0, s = 0;
        uint32_t par = 0;
        float nw = nk > 0 ? __ldg(sw) : 0.0f;
        for (int i = 0; i < nk; ++i) {
            const float wsc = nw;
            if (i + 1 < nk) nw = __ldg(sw + i + 1);
            if (!f8_wait(&bars.done[s], par, &bars, a.err)) break;
            tc_fence_after();
            const uint32_t ta = tmem + (static_cast<uint32_t>(32 * q) << 16) + b * NT;
            const float* sc = sxs + i * NT;
#pragma unroll
            for (int c = 0; c < kCols; c += 16) {
                float v[16];
                tmem_ldw16(ta + c, v);
                if (c + 16 == kCols) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars.acc_empty[b]);
                }
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const float4 f = *reinterpret_cast<const float4*>(sc + c + j);
                    acc[c + j] = fmaf(v[j], f.x * wsc, acc[c + j]);
                    acc[c + j + 1] = fmaf(v[j + 1], f.y * wsc, acc[c + j + 1]);
                    acc[c + j + 2] = fmaf(v[j + 2], f.z * wsc, acc[c + j + 2]);
                    acc[c + j + 3] = fmaf(v[j + 3], f.w * wsc, acc[c + j + 3]);
                }
            }
            if (++b == kBuf) b = 0;
            if (++s == a.stages) {
                s = 0;
                par ^= 1;
            }
        }
        // every MMA has read its stages (the last accumulator was waited for),
        // so their memory holds the sums now: [token][weight row]
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpi) : "memory");
#pragma unroll
        for (int i = 0; i < kCols; ++i) red[i * 128 + 32 * q + lane] = acc[i];
    }
    tc_fence_before();
    __syncthreads();
    pdl_launch_dependents();
    if (warp == 1) tmem_dealloc(tmem, kTmem);
    if (splits > 1) cluster_sync_all();
    // the cluster's ranks each finish a share of the tokens
    TY* const y = static_cast<TY*>(a.y);
    const int n = static_cast<int>(a.N);
    for (int i = threadIdx.x; i < ((n + splits - 1) / splits) * 128; i += blockDim.x) {
        const int t = (i >> 7) * splits + rank, r = i & 127;
        const int64_t m = static_cast<int64_t>(mt) * 128 + r;
        if (t >= n || m >= a.M) continue;
        float v = 0.0f;
        if (splits == 1) {
            v = red[t * 128 + r];
        } else {
            const float* p = red + t * 128 + r;
            for (int k = 0; k < splits; ++k) v += ld_cluster_f32(cluster_addr(p, k));
        }
        if (a.bias) v += __ldg(a.bias + m);
        y[static_cast<int64_t>(t) * a.M + m] = Elem<TY>::put(v);
    }
    if (splits > 1) cluster_sync_all();  // a rank's sums stay until every rank has read them
}

// ---- host ---------------------------------------------------------------------

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
    static const EncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

// Map of a [rows x cols] matrix of bytes with row stride ld, in boxes of
// box_rows x 128 bytes.
cudaError_t byte_map(CUtensorMap* m, const void* p, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
    EncodeFn fn = encode_fn();
    if (!fn) return cudaErrorNotSupported;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
    const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t steps[2] = {1, 1};
    CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, box, steps,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <typename... Params, typename... Args>
cudaError_t launch_cluster(void (*kernel)(Params...), int grid, int threads, int cluster, size_t smem, cudaStream_t s,
                           Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 0 ? 2 : 1;  // 0: the kernel's own __cluster_dims__
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
    return e == cudaSuccess ? cudaGetLastError() : e;
}

template <int BN, typename TY>
cudaError_t launch_pair(const F8Linear& l, F8Args a, cudaStream_t s) {
    constexpr int kStage = 128 * 128 + (BN / 2) * 128;
    CUtensorMap mx, mw;
    if (cudaError_t e = byte_map(&mx, l.x, l.N, l.K, l.x_ld, 128); e != cudaSuccess) return e;
    if (cudaError_t e = byte_map(&mw, l.w, l.M, l.K, l.w_ld, BN / 2); e != cudaSuccess) return e;
    a.tiles_n = static_cast<int>((l.N + 255) / 256);
    a.tiles_m = static_cast<int>((l.M + BN - 1) / BN);
    a.nbuf = 512 / BN;
    constexpr int kOut = 8 * kOutWarpBytes;
    a.stages = std::min(kMaxF8Stages, (224 * 1024 - 1024 - kOut) / kStage);
    static_assert(512 / BN <= (224 * 1024 - 1024 - kOut) / kStage, "an accumulator buffer needs a stage of its own");
    const int smem = a.stages * kStage + kOut + 1024;
    static std::atomic<int> cfg[64];
    if (cudaError_t e = ensure_dyn_smem(f8_pair_kernel<BN, TY>, smem, cfg); e != cudaSuccess) return e;
    const int64_t tiles = int64_t(a.tiles_n) * a.tiles_m;
    if (tiles >= (int64_t(1) << 31)) return cudaErrorInvalidValue;
    const int pairs = static_cast<int>(std::min<int64_t>(tiles, device_sm_count() / 2));
    return launch_cluster(f8_pair_kernel<BN, TY>, 2 * pairs, kPairThreads, 0, smem, s, mx, mw, a);
}

// Clusters of the skinny kernel: CTAs that split K so that about two per SM are
// at work, each with at least two blocks.
int skinny_splits(int64_t M, int nkb) {
    const int64_t tiles = (M + 127) / 128;
    int splits = 1;
    while (splits < 8 && tiles * splits * 2 <= 2 * device_sm_count() && splits * 4 <= nkb) splits *= 2;
    return splits;
}

template <int NT, typename TY, typename TX>
cudaError_t launch_skinny(const F8Linear& l, F8Args a, cudaStream_t s) {
    constexpr bool kPack = !std::is_void_v<TX>;
    constexpr int kStage = 128 * 128 + (kPack ? 0 : NT * 128);
    CUtensorMap mx, mw;
    if (cudaError_t e = byte_map(&mw, l.w, l.M, l.K, l.w_ld, 128); e != cudaSuccess) return e;
    if constexpr (kPack) {
        mx = mw;  // unused
        a.x = l.x;
        a.K = l.K;
        a.xvec = reinterpret_cast<uintptr_t>(l.x) % 16 == 0 && l.K * sizeof(TX) % 16 == 0;
    } else {
        if (cudaError_t e = byte_map(&mx, l.x, l.N, l.K, l.x_ld, NT); e != cudaSuccess) return e;
    }
    const int64_t tiles = (l.M + 127) / 128;
    const int splits = skinny_splits(l.M, a.nkb);
    const int per = (a.nkb + splits - 1) / splits;  // blocks of K of one CTA
    // two CTAs per SM, unless the scales of X take the room
    const int64_t own = (static_cast<int64_t>(per) * (NT * 4 + (kPack ? NT * 128 : 0)) + 127) / 128 * 128;
    int64_t budget = 110 * 1024 - 1024 - own;
    if (budget < 3 * kStage) budget = 224 * 1024 - 1024 - own;
    const int sums = (NT * 512 + kStage - 1) / kStage;  // stages that the sums take: NT x 128 floats
    const int64_t fit = budget < 0 ? 0 : budget / kStage;
    if (fit < std::max(2, sums)) {  // K so long that the scales of X fill shared memory
        if constexpr (kPack) return cudaErrorInvalidConfiguration;
        else return launch_pair<128, TY>(l, a, s);
    }
    a.stages = static_cast<int>(std::min<int64_t>({int64_t(kMaxF8Stages), int64_t(std::max({per, 2, sums})), fit}));
    const int smem = static_cast<int>(a.stages * kStage + own + 1024);
    static std::atomic<int> cfg[64];
    if (cudaError_t e = ensure_dyn_smem(f8_skinny_kernel<NT, TY, TX>, smem, cfg); e != cudaSuccess) return e;
    return launch_cluster(f8_skinny_kernel<NT, TY, TX>, static_cast<int>(tiles * splits), kSkinnyThreads, splits,
                          smem, s, mx, mw, a, splits);
}

F8Args args_of(const F8Linear& l) {
    F8Args a{};
    a.sx = l.x_scales;
    a.sw = l.w_scales;
    a.bias = l.bias;
    a.y = l.y;
    a.M = l.M;
    a.N = l.N;
    a.nkb = static_cast<int>((l.K + kF8Block - 1) / kF8Block);
    a.err = l.err;
    return a;
}

}  // namespace

// Few tokens whose K range of a CTA is at most 32 blocks: one round of loads,
// which cost less than a packing kernel (4096 x 4096: 6.6 against 8.4 us for one
// token); more rounds cost more (11008 x 4096, 16 tokens: 35 against 16 us).
bool f8_gemm_packs(int64_t M, int64_t K, int64_t N) {
    const int nkb = static_cast<int>((K + kF8Block - 1) / kF8Block);
    const int splits = skinny_splits(M, nkb);
    return N <= 16 && N * ((nkb + splits - 1) / splits) <= 32;
}

cudaError_t f8_gemm_unpacked_dispatch(const F8Linear& l, int x_dtype, cudaStream_t s) {
    const F8Args a = args_of(l);
    return with_dtype(x_dtype, [&](auto* xt) {
        using TX = std::remove_pointer_t<decltype(xt)>;
        return with_dtype(l.y_dtype, [&](auto* yt) {
            using TY = std::remove_pointer_t<decltype(yt)>;
            return launch_skinny<16, TY, TX>(l, a, s);
        });
    });
}

cudaError_t f8_gemm_dispatch(const F8Linear& l, cudaStream_t s) {
    const F8Args a = args_of(l);
    return with_dtype(l.y_dtype, [&](auto* tag) {
        using TY = std::remove_pointer_t<decltype(tag)>;
        if (l.N <= 16) return launch_skinny<16, TY, void>(l, a, s);
        if (l.N <= 32) return launch_skinny<32, TY, void>(l, a, s);
        if (l.N <= 64) return launch_skinny<64, TY, void>(l, a, s);
        // more tokens: the pair kernel is faster even where half of its 256 rows are padding (128 tokens: 28672 x 8192
        // 76 against 93 us, 4096 x 4096 18 against 32)
        const int64_t wide = (l.N + 255) / 256 * ((l.M + 255) / 256);
        return wide * 2 >= device_sm_count() ? launch_pair<256, TY>(l, a, s) : launch_pair<128, TY>(l, a, s);
    });
}

}  // namespace axq
