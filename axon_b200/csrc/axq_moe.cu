// Mixture-of-experts layer for a few tokens on packed expert weights:
//   ids, p = top_k of softmax(x . W_router^T)
//   y[t]   = sum_j p[t][j] * W_down[e] . (silu(W_gate[e] . x) * (W_up[e] . x)),
//            e = ids[t][j].
//
// It has to read the packed bytes of the experts that some token chose; each is
// read once per group of up to 8 of its tokens.  What bounds it is decoding them.
//
//  * moe_route_kernel: a cluster of 8 CTAs per 4 tokens splits the experts, its
//    first CTA picks the top_k (latency: 5 to 8 us, of loads, the cluster's
//    exchange and top_k rounds of warp maxima) and, if it has all tokens, makes the
//    plan: the tokens' choices sorted by expert, in groups.  Other clusters write
//    the records of x: per 256 elements one or two fp16 terms (x 2^-e = hi or ~ hi +
//    lo, 22 bits) in the order of the weights' MMA fragments, and sums for the
//    minimums.
//  * moe_prep_kernel: plan and records where the router's kernel did not make them,
//    and the records of the hidden activations.
//  * moe_expert_kernel: a producer warp streams packed rows through a ring of
//    shared-memory stages (bulk copies); eight consumer warps decode them into
//    exact fp16 fragments (axq_moe_decode.cuh) and multiply with mma.sync
//    m16n8k16, whose 8 columns are eight tokens or the two terms of four.  Runs
//    twice: gate and up (half of a unit's rows each, joined by silu), and down.  A
//    finisher warp joins the consumers' sums of a round beside the next one.
//    mma.sync and not tcgen05: the weights are decoded in registers, and with at
//    most 8 columns the tensor pipe is idle most of the time either way.  Bound by
//    the decoders' integer and fp16 instructions (3 per weight of Q4_K, 5.7 of
//    Q6_K, 5 of Q3_K) at 55 to 60 % of the issue rate, which 20 warps of 96
//    registers reach: 304 MB of Q4_K in 95 us (3.2 TB/s), 222 MB of Q6_K in 94 (fp32
//    results; 88 and 88 without the joins of kChain, before which the other figures
//    for four tokens in this file were taken), 114 MB of Q3_K in 72; 185 MB of e4m3,
//    which needs few instructions, in 39 (4.7 TB/s).  At 96 registers most kernels
//    spill a little, most of all Q6_K with two terms and two blocks of columns (168
//    bytes stored, 208 loaded; the limit of 96 is what two CTAs an SM leave).
//  * moe_combine_kernel: y from the experts' products, in the order of the
//    token's choices (no atomics on values: results do not depend on timing).
//    It, the plan and the hidden records take 2 to 5 us each, mostly their start.
//
// A form of three kernels for few choices, where every CTA made the plan and the
// last to finish a part wrote the hidden records and y, was no faster for one token
// (44.7 us) and slower for four (194 against 180): the counting of parts, with its
// fences, kept the finisher behind the consumers.
#include <algorithm>

#include "axq_common.cuh"
#include "axq_f8.cuh"
#include "axq_internal.h"
#include "axq_moe.cuh"
#include "axq_moe_decode.cuh"
#include "axq_ptx.cuh"
#include "axq_tc.cuh"

namespace axq {
namespace {

// ---- activation records -----------------------------------------------------------

// Record of one row and CG with T terms: eight lines (one for each pair of MMAs:
// [term][lane part][16 bytes]), the sums as two terms [2][lane part][8 bytes],
// the scale.
// The largest of the 256 is scaled to 2^8 .. 2^9 and fp16's smallest step is 2^-24, so
// every element is held to within 2^-33 of the largest.  Above that one term holds
// 16-bit activations: exactly down to 2^-25 (bf16) or 2^-22 (fp16) of the largest; two
// hold fp32 ones to 22 bits.
template <int T> constexpr int kRecSums = 512 * T;
template <int T> constexpr int kRecScale = kRecSums<T> + 64;
template <int T> constexpr int kRec = (kRecScale<T> + 4 + 63) / 64 * 64;
__host__ __device__ __forceinline__ int rec_bytes(int terms) { return terms == 1 ? kRec<1> : kRec<2>; }

// Two fp16 terms of v (already scaled): v = hi + lo within 2^-22 of it.
__device__ __forceinline__ void split2(float v, __half& hi, __half& lo) {
    hi = __float2half_rn(v);
    const float r = v - __half2float(hi);
    lo = __float2half_rn(isfinite(r) ? r : 0.0f);
}

// One warp: the record of 256 elements in s (shared memory, zero past the end)
// for weights of format fmt.
__device__ __forceinline__ void write_record(int fmt, int terms, const float* s, uint8_t* rec, int lane) {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(s[32 * j + lane]));
#pragma unroll
    for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
    // A power of two brings the largest element to [2^8, 2^9): fp16 then holds
    // sums of 32 elements, and terms down to 2^-33 of the largest.
    const int e = min(max(static_cast<int>(__float_as_uint(m) >> 23) - 127 - 8, -118), 118);
    const float up = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    const int mp = lane >> 2, i = lane & 3;
    __half hi[8], lo[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) split2(s[order_elem(fmt, 2 * mp + (k >> 2), i, k & 3)] * up, hi[k], lo[k]);
    uint4 a;
    memcpy(&a, hi, 16);
    *reinterpret_cast<uint4*>(rec + mp * 64 * terms + i * 16) = a;
    if (terms == 2) {
        memcpy(&a, lo, 16);
        *reinterpret_cast<uint4*>(rec + mp * 128 + 64 + i * 16) = a;
    }
    const int sums = order_sums(fmt), at = 512 * terms;
    if (sums && lane < 16) {  // lane part lane / 4, slot lane % 4
        const int n = 256 / sums, sb = order_sum(fmt, lane >> 2, lane & 3);
        float v = 0.0f;
        if (sb >= 0) {
            for (int k = 0; k < n; ++k) {
                const float x = s[sb * n + ((k + lane) & (n - 1))] * up;
                // what the codes are multiplied with: with one term, its rounding
                v += terms == 2 ? x : __half2float(__float2half_rn(x));
            }
        }
        __half h, l;
        split2(v, h, l);
        reinterpret_cast<__half*>(rec + at)[lane] = h;
        reinterpret_cast<__half*>(rec + at + 32)[lane] = l;
    }
    if (lane == 0) *reinterpret_cast<float*>(rec + at + 64) = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}

// Records of rows of x (or of the hidden activations).
struct RecordArgs {
    int fmt, terms;
    int64_t rows, cols;
    int ncg;
    uint8_t* rec;
    const int* need;  // rows whose expert id is out of range are skipped; null: none
    int experts;
};

// Record `it` (row-major over rows and CGs) by one warp, through its 256 floats.
template <typename T>
__device__ __forceinline__ void record_of(const RecordArgs& a, const T* x, int64_t it, float* buf, int lane) {
    if (it >= a.rows * a.ncg) return;
    const int64_t r = it / a.ncg;
    const int cg = static_cast<int>(it - r * a.ncg);
    if (a.need && static_cast<unsigned>(a.need[r]) >= static_cast<unsigned>(a.experts)) return;
    const int64_t k0 = static_cast<int64_t>(cg) * 256;
    const T* xr = x + r * a.cols;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int64_t k = k0 + 32 * j + lane;
        buf[32 * j + lane] = k < a.cols ? Elem<T>::get(xr[k]) : 0.0f;
    }
    __syncwarp();
    write_record(a.fmt, a.terms, buf, a.rec + it * rec_bytes(a.terms), lane);
}

constexpr int kPrepWarps = 8;

// Records of all rows; block 0 also makes the plan when ids are given.
template <typename T>
__global__ void __launch_bounds__(32 * kPrepWarps) moe_prep_kernel(const T* __restrict__ x, RecordArgs a, MoePlan plan) {
    __shared__ float buf[kPrepWarps][256];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_launch_dependents();
    if (plan.ids && blockIdx.x == 0) {
        moe_make_plan<32 * kPrepWarps>(plan);
        return;
    }
    const int64_t b = blockIdx.x - (plan.ids ? 1 : 0);
    record_of(a, x, b * kPrepWarps + warp, buf[warp], lane);
}

// ---- router ---------------------------------------------------------------------

constexpr int kRouteCtas = 8, kRouteWarps = 16, kRouteTokens = 4;

__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// The top_k of a token of the cluster, by one warp.  Logits become keys whose order
// as integers is theirs (NaN 1, chosen ones 0); lane e % 32 holds the best of its own.
__device__ __forceinline__ void route_token(float* logits, int* ids, float* wt, int token, int lane, int experts, int top_k,
                                            int slices, int normalize) {
    uint32_t* keys = reinterpret_cast<uint32_t*>(logits) + token * experts;
    uint32_t best = 0;
    int best_e = INT32_MAX;
    for (int e = lane; e < experts; e += 32) {
        const float* l = logits + token * experts + e;
        float v = l[0];
        for (int sl = 1; sl < slices; ++sl) v += l[sl * kRouteTokens * experts];
        const uint32_t b = __float_as_uint(v);
        const uint32_t k = isnan(v) ? 1u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
        keys[e] = k;
        if (k > best) {
            best = k;
            best_e = e;
        }
    }
    auto value = [](uint32_t k) {
        return k == 1u ? __uint_as_float(0x7FFFFFFFu) : __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k);
    };
    float mine = 0.0f, sum = 0.0f, mx = 0.0f;
    int my_id = 0;
    if (!normalize) {  // the sum over all experts, before the chosen ones are marked
        mx = value(__reduce_max_sync(0xFFFFFFFFu, best));
        for (int e = lane; e < experts; e += 32) sum += expf(value(keys[e]) - mx);
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    }
    for (int j = 0; j < top_k; ++j) {
        const uint32_t m = __reduce_max_sync(0xFFFFFFFFu, best);
        const int e = __reduce_min_sync(0xFFFFFFFFu, best == m ? best_e : INT32_MAX);  // ties: the lowest index
        if (j == 0) mx = value(m);
        const float p = expf(value(m) - mx);
        if (normalize) sum += p;
        if (lane == j) {
            mine = p;
            my_id = e;
        }
        if (lane == (e & 31)) {
            keys[e] = 0;
            best = 0;
            best_e = INT32_MAX;
            for (int q = lane; q < experts; q += 32)
                if (keys[q] > best) {
                    best = keys[q];
                    best_e = q;
                }
        }
        __syncwarp();
    }
    if (lane < top_k) {
        ids[lane] = my_id;
        wt[lane] = mine / sum;
    }
}

// Logits in fp32 (FMAs over lanes of 128 columns, then a tree over the lanes,
// then the slices in order); ties go to the lowest index, NaN logits are chosen
// last.  The cluster's 128 warps take (expert, slice of the columns) each:
// latency counts here, so few experts are cut into slices.
template <typename T>
__global__ void __cluster_dims__(kRouteCtas, 1, 1) __launch_bounds__(32 * kRouteWarps)
    moe_route_kernel(const T* __restrict__ x, const float* __restrict__ w, int* ids, float* wt,
                     int64_t tokens, int experts, int top_k, int64_t hidden, int slices, int normalize, bool vec,
                     RecordArgs records, MoePlan plan) {
    extern __shared__ float logits[];  // [slice][kRouteTokens][experts], of the cluster's first CTA
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int64_t t0 = static_cast<int64_t>(blockIdx.x / kRouteCtas) * kRouteTokens;
    if (t0 >= tokens) {
        // clusters past the tokens': the layer's activation records, which do not wait for the choice of experts
        __shared__ float buf[kRouteWarps][256];
        const int first = static_cast<int>((tokens + kRouteTokens - 1) / kRouteTokens) * kRouteCtas;
        const int b = static_cast<int>(blockIdx.x) - first;
        pdl_wait();
        pdl_launch_dependents();
        record_of(records, x, static_cast<int64_t>(b) * kRouteWarps + warp, buf[warp], lane);
        return;
    }
    const int nt = static_cast<int>(min64(kRouteTokens, tokens - t0));
    cluster_arrive();  // waited for before the first store to the first CTA's shared memory
    pdl_wait();
    pdl_launch_dependents();
    bool there = false;
    const int64_t per = ((hidden + slices - 1) / slices + 127) / 128 * 128;  // columns of a slice
    for (int o = static_cast<int>(rank) * kRouteWarps + warp; o < experts * slices; o += kRouteCtas * kRouteWarps) {
        const int e = o / slices, sl = o - e * slices;
        const int64_t k0 = sl * per, k1 = min64(k0 + per, hidden);
        float acc[kRouteTokens] = {};
        const float* we = w + static_cast<int64_t>(e) * hidden;
        const T* xt = x + t0 * hidden;
        if (vec) {
#pragma unroll 4
            for (int64_t k = k0 + 4 * lane; k < k1; k += 128) {
                const float4 a = __ldg(reinterpret_cast<const float4*>(we + k));
#pragma unroll
                for (int t = 0; t < kRouteTokens; ++t) {
                    if (t < nt) {
                        const T* xp = xt + t * hidden + k;
                        float v[4];
                        if constexpr (sizeof(T) == 4) {
                            const float4 b = __ldg(reinterpret_cast<const float4*>(xp));
                            v[0] = b.x; v[1] = b.y; v[2] = b.z; v[3] = b.w;
                        } else {
                            const uint2 b = __ldg(reinterpret_cast<const uint2*>(xp));
                            T h[4];
                            memcpy(h, &b, 8);
#pragma unroll
                            for (int i = 0; i < 4; ++i) v[i] = Elem<T>::get(h[i]);
                        }
                        acc[t] = fmaf(a.x, v[0], fmaf(a.y, v[1], fmaf(a.z, v[2], fmaf(a.w, v[3], acc[t]))));
                    }
                }
            }
        } else {
            for (int64_t k = k0 + lane; k < k1; k += 32)
#pragma unroll
                for (int t = 0; t < kRouteTokens; ++t)
                    if (t < nt) acc[t] = fmaf(we[k], Elem<T>::get(xt[t * hidden + k]), acc[t]);
        }
        if (!there) cluster_wait();
        there = true;
#pragma unroll
        for (int t = 0; t < kRouteTokens; ++t) {
            if (t >= nt) break;
#pragma unroll
            for (int d = 16; d; d >>= 1) acc[t] += __shfl_xor_sync(0xFFFFFFFFu, acc[t], d);
            if (lane == 0)
                st_cluster_f32(cluster_addr(logits + (sl * kRouteTokens + t) * experts + e, 0), acc[t]);
        }
    }
    if (!there) cluster_wait();
    cluster_sync_all();
    if (rank != 0) return;
    if (warp < nt) route_token(logits, ids + (t0 + warp) * top_k, wt + (t0 + warp) * top_k, warp, lane, experts, top_k, slices, normalize);
    if (!plan.ids) return;  // else this is the only cluster with tokens
    __syncthreads();
    moe_make_plan<32 * kRouteWarps>(plan);
}

// ---- experts -------------------------------------------------------------------------

constexpr int kConsumers = 8;
constexpr int kMoeThreads = (kConsumers + 2) * 32;  // and the producer and the finisher
constexpr int kMoeStages = 8;  // most
// The rounds a CTA has named to its warps and not all of them have done with: one
// for each stage at most, one being named, three by which the finisher lags.
constexpr int kMoeNamed = 16;
static_assert(kMoeStages + 4 < kMoeNamed);
constexpr int kMoeGroup = 8;  // tokens of a group, at most

struct MoeBars {
    uint64_t full[kMoeStages], empty[kMoeStages];
    uint64_t sums[2], joined[2];  // a round's partial sums are written, and joined
    uint64_t named[kMoeNamed];    // the q-th round of this CTA is at q % kMoeNamed:
    int4 round[kMoeNamed];        // expert, tokens, group (-1: no more), first unit
    int2 entry[kMoeNamed][kMoeGroup];
    int abort;
};

struct ExpertArgs {
    const uint8_t* w[2];   // tile 0's and tile 1's matrix
    const float* sc[2];    // e4m3: their scales
    int64_t w_bytes;       // bytes of each (all experts)
    int64_t rb;            // bytes from row to row
    int64_t rows;          // rows of an expert
    int64_t row_bytes;     // packed bytes of a row
    int ncg, nblk;         // CGs and (32- or 128-element) blocks of a row
    int gate_up;           // tile 1 is `up` and the result silu(tile 0) * tile 1; else tile 1 follows tile 0
    int tiles;             // units of an expert
    int slots, wps;        // units a stage holds, warps (and CGs of a stage) per unit: slots * wps = 8
    int rs, stage_bytes, stages;
    const uint8_t* rec;    // activation records
    int64_t rec_row;       // bytes of a record row
    int rec_token;         // a pair's record row is its token's, else its own
    float* out;            // [pair][rows]
    int* next;             // rounds taken beyond the first of each CTA
    MoePlan plan;
    int* err;
};
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Compile-time loop over MMA pairs 0..7.
template <class Fn, int... Js>
__device__ __forceinline__ void each_pair_impl(Fn&& f, std::integer_sequence<int, Js...>) {
    (f(std::integral_constant<int, Js>{}), ...);
}
template <class Fn>
__device__ __forceinline__ void each_pair(Fn&& f) {
    each_pair_impl(f, std::make_integer_sequence<int, 8>{});
}

// The same for 0 .. N - 1.
template <int N, class Fn>
__device__ __forceinline__ void static_for_pairs(Fn&& f) {
    each_pair_impl(f, std::make_integer_sequence<int, N>{});
}

// Sums of codes of one tile's CG over one pair of MMAs.
template <int F, int MP, int NB>
__device__ __forceinline__ void moe_pair(MoeRow<F> (&r)[2], const uint4 (&b)[NB], float (&acc)[NB][4]) {
    uint32_t x[4], y[4];
    if constexpr (F == F_Q6_K) {
        uint32_t xh[4], yh[4];
        r[0].template pair<MP>(x, xh);
        r[1].template pair<MP>(y, yh);
        const uint32_t h0[4] = {xh[0], yh[0], xh[1], yh[1]}, h1[4] = {xh[2], yh[2], xh[3], yh[3]};
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            mma16816(acc[n], h0, b[n].x, b[n].y);
            mma16816(acc[n], h1, b[n].z, b[n].w);
        }
    } else {
        r[0].template pair<MP>(x);
        r[1].template pair<MP>(y);
    }
    const uint32_t a0[4] = {x[0], y[0], x[1], y[1]}, a1[4] = {x[2], y[2], x[3], y[3]};
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        mma16816(acc[n], a0, b[n].x, b[n].y);
        mma16816(acc[n], a1, b[n].z, b[n].w);
    }
}

// Scales of a block of rows g and g + 8 where they are per block.
template <int F>
__device__ __forceinline__ float2 block_scales(const MoeRow<F> (&r)[2], const float* w) {
    if constexpr (F == F_F8) {
        const float d = __ldg(w);
        return make_float2(d, d);
    } else if constexpr (F == F_Q8_0 || F == F_Q4_0) {
        return make_float2(r[0].d(), r[1].d());
    } else {
        return make_float2(0.0f, 0.0f);
    }
}

// Columns of an MMA with T terms: column c is term c % T of token c / T.  A lane
// reads column g = lane / 4 of B and holds columns 2 i and 2 i + 1 of the sums:
// two tokens, or the two terms of one.
template <int T>
struct Cols {
    static constexpr int kTokens = 8 / T;  // of a block of columns
    static constexpr int kOwn = 2 / T;     // of a lane's sums
    __device__ __forceinline__ static int token(int g) { return g / T; }
    __device__ __forceinline__ static int own(int i, int u) { return kOwn * i + u; }
    __device__ __forceinline__ static int offset(int g, int i) { return (T == 2 ? (g & 1) * 64 : 0) + i * 16; }
    // the lane's sums of row r (0: g, 1: g + 8)
    __device__ __forceinline__ static float sum(const float (&c)[4], int r, int u) {
        return T == 2 ? c[2 * r] + c[2 * r + 1] : c[2 * r + u];
    }
};

// Lines of the activation record loaded ahead of their use, as far as the
// format's registers allow; the first are loaded before the wait for the stage.
// e4m3, whose decoder needs next to none, holds all eight of a CG for both tiles.
template <int F, int NB>
constexpr int kAhead = (F == F_F8 ? 8 : F == F_Q8_0 || F == F_Q4_0 ? 3 : 2) / NB;

template <int F, int T, int NB>
struct ActLines {
    uint4 b[NB][kAhead<F, NB> + 1];
    template <int MP>
    __device__ __forceinline__ void load(const uint8_t* const (&rec)[NB]) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
            b[n][MP % (kAhead<F, NB> + 1)] = __ldg(reinterpret_cast<const uint4*>(rec[n] + MP * 64 * T));
    }
};

// Pairs of MMAs whose sums follow one another in the tensor core before fp32
// registers take them.  Its additions truncate, always toward zero, so a long chain
// loses bits: fp32 layers of 256-element formats were 1 to 2.4e-6 off with all 16 or
// (Q6_K) 32 MMAs of a CG in one chain, up to 1.3e-6 with half of it, 0.8 with a
// quarter, 0.64 with an eighth, where fp32 alone gives 0.2 to 1.6.  EX, for results in
// fp32: four MMAs (Q4_K / Q6_K, 4 tokens: 173 -> 183 us; Q3_K / Q5_K, 33 tokens, whose
// two blocks of columns leave few registers: 143 -> 166); results of 16 bits show none
// of it.
template <int F, bool EX>
constexpr int kChain = !EX ? 8 : F == F_Q6_K ? 1 : 2;

// One CG of TL tiles (rows g and g + 8 of tile t at p[t][0], p[t][1]) times NB
// blocks of eight columns: tot[t][n][r][u] += row r's product with this lane's
// u-th token of block n (see Cols).
// Tiles taken together share the loads of the activations, whose first kAhead
// lines are in `x`.
template <int F, int T, int NB, bool EX, int TL>
__device__ __forceinline__ void moe_cg(const uint8_t* const (*p)[2], int g, int i, const uint8_t* const (&rec)[NB],
                                       ActLines<F, T, NB>& x, const float (&xs)[NB][Cols<T>::kOwn], int blocks,
                                       const float* const* wsc, float (*tot)[NB][2][Cols<T>::kOwn]) {
    using C = Cols<T>;
    constexpr int kPairs = kChain<F, EX>;
    MoeRow<F> r[TL][2];
    float acc[TL][NB][4];
    [[maybe_unused]] float part[TL][NB][4];  // the chain of MMAs at work
#pragma unroll
    for (int t = 0; t < TL; ++t) {
        r[t][0].load(p[t][0], i);
        r[t][1].load(p[t][1], i);
#pragma unroll
        for (int n = 0; n < NB; ++n) acc[t][n][0] = acc[t][n][1] = acc[t][n][2] = acc[t][n][3] = 0.0f;
    }
    each_pair([&](auto MPc) {
        constexpr int MP = decltype(MPc)::value;
        constexpr int D = kAhead<F, NB>;
        if constexpr (MP + D < 8) x.template load<MP + D>(rec);
        uint4 b[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) b[n] = x.b[n][MP % (D + 1)];
#pragma unroll
        for (int t = 0; t < TL; ++t) {
            if constexpr (kPairs < 8) {
                if constexpr (MP % kPairs == 0)
#pragma unroll
                    for (int n = 0; n < NB; ++n) part[t][n][0] = part[t][n][1] = part[t][n][2] = part[t][n][3] = 0.0f;
                moe_pair<F, MP, NB>(r[t], b, part[t]);
                if constexpr (MP % kPairs == kPairs - 1)
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int k = 0; k < 4; ++k) acc[t][n][k] += part[t][n][k];
            } else {
                moe_pair<F, MP, NB>(r[t], b, acc[t]);
            }
            if constexpr (F == F_Q8_0 || F == F_Q4_0 || (F == F_F8 && MP % 4 == 3)) {
                // a block is done: its scales in fp32 (blocks past the row's end hold other rows' bytes)
                constexpr int B = F == F_F8 ? MP / 4 : MP;
                if (B < blocks) {
                    const float2 d = block_scales<F>(r[t], wsc[t] + B);
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int u = 0; u < C::kOwn; ++u) {
                            tot[t][n][0][u] = fmaf(xs[n][u] * d.x, C::sum(acc[t][n], 0, u), tot[t][n][0][u]);
                            tot[t][n][1][u] = fmaf(xs[n][u] * d.y, C::sum(acc[t][n], 1, u), tot[t][n][1][u]);
                        }
                }
#pragma unroll
                for (int n = 0; n < NB; ++n) acc[t][n][0] = acc[t][n][1] = acc[t][n][2] = acc[t][n][3] = 0.0f;
            }
        }
    });
    if constexpr (Order<F>::SUMS > 0) {
        // the sums of this lane's column and part: with one term the two terms of a sum are two MMAs
        uint2 b[NB], bl[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const uint8_t* q = rec[n] + (kRecSums<T> - C::offset(g, i)) + (T == 2 ? (g & 1) * 32 : 0) + i * 8;
            b[n] = __ldg(reinterpret_cast<const uint2*>(q));
            if constexpr (T == 1) bl[n] = __ldg(reinterpret_cast<const uint2*>(q + 32));
        }
#pragma unroll
        for (int t = 0; t < TL; ++t) {
            uint32_t m0[2], m1[2];
            r[t][0].mins(m0);
            r[t][1].mins(m1);
            const uint32_t a[4] = {m0[0], m1[0], m0[1], m1[1]};
            const float2 s0 = r[t][0].scales(), s1 = r[t][1].scales();
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                mma16816(c, a, b[n].x, b[n].y);
                if constexpr (T == 1) mma16816(c, a, bl[n].x, bl[n].y);
#pragma unroll
                for (int u = 0; u < C::kOwn; ++u) {
                    tot[t][n][0][u] =
                        fmaf(xs[n][u], fmaf(s0.x, C::sum(acc[t][n], 0, u), -s0.y * C::sum(c, 0, u)), tot[t][n][0][u]);
                    tot[t][n][1][u] =
                        fmaf(xs[n][u], fmaf(s1.x, C::sum(acc[t][n], 1, u), -s1.y * C::sum(c, 1, u)), tot[t][n][1][u]);
                }
            }
        }
    }
}

// Tiles of a unit that a stage holds and a warp takes at once: both where the
// decoder's state of four rows fits the registers and two stages of them fit
// half an SM's shared memory, else one after the other.
template <int F, int NB>
constexpr int kStageTiles = NB == 1 && (F == F_Q4_K || F == F_Q4_0) ? 2 : 1;
// Tiles of a unit.  Two hold 16 rows of gate and 16 of up, or 32 rows of down; one
// 8 and 8, or 16.  The smaller unit shares the SMs better (Q6_K, four tokens: 173
// against 180 us for the layer); the larger one lets its tiles share the
// activations, where they are taken together or stay in registers.
template <int F, int NB>
constexpr int kUnitTiles = F == F_F8 ? 2 : kStageTiles<F, NB>;
// Rows whose packed length is a multiple of 16 start on one.
template <int F>
constexpr bool kAlignedRows = F == F_Q4_K || F == F_Q5_K || F == F_F8;

// Bounded wait of a whole warp (see MoeBars::abort).
__device__ __forceinline__ bool moe_wait(uint64_t* bar, uint32_t parity, MoeBars* b, int* err) {
    bool ok = mbar_try_wait(bar, parity);
    if (__builtin_expect(!ok, 0)) ok = mbar_wait_bounded(bar, parity, &b->abort);
    ok = __all_sync(0xFFFFFFFFu, ok);
    if (__builtin_expect(!ok, 0)) {
        *const_cast<volatile int*>(&b->abort) = 1;
        atomicExch(err, 1);
    }
    return ok;
}

// sum_j p[t][j] z[t top_k + j][c], j in order; ids out of range add nothing.
// Loads of four choices are in flight together (z has a row for every choice,
// written or not).
__device__ __forceinline__ float moe_combined(const float* z, const int* ids, const float* wt, int64_t t, int64_t c,
                                              int64_t hidden, int top_k, int experts) {
    float v = 0.0f;
    for (int j0 = 0; j0 < top_k; j0 += 4) {
        int id[4];
        float w[4], x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t p = t * top_k + min(j0 + j, top_k - 1);
            id[j] = j0 + j < top_k ? __ldg(ids + p) : -1;
            w[j] = __ldg(wt + p);
            x[j] = __ldcg(z + p * hidden + c);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (static_cast<unsigned>(id[j]) < static_cast<unsigned>(experts)) v = fmaf(w[j], x[j], v);
    }
    return v;
}

// Row (of the expert) of tile `tile` and row r of unit `unit`.
template <int UT>
__device__ __forceinline__ int64_t stage_row(const ExpertArgs& a, int unit, int tile, int r) {
    return a.gate_up ? static_cast<int64_t>(unit) * (8 * UT) + (UT == 1 ? r & 7 : r)
                     : static_cast<int64_t>(unit) * (16 * UT) + 16 * tile + r;
}

// A round: `slots` units of one group, from unit t0.
struct MoeRound {
    int expert, tokens, grp, t0;
    const int2* entries;
};
// The CTA's q-th round; grp < 0: there is none.
__device__ __forceinline__ MoeRound moe_round(MoeBars& bars, int q, int* err) {
    const int at = q % kMoeNamed;
    if (!moe_wait(&bars.named[at], (q / kMoeNamed) & 1, &bars, err)) return MoeRound{0, 0, -1, 0, nullptr};
    const int4 r = bars.round[at];
    return MoeRound{r.x, r.y, r.z, r.w, bars.entry[at]};
}

// Joins the warps' partial sums (rb) of a round and writes its results (one warp).
template <int kTok, int UT>
__device__ __forceinline__ void moe_results(const ExpertArgs& a, const float* rb, const MoeRound& rd, int lane) {
    const int rs = (a.gate_up ? 2 : 3) + UT;  // log2 of a unit's rows
    const int outputs = rd.tokens << rs;         // of a unit
    for (int un = 0; un < a.slots && rd.t0 + un < a.tiles; ++un) {
        for (int o = lane; o < outputs; o += 32) {
            const int rr = o & ((1 << rs) - 1), t = o >> rs;
            const int64_t row = (static_cast<int64_t>(rd.t0 + un) << rs) + rr;
            // the warps' parts are loaded together and added in order
            float part[2][kConsumers];
            const float* q = rb + (un * a.wps * UT * kTok + t) * 16 + (rr >> 4) * kTok * 16 + (rr & 15);
            const int up = UT == 2 ? kTok * 16 : 8;  // from a row of gate to that of up
#pragma unroll
            for (int w = 0; w < kConsumers; ++w) {
                part[0][w] = w < a.wps ? q[w * UT * kTok * 16] : 0.0f;
                part[1][w] = a.gate_up && w < a.wps ? q[w * UT * kTok * 16 + up] : 0.0f;
            }
            float v[2] = {0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < kConsumers; ++w) {
                v[0] += part[0][w];
                v[1] += part[1][w];
            }
            const float z = a.gate_up ? v[0] / (1.0f + expf(-v[0])) * v[1] : v[0];
            if (row < a.rows) a.out[static_cast<int64_t>(rd.entries[t].x) * a.rows + row] = z;
        }
    }
}

template <int F, int T, int NB, bool EX>
__global__ void __launch_bounds__(kMoeThreads, 2) moe_expert_kernel(const __grid_constant__ ExpertArgs a) {
    using C = Cols<T>;
    constexpr int CGB = moe_cg_bytes<F>();
    constexpr int kTok = C::kTokens * NB;
    constexpr int TL = kStageTiles<F, NB>, UT = kUnitTiles<F, NB>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = smem_raw + ((128 - (smem_u32(smem_raw) & 127)) & 127);
    float* red = reinterpret_cast<float*>(ring + a.stages * a.stage_bytes);  // the warps' sums of two rounds
    __shared__ MoeBars bars;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kMoeStages; ++s) {
            mbar_init(&bars.full[s], 1);
            mbar_init(&bars.empty[s], kConsumers);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&bars.sums[s], kConsumers);
            mbar_init(&bars.joined[s], 1);
        }
        for (int s = 0; s < kMoeNamed; ++s) mbar_init(&bars.named[s], 1);
        bars.abort = 0;
        fence_mbar_init();
    }
    __syncthreads();
    // The producer of the down product starts before the records of the hidden activations are there: the kernel that
    // writes them lets this one start only after gate and up have finished, and those began after the plan was made.
    if (a.gate_up || warp != kConsumers) {
        pdl_wait();
        pdl_launch_dependents();
    }
    const int ksteps = (a.ncg + a.wps - 1) / a.wps;

    if (warp == kConsumers) {
        const uint64_t policy = l2_evict_first_policy();
        int s = 0;
        uint32_t par = 0;
        bool ok = true;
        int64_t issued = 0;
        constexpr int kMost = TL == 2 ? 4 : 2;  // rows of a stage that a lane copies, at most (four slots)
        const int srows = a.slots * 16 * TL;
        // A CTA's share of the rounds, rounded down, is consecutive (mostly of one group, whose activations stay in L1);
        // the rest are taken by whoever is free, their numbers asked for a round ahead.  All of them shared out
        // beforehand left SMs idle (194 against 173 us for four tokens); three quarters beforehand, the rest taken: 180.
        const int per = (a.tiles + a.slots - 1) / a.slots;  // rounds of a group; all fit 32 bits (checked on the host)
        const int rounds = __ldcg(a.plan.ngroups) * per;
        const int own = max(1, rounds / static_cast<int>(gridDim.x));
        int n = blockIdx.x * own;
        for (int q = 0; ok; ++q) {
            const int at = q % kMoeNamed;
            if (n >= rounds) {
                if (lane == 0) {
                    bars.round[at] = make_int4(0, 0, -1, 0);
                    mbar_arrive(&bars.named[at]);
                }
                break;
            }
            int after = n + 1;
            if (q + 1 >= own && lane == 0) after = static_cast<int>(gridDim.x) * own + atomicAdd(a.next, 1);
            const int grp = n / per;
            const int4 gd = __ldcg(a.plan.groups + grp);  // expert, first entry, number of entries
            const MoeRound rd{gd.x, gd.z, grp, (n - grp * per) * a.slots, nullptr};
            if (lane < gd.z) bars.entry[at][lane] = __ldcg(a.plan.entries + gd.y + lane);
            if (lane == 0) bars.round[at] = make_int4(rd.expert, rd.tokens, grp, rd.t0);
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.named[at]);
            // where this lane's rows of a stage begin (of tile 0, if a stage holds one tile); -1: no such row
            const int64_t expert = rd.expert;
            int64_t at0[kMost];
#pragma unroll
            for (int j = 0; j < kMost; ++j) {
                const int sr = lane + 32 * j, u = sr / (16 * TL), r = sr & (16 * TL - 1);
                const int64_t row = stage_row<UT>(a, rd.t0 + u, TL == 2 ? r >> 4 : 0, r & 15);
                at0[j] = sr < srows && rd.t0 + u < a.tiles && row < a.rows ? (expert * a.rows + row) * a.rb : -1;
            }
            for (int step = 0; step < ksteps * (UT / TL); ++step) {
                const int k = step / (UT / TL), tile = step & (UT / TL - 1);
                // the matrix of row sr of the stage (both are the same for the down product)
                auto matrix = [&](int sr) { return a.w[UT == 1 ? (sr >> 3) & 1 : TL == 2 ? (sr >> 4) & 1 : tile]; };
                // tile 1 of the down product is 16 rows on, and may lie past the last row
                const int64_t skip = tile && !a.gate_up ? 16 * a.rb : 0;
                const int64_t end = (expert + 1) * a.rows * a.rb;
                const int64_t off = static_cast<int64_t>(k) * a.wps * CGB;
                const int64_t seg = min64(static_cast<int64_t>(a.wps) * CGB, a.row_bytes - off);
                ok = moe_wait(&bars.empty[s], par ^ 1, &bars, a.err);
                if (!ok) break;
                uint8_t* st = ring + s * a.stage_bytes;
                // The bytes come from the 16-byte rounded range around a row's segment.
                uint32_t tx = 0, len[kMost];
#pragma unroll
                for (int j = 0; j < kMost; ++j) {
                    len[j] = 0;
                    const int64_t at = at0[j] + skip + off;
                    if (at0[j] < 0 || at0[j] + skip >= end) continue;
                    const int64_t from = at & ~int64_t(15), to = (at + seg + 15) & ~int64_t(15);
                    const int sr = lane + 32 * j;
                    if (to <= a.w_bytes) {
                        tx += len[j] = static_cast<uint32_t>(to - from);
                    } else {  // the rounded end would leave the buffer: bytes one by one
                        const uint8_t* src = matrix(sr) + at;
                        uint8_t* dst = st + sr * a.rs + (at & 15);
                        for (int64_t c = 0; c < seg; ++c) dst[c] = src[c];
                    }
                }
                tx = __reduce_add_sync(0xFFFFFFFFu, tx);
                __syncwarp();  // bytes copied by lanes come before the arrival
                if (lane == 0) mbar_arrive_expect_tx(&bars.full[s], tx);
                __syncwarp();
#pragma unroll
                for (int j = 0; j < kMost; ++j) {
                    const int sr = lane + 32 * j;
                    if (len[j])
                        bulk_g2s_hint(st + sr * a.rs, matrix(sr) + ((at0[j] + skip + off) & ~int64_t(15)), len[j],
                                      &bars.full[s], policy);
                }
                ++issued;
                if (++s == a.stages) {
                    s = 0;
                    par ^= 1;
                }
            }
            n = __shfl_sync(0xFFFFFFFFu, after, 0);
        }
        if (!ok)  // copies still in flight land before the shared memory goes away
            for (int64_t i = max(int64_t(0), issued - a.stages); i < issued; ++i)
                mbar_wait_bounded(&bars.full[i % a.stages], static_cast<uint32_t>((i / a.stages) & 1));
        return;
    }

    constexpr int kSums = kConsumers * UT * kTok * 16;  // [warp][tile][token][16 rows]
    if (warp > kConsumers) {
        // The finisher joins each round's sums beside the consumers, which go on; it needs no registers that the SM has
        // not left over (18 and 20 warps share its schedulers alike).
        for (int q = 0;; ++q) {
            const MoeRound rd = moe_round(bars, q, a.err);
            if (rd.grp < 0 || !moe_wait(&bars.sums[q & 1], (q >> 1) & 1, &bars, a.err)) break;
            moe_results<kTok, UT>(a, red + (q & 1) * kSums, rd, lane);
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.joined[q & 1]);
        }
        return;
    }

    const int g = lane >> 2, i = lane & 3;
    const int u = warp / a.wps, col = warp - u * a.wps;
    int s = 0;
    uint32_t par = 0;
    bool ok = true;
    for (int q = 0;; ++q) {
        const MoeRound rd = moe_round(bars, q, a.err);
        if (rd.grp < 0) break;
        const int unit = rd.t0 + u;
        // this lane's B column, and the scales of its sums' columns (columns past the group's end: its first token's)
        const uint8_t *rec0[NB], *scale0[NB][C::kOwn];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const int t = n * C::kTokens + C::token(g);
            const int2 e = rd.entries[t < rd.tokens ? t : 0];
            rec0[n] = a.rec + (a.rec_token ? e.y : e.x) * a.rec_row + C::offset(g, i);
#pragma unroll
            for (int v = 0; v < C::kOwn; ++v) {
                const int ts = n * C::kTokens + C::own(i, v);
                const int2 es = rd.entries[ts < rd.tokens ? ts : 0];
                scale0[n][v] = a.rec + (a.rec_token ? es.y : es.x) * a.rec_row + kRecScale<T>;
            }
        }
        float tot[UT][NB][2][C::kOwn];
#pragma unroll
        for (int t = 0; t < UT; ++t)
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int v = 0; v < C::kOwn; ++v) tot[t][n][0][v] = tot[t][n][1][v] = 0.0f;
        const int64_t row0 = rd.expert * a.rows + stage_row<UT>(a, unit, 0, 0);
        for (int k = 0; k < ksteps; ++k) {
            const int cg = k * a.wps + col;
            const bool mine = cg < a.ncg && unit < a.tiles;
            const uint8_t* rec[NB];
            float xs[NB][C::kOwn];
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const int64_t at = static_cast<int64_t>(mine ? cg : 0) * kRec<T>;
                rec[n] = rec0[n] + at;
#pragma unroll
                for (int v = 0; v < C::kOwn; ++v) xs[n][v] = __ldg(reinterpret_cast<const float*>(scale0[n][v] + at));
            }
            // bytes of the first row's segment past a multiple of 16 (low bits suffice)
            const uint32_t ph0 = kAlignedRows<F> ? 0u : static_cast<uint32_t>(row0) * static_cast<uint32_t>(a.rb) +
                                                            static_cast<uint32_t>(k * a.wps) * CGB;
            // e4m3: scales of the unit's rows (16 or 32 rows from a multiple of 16, so one block of 128)
            const int64_t sc0 = F == F_F8 ? min64(row0, (rd.expert + 1) * a.rows - 1) / 128 * a.nblk + 2 * cg : 0;
            const int blocks = a.nblk - (F == F_F8 ? 2 : 8) * cg;
            ActLines<F, T, NB> x;
#pragma unroll
            for (int h = 0; h < UT / TL; ++h) {
                if (h == 0 || kAhead<F, NB> < 8)
                    static_for_pairs<kAhead<F, NB>>([&](auto J) { x.template load<decltype(J)::value>(rec); });
                if (ok) ok = moe_wait(&bars.full[s], par, &bars, a.err);
                if (ok && mine) {
                    const uint8_t* st = ring + s * a.stage_bytes + u * (16 * TL) * a.rs + col * CGB;
                    const uint8_t* p[TL][2];
                    const float* wsc[TL];  // e4m3, whose units have two tiles
#pragma unroll
                    for (int t = 0; t < TL; ++t) {
                        const int tile = TL == 2 ? t : h;
                        p[t][0] = st + (16 * t + g) * a.rs;
                        p[t][1] = p[t][0] + 8 * a.rs;
                        if constexpr (!kAlignedRows<F>) {
                            // rows start where they do within their 16 bytes in memory
                            const uint32_t ph = ph0 + (g + (a.gate_up ? 0 : 16 * tile)) * static_cast<uint32_t>(a.rb);
                            p[t][0] += ph & 15u;  // the second row is 8 on, but with 8 and 8 rows the same one of up
                            p[t][1] += (ph + (UT == 1 && a.gate_up ? 0u : 8 * static_cast<uint32_t>(a.rb))) & 15u;
                        }
                        wsc[t] = F == F_F8 ? a.sc[tile] + sc0 : nullptr;
                    }
                    moe_cg<F, T, NB, EX, TL>(p, g, i, rec, x, xs, blocks, wsc, tot + (TL == 2 ? 0 : h));
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.empty[s]);
                if (++s == a.stages) {
                    s = 0;
                    par ^= 1;
                }
            }
        }
        // The sums of two rounds before, in the same buffer, have been joined.  (One buffer and a deeper ring were slower:
        // 90 against 77 us for 16 tokens on e4m3 experts.)
        if (ok && q > 1) ok = moe_wait(&bars.joined[q & 1], ((q >> 1) - 1) & 1, &bars, a.err);
        float* rb = red + (q & 1) * kSums;
#pragma unroll
        for (int t = 0; t < UT; ++t)
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int v = 0; v < C::kOwn; ++v) {
                    float* to = rb + ((warp * UT + t) * kTok + n * C::kTokens + C::own(i, v)) * 16;
                    to[g] = tot[t][n][0][v];
                    to[g + 8] = tot[t][n][1][v];
                }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.sums[q & 1]);
    }
}

template <typename T>
__global__ void __launch_bounds__(256) moe_combine_kernel(const float* __restrict__ z, const int* __restrict__ ids,
                                                          const float* __restrict__ wt, T* __restrict__ y, int64_t tokens,
                                                          int64_t hidden, int top_k, int experts) {
    pdl_wait();
    pdl_launch_dependents();
    const int64_t n = tokens * hidden;
    for (int64_t o = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; o < n;
         o += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t t = o / hidden, c = o - t * hidden;
        y[o] = Elem<T>::put(moe_combined(z, ids, wt, t, c, hidden, top_k, experts));
    }
}

// ---- host -----------------------------------------------------------------------------

template <class Fn>
cudaError_t with_moe_fmt(int fmt, Fn&& f) {
    switch (fmt) {
        case F_Q8_0: return f(std::integral_constant<int, F_Q8_0>{});
        case F_Q4_0: return f(std::integral_constant<int, F_Q4_0>{});
        case F_Q2_K: return f(std::integral_constant<int, F_Q2_K>{});
        case F_Q3_K: return f(std::integral_constant<int, F_Q3_K>{});
        case F_Q4_K: return f(std::integral_constant<int, F_Q4_K>{});
        case F_Q5_K: return f(std::integral_constant<int, F_Q5_K>{});
        case F_Q6_K: return f(std::integral_constant<int, F_Q6_K>{});
        case F_F8: return f(std::integral_constant<int, F_F8>{});
        default: return cudaErrorInvalidValue;
    }
}

template <int F, int T, int NB, bool EX>
cudaError_t launch_expert(ExpertArgs a, int64_t cols, cudaStream_t s) {
    constexpr int CGB = moe_cg_bytes<F>();
    a.ncg = static_cast<int>((cols + 255) / 256);
    if constexpr (F == F_F8) {
        a.nblk = static_cast<int>((cols + 127) / 128);
        a.row_bytes = cols;
    } else {
        constexpr int BE = Traits<F>::BE;
        const int64_t blocks = (cols + BE - 1) / BE;
        a.nblk = static_cast<int>(blocks) * (BE == 256 ? 8 : 1);
        a.row_bytes = a.rb = blocks * Traits<F>::BB;
    }
    // short rows: several units share a stage, so that every warp has a CG
    a.slots = a.ncg <= 2 ? 4 : a.ncg <= 4 ? 2 : 1;
    a.wps = kConsumers / a.slots;
    const int unit_rows = (a.gate_up ? 8 : 16) * kUnitTiles<F, NB>;
    a.tiles = static_cast<int>((a.rows + unit_rows - 1) / unit_rows);
    // row stride of a stage: the segment, its phase of up to 15 bytes, the 4 that word loads read past it, rounded
    // to an odd multiple of 16 so that eight rows start in different banks
    const int cgs = std::min(a.wps, a.ncg);
    a.rs = (cgs * CGB + 15 + 4 + 15) / 16 * 16;
    while (a.rs % 128 != 16) a.rs += 16;
    a.stage_bytes = a.slots * 16 * kStageTiles<F, NB> * a.rs;
    // sums of two rounds
    const int red = 2 * kConsumers * kUnitTiles<F, NB> * (8 / T) * NB * 16 * 4;
    // two CTAs per SM, each with up to 3 KB besides (barriers and rounds, the driver's 1 KB)
    const int budget = 109 * 1024 - 512 - red;
    a.stages = std::min(kMoeStages, budget / a.stage_bytes);
    int per_sm = 2;
    if (a.stages < 2) {
        a.stages = std::min(kMoeStages, (224 * 1024 - 512 - red) / a.stage_bytes);
        per_sm = 1;
    }
    if (a.stages < 2) return cudaErrorInvalidConfiguration;
    const int smem = a.stages * a.stage_bytes + red + 128;
    static std::atomic<int> cfg[64];
    if (cudaError_t e = ensure_dyn_smem(moe_expert_kernel<F, T, NB, EX>, smem, cfg); e != cudaSuccess) return e;
    cudaError_t e = launch_pdl(moe_expert_kernel<F, T, NB, EX>, dim3(static_cast<unsigned>(device_sm_count() * per_sm)),
                               dim3(kMoeThreads), smem, s, a);
    return e == cudaSuccess ? cudaGetLastError() : e;
}

// One term: eight columns are up to 8 tokens.  Two terms: a block of columns is 4
// tokens, and groups of up to 8 take two blocks.
cudaError_t launch_experts(int fmt, const ExpertArgs& a, int64_t cols, int terms, int group, bool exact, cudaStream_t s) {
    return with_moe_fmt(fmt, [&](auto f) {
        constexpr int F = decltype(f)::value;
        constexpr bool kLong = Order<F>::SUMS > 0;  // the other formats' sums leave the tensor core after a block
        if (terms == 1) return launch_expert<F, 1, 1, false>(a, cols, s);
        if (kLong && exact) return group == 4 ? launch_expert<F, 2, 1, kLong>(a, cols, s) : launch_expert<F, 2, 2, kLong>(a, cols, s);
        return group == 4 ? launch_expert<F, 2, 1, false>(a, cols, s) : launch_expert<F, 2, 2, false>(a, cols, s);
    });
}

template <typename T>
cudaError_t launch_prep(const T* x, const RecordArgs& a, const MoePlan& plan, cudaStream_t s) {
    const int64_t grid = (a.rows * a.ncg + kPrepWarps - 1) / kPrepWarps + (plan.ids ? 1 : 0);
    cudaError_t e = launch_pdl(moe_prep_kernel<T>, dim3(static_cast<unsigned>(grid)), dim3(32 * kPrepWarps), 0, s, x, a, plan);
    return e == cudaSuccess ? cudaGetLastError() : e;
}

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// Tokens of one pass: their choices fit the plan.
int64_t pass_tokens(int top_k) { return std::max<int64_t>(1, kMoePairs / top_k); }

struct MoeSpace {
    size_t plan, rec_x, rec_h, h, z, total;
};

MoeSpace moe_space(int64_t tokens, int top_k, int64_t hidden, int64_t ffn) {
    const int64_t t = std::min(tokens, pass_tokens(top_k)), p = t * top_k;
    MoeSpace w{};
    size_t at = 256;  // status word
    auto take = [&](size_t n) {
        const size_t r = at;
        at += up256(n);
        return r;
    };
    w.plan = take(kMoePlanBytes);
    w.rec_x = take(static_cast<size_t>(t) * ((hidden + 255) / 256) * kRec<2>);
    w.rec_h = take(static_cast<size_t>(p) * ((ffn + 255) / 256) * kRec<2>);
    w.h = take(static_cast<size_t>(p) * ffn * 4);
    w.z = take(static_cast<size_t>(p) * hidden * 4);
    w.total = at;
    return w;
}

cudaError_t launch_route(int dtype, const void* x, const float* w, int* ids, float* weights, int64_t tokens, int experts,
                         int top_k, int64_t hidden, int normalize, const RecordArgs& records, const MoePlan& plan, cudaStream_t s) {
    return with_dtype(dtype, [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        const bool vec = hidden % 4 == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0 &&
                         reinterpret_cast<uintptr_t>(x) % (4 * sizeof(T)) == 0;
        const int64_t clusters = (tokens + kRouteTokens - 1) / kRouteTokens;
        const int64_t nrec = records.rows * records.ncg;
        const int64_t extra = (nrec + kRouteWarps * kRouteCtas - 1) / (kRouteWarps * kRouteCtas);  // clusters
        int slices = 1;
        while (2 * slices * experts <= kRouteCtas * kRouteWarps && hidden >= 256 * slices) slices *= 2;
        const size_t smem = static_cast<size_t>(slices) * kRouteTokens * experts * 4;
        cudaError_t e = launch_pdl(moe_route_kernel<T>, dim3(static_cast<unsigned>((clusters + extra) * kRouteCtas)),
                                   dim3(32 * kRouteWarps), smem, s, static_cast<const T*>(x), w, ids, weights, tokens,
                                   experts, top_k, hidden, slices, normalize, vec, records, plan);
        return e == cudaSuccess ? cudaGetLastError() : e;
    });
}

}  // namespace

size_t moe_workspace_bytes(int64_t tokens, int top_k, int64_t hidden, int64_t ffn) {
    return moe_space(tokens, top_k, hidden, ffn).total;
}

cudaError_t moe_route_dispatch(int dtype, const void* x, const float* w, int* ids, float* weights, int64_t tokens,
                               int experts, int top_k, int64_t hidden, int normalize, cudaStream_t s) {
    return launch_route(dtype, x, w, ids, weights, tokens, experts, top_k, hidden, normalize, RecordArgs{}, MoePlan{}, s);
}

// Passes of up to kMoePairs choices.  A pass is five kernels: router, with the
// records of x and the plan; gate and up; records of the hidden activations; down;
// y.  Without a router, or with more tokens than one cluster routes, the plan is a
// kernel too (and with several passes or no router the records are with it).
cudaError_t moe_mlp_dispatch(const MoeMlp& m, void* ws, int* err, cudaStream_t s) {
    const MoeSpace w = moe_space(m.tokens, m.top_k, m.hidden, m.ffn);
    auto* base = static_cast<uint8_t*>(ws);
    const int64_t step = pass_tokens(m.top_k);
    const int size = host_dtype_size(m.dtype);
    // 16-bit x is one term; fp32 x and the hidden activations, which are fp32 whatever the result's type, are two
    const int terms_x = m.dtype == AXQ_DT_F32 ? 2 : 1, terms_h = 2;
    const bool exact = m.dtype == AXQ_DT_F32;
    const bool several = m.tokens > step;  // passes
    if (m.w_router && several) {
        cudaError_t e = moe_route_dispatch(m.dtype, m.x, m.w_router, m.ids, m.weights, m.tokens, m.experts, m.top_k, m.hidden,
                                           m.normalize, s);
        if (e != cudaSuccess) return e;
    }
    for (int64_t t0 = 0; t0 < m.tokens; t0 += step) {
        const int64_t t = std::min(step, m.tokens - t0), p = t * m.top_k;
        // Tokens of a group.  With one-term x gate and up take 8 at once, so 8 unless no expert can have more than 4, whose
        // down product then does without the second block of columns (1 token Q4_K / Q6_K, 8 of 64 experts: 39.3 against
        // 43.1 us; 4 tokens, 2 of 8: 179 against 204; but 16 tokens 130 against 117).  With two-term x by the average.
        const int group = (terms_x == 1 ? t > 4 : p > 4 * m.experts) ? 8 : 4;
        MoePlan plan = moe_plan_at(base + w.plan);
        plan.ids = m.ids + t0 * m.top_k;
        plan.npairs = static_cast<int>(p);
        plan.experts = m.experts;
        plan.group = group;
        plan.top_k = m.top_k;
        plan.err = t0 == 0 ? err : nullptr;
        const void* x = static_cast<const uint8_t*>(m.x) + t0 * m.hidden * size;
        void* y = static_cast<uint8_t*>(m.y) + t0 * m.hidden * size;
        float* h = reinterpret_cast<float*>(base + w.h);
        float* z = reinterpret_cast<float*>(base + w.z);
        RecordArgs rx{};
        rx.fmt = m.fmt;
        rx.terms = terms_x;
        rx.rows = t;
        rx.cols = m.hidden;
        rx.ncg = static_cast<int>((m.hidden + 255) / 256);
        rx.rec = base + w.rec_x;
        cudaError_t e;
        const bool routed = m.w_router && !several;  // the router's kernel writes the records too
        const bool planned = routed && t <= kRouteTokens;  // and makes the plan, if one cluster has all tokens
        if (routed) {
            e = launch_route(m.dtype, x, m.w_router, m.ids, m.weights, t, m.experts, m.top_k, m.hidden, m.normalize, rx,
                             planned ? plan : MoePlan{}, s);
            if (e != cudaSuccess) return e;
            rx.rows = 0;
        }
        if (!planned) {
            e = with_dtype(m.dtype, [&](auto* tag) {
                using T = std::remove_pointer_t<decltype(tag)>;
                return launch_prep<T>(static_cast<const T*>(x), rx, plan, s);
            });
            if (e != cudaSuccess) return e;
        }
        ExpertArgs a{};
        a.w[0] = static_cast<const uint8_t*>(m.w_gate);
        a.w[1] = static_cast<const uint8_t*>(m.w_up);
        a.sc[0] = m.s_gate;
        a.sc[1] = m.s_up;
        a.rb = m.hidden;  // e4m3; the packed formats set their own
        a.w_bytes = m.gate_bytes;
        a.rows = m.ffn;
        a.gate_up = 1;
        a.rec = rx.rec;
        a.rec_row = static_cast<int64_t>(rx.ncg) * rec_bytes(terms_x);
        a.rec_token = 1;
        a.out = h;
        a.plan = plan;
        a.next = plan.taken;
        a.err = err;
        if (e = launch_experts(m.fmt, a, m.hidden, terms_x, group, exact, s); e != cudaSuccess) return e;
        RecordArgs rh{};
        rh.fmt = m.fmt_down;
        rh.terms = terms_h;
        rh.rows = p;
        rh.cols = m.ffn;
        rh.ncg = static_cast<int>((m.ffn + 255) / 256);
        rh.rec = base + w.rec_h;
        rh.need = plan.ids;
        rh.experts = m.experts;
        if (e = launch_prep<float>(h, rh, MoePlan{}, s); e != cudaSuccess) return e;
        a.w[0] = a.w[1] = static_cast<const uint8_t*>(m.w_down);
        a.sc[0] = a.sc[1] = m.s_down;
        a.rb = m.ffn;
        a.w_bytes = m.down_bytes;
        a.rows = m.hidden;
        a.gate_up = 0;
        a.rec = rh.rec;
        a.rec_row = static_cast<int64_t>(rh.ncg) * rec_bytes(terms_h);
        a.rec_token = 0;
        a.out = z;
        a.next = plan.taken + 1;
        if (e = launch_experts(m.fmt_down, a, m.ffn, terms_h, group, exact, s); e != cudaSuccess) return e;
        const float* wt = m.weights + t0 * m.top_k;
        e = with_dtype(m.dtype, [&](auto* tag) {
            using T = std::remove_pointer_t<decltype(tag)>;
            const int64_t grid = std::min<int64_t>((t * m.hidden + 255) / 256, int64_t(device_sm_count()) * 8);
            cudaError_t r = launch_pdl(moe_combine_kernel<T>, dim3(static_cast<unsigned>(grid)), dim3(256), 0, s,
                                       static_cast<const float*>(z), plan.ids, wt, static_cast<T*>(y), t, m.hidden, m.top_k,
                                       m.experts);
            return r == cudaSuccess ? cudaGetLastError() : r;
        });
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace axq
