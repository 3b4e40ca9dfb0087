// The plan of a mixture-of-experts pass: the tokens' choices ("pairs", p = token
// * top_k + j) sorted by expert, cut into groups of tokens that share a read of
// the expert's weights.
#pragma once

#include <cstdint>

namespace axq {

constexpr int kMoePairs = 512;     // choices of one pass, at most
constexpr int kMoeExperts = 1024;  // experts, at most

struct MoePlan {
    const int* ids;  // null: no plan to make
    int npairs, experts, group, top_k;
    int* ngroups;
    int* taken;      // counters of the rounds that the two products' CTAs have taken, set to 0
    int4* groups;    // expert, first entry, number of entries
    int2* entries;   // pair and its token, sorted by expert
    int* err;        // status word to clear, or null
};

constexpr size_t kMoePlanBytes = 256 + kMoePairs * 16 + kMoePairs * 8;

inline MoePlan moe_plan_at(uint8_t* p) {
    MoePlan m{};
    m.ngroups = reinterpret_cast<int*>(p);
    m.taken = m.ngroups + 1;
    m.groups = reinterpret_cast<int4*>(p + 256);
    m.entries = reinterpret_cast<int2*>(p + 256 + kMoePairs * 16);
    return m;
}

// Makes the plan with one block of kThreads threads.  Ids out of range (a padded
// token, an expert held elsewhere) appear in no group.
template <int kThreads>
__device__ __forceinline__ void moe_make_plan(const MoePlan& m) {
    constexpr int kOwn = kMoeExperts / kThreads;  // experts of a thread
    __shared__ int4 ids4[kMoePairs / 4];
    __shared__ int first[kMoeExperts];  // counts, then first entries
    __shared__ int warp_sum[2][kThreads / 32];
    int* ids = reinterpret_cast<int*>(ids4);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid < 2) m.taken[tid] = 0;
    if (tid == 0 && m.err) *m.err = 0;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) first[kOwn * tid + j] = 0;
    for (int p = tid; p < (m.npairs + 3) / 4 * 4; p += kThreads) {
        const int e = p < m.npairs ? m.ids[p] : -1;
        ids[p] = static_cast<unsigned>(e) < static_cast<unsigned>(m.experts) ? e : -1;
    }
    __syncthreads();
    for (int p = tid; p < m.npairs; p += kThreads)
        if (ids[p] >= 0) atomicAdd(&first[ids[p]], 1);
    __syncthreads();
    // sums over the experts before those of this thread
    int cnt[kOwn];
#pragma unroll
    for (int j = 0; j < kOwn; ++j) cnt[j] = first[kOwn * tid + j];
    int c = 0, g = 0;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        c += cnt[j];
        g += (cnt[j] + m.group - 1) / m.group;
    }
    int ci = c, gi = g;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int a = __shfl_up_sync(0xFFFFFFFFu, ci, d), b = __shfl_up_sync(0xFFFFFFFFu, gi, d);
        if (lane >= d) {
            ci += a;
            gi += b;
        }
    }
    if (lane == 31) {
        warp_sum[0][warp] = ci;
        warp_sum[1][warp] = gi;
    }
    __syncthreads();
    int cb = ci - c, gb = gi - g;
    for (int w = 0; w < warp; ++w) {
        cb += warp_sum[0][w];
        gb += warp_sum[1][w];
    }
    if (tid == kThreads - 1) *m.ngroups = gb + g;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        first[kOwn * tid + j] = cb;
        for (int k = 0; k * m.group < cnt[j]; ++k)
            m.groups[gb + k] = make_int4(kOwn * tid + j, cb + k * m.group, min(m.group, cnt[j] - k * m.group), 0);
        cb += cnt[j];
        gb += (cnt[j] + m.group - 1) / m.group;
    }
    __syncthreads();
    // a pair's place: after the earlier pairs of its expert
    for (int p = tid; p < m.npairs; p += kThreads) {
        const int e = ids[p];
        if (e < 0) continue;
        int r = first[e];
#pragma unroll 4
        for (int q = 0; q < p; q += 4) {
            const int4 o = ids4[q / 4];
            r += (o.x == e) + (o.y == e && q + 1 < p) + (o.z == e && q + 2 < p) + (o.w == e && q + 3 < p);
        }
        m.entries[r] = make_int2(p, p / m.top_k);
    }
}

}  // namespace axq
