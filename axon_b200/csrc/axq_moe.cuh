// The plan of a mixture-of-experts pass: the tokens' choices ("pairs", p = token
// * top_k + j) sorted by expert, cut into groups of tokens that share a read of
// the expert's weights.
#pragma once

#include <cstdint>

namespace axq {

constexpr int kMoePairs = 512;     // choices of one pass, at most
constexpr int kMoeFew = 64;        // choices that each CTA plans for itself, at most
constexpr int kMoeExperts = 1024;  // experts, at most

struct MoePlan {
    const int* ids;  // null once the plan is made
    int npairs, experts, group;
    int* ngroups;
    int4* groups;    // expert, first entry, number of entries
    int2* entries;   // pair and its token, sorted by expert
    int top_k;
    int* err;        // status word to clear, or null
};

// The plan of few choices, made by every CTA in its shared memory (no kernel
// has to come between the choice of experts and their products).
struct MoeFewPlan {
    int4 groups[kMoeFew];
    int2 entries[kMoeFew];
    int ids[kMoeFew], rank[kMoeFew];
    int ngroups;
};

// All threads of the block (at least kMoeFew) call it.
__device__ __forceinline__ void moe_few_plan(MoeFewPlan& p, const MoePlan& m) {
    const int tid = threadIdx.x;
    if (tid < kMoeFew) p.ids[tid] = tid < m.npairs ? m.ids[tid] : -1;
    __syncthreads();
    const int mine = tid < kMoeFew ? p.ids[tid] : -1;
    const bool valid = static_cast<unsigned>(mine) < static_cast<unsigned>(m.experts);
    int before = 0, rank = 0, total = 0;
    if (valid) {
        for (int q = 0; q < m.npairs; ++q) {
            const int e = p.ids[q];
            before += (e >= 0 && e < mine) || (e == mine && q < tid) ? 1 : 0;
            rank += e == mine && q < tid ? 1 : 0;
            total += e == mine ? 1 : 0;
        }
    }
    if (tid < kMoeFew) p.rank[tid] = valid ? rank % m.group : -1;
    __syncthreads();
    int starts = 0;  // groups that begin before this pair, and in all
    int all = 0;
    for (int q = 0; q < m.npairs; ++q) {
        const int e = p.ids[q], s = p.rank[q] == 0 ? 1 : 0;
        all += s;
        starts += s && (e < mine || (e == mine && q < tid)) ? 1 : 0;
    }
    if (valid) {
        p.entries[before] = make_int2(tid, tid / m.top_k);
        if (rank % m.group == 0) p.groups[starts] = make_int4(mine, before, min(m.group, total - rank), 0);
    }
    if (tid == 0) p.ngroups = all;
    __syncthreads();
}

constexpr size_t kMoePlanBytes = 256 + kMoePairs * 16 + kMoePairs * 8;

inline MoePlan moe_plan_at(uint8_t* p) {
    MoePlan m{};
    m.ngroups = reinterpret_cast<int*>(p);
    m.groups = reinterpret_cast<int4*>(p + 256);
    m.entries = reinterpret_cast<int2*>(p + 256 + kMoePairs * 16);
    return m;
}

// Makes the plan with one block of 256 threads.  Ids out of range (a padded
// token, an expert held elsewhere) appear in no group.
__device__ __forceinline__ void moe_make_plan(const MoePlan& m) {
    __shared__ int ids[kMoePairs];
    __shared__ int first[kMoeExperts];
    __shared__ int warp_sum[2][8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0 && m.err) *m.err = 0;
    for (int p = tid; p < m.npairs; p += 256) ids[p] = m.ids[p];
    __syncthreads();
    // counts of experts 4 tid .. 4 tid + 3, then sums over the experts before
    int cnt[4] = {0, 0, 0, 0};
    for (int p = 0; p < m.npairs; ++p) {
        const int d = ids[p] - 4 * tid;
#pragma unroll
        for (int j = 0; j < 4; ++j) cnt[j] += (d == j && ids[p] < m.experts) ? 1 : 0;
    }
    int c = 0, g = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
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
    if (tid == 255) *m.ngroups = gb + g;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        first[4 * tid + j] = cb;
        for (int k = 0; k * m.group < cnt[j]; ++k)
            m.groups[gb + k] = make_int4(4 * tid + j, cb + k * m.group, min(m.group, cnt[j] - k * m.group), 0);
        cb += cnt[j];
        gb += (cnt[j] + m.group - 1) / m.group;
    }
    __syncthreads();
    // a pair's place: after the earlier pairs of its expert
    for (int p = tid; p < m.npairs; p += 256) {
        const int e = ids[p];
        if (static_cast<unsigned>(e) >= static_cast<unsigned>(m.experts)) continue;
        int r = first[e];
        for (int q = 0; q < p; ++q) r += ids[q] == e ? 1 : 0;
        m.entries[r] = make_int2(p, p / m.top_k);
    }
}

}  // namespace axq
