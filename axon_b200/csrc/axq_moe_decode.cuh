// Decoders of packed weight rows into mma.sync m16n8k16 A fragments (fp16,
// exact) for the mixture-of-experts kernels.
//
// A column group (CG) is 256 elements of a row.  Lane (g, i) = (lane / 4,
// lane % 4) of a warp holds, of each of its rows, 64 of a CG's elements: which
// ones is each format's choice, as long as the activation records hold x in the
// same order (order_elem).  In the formats with integer sub-block scales a
// lane owns whole sub-blocks, so that it decodes only their scales.
//
// fp16 holds integers up to 2048 exactly, and 0x6400 | c is 1024 + c.  So
// (1024 + c * 2^s) * (sc / 2^s) - 1024 * sc / 2^s, one FMA on two codes, is
// sc * c exactly wherever |sc * c| <= 2048 (or has at most 11 significant
// bits): code extraction, conversion and sub-block scale cost a mask and an FMA
// for two elements, and the MMAs add a whole CG without touching the sums.  The
// block's fp16 d and dmin are applied in fp32 once per CG.
#pragma once

#include "axq_common.cuh"
#include "axq_f8.cuh"
#include "axq_ptx.cuh"

namespace axq {

constexpr int F_F8 = 64;  // AXQ_F8_E4M3: e4m3 codes with 128 x 128 scales

// Order of a CG's elements and sub-blocks over the lanes, by format.
//
// SUMS: sub-blocks whose sums of x weigh the minimums (0: none).
template <int F> struct Order {
    static constexpr bool K4 = F == F_Q4_K || F == F_Q5_K;
    static constexpr bool K16 = F == F_Q2_K || F == F_Q3_K || F == F_Q6_K;
    static constexpr int SUMS = K4 ? 8 : K16 ? 16 : 0;
};

// Element (0..255) of the CG at slot 0..3 of MMA m (0..15) of lane part i.
// Slots 0, 1 are the low and high half of the first fragment register, 2, 3 of
// the second.
__device__ __forceinline__ int order_elem(int fmt, int m, int i, int slot) {
    const int bo = slot == 1 ? 2 : slot == 2 ? 1 : slot;  // bytes 0, 2 of a word, then 1, 3
    if (fmt == F_Q4_K || fmt == F_Q5_K) return 64 * i + 32 * (m & 1) + 4 * (m >> 1) + bo;
    if (fmt == F_Q2_K || fmt == F_Q3_K || fmt == F_Q6_K) {
        // Q2_K: lane part i starts at word i of its four (conflict-free loads)
        const int v = fmt == F_Q2_K ? ((m >> 2) + i) & 3 : m >> 2;
        return 128 * (i >> 1) + 32 * (m & 3) + 16 * (i & 1) + 4 * v + bo;
    }
    if (fmt == F_Q8_0) return 32 * (m >> 1) + 8 * i + 4 * (m & 1) + slot;
    if (fmt == F_Q4_0) return 32 * (m >> 1) + 2 * (4 * i + bo) + (m & 1);
    return 128 * (m >> 3) + 32 * i + 4 * (m & 7) + slot;  // e4m3
}

// Sub-blocks of the format that have sums (0: none), and the one at slot j of
// lane part i (-1: none).
__device__ __forceinline__ int order_sums(int fmt) {
    return fmt == F_Q4_K || fmt == F_Q5_K ? 8 : fmt == F_Q2_K || fmt == F_Q3_K || fmt == F_Q6_K ? 16 : 0;
}
__device__ __forceinline__ int order_sum(int fmt, int i, int j) {
    if (fmt == F_Q4_K || fmt == F_Q5_K) return j < 2 ? 2 * i + j : -1;
    return 8 * (i >> 1) + 2 * j + (i & 1);
}

template <int F> constexpr int moe_cg_bytes() {
    return F == F_F8 ? 256 : F == F_Q8_0 ? 8 * 34 : F == F_Q4_0 ? 8 * 18 : Traits<F == F_F8 ? F_Q4_K : F>::BB;
}

__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t h2_const(float v) {
    const __half2 h = __float2half2_rn(v);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// Two integers 0 .. 1023 in the halves of v, less K, as an fp16 pair.
template <int K>
__device__ __forceinline__ uint32_t ints_h2(uint32_t v) {
    uint32_t d;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(v | 0x64006400u), "r"(h2_const(-1024.0f - K)));
    return d;
}
// (v.low, v.low) and (v.high, v.high)
__device__ __forceinline__ uint32_t h2_low(uint32_t v) { return __byte_perm(v, 0u, 0x1010u); }
__device__ __forceinline__ uint32_t h2_high(uint32_t v) { return __byte_perm(v, 0u, 0x3232u); }
__host__ __device__ constexpr uint32_t h2_pow2(int lo, int hi) {  // (2^lo, 2^hi), exponents -14 .. 15
    return static_cast<uint32_t>((lo + 15) << 10) | (static_cast<uint32_t>((hi + 15) << 10) << 16);
}
constexpr uint32_t kNeg2 = 0x80008000u;  // signs of both halves
// (w & m) | o in one LOP3: two constants do not fit its immediate, and the
// compiler splits the expression where it is not spelled out.
__device__ __forceinline__ uint32_t lop_and_or(uint32_t w, uint32_t m, uint32_t o) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(w), "r"(m), "r"(o));
    return d;
}
template <uint32_t MASK, uint32_t OR>
__device__ __forceinline__ uint32_t and_or(uint32_t w) { return lop_and_or(w, MASK, OR); }
// Both halves of a block header (d, dmin), subnormals as zero (the formats'
// definition), to fp32.
__device__ __forceinline__ float2 h2_flush(uint32_t hd) {
    uint32_t r;
    asm("fma.rn.ftz.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(hd), "r"(0x3C003C00u), "r"(0x80008000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&r));
}
constexpr uint32_t kMagic = 0x64006400u;  // 1024 in both halves

// Words of a block at a 2-byte aligned shared address: one aligned base for the
// whole block, since every offset asked for is a multiple of 4; each word is cut
// out of the two aligned ones around it.
struct Words2 {
    const uint32_t* b;
    uint32_t sh;
    __device__ __forceinline__ explicit Words2(const uint8_t* p) {
        // the base by pointer arithmetic keeps a shared pointer shared
        const uint32_t mis = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 3u;
        b = reinterpret_cast<const uint32_t*>(p - mis);
        sh = mis * 8;
    }
    template <int N>
    __device__ __forceinline__ void load(int off, uint32_t (&out)[N]) const {
        uint32_t w[N + 1];
#pragma unroll
        for (int k = 0; k <= N; ++k) w[k] = b[off / 4 + k];
#pragma unroll
        for (int k = 0; k < N; ++k) out[k] = __funnelshift_r(w[k], w[k + 1], sh);
    }
};

__device__ __forceinline__ uint32_t ld_half2b(const uint8_t* p) { return *reinterpret_cast<const uint16_t*>(p); }

// Row<F>: one row's part of one CG.  load(p, i) reads the header; pair<MP>(a)
// gives the fragments of MMAs 2 MP (a[0], a[1]) and 2 MP + 1 (a[2], a[3]);
// mins(a) those of the minimums' MMA (sub-block sums of x against them);
// scales() those of the sums of codes and of minimums.
template <int F> struct MoeRow;

// Q4_K {d, dmin, scales[12], qs[128]}: lane part i owns qs[32i ..], the
// sub-blocks 2i (low nibbles) and 2i + 1 (high nibbles): 63 * 15 <= 2048.
// Q5_K {d, dmin, scales[12], qh[32], qs[128]}: the fifth bit of sub-block s is
// bit s of qh[l]: 63 * 31 <= 2048.
template <int F> struct MoeRowK45 {
    const uint8_t* q;
    uint32_t hd, w[4], h[4];
    uint32_t scl, cl, sch, ch, mn;
    int sh;
    const uint8_t* qh;
    __device__ __forceinline__ void load(const uint8_t* p, int i) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        hd = v.x;
        // 6-bit scales and minimums j = 2i, 2i + 1 (get_scale_min_k4): bytes 0-3 hold scales 0-3, 4-7 minimums 0-3,
        // 8-11 the low halves of both for 4-7, whose high two bits are the top bits of the first eight bytes.  The
        // two bytes of this lane go to the halves of one register.
        const uint32_t sel = (i & 1) ? 0x4342u : 0x4140u;
        const uint32_t x = __byte_perm(v.y, 0u, sel), y = __byte_perm(v.z, 0u, sel), t = __byte_perm(v.w, 0u, sel);
        const uint32_t sp = i < 2 ? x & 0x003F003Fu : (t & 0x000F000Fu) | ((x >> 2) & 0x00300030u);
        const uint32_t mp = i < 2 ? y & 0x003F003Fu : ((t >> 4) & 0x000F000Fu) | ((y >> 2) & 0x00300030u);
        mn = ints_h2<0>(mp);
        const uint32_t s2 = hmul2(ints_h2<0>(sp), h2_pow2(0, -4));  // the high nibbles stay in place (x 16)
        const uint32_t c2 = hmul2(s2, h2_pow2(10, 10) | kNeg2);
        scl = h2_low(s2);
        sch = h2_high(s2);
        cl = h2_low(c2);
        ch = h2_high(c2);
        q = p + (F == F_Q4_K ? 16 : 48) + 32 * i;
        qh = p + 16;
        sh = 2 * i;
    }
    template <int MP>
    __device__ __forceinline__ void pair(uint32_t (&a)[4]) {
        if constexpr (MP % 4 == 0) {
            const uint4 v = *reinterpret_cast<const uint4*>(q + 4 * MP);
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
            if constexpr (F == F_Q5_K) {
                const uint4 u = *reinterpret_cast<const uint4*>(qh + 4 * MP);
                h[0] = u.x >> sh; h[1] = u.y >> sh; h[2] = u.z >> sh; h[3] = u.w >> sh;
            }
        }
        const uint32_t x = w[MP % 4], y = x >> 8;
        uint32_t t0 = and_or<0x000F000Fu, kMagic>(x), t1 = and_or<0x000F000Fu, kMagic>(y);
        uint32_t t2 = and_or<0x00F000F0u, kMagic>(x), t3 = and_or<0x00F000F0u, kMagic>(y);
        if constexpr (F == F_Q5_K) {
            const uint32_t b = h[MP % 4];
            t0 = lop_and_or(b << 4, 0x00100010u, t0);
            t1 = lop_and_or(b >> 4, 0x00100010u, t1);
            t2 = lop_and_or(b << 7, 0x01000100u, t2);
            t3 = lop_and_or(b >> 1, 0x01000100u, t3);
        }
        a[0] = hfma2(t0, scl, cl);
        a[1] = hfma2(t1, scl, cl);
        a[2] = hfma2(t2, sch, ch);
        a[3] = hfma2(t3, sch, ch);
    }
    __device__ __forceinline__ void mins(uint32_t (&a)[2]) const { a[0] = mn; a[1] = 0; }
    __device__ __forceinline__ float2 scales() const { return h2_flush(hd); }
};
template <> struct MoeRow<F_Q4_K> : MoeRowK45<F_Q4_K> {};
template <> struct MoeRow<F_Q5_K> : MoeRowK45<F_Q5_K> {};

// Q2_K {d, dmin, scales[16], qs[64]}: lane part i owns qs[16i .. 16i + 15],
// whose four 2-bit fields are sub-blocks 8(i/2) + 2j + (i%2), j = 0..3: 15 * 3.
template <> struct MoeRow<F_Q2_K> {
    const uint8_t* q;
    uint32_t hd, sc[4], c[4], mn[2], w;
    int rot;
    __device__ __forceinline__ void load(const uint8_t* p, int i) {
        hd = *reinterpret_cast<const uint32_t*>(p);
        const uint32_t* s = reinterpret_cast<const uint32_t*>(p + 4 + 8 * (i >> 1));
        const int by = 8 * (i & 1);
        const uint32_t a = s[0] >> by, b = s[1] >> by;  // bytes 2j + (i & 1) in the halves
        const uint32_t s01 = hmul2(ints_h2<0>(a & 0x000F000Fu), h2_pow2(0, -2));
        const uint32_t s23 = hmul2(ints_h2<0>(b & 0x000F000Fu), h2_pow2(-4, -6));
        const uint32_t c01 = hmul2(s01, h2_pow2(10, 10) | kNeg2), c23 = hmul2(s23, h2_pow2(10, 10) | kNeg2);
        sc[0] = h2_low(s01); sc[1] = h2_high(s01); sc[2] = h2_low(s23); sc[3] = h2_high(s23);
        c[0] = h2_low(c01); c[1] = h2_high(c01); c[2] = h2_low(c23); c[3] = h2_high(c23);
        mn[0] = ints_h2<0>((a >> 4) & 0x000F000Fu);
        mn[1] = ints_h2<0>((b >> 4) & 0x000F000Fu);
        q = p + 20 + 16 * i;
        rot = i;
    }
    template <int MP>
    __device__ __forceinline__ void pair(uint32_t (&a)[4]) {
        if constexpr (MP % 2 == 0) w = reinterpret_cast<const uint32_t*>(q)[(MP / 2 + rot) & 3];
        constexpr int j = 2 * (MP % 2);  // MMA 2 MP: field j, MMA 2 MP + 1: field j + 1
        constexpr uint32_t m0 = 0x00030003u << (2 * j), m1 = 0x00030003u << (2 * j + 2);
        const uint32_t y = w >> 8;
        a[0] = hfma2(and_or<m0, kMagic>(w), sc[j], c[j]);
        a[1] = hfma2(and_or<m0, kMagic>(y), sc[j], c[j]);
        a[2] = hfma2(and_or<m1, kMagic>(w), sc[j + 1], c[j + 1]);
        a[3] = hfma2(and_or<m1, kMagic>(y), sc[j + 1], c[j + 1]);
    }
    __device__ __forceinline__ void mins(uint32_t (&a)[2]) const { a[0] = mn[0]; a[1] = mn[1]; }
    __device__ __forceinline__ float2 scales() const { return h2_flush(hd); }
};

// Q3_K {hmask[32], qs[64], scales[12], d}: the fields of Q2_K with a third bit,
// bit 4(i/2) + j of hmask[16(i%2) + l]; value = d * sc * (code - 4), sc = 6 bits
// - 32.  The codes (0..7) go through the MMAs, 4 sc through the minimums'.  A
// word's 16 fields and their high bits are merged into two words of 3-bit codes:
// fields 0 and 2 at bits 0 and 4 of each byte, fields 1 and 3 likewise.
template <> struct MoeRow<F_Q3_K> {
    uint32_t hd, sc[4], c[4], mn[2], w[4], h[4];
    uint32_t e, o;  // fields 0, 2 and 1, 3 of the word at work
    __device__ __forceinline__ void load(const uint8_t* p, int i) {
        hd = ld_half2b(p + 108);
        const Words2 words(p);
        uint32_t s[3];
        words.load(96, s);
        // scale is = 8n + 2j + lh: low 4 bits in nibble n of byte 2j + lh of the first eight, high 2 bits at
        // 2 (is >> 2) of byte 8 + (is & 3)
        const int n = i >> 1, lh = i & 1;
        const int by = 8 * lh + 4 * n;
        const uint32_t hb = s[2] >> by;
        const uint32_t v01 = ((s[0] >> by) & 0x000F000Fu) | ((hb << 4) & 0x00300030u);
        const uint32_t v23 = ((s[1] >> by) & 0x000F000Fu) | ((hb << 2) & 0x00300030u);
        const uint32_t x01 = ints_h2<32>(v01), x23 = ints_h2<32>(v23);
        mn[0] = hmul2(x01, h2_pow2(2, 2));
        mn[1] = hmul2(x23, h2_pow2(2, 2));
        const uint32_t s23 = hmul2(x23, h2_pow2(-4, -4));  // fields 2 and 3 stay in place (x 16)
        const uint32_t c01 = hmul2(x01, h2_pow2(10, 10) | kNeg2), c23 = hmul2(s23, h2_pow2(10, 10) | kNeg2);
        sc[0] = h2_low(x01); sc[1] = h2_high(x01); sc[2] = h2_low(s23); sc[3] = h2_high(s23);
        c[0] = h2_low(c01); c[1] = h2_high(c01); c[2] = h2_low(c23); c[3] = h2_high(c23);
        words.load(32 + 16 * i, w);
        words.load(16 * lh, h);
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] >>= 4 * n;
    }
    template <int MP>
    __device__ __forceinline__ void pair(uint32_t (&a)[4]) {
        if constexpr (MP % 2 == 0) {
            // high bits 0 / 2 to bits 2 / 6 in one multiply: x * 20 puts bit 0 at bits 2 and 4 and bit 2 at bits 4 and 6;
            // bits 4-5 (the sum of the two, never carrying into bit 6) are taken from w.  Likewise bits 1 / 3 by 10.
            e = lop_and_or(w[MP / 2], 0x33333333u, ((h[MP / 2] & 0x05050505u) * 20u) & 0x44444444u);
            o = lop_and_or(w[MP / 2] >> 2, 0x33333333u, ((h[MP / 2] & 0x0A0A0A0Au) * 10u) & 0x44444444u);
        }
        constexpr int j = 2 * (MP % 2);  // fields j, j + 1
        constexpr uint32_t m = j ? 0x00700070u : 0x00070007u;
        a[0] = hfma2(and_or<m, kMagic>(e), sc[j], c[j]);
        a[1] = hfma2(and_or<m, kMagic>(e >> 8), sc[j], c[j]);
        a[2] = hfma2(and_or<m, kMagic>(o), sc[j + 1], c[j + 1]);
        a[3] = hfma2(and_or<m, kMagic>(o >> 8), sc[j + 1], c[j + 1]);
    }
    __device__ __forceinline__ void mins(uint32_t (&a)[2]) const { a[0] = mn[0]; a[1] = mn[1]; }
    __device__ __forceinline__ float2 scales() const {
        const float d = h2_flush(hd).x;
        return make_float2(d, d);
    }
};

// Q6_K {ql[128], qh[64], scales[16], d}: field t of lane part i is sub-block
// 8(i/2) + 2t + (i%2); code = 4 bits of ql + 16 * 2 bits of qh, value = d * sc *
// (code - 32) with sc of 8 bits.  sc * code does not fit fp16, its two parts do:
// |sc| * 15 <= 1920 and |sc| * 16 * {0..3}, so each MMA is issued twice, on the
// low and on the high bits; 32 sc goes through the minimums'.  Scales are kept /
// 4, so that 1024 * sc / 4 is finite.
template <> struct MoeRow<F_Q6_K> {
    uint32_t hd, sc[4], c[4], mn[2], lo[8], hi[4];
    __device__ __forceinline__ void load(const uint8_t* p, int i) {
        const int n = i >> 1, lh = i & 1;
        hd = ld_half2b(p + 208);
        const Words2 words(p);
        uint32_t s[2];
        words.load(192 + 8 * n, s);
        const int by = 8 * lh;
        mn[0] = hmul2(ints_h2<128>(((s[0] >> by) & 0x00FF00FFu) ^ 0x00800080u), h2_pow2(-2, -2));
        mn[1] = hmul2(ints_h2<128>(((s[1] >> by) & 0x00FF00FFu) ^ 0x00800080u), h2_pow2(-2, -2));
        const uint32_t c01 = hmul2(mn[0], h2_pow2(10, 10) | kNeg2), c23 = hmul2(mn[1], h2_pow2(10, 10) | kNeg2);
        sc[0] = h2_low(mn[0]); sc[1] = h2_high(mn[0]); sc[2] = h2_low(mn[1]); sc[3] = h2_high(mn[1]);
        c[0] = h2_low(c01); c[1] = h2_high(c01); c[2] = h2_low(c23); c[3] = h2_high(c23);
        uint32_t a[4], b[4];
        words.load(64 * n + 16 * lh, a);
        words.load(64 * n + 32 + 16 * lh, b);
        words.load(128 + 16 * i, hi);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            lo[k] = a[k];      // fields 0 (low nibbles) and 2 (high)
            lo[4 + k] = b[k];  // fields 1 and 3
        }
    }
    // low bits (a) and high bits (b) of MMAs 2 MP, 2 MP + 1: fields t, t + 1 of word MP / 2
    template <int MP>
    __device__ __forceinline__ void pair(uint32_t (&a)[4], uint32_t (&b)[4]) {
        constexpr int t = 2 * (MP % 2), v = MP / 2;
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            const uint32_t x = lo[4 * f + v], z = hi[v];
            const uint32_t s = sc[t + f], k = c[t + f];
            // the nibble at bit 0 (fields 0, 1) or 4 (fields 2, 3) of bytes 0, 2, then of bytes 1, 3
            a[2 * f] = hfma2(and_or<0x000F000Fu, kMagic>(t ? x >> 4 : x), s, k);
            a[2 * f + 1] = hfma2(and_or<0x000F000Fu, kMagic>(t ? x >> 12 : x >> 8), s, k);
            // the 2 bits at 2 (t + f), moved to bits 4 and 5: 16 * field
            const int up = 4 - 2 * (t + f);
            b[2 * f] = hfma2(and_or<0x00300030u, kMagic>(up >= 0 ? z << up : z >> -up), s, k);
            b[2 * f + 1] = hfma2(and_or<0x00300030u, kMagic>(z >> (8 - up)), s, k);
        }
    }
    __device__ __forceinline__ void mins(uint32_t (&a)[2]) const { a[0] = mn[0]; a[1] = mn[1]; }
    __device__ __forceinline__ float2 scales() const {
        const float d = h2_flush(hd).x;
        return make_float2(d * 4.0f, d * 128.0f);
    }
};

// Q8_0 {d, qs[32]} x 8 and Q4_0 {d, qs[16]} x 8: a block's d is fp16, so its
// two MMAs (2 MP and 2 MP + 1 are block MP) are scaled in fp32; lane part i
// holds 8 elements of every block.
template <> struct MoeRow<F_Q8_0> {
    const uint8_t* p;
    int i;
    uint32_t hd;
    __device__ __forceinline__ void load(const uint8_t* q, int part) { p = q; i = part; }
    template <int MP>
    __device__ __forceinline__ void pair(uint32_t (&a)[4]) {
        hd = ld_half2b(p + 34 * MP);
        uint32_t w[2];
        Words2(p + 34 * MP + 2 + 8 * i).load(0, w);
        const uint32_t off = h2_const(-1152.0f), unit = h2_const(1.0f);  // 1024 + 128
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint32_t u = w[k] ^ 0x80808080u;
            a[2 * k] = hfma2(__byte_perm(u, 0x64646464u, 0x4140u), unit, off);
            a[2 * k + 1] = hfma2(__byte_perm(u, 0x64646464u, 0x4342u), unit, off);
        }
    }
    __device__ __forceinline__ float d() const { return h2_flush(hd).x; }
};
template <> struct MoeRow<F_Q4_0> {
    const uint8_t* p;
    int i;
    uint32_t hd;
    __device__ __forceinline__ void load(const uint8_t* q, int part) { p = q; i = part; }
    template <int MP>
    __device__ __forceinline__ void pair(uint32_t (&a)[4]) {
        hd = ld_half2b(p + 18 * MP);
        uint32_t w[1];
        Words2(p + 18 * MP + 2 + 4 * i).load(0, w);
        const uint32_t x = w[0], y = x >> 8;
        const uint32_t unit = h2_const(1.0f), o0 = h2_const(-1032.0f), s = h2_const(0.0625f), o1 = h2_const(-72.0f);
        a[0] = hfma2(and_or<0x000F000Fu, kMagic>(x), unit, o0);
        a[1] = hfma2(and_or<0x000F000Fu, kMagic>(y), unit, o0);
        a[2] = hfma2(and_or<0x00F000F0u, kMagic>(x), s, o1);
        a[3] = hfma2(and_or<0x00F000F0u, kMagic>(y), s, o1);
    }
    __device__ __forceinline__ float d() const { return h2_flush(hd).x; }
};

// e4m3: MMAs 0-7 are the first 128 columns, 8-15 the second; each half has one
// fp32 scale for the whole tile of rows.
template <> struct MoeRow<F_F8> {
    const uint8_t* p;
    uint32_t w[4];
    __device__ __forceinline__ void load(const uint8_t* q, int i) { p = q + 32 * i; }
    __device__ __forceinline__ static uint32_t cvt(uint32_t two) {
        uint32_t r;
        asm("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(two));
        return r;
    }
    template <int MP>
    __device__ __forceinline__ void pair(uint32_t (&a)[4]) {
        if constexpr (MP % 2 == 0) {
            const uint4 v = *reinterpret_cast<const uint4*>(p + 128 * (MP / 4) + 8 * (MP % 4));
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint32_t x = w[2 * (MP % 2) + k];
            a[2 * k] = cvt(x);
            a[2 * k + 1] = cvt(x >> 16);
        }
    }
};

}  // namespace axq
