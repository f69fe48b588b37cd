// Decode attention over int4-g32 pages, and over fp16 pages with the weight
// of every cached token added to an array.
//
// k_attn: a block of 8 wavefronts takes every splits-th pair of pages of one
// kv head for up to 8 of its query heads, keeps an online softmax per head,
// merges its wavefronts through LDS and writes one record (O, M, L), or the
// fp16 output where it has the kv head to itself.  With weights it also writes
// the scores, and with the kv head to itself it adds the weights as well.
// k_join: merges the records and, with weights, turns the scores into exp(s - M)
// / L, whose sum over the query heads of the kv head it adds to the weights.
// (The scores need M and L of all splits, which no block of k_attn has; reading
// them back costs 8 bytes a token and query head, the pages again would cost
// 9/16 byte or more a value.  Merging the records in the last block of k_attn
// instead took as long for 8 splits and longer for more: 18.3 against 15.5 us
// for 64.)
//
// Products are v_mfma_f32_16x16x32_f16 (A: lane l holds row l%16, k = 8 (l/16)
// .. +7; B: column l%16, the same k; C: column l%16, rows 4 (l/16) .. +3).
// S = K q^T: rows are a page's 16 tokens, columns 0-7 the query heads' fp16
// high parts and columns 8-15 their low parts (q = hi + lo to 2^-22), so one
// product gives both and a lane adds the column eight over.  O = P V: rows are
// heads, k the 32 tokens of a pair of pages in the order in which the lane
// already holds their scores (4 g .. +3 of page a, then of page b).
//
// int4-g32: a step of 32 dimensions is one scale group, so codes enter the
// products as exact fp16 integers and the scales stay outside: fp32 behind K's
// product, in front of V's with the probability.  Between two bounds: vector
// instructions beside the products (347 a pair of pages of 128 dimensions, 283
// more a wavefront) take 57 % of the SIMDs' time, and a wavefront, which has half
// a pair in flight, waits for memory in 47 % of its own: 32768 tokens of 8 kv heads
// (38 MB) 12.8 us and a join of 3.9.
#include <algorithm>
#include <type_traits>

#include "nx_attn_dev.h"
#include "nx_kvc.h"

namespace nx {
namespace kvc {

namespace {

using at::f4_t;
using at::h8_t;

constexpr int kWaves = 8;
constexpr int kThreads = kWaves * kWave;
constexpr int kMaxSplits = 64;
constexpr int kRowRor8 = 0x128;
constexpr float kUp = 11.0f, kLead = 4.0f, kFar = 1048576.0f;
constexpr float kLog2e = 1.4426950408889634f;

// Lane l's and lane l ^ 16's (32's) larger value, and their sum.
__device__ inline float max_x16(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    const uint32_t x = a[0], y = a[1];
    return fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}
__device__ inline float sum_x16(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    const uint32_t x = a[0], y = a[1];
    return __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
}
__device__ inline float sum_x32(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    const uint32_t x = a[0], y = a[1];
    return __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
}
// Lower lanes: the sum of a's two halves, upper lanes: of b's.
__device__ inline float halves_sum(float a, float b) {
    const auto v = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), false, false);
    const uint32_t x = v[0], y = v[1];
    return __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
}
__device__ inline float max_x32(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    const uint32_t x = a[0], y = a[1];
    return fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}

// ------------------------------------------------------------------- pages --
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h4_t __attribute__((ext_vector_type(4)));

// A lane's share of a pair of pages.
template <int HD>
struct PairI4 {
    uint32_t k[2][HD / 32], v[2][HD / 32];  // codes: K of token l%16, V of tokens 4 g .. +3
    h4_t ks[2][HD / 32], vs[2][HD / 32];    // scales of tokens 4 g .. +3 per group
};

// N dwords that start at a multiple of 4 N bytes (of 16 where N is above 4).
template <int N>
__device__ inline void load_words(uint32_t (&r)[N], const uint8_t* p) {
    if constexpr (N == 2) {
        const u2_t w = *reinterpret_cast<const u2_t*>(p);
        r[0] = w.x, r[1] = w.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const u4_t w = reinterpret_cast<const u4_t*>(p)[i / 4];
            r[i] = w.x, r[i + 1] = w.y, r[i + 2] = w.z, r[i + 3] = w.w;
        }
    }
}
template <int N>
__device__ inline void load_scales(h4_t (&r)[N], const uint8_t* p) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const h8_t w = reinterpret_cast<const h8_t*>(p)[i / 2];
        r[i] = __builtin_shufflevector(w, w, 0, 1, 2, 3), r[i + 1] = __builtin_shufflevector(w, w, 4, 5, 6, 7);
    }
}

// (Kept apart from the page's address, which is the same in all lanes: as sums
// of 64 bits the four addresses would take eight registers over the loop.)
__device__ inline uint32_t lane_offset(uint32_t v) {
    asm("" : "+v"(v));
    return v;
}

template <int HD>
__device__ inline void load_k(PairI4<HD>& r, const AttnArgs& a, const int (&blk)[2], int kvh, int lane) {
    constexpr int S = HD / 32;
    const uint32_t g = lane >> 4, t = lane & 15;
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
        const uint8_t* p = a.kpool + ((size_t)(uint32_t)blk[pg] * (uint32_t)a.hkv + (uint32_t)kvh) * page_bytes(HD);
        load_words<S>(r.k[pg], p + lane_offset((t * 4 + g) * (4 * S)));
        load_scales<S>(r.ks[pg], p + 8 * HD + lane_offset(g * (8 * S)));
    }
}
template <int HD>
__device__ inline void load_v(PairI4<HD>& r, const AttnArgs& a, const int (&blk)[2], int kvh, int lane) {
    constexpr int S = HD / 32;
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
        const uint8_t* p = a.vpool + ((size_t)(uint32_t)blk[pg] * (uint32_t)a.hkv + (uint32_t)kvh) * page_bytes(HD);
        load_words<S>(r.v[pg], p + lane_offset((uint32_t)lane * (4 * S)));
        load_scales<S>(r.vs[pg], p + 8 * HD + lane_offset(((uint32_t)lane >> 4) * (8 * S)));
    }
}

// (Loaded as data used once, 8 sequences of 4096 took 28.3 us in place of 29.4, but
// 5 of 3000 17.6 in place of 15.9 and most smaller ones longer, too.)
template <int HD>
struct PairF16 {
    h8_t k[2][HD / 32];
    u2_t v[HD / 16][2];
};

template <int HD>
__device__ inline void load_k(PairF16<HD>& r, const AttnArgs& a, const int (&blk)[2], int kvh, int lane) {
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
        const uint8_t* p = a.kpool + ((size_t)(uint32_t)blk[pg] * (uint32_t)a.hkv + (uint32_t)kvh) * (2 * kPage * HD);
#pragma unroll
        for (int s = 0; s < HD / 32; ++s) r.k[pg][s] = *reinterpret_cast<const h8_t*>(p + 2u * ((lane & 15u) * HD + 8u * ((uint32_t)lane >> 4)) + 64 * s);
    }
}
template <int HD>
__device__ inline void load_v(PairF16<HD>& r, const AttnArgs& a, const int (&blk)[2], int kvh, int lane) {
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
        const uint8_t* p = a.vpool + ((size_t)(uint32_t)blk[pg] * (uint32_t)a.hkv + (uint32_t)kvh) * (2 * kPage * HD);
#pragma unroll
        for (int nt = 0; nt < HD / 16; ++nt) r.v[nt][pg] = *reinterpret_cast<const u2_t*>(p + 2u * ((lane & 15u) * kPage + 4u * ((uint32_t)lane >> 4)) + 32 * kPage * nt);
    }
}

struct H2x4 {
    half2_t h[4];
};

// Codes of half a dword (nibbles 0 and 4, 1 and 5) as fp16 values code - 8:
// 0x6400 is 1024, whose last bits a nibble sets; both steps are exact.
__device__ inline uint32_t and_or(uint32_t w, uint32_t mask, uint32_t bits) {
    uint32_t v;  // (the compiler takes two instructions for it, as two of the operands are constants)
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(v) : "v"(w), "s"(mask), "v"(bits));
    return v;
}
__device__ inline half2_t low_codes(uint32_t w) {
    const half2_t v = __builtin_bit_cast(half2_t, and_or(w, 0x000F000Fu, 0x64006400u));
    return v + half2_t{(_Float16)-1032.0f, (_Float16)-1032.0f};
}
__device__ inline half2_t high_codes(uint32_t w) {  // 1024 + 16 code
    const half2_t v = __builtin_bit_cast(half2_t, and_or(w, 0x00F000F0u, 0x64006400u));
    return __builtin_elementwise_fma(v, half2_t{(_Float16)0.0625f, (_Float16)0.0625f}, half2_t{(_Float16)-72.0f, (_Float16)-72.0f});
}
__device__ inline h8_t codes8(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(h8_t, H2x4{low_codes(a), high_codes(a), low_codes(b), high_codes(b)});
}

// K's codes as they are: a nibble in the last bits of a half is the subnormal
// number code 2^-24, in the next four code 2^-20, and the products take both
// exactly, so a mask is all that a pair of codes takes.  q's dimensions 2, 3, 6
// and 7 of eight are 1/16 of what they were, and a product begins at -8 times
// q's sum over its 32 dimensions.  (V's cannot go so: what taking off 8 p leaves,
// 2^-21 of a scale, would stand where every value is 0.)
struct W4 {
    uint32_t w[4];
};
__device__ inline h8_t raw_codes8(uint32_t w) {
    return __builtin_bit_cast(h8_t, W4{w & 0x000F000Fu, w & 0x00F000F0u, w >> 8 & 0x000F000Fu, w >> 8 & 0x00F000F0u});
}

// ------------------------------------------------------------ scores of a pair --
template <int HD>
__device__ inline void scores(const PairI4<HD>& r, const h8_t* q, const f4_t* off, f4_t (&s)[2]) {
    s[0] = s[1] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
        const h8_t qi = q[i * kWave];
        const f4_t o = off[i * 16];
#pragma unroll
        for (int pg = 0; pg < 2; ++pg) {
            const f4_t d = __builtin_amdgcn_mfma_f32_16x16x32_f16(raw_codes8(r.k[pg][i]), qi, o, 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) s[pg][j] = __builtin_fmaf(d[j], (float)r.ks[pg][i][j], s[pg][j]);
        }
        if (i % 2) __builtin_amdgcn_sched_barrier(0);
    }
}

template <int HD>
__device__ inline void scores(const PairF16<HD>& r, const h8_t* q, const f4_t*, f4_t (&s)[2]) {
    s[0] = s[1] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
        const h8_t qi = q[i * kWave];
#pragma unroll
        for (int pg = 0; pg < 2; ++pg) s[pg] = __builtin_amdgcn_mfma_f32_16x16x32_f16(r.k[pg][i], qi, s[pg], 0, 0, 0);
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
}

// Tokens past a page's valid ones may hold anything, and their probability, 0,
// must not meet a NaN: the int4 scales and the fp16 values become zeros.
template <int HD>
__device__ inline void clear_past(PairI4<HD>& r, int na, int nb, int lane) {
    const uint2 m[2] = {at::vmask_of(na, lane >> 4), at::vmask_of(nb, lane >> 4)};
#pragma unroll
    for (int pg = 0; pg < 2; ++pg)
#pragma unroll
        for (int i = 0; i < HD / 32; ++i)
            r.vs[pg][i] = __builtin_bit_cast(h4_t, __builtin_bit_cast(u2_t, r.vs[pg][i]) & u2_t{m[pg].x, m[pg].y});
}
template <int HD>
__device__ inline void clear_past(PairF16<HD>& r, int na, int nb, int lane) {
    const uint2 m[2] = {at::vmask_of(na, lane >> 4), at::vmask_of(nb, lane >> 4)};
#pragma unroll
    for (int pg = 0; pg < 2; ++pg)
#pragma unroll
        for (int nt = 0; nt < HD / 16; ++nt) r.v[nt][pg] &= u2_t{m[pg].x, m[pg].y};
}

// One wavefront's state over its pairs of pages: a column's reference m (of
// scores times log2 e), this lane's part of its sum, and O.  Probabilities are
// exp2(s - m + up), up to 2^15 instead of 1, so that small ones stay normal
// fp16 numbers (below 2^-14 fp16 loses bits); L and O have the same factor.
// The reference is the first pair's maximum and follows a larger one only when
// that is more than 2^kLead ahead (kUp + kLead is 15): O is hardly ever
// multiplied through.  int4 pages: `up` is kUp less what large scales ask for, and
// O of a group of 32 dimensions has 2^(kUp - down) in place of 2^up (make_room; the
// same in all lanes).
template <int HD>
struct Fold {
    float m = -__builtin_inff(), l = 0.0f, up = kUp;
    int down[HD / 32] = {};
    f4_t o[HD / 16];
};

// ------------------------------------------------------------ values of a pair --
// P V takes p times the token's scale as fp16 numbers (below).  p is 2^15 at
// most, and as much more as the roundings of scores below kFar give (a tenth in
// the exponent), so with a scale of 1 or more (a value of 8 and up among a
// group) the product could pass the largest fp16 number: from such a pair on
// the wavefront's products for that group go without as many powers of two,
// `down`.  Half of the most that a group asks for is taken from p, for all, and the
// rest from (or back to) the scales, so that neither loses bits to fp16's smallest
// number.  What that leaves out of a token's term is 2^-34 of the group's largest |V|
// among the wavefront's tokens and 2^-28 of its own.
template <int HD>
__device__ inline void make_room(Fold<HD>& f, PairI4<HD>& r) {
    typedef uint16_t us2_t __attribute__((ext_vector_type(2)));
    typedef uint16_t us4_t __attribute__((ext_vector_type(4)));
    us2_t any = {0, 0};
#pragma unroll
    for (int pg = 0; pg < 2; ++pg)
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
            const us4_t w = __builtin_bit_cast(us4_t, r.vs[pg][i]);
            any = __builtin_elementwise_max(any, __builtin_elementwise_max(__builtin_shufflevector(w, w, 0, 1), __builtin_shufflevector(w, w, 2, 3)));
        }
    // biased exponents: 15 is 2^0 (31 no number, 32 and up a negative one's)
    if (!__any(max((int)any.x, (int)any.y) >= 15 << 10) && f.up == kUp) return;
    int top = 0;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
        us4_t most = {0, 0, 0, 0};
#pragma unroll
        for (int pg = 0; pg < 2; ++pg) {
            const us4_t size = __builtin_bit_cast(us4_t, r.vs[pg][i]) & (uint16_t)0x7FFFu;
            most = __builtin_elementwise_max(most, size & __builtin_bit_cast(us4_t, size < (uint16_t)0x7C00u));  // (no factor makes the others' products finite)
        }
        const int e = max(max((int)most[0], (int)most[1]), max((int)most[2], (int)most[3])) >> 10;
        const int d = max(f.down[i], __builtin_amdgcn_readfirstlane((int)wave_max((float)e)) - 14);
        const float by = ldexpf(1.0f, f.down[i] - d);
        f.o[2 * i] *= by;
        f.o[2 * i + 1] *= by;
        f.down[i] = d;
        top = max(top, d);
        __builtin_amdgcn_sched_barrier(0);
    }
    const int half = (top + 1) / 2;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
        const _Float16 by = (_Float16)ldexpf(1.0f, half - f.down[i]);  // 2^-8 to 2^8
        r.vs[0][i] *= h4_t{by, by, by, by};
        r.vs[1][i] *= h4_t{by, by, by, by};
    }
    const float up = kUp - (float)half;
    f.l *= __builtin_amdgcn_exp2f(up - f.up);
    f.up = up;
}
template <int HD>
__device__ inline void make_room(Fold<HD>&, const PairF16<HD>&) {}

// The lanes of columns 8-15 (those with bit 3), which hold the same
// probabilities as columns 0-7: rows 0-7 of a product take the fp16 high parts
// of the heads' factors and rows 8-15 the low parts.
__device__ inline bool low_part() { return __builtin_amdgcn_inverse_ballot_w64(0xFF00FF00FF00FF00ull); }

// o += P V.  p: probabilities of tokens 4 g + j of page a (j < 4) and page b.
// int4 pages: the factors are p times the token's scale.  The high part is the
// rounded product of p's high part and the scale, the low part what that
// rounding left out (exactly: one fused step) and the product with p's low
// part, so both are 2^-21 of a factor, or fp16's smallest number.  (The high
// part alone, 2^-11, is what an output rounds to, but of its terms'
// magnitudes, not of their sum: it made outputs differ by 3e-4.)
template <int HD>
__device__ inline void values(const PairI4<HD>& r, const float (&p)[8], f4_t (&o)[HD / 16], int) {
    H2x4 part, less;  // p's own part; in lanes of low parts p's high one, negative, else 0
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const half2_t hi = {(_Float16)p[2 * j], (_Float16)p[2 * j + 1]};
        const half2_t lo = {(_Float16)(p[2 * j] - (float)hi.x), (_Float16)(p[2 * j + 1] - (float)hi.y)};
        const uint32_t h = __builtin_bit_cast(uint32_t, hi), l = __builtin_bit_cast(uint32_t, lo);
        part.h[j] = __builtin_bit_cast(half2_t, low_part() ? l : h);
        less.h[j] = __builtin_bit_cast(half2_t, low_part() ? h ^ 0x80008000u : 0u);
    }
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
        const H2x4 vs = __builtin_bit_cast(H2x4, __builtin_shufflevector(r.vs[0][i], r.vs[1][i], 0, 1, 2, 3, 4, 5, 6, 7));
        H2x4 ps;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            ps.h[j] = __builtin_elementwise_fma(part.h[j], vs.h[j], __builtin_elementwise_fma(-less.h[j], vs.h[j], less.h[j] * vs.h[j]));
        const h8_t a = __builtin_bit_cast(h8_t, ps);
        o[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, codes8(r.v[0][i], r.v[1][i]), o[2 * i], 0, 0, 0);
        o[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, codes8(r.v[0][i] >> 8, r.v[1][i] >> 8), o[2 * i + 1], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// fp16 pages: the factors are the probabilities themselves.
template <int HD>
__device__ inline void values(const PairF16<HD>& r, const float (&p)[8], f4_t (&o)[HD / 16], int lane) {
    const bool low = lane & 8;
    h8_t ps;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const _Float16 hi = (_Float16)p[j];
        ps[j] = low ? (_Float16)(p[j] - (float)hi) : hi;
    }
#pragma unroll
    for (int nt = 0; nt < HD / 16; ++nt) {
        const h8_t v = __builtin_bit_cast(h8_t, __builtin_shufflevector(r.v[nt][0], r.v[nt][1], 0, 1, 2, 3));
        o[nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ps, v, o[nt], 0, 0, 0);
    }
}

// ------------------------------------------------------------------- k_attn --
// q as operands in LDS, by the whole block: [step][lane] 8 fp16 values.  Column
// t < 8 is the high part of head h0 + t (zero past H), column 8 + t its low
// part.  A power of two per head brings its largest value to 512 and up, so
// that low parts are normal fp16 numbers and no high part overflows; scale[t]
// takes it back.
template <int HD, bool INT4>
struct StageQ {
    static constexpr int T = HD / 4;  // threads of a head, four dimensions each
    static_assert(T * kHeadsPerBlock <= kThreads && kWave % T == 0, "a head lies in one wavefront");
    f4_t x;
    __device__ void request(const float* q, int H) {
        const int h = threadIdx.x / T, d = 4 * (threadIdx.x % T);
        x = h < H ? *reinterpret_cast<const f4_t*>(q + (size_t)h * HD + d) : f4_t{0.f, 0.f, 0.f, 0.f};
    }
    __device__ void store(_Float16* ops, float* scale, f4_t* off) const {
        const int h = threadIdx.x / T, d = 4 * (threadIdx.x % T);
        if (h >= kHeadsPerBlock) return;
        float top = row16_max(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
        if (T >= 32) top = max_x16(top);
        if (T >= 64) top = max_x32(top);
        const int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23);
        const int up = e == 0 || e == 255 ? 0 : min(136 - e, 126);
        h4_t hi, lo;
        float sum[2] = {0.0f, 0.0f};  // of the parts, times -8 2^-24
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float part = INT4 && j >= 2 ? 0.0625f : 1.0f, y = ldexpf(x[j], up) * part;  // (raw_codes8)
            hi[j] = (_Float16)y;
            lo[j] = (_Float16)(y - (float)hi[j]);
            sum[0] = __builtin_fmaf((float)hi[j], -0x1p-21f / part, sum[0]);
            sum[1] = __builtin_fmaf((float)lo[j], -0x1p-21f / part, sum[1]);
        }
        if (INT4)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float v = sum[i] + dpp<kQuadXor1>(sum[i]);
                v += dpp<kQuadXor2>(v);
                v += dpp<kRowHalfMirror>(v);
                if (d % 32 == 0) off[d / 32 * 16 + h + 8 * i] = f4_t{v, v, v, v};
            }
        const int at = ((d / 32) * kWave + 16 * (d % 32 / 8)) * 8 + d % 8;
        *reinterpret_cast<h4_t*>(ops + at + 8 * h) = hi;
        *reinterpret_cast<h4_t*>(ops + at + 8 * (h + 8)) = lo;
        // codes enter as code 2^-24 (2^120 at most: scores of such a q are far apart anyway)
        if (d == 0) scale[h] = ldexpf(kLog2e / sqrtf((float)HD), INT4 ? min(24 - up, 120) : -up);
    }
};

// A pair of pages into the state.  The next pair's K is requested once this
// one's has become scores, its V once this one's is added: half a pair is in
// flight all the time, in registers that are free anyway.
template <int HD, bool ACC, class Pair, class Next>
__device__ inline void fold(Fold<HD>& f, Pair& r, const h8_t* q, const f4_t* off, float scale, int na, int nb, float* raw, int lane, Next next_k) {
    const int g = lane >> 4;
    f4_t s[2];
    scores<HD>(r, q, off, s);
    // (here, not after the next request, whose registers these were)
    asm volatile("" : "+v"(s[0]), "+v"(s[1]));
    next_k();
    float p[8], top = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        p[j] = s[j / 4][j % 4] + dpp<kRowRor8>(s[j / 4][j % 4]);
        // An infinite key gives infinities and NaN by the signs of q's two parts:
        // NaN for any.  (No finite one passes fp32 here.)
        p[j] = __builtin_fmaf(p[j], 0.0f, p[j]);
    }
    if (nb < kPage) {
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = 4 * g + j % 4 < (j < 4 ? na : nb) ? p[j] : -__builtin_inff();
        clear_past<HD>(r, na, nb, lane);
    }
    if constexpr (ACC) {
        if (raw) {
            reinterpret_cast<f4_t*>(raw)[0] = f4_t{p[0], p[1], p[2], p[3]} * scale;
            if (nb > 0) reinterpret_cast<f4_t*>(raw)[4] = f4_t{p[4], p[5], p[6], p[7]} * scale;
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, p[j]);
    top = max_x32(max_x16(top)) * scale;  // over the column's four lanes
    // Far from 0 (kFar) a step of the scores' 24 bits is near the powers of two
    // that p has to spare: there they are rounded and taken from the maximum
    // itself before anything is added.
    const bool far = fabsf(top) > kFar && top != -__builtin_inff();  // (of a column: heads go by their own scores)
    const float mn = top > (far ? f.m : f.m + kLead) ? top : f.m;
    const bool none = mn == -__builtin_inff();  // no token, or NaN scores alone
    make_room<HD>(f, r);
    const float up = f.up;
    const float corr = none ? 1.0f : __builtin_amdgcn_exp2f(f.m - mn);
    float by = scale, from = none ? 0.0f : mn - up, sum = 0.0f;
    if (__any(far)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = far ? p[j] * scale - mn : p[j];
        by = far ? 1.0f : by;
        from = far ? -up : from;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[j], by, -from));
        sum += p[j];
    }
    f.l = f.l * corr + sum;
    // rows of O are heads: their factors lie in the lanes of that column (there
    // is no O yet where the maximum was not one)
    if (__any(corr != 1.0f && f.m != -__builtin_inff())) {
        float c[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = __shfl(corr, 4 * g + j, 64);
#pragma unroll
        for (int nt = 0; nt < HD / 16; ++nt)
#pragma unroll
            for (int j = 0; j < 4; ++j) f.o[nt][j] *= c[j];
    }
    f.m = mn;
    values<HD>(r, p, f.o, lane);
}

__device__ inline void store_out(uint16_t* out, f4_t v) {
    *reinterpret_cast<uint2*>(out) =
        make_uint2((uint32_t)f2h_bits(v[0]) | ((uint32_t)f2h_bits(v[1]) << 16), (uint32_t)f2h_bits(v[2]) | ((uint32_t)f2h_bits(v[3]) << 16));
}

// The weight of a score, from its head's M and 1 / L.
__device__ inline float part_of(float score, float2 norm) { return __builtin_amdgcn_exp2f(score - norm.x + kUp) * norm.y; }

template <int HD, bool INT4, bool ACC>
__global__ __launch_bounds__(kThreads, HD * (INT4 ? 1 : 2) <= 128 ? 4 : 2) void k_attn(AttnArgs a) {
    using Pair = typename std::conditional<INT4, PairI4<HD>, PairF16<HD>>::type;
    constexpr int kRec = kHeadsPerBlock * (HD + 2);
    __shared__ __align__(16) float lds[kWaves * kRec];
    __shared__ h8_t qops[HD / 32 * kWave];
    __shared__ float qscale[kHeadsPerBlock];
    __shared__ f4_t qoff[INT4 ? HD / 32 * 16 : 1];  // what K's products begin at
    __shared__ float2 norm[kHeadsPerBlock];  // without a join: a head's M (NaN: refused) and 1 / L
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, t = lane & 15;
    const int split = blockIdx.x, kvh = blockIdx.y / a.plan.groups, grp = blockIdx.y % a.plan.groups, b = blockIdx.z;
    const int G = a.hq / a.hkv, H = min(kHeadsPerBlock, G - kHeadsPerBlock * grp), h0 = kvh * G + kHeadsPerBlock * grp;
    const int cap = a.max_blocks * kPage;
    const int stride = a.plan.splits * kWaves, first = split + a.plan.splits * wave;
    // q and the table entries of the first 32 pairs (two lanes each) are
    // requested with the length, not behind it
    StageQ<HD, INT4> stage;
    stage.request(a.q + ((size_t)b * a.hq + h0) * HD, H);
    const int32_t* table = a.table + (size_t)b * a.max_blocks;
    auto entry_of = [&](int i) {
        const int page = 2 * (first + stride * (i + lane / 2)) + (lane & 1);
        return page < a.max_blocks ? table[page] : 0;
    };
    int entry = entry_of(0);
    int ctx = a.lens[b];
    bool bad = ctx < 0 || ctx > cap;
    ctx = bad ? 0 : ctx;
    const int npages = (ctx + kPage - 1) / kPage, npairs = (npages + 1) / 2;
    const int mine = first < npairs ? (npairs - first + stride - 1) / stride : 0;
    int blk[2];
    Pair r;
    // the pages of pair i of this wavefront, in order
    auto turn_to = [&](int i) {
        if (i % (kWave / 2) == 0) {
            if (i > 0) entry = entry_of(i);
            const bool used = 2 * (first + stride * (i + lane / 2)) + (lane & 1) < npages, out = entry < 0 || entry >= a.num_blocks;
            bad = bad || __any(used && out);
            entry = used && !out ? entry : 0;
        }
        // (a page that the sequence does not have has entry 0 and no valid token)
        blk[0] = __builtin_amdgcn_readlane(entry, 2 * (i % (kWave / 2)));
        blk[1] = __builtin_amdgcn_readlane(entry, 2 * (i % (kWave / 2)) + 1);
    };
    if (mine > 0) {
        turn_to(0);
        load_k<HD>(r, a, blk, kvh, lane);
    }
    stage.store(reinterpret_cast<_Float16*>(qops), qscale, qoff);
    __syncthreads();
    const h8_t* q = qops + lane;
    const f4_t* off = qoff + t;
    const float scale = qscale[t & 7];
    Fold<HD> f;
#pragma unroll
    for (int nt = 0; nt < HD / 16; ++nt) f.o[nt] = f4_t{0.f, 0.f, 0.f, 0.f};
    auto use = [&](int i, auto next_k) {
        const int page = 2 * (first + stride * i);
        float* raw = ACC && t < H ? a.raw + ((size_t)b * a.hq + h0 + t) * cap + page * kPage + 4 * g : nullptr;
        fold<HD, ACC>(f, r, q, off, scale, min(ctx - page * kPage, kPage), min(max(ctx - (page + 1) * kPage, 0), kPage), raw, lane, next_k);
    };
    // (the last pair apart: a request that may not come makes the waits for
    // others wait for all; heads of 256 need one branch around all requests for
    // that, which costs the others registers)
    auto fold_all = [&] {
        for (int i = 0; i + 1 < mine; ++i) {
            use(i, [&] {
                turn_to(i + 1);
                load_k<HD>(r, a, blk, kvh, lane);
            });
            load_v<HD>(r, a, blk, kvh, lane);
        }
    };
    if constexpr (INT4 && HD == 256) {
        if (mine > 0) {
            load_v<HD>(r, a, blk, kvh, lane);
            fold_all();
            use(mine - 1, [] {});
        }
    } else {
        if (mine > 0) load_v<HD>(r, a, blk, kvh, lane);
        fold_all();
        if (mine > 0) use(mine - 1, [] {});
    }
    const float l = ldexpf(sum_x32(sum_x16(f.l)), (int)(kUp - f.up));  // records have 2^kUp
    // rows 8-15 onto rows 0-7: tile 2 k's sums in the lower half of the lanes, tile
    // 2 k + 1's in the upper
#pragma unroll
    for (int nt = 0; nt < HD / 16; nt += 2)
#pragma unroll
        for (int j = 0; j < 4; ++j) f.o[nt / 2][j] = halves_sum(f.o[nt][j], f.o[nt + 1][j]);
    // one record per wavefront in LDS: O[8][HD], M[8], L[8] (rows past H hold anything)
    constexpr int MO = kHeadsPerBlock * HD, LO = MO + kHeadsPerBlock;
    float* my = lds + wave * kRec;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) my[(4 * (g & 1) + j) * HD + 32 * i + 16 * (g >> 1) + t] = ldexpf(f.o[i][j], f.down[i]);
    if (lane < kHeadsPerBlock) {
        // M is NaN where the length or the table is out of range
        my[MO + lane] = bad ? __builtin_nanf("") : f.m;
        my[LO + lane] = l;
    }
    __syncthreads();
    const size_t row = (size_t)b * a.hkv * a.plan.groups + blockIdx.y;
    float* part = a.part + (row * a.plan.splits + split) * a.plan.rec;
    const int MP = a.plan.heads * HD, LP = MP + a.plan.heads;  // of a record in memory
    uint16_t* out = a.out + ((size_t)b * a.hq + h0) * HD;
    for (int x = 4 * threadIdx.x; x < H * HD; x += 4 * kThreads) {
        const int h = x / HD;
        float mw[kWaves], M = -__builtin_inff(), L = 0.0f;
        bool no = false;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            mw[w] = lds[w * kRec + MO + h];
            no = no || mw[w] != mw[w];
            M = fmaxf(M, mw[w]);
        }
        f4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float e = M == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(mw[w] - M);
            acc += e * *reinterpret_cast<const f4_t*>(lds + w * kRec + x);
            L = fmaf(e, lds[w * kRec + LO + h], L);
        }
        if (a.plan.join) {
            *reinterpret_cast<f4_t*>(part + x) = acc;
            if (x % HD == 0) {
                part[MP + h] = no ? __builtin_nanf("") : M;
                part[LP + h] = L;
            }
        } else {  // the one block of its kv head
            const float il = no ? __builtin_nanf("") : L == 0.0f ? 0.0f : 1.0f / L;
            store_out(out + x, acc * il);
            if (ACC && x % HD == 0) norm[h] = make_float2(no ? __builtin_nanf("") : M, il);
        }
    }
    if constexpr (ACC) {
        if (a.plan.join) return;
        __syncthreads();
        if (norm[0].x != norm[0].x) return;
        const float* raw = a.raw + ((size_t)b * a.hq + h0) * cap;
        float* weights = a.weights + ((size_t)b * a.hkv + kvh) * cap;
        for (int s = threadIdx.x; s < ctx; s += kThreads) {
            float acc = 0.0f;
#pragma unroll
            for (int h = 0; h < kHeadsPerBlock; ++h)
                if (h < H) acc += part_of(raw[(size_t)h * cap + s], norm[h]);
            weights[s] += acc;
        }
    }
}

// ------------------------------------------------------------------- k_join --
// The first `outs` blocks of a (kv head, sequence) merge the
// records into 32 float4 columns of the output each, eight threads to a column;
// the others turn 256 slots' scores into weights at a time.
constexpr int kJoinThreads = 256, kJoinCols = 32;
constexpr int kJoinHeads = 64;  // query heads of a kv head

template <int HD>
__global__ __launch_bounds__(kJoinThreads) void k_join(AttnArgs a, int outs) {
    __shared__ float fac[kJoinHeads * kMaxSplits];
    __shared__ float2 norm[kJoinHeads];
    __shared__ f4_t sums[kJoinThreads];
    __shared__ int refused;
    const int kvh = blockIdx.y, b = blockIdx.z, G = a.hq / a.hkv, ns = a.plan.splits, tid = threadIdx.x, rec = a.plan.rec;
    const float* parts = a.part + ((size_t)b * a.hkv + kvh) * a.plan.groups * ns * rec;
    const bool output = (int)blockIdx.x < outs;
    // the thread's first slot's scores and weight are requested ahead of all else
    const int cap = a.max_blocks * kPage, slot = ((int)blockIdx.x - outs) * kJoinThreads + tid;
    const float* raw = a.raw + ((size_t)b * a.hq + (size_t)kvh * G) * cap;
    float* weights = a.weights + ((size_t)b * a.hkv + kvh) * cap;
    // (an output block's: its first eight splits' columns)
    const int total = G * HD / 4, col = blockIdx.x * kJoinCols + tid % kJoinCols, c = min(col, total - 1), split0 = tid / kJoinCols;
    constexpr int step = kJoinThreads / kJoinCols, kAhead = 8;
    const float* column = parts + (size_t)(4 * c / HD / kHeadsPerBlock) * ns * rec + 4 * c % (kHeadsPerBlock * HD);
    float early[8], was = 0.0f;
    f4_t v[kAhead];
    if (output) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) v[u] = *reinterpret_cast<const f4_t*>(column + (size_t)min(split0 + u * step, ns - 1) * rec);
    } else {
        const int s = min(slot, cap - 1);
#pragma unroll
        for (int h = 0; h < 8; ++h) early[h] = raw[(size_t)min(h, G - 1) * cap + s];
        was = weights[s];
    }
    if (tid == 0) refused = 0;
    __syncthreads();
    // wavefront w: heads w, w + 4, ..; lane s: split s
    const int lane = tid & 63, slane = min(lane, ns - 1);
    for (int h0 = tid / kWave; h0 < G; h0 += 4 * kJoinThreads / kWave) {
        float m[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int h = min(h0 + i * kJoinThreads / kWave, G - 1);
            const float* p = parts + ((size_t)(h / kHeadsPerBlock) * ns + slane) * rec + a.plan.heads * HD + h % kHeadsPerBlock;
            m[i] = p[0];
            l[i] = p[a.plan.heads];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int h = h0 + i * kJoinThreads / kWave;
            if (h >= G) break;
            const float M = wave_max(m[i]);  // (past the last split: that one again)
            const float e = lane >= ns ? 0.0f : M == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m[i] - M), L = wave_sum(lane < ns ? e * l[i] : 0.0f);
            const bool no = __any(m[i] != m[i]);
            const float il = no ? __builtin_nanf("") : L == 0.0f ? 0.0f : 1.0f / L;
            if (lane < ns) fac[h * kMaxSplits + lane] = no ? il : e * il;
            if (lane == 0) {
                norm[h] = make_float2(M, il);
                if (no) refused = 1;
            }
        }
    }
    __syncthreads();
    if (output) {
        static_assert(kAhead * step >= kMaxSplits, "all of a column's splits");
        const int h = 4 * c / HD;
        f4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (split0 + u * step < ns) acc += fac[h * kMaxSplits + split0 + u * step] * v[u];
        sums[tid] = acc;
        __syncthreads();
        if (tid < kJoinCols && col < total) {
            for (int i = 1; i < step; ++i) acc += sums[i * kJoinCols + tid];
            store_out(a.out + ((size_t)b * a.hq + (size_t)kvh * G) * HD + 4 * col, acc);
        }
        return;
    }
    if (refused) return;
    const int ctx = a.lens[b], stride = ((int)gridDim.x - outs) * kJoinThreads;
    if (slot < ctx) {
        float acc = 0.0f;
#pragma unroll
        for (int h = 0; h < 8; ++h)
            if (h < G) acc += part_of(early[h], norm[h]);
        for (int h = 8; h < G; ++h) acc += part_of(raw[(size_t)h * cap + slot], norm[h]);
        weights[slot] = was + acc;
    }
    for (int64_t s = (int64_t)slot + stride; s < ctx; s += stride) {
        float acc = 0.0f;
#pragma unroll 8
        for (int h = 0; h < G; ++h) acc += part_of(raw[(size_t)h * cap + s], norm[h]);
        weights[s] += acc;
    }
}

template <int HD, bool INT4>
hipError_t attn_case(const AttnArgs& a, hipStream_t st) {
    const dim3 grid(a.plan.splits, a.hkv * a.plan.groups, a.batch);
    if (a.weights)
        hipLaunchKernelGGL((k_attn<HD, INT4, true>), grid, dim3(kThreads), 0, st, a);
    else if constexpr (INT4)  // (fp16 pages without weights are nx_attn.hip's)
        hipLaunchKernelGGL((k_attn<HD, true, false>), grid, dim3(kThreads), 0, st, a);
    if (!a.plan.join) return hipGetLastError();
    const int outs = (a.hq / a.hkv * HD / 4 + kJoinCols - 1) / kJoinCols;
    const int slots = a.weights ? std::min(128, (a.max_blocks * kPage + kJoinThreads - 1) / kJoinThreads) : 0;
    hipLaunchKernelGGL(k_join<HD>, dim3(outs + slots, a.hkv, a.batch), dim3(kJoinThreads), 0, st, a, outs);
    return hipGetLastError();
}

// The part of a plan that the heads decide.
AttnPlan heads_plan(int hq, int hkv, int hd) {
    const int G = hq / hkv, heads = std::min(G, kHeadsPerBlock);
    return {(G + kHeadsPerBlock - 1) / kHeadsPerBlock, heads, 1, (heads * (hd + 2) + 3) / 4 * 4, true};
}

}  // namespace

AttnPlan attn_plan(int batch, int hq, int hkv, int hd, int max_blocks, bool int4, bool weights) {
    AttnPlan p = heads_plan(hq, hkv, hd);
    const int pairs = (max_blocks + 1) / 2;
    // The splits of the least time, in steps of 10 ns, from sweeps over 1 to 64
    // splits of contexts of 100 to 16384: 2.1 us for the launch; 1 us for each
    // block that a compute unit gets, and for eight pairs of it 0.8 us (int4) or
    // 1.4 us (fp16) per 64 dimensions, 15 % less where it holds two blocks at
    // once, 0.4 of that and up for fewer than eight pairs; 3 us and a little per
    // split for records and join, or without a join half a microsecond for eight
    // pairs' weights.  (8 kv heads of 128, int4: 512 tokens 6.9 us in one block
    // each and 8.5 in eight with a join, 1024 tokens 10.1 and 8.5; 8 sequences of
    // 8192 21.2 us in four, 19.5 in eight; 6 of 2500, 8 heads of 64, fp16: 11.5 us
    // in five, 12.8 in twelve.)
    const int64_t rows = (int64_t)batch * hkv * p.groups, cus = device_cus(), pair = (int4 ? 80 : 140) * (hd / 64);
    const bool joined = weights && p.groups > 1, two = hd * (int4 ? 1 : 2) <= 128;
    int64_t least = INT64_MAX;
    for (int s = 1; s <= std::min(kMaxSplits, pairs); ++s) {
        const bool join = s > 1 || joined;
        const int64_t of = (pairs + s - 1) / s, blocks = (rows * s + cus - 1) / cus;  // pairs of a block, blocks of a compute unit
        const int64_t busy = of <= 4 ? 16 + 3 * of : of < 8 ? 24 + 2 * of : 5 * of;     // 40: eight pairs
        const int64_t block = 100 + pair * busy * (two && blocks > 1 ? 17 : 20) / 800 + (weights && !join ? 50 * of / 8 : 0);
        const int64_t cost = 210 + blocks * block + (join ? 300 + 3 * s : 0);
        if (cost < least) {
            least = cost;
            p.splits = s;
        }
    }
    p.join = p.splits > 1 || joined;
    return p;
}

size_t attn_part_floats(const AttnPlan& p, int batch, int hkv) { return (size_t)batch * hkv * p.groups * p.splits * p.rec; }
// (Records grow with the heads that share a kv head but for steps of eight, so
// fewer kv heads can take more: each number with the most heads for it.  A call of
// fewer rows may split its pages further: up to the most splits.)
size_t attn_most_part_floats(int batch, int hq, int hkv, int hd, int max_blocks, int max_group) {
    size_t most = 0;
    for (int h = 1; h <= std::min(hq, hkv); ++h) {
        AttnPlan p = heads_plan(std::min(hq / h, max_group) * h, h, hd);
        p.splits = std::min(kMaxSplits, (max_blocks + 1) / 2);
        most = std::max(most, attn_part_floats(p, batch, h));
    }
    return most;
}

hipError_t attn_launch(const AttnArgs& a, bool int4, hipStream_t st) {
    switch (a.hd) {
        case 64: return int4 ? attn_case<64, true>(a, st) : attn_case<64, false>(a, st);
        case 128: return int4 ? attn_case<128, true>(a, st) : attn_case<128, false>(a, st);
        case 256: return int4 ? attn_case<256, true>(a, st) : attn_case<256, false>(a, st);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace kvc
}  // namespace nx
