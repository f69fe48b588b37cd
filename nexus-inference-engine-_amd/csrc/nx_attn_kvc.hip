// Decode attention over int4-g32 pages, and over fp16 pages with the weight
// of every cached token added to an array.
//
// Two launches.  k_attn: a block of 8 wavefronts takes every splits-th pair of
// pages of one kv head for up to 8 of its query heads, keeps an online softmax
// per head, merges its wavefronts through LDS and writes one record (O, M, L);
// with weights it also writes the scores.  k_join: blocks share the merge of
// the records into the fp16 output and, with weights, turn the scores into
// exp(s - M) / L and add their sum over the query heads of the kv head.  (The
// scores need M and L of all splits, which no block of k_attn has; reading
// them back costs 8 bytes a token and query head, the pages again would cost 9/16
// byte or more a value.)
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
// product, in front of V's with the probability.
#include <algorithm>
#include <type_traits>

#include "nx_attn_dev.h"
#include "nx_kvc.h"

namespace nx {
namespace kvc {

namespace {

using at::as_h8;
using at::f4_t;
using at::h8_t;

constexpr int kWaves = 8;
constexpr int kThreads = kWaves * kWave;
constexpr int kMaxSplits = 64;
constexpr int kRowRor8 = 0x128;
// Probabilities are exp2(s - max + kUp): up to 2^15 instead of 1, so that the
// small ones stay normal fp16 numbers (below 2^-14 fp16 loses bits).  L is the
// sum of the same values, and O / L does not see the factor.
constexpr float kUp = 15.0f;
constexpr float kLog2e = 1.4426950408889634f;

// ------------------------------------------------------------------- pages --
// A lane's share of a pair of pages.
template <int HD>
struct PairI4 {
    uint32_t k[2][HD / 32], v[2][HD / 32];  // codes: K of token l%16, V of tokens 4 g .. +3
    uint2 ks[2][HD / 32], vs[2][HD / 32];   // scales of tokens 4 g .. +3 per group
};

// N dwords that start at a multiple of 4 N bytes (of 16 where N is above 4).
template <int N>
__device__ inline void load_words(uint32_t (&r)[N], const uint8_t* p) {
    if constexpr (N == 2) {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        r[0] = w.x, r[1] = w.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 w = reinterpret_cast<const uint4*>(p)[i / 4];
            r[i] = w.x, r[i + 1] = w.y, r[i + 2] = w.z, r[i + 3] = w.w;
        }
    }
}
template <int N>
__device__ inline void load_pairs(uint2 (&r)[N], const uint8_t* p) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const uint4 w = reinterpret_cast<const uint4*>(p)[i / 2];
        r[i] = make_uint2(w.x, w.y), r[i + 1] = make_uint2(w.z, w.w);
    }
}

template <int HD>
__device__ inline void load_pair(PairI4<HD>& r, const AttnArgs& a, int blka, int blkb, int kvh, int lane) {
    constexpr int S = HD / 32;
    const int g = lane >> 4, t = lane & 15;
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
        const size_t base = ((size_t)(pg ? blkb : blka) * a.hkv + kvh) * page_bytes(HD);
        load_words<S>(r.k[pg], a.kpool + base + (t * 4 + g) * (4 * S));
        load_pairs<S>(r.ks[pg], a.kpool + base + 8 * HD + g * (8 * S));
        load_words<S>(r.v[pg], a.vpool + base + lane * (4 * S));
        load_pairs<S>(r.vs[pg], a.vpool + base + 8 * HD + g * (8 * S));
    }
}

template <int HD>
struct PairF16 {
    uint4 k[2][HD / 32];
    uint2 v[HD / 16][2];
};

template <int HD>
__device__ inline void load_pair(PairF16<HD>& r, const AttnArgs& a, int blka, int blkb, int kvh, int lane) {
    const int g = lane >> 4, t = lane & 15;
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
        const size_t base = ((size_t)(pg ? blkb : blka) * a.hkv + kvh) * (2 * kPage * HD);
#pragma unroll
        for (int s = 0; s < HD / 32; ++s)
            r.k[pg][s] = *reinterpret_cast<const uint4*>(a.kpool + base + 2 * (t * HD + 32 * s + 8 * g));
#pragma unroll
        for (int nt = 0; nt < HD / 16; ++nt)
            r.v[nt][pg] = *reinterpret_cast<const uint2*>(a.vpool + base + 2 * ((16 * nt + t) * kPage + 4 * g));
    }
}

// Codes of half a dword (nibbles 0 and 4, 1 and 5) as fp16 values code - 8:
// 0x6400 is 1024, whose last bits a nibble sets; both steps are exact.
__device__ inline half2_t low_codes(uint32_t w) {
    const half2_t v = __builtin_bit_cast(half2_t, (w & 0x000F000Fu) | 0x64006400u);
    return v + half2_t{(_Float16)-1032.0f, (_Float16)-1032.0f};
}
__device__ inline half2_t high_codes(uint32_t w) {  // 1024 + 16 code
    const half2_t v = __builtin_bit_cast(half2_t, (w & 0x00F000F0u) | 0x64006400u);
    return __builtin_elementwise_fma(v, half2_t{(_Float16)0.0625f, (_Float16)0.0625f}, half2_t{(_Float16)-72.0f, (_Float16)-72.0f});
}
struct H2x4 {
    half2_t h[4];
};
__device__ inline h8_t codes8(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(h8_t, H2x4{low_codes(a), high_codes(a), low_codes(b), high_codes(b)});
}

__device__ inline float half_of(uint2 w, int i) { return h2f_bits((uint16_t)((i < 2 ? w.x : w.y) >> (16 * (i & 1)))); }

// ------------------------------------------------------------ scores of a pair --
template <int HD>
__device__ inline void scores(const PairI4<HD>& r, const h8_t (&q)[HD / 32], f4_t (&s)[2]) {
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
        f4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
            const h8_t k = codes8(r.k[pg][i], r.k[pg][i] >> 8);
            const f4_t d = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[i], f4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] = fmaf(d[j], half_of(r.ks[pg][i], j), acc[j]);
        }
        s[pg] = acc;
    }
}

template <int HD>
__device__ inline void scores(const PairF16<HD>& r, const h8_t (&q)[HD / 32], f4_t (&s)[2]) {
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
        f4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(r.k[pg][i]), q[i], acc, 0, 0, 0);
        s[pg] = acc;
    }
}

// ------------------------------------------------------------ values of a pair --
// o += P V.  p: probabilities of tokens 4 g + j of page a (j < 4) and page b.
// The product takes p times the token's scale, rounded to fp16: at most
// 2^-11 of a term, which stays linear in the output (an fp16 number itself).
// p is up to 2^15, so a scale of 2 or more (a value of 16 and up among a
// group) could pass the largest fp16 number: such a pair goes without the factor
// 2^15 and its sums get it afterwards.
template <int HD>
__device__ inline void values(const PairI4<HD>& r, const float (&p)[8], int na, int nb, f4_t (&o)[HD / 16], int lane) {
    constexpr int S = HD / 32;
    const int g = lane >> 4;
    uint2 vs[2][S];
    uint32_t seen = 0u;
    // scales of tokens past the page's valid ones may be anything
    const uint2 m[2] = {at::vmask_of(na, g), at::vmask_of(nb, g)};
#pragma unroll
    for (int pg = 0; pg < 2; ++pg)
#pragma unroll
        for (int i = 0; i < S; ++i) {
            vs[pg][i] = make_uint2(r.vs[pg][i].x & m[pg].x, r.vs[pg][i].y & m[pg].y);
            seen |= vs[pg][i].x | vs[pg][i].y;
        }
    const bool large = __any((seen & 0x40004000u) != 0u);  // an exponent of 2^1 and up
    const float down = large ? 1.0f / 32768.0f : 1.0f;
#pragma unroll
    for (int i = 0; i < S; ++i) {
        h8_t ps;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float sc = half_of(vs[j / 4][i], j % 4);
            ps[j] = (_Float16)(large ? p[j] * down * sc : p[j] * sc);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t wa = e ? r.v[0][i] >> 8 : r.v[0][i], wb = e ? r.v[1][i] >> 8 : r.v[1][i];
            const h8_t v = codes8(wa, wb);
            f4_t& acc = o[2 * i + e];
            if (large) {
                const f4_t d = __builtin_amdgcn_mfma_f32_16x16x32_f16(ps, v, f4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j] = fmaf(d[j], 32768.0f, acc[j]);
            } else {
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ps, v, acc, 0, 0, 0);
            }
        }
    }
}

// fp16 pages: rows 0-7 of the product take the fp16 high parts of the heads'
// probabilities and rows 8-15 (the lanes of columns 8-15) the low parts.
template <int HD>
__device__ inline void values(const PairF16<HD>& r, const float (&p)[8], int na, int nb, f4_t (&o)[HD / 16], int lane) {
    const int g = lane >> 4;
    const bool low = lane & 8;
    h8_t ps;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const _Float16 hi = (_Float16)p[j];
        ps[j] = low ? (_Float16)(p[j] - (float)hi) : hi;
    }
    // V words of tokens past the valid ones may be anything
    const uint2 ma = at::vmask_of(na, g), mb = at::vmask_of(nb, g);
#pragma unroll
    for (int nt = 0; nt < HD / 16; ++nt) {
        const h8_t v = as_h8(make_uint4(r.v[nt][0].x & ma.x, r.v[nt][0].y & ma.y, r.v[nt][1].x & mb.x, r.v[nt][1].y & mb.y));
        o[nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ps, v, o[nt], 0, 0, 0);
    }
}

// ------------------------------------------------------------------- k_attn --
template <int HD, bool INT4, bool ACC>
__global__ __launch_bounds__(kThreads) void k_attn(AttnArgs a) {
    __shared__ __align__(16) float lds[kWaves * kHeadsPerBlock * (HD + 2)];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, t = lane & 15;
    const int split = blockIdx.x, kvh = blockIdx.y / a.plan.groups, grp = blockIdx.y % a.plan.groups, b = blockIdx.z;
    const int G = a.hq / a.hkv, H = min(kHeadsPerBlock, G - kHeadsPerBlock * grp), h0 = kvh * G + kHeadsPerBlock * grp;
    const int cap = a.max_blocks * kPage;
    int ctx = a.lens[b];
    bool bad = ctx < 0 || ctx > cap;
    ctx = bad ? 0 : ctx;
    // q: column t % 8 is head h0 + t % 8 (zero past H), the low part from
    // column 8 on.  A power of two per head brings its largest value to 512 and
    // up, so that low parts are normal fp16 numbers and no high part overflows.
    h8_t q[HD / 32];
    float scale = kLog2e / sqrtf((float)HD);
    {
        const bool on = (t & 7) < H;
        const float* src = a.q + ((size_t)b * a.hq + h0 + (on ? t & 7 : 0)) * HD + 8 * g;
        float x[HD / 32][8], top = 0.0f;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
            const float4 lo = reinterpret_cast<const float4*>(src + 32 * i)[0], hi = reinterpret_cast<const float4*>(src + 32 * i)[1];
            const float y[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[i][j] = y[j];
                top = fmaxf(top, fabsf(y[j]));
            }
        }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23);
        const int up = e == 0 || e == 255 ? 0 : min(136 - e, 126);
        scale = ldexpf(scale, -up);
#pragma unroll
        for (int i = 0; i < HD / 32; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = ldexpf(x[i][j], up);
                const _Float16 hi = (_Float16)y;
                const _Float16 v = t < 8 ? hi : (_Float16)(y - (float)hi);
                q[i][j] = on ? v : (_Float16)0.0f;
            }
    }
    const int npages = (ctx + kPage - 1) / kPage, npairs = (npages + 1) / 2;
    const int stride = a.plan.splits * kWaves, first = split + a.plan.splits * wave;
    const int mine = first < npairs ? (npairs - first + stride - 1) / stride : 0;
    float m = -__builtin_inff(), l = 0.0f;
    f4_t o[HD / 16];
#pragma unroll
    for (int nt = 0; nt < HD / 16; ++nt) o[nt] = f4_t{0.f, 0.f, 0.f, 0.f};
    for (int base = 0; base < mine; base += kWave / 2) {
        // the table entries of the next 32 pairs, two lanes each
        const int my_page = 2 * (first + stride * (base + lane / 2)) + (lane & 1);
        int entry = my_page < npages ? a.table[(size_t)b * a.max_blocks + my_page] : 0;
        const bool out = entry < 0 || entry >= a.num_blocks;
        bad = bad || __any(out);
        entry = out ? 0 : entry;
        const int n = min(mine - base, kWave / 2);
        for (int i = 0; i < n; ++i) {
            const int page = 2 * (first + stride * (base + i));
            const int na = min(ctx - page * kPage, kPage), nb = min(max(ctx - (page + 1) * kPage, 0), kPage);
            const int blka = __builtin_amdgcn_readlane(entry, 2 * i), blkb = nb > 0 ? __builtin_amdgcn_readlane(entry, 2 * i + 1) : blka;
            typename std::conditional<INT4, PairI4<HD>, PairF16<HD>>::type r;
            load_pair<HD>(r, a, blka, blkb, kvh, lane);
            f4_t s[2];
            scores<HD>(r, q, s);
            float p[8];
            float top = -__builtin_inff();
#pragma unroll
            for (int pg = 0; pg < 2; ++pg)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x = (s[pg][j] + dpp<kRowRor8>(s[pg][j])) * scale;
                    p[4 * pg + j] = 4 * g + j < (pg ? nb : na) ? x : -__builtin_inff();
                    top = fmaxf(top, p[4 * pg + j]);
                }
            if constexpr (ACC) {
                if (t < H) {
                    float4* dst = reinterpret_cast<float4*>(a.raw + ((size_t)b * a.hq + h0 + t) * cap + page * kPage + 4 * g);
                    dst[0] = make_float4(p[0], p[1], p[2], p[3]);
                    if (nb > 0) dst[4] = make_float4(p[4], p[5], p[6], p[7]);
                }
            }
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float mn = fmaxf(m, top);
            const bool none = mn == -__builtin_inff();
            const float corr = none ? 1.0f : __builtin_amdgcn_exp2f(m - mn), at0 = mn - kUp;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                p[j] = none ? (p[j] == p[j] ? 0.0f : p[j]) : __builtin_amdgcn_exp2f(p[j] - at0);
                sum += p[j];
            }
            l = l * corr + sum;
            m = mn;
            // rows of O are heads: their factors lie in the lanes of that column
            if (__any(corr != 1.0f)) {
                float c[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) c[j] = __shfl(corr, 4 * g + j, 64);
#pragma unroll
                for (int nt = 0; nt < HD / 16; ++nt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[nt][j] *= c[j];
            }
            values<HD>(r, p, na, nb, o, lane);
        }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if constexpr (!INT4) {  // the low parts' rows
#pragma unroll
        for (int nt = 0; nt < HD / 16; ++nt)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[nt][j] += __shfl_xor(o[nt][j], 32, 64);
    }
    // one record per wavefront in LDS: O[H][HD], M[H], L[H]
    const int rec = H * (HD + 2);
    float* my = lds + wave * rec;
#pragma unroll
    for (int nt = 0; nt < HD / 16; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (4 * g + j < H) my[(4 * g + j) * HD + 16 * nt + t] = o[nt][j];
    if (g == 0 && t < H) {
        // M is NaN where the length or the table is out of range
        my[H * HD + t] = bad ? __builtin_nanf("") : m;
        my[H * HD + H + t] = l;
    }
    __syncthreads();
    float* part = a.part + (((size_t)b * a.hkv * a.plan.groups + blockIdx.y) * a.plan.splits + split) * a.plan.rec;
    for (int x = threadIdx.x; x < H * HD; x += kThreads) {
        const int h = x / HD;
        float M = -__builtin_inff(), acc = 0.0f, L = 0.0f;
        bool no = false;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float mw = lds[w * rec + H * HD + h];
            no = no || mw != mw;
            M = fmaxf(M, mw);
        }
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = M == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(lds[w * rec + H * HD + h] - M);
            acc = fmaf(f, lds[w * rec + x], acc);
            L = fmaf(f, lds[w * rec + H * HD + H + h], L);
        }
        part[x] = acc;
        if (x % HD == 0) {
            part[a.plan.heads * HD + h] = no ? __builtin_nanf("") : M;
            part[a.plan.heads * HD + a.plan.heads + h] = L;
        }
    }
}

// ------------------------------------------------------------------- k_join --
// Block (j, kv head, sequence): the j-th share of the kv head's output and, with
// weights, of its slots.
constexpr int kJoinThreads = 256;
constexpr int kJoinHeads = 64;  // query heads of a kv head

template <int HD, bool ACC>
__global__ __launch_bounds__(kJoinThreads) void k_join(AttnArgs a) {
    __shared__ float fac[kJoinHeads * kMaxSplits], top[kJoinHeads], inv[kJoinHeads];
    __shared__ int refused;
    const int kvh = blockIdx.y, b = blockIdx.z, G = a.hq / a.hkv, ns = a.plan.splits, tid = threadIdx.x;
    const float* parts = a.part + ((size_t)b * a.hkv + kvh) * a.plan.groups * ns * a.plan.rec;
    if (tid == 0) refused = 0;
    __syncthreads();
    // wavefront w: heads w, w + 4, ..; lane s: split s
    const int lane = tid & 63;
    for (int h = tid / kWave; h < G; h += kJoinThreads / kWave) {
        const float* p = parts + ((size_t)(h / kHeadsPerBlock) * ns + min(lane, ns - 1)) * a.plan.rec + a.plan.heads * HD + h % kHeadsPerBlock;
        const float m = lane < ns ? p[0] : -__builtin_inff(), l = lane < ns ? p[a.plan.heads] : 0.0f;
        const float M = wave_max(m);
        const bool none = M == -__builtin_inff();
        const float e = none ? 1.0f : __builtin_amdgcn_exp2f(m - M), L = wave_sum(e * l);
        const bool no = __any(m != m);
        const float il = no ? __builtin_nanf("") : L == 0.0f ? 0.0f : 1.0f / L;
        if (lane < ns) fac[h * kMaxSplits + lane] = no ? il : e * il;
        if (lane == 0) {
            top[h] = M - kUp;
            inv[h] = il;
            if (no) refused = 1;
        }
    }
    __syncthreads();
    const int total = G * HD, per = ((total + (int)gridDim.x - 1) / (int)gridDim.x + 3) / 4 * 4;
    uint16_t* out = a.out + ((size_t)b * a.hq + (size_t)kvh * G) * HD;
    const int end = min(total, (int)(blockIdx.x + 1) * per);
    for (int x = (int)blockIdx.x * per + 4 * tid; x < end; x += 4 * kJoinThreads) {
        const int h = x / HD;
        const float* p = parts + (size_t)(h / kHeadsPerBlock) * ns * a.plan.rec + (h % kHeadsPerBlock) * HD + x % HD;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int s = 0; s < ns; ++s) {
            const float4 v = *reinterpret_cast<const float4*>(p + (size_t)s * a.plan.rec);
            const float f = fac[h * kMaxSplits + s];
            acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
        }
        *reinterpret_cast<uint2*>(out + x) = make_uint2((uint32_t)f2h_bits(acc.x) | ((uint32_t)f2h_bits(acc.y) << 16),
                                                        (uint32_t)f2h_bits(acc.z) | ((uint32_t)f2h_bits(acc.w) << 16));
    }
    if constexpr (ACC) {
        if (refused) return;
        const int cap = a.max_blocks * kPage, ctx = a.lens[b];
        float* w = a.weights + ((size_t)b * a.hkv + kvh) * cap;
        const float* raw = a.raw + ((size_t)b * a.hq + (size_t)kvh * G) * cap;
        for (int s = (int)blockIdx.x * kJoinThreads + tid; s < ctx; s += (int)gridDim.x * kJoinThreads) {
            float acc = 0.0f;
            for (int h = 0; h < G; ++h) acc = fmaf(__builtin_amdgcn_exp2f(raw[(size_t)h * cap + s] - top[h]), inv[h], acc);
            w[s] += acc;
        }
    }
}

template <int HD, bool INT4>
hipError_t attn_case(const AttnArgs& a, hipStream_t st) {
    const dim3 grid(a.plan.splits, a.hkv * a.plan.groups, a.batch);
    const int slots = a.max_blocks * kPage;
    if (a.weights) {
        hipLaunchKernelGGL((k_attn<HD, INT4, true>), grid, dim3(kThreads), 0, st, a);
        const unsigned n = (unsigned)std::min(64, std::max(1, slots / (2 * kJoinThreads)));
        hipLaunchKernelGGL((k_join<HD, true>), dim3(n, a.hkv, a.batch), dim3(kJoinThreads), 0, st, a);
    } else {
        hipLaunchKernelGGL((k_attn<HD, INT4, false>), grid, dim3(kThreads), 0, st, a);
        const unsigned n = (unsigned)std::max(1, a.hq / a.hkv * HD / 128);
        hipLaunchKernelGGL((k_join<HD, false>), dim3(n, a.hkv, a.batch), dim3(kJoinThreads), 0, st, a);
    }
    return hipGetLastError();
}

}  // namespace

AttnPlan attn_plan(int batch, int hq, int hkv, int hd, int max_blocks) {
    AttnPlan p;
    const int G = hq / hkv, pairs = (max_blocks + 1) / 2;
    p.groups = (G + kHeadsPerBlock - 1) / kHeadsPerBlock;
    p.heads = std::min(G, kHeadsPerBlock);
    p.rec = (p.heads * (hd + 2) + 3) / 4 * 4;
    // two blocks to a compute unit, and a pair of pages at least to a wavefront
    const int64_t rows = (int64_t)batch * hkv * p.groups;
    const int64_t want = (2 * (int64_t)device_cus() + rows - 1) / rows;
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({want, (pairs + kWaves - 1) / kWaves, kMaxSplits}));
    return p;
}

size_t attn_part_floats(const AttnPlan& p, int batch, int hkv) { return (size_t)batch * hkv * p.groups * p.splits * p.rec; }

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
