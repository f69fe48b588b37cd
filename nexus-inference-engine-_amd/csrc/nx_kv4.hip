// Rows into and out of int4-g32 KV pages.
//
// A block takes one page of one kv head, K and V: 16 tokens x hd values of
// each, eight of each to a thread.  Four neighbouring threads hold a group of
// 32 and agree on its scale through DPP.  Both directions are bound by memory
// (4.5625 bytes a value), so everything a block reads is requested together:
// the rows with the table entry, which they do not depend on, K's with V's.  K
// codes leave the threads as the dwords of their page, V codes, whose dwords
// hold four tokens each, cross through LDS.  8192 tokens of 8 kv heads of 128
// (76 MB): 18 us in and 13 us out by turns, when each waits for the other's rows
// to leave the caches.
#include "nx_kvc.h"

namespace nx {
namespace kvc {

namespace {

template <int CTRL>
__device__ inline uint32_t dpp_u(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}

// Offset of a page's record of head h in its pool: -1 where no row lies in the
// page, the positions are refused or the table names no block of the pool.
template <int HD>
__device__ inline int64_t page_record(const RowArgs& a, const RowPage& p, int b, int h) {
    if (p.none || p.refused) return -1;
    const int blk = a.table[(size_t)b * a.max_blocks + p.page];
    return blk < 0 || blk >= a.num_blocks ? -1 : ((int64_t)blk * a.hkv + h) * page_bytes(HD);
}

// Scale of a group from the largest magnitude's bits over the thread's
// eight values: fp16(amax / 7), at most the largest finite one; NaN for a
// group that holds a NaN or an infinity.
__device__ inline uint16_t group_scale(uint32_t amax) {
    amax = max(amax, dpp_u<kQuadXor1>(amax));
    amax = max(amax, dpp_u<kQuadXor2>(amax));
    if (amax >= 0x7F800000u) return 0x7E00u;
    return f2h_bits(fminf(__fdiv_rn(__builtin_bit_cast(float, amax), 7.0f), 65504.0f));
}

// code - 8 of x, as a float: the quotient x / s rounded to fp32, then half away
// from zero, in [-8, 7]; `r` is 1 / s, rounded.  With a rounded reciprocal one
// step of Markstein's iteration gives the rounded quotient (IBM J. Res. Dev. 34
// (1), 1990; s has 11 bits, and quotients that underflow are far from a half): 3
// instructions a value where a division takes ten (one token of 8 sequences: 3.7
// against 4.0 us).
__device__ inline float step_of(float x, float s, float r) {
    const float q0 = x * r, q = __builtin_fmaf(__builtin_fmaf(-q0, s, x), r, q0);
    const float t = __builtin_truncf(q);
    const float n = t + (fabsf(q - t) >= 0.5f ? __builtin_copysignf(1.0f, q) : 0.0f);
    return __builtin_amdgcn_fmed3f(n, -8.0f, 7.0f);
}

typedef float f4_t __attribute__((ext_vector_type(4)));

// A thread's eight values of a row, zeros where it has none.  Rows are read
// once and are loaded as such: 8192 tokens took 25 us otherwise, with what the
// last call left in the caches, and 18.6 so.
struct Eight {
    f4_t lo, hi;
    __device__ void load(const float* p) {
        lo = __builtin_nontemporal_load(reinterpret_cast<const f4_t*>(p));
        hi = __builtin_nontemporal_load(reinterpret_cast<const f4_t*>(p) + 1);
    }
    __device__ float operator[](int j) const { return j < 4 ? lo[j] : hi[j - 4]; }
    __device__ uint16_t scale() const {
        uint32_t amax = 0u;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = (*this)[j];
            amax = max(amax, __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu);
        }
        return group_scale(amax);
    }
    // the values' codes less 8 (zeros for a scale of 0 or NaN)
    __device__ void steps(uint16_t s16, float (&n)[8]) const {
        const float s = h2f_bits(s16), r = __fdiv_rn(1.0f, s);
#pragma unroll
        for (int j = 0; j < 8; ++j) n[j] = s > 0.0f ? step_of((*this)[j], s, r) : 0.0f;
    }
};

template <int HD>
__global__ __launch_bounds__(2 * HD) void k_append_int4(RowArgs a) {
    constexpr int C = HD / 8;
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const RowPage pr = row_page(a.start[b], a.tokens, a.max_blocks, blockIdx.x);
    if (pr.none || pr.refused) return;
    const int t = tid / C, c = tid % C, row = pr.row0 + t;
    const bool have = row >= 0 && row < a.tokens;
    Eight xk{}, xv{};
    if (have) {
        const size_t at = (((size_t)b * a.tokens + row) * a.hkv + h) * HD + 8 * c;
        xk.load(a.k + at);
        xv.load(a.v + at);
    }
    const int64_t rec = page_record<HD>(a, pr, b, h);
    if (rec < 0) return;
    const uint16_t sk = xk.scale(), sv = xv.scale();
    __shared__ uint8_t codes[kPage * HD];
    // codes are gathered as digits of exact floats: four of 4 bits for K (even
    // j in the low half of the dword, odd j in the high), two of 8 for V
    float q[8];
    xk.steps(sk, q);
    auto digits = [](float a, float b, float c, float d) {
        return (uint32_t)__builtin_fmaf(__builtin_fmaf(__builtin_fmaf(d, 16.0f, c), 16.0f, b), 16.0f, a + (float)0x8888);
    };
    const uint32_t w = digits(q[0], q[2], q[4], q[6]) | digits(q[1], q[3], q[5], q[7]) << 16;
    xv.steps(sv, q);
    auto bytes = [](float a, float b) { return (uint32_t)__builtin_fmaf(b, 256.0f, a + (float)0x0808); };
    const uint32_t w2[2] = {bytes(q[0], q[1]) | bytes(q[2], q[3]) << 16, bytes(q[4], q[5]) | bytes(q[6], q[7]) << 16};
    if (have) {
        reinterpret_cast<uint32_t*>(a.kpool + rec)[k_word(HD, t, 8 * c)] = w;
        if (c % 4 == 0) {
            reinterpret_cast<uint16_t*>(a.kpool + rec + 8 * HD)[scale_at(HD, t, c / 4)] = sk;
            reinterpret_cast<uint16_t*>(a.vpool + rec + 8 * HD)[scale_at(HD, t, c / 4)] = sv;
        }
    }
    *reinterpret_cast<uint2*>(codes + t * HD + 8 * c) = make_uint2(w2[0], w2[1]);
    __syncthreads();
    // thread tid owns dword tid of V: tokens 4 g + j of dimensions d and d + 16
    const int g = v_word(HD, tid).g, d = v_word(HD, tid).d;
    uint32_t out = 0u, mask = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int r = pr.row0 + 4 * g + j;
        if (r < 0 || r >= a.tokens) continue;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int nib = 4 * v_nib(j, 16 * e);
            out |= (uint32_t)codes[(4 * g + j) * HD + d + 16 * e] << nib;
            mask |= 15u << nib;
        }
    }
    // tokens of the dword that are not this call's keep their codes
    uint32_t* words = reinterpret_cast<uint32_t*>(a.vpool + rec);
    if (mask == 0xFFFFFFFFu)
        words[tid] = out;
    else if (mask)
        words[tid] = (words[tid] & ~mask) | out;
}

// Four values to a thread of each of two tokens, so that a store's lanes write
// whole lines (with eight of one token 4096 tokens took 14.0 us in place of 12.3).
template <int HD>
__global__ __launch_bounds__(2 * HD) void k_read_int4(RowArgs a) {
    constexpr int C = HD / 4;
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const RowPage pr = row_page(a.start[b], a.tokens, a.max_blocks, blockIdx.x);
    if (pr.none) return;
    const int c = tid % C, t0 = tid / C;
    bool have[2];
    size_t at[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int row = pr.row0 + t0 + 8 * u;
        have[u] = row >= 0 && row < a.tokens;
        at[u] = have[u] ? (((size_t)b * a.tokens + row) * a.hkv + h) * HD + 4 * c : 0;
    }
    const int64_t rec = page_record<HD>(a, pr, b, h);
    if (rec < 0) {
        const float nan = __builtin_nanf("");
#pragma unroll
        for (int u = 0; u < 2; ++u)
            if (have[u])
                for (float* p : {a.k + at[u], a.v + at[u]}) *reinterpret_cast<f4_t*>(p) = f4_t{nan, nan, nan, nan};
        return;
    }
    const uint32_t wv = reinterpret_cast<const uint32_t*>(a.vpool + rec)[tid];
    uint16_t s16[2][2];
    uint32_t wk[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int t = t0 + 8 * u, sat = scale_at(HD, t, c / 8);
        s16[u][0] = reinterpret_cast<const uint16_t*>(a.kpool + rec + 8 * HD)[sat];
        s16[u][1] = reinterpret_cast<const uint16_t*>(a.vpool + rec + 8 * HD)[sat];
        wk[u] = reinterpret_cast<const uint32_t*>(a.kpool + rec)[k_word(HD, t, 4 * c)] >> (c % 2 * 8);
    }
    __shared__ uint8_t codes[kPage * HD];
    const int g = v_word(HD, tid).g, d = v_word(HD, tid).d;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) codes[(4 * g + j) * HD + d + 16 * e] = (uint8_t)((wv >> (4 * v_nib(j, 16 * e))) & 15u);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const uint32_t q = *reinterpret_cast<const uint32_t*>(codes + (t0 + 8 * u) * HD + 4 * c);
        f4_t k, v;
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // (dimensions 4 .. 7 of eight lie one byte on)
            k[j] = (float)((int)((wk[u] >> (4 * k_nib(j))) & 15u) - 8) * h2f_bits(s16[u][0]);
            v[j] = (float)((int)((q >> (8 * j)) & 255u) - 8) * h2f_bits(s16[u][1]);
        }
        if (have[u]) {
            *reinterpret_cast<f4_t*>(a.k + at[u]) = k;
            *reinterpret_cast<f4_t*>(a.v + at[u]) = v;
        }
    }
}

dim3 row_grid(const RowArgs& a) { return dim3((unsigned)row_pages(a.tokens), (unsigned)a.hkv, (unsigned)a.batch); }

}  // namespace

hipError_t append_int4_launch(const RowArgs& a, hipStream_t st) {
    if (a.hd == 64)
        hipLaunchKernelGGL(k_append_int4<64>, row_grid(a), dim3(128), 0, st, a);
    else if (a.hd == 128)
        hipLaunchKernelGGL(k_append_int4<128>, row_grid(a), dim3(256), 0, st, a);
    else if (a.hd == 256)
        hipLaunchKernelGGL(k_append_int4<256>, row_grid(a), dim3(512), 0, st, a);
    else
        return hipErrorInvalidValue;
    return hipGetLastError();
}

hipError_t read_int4_launch(const RowArgs& a, hipStream_t st) {
    if (a.hd == 64)
        hipLaunchKernelGGL(k_read_int4<64>, row_grid(a), dim3(128), 0, st, a);
    else if (a.hd == 128)
        hipLaunchKernelGGL(k_read_int4<128>, row_grid(a), dim3(256), 0, st, a);
    else if (a.hd == 256)
        hipLaunchKernelGGL(k_read_int4<256>, row_grid(a), dim3(512), 0, st, a);
    else
        return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace kvc
}  // namespace nx
