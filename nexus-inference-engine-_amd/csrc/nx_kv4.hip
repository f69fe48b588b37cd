// Rows into and out of int4-g32 KV pages.
//
// A block takes one page of one kv head, K or V: 16 tokens x hd values, eight
// to a thread.  Four neighbouring threads hold a group of 32 and agree on its
// scale through DPP.  Both directions are bound by memory (4.5625 bytes a
// value); K codes leave the threads as the dwords of their page, V codes, whose
// dwords hold four tokens each, cross through LDS.
#include "nx_kvc.h"

namespace nx {
namespace kvc {

namespace {

template <int CTRL>
__device__ inline uint32_t dpp_u(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}

// The page a block works on (row_page), and its record of head h: null where
// no row lies in it, the positions are refused or the table names no block of
// the pool.
template <int HD>
__device__ inline uint8_t* page_record(const RowArgs& a, const RowPage& p, int b, int h, bool v) {
    if (p.none || p.refused) return nullptr;
    const int blk = a.table[(size_t)b * a.max_blocks + p.page];
    if (blk < 0 || blk >= a.num_blocks) return nullptr;
    return (v ? a.vpool : a.kpool) + ((size_t)blk * a.hkv + h) * page_bytes(HD);
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

// Code 0..15 of x: the quotient rounded to fp32, then half away from zero.
__device__ inline uint32_t code_of(float x, float s) {
    if (!(s > 0.0f)) return 8u;  // scale 0 or NaN
    const float r = fminf(fmaxf(roundf(__fdiv_rn(x, s)), -8.0f), 7.0f);
    return (uint32_t)((int)r + 8);
}

template <int HD>
__global__ __launch_bounds__(2 * HD) void k_append_int4(RowArgs a) {
    constexpr int S = HD / 32, C = HD / 8;
    const int h = blockIdx.y >> 1, b = blockIdx.z, tid = threadIdx.x;
    const bool v = blockIdx.y & 1;
    const RowPage pr = row_page(a.start[b], a.tokens, a.max_blocks, blockIdx.x);
    uint8_t* rec = page_record<HD>(a, pr, b, h, v);
    if (!rec) return;
    const int t = tid / C, c = tid % C, row = pr.row0 + t;
    const bool have = row >= 0 && row < a.tokens;
    float x[8] = {};
    if (have) {
        const float4* src = reinterpret_cast<const float4*>((v ? a.v : a.k) + (((size_t)b * a.tokens + row) * a.hkv + h) * HD + 8 * c);
        const float4 lo = src[0], hi = src[1];
        x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w, x[4] = hi.x, x[5] = hi.y, x[6] = hi.z, x[7] = hi.w;
    }
    uint32_t amax = 0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = max(amax, __builtin_bit_cast(uint32_t, x[j]) & 0x7FFFFFFFu);
    const uint16_t s16 = group_scale(amax);
    const float s = h2f_bits(s16);
    uint16_t* scales = reinterpret_cast<uint16_t*>(rec + 8 * HD);
    if (have && c % 4 == 0) scales[scale_at(HD, t, c / 4)] = s16;
    uint32_t* words = reinterpret_cast<uint32_t*>(rec);
    if (!v) {
        uint32_t w = 0u;
#pragma unroll
        for (int j = 0; j < 8; ++j) w |= code_of(x[j], s) << (4 * k_nib(j));
        if (have) words[k_word(HD, t, 8 * c)] = w;
        return;
    }
    __shared__ uint8_t codes[kPage * HD];
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j / 4] |= code_of(x[j], s) << (8 * (j % 4));
    *reinterpret_cast<uint2*>(codes + t * HD + 8 * c) = make_uint2(w[0], w[1]);
    __syncthreads();
    // thread tid owns dword tid: tokens 4 g + j of dimensions d and d + 16
    const int i = tid % S, n = (tid / S) % 16, g = tid / S / 16, d = 32 * i + n;
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
    if (mask == 0xFFFFFFFFu)
        words[tid] = out;
    else if (mask)
        words[tid] = (words[tid] & ~mask) | out;
}

template <int HD>
__global__ __launch_bounds__(2 * HD) void k_read_int4(RowArgs a) {
    constexpr int S = HD / 32, C = HD / 8;
    const int h = blockIdx.y >> 1, b = blockIdx.z, tid = threadIdx.x;
    const bool v = blockIdx.y & 1;
    const RowPage pr = row_page(a.start[b], a.tokens, a.max_blocks, blockIdx.x);
    if (pr.none) return;
    const uint8_t* rec = page_record<HD>(a, pr, b, h, v);
    const int t = tid / C, c = tid % C, row = pr.row0 + t;
    const bool have = row >= 0 && row < a.tokens;
    float* dst = (v ? a.v : a.k) + (((size_t)b * a.tokens + row) * a.hkv + h) * HD + 8 * c;
    if (!rec) {
        const float nan = __builtin_nanf("");
        if (have) {
            reinterpret_cast<float4*>(dst)[0] = make_float4(nan, nan, nan, nan);
            reinterpret_cast<float4*>(dst)[1] = make_float4(nan, nan, nan, nan);
        }
        return;
    }
    const float s = h2f_bits(reinterpret_cast<const uint16_t*>(rec + 8 * HD)[scale_at(HD, t, c / 4)]);
    const uint32_t* words = reinterpret_cast<const uint32_t*>(rec);
    float x[8];
    if (!v) {
        const uint32_t w = words[k_word(HD, t, 8 * c)];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (float)((int)((w >> (4 * k_nib(j))) & 15u) - 8) * s;
    } else {
        __shared__ uint8_t codes[kPage * HD];
        const uint32_t w = words[tid];
        const int i = tid % S, n = (tid / S) % 16, g = tid / S / 16, d = 32 * i + n;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) codes[(4 * g + j) * HD + d + 16 * e] = (uint8_t)((w >> (4 * v_nib(j, 16 * e))) & 15u);
        __syncthreads();
        const uint2 q = *reinterpret_cast<const uint2*>(codes + t * HD + 8 * c);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (float)((int)(((j < 4 ? q.x : q.y) >> (8 * (j % 4))) & 255u) - 8) * s;
    }
    if (have) {
        reinterpret_cast<float4*>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
}

dim3 row_grid(const RowArgs& a) { return dim3((unsigned)row_pages(a.tokens), (unsigned)(2 * a.hkv), (unsigned)a.batch); }

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
