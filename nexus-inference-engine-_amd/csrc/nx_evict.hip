// Eviction of cached tokens by the attention weight they gathered.
//
// Per sequence and kv head the `keep` slots of highest rank stay (recent
// tokens first, then by weight, then the lower slot), and the tokens kept from
// slots beyond `keep` move into the slots that others left below it, the i-th
// to the i-th, both in ascending order.  Attention does not ask for an order of
// its slots, so nothing else moves: sources lie at keep and above,
// destinations below, and no copy can overtake another.
//
// k_pick, one block per (sequence, kv head): a radix selection over 32-bit
// keys (11, 11 and 10 bits) finds the keep-th largest, ballots number the
// equal ones, the free slots and the tokens that move in slot order, and the
// weights and tags are written.  k_move, one wavefront per destination page:
// K vectors as they are; V, whose pages are dimension-major, by rewriting the
// page's words, each of which one lane owns.
#include <algorithm>

#include "nx_kvc.h"

namespace nx {
namespace kvc {

namespace {

constexpr int kPickThreads = 1024, kPickWaves = kPickThreads / kWave;
constexpr int kBins = 2048;

// The words a (sequence, kv head) has in the workspace: keys, then where each
// kept slot's token comes from (-1: it stays), then the tokens that move.
struct Row {
    uint32_t* keys;
    int32_t *src, *from;
};
__host__ __device__ inline int kept_slots(int max_blocks, int keep) {
    const int cap = max_blocks * kPage;
    return keep < cap ? (keep + kPage - 1) / kPage * kPage : cap;
}
__device__ inline Row row_of(const EvictArgs& a, int b, int h) {
    const size_t cap = (size_t)a.max_blocks * kPage, ks = kept_slots(a.max_blocks, a.keep);
    uint32_t* p = a.ws + ((size_t)b * a.hkv + h) * (cap + 2 * ks);
    return {p, reinterpret_cast<int32_t*>(p + cap), reinterpret_cast<int32_t*>(p + cap + ks)};
}
__device__ inline int32_t* new_lens(const EvictArgs& a) {
    const size_t cap = (size_t)a.max_blocks * kPage, ks = kept_slots(a.max_blocks, a.keep);
    return reinterpret_cast<int32_t*>(a.ws + (size_t)a.batch * a.hkv * (cap + 2 * ks));
}

// Order of weights as unsigned numbers: NaN below every other, -0 as 0.
__device__ inline uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive sums of v over the block in thread order, and their total.
__device__ inline int block_scan(int v, int* lds, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int y = __shfl_up(x, o, kWave);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == kWave - 1) lds[wave] = x;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int w = 0; w < kPickWaves; ++w) {
        before += w < wave ? lds[w] : 0;
        total += lds[w];
    }
    return before + x - v;
}

__global__ __launch_bounds__(kPickThreads) void k_pick(EvictArgs a) {
    __shared__ uint32_t hist[kBins];
    __shared__ int sums[kPickWaves], found_bin, found_left;
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int cap = a.max_blocks * kPage, keep = a.keep, L = a.lens_in[b], N = a.seen[b], ks = kept_slots(a.max_blocks, keep);
    const Row r = row_of(a, b, h);
    const size_t at = ((size_t)b * a.hkv + h) * cap;
    const float* w_in = a.weights_in + at;
    const int32_t* t_in = a.tags_in + at;
    float* w_out = a.weights_out + at;
    int32_t* t_out = a.tags_out + at;
    bool bad = L < 0 || L > cap || N < L;
    if (!bad)
        for (int p = tid; p < (L + kPage - 1) / kPage; p += kPickThreads) {
            const int blk = a.table[(size_t)b * a.max_blocks + p];
            bad = bad || blk < 0 || blk >= a.num_blocks;
        }
    bad = __syncthreads_or(bad);
    if (tid == 0 && h == 0) new_lens(a)[b] = bad ? -1 : min(L, keep);
    // a token's position + 1: its tag, or its place among the tokens
    // appended since the last call
    auto tag_of = [&](int s) {
        const int t = t_in[s];
        return t > 0 ? t : N - L + s + 1;
    };
    if (bad || L <= keep) {
        for (int s = tid; s < ks; s += kPickThreads) r.src[s] = -1;
        if (bad) return;
        for (int s = tid; s < cap; s += kPickThreads) {
            const float w = s < L ? w_in[s] : 0.0f;
            const int t = s < L ? tag_of(s) : 0;
            w_out[s] = w;
            t_out[s] = t;
        }
        return;
    }
    // a wavefront takes a run of slots, 64 at a time
    const int run = (L + kPickThreads - 1) / kPickThreads * kWave, s0 = wave * run, s1 = min(L, s0 + run);
    // ---- the keep-th largest key
    uint32_t prefix = 0u, mask = 0u;
    int left = keep;
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
        for (int i = tid; i < kBins; i += kPickThreads) hist[i] = 0u;
        __syncthreads();
        for (int s = s0 + lane; s < s1; s += kWave) {
            uint32_t key;
            if (pass == 0) {
                key = tag_of(s) > N - a.recent ? 0xFFFFFFFFu : weight_key(w_in[s]);
                r.keys[s] = key;
            } else {
                key = r.keys[s];
            }
            if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & (bins - 1)], 1u);
        }
        __syncthreads();
        // thread i: bins 2047 - 2 i and 2046 - 2 i, the largest keys first
        const int hi = (int)hist[kBins - 1 - 2 * tid], lo = (int)hist[kBins - 2 - 2 * tid];
        int total;
        const int before = block_scan(hi + lo, sums, total);
        if (before < left && left <= before + hi + lo) {
            const bool first = left <= before + hi;
            found_bin = first ? kBins - 1 - 2 * tid : kBins - 2 - 2 * tid;
            found_left = left - before - (first ? 0 : hi);
        }
        __syncthreads();
        prefix |= (uint32_t)found_bin << shift;
        mask |= (uint32_t)(bins - 1) << shift;
        left = found_left;
        __syncthreads();
    }
    // ---- keys above the prefix stay, of the equal ones the `left` lowest slots
    int total, equal = 0;
    for (int s = s0 + lane; s < s1; s += kWave) equal += r.keys[s] == prefix;
    // (a wavefront's lanes in one sum: the scan is by thread, its run by wavefront)
    for (int o = 1; o < kWave; o <<= 1) equal += __shfl_xor(equal, o, kWave);
    const int eq0 = __shfl(block_scan(lane == 0 ? equal : 0, sums, total), 0, kWave);
    int holes0 = 0, moves0 = 0;
    for (int write = 0; write < 2; ++write) {
        int eq = eq0, holes = holes0, moves = moves0;
        for (int s = s0 + lane; s - lane < s1; s += kWave) {
            const uint32_t key = s < s1 ? r.keys[s] : 0u;
            const unsigned long long below = (1ull << lane) - 1ull;
            const unsigned long long same = __ballot(s < s1 && key == prefix);
            const bool kept = s < s1 && (key > prefix || (key == prefix && eq + __popcll(same & below) < left));
            const unsigned long long hole = __ballot(s < s1 && s < keep && !kept), move = __ballot(kept && s >= keep);
            if (write) {
                const bool mine = hole >> lane & 1ull;
                if (s < min(s1, keep)) r.src[s] = mine ? holes + __popcll(hole & below) : -1;
                if (move >> lane & 1ull) r.from[moves + __popcll(move & below)] = s;
            }
            eq += __popcll(same);
            holes += __popcll(hole);
            moves += __popcll(move);
        }
        if (!write) {
            const int x = block_scan(lane == 0 ? holes : 0, sums, total), y = block_scan(lane == 0 ? moves : 0, sums, total);
            holes0 = __shfl(x, 0, kWave);
            moves0 = __shfl(y, 0, kWave);
        }
    }
    __syncthreads();
    // ---- the kept slots' weights and tags; then nothing beyond them
    for (int s = tid; s < ks; s += kPickThreads) {
        if (s >= keep) {
            r.src[s] = -1;
            continue;
        }
        const int i = r.src[s], m = i < 0 ? s : r.from[i];
        if (i >= 0) r.src[s] = m;
        const float w = w_in[m];
        const int t = tag_of(m);
        w_out[s] = w;
        t_out[s] = t;
    }
    __syncthreads();
    for (int s = keep + tid; s < cap; s += kPickThreads) {
        w_out[s] = 0.0f;
        t_out[s] = 0;
    }
}

constexpr int kMoveWaves = 4;

// Where slot s of sequence b lies: its page's record of head h, and the token in it.
template <int BYTES>
__device__ inline size_t page_at(const EvictArgs& a, int b, int h, int s) {
    return ((size_t)a.table[(size_t)b * a.max_blocks + s / kPage] * a.hkv + h) * BYTES;
}

template <int HD, bool INT4>
__global__ __launch_bounds__(kMoveWaves * kWave) void k_move(EvictArgs a) {
    constexpr int BYTES = INT4 ? page_bytes(HD) : 2 * kPage * HD, S = HD / 32;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = blockIdx.y, b = blockIdx.z;
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) a.lens_out[b] = new_lens(a)[b];
    const int page = blockIdx.x * kMoveWaves + wave, ks = kept_slots(a.max_blocks, a.keep);
    if (page * kPage >= ks) return;
    // lane t < 16: where the page's slot t gets its token from
    const int from = lane < kPage ? row_of(a, b, h).src[page * kPage + lane] : -1;
    const unsigned moved = (unsigned)__ballot(from >= 0);
    if (!moved) return;
    const size_t dst = page_at<BYTES>(a, b, h, page * kPage);
    const size_t src = from >= 0 ? page_at<BYTES>(a, b, h, from) : 0;
    for (unsigned left = moved; left; left &= left - 1) {
        const int t = __builtin_ctz(left), u = __builtin_amdgcn_readlane(from, t) % kPage;
        const size_t sp = ((size_t)(uint32_t)__builtin_amdgcn_readlane((int)(src >> 32), t) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)src, t);
        if constexpr (INT4) {
            const uint32_t* ks32 = reinterpret_cast<const uint32_t*>(a.kpool + sp);
            uint32_t* kd32 = reinterpret_cast<uint32_t*>(a.kpool + dst);
            if (lane < HD / 8) kd32[t * (HD / 8) + lane] = ks32[u * (HD / 8) + lane];
            if (lane < 2 * S) {  // scales: K's, then V's
                uint8_t* pool = lane < S ? a.kpool : a.vpool;
                reinterpret_cast<uint16_t*>(pool + dst + 8 * HD)[scale_at(HD, t, lane % S)] =
                    reinterpret_cast<const uint16_t*>(pool + sp + 8 * HD)[scale_at(HD, u, lane % S)];
            }
            // V: lane n < 16 of quad t / 4 takes the two nibbles of its S dwords
            if (lane >> 4 == t >> 2) {
                const uint32_t* vs32 = reinterpret_cast<const uint32_t*>(a.vpool + sp);
                uint32_t* vd32 = reinterpret_cast<uint32_t*>(a.vpool + dst);
#pragma unroll
                for (int i = 0; i < S; ++i) {
                    const uint32_t w = vs32[(16 * (u >> 2) + (lane & 15)) * S + i];
                    uint32_t d = vd32[lane * S + i];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int ns = 4 * v_nib(u, 16 * e), nd = 4 * v_nib(t, 16 * e);
                        d = (d & ~(15u << nd)) | ((w >> ns & 15u) << nd);
                    }
                    vd32[lane * S + i] = d;
                }
            }
        } else {
            const uint4* k4 = reinterpret_cast<const uint4*>(a.kpool + sp);
            uint4* kd4 = reinterpret_cast<uint4*>(a.kpool + dst);
            if (lane < HD / 8) kd4[t * (HD / 8) + lane] = k4[u * (HD / 8) + lane];
            const uint16_t* vs = reinterpret_cast<const uint16_t*>(a.vpool + sp);
            uint16_t* vd = reinterpret_cast<uint16_t*>(a.vpool + dst);
            for (int d = lane; d < HD; d += kWave) vd[d * kPage + t] = vs[d * kPage + u];
        }
    }
}

template <int HD, bool INT4>
void move_case(const EvictArgs& a, hipStream_t st) {
    const int pages = kept_slots(a.max_blocks, a.keep) / kPage;
    hipLaunchKernelGGL((k_move<HD, INT4>), dim3((unsigned)((pages + kMoveWaves - 1) / kMoveWaves), (unsigned)a.hkv, (unsigned)a.batch),
                       dim3(kMoveWaves * kWave), 0, st, a);
}

}  // namespace

size_t evict_ws_words(int batch, int hkv, int max_blocks, int keep) {
    return (size_t)batch * hkv * ((size_t)max_blocks * kPage + 2 * (size_t)kept_slots(max_blocks, keep)) + batch;
}

hipError_t evict_launch(const EvictArgs& a, bool int4, hipStream_t st) {
    if (a.hd != 64 && a.hd != 128 && a.hd != 256) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_pick, dim3((unsigned)a.hkv, (unsigned)a.batch), dim3(kPickThreads), 0, st, a);
    if (a.hd == 64)
        int4 ? move_case<64, true>(a, st) : move_case<64, false>(a, st);
    else if (a.hd == 128)
        int4 ? move_case<128, true>(a, st) : move_case<128, false>(a, st);
    else
        int4 ? move_case<256, true>(a, st) : move_case<256, false>(a, st);
    return hipGetLastError();
}

}  // namespace kvc
}  // namespace nx
