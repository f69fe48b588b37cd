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
// keys (11, 11 and 10 bits), which stay in LDS, finds the keep-th largest;
// ballots number the equal ones, the free slots and the tokens that move in
// slot order.  k_move, a wavefront per destination page of int4 pages and 1 + hd /
// 64 of fp16 ones (K, and 64 dimensions of V each): weights and tags; K vectors
// as they are; V, whose pages are dimension-major, by rewriting the page's words
// (fp16: half rows of eight tokens), each of which one lane owns.
#include <algorithm>

#include "nx_kvc.h"

namespace nx {
namespace kvc {

namespace {

constexpr int kPickThreads = 1024, kPickWaves = kPickThreads / kWave;
constexpr int kBins = 2048, kListed = 2048, kRanked = 128;
constexpr int kKeyPad = 8 * kWave;  // keys past a row's that a wavefront may read
constexpr int kLdsSlots = 32768;  // slots whose keys a block holds in LDS

__host__ __device__ inline int kept_slots(int max_blocks, int keep) {
    const int cap = max_blocks * kPage;
    return keep < cap ? (keep + kPage - 1) / kPage * kPage : cap;
}
// Slots whose keys go through memory: longer rows than LDS holds.
__host__ __device__ inline size_t stored_keys(int max_blocks) {
    const size_t cap = (size_t)max_blocks * kPage;
    return cap > (size_t)kLdsSlots ? (cap + kPickThreads - 1) / kPickThreads * kPickThreads + 8 * kWave : 0;
}

// What k_pick leaves for k_move.  Of a sequence: its new length (-1: refused),
// whether it was cut, and what a slot's number lacks to the tag of a token
// appended since the last call.  Of a (sequence, kv head) that is cut: a bit
// for each slot that stays, 64 to a word; for each word how many slots below
// keep came free before it; and the slots of the tokens that move, in order.
struct Seq {
    int len, cut, ahead;
};
constexpr int kSeqWords = 4;
__device__ inline Seq* seq_of(const EvictArgs& a, int b) { return reinterpret_cast<Seq*>(a.ws + (size_t)b * kSeqWords); }
__host__ __device__ inline size_t bit_words(int max_blocks) { return ((size_t)max_blocks * kPage + kWave - 1) / kWave; }
__host__ __device__ inline size_t row_words(int max_blocks, int keep) {
    return (3 * bit_words(max_blocks) + kept_slots(max_blocks, keep) + stored_keys(max_blocks) + 1) / 2 * 2;
}
struct Row {
    unsigned long long* stays;
    int32_t *free_before, *from;
    uint32_t* keys;
};
__device__ inline Row row_of(const EvictArgs& a, int b, int h) {
    const size_t nw = bit_words(a.max_blocks);
    uint32_t* p = a.ws + (size_t)a.batch * kSeqWords + ((size_t)b * a.hkv + h) * row_words(a.max_blocks, a.keep);
    int32_t* q = reinterpret_cast<int32_t*>(p + 2 * nw);
    return {reinterpret_cast<unsigned long long*>(p), q, q + nw, p + 3 * nw + kept_slots(a.max_blocks, a.keep)};
}

// Order of weights as unsigned numbers: NaN below every other, -0 as 0; no
// weight has key 0, which stands for no token.
__device__ inline uint32_t weight_key(float w) {
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);
    return w != w ? 1u : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

// base + the bits of v below this lane.
__device__ inline int below_lane(unsigned long long v, int base) {
    return (int)__builtin_amdgcn_mbcnt_hi((unsigned)(v >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)v, (unsigned)base));
}

template <int CTRL, int ROWS = 0xF>
__device__ inline int dpp_add(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
// Inclusive sums over the 16 lanes of a row.
__device__ inline int row_scan(int v) {
    v = dpp_add<0x111>(v);  // row_shr:1, 2, 4, 8
    v = dpp_add<0x112>(v);
    v = dpp_add<0x114>(v);
    return dpp_add<0x118>(v);
}
// Inclusive sums over the wavefront's lanes.
__device__ inline int wave_scan(int v) { return dpp_add<kRowBcast31, 0xC>(dpp_add<kRowBcast15, 0xA>(row_scan(v))); }
// Exclusive sums over the block in thread order of two numbers, and their totals.
__device__ inline int2 block_scan(int2 v, int2* lds, int2& total) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int x = wave_scan(v.x), y = wave_scan(v.y);
    __syncthreads();
    if (lane == kWave - 1) lds[wave] = make_int2(x, y);
    __syncthreads();
    static_assert(kPickWaves == 16, "one row of lanes holds the wavefronts' sums");
    const int2 w = lds[lane & 15];
    const int wx = row_scan(w.x), wy = row_scan(w.y);
    total = make_int2(__builtin_amdgcn_readlane(wx, 15), __builtin_amdgcn_readlane(wy, 15));
    const int2 before = wave > 0 ? make_int2(__builtin_amdgcn_readlane(wx, wave - 1), __builtin_amdgcn_readlane(wy, wave - 1)) : make_int2(0, 0);
    return make_int2(before.x + x - v.x, before.y + y - v.y);
}

// SLOTS: the longest row whose keys stay in LDS; 0: they go through memory.
// A block is one compute unit's work: the first loop is bound by what one
// compute unit can request and count (32768 slots: 11000 of 37000 cycles), the
// others by its instructions.  A row's slots are passed three times: keys and
// their top bits are counted, the keys of the bin that holds the keep-th are
// listed, and the keys are compared with the keep-th (twice more where some of
// its equals stay and some go).  8 kv heads of 32768 slots: 18.0 us, of 4352: 8.2 us.
template <int SLOTS>
__global__ __launch_bounds__(kPickThreads) void k_pick(EvictArgs a) {
    // two counters per bin, by lane: weights crowd into few bins
    __shared__ uint2 hist[kBins];
    __shared__ uint32_t lds_keys[SLOTS > 0 ? SLOTS + kKeyPad : 1], list[kListed];
    __shared__ int2 sums[kPickWaves];
    __shared__ int found, found_left, found_all, listed;
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int cap = a.max_blocks * kPage, keep = a.keep, L = a.lens_in[b], N = a.seen[b];
    const Row r = row_of(a, b, h);
    const size_t at = ((size_t)b * a.hkv + h) * cap;
    const float* w_in = a.weights_in + at;
    const int32_t* t_in = a.tags_in + at;
    // The first weights and tags are requested ahead of the lengths, as those of a
    // row that fills its slots (most often right where rows are cut), and the
    // table's entries, which are looked at behind the first loop.
    float w[8];
    int t[8];
    const int guess = (cap + kPickThreads - 1) / kPickThreads;
    auto request_upto = [&](int s, int last) {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = w_in[min(s + j * kWave, last)];
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = t_in[min(s + j * kWave, last)];
    };
    request_upto(wave * guess * kWave + lane, cap - 1);
    const int32_t* table = a.table + (size_t)b * a.max_blocks;
    const int entry[2] = {table[min(tid, a.max_blocks - 1)], table[min(tid + kPickThreads, a.max_blocks - 1)]};
    for (int i = tid; i < kBins; i += kPickThreads) hist[i] = make_uint2(0u, 0u);
    if (tid == 0) listed = 0;
    asm volatile("" ::: "memory");  // (all of this before the wait for the lengths)
    bool bad = L < 0 || L > cap || N < L;
    const int pages = bad ? 0 : (L + kPage - 1) / kPage, ahead = (int)((unsigned)N - (unsigned)L + 1u);
    auto outside = [&] {
        auto out = [&](int e) { return e < 0 || e >= a.num_blocks; };
        bool any = (tid < pages && out(entry[0])) || (tid + kPickThreads < pages && out(entry[1]));
        for (int p = tid + 2 * kPickThreads; p < pages; p += kPickThreads) any = any || out(table[p]);
        return any;
    };
    if (bad || L <= keep) {
        bad = __syncthreads_or(bad || outside());
        if (tid == 0 && h == 0) *seq_of(a, b) = {bad ? -1 : L, 0, ahead};
        return;
    }
    __syncthreads();
    uint32_t* keys;
    if constexpr (SLOTS > 0)
        keys = lds_keys;
    else
        keys = r.keys;
    // a wavefront takes a run of slots, lane l of step u slot s0 + 64 u + l
    // (no thread uses a key that another wrote); slots past the row's last
    // token have key 0, kKeyPad more may be read
    const int steps = (L + kPickThreads - 1) / kPickThreads, s0 = wave * steps * kWave, s1 = min(L, s0 + steps * kWave);
    const int mine_n = (max(s1 - s0, 0) + kWave - 1) / kWave;  // steps of this wavefront
    // f(step, key) over n steps from slot `first` on, eight keys requested together
    auto over = [&](int first, int n, auto&& f) {
        for (int u0 = 0; u0 < n; u0 += 8) {
            const uint32_t* p = keys + first + u0 * kWave + lane;
            uint32_t k[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) k[j] = p[j * kWave];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (u0 + j < n) f(u0 + j, k[j]);
        }
    };
    // ---- the keep-th largest key.  Recent tokens have the largest, in a bin of
    // their own (no weight's key is above an infinity's, 0xFF800000).
    uint32_t* count = reinterpret_cast<uint32_t*>(hist) + (lane & 1);
    auto key_of = [&](int s, float w, int t) {
        uint32_t key = weight_key(w);
        asm("" : "+v"(key));  // (or it becomes a branch for each key)
        return (t > 0 ? t : s + ahead) > N - a.recent ? 0xFFFFFFFFu : key;
    };
    auto put = [&](int s, uint32_t key) {
        keys[s] = key;
        atomicAdd(count + 2 * (key >> 21), 1u);
    };
    // eight steps at a time, the next eight requested ahead; then the last few
    const int full = max(s1 - s0, 0) / (8 * kWave) * 8;
    if (steps != guess && mine_n > 0) request_upto(s0 + lane, s1 - 1);
    for (int u0 = 0; u0 < full; u0 += 8) {
        const int s = s0 + u0 * kWave + lane, next = s0 + min(u0 + 8, full - 8) * kWave + lane;
        uint32_t key[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) key[j] = key_of(s + j * kWave, w[j], t[j]);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = w_in[next + j * kWave];
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = t_in[next + j * kWave];
#pragma unroll
        for (int j = 0; j < 8; ++j) put(s + j * kWave, key[j]);
    }
    if (full < mine_n) {
        if (full > 0) request_upto(s0 + full * kWave + lane, s1 - 1);
        uint32_t key[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int s = s0 + (full + j) * kWave + lane;
            key[j] = s < s1 ? key_of(s, w[j], t[j]) : 0u;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int s = s0 + (full + j) * kWave + lane;
            if (s < s1)
                put(s, key[j]);
            else if (full + j < mine_n)
                keys[s] = 0u;
        }
    }
    bad = __syncthreads_or(outside());
    if (tid == 0 && h == 0) *seq_of(a, b) = {bad ? -1 : keep, !bad, ahead};
    if (bad) return;
    int2 total;
    uint32_t prefix = 0u;
    int left = keep, all = 0;
    // The bin of the counts in which the left-th largest lies: thread i adds up
    // bins 2047 - 2 i and 2046 - 2 i, the largest keys first.
    auto find = [&](int shift) {
        const uint2 x = hist[kBins - 1 - 2 * tid], y = hist[kBins - 2 - 2 * tid];
        const int hi = (int)(x.x + x.y), lo = (int)(y.x + y.y);
        const int before = block_scan(make_int2(hi + lo, 0), sums, total).x;
        if (before < left && left <= before + hi + lo) {
            const bool first = left <= before + hi;
            found = first ? kBins - 1 - 2 * tid : kBins - 2 - 2 * tid;
            found_left = left - before - (first ? 0 : hi);
            found_all = first ? hi : lo;
        }
        __syncthreads();
        prefix |= (uint32_t)found << shift;
        left = found_left;
        all = found_all;
    };
    find(21);
    // the bin's keys in a list, if they are few, so that the other bits take no
    // more passes over the row
    uint32_t base = max(prefix, 1u), span = prefix + (1u << 21) - base;
    const bool few = all <= kListed;
    if (few)
        for (int u0 = 0; u0 < mine_n; u0 += 32) {
            uint32_t hits = 0u;
            over(s0 + u0 * kWave, min(mine_n - u0, 32), [&](int u, uint32_t key) { hits |= (uint32_t)(key - base < span) << u; });
            const int n = __popc(hits), upto = wave_scan(n);
            int at = 0;
            if (lane == kWave - 1) at = atomicAdd(&listed, upto);
            at = __builtin_amdgcn_readlane(at, kWave - 1) + upto - n;
            for (; hits; hits &= hits - 1u) list[at++] = keys[s0 + (u0 + __ffs(hits) - 1) * kWave + lane];
        }
    if (all <= kRanked) {
        // each key's number of larger ones (<< 16) and of equal ones, wavefront w
        // against keys w, w + 16, ..: two passes over the other bits take longer
        // (4352 slots: 4100 against 1500 cycles)
        uint32_t* rank = reinterpret_cast<uint32_t*>(hist);
        const int n = all;
        if (tid < n) rank[tid] = 0u;
        __syncthreads();
        for (int i0 = 0; i0 < n; i0 += kWave) {
            const uint32_t key = list[min(i0 + lane, n - 1)];
            uint32_t c = 0u;
            for (int j = wave; j < n; j += kPickWaves) {
                const uint32_t other = list[j];
                c += other > key ? 1u << 16 : other == key ? 1u : 0u;
            }
            if (i0 + lane < n) atomicAdd(rank + i0 + lane, c);
        }
        __syncthreads();
        if (tid < n) {
            const int larger = (int)(rank[tid] >> 16), same = (int)(rank[tid] & 0xFFFFu);
            if (larger < left && left <= larger + same) {  // (equal keys all write the same)
                found = (int)list[tid];
                found_left = left - larger;
                found_all = same;
            }
        }
        __syncthreads();
        prefix = (uint32_t)found;
        left = found_left;
        all = found_all;
    } else {
        for (int shift = 10; shift >= 0; shift -= 10) {
            const uint32_t last = shift ? 2047u : 1023u;
            for (int i = tid; i < kBins; i += kPickThreads) hist[i] = make_uint2(0u, 0u);
            __syncthreads();
            auto add = [&](int, uint32_t key) {
                if (key - base < span) atomicAdd(count + 2 * ((key >> shift) & last), 1u);
            };
            if (few)
                for (int i = tid; i < listed; i += kPickThreads) add(0, list[i]);
            else
                over(s0, mine_n, add);
            __syncthreads();
            find(shift);
            base = max(prefix, 1u);
            span = prefix + (1u << shift) - base;
            __syncthreads();
        }
    }
    // ---- keys above the prefix stay, of the `all` equal ones the `left`
    // lowest slots.  Each step's comparison is a word of 64 bits, which lane u
    // keeps for step u of a round; counts and running sums over the steps are
    // then one vector operation (the scalar unit, which all of the block's
    // wavefronts share, took longer for them step by step).
    typedef unsigned long long Bits;
    const bool ties = all != left;
    const int rounds = (steps + kWave - 1) / kWave;
    auto bits_of = [&](int round, auto&& f) {
        uint32_t lo = 0u, hi = 0u;
        over(s0 + round * kWave * kWave, min(mine_n - round * kWave, kWave), [&](int u, uint32_t key) {
            const Bits v = __ballot(f(u, key));
            lo = lane == u ? (uint32_t)v : lo;
            hi = lane == u ? (uint32_t)(v >> 32) : hi;
        });
        return (Bits)hi << 32 | lo;
    };
    auto lane_bits = [&](Bits v, int u) {
        return (Bits)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), u) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, u);
    };
    // lane u: the word of keys equal to the prefix in step u, and how many came before it
    auto find_same = [&](int round, int& eq, int& before) {
        const Bits same = bits_of(round, [&](int, uint32_t key) { return key == prefix; });
        const int n = __popcll(same), x = wave_scan(n);
        before = eq + x - n;
        eq += __builtin_amdgcn_readlane(x, kWave - 1);
        return same;
    };
    auto find_kept = [&](int round, int& eq) {
        if (!ties) return bits_of(round, [&](int, uint32_t key) { return key >= prefix; });
        int before;
        const Bits same = find_same(round, eq, before);
        return bits_of(round, [&](int u, uint32_t key) {
            return key > prefix || (key == prefix && below_lane(lane_bits(same, u), __builtin_amdgcn_readlane(before, u)) < left);
        });
    };
    auto below_keep = [&](int round) {
        // (a lane without a step of this wavefront has no slots)
        const int first = s0 + (round * kWave + lane) * kWave, n = keep - first;
        return first >= s1 || n <= 0 ? 0ull : n >= kWave ? ~0ull : (1ull << n) - 1ull;
    };
    int eq0 = 0;
    if (ties) {
        int before;
        for (int round = 0; round < rounds; ++round) (void)find_same(round, eq0, before);
        eq0 = __builtin_amdgcn_readfirstlane(block_scan(make_int2(lane == 0 ? eq0 : 0, 0), sums, total).x);
    }
    int eq = eq0;
    Bits kept = 0;
    int2 mine = make_int2(0, 0);  // free slots below keep, moving tokens
    for (int round = 0; round < rounds; ++round) {
        kept = find_kept(round, eq);
        const Bits low = below_keep(round);
        mine.x += __popcll(low & ~kept);
        mine.y += __popcll(kept & ~low);
    }
    const int2 at0 = block_scan(mine, sums, total);
    int free0 = __builtin_amdgcn_readfirstlane(at0.x), move0 = __builtin_amdgcn_readfirstlane(at0.y);
    eq = eq0;
    for (int round = 0; round < rounds; ++round) {
        if (rounds > 1) kept = find_kept(round, eq);
        const Bits low = below_keep(round);
        const int f = __popcll(low & ~kept), m = __popcll(kept & ~low), fs = wave_scan(f), ms = wave_scan(m);
        const int first = s0 + round * kWave * kWave, word = first / kWave + lane, moves_before = move0 + ms - m;
        if (word * kWave < s1) {
            r.stays[word] = kept;
            r.free_before[word] = free0 + fs - f;
        }
        const Bits move = kept & ~low;
        const int n = min(mine_n - round * kWave, kWave);
        for (int u = max(0, (keep - first) / kWave); u < n; ++u) {
            const Bits v = lane_bits(move, u);
            if (__builtin_amdgcn_inverse_ballot_w64(v)) r.from[below_lane(v, __builtin_amdgcn_readlane(moves_before, u))] = first + u * kWave + lane;
        }
        free0 += __builtin_amdgcn_readlane(fs, kWave - 1);
        move0 += __builtin_amdgcn_readlane(ms, kWave - 1);
    }
}

constexpr int kMoveWaves = 4, kMoveThreads = kMoveWaves * kWave;
constexpr int kClearSlots = 4 * kMoveThreads;
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));

__device__ inline size_t lane64(size_t v, int l) {
    return ((size_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)v, l);
}

// Tokens into one page of one kv head.  Lane t < 16 has the record (byte
// offset `src`) and the slot there (`u`) of the token that slot t takes, `moved`
// has a bit for each t that takes one.  All of a wavefront's loads are requested
// before its stores; a lane alone writes the words it reads.
// fp16 pages: part 0 is K, part 1 + i the 64 dimensions from 64 i on of V.
template <int HD>
__device__ inline void move_f16(const EvictArgs& a, int part, size_t dst, size_t src, int u, unsigned moved, int lane) {
    if (part == 0) {  // 16 bytes of a vector a lane
        constexpr int KL = HD / 8, KT = kWave / KL < kPage ? kWave / KL : kPage, KN = kPage / KT;  // lanes of a vector, vectors and steps
        u4_t k[KN] = {};
#pragma unroll
        for (int i = 0; i < KN; ++i) {
            const int t = i * KT + lane / KL;
            const size_t p = __shfl(src, t, kWave) + 2 * HD * __shfl(u, t, kWave);
            if (moved >> t & 1u) k[i] = __builtin_nontemporal_load(reinterpret_cast<const u4_t*>(a.kpool + p) + lane % KL);
        }
#pragma unroll
        for (int i = 0; i < KN; ++i) {
            const int t = i * KT + lane / KL;
            if (moved >> t & 1u) reinterpret_cast<u4_t*>(a.kpool + dst + 2 * HD * t)[lane % KL] = k[i];
        }
        return;
    }
    // Half a dimension's row (eight tokens) a lane, of dimensions r and r + 32: a
    // store's lanes write whole lines.
    const int half = lane & 1, r = (part - 1) * kWave + lane / 2;
    const unsigned mine = moved >> (8 * half) & 0xFFu;
    uint16_t v[8][2] = {};
    u4_t row[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) row[i] = reinterpret_cast<const u4_t*>(a.vpool + dst)[2 * (r + 32 * i) + half];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        if (!(moved >> k & 0x101u)) continue;
        const size_t from = (half ? lane64(src, 8 + k) : lane64(src, k)) + 2 * (half ? __builtin_amdgcn_readlane(u, 8 + k) : __builtin_amdgcn_readlane(u, k));
        if (mine >> k & 1u)
#pragma unroll
            for (int i = 0; i < 2; ++i) v[k][i] = reinterpret_cast<const uint16_t*>(a.vpool + from)[(uint32_t)(r + 32 * i) * kPage];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t w = row[i][k / 2], x = k % 2 ? (w & 0xFFFFu) | (uint32_t)v[k][i] << 16 : (w & 0xFFFF0000u) | v[k][i];
            row[i][k / 2] = mine >> k & 1u ? x : w;
        }
        reinterpret_cast<u4_t*>(a.vpool + dst)[2 * (r + 32 * i) + half] = row[i];
    }
}

template <int HD>
__device__ inline void move_int4(const EvictArgs& a, size_t dst, size_t src, int u, unsigned moved, int lane) {
    constexpr int S = HD / 32;
    // K: 16 bytes of a token's codes a lane
    constexpr int KL = HD / 32, KT = kWave / KL < kPage ? kWave / KL : kPage, KN = kPage / KT;
    u4_t k[KN] = {};
#pragma unroll
    for (int i = 0; i < KN; ++i) {
        const int t = i * KT + lane / KL;
        const size_t p = __shfl(src, t & 15, kWave) + HD / 2 * __shfl(u, t & 15, kWave);
        if (t < kPage && (moved >> t & 1u)) k[i] = reinterpret_cast<const u4_t*>(a.kpool + p)[lane % KL];
    }
    // scales: a token's S of K, then of V
    constexpr int SN = 2 * S * kPage / kWave;
    uint16_t sc[SN] = {};
#pragma unroll
    for (int i = 0; i < SN; ++i) {
        const int x = i * kWave + lane, t = x / (2 * S), g = x % (2 * S);
        const size_t p = __shfl(src, t, kWave);
        const int from = __shfl(u, t, kWave);
        if (moved >> t & 1u) sc[i] = reinterpret_cast<const uint16_t*>((g < S ? a.kpool : a.vpool) + p + 8 * HD)[scale_at(HD, from, g % S)];
    }
    // V: lane (g, n) has the S dwords of quad g, and of its four tokens the
    // dwords that hold them elsewhere
    const int q = lane >> 4, n = lane & 15;
    uint32_t* own = reinterpret_cast<uint32_t*>(a.vpool + dst) + lane * S;
    const bool mine = moved >> (4 * q) & 15u;
    uint32_t d[S] = {}, w[4][S] = {};
    int from[4];
    if (mine)
#pragma unroll
        for (int i = 0; i < S; ++i) d[i] = own[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const size_t p = __shfl(src, 4 * q + j, kWave);
        from[j] = __shfl(u, 4 * q + j, kWave);
        if (moved >> (4 * q + j) & 1u)
#pragma unroll
            for (int i = 0; i < S; ++i) w[j][i] = reinterpret_cast<const uint32_t*>(a.vpool + p)[(16 * (from[j] >> 2) + n) * S + i];
    }
#pragma unroll
    for (int i = 0; i < KN; ++i) {
        const int t = i * KT + lane / KL;
        if (t < kPage && (moved >> t & 1u)) reinterpret_cast<u4_t*>(a.kpool + dst + HD / 2 * t)[lane % KL] = k[i];
    }
#pragma unroll
    for (int i = 0; i < SN; ++i) {
        const int x = i * kWave + lane, t = x / (2 * S), g = x % (2 * S);
        if (moved >> t & 1u) reinterpret_cast<uint16_t*>((g < S ? a.kpool : a.vpool) + dst + 8 * HD)[scale_at(HD, t, g % S)] = sc[i];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (moved >> (4 * q + j) & 1u)
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int ns = 4 * v_nib(from[j], 16 * e), nd = 4 * v_nib(j, 16 * e);
                    d[i] = (d[i] & ~(15u << nd)) | ((w[j][i] >> ns & 15u) << nd);
                }
    if (mine)
#pragma unroll
        for (int i = 0; i < S; ++i) own[i] = d[i];
}

// The first blocks of a (kv head, sequence) take the pages of kept slots,
// kParts wavefronts to a page, the others clear kClearSlots slots' weights and
// tags beyond them.  The weights' outputs may be their inputs: a slot that a
// token leaves is cleared by the lane that has read it, every other by its own.
// fp16: bound by memory, since V's pages are dimension-major, so that a token
// moves with whole pages: 8 sequences of 8192 tokens of 8 kv heads of 128 cut to
// 2048 read 173 MB and write 65, 51 us; int4, one of 32768 cut to 4096: 8.0 us.
template <int HD, bool INT4>
constexpr int kParts = INT4 ? 1 : 1 + HD / kWave;  // wavefronts of a page

template <int HD, bool INT4>
__global__ __launch_bounds__(kMoveThreads) void k_move(EvictArgs a) {
    constexpr int BYTES = INT4 ? page_bytes(HD) : 2 * kPage * HD;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = blockIdx.y, b = blockIdx.z;
    const int cap = a.max_blocks * kPage, ks = kept_slots(a.max_blocks, a.keep), blocks = (ks / kPage * kParts<HD, INT4> + kMoveWaves - 1) / kMoveWaves;
    const size_t at = ((size_t)b * a.hkv + h) * cap;
    const Row r = row_of(a, b, h);
    if ((int)blockIdx.x >= blocks) {
        const Seq seq = *seq_of(a, b);
        if (seq.len < 0) return;
        const int tokens = seq.cut ? a.seen[b] - seq.ahead + 1 : seq.len;  // cached before
        const int first = ks + ((int)blockIdx.x - blocks) * kClearSlots, end = min(cap, first + kClearSlots);
        for (int s = first + (int)threadIdx.x; s < end; s += kMoveThreads) {
            if (s < tokens && (r.stays[s / kWave] >> (s % kWave) & 1ull)) continue;
            a.weights_out[at + s] = 0.0f;
            a.tags_out[at + s] = 0;
        }
        return;
    }
    const int unit = blockIdx.x * kMoveWaves + wave, page = unit / kParts<HD, INT4>, part = unit % kParts<HD, INT4>;
    if (page * kPage >= ks) return;
    // A wavefront's time is the chain from here to the tokens' bytes: what does
    // not depend on the sequence's state is requested with it (stays and
    // free_before hold anything where nothing is cut, the table's entry
    // where the sequence is refused or too short).
    const int32_t* table = a.table + (size_t)b * a.max_blocks;
    const Seq seq = *seq_of(a, b);
    const int seen = a.seen[b], here = table[page];
    unsigned long long stays = r.stays[page * kPage / kWave];
    int free_before = r.free_before[page * kPage / kWave];
    asm volatile("" : "+v"(stays), "+v"(free_before) : "v"(seen), "v"(here));
    if (unit == 0 && h == 0 && lane == 0) a.lens_out[b] = seq.len;
    if (seq.len < 0) return;
    const int tokens = seq.cut ? seen - seq.ahead + 1 : seq.len;
    if (!seq.cut) {
        stays = ~0ull;
        free_before = 0;
    }
    // lane t < 16: slot t of the page
    const int s = page * kPage + (lane & 15), bit = s % kWave;
    const bool used = s < seq.len && lane < kPage;
    const bool takes = used && !(stays >> bit & 1ull);
    int from = 0, tag = 0;
    float w = 0.0f;
    if (used) from = takes ? r.from[free_before + __popcll(~stays & ((1ull << bit) - 1ull))] : s;
    if (used && part == 0) {
        const int t = a.tags_in[at + from];
        tag = t > 0 ? t : seq.ahead + from;
        w = a.weights_in[at + from];
    }
    const unsigned moved = (unsigned)__ballot(takes);
    if (moved) {
        const size_t src = takes ? ((size_t)table[from / kPage] * a.hkv + h) * BYTES : 0;
        const size_t dst = ((size_t)here * a.hkv + h) * BYTES;
        if constexpr (INT4)
            move_int4<HD>(a, dst, src, from % kPage, moved, lane);
        else
            move_f16<HD>(a, part, dst, src, from % kPage, moved, lane);
    }
    if (part > 0) return;
    if (lane < kPage && (used || s >= tokens || !(stays >> bit & 1ull))) {
        a.weights_out[at + s] = w;
        a.tags_out[at + s] = tag;
    }
    if (takes) {
        a.weights_out[at + from] = 0.0f;
        a.tags_out[at + from] = 0;
    }
}

template <int HD, bool INT4>
void move_case(const EvictArgs& a, hipStream_t st) {
    const int ks = kept_slots(a.max_blocks, a.keep), rest = a.max_blocks * kPage - ks;
    const unsigned blocks = (unsigned)((ks / kPage * kParts<HD, INT4> + kMoveWaves - 1) / kMoveWaves + (rest + kClearSlots - 1) / kClearSlots);
    hipLaunchKernelGGL((k_move<HD, INT4>), dim3(blocks, (unsigned)a.hkv, (unsigned)a.batch), dim3(kMoveThreads), 0, st, a);
}

}  // namespace

size_t evict_ws_words(int batch, int hkv, int max_blocks, int keep) {
    return (size_t)batch * kSeqWords + (size_t)batch * hkv * row_words(max_blocks, keep);
}

hipError_t evict_launch(const EvictArgs& a, bool int4, hipStream_t st) {
    if (a.hd != 64 && a.hd != 128 && a.hd != 256) return hipErrorInvalidValue;
    const dim3 rows((unsigned)a.hkv, (unsigned)a.batch), threads(kPickThreads);
    const int cap = a.max_blocks * kPage;
    if (cap <= 8192)
        hipLaunchKernelGGL(k_pick<8192>, rows, threads, 0, st, a);
    else if (cap <= kLdsSlots)
        hipLaunchKernelGGL(k_pick<kLdsSlots>, rows, threads, 0, st, a);
    else
        hipLaunchKernelGGL(k_pick<0>, rows, threads, 0, st, a);
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
