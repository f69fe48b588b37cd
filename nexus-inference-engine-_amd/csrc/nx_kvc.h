// The compact KV cache: int4-g32 pages, attention over them and over fp16
// pages that accumulates the weight of every cached token, and eviction by
// that weight.  Layout of the pages, kernel arguments and launchers.
#pragma once

#include <stddef.h>

#include "nx_common.h"

namespace nx {
namespace kvc {

// --------------------------------------------------------- int4-g32 pages --
// One page of one kv head is a record of 9 hd bytes: 8 hd of codes (16 tokens
// x hd, 4 bits each), then 16 x hd / 32 fp16 scales.  A value is (code - 8) *
// scale of its token and group of 32 dimensions.  The codes lie in the order
// in which the attention's matrix products take them, so that a lane's share
// of a page is one run of hd / 32 dwords:
//   K: dword g S + s of a token's hd / 8 (S = hd / 32) holds dimensions
//      32 s + 8 g + j, j < 8: lane (token, g) reads its S steps together;
//   V: dword (16 g + n) S + i holds tokens 4 g + j, j < 4, of dimensions
//      32 i + n (e = 0) and 32 i + 16 + n (e = 1): lane (g, n) reads all its
//      tiles together.
// Neighbours along a product's k sit four nibbles apart (0 and 4, 1 and 5,
// ..), so a mask and an or give two of them as one register of fp16 pairs.
__host__ __device__ constexpr int page_bytes(int hd) { return 9 * hd; }
__host__ __device__ constexpr int k_word(int hd, int t, int d) { return t * (hd / 8) + ((d >> 3) & 3) * (hd / 32) + (d >> 5); }
__host__ __device__ constexpr int k_nib(int d) { return ((d & 7) >> 1) + 4 * (d & 1); }
// what V's dword w holds: tokens 4 g .. + 3 of dimensions d and d + 16
struct VWord {
    int g, d;
};
__host__ __device__ constexpr VWord v_word(int hd, int w) { return {w / (hd / 32) / 16, 32 * (w % (hd / 32)) + w / (hd / 32) % 16}; }
__host__ __device__ constexpr int v_nib(int t, int d) { return ((t & 3) >> 1) + 2 * ((d >> 4) & 1) + 4 * (t & 1); }
// index of a scale among the page's halves: the four tokens of a lane together
__host__ __device__ constexpr int scale_at(int hd, int t, int grp) { return ((t >> 2) * (hd / 32) + grp) * 4 + (t & 3); }

// The i-th page that rows of positions first .. first + tokens - 1 touch.
struct RowPage {
    int page, row0;      // its place in the block table, and the row of its token 0
    bool none, refused;  // no row lies in it; the positions are out of range (rows as from 0)
};
NX_HD RowPage row_page(int first, int tokens, int max_blocks, int i) {
    const bool refused = first < 0 || (int64_t)first + tokens > (int64_t)max_blocks * kPage;
    const int s = refused ? 0 : first, page = s / kPage + i;
    const int64_t row0 = (int64_t)page * kPage - s;
    return {page, (int)row0, row0 >= tokens, refused};
}
// Pages that `tokens` rows may touch, wherever they begin.
NX_HD int row_pages(int tokens) { return (int)(((int64_t)tokens + kPage - 2) / kPage + 1); }

struct RowArgs {             // append and read: rows fp32 [batch][tokens][hkv][hd]
    float *k, *v;
    uint8_t *kpool, *vpool;  // [num_blocks][hkv][9 hd]
    const int32_t *table;    // [batch][max_blocks]
    const int32_t *start;    // [batch] position of a sequence's first row
    int batch, tokens, hkv, hd, max_blocks, num_blocks;
};
hipError_t append_int4_launch(const RowArgs& a, hipStream_t st);
hipError_t read_int4_launch(const RowArgs& a, hipStream_t st);

// --------------------------------------------------------------- attention --
constexpr int kHeadsPerBlock = 8;  // query heads that share a block's pages (hi and lo parts fill 16 columns)

struct AttnPlan {
    int groups;  // blocks of up to kHeadsPerBlock query heads per kv head
    int heads;   // query heads of a block's record
    int splits;  // blocks that share the pages of one (sequence, kv head)
    int rec;     // floats of a record: O[heads][hd], M[heads], L[heads]
    bool join;   // a second launch merges the records
};
AttnPlan attn_plan(int batch, int hq, int hkv, int hd, int max_blocks, bool int4, bool weights);

struct AttnArgs {
    const float* q;          // [batch][hq][hd]
    const uint8_t *kpool, *vpool;
    const int32_t *table, *lens;
    uint16_t* out;           // [batch][hq][hd]
    float* weights;          // [batch][hkv][max_blocks * 16], added to; or null
    float* part;             // records [batch][hkv * groups][splits][rec]
    float* raw;              // with weights: scores [batch][hq][max_blocks * 16]
    int batch, hq, hkv, hd, max_blocks, num_blocks;
    AttnPlan plan;
};
// Floats of the workspace: the records, and the scores with weights.
size_t attn_part_floats(const AttnPlan& p, int batch, int hkv);
size_t attn_most_part_floats(int batch, int hq, int hkv, int hd, int max_blocks, int max_group);  // of any call up to these sizes
inline size_t attn_raw_floats(int batch, int hq, int max_blocks) { return (size_t)batch * hq * max_blocks * kPage; }
hipError_t attn_launch(const AttnArgs& a, bool int4, hipStream_t st);

// ---------------------------------------------------------------- eviction --
struct EvictArgs {
    uint8_t *kpool, *vpool;
    const int32_t *table, *lens_in, *seen;
    const float* weights_in;   // [batch][hkv][max_blocks * 16]
    const int32_t* tags_in;
    int32_t* lens_out;
    float* weights_out;
    int32_t* tags_out;
    uint32_t* ws;              // evict_ws_words words
    int batch, hkv, hd, max_blocks, num_blocks, keep, recent;
};
size_t evict_ws_words(int batch, int hkv, int max_blocks, int keep);
hipError_t evict_launch(const EvictArgs& a, bool int4, hipStream_t st);

}  // namespace kvc
}  // namespace nx
