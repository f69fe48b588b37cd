// Entry points of the compact KV cache (nx_kvc.h): checks of shapes and
// buffers on the host, the workspace, the launches.  Lengths, positions and
// block tables are checked by the kernels, so no call waits for the device
// (but where its workspace grows outside a token batch) and every call may be
// captured into a token batch.
#include <algorithm>

#include "nx_internal.h"
#include "nx_kvc.h"

using nx::fail;

namespace {

template <class T>
T* dptr(nx_buf b) {
    return reinterpret_cast<T*>(static_cast<uintptr_t>(b));
}

// NX_NEED, which knows the numbers of a context without a device as well: these
// calls end before they would be taken for addresses.
nx_status need(nx_ctx* ctx, nx_buf b, size_t bytes, const char* name) {
    if (ctx->device >= 0 || !ctx->numbers.count(b)) {
        NX_NEED(ctx, b, bytes, name);
        return NX_OK;
    }
    const size_t has = ctx->numbers[b];
    return has < bytes ? fail(ctx, NX_ERR_INVALID, "%s: buffer has %zu bytes, needs %zu", name, has, bytes) : NX_OK;
}
#define NEED(ctx, b, bytes, name)                                  \
    do {                                                           \
        const nx_status nx_s_ = need((ctx), (b), (bytes), (name)); \
        if (nx_s_ != NX_OK) return nx_s_;                          \
    } while (0)

// The context's device for the time of a call.
struct OnDevice {
    int before = -1;
    explicit OnDevice(int device) {
        if (hipGetDevice(&before) != hipSuccess || before == device || hipSetDevice(device) != hipSuccess) before = -1;
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

// Largest sizes the kernels' grids and 32-bit slot numbers take.
constexpr int kMaxBatch = 65535, kMaxHkv = 4096, kMaxGroup = 64, kMaxSlotBlocks = 1 << 22;

nx_status cache_shape(nx_ctx* ctx, const char* name, int batch, int hkv, int hd, int max_blocks, int num_blocks) {
    if (batch < 1 || hkv < 1 || hd < 1 || max_blocks < 1 || num_blocks < 1)
        return fail(ctx, NX_ERR_INVALID, "%s: bad shape (batch=%d hkv=%d head_dim=%d max_blocks=%d num_blocks=%d)", name, batch, hkv, hd,
                    max_blocks, num_blocks);
    if (hd != 64 && hd != 128 && hd != 256) return fail(ctx, NX_ERR_UNSUPPORTED, "%s: head_dim %d (64, 128 and 256 are built)", name, hd);
    if (batch > kMaxBatch || hkv > kMaxHkv || max_blocks > kMaxSlotBlocks)
        return fail(ctx, NX_ERR_UNSUPPORTED, "%s: batch %d above %d, hkv %d above %d or max_blocks %d above %d", name, batch, kMaxBatch, hkv,
                    kMaxHkv, max_blocks, kMaxSlotBlocks);
    return NX_OK;
}

size_t pool_bytes(bool int4, int hkv, int hd, int num_blocks) {
    return (size_t)num_blocks * hkv * (int4 ? nx::kvc::page_bytes(hd) : 2 * nx::kPage * hd);
}

// The workspace of attention and eviction, grown when a call needs more: the
// old one goes first, behind a wait for its last call.  In a token batch,
// whose launches name the old one, it is kept until the batch has run, and the
// allocation is declared as no part of the capture.
nx_status kvc_ws(nx_ctx* ctx, size_t bytes, const char* name) {
    if (bytes <= ctx->kvc_ws_bytes) return NX_OK;
    void* ws = nullptr;
    if (!ctx->capturing) {
        if (ctx->kvc_ws) {
            NX_HIP(ctx, hipStreamSynchronize(ctx->stream));
            (void)hipFree(ctx->kvc_ws);
            ctx->kvc_ws = nullptr;
            ctx->kvc_ws_bytes = 0;
        }
        const hipError_t e = nx::dev_malloc(ctx, &ws, bytes);
        if (e != hipSuccess) return nx::hip_fail(ctx, e, name);
    } else {
        if (ctx->kvc_ws) {
            try {
                ctx->outgrown.reserve(ctx->outgrown.size() + 1);
            } catch (...) {
                return fail(ctx, NX_ERR_OOM, "%s: no memory for the list of old workspaces", name);
            }
        }
        hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
        NX_HIP(ctx, hipThreadExchangeStreamCaptureMode(&mode));
        const hipError_t e = nx::dev_malloc(ctx, &ws, bytes);
        (void)hipThreadExchangeStreamCaptureMode(&mode);
        if (e != hipSuccess) return nx::hip_fail(ctx, e, name);
        if (ctx->kvc_ws) ctx->outgrown.push_back(ctx->kvc_ws);
    }
    ctx->kvc_ws = ws;
    ctx->kvc_ws_bytes = bytes;
    return NX_OK;
}

size_t attn_ws_bytes(const nx::kvc::AttnPlan& p, int batch, int hq, int hkv, int max_blocks, bool weights) {
    return 4 * (nx::kvc::attn_part_floats(p, batch, hkv) + (weights ? nx::kvc::attn_raw_floats(batch, hq, max_blocks) : 0));
}

nx_status rows_int4(nx_ctx* ctx, const char* name, bool append, nx_buf k, nx_buf v, nx_buf kpool, nx_buf vpool, nx_buf bt, nx_buf pos, int batch,
                    int tokens, int hkv, int hd, int max_blocks, int num_blocks) {
    if (!ctx) return NX_ERR_INVALID;
    const nx_status s = cache_shape(ctx, name, batch, hkv, hd, max_blocks, num_blocks);
    if (s != NX_OK) return s;
    if (tokens < 1) return fail(ctx, NX_ERR_INVALID, "%s: tokens must be positive", name);
    if (tokens > max_blocks * nx::kPage)
        return fail(ctx, NX_ERR_CAPACITY, "%s: %d tokens exceed %d blocks of %d", name, tokens, max_blocks, nx::kPage);
    const size_t rows = (size_t)batch * tokens * hkv * hd * 4, pool = pool_bytes(true, hkv, hd, num_blocks);
    NEED(ctx, k, rows, "k");
    NEED(ctx, v, rows, "v");
    NEED(ctx, kpool, pool, "kpool");
    NEED(ctx, vpool, pool, "vpool");
    NEED(ctx, bt, (size_t)batch * max_blocks * 4, "block_table");
    NEED(ctx, pos, (size_t)batch * 4, "positions");
    const nx_buf all[] = {k, v, kpool, vpool, bt, pos}, outs[] = {append ? kpool : k, append ? vpool : v};
    for (nx_buf o : outs) {
        int n = 0;
        for (nx_buf b : all) n += b == o;
        if (n > 1) return fail(ctx, NX_ERR_INVALID, "%s: an output is another buffer of the call", name);
    }
    nx::kvc::RowArgs a{};
    a.k = dptr<float>(k);
    a.v = dptr<float>(v);
    a.kpool = dptr<uint8_t>(kpool);
    a.vpool = dptr<uint8_t>(vpool);
    a.table = dptr<const int32_t>(bt);
    a.start = dptr<const int32_t>(pos);
    a.batch = batch;
    a.tokens = tokens;
    a.hkv = hkv;
    a.hd = hd;
    a.max_blocks = max_blocks;
    a.num_blocks = num_blocks;
    if (ctx->device < 0) return fail(ctx, NX_ERR_NO_DEVICE, "%s: no device", name);
    const OnDevice on(ctx->device);
    const hipError_t e = append ? nx::kvc::append_int4_launch(a, ctx->stream) : nx::kvc::read_int4_launch(a, ctx->stream);
    return e == hipSuccess ? NX_OK : nx::hip_fail(ctx, e, name);
}

nx_status attn_kvc(nx_ctx* ctx, const char* name, bool int4, nx_buf q, nx_buf kpool, nx_buf vpool, nx_buf bt, nx_buf lens, nx_buf out, nx_buf weights,
                   int batch, int hq, int hkv, int hd, int max_blocks, int num_blocks) {
    if (!ctx) return NX_ERR_INVALID;
    nx_status s = cache_shape(ctx, name, batch, hkv, hd, max_blocks, num_blocks);
    if (s != NX_OK) return s;
    if (hq < 1 || hq % hkv) return fail(ctx, NX_ERR_INVALID, "%s: hq %d is no multiple of hkv %d", name, hq, hkv);
    if (hq / hkv > kMaxGroup) return fail(ctx, NX_ERR_UNSUPPORTED, "%s: hq/hkv = %d above %d", name, hq / hkv, kMaxGroup);
    const size_t pool = pool_bytes(int4, hkv, hd, num_blocks);
    NEED(ctx, q, (size_t)batch * hq * hd * 4, "q");
    NEED(ctx, kpool, pool, "kpool");
    NEED(ctx, vpool, pool, "vpool");
    NEED(ctx, bt, (size_t)batch * max_blocks * 4, "block_table");
    NEED(ctx, lens, (size_t)batch * 4, "ctx_lens");
    NEED(ctx, out, (size_t)batch * hq * hd * 2, "out");
    if (weights || !int4) NEED(ctx, weights, (size_t)batch * hkv * max_blocks * nx::kPage * 4, "weights");
    const nx_buf in[] = {q, kpool, vpool, bt, lens};
    bool clash = out == weights;
    for (nx_buf b : in) clash = clash || b == out || (weights && b == weights);
    if (clash) return fail(ctx, NX_ERR_INVALID, "%s: an output is another buffer of the call", name);
    nx::kvc::AttnArgs a{};
    if (ctx->device < 0) return fail(ctx, NX_ERR_NO_DEVICE, "%s: no device", name);
    const OnDevice on(ctx->device);
    a.plan = nx::kvc::attn_plan(batch, hq, hkv, hd, max_blocks, int4, weights != 0);
    s = kvc_ws(ctx, attn_ws_bytes(a.plan, batch, hq, hkv, max_blocks, weights != 0), name);
    if (s != NX_OK) return s;
    a.q = dptr<const float>(q);
    a.kpool = dptr<const uint8_t>(kpool);
    a.vpool = dptr<const uint8_t>(vpool);
    a.table = dptr<const int32_t>(bt);
    a.lens = dptr<const int32_t>(lens);
    a.out = dptr<uint16_t>(out);
    a.weights = weights ? dptr<float>(weights) : nullptr;
    a.part = static_cast<float*>(ctx->kvc_ws);
    a.raw = a.part + nx::kvc::attn_part_floats(a.plan, batch, hkv);
    a.batch = batch;
    a.hq = hq;
    a.hkv = hkv;
    a.hd = hd;
    a.max_blocks = max_blocks;
    a.num_blocks = num_blocks;
    const hipError_t e = nx::kvc::attn_launch(a, int4, ctx->stream);
    return e == hipSuccess ? NX_OK : nx::hip_fail(ctx, e, name);
}

nx_status evict(nx_ctx* ctx, const char* name, bool int4, nx_buf kpool, nx_buf vpool, nx_buf bt, nx_buf lens_in, nx_buf seen, nx_buf w_in, nx_buf t_in,
                nx_buf lens_out, nx_buf w_out, nx_buf t_out, int batch, int hkv, int hd, int max_blocks, int num_blocks, int keep, int recent) {
    if (!ctx) return NX_ERR_INVALID;
    nx_status s = cache_shape(ctx, name, batch, hkv, hd, max_blocks, num_blocks);
    if (s != NX_OK) return s;
    if (keep < 1 || recent < 0 || recent > keep)
        return fail(ctx, NX_ERR_INVALID, "%s: keep %d must be positive and recent %d within it", name, keep, recent);
    const size_t pool = pool_bytes(int4, hkv, hd, num_blocks), slots = (size_t)batch * hkv * max_blocks * nx::kPage * 4;
    NEED(ctx, kpool, pool, "kpool");
    NEED(ctx, vpool, pool, "vpool");
    NEED(ctx, bt, (size_t)batch * max_blocks * 4, "block_table");
    NEED(ctx, lens_in, (size_t)batch * 4, "ctx_lens");
    NEED(ctx, seen, (size_t)batch * 4, "seen");
    NEED(ctx, w_in, slots, "weights");
    NEED(ctx, t_in, slots, "tags");
    NEED(ctx, lens_out, (size_t)batch * 4, "lens_out");
    NEED(ctx, w_out, slots, "weights_out");
    NEED(ctx, t_out, slots, "tags_out");
    // What is written is no other buffer of the call, but that each of the last
    // three may be the input of its kind.  (The places count: an input that is
    // given twice may not be one output's own and stand for another input.)
    const nx_buf all[] = {kpool, vpool, lens_out, w_out, t_out, bt, seen, lens_in, w_in, t_in};
    constexpr int kWritten = 5, kAll = 10;
    bool clash = false;
    for (int i = 0; i < kWritten; ++i)
        for (int j = 0; j < kAll; ++j) clash = clash || (j != i && all[j] == all[i] && !(i >= 2 && j == i + 5));
    if (clash) return fail(ctx, NX_ERR_INVALID, "%s: an output is another buffer of the call", name);
    if (ctx->device < 0) return fail(ctx, NX_ERR_NO_DEVICE, "%s: no device", name);
    const OnDevice on(ctx->device);
    s = kvc_ws(ctx, 4 * nx::kvc::evict_ws_words(batch, hkv, max_blocks, keep), name);
    if (s != NX_OK) return s;
    nx::kvc::EvictArgs a{};
    a.kpool = dptr<uint8_t>(kpool);
    a.vpool = dptr<uint8_t>(vpool);
    a.table = dptr<const int32_t>(bt);
    a.lens_in = dptr<const int32_t>(lens_in);
    a.seen = dptr<const int32_t>(seen);
    a.weights_in = dptr<const float>(w_in);
    a.tags_in = dptr<const int32_t>(t_in);
    a.lens_out = dptr<int32_t>(lens_out);
    a.weights_out = dptr<float>(w_out);
    a.tags_out = dptr<int32_t>(t_out);
    a.ws = static_cast<uint32_t*>(ctx->kvc_ws);
    a.batch = batch;
    a.hkv = hkv;
    a.hd = hd;
    a.max_blocks = max_blocks;
    a.num_blocks = num_blocks;
    a.keep = keep;
    a.recent = recent;
    const hipError_t e = nx::kvc::evict_launch(a, int4, ctx->stream);
    return e == hipSuccess ? NX_OK : nx::hip_fail(ctx, e, name);
}

}  // namespace

extern "C" {

// Not part of the interface: the pages that the row kernels work on, for a
// test to walk (row_page: place, row of token 0, none, refused).
int nx_kvc_row_page(int first, int tokens, int max_blocks, int i, int* out) {
    const nx::kvc::RowPage p = nx::kvc::row_page(first, tokens, max_blocks, i);
    out[0] = p.page;
    out[1] = p.row0;
    out[2] = p.none;
    out[3] = p.refused;
    return nx::kvc::row_pages(tokens);
}

nx_status nx_reserve_kv_compact(nx_ctx* ctx, int batch, int hq, int hkv, int hd, int max_ctx) {
    const char* name = "nx_reserve_kv_compact";
    if (!ctx) return NX_ERR_INVALID;
    if (hq < 1 || max_ctx < 1) return fail(ctx, NX_ERR_INVALID, "%s: bad sizes (n_heads=%d max_ctx=%d)", name, hq, max_ctx);
    const int blocks = (int)(((int64_t)max_ctx + nx::kPage - 1) / nx::kPage);
    const nx_status s = cache_shape(ctx, name, batch, hkv, hd, blocks, 1);
    if (s != NX_OK) return s;
    if (ctx->capturing) return fail(ctx, NX_ERR_STATE, "%s inside a token batch", name);
    if (ctx->device < 0) return fail(ctx, NX_ERR_NO_DEVICE, "%s: no device", name);
    const OnDevice on(ctx->device);
    const size_t attn = 4 * (nx::kvc::attn_most_part_floats(batch, hq, hkv, hd, blocks, kMaxGroup) + nx::kvc::attn_raw_floats(batch, hq, blocks));
    return kvc_ws(ctx, std::max(4 * nx::kvc::evict_ws_words(batch, hkv, blocks, blocks * nx::kPage), attn), name);
}

nx_status nx_kv_append_int4(nx_ctx* ctx, nx_buf k, nx_buf v, nx_buf kpool, nx_buf vpool, nx_buf bt, nx_buf pos, int batch, int tokens, int hkv,
                            int hd, int max_blocks, int num_blocks) {
    return rows_int4(ctx, "nx_kv_append_int4", true, k, v, kpool, vpool, bt, pos, batch, tokens, hkv, hd, max_blocks, num_blocks);
}

nx_status nx_kv_read_int4(nx_ctx* ctx, nx_buf kpool, nx_buf vpool, nx_buf bt, nx_buf pos, nx_buf k, nx_buf v, int batch, int tokens, int hkv, int hd,
                          int max_blocks, int num_blocks) {
    return rows_int4(ctx, "nx_kv_read_int4", false, k, v, kpool, vpool, bt, pos, batch, tokens, hkv, hd, max_blocks, num_blocks);
}

nx_status nx_attn_decode_paged_int4(nx_ctx* ctx, nx_buf q, nx_buf kpool, nx_buf vpool, nx_buf bt, nx_buf lens, nx_buf out, nx_buf weights, int batch,
                                    int hq, int hkv, int hd, int max_blocks, int num_blocks) {
    return attn_kvc(ctx, "nx_attn_decode_paged_int4", true, q, kpool, vpool, bt, lens, out, weights, batch, hq, hkv, hd, max_blocks, num_blocks);
}

nx_status nx_attn_decode_paged_f16_acc(nx_ctx* ctx, nx_buf q, nx_buf kpool, nx_buf vpool, nx_buf bt, nx_buf lens, nx_buf out, nx_buf weights,
                                       int batch, int hq, int hkv, int hd, int max_blocks, int num_blocks) {
    return attn_kvc(ctx, "nx_attn_decode_paged_f16_acc", false, q, kpool, vpool, bt, lens, out, weights, batch, hq, hkv, hd, max_blocks, num_blocks);
}

nx_status nx_kv_evict_f16(nx_ctx* ctx, nx_buf kpool, nx_buf vpool, nx_buf bt, nx_buf lens, nx_buf seen, nx_buf weights, nx_buf tags, nx_buf lens_out,
                          nx_buf weights_out, nx_buf tags_out, int batch, int hkv, int hd, int max_blocks, int num_blocks, int keep, int recent) {
    return evict(ctx, "nx_kv_evict_f16", false, kpool, vpool, bt, lens, seen, weights, tags, lens_out, weights_out, tags_out, batch, hkv, hd,
                 max_blocks, num_blocks, keep, recent);
}

nx_status nx_kv_evict_int4(nx_ctx* ctx, nx_buf kpool, nx_buf vpool, nx_buf bt, nx_buf lens, nx_buf seen, nx_buf weights, nx_buf tags, nx_buf lens_out,
                           nx_buf weights_out, nx_buf tags_out, int batch, int hkv, int hd, int max_blocks, int num_blocks, int keep, int recent) {
    return evict(ctx, "nx_kv_evict_int4", true, kpool, vpool, bt, lens, seen, weights, tags, lens_out, weights_out, tags_out, batch, hkv, hd,
                 max_blocks, num_blocks, keep, recent);
}

}  // extern "C"
