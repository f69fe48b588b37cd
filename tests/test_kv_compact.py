"""The compact KV cache: int4-g32 pages (append, read, attention), attention
that accumulates weights, eviction by weight.  Everything is compared with
plain numpy forms in 64 bits written here from the definitions; codes, moved
tokens, tags and lengths bit for bit.

Tolerances count roundings.  With A = sum_t p_t |v_t| of an output element:
  scores    q enters as fp16 hi + lo (2^-22 of q, 2^-30 of the head's largest), products add in fp32, and
            1/sqrt(hd) log2(e) is one more rounding: at most
            es = (hd + 32) 2^-24 max_t sum_i |q_i k_i| / sqrt(hd) each way
  weights   p is off by at most e = 2 es + 2^-19 of itself (exp2 and its
            argument, up to 32: 32 * 2^-24; the sum over a row; 1 / L)
  fp16 pages: p as fp16 hi + lo (2^-22), fp32 sums: e A + 2^-19 A
  int4 pages: p times scale rounded to fp16: 2^-11 A on top of that
  output    fp16: 2^-11 |out| + 2^-25 (half a step of the smallest numbers)
"""
import ctypes as C

import numpy as np
import pytest

import nexus_amd

PAGE = 16


# ------------------------------------------------------------ plain forms --
def quantize(x):
    """Codes 0..15 and fp16 scales of x [..., hd]."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], -1, 32)
    finite = np.isfinite(g).all(-1)
    amax = np.where(finite, np.abs(np.where(np.isfinite(g), g, 0)).max(-1), 0).astype(np.float32)
    with np.errstate(all="ignore"):
        s = np.minimum(amax / np.float32(7), np.float32(65504)).astype(np.float16)
        sf = s.astype(np.float32)[..., None]
        r = np.where((sf > 0) & finite[..., None], g / np.where(sf > 0, sf, 1), 0).astype(np.float32).astype(np.float64)
    q = np.clip(np.sign(r) * np.floor(np.abs(r) + 0.5), -8, 7) + 8
    s = np.where(finite, s, np.float16(np.nan)).astype(np.float16)
    return q.astype(np.uint8).reshape(x.shape), s


def places(hd, value):
    """(dword, nibble) of code [t][d] in a page, and the half of scale [t][group]."""
    t, d = np.arange(PAGE)[:, None], np.arange(hd)[None, :]
    S = hd // 32
    if value:
        word, nib = (16 * (t // 4) + d % 16) * S + d // 32, (t % 4) // 2 + 2 * ((d // 16) % 2) + 4 * (t % 2)
    else:
        word, nib = t * (hd // 8) + ((d // 8) % 4) * S + d // 32, (d % 8) // 2 + 4 * (d % 2) + 0 * t
    return word, nib, ((t // 4) * S + np.arange(S)[None, :]) * 4 + t % 4


def pack(q, s, value):
    """Records [..., 9 hd] of pages' codes [..., 16, hd] and scales [..., 16, S]."""
    hd = q.shape[-1]
    word, nib, half = places(hd, value)
    words = np.zeros((*q.shape[:-2], 2 * hd), np.uint32)
    for t in range(PAGE):
        for e in range(8):
            at = nib[t] == e
            words[..., word[t][at]] |= q[..., t, :][..., at].astype(np.uint32) << np.uint32(4 * e)
    halves = np.zeros((*q.shape[:-2], hd // 2), np.float16)
    halves[..., half] = s
    return np.concatenate([words.view(np.uint8), halves.view(np.uint8)], -1)


def unpack(rec, hd, value):
    """Values [..., 16, hd] (64 bits) of records [..., 9 hd]."""
    word, nib, half = places(hd, value)
    words = np.ascontiguousarray(rec[..., :8 * hd]).view(np.uint32)
    halves = np.ascontiguousarray(rec[..., 8 * hd:]).view(np.float16).astype(np.float64)
    q = (words[..., word] >> (4 * nib).astype(np.uint32)) & 15
    return (q.astype(np.float64) - 8) * np.repeat(halves[..., half], 32, -1)


def to_pages(x, table, nblk, fill):
    """Pages [nblk][hkv][16][hd] that hold x[b] = [n][hkv][hd] through table; other tokens hold `fill`."""
    hkv, hd = x[0].shape[1:]
    pages = np.full((nblk, hkv, PAGE, hd), fill, np.float32)
    for b, rows in enumerate(x):
        for p in range(rows.shape[0]):
            pages[table[b, p // PAGE], :, p % PAGE] = rows[p]
    return pages


def in_order(pages, table, n):
    """[n][hkv][hd] of one sequence."""
    if n == 0:
        return np.zeros((0, pages.shape[1], pages.shape[3]))
    return pages[table[:-(-n // PAGE)]].transpose(0, 2, 1, 3).reshape(-1, pages.shape[1], pages.shape[3])[:n]


def attention(q, k, v):
    """out [hq][hd], weights [hkv][n], and what the tolerances need, for one
    sequence's q [hq][hd] and k, v [n][hkv][hd]."""
    hq, hd = q.shape
    n, hkv, _ = k.shape
    G = hq // hkv
    out, A, W, es = np.zeros((hq, hd)), np.zeros((hq, hd)), np.zeros((hkv, n)), 0.0
    q = q.astype(np.float64)
    for h in range(hq if n else 0):
        j = h // G
        s = k[:, j] @ q[h] / np.sqrt(hd)
        es = max(es, (hd + 32) * 2.0**-24 * (np.abs(k[:, j]) @ np.abs(q[h])).max() / np.sqrt(hd))
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h], A[h] = p @ v[:, j], p @ np.abs(v[:, j])
        W[j] += p
    return out, W, A, 2 * es + 2.0**-19


# ------------------------------------------------------------------- helpers --
def up(ctx, a):
    return ctx.upload(np.ascontiguousarray(a))


class Held:
    """Buffers of one test, given back at its end."""

    def __init__(self, ctx, **arrays):
        self.ctx, self.b, self.a = ctx, {}, {}
        for n, v in arrays.items():
            self.put(n, v)

    def put(self, name, value):
        self.a[name] = np.ascontiguousarray(value)
        self.b[name] = self.ctx.upload(self.a[name], self.b.get(name))

    def __getitem__(self, name):
        return self.b[name]

    def get(self, name):
        return self.ctx.download(self.b[name], self.a[name].shape, self.a[name].dtype)

    def free(self):
        for v in self.b.values():
            self.ctx.free(v)


def table_of(rng, B, max_blocks, nblk):
    return rng.permutation(nblk)[:B * max_blocks].reshape(B, max_blocks).astype(np.int32)


def cache(rng, int4, lens, hkv, hd, max_blocks, nblk, amp=1.0, stale=np.nan):
    """Pools as the library holds them, their values in 64 bits, and the table.
    Tokens past the lengths hold `stale`, table entries past them nonsense."""
    B = len(lens)
    if nblk >= B * max_blocks:
        table = table_of(rng, B, max_blocks, nblk)
    else:  # pages for the tokens alone
        table, free = np.zeros((B, max_blocks), np.int32), rng.permutation(nblk).astype(np.int32)
        for b, n in enumerate(lens):
            table[b, :-(-n // PAGE)], free = np.split(free, [-(-n // PAGE)])
    ks, vs = ([(rng.normal(0, 1, (n, hkv, hd)) * amp).astype(np.float32) for n in lens] for _ in range(2))
    pk, pv = to_pages(ks, table, nblk, stale), to_pages(vs, table, nblk, stale)
    if int4:
        kp, vp = pack(*quantize(pk), False), pack(*quantize(pv), True)
        k64, v64 = unpack(kp, hd, False), unpack(vp, hd, True)
    else:
        kp, vp = pk.astype(np.float16), np.ascontiguousarray(pv.astype(np.float16).transpose(0, 1, 3, 2))
        k64, v64 = kp.astype(np.float64), vp.astype(np.float64).transpose(0, 1, 3, 2)
    for b, n in enumerate(lens):
        table[b, -(-n // PAGE):] = [-1, 1 << 30, nblk, -(1 << 31)][b % 4]
    return kp, vp, k64, v64, table


# ------------------------------------------------------ on the CPU: layout --
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("value", [False, True])
def test_every_code_has_a_nibble_of_its_own(hd, value):
    word, nib, half = places(hd, value)
    at = word * 8 + nib
    assert sorted(at.ravel()) == list(range(PAGE * hd))
    assert sorted(half.ravel()) == list(range(PAGE * hd // 32))
    rng = np.random.default_rng(hd)
    q, s = quantize(rng.normal(0, 1, (3, 2, PAGE, hd)))
    want = (q.astype(np.float64) - 8) * np.repeat(s.astype(np.float64), 32, -1)
    assert np.array_equal(unpack(pack(q, s, value), hd, value), want)


@pytest.mark.parametrize("max_blocks", [1, 2, 5, 1 << 22])
def test_row_pages_stay_inside_the_table(max_blocks):
    """The pages of an append: inside the table, every row in exactly one,
    no more than the launch has; out of range: refused."""
    L = nexus_amd.lib()
    L.nx_kvc_row_page.argtypes = [C.c_int] * 4 + [C.POINTER(C.c_int)]
    out = (C.c_int * 4)()
    cap = max_blocks * PAGE
    firsts = {f for f in (-(1 << 31), -1, 0, 1, 15, 16, 17, 31, cap - 17, cap - 16, cap - 1, cap, (1 << 31) - 1) if f < 1 << 31}
    for first in firsts:
        for tokens in (1, 2, 15, 16, 17, 18, 33, 80):
            if tokens > cap:
                continue
            n = L.nx_kvc_row_page(first, tokens, max_blocks, 0, out)
            rows = []
            ok = 0 <= first and first + tokens <= cap
            for i in range(n):
                L.nx_kvc_row_page(first, tokens, max_blocks, i, out)
                page, row0, none, refused = out
                assert bool(refused) == (not ok)
                if none:
                    continue
                assert not ok or 0 <= page < max_blocks
                rows += [r for r in range(row0, row0 + PAGE) if 0 <= r < tokens]
                if ok:
                    assert page * PAGE == first + row0
            assert rows == list(range(tokens))


# --------------------------------------------------- on the CPU: refusals --
SHAPE = dict(batch=2, hq=8, hkv=2, hd=64, max_blocks=3, num_blocks=7, tokens=20, keep=9, recent=4)


def sizes(op, s):
    """Bytes that each buffer of a call needs, in the call's order."""
    pool = s["num_blocks"] * s["hkv"] * (9 * s["hd"] if "int4" in op else 32 * s["hd"])
    rows, tab, lens = s["batch"] * s["tokens"] * s["hkv"] * s["hd"] * 4, s["batch"] * s["max_blocks"] * 4, s["batch"] * 4
    slots, q = s["batch"] * s["hkv"] * s["max_blocks"] * 64, s["batch"] * s["hq"] * s["hd"]
    return {"nx_kv_append_int4": [rows, rows, pool, pool, tab, lens],
            "nx_kv_read_int4": [pool, pool, tab, lens, rows, rows],
            "nx_attn_decode_paged_int4": [4 * q, pool, pool, tab, lens, 2 * q, slots],
            "nx_attn_decode_paged_f16_acc": [4 * q, pool, pool, tab, lens, 2 * q, slots],
            "nx_kv_evict_f16": [pool, pool, tab, lens, lens, slots, slots, lens, slots, slots],
            "nx_kv_evict_int4": [pool, pool, tab, lens, lens, slots, slots, lens, slots, slots]}[op]


OPS = ["nx_kv_append_int4", "nx_kv_read_int4", "nx_attn_decode_paged_int4", "nx_attn_decode_paged_f16_acc", "nx_kv_evict_f16",
       "nx_kv_evict_int4"]


def numbers(op, s):
    if "attn" in op:
        return [s[n] for n in ("batch", "hq", "hkv", "hd", "max_blocks", "num_blocks")]
    if "evict" in op:
        return [s[n] for n in ("batch", "hkv", "hd", "max_blocks", "num_blocks", "keep", "recent")]
    return [s[n] for n in ("batch", "tokens", "hkv", "hd", "max_blocks", "num_blocks")]


def call(op, bufs, s, need=None):
    """Status and message of a call on a context whose buffers are numbers
    alone: a call that refuses nothing answers that there is no device (6)."""
    L = nexus_amd.lib()
    need = sizes(op, SHAPE) if need is None else need
    L.nx_deviceless.restype = C.c_void_p
    ctx = C.c_void_p(L.nx_deviceless((C.c_size_t * len(need))(*need), len(need)))
    st = getattr(L, op)(ctx, *bufs, *numbers(op, s))
    msg = L.nx_last_error(ctx).decode()
    L.nx_destroy(ctx)
    return st, msg


@pytest.mark.parametrize("op", OPS)
def test_refusals(op):
    n = len(sizes(op, SHAPE))
    ids = list(range(1, n + 1))
    assert call(op, ids, SHAPE)[0] == 6  # the call itself is in order
    assert getattr(nexus_amd.lib(), op)(None, *ids, *numbers(op, SHAPE)) == 1
    for name in ("batch", "hkv", "hd", "max_blocks", "num_blocks"):
        for bad in (0, -1):
            assert call(op, ids, dict(SHAPE, **{name: bad}))[0] == 1, name
    for hd in (32, 96, 80, 512):
        assert call(op, ids, dict(SHAPE, hd=hd))[0] == 4
    for name, big in (("batch", 65536), ("hkv", 4097), ("max_blocks", (1 << 22) + 1), ("max_blocks", (1 << 31) - 1)):
        assert call(op, ids, dict(SHAPE, hq=big * 4 if name == "hkv" else 8, **{name: big}))[0] == 4, name
    # sizes whose product passes 64 bits would wrap: they are larger than any buffer
    assert call(op, ids, dict(SHAPE, num_blocks=(1 << 31) - 1))[0] == 1
    for i in range(n):
        need = sizes(op, SHAPE)
        need[i] -= 1
        st, msg = call(op, ids, SHAPE, need)
        assert st == 1 and "needs" in msg, i
        st, msg = call(op, ids[:i] + [999] + ids[i + 1:], SHAPE)
        assert st == 1 and "unknown buffer" in msg, i
        if not (op == "nx_attn_decode_paged_int4" and i == 6):  # no weights is a choice there
            assert call(op, ids[:i] + [0] + ids[i + 1:], SHAPE)[0] == 1, i
    if "attn" in op:
        assert call(op, ids, dict(SHAPE, hq=7))[0] == 1
        assert call(op, ids, dict(SHAPE, hq=0))[0] == 1
        assert call(op, ids, dict(SHAPE, hq=130))[0] == 4
        assert call(op, ids[:6] + [0], SHAPE)[0] == (6 if "int4" in op else 1)
        for out in (5, 6):  # the output and the weights are buffers of their own
            for i in range(n):
                if i != out:
                    assert call(op, ids[:out] + [ids[i]] + ids[out + 1:], SHAPE, [1 << 20] * n)[0] == 1
    elif "evict" in op:
        for keep, recent in ((0, 0), (-1, 0), (4, 5), (4, -1)):
            assert call(op, ids, dict(SHAPE, keep=keep, recent=recent))[0] == 1
        assert call(op, ids, dict(SHAPE, keep=1 << 30, recent=1 << 30))[0] == 6
        big = [1 << 20] * n
        for out, src in ((7, 3), (8, 5), (9, 6)):  # an output may be the input of its kind alone
            for i in range(n):
                if i != out:
                    st, _ = call(op, ids[:out] + [ids[i]] + ids[out + 1:], SHAPE, big)
                    assert st == (6 if i == src else 1), (out, i)
        assert call(op, [1, 1] + ids[2:], SHAPE, big)[0] == 1
    else:
        assert call(op, ids, dict(SHAPE, tokens=0))[0] == 1
        assert call(op, ids, dict(SHAPE, tokens=49))[0] == 7
        for out in ((2, 3) if "append" in op else (4, 5)):
            for i in range(n):
                if i != out:
                    assert call(op, ids[:out] + [ids[i]] + ids[out + 1:], SHAPE, [1 << 20] * n)[0] == 1


# ---------------------------------------------------------- append and read --
def odd_rows(rng, B, T, hkv, hd):
    """Rows with what a quantizer meets: zeros, values on a half step, tiny, huge and non-finite groups."""
    x = rng.normal(0, 1, (B, T, hkv, hd)).astype(np.float32)
    flat = x.reshape(-1, 32)
    for i, row in enumerate(flat[:: max(1, len(flat) // 97)]):
        kind = i % 9
        if kind == 0:
            row[:] = 0
        elif kind == 1:
            row[:] = (rng.integers(-15, 16, 32) / 2).astype(np.float32)
            row[0] = 7.0
        elif kind == 2:
            row *= np.float32(1e-7)
        elif kind == 3:
            row *= np.float32(1e7)
        elif kind == 4:
            row[3] = np.nan
        elif kind == 5:
            row[31] = -np.inf
        elif kind == 6:
            row *= np.float32(1e-39)
        elif kind == 7:
            row[:] = -0.0
        else:
            row[:] = -np.abs(row)
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("hd,hkv,parts,starts", [
    (64, 1, [1], [0]), (64, 2, [3, 1, 20], [5, 0]), (128, 8, [1], [47, 15, 0, 31]), (128, 3, [16, 17, 15], [0]),
    (128, 2, [300], [7, 16]), (256, 1, [2, 2, 2, 2, 2], [13]), (256, 5, [33], [0, 31, 16])])
def test_append_and_read_bit_exact(ctx, hd, hkv, parts, starts):
    """Pages as the plain form packs them, whatever the parts the rows come
    in; every other byte as it was; and the same values read back."""
    rng = np.random.default_rng(hd * 31 + hkv + sum(parts))
    B, T = len(starts), sum(parts)
    mb = -(-(max(starts) + T) // PAGE)
    nblk = B * mb + 3
    table = table_of(rng, B, mb, nblk)
    k, v = odd_rows(rng, B, T, hkv, hd), odd_rows(rng, B, T, hkv, hd)
    kp0, vp0 = (rng.integers(0, 256, (nblk, hkv, 9 * hd), dtype=np.uint8) for _ in range(2))
    h = Held(ctx, kp=kp0, vp=vp0, table=table, pos=np.array(starts, np.int32))
    done = 0
    for n in parts:
        ids = [up(ctx, k[:, done:done + n]), up(ctx, v[:, done:done + n])]
        h.put("pos", np.array(starts, np.int32) + np.int32(done))
        ctx.kv_append_int4(*ids, h["kp"], h["vp"], h["table"], h["pos"], B, n, hkv, hd, mb, nblk)
        ctx.sync()
        for i in ids:
            ctx.free(i)
        done += n
    for name, rows, was, value in (("kp", k, kp0, False), ("vp", v, vp0, True)):
        q, s = quantize(rows)
        word, nib, half = places(hd, value)
        words, halves = was[..., :8 * hd].copy().view(np.uint32), was[..., 8 * hd:].copy().view(np.uint16)
        for b in range(B):
            for i in range(T):
                blk, t = table[b, (starts[b] + i) // PAGE], (starts[b] + i) % PAGE
                for e in range(8):
                    at = nib[t] == e
                    w = word[t][at]
                    words[blk][:, w] = (words[blk][:, w] & ~np.uint32(15 << 4 * e)) | (q[b, i][:, at].astype(np.uint32) << np.uint32(4 * e))
                bits = s[b, i].view(np.uint16)
                halves[blk][:, half[t]] = np.where(np.isnan(s[b, i]), np.uint16(0x7E00), bits)
        want = np.concatenate([words.view(np.uint8), halves.view(np.uint8)], -1)
        got = h.get(name)
        assert np.array_equal(got, want), f"{name}: {np.argwhere(got != want)[:5]}"
    h.put("pos", np.array(starts, np.int32))
    h.put("ko", np.full((B, T, hkv, hd), 77, np.float32))
    h.put("vo", np.full((B, T, hkv, hd), 77, np.float32))
    ctx.kv_read_int4(h["kp"], h["vp"], h["table"], h["pos"], h["ko"], h["vo"], B, T, hkv, hd, mb, nblk)
    for name, rows in (("ko", k), ("vo", v)):
        q, s = quantize(rows)
        want = (q.astype(np.float32) - 8) * np.repeat(s.astype(np.float32), 32, -1)
        assert np.array_equal(h.get(name), want, equal_nan=True)
    h.free()


@pytest.mark.gpu
def test_append_and_read_out_of_range(ctx):
    """Sequences out of range write nothing and read NaN; a page whose table
    entry lies outside the pool likewise, with the other pages in order."""
    rng = np.random.default_rng(5)
    hd, hkv, T, mb, nblk = 64, 2, 20, 4, 19
    starts = np.array([-1, 45, 44, 0, (1 << 31) - 1, -(1 << 31)], np.int32)
    B = len(starts)
    table = np.arange(B * mb, dtype=np.int32).reshape(B, mb) % nblk
    table[0], table[1], table[4], table[5] = 0, 1, 2, 3   # in the pool: their positions are at fault
    table[2], table[3] = [5, 6, 7, 8], [9, nblk, 10, -1]   # 44..63: pages 2, 3; 0..19: pages 0 and 1 (outside)
    k, v = rng.normal(0, 1, (2, B, T, hkv, hd)).astype(np.float32)
    pool = rng.integers(0, 256, (nblk, hkv, 9 * hd), dtype=np.uint8)
    h = Held(ctx, k=k, v=v, kp=pool, vp=pool, table=table, pos=starts, ko=np.zeros_like(k), vo=np.zeros_like(k))
    ctx.kv_append_int4(h["k"], h["v"], h["kp"], h["vp"], h["table"], h["pos"], B, T, hkv, hd, mb, nblk)
    ctx.kv_read_int4(h["kp"], h["vp"], h["table"], h["pos"], h["ko"], h["vo"], B, T, hkv, hd, mb, nblk)
    touched = {7, 8, 9}
    for name in ("kp", "vp"):
        got = h.get(name)
        assert np.array_equal(got[[i for i in range(nblk) if i not in touched]], pool[[i for i in range(nblk) if i not in touched]])
    for name, rows in (("ko", k), ("vo", v)):
        q, s = quantize(rows)
        want = (q.astype(np.float32) - 8) * np.repeat(s.astype(np.float32), 32, -1)
        want[[0, 1, 4, 5]] = np.nan
        want[3, 16:] = np.nan
        assert np.array_equal(h.get(name), want, equal_nan=True)
    h.free()


# ------------------------------------------------------------------ attention --
def check_attention(ctx, int4, hq, hkv, hd, lens, weights=True, amp=1.0, spare=2, qamp=1.0, twice=False, seed=0, nblk=0):
    rng = np.random.default_rng(seed + hq * 7 + hd + sum(lens))
    B, mb = len(lens), max(1, -(-max(lens) // PAGE)) + spare
    nblk = nblk or B * mb + 1
    kp, vp, k64, v64, table = cache(rng, int4, lens, hkv, hd, mb, nblk, amp)
    q = (rng.normal(0, 1, (B, hq, hd)) * qamp).astype(np.float32)
    w0 = rng.exponential(1, (B, hkv, mb * PAGE)).astype(np.float32)
    h = Held(ctx, q=q, kp=kp, vp=vp, table=table, lens=np.array(lens, np.int32), out=np.full((B, hq, hd), 9, np.float16), w=w0)
    f = ctx.attn_decode_paged_int4 if int4 else ctx.attn_decode_paged_f16_acc
    for _ in range(2 if twice else 1):
        f(h["q"], h["kp"], h["vp"], h["table"], h["lens"], h["out"], h["w"] if weights else 0, B, hq, hkv, hd, mb, nblk)
    out, w = h.get("out").astype(np.float64), h.get("w")
    h.free()
    for b, n in enumerate(lens):
        want, W, A, e = attention(q[b], in_order(k64, table[b], n), in_order(v64, table[b], n))
        tol = 2.0**-11 * (np.abs(want) + (A if int4 else 0)) + (e + 2.0**-19) * A + 2.0**-25
        off = np.abs(out[b] - want)
        assert (off <= tol).all(), f"sequence {b}: out off by {(off / tol).max():.3g} of the bound"
        add = (2 if twice else 1) * W if weights else 0 * W
        full = w0[b].astype(np.float64)
        full[:, :n] += add
        # one or two fp32 additions, and p itself
        tol = 2.0**-23 * np.abs(full)
        tol[:, :n] += e * add
        off = np.abs(w[b] - full)
        assert (off <= tol).all(), f"sequence {b}: weights off by {(off / np.maximum(tol, 1e-30)).max():.3g} of the bound"
        assert np.array_equal(w[b][:, n:], w0[b][:, n:])


@pytest.mark.gpu
@pytest.mark.parametrize("int4", [True, False], ids=["int4", "f16"])
@pytest.mark.parametrize("hq,hkv,hd,lens", [
    (1, 1, 64, [1]), (4, 2, 64, [0, 1, 2, 15, 16, 17, 31, 32, 33]), (8, 8, 128, [100, 0]), (32, 8, 128, [257, 513, 1]),
    (6, 2, 128, [48, 49]), (5, 1, 64, [1000]), (14, 2, 256, [16, 700]), (9, 1, 128, [130]), (36, 3, 64, [77, 5]),
    (64, 1, 64, [300]), (16, 1, 256, [33, 2000]), (32, 8, 128, [4096] * 2), (8, 2, 128, [20000]), (2, 2, 256, [9001])])
def test_attention(ctx, int4, hq, hkv, hd, lens):
    print(f"[case] {'int4' if int4 else 'f16'} hq={hq} hkv={hkv} hd={hd} lens={lens}", flush=True)
    check_attention(ctx, int4, hq, hkv, hd, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,hd,lens", [(4, 2, 64, [0, 40]), (32, 8, 128, [300]), (12, 1, 256, [999, 16])])
def test_attention_int4_without_weights(ctx, hq, hkv, hd, lens):
    check_attention(ctx, True, hq, hkv, hd, lens, weights=False)


@pytest.mark.gpu
@pytest.mark.parametrize("int4,weights", [(True, True), (True, False), (False, True)], ids=["int4", "int4-plain", "f16"])
def test_attention_of_many_rows(ctx, int4, weights):
    """More rows than the device holds blocks, so one block to a row or two, and
    one long sequence among short ones: a wavefront's pages pass 64 of the table."""
    check_attention(ctx, int4, 256, 4, 64, [18001] + [1, 17, 0, 40] * 47, weights=weights, nblk=1500)


@pytest.mark.gpu
@pytest.mark.parametrize("int4", [True, False], ids=["int4", "f16"])
def test_attention_past_the_joins_first_slots(ctx, int4):
    check_attention(ctx, int4, 9, 1, 64, [40000, 32769])


@pytest.mark.gpu
@pytest.mark.parametrize("int4", [True, False], ids=["int4", "f16"])
@pytest.mark.parametrize("amp", [1e-3, 30.0, 2000.0])
def test_attention_amplitudes(ctx, int4, amp):
    """Scales from fp16's smallest normal numbers to above 2 (whose products
    go without the probabilities' factor); q scaled so that scores stay moderate."""
    check_attention(ctx, int4, 8, 2, 128, [500, 31], amp=amp, qamp=1.0 / amp)


@pytest.mark.gpu
@pytest.mark.parametrize("int4", [True, False], ids=["int4", "f16"])
def test_attention_peaked_rows_and_calls_in_a_row(ctx, int4):
    check_attention(ctx, int4, 8, 2, 64, [600, 3], qamp=8.0, twice=True)
    check_attention(ctx, int4, 4, 1, 64, [2], twice=True)


@pytest.mark.gpu
@pytest.mark.parametrize("int4", [True, False], ids=["int4", "f16"])
@pytest.mark.parametrize("qamp", [0.0, 1e-42, 1e-30, 1e30, 3e37])
def test_attention_extreme_queries(ctx, int4, qamp):
    """Queries far below and above 1: all tokens weigh the same, or one weighs 1
    (p is exact then, so an output is off by the rounding of p times the scale
    and its own, 2^-11 of it each)."""
    rng = np.random.default_rng(12)
    hq, hkv, hd, n, mb = 4, 2, 64, 50, 4
    kp, vp, k64, v64, table = cache(rng, int4, [n], hkv, hd, mb, mb)
    q = (rng.uniform(-1, 1, (1, hq, hd)) * qamp).astype(np.float32)
    h = Held(ctx, q=q, kp=kp, vp=vp, table=table, lens=np.array([n], np.int32), out=np.zeros((1, hq, hd), np.float16),
             w=np.zeros((1, hkv, mb * PAGE), np.float32))
    f = ctx.attn_decode_paged_int4 if int4 else ctx.attn_decode_paged_f16_acc
    f(h["q"], h["kp"], h["vp"], h["table"], h["lens"], h["out"], h["w"], 1, hq, hkv, hd, mb, mb)
    out, w = h.get("out")[0].astype(np.float64), h.get("w")[0]
    h.free()
    want, W, A, e = attention(q[0], in_order(k64, table[0], n), in_order(v64, table[0], n))
    if qamp > 1:
        assert np.array_equal(W, np.round(W)) and np.array_equal(w[:, :n], W)
        e = 0.0
    assert (np.abs(out - want) <= 2.0**-11 * (np.abs(want) + A) + (e + 2.0**-19) * A + 2.0**-25).all()
    assert np.abs(w[:, :n] - W).max() <= e * W.max() + 2.0**-22


@pytest.mark.gpu
@pytest.mark.parametrize("int4", [True, False], ids=["int4", "f16"])
def test_attention_out_of_range(ctx, int4):
    """A length or a table entry out of range: NaN rows, weights as they were,
    the other sequences unharmed."""
    rng = np.random.default_rng(3)
    hq, hkv, hd, mb = 8, 2, 64, 40
    good = [600, 33, 40, 20, 50]
    B, nblk = len(good), 5 * mb
    kp, vp, k64, v64, table = cache(rng, int4, good, hkv, hd, mb, nblk)
    lens = np.array(good, np.int32)
    lens[1], lens[2] = mb * PAGE + 1, -1
    table[3, 1], table[4, 0] = nblk, -1
    q = rng.normal(0, 1, (B, hq, hd)).astype(np.float32)
    w0 = rng.exponential(1, (B, hkv, mb * PAGE)).astype(np.float32)
    h = Held(ctx, q=q, kp=kp, vp=vp, table=table, lens=lens, out=np.zeros((B, hq, hd), np.float16), w=w0)
    f = ctx.attn_decode_paged_int4 if int4 else ctx.attn_decode_paged_f16_acc
    f(h["q"], h["kp"], h["vp"], h["table"], h["lens"], h["out"], h["w"], B, hq, hkv, hd, mb, nblk)
    out, w = h.get("out"), h.get("w")
    h.free()
    assert np.isnan(out[1:]).all() and np.array_equal(w[1:], w0[1:])
    want, W, A, e = attention(q[0], in_order(k64, table[0], 600), in_order(v64, table[0], 600))
    assert (np.abs(out[0] - want) <= 2.0**-11 * (np.abs(want) + A) + (e + 2.0**-19) * A + 2.0**-25).all()
    assert not np.array_equal(w[0], w0[0])


@pytest.mark.gpu
@pytest.mark.parametrize("int4", [True, False], ids=["int4", "f16"])
def test_attention_non_finite_tokens(ctx, int4):
    """A NaN among the cached keys makes its kv head's rows and weights NaN,
    one among the values the outputs of its dimensions (int4: of its group)."""
    rng = np.random.default_rng(4)
    hq, hkv, hd, n, mb = 4, 2, 64, 50, 4
    table = np.arange(mb, dtype=np.int32)[None]
    k, v = rng.normal(0, 1, (2, n, hkv, hd)).astype(np.float32)
    k[20, 0, 5] = np.nan
    v[49, 1, 40] = np.nan
    pk, pv = to_pages([k], table, mb, 0), to_pages([v], table, mb, 0)
    kp, vp = (pack(*quantize(pk), False), pack(*quantize(pv), True)) if int4 else (
        pk.astype(np.float16), pv.astype(np.float16).transpose(0, 1, 3, 2))
    h = Held(ctx, q=rng.normal(0, 1, (1, hq, hd)).astype(np.float32), kp=kp, vp=vp, table=table, lens=np.array([n], np.int32),
             out=np.zeros((1, hq, hd), np.float16), w=np.zeros((1, hkv, mb * PAGE), np.float32))
    f = ctx.attn_decode_paged_int4 if int4 else ctx.attn_decode_paged_f16_acc
    f(h["q"], h["kp"], h["vp"], h["table"], h["lens"], h["out"], h["w"], 1, hq, hkv, hd, mb, mb)
    out, w = h.get("out")[0], h.get("w")[0]
    h.free()
    assert np.isnan(out[:2]).all() and np.isnan(w[0, :n]).all() and (w[0, n:] == 0).all()
    hit = np.zeros(hd, bool)
    hit[32:64 if int4 else 0] = True
    hit[40] = True
    assert np.array_equal(np.isnan(out[2:]), np.broadcast_to(hit, (2, hd)))
    assert np.isfinite(w[1]).all() and abs(w[1].sum() - 2) < 1e-4


# ------------------------------------------------------------------- eviction --
def evict(lens, seen, w, tags, keep, recent):
    """The plain form: per (b, h) the slot that each new slot takes its token
    from, and the new lengths, weights and tags."""
    B, hkv, cap = w.shape
    src = np.tile(np.arange(cap), (B, hkv, 1))
    w2, t2, lens2 = np.zeros_like(w), np.zeros_like(tags), np.zeros(B, np.int32)
    for b in range(B):
        L, N = int(lens[b]), int(seen[b])
        lens2[b] = min(L, keep)
        for h in range(hkv):
            pos = np.where(tags[b, h, :L] > 0, tags[b, h, :L].astype(np.int64) - 1, N - L + np.arange(L))
            if L > keep:
                x = w[b, h, :L].astype(np.float64)
                rank = sorted(range(L), key=lambda s: (not pos[s] >= N - recent, 0 if pos[s] >= N - recent else 1 if x[s] == x[s] else 2,
                                                       -x[s] if x[s] == x[s] and pos[s] < N - recent else 0, s))
                kept = np.zeros(L, bool)
                kept[rank[:keep]] = True
                src[b, h, np.flatnonzero(~kept[:keep])] = keep + np.flatnonzero(kept[keep:])
            n = lens2[b]
            w2[b, h, :n] = w[b, h, src[b, h, :n]]
            t2[b, h, :n] = pos[src[b, h, :n]] + 1
    return src, lens2, w2, t2


def tokens_of(int4, pools, hd):
    """What identifies a token's K and V: the values that the pages stand for [blk][hkv][16][hd]."""
    kp, vp = pools
    return (unpack(kp, hd, False), unpack(vp, hd, True)) if int4 else (kp, vp.transpose(0, 1, 3, 2))


def run_evict(ctx, int4, h, B, hkv, hd, mb, nblk, keep, recent, alias):
    o = ("lens", "w", "tags") if alias else ("lens_o", "w_o", "tags_o")
    f = ctx.kv_evict_int4 if int4 else ctx.kv_evict_f16
    f(h["kp"], h["vp"], h["table"], h["lens"], h["seen"], h["w"], h["tags"], *[h[n] for n in o], B, hkv, hd, mb, nblk, keep, recent)
    return o


@pytest.mark.gpu
@pytest.mark.parametrize("int4", [True, False], ids=["int4", "f16"])
@pytest.mark.parametrize("hd,hkv,lens,keep,recent,alias", [
    (64, 1, [2], 1, 0, False), (64, 2, [1, 17, 16, 0, 40], 16, 3, True), (128, 2, [100, 33], 37, 37, False),
    (128, 8, [257], 256, 64, True), (256, 1, [300, 64], 63, 0, False), (64, 3, [1500], 700, 100, True),
    (128, 1, [5000, 4000], 4001, 9, False), (64, 1, [20, 48], 48, 5, False), (64, 1, [20, 48], 1000, 900, True),
    (64, 1, [20000], 3000, 100, False), (64, 1, [40000], 9000, 500, False), (64, 1, [70000, 33000], 30000, 1000, True),
    (64, 1, [70000], 69990, 69000, False)])
def test_eviction(ctx, int4, hd, hkv, lens, keep, recent, alias):
    """Tokens, weights, tags and lengths as the plain form has them, twice in a
    row with tokens appended between; no other byte of the pools changes."""
    print(f"[case] {'int4' if int4 else 'f16'} hd={hd} hkv={hkv} lens={lens} keep={keep} recent={recent}", flush=True)
    rng = np.random.default_rng(hd + keep + recent)
    B, mb = len(lens), max(1, -(-max(lens) // PAGE))
    nblk = B * mb + 1
    cap = mb * PAGE
    kp, vp, _, _, table = cache(rng, int4, lens, hkv, hd, mb, nblk, stale=3.0)
    w = np.where(np.arange(cap) < np.array(lens)[:, None, None], np.exp(2 * rng.normal(0, 1, (B, hkv, cap))), 0).astype(np.float32)
    for x, share in ((0.0, 0.1), (-0.0, 0.1), (1.0, 0.2), (np.nan, 0.05), (np.inf, 0.02), (-np.inf, 0.02), (-1.5, 0.03), (1e-40, 0.03)):
        w[rng.random(w.shape) < share] = x
    seen = np.array(lens, np.int32) + rng.integers(0, 50, B).astype(np.int32)
    z = np.zeros_like(w)
    h = Held(ctx, kp=kp, vp=vp, table=table, lens=np.array(lens, np.int32), seen=seen, w=w, tags=z.astype(np.int32),
             lens_o=np.full(B, 7, np.int32), w_o=z + 5, tags_o=(z + 5).astype(np.int32))
    for again in range(2):
        before = [h.get(n) for n in ("kp", "vp", "w", "tags")]
        src, lens2, w2, t2 = evict(h.get("lens"), h.get("seen"), before[2], before[3], keep, recent)
        o = run_evict(ctx, int4, h, B, hkv, hd, mb, nblk, keep, recent, alias)
        assert np.array_equal(h.get(o[0]), lens2)
        assert np.array_equal(h.get(o[1]).view(np.uint32), w2.view(np.uint32))
        assert np.array_equal(h.get(o[2]), t2)
        was, now = tokens_of(int4, before[:2], hd), tokens_of(int4, (h.get("kp"), h.get("vp")), hd)
        for x, y in zip(was, now):
            want = x.copy()
            for b in range(B):
                for hh in range(hkv):
                    for s in np.flatnonzero(src[b, hh] != np.arange(cap)):
                        f = src[b, hh, s]
                        want[table[b, s // PAGE], hh, s % PAGE] = x[table[b, f // PAGE], hh, f % PAGE]
            assert np.array_equal(y, want)
        # some tokens more, in fresh slots, with little weight
        n = np.minimum(lens2 + 5, np.array(lens))
        w3, t3 = w2.copy(), t2.copy()
        for b in range(B):
            w3[b, :, lens2[b]:n[b]] = 0.25
        h.put("lens", n.astype(np.int32))
        h.put("seen", seen + (again + 1) * 5)
        h.put("w", w3)
        h.put("tags", t3)
    h.free()


@pytest.mark.gpu
@pytest.mark.parametrize("int4", [True, False], ids=["int4", "f16"])
def test_eviction_out_of_range(ctx, int4):
    """A length out of range, more cached than seen, a table entry outside the
    pool: length -1, nothing else written; the other sequence is cut."""
    rng = np.random.default_rng(8)
    hd, hkv, mb, keep = 64, 2, 4, 20
    good = [60, 64, 64, 64, 50]
    B, nblk = len(good), 5 * 4
    kp, vp, _, _, table = cache(rng, int4, good, hkv, hd, mb, nblk, stale=3.0)
    lens, seen = np.array(good, np.int32), np.array(good, np.int32) + 3
    lens[1], lens[2], seen[3] = mb * PAGE + 1, -5, 63
    table[4, 2] = nblk
    w = rng.exponential(1, (B, hkv, mb * PAGE)).astype(np.float32)
    h = Held(ctx, kp=kp, vp=vp, table=table, lens=lens, seen=seen, w=w, tags=np.zeros(w.shape, np.int32), lens_o=np.zeros(B, np.int32),
             w_o=np.full(w.shape, 5, np.float32), tags_o=np.full(w.shape, 5, np.int32))
    run_evict(ctx, int4, h, B, hkv, hd, mb, nblk, keep, 2, False)
    assert h.get("lens_o").tolist() == [keep, -1, -1, -1, -1]
    assert (h.get("w_o")[1:] == 5).all() and (h.get("tags_o")[1:] == 5).all()
    src, _, w2, t2 = evict(lens[:1], seen[:1], w[:1], np.zeros(w[:1].shape, np.int32), keep, 2)
    assert np.array_equal(h.get("w_o")[:1], w2) and np.array_equal(h.get("tags_o")[:1], t2)
    others = [i for i in range(nblk) if i not in table[0]]
    assert np.array_equal(h.get("kp")[others], kp[others]) and np.array_equal(h.get("vp")[others], vp[others])
    h.free()


# ------------------------------------------------------------------ together --
class Session:
    """A small decoder's cache: rows appended, attended to and evicted, with
    the plain forms beside the calls, which start from the library's own
    weights (a choice between near-equal weights is then the same)."""

    def __init__(self, ctx, int4, B=2, hq=6, hkv=2, hd=64, mb=6, seed=1):
        self.ctx, self.int4, self.B, self.hq, self.hkv, self.hd, self.mb = ctx, int4, B, hq, hkv, hd, mb
        self.rng = np.random.default_rng(seed)
        self.nblk = B * mb
        pool = np.zeros((self.nblk, hkv, 9 * hd), np.uint8) if int4 else np.zeros((self.nblk, hkv, 16, hd), np.float16)
        slots = np.zeros((B, hkv, mb * PAGE), np.float32)
        self.h = Held(ctx, kp=pool, vp=pool if int4 else pool.transpose(0, 1, 3, 2), table=table_of(self.rng, B, mb, self.nblk),
                      lens=np.zeros(B, np.int32), pos=np.zeros(B, np.int32), seen=np.zeros(B, np.int32), w=slots,
                      tags=slots.astype(np.int32), q=np.zeros((B, hq, hd), np.float32), out=np.zeros((B, hq, hd), np.float16),
                      k=np.zeros((B, 1, hkv, hd), np.float32), v=np.zeros((B, 1, hkv, hd), np.float32))
        self.lens = np.zeros(B, np.int32)
        self.seen = 0

    def inputs(self):
        """A new token's rows and query; lengths as the host keeps them."""
        h, r = self.h, self.rng
        h.put("k", r.normal(0, 1, (self.B, 1, self.hkv, self.hd)).astype(np.float32))
        h.put("v", r.normal(0, 1, (self.B, 1, self.hkv, self.hd)).astype(np.float32))
        h.put("q", 2 * r.normal(0, 1, (self.B, self.hq, self.hd)).astype(np.float32))
        h.put("pos", self.lens)
        self.lens = self.lens + 1
        self.seen += 1
        h.put("lens", self.lens)
        h.put("seen", np.full(self.B, self.seen, np.int32))

    def step(self, keep, recent, attend=True):
        h, c = self.h, self.ctx
        shape = (self.B, self.hkv, self.hd, self.mb, self.nblk)
        if self.int4:
            c.kv_append_int4(h["k"], h["v"], h["kp"], h["vp"], h["table"], h["pos"], self.B, 1, *shape[1:])
        f = c.attn_decode_paged_int4 if self.int4 else c.attn_decode_paged_f16_acc
        f(h["q"], h["kp"], h["vp"], h["table"], h["lens"], h["out"], h["w"], self.B, self.hq, *shape[1:])
        run_evict(c, self.int4, h, *shape, keep, recent, True)

    def append_f16(self):
        h = self.h
        self.ctx.check(self.ctx.L.nx_kv_append_f16(self.ctx.h, h["k"], h["v"], h["kp"], h["vp"], h["table"], h["pos"], self.B, self.hkv,
                                                   self.hd, self.mb, self.nblk), "append")

    def values(self):
        return tokens_of(self.int4, (self.h.get("kp"), self.h.get("vp")), self.hd)

    def state(self):
        return [self.h.get(n) for n in ("kp", "vp", "w", "tags", "lens", "out")]


@pytest.mark.gpu
@pytest.mark.parametrize("int4", [True, False], ids=["int4", "f16"])
def test_a_bounded_cache_over_many_steps(ctx, int4):
    """90 tokens through a cache of at most 32: each step's output is
    attention over the tokens the plain eviction has kept so far."""
    s = Session(ctx, int4)
    keep, recent = 32, 8
    B, hkv = s.B, s.hkv
    kept = [[[] for _ in range(hkv)] for _ in range(B)]   # (k, v) in slot order
    for step in range(90):
        s.inputs()
        if not int4:
            s.append_f16()
        k, v = s.h.a["k"], s.h.a["v"]
        for b in range(B):
            for j in range(hkv):
                if int4:
                    row = [(q.astype(np.float64) - 8) * np.repeat(sc.astype(np.float64), 32) for q, sc in (quantize(k[b, 0, j]), quantize(v[b, 0, j]))]
                else:
                    row = [k[b, 0, j].astype(np.float16).astype(np.float64), v[b, 0, j].astype(np.float16).astype(np.float64)]
                kept[b][j].append(row)
        w0, tags0, lens0 = s.h.get("w"), s.h.get("tags"), s.lens.copy()
        s.step(keep, recent)
        out = s.h.get("out").astype(np.float64)
        w1 = w0.astype(np.float64)
        for b in range(B):
            kk, vv = (np.stack([np.stack([r[i] for r in kept[b][j]]) for j in range(hkv)], 1) for i in range(2))
            want, W, A, e = attention(s.h.a["q"][b], kk, vv)
            tol = 2.0**-11 * (np.abs(want) + A) + (e + 2.0**-19) * A + 2.0**-25
            assert (np.abs(out[b] - want) <= tol).all(), step
            w1[b][:, :lens0[b]] += W
        # which tokens stayed: by tag; their weights as accumulated
        tags, w, lens = s.h.get("tags"), s.h.get("w"), s.h.get("lens")
        assert lens.tolist() == [min(int(n), keep) for n in lens0]
        for b in range(B):
            for j in range(hkv):
                n = lens0[b]
                pos = np.where(tags0[b, j, :n] > 0, tags0[b, j, :n] - 1, s.seen - n + np.arange(n))
                assert sorted(set(pos)) == sorted(pos)
                where = {int(p): i for i, p in enumerate(pos)}
                order = [where[int(t) - 1] for t in tags[b, j, :lens[b]]]
                assert len(set(order)) == lens[b]
                gone = [i for i in range(n) if i not in order]
                for i in gone:  # of those that could go, none had clearly more weight than one that stayed
                    assert pos[i] < s.seen - recent
                    for o in order:
                        assert pos[o] >= s.seen - recent or w1[b, j, o] >= w1[b, j, i] * (1 - 1e-4)
                assert np.abs(w[b, j, :lens[b]] - w1[b, j, order]).max() <= 1e-4 * w1[b, j].max()
                kept[b][j] = [kept[b][j][i] for i in order]
        s.lens = lens.astype(np.int32)
    s.h.free()


@pytest.mark.gpu
@pytest.mark.parametrize("int4", [True, False], ids=["int4", "f16"])
def test_captured_steps_equal_eager_ones(ctx, int4):
    """A token batch that appends, attends and evicts, replayed step after step
    with eager work between, leaves what the same calls leave one by one."""
    a, b = Session(ctx, int4, seed=9), Session(ctx, int4, seed=9)
    scratch = ctx.alloc(4096)
    for step in range(40):
        for s, capture in ((a, False), (b, True)):
            s.inputs()
            if not int4:
                s.append_f16()
            if capture:
                ctx.check(ctx.L.nx_token_begin(ctx.h), "begin")
            s.step(20, 4)
            if capture:
                ctx.check(ctx.L.nx_token_end(ctx.h), "end")
            ctx.check(ctx.L.nx_residual_add(ctx.h, scratch, scratch, scratch, 1024), "eager work")
            s.lens = s.h.get("lens").astype(np.int32)
        for x, y in zip(a.state(), b.state()):
            assert np.array_equal(x.view(np.uint8), y.view(np.uint8)), step
    ctx.free(scratch)
    a.h.free()
    b.h.free()


@pytest.mark.gpu
def test_workspace_grows_inside_a_token_batch():
    """The first calls of a context come under capture: the workspace grows
    there, twice, and the results are those of eager calls."""
    def outputs(capture, reserve):
        with nexus_amd.Context(0) as c:
            if reserve:
                c.check(c.L.nx_reserve_workspace(c.h, 2, 0, 0, 8, 2, 64, 2048), "reserve")
            got = []
            cases = []
            for n, B in ((40, 1), (1500, 2)):
                rng = np.random.default_rng(n)
                mb = -(-n // PAGE)
                kp, vp, _, _, table = cache(rng, True, [n] * B, 2, 64, mb, B * mb, stale=0.0)
                cases.append((Held(c, q=rng.normal(0, 1, (B, 8, 64)).astype(np.float32), kp=kp, vp=vp, table=table,
                                   lens=np.array([n] * B, np.int32), out=np.zeros((B, 8, 64), np.float16),
                                   plain=np.zeros((B, 8, 64), np.float16), w=np.zeros((B, 2, mb * PAGE), np.float32)), B, mb))
            if capture:
                c.check(c.L.nx_token_begin(c.h), "begin")
            for h, B, mb in cases:
                c.attn_decode_paged_int4(h["q"], h["kp"], h["vp"], h["table"], h["lens"], h["plain"], 0, B, 8, 2, 64, mb, B * mb)
                c.attn_decode_paged_int4(h["q"], h["kp"], h["vp"], h["table"], h["lens"], h["out"], h["w"], B, 8, 2, 64, mb, B * mb)
            if capture:
                c.check(c.L.nx_token_end(c.h), "end")
            for h, _, _ in cases:
                got += [h.get("out"), h.get("w"), h.get("plain")]
            return got

    want = outputs(False, False)
    for capture, reserve in ((True, False), (True, True)):
        for x, y in zip(outputs(capture, reserve), want):
            assert np.array_equal(x, y)


@pytest.mark.gpu
def test_two_contexts_at_once(ctx):
    """Calls queued on two contexts' streams without a wait between them."""
    with nexus_amd.Context(0) as other:
        held = []
        for c in (ctx, other):
            rng = np.random.default_rng(77)
            kp, vp, _, _, table = cache(rng, True, [3000, 2000], 4, 128, 188, 376, stale=0.0)
            held.append(Held(c, q=rng.normal(0, 1, (2, 16, 128)).astype(np.float32), kp=kp, vp=vp, table=table,
                             lens=np.array([3000, 2000], np.int32), out=np.zeros((2, 16, 128), np.float16),
                             w=np.zeros((2, 4, 3008), np.float32)))
        for _ in range(20):
            for c, h in zip((ctx, other), held):
                c.attn_decode_paged_int4(h["q"], h["kp"], h["vp"], h["table"], h["lens"], h["out"], h["w"], 2, 16, 4, 128, 188, 376)
        a, b = ([h.get("out"), h.get("w")] for h in held)
        assert all(np.array_equal(x, y) for x, y in zip(a, b)) and abs(a[1].sum() - 20 * 2 * 16) < 0.1
        for h in held:
            h.free()


@pytest.mark.gpu
def test_no_memory_for_the_workspace(poor):
    """Without memory for its workspace a call fails with NX_ERR_OOM, and the
    next one with memory runs."""
    rng = np.random.default_rng(2)
    kp, vp, k64, v64, table = cache(rng, True, [64], 1, 64, 4, 4)
    h = Held(poor, q=rng.normal(0, 1, (1, 4, 64)).astype(np.float32), kp=kp, vp=vp, table=table, lens=np.array([64], np.int32),
             out=np.zeros((1, 4, 64), np.float16))
    poor.limit(64)
    with pytest.raises(nexus_amd.NxError) as e:
        poor.attn_decode_paged_int4(h["q"], h["kp"], h["vp"], h["table"], h["lens"], h["out"], 0, 1, 4, 1, 64, 4, 4)
    assert e.value.code == 3
    poor.limit(0)
    poor.attn_decode_paged_int4(h["q"], h["kp"], h["vp"], h["table"], h["lens"], h["out"], 0, 1, 4, 1, 64, 4, 4)
    want, _, A, e = attention(h.a["q"][0], in_order(k64, table[0], 64), in_order(v64, table[0], 64))
    assert (np.abs(h.get("out")[0] - want) <= 2.0**-11 * (np.abs(want) + A) + (e + 2.0**-19) * A + 2.0**-25).all()
    h.free()


@pytest.mark.gpu
@pytest.mark.parametrize("int4", [True, False], ids=["int4", "f16"])
def test_pages_past_four_gib(ctx, int4):
    """Pages that lie beyond 2^32 bytes of their pools: append (int4),
    attention and eviction reach them and none below."""
    hd, hkv, n, keep = 256, 8, 40, 24
    per = hkv * (9 * hd if int4 else 32 * hd)
    nblk = (1 << 32) // per + 5
    rng = np.random.default_rng(6)
    small = np.arange(3, dtype=np.int32)[None]
    far = small + np.int32(nblk - 3)
    k, v = rng.normal(0, 1, (2, 1, n, hkv, hd)).astype(np.float32)
    kp, vp = (np.ascontiguousarray(x) for x in (to_pages([k[0]], small, 3, 0).astype(np.float16),
                                                to_pages([v[0]], small, 3, 0).astype(np.float16).transpose(0, 1, 3, 2)))
    if int4:
        kp = vp = np.zeros(3 * per, np.uint8)
    q = rng.normal(0, 1, (1, 16, hd)).astype(np.float32)
    w0 = rng.exponential(1, (1, hkv, 48)).astype(np.float32)

    def run(pools, table, blocks):
        h = Held(ctx, table=table, lens=np.array([n], np.int32), seen=np.array([n], np.int32), pos=np.zeros(1, np.int32), q=q, w=w0,
                 out=np.zeros((1, 16, hd), np.float16), tags=np.zeros((1, hkv, 48), np.int32), k=k, v=v)
        h.b.update(kp=pools[0], vp=pools[1])
        if int4:
            ctx.kv_append_int4(h["k"], h["v"], h["kp"], h["vp"], h["table"], h["pos"], 1, n, hkv, hd, 3, blocks)
        f = ctx.attn_decode_paged_int4 if int4 else ctx.attn_decode_paged_f16_acc
        f(h["q"], h["kp"], h["vp"], h["table"], h["lens"], h["out"], h["w"], 1, 16, hkv, hd, 3, blocks)
        run_evict(ctx, int4, h, 1, hkv, hd, 3, blocks, keep, 4, True)
        got = [h.get(x) for x in ("out", "w", "tags", "lens")]
        at = (blocks - 3) * per
        for p in pools:
            x = np.empty(3 * per, np.uint8)
            ctx.check(ctx.L.nx_download(ctx.h, x.ctypes.data, p, at, x.nbytes), "download")
            got.append(x)
            y = np.empty(1 << 16, np.uint8)
            if blocks > 3:
                ctx.check(ctx.L.nx_download(ctx.h, y.ctypes.data, p, at - (1 << 32) if at > 1 << 32 else 0, y.nbytes), "download")
                assert not y.any()
        h.free()
        return got

    want = run([up(ctx, kp), up(ctx, vp)], small, 3)
    pools = [ctx.alloc(nblk * per) for _ in range(2)]
    if not int4:
        for p, x in zip(pools, (kp, vp)):
            ctx.check(ctx.L.nx_upload(ctx.h, p, (nblk - 3) * per, x.ctypes.data, x.nbytes), "upload")
    got = run(pools, far, nblk)
    for x, y in zip(got, want):
        assert np.array_equal(x, y)
