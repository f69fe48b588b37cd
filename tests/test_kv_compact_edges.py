"""The compact KV cache where its arithmetic and its checks have an edge:
precision against 64 bits with next to nothing but roundings in the
tolerance, scores and scales at the ends of their ranges, buffers that may not
be shared, memory that is short."""
import numpy as np
import pytest

import test_kv_compact as kvc
from test_kv_compact import PAGE, Held, attention, call, in_order, numbers, pack, quantize, sizes, to_pages, unpack


def one_sequence(rng, k, v, mb):
    """int4 pools of one sequence's k and v [n][hkv][hd], their values in 64 bits, the table."""
    table = rng.permutation(mb).astype(np.int32)[None]
    kp, vp = pack(*quantize(to_pages([k], table, mb, np.nan)), False), pack(*quantize(to_pages([v], table, mb, np.nan)), True)
    n, hd = k.shape[0], k.shape[2]
    return kp, vp, in_order(unpack(kp, hd, False), table[0], n), in_order(unpack(vp, hd, True), table[0], n), table


def attend(ctx, q, kp, vp, table, n, weights=True, int4=True):
    """out [hq][hd] and weights [hkv][n] of one sequence, weights from 0."""
    (hq, hd), mb = q.shape, table.shape[1]
    hkv = kp.shape[1]
    h = Held(ctx, q=q.astype(np.float32), kp=kp, vp=vp, table=table, lens=np.array([n], np.int32), out=np.zeros((hq, hd), np.float16),
             w=np.zeros((hkv, mb * PAGE), np.float32))
    f = ctx.attn_decode_paged_int4 if int4 else ctx.attn_decode_paged_f16_acc
    f(h["q"], h["kp"], h["vp"], h["table"], h["lens"], h["out"], h["w"] if weights else 0, 1, hq, hkv, hd, mb, kp.shape[0])
    got = h.get("out").astype(np.float64), h.get("w")[:, :n].astype(np.float64)
    h.free()
    return got


# --------------------------------------------------- roundings of the products --
@pytest.mark.gpu
@pytest.mark.parametrize("weights", [True, False], ids=["weights", "plain"])
@pytest.mark.parametrize("hq,hkv,hd,n", [(4, 1, 64, 31), (8, 2, 128, 60), (2, 2, 256, 500), (20, 1, 128, 1000)])
def test_probabilities_keep_more_than_fp16(ctx, hq, hkv, hd, n, weights):
    """Each query looks at one dimension of K alone, with a power of two there,
    so a score is one exact product, its scale and one factor: it is off by
    3 * 2^-24 of itself (the scale's product, the factor, its product) and e is
    2 es + 2^-19 as elsewhere.  p * scale as fp16 hi + lo: 2^-21 of a term, or
    half a step of the smallest numbers, 2^-25 of 2^11 and more, times a code
    of at most 8: n 2^-33 in all.  A single fp16 number would be 2^-12 of a
    term, which the outputs here, far smaller than their terms, do not hide."""
    rng = np.random.default_rng(hd + n)
    mb = -(-n // PAGE)
    kp, vp, k64, v64, table = one_sequence(rng, rng.normal(0, 1, (n, hkv, hd)).astype(np.float32),
                                           rng.normal(0, 1, (n, hkv, hd)).astype(np.float32), mb)
    q = np.zeros((hq, hd))
    q[np.arange(hq), rng.integers(0, hd, hq)] = rng.choice([-2.0, -1.0, 1.0, 2.0], hq) * 8
    out, w = attend(ctx, q, kp, vp, table, n, weights)
    want, W, A, _ = attention(q, k64, v64)
    score = max(np.abs(k64[:, j] @ q[j * (hq // hkv):(j + 1) * (hq // hkv)].T).max() for j in range(hkv)) / np.sqrt(hd)
    e = 6 * 2.0**-24 * score + 2.0**-19
    tol = 2.0**-11 * np.abs(want) + (e + 2.0**-19) * A + n * 2.0**-33 + 2.0**-25
    off = np.abs(out - want)
    assert (off <= tol).all(), f"off by {(off / tol).max():.3g} of the bound"
    if weights:
        assert (np.abs(w - W) <= (e + 2.0**-22) * W + 2.0**-40).all()


@pytest.mark.gpu
@pytest.mark.parametrize("big,first,code,second,score", [
    (224.875, 1.669921875, 1, 3.408203125, 18168), (1614.0, 1.1396484375, 3, 3.6640625, 130397),
    (6976.0, 2.4296875, 6, 5.23828125, 563600)])
def test_largest_probability_times_largest_scale(ctx, big, first, code, second, score):
    """Scores far from 0 (`score`, times log2 e) whose maximum moves by 4 in log2
    and, by the roundings of fp32 there, up to 2^-5 more than a wavefront can see:
    it keeps its reference, and a probability passes 2^15.  With a scale of
    nearly 2 the product passes 65504, fp16's largest number, though every input is far
    from any limit.  All tokens have the same V, so that is the output, whatever
    the weights: the sum of p times V over the sum of p, 2^-19 off, and rounded.  A
    weight comes from its score, rounded, and from L, whose references are: 3
    roundings of numbers of about `score` in an exponent."""
    rng = np.random.default_rng(score)
    hd, n = 64, 512 * 2 * PAGE  # pairs of pages 0..255 hold the first maximum, the others the second
    k, v = np.zeros((n, 1, hd), np.float32), np.zeros((n, 1, hd), np.float32)
    at = np.arange(512) * 2 * PAGE + rng.integers(0, 2 * PAGE, 512)
    k[at, 0, 0] = 7 * big
    k[at[:256], 0, 32], k[at[:256], 0, 33] = code * first, 7 * first
    k[at[256:], 0, 32] = 7 * second
    v[:, 0] = rng.integers(-7, 8, hd) * np.float32(1.9990234375)
    v[:, 0, 5] = v[:, 0, 40] = 7 * 1.9990234375
    q = np.zeros((1, hd))
    q[0, 0], q[0, 32] = 64, 1
    kp, vp, k64, v64, table = one_sequence(rng, k, v, n // PAGE)
    assert np.array_equal(k64, k) and np.array_equal(v64, v)
    assert abs((k64[at[0], 0] @ q[0]) / 8 * np.log2(np.e) - score) < 1
    out, w = attend(ctx, q, kp, vp, table, n)
    assert (np.abs(out[0] - v[0, 0]) <= (2.0**-11 + 2.0**-19) * np.abs(v[0, 0])).all()
    assert abs(w.sum() - 1) <= 3 * 2.0**-24 * score * np.log(2) + 2.0**-19


@pytest.mark.gpu
@pytest.mark.parametrize("hd,n", [(64, 31), (128, 600), (256, 90)])
def test_scales_of_either_sign(ctx, hd, n):
    """The format's value is (code - 8) * scale: negated scales with negated
    codes are the same values, and give the same outputs (the tolerance of
    test_probabilities_keep_more_than_fp16)."""
    rng = np.random.default_rng(hd * n)
    mb = -(-n // PAGE)
    table = rng.permutation(mb).astype(np.int32)[None]
    pools, vals = [], []
    for value in (False, True):
        codes, s = quantize(to_pages([rng.normal(0, 1, (n, 1, hd)).astype(np.float32)], table, mb, 0))
        codes = np.maximum(codes, 1)  # (code 0 has no negative)
        flip = rng.random(s.shape) < 0.5
        codes = np.where(np.repeat(flip, 32, -1), 16 - codes, codes).astype(np.uint8)
        pools.append(pack(codes, np.where(flip, -s, s).astype(np.float16), value))
        vals.append(in_order(unpack(pools[-1], hd, value), table[0], n))
    q = np.zeros((3, hd))
    q[np.arange(3), [3, hd // 2, hd - 1]] = [16, -8, 8]
    out, w = attend(ctx, q, *pools, table, n)
    want, W, A, _ = attention(q, *vals)
    e = 6 * 2.0**-24 * np.abs(vals[0][:, 0] @ q.T).max() / np.sqrt(hd) + 2.0**-19
    tol = 2.0**-11 * np.abs(want) + (e + 2.0**-19) * A + n * 2.0**-33 + 2.0**-25
    off = np.abs(out - want)
    assert (off <= tol).all(), f"off by {(off / tol).max():.3g} of the bound"
    assert (np.abs(w - W) <= (e + 2.0**-22) * W + 2.0**-40).all()


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("value", [np.inf, -np.inf])
def test_an_infinite_key_of_fp16_pages(ctx, hd, value):
    """Whatever the signs of q and of its rounding to fp16, and whether that
    leaves a rest: an infinite element of K makes every row and weight of its
    kv head NaN, and no other head's."""
    rng = np.random.default_rng(hd)
    hq, hkv, n, mb = 16, 2, 50, 4
    table = np.arange(mb, dtype=np.int32)[None]
    k, v = rng.normal(0, 1, (2, n, hkv, hd)).astype(np.float32)
    k[20, 0, 5] = value
    kp, vp = to_pages([k], table, mb, 0).astype(np.float16), to_pages([v], table, mb, 0).astype(np.float16).transpose(0, 1, 3, 2)
    q = rng.normal(0, 1, (hq, hd))
    # of the first kv head's eight: either sign, a rest of either sign and none
    q[:8, 5] = [1, -1, 1 + 2.0**-13, 1 - 2.0**-13, -1 - 2.0**-13, -1 + 2.0**-13, 2, 1e-3]
    out, w = attend(ctx, q, kp, vp, table, n, int4=False)
    assert np.isnan(out[:8]).all() and np.isnan(w[0]).all()
    assert np.isfinite(out[8:]).all() and abs(w[1].sum() - 8) < 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("int4", [True, False], ids=["int4", "f16"])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan, 1e9])
def test_a_query_far_from_the_others(ctx, int4, value):
    """One that is not finite: its row and its kv head's weights are NaN, the other heads' rows are
    theirs, bit for bit: what a head computes goes by its own scores."""
    rng = np.random.default_rng(1)
    hq, hkv, hd, n, mb = 12, 2, 64, 50, 4
    table = np.arange(mb, dtype=np.int32)[None]
    pk, pv = (to_pages([rng.normal(0, 1, (n, hkv, hd)).astype(np.float32)], table, mb, 0) for _ in range(2))
    kp, vp = (pack(*quantize(pk), False), pack(*quantize(pv), True)) if int4 else (pk.astype(np.float16), pv.astype(np.float16).transpose(0, 1, 3, 2))
    q = rng.normal(0, 1, (hq, hd))
    want, _ = attend(ctx, q, kp, vp, table, n, int4=int4)
    q[2, 7] = value
    out, w = attend(ctx, q, kp, vp, table, n, int4=int4)
    if not np.isfinite(value):
        assert np.isnan(out[2]).all() and np.isnan(w[0]).all()
    assert np.isfinite(w[1]).all()
    assert np.array_equal(np.delete(out, 2, 0), np.delete(want, 2, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("value", [np.inf, -np.inf])
def test_an_infinite_scale_of_int4_pages(ctx, hd, value):
    """The same for pages that some other program wrote with an infinite scale."""
    rng = np.random.default_rng(hd)
    n, mb = 50, 4
    table = np.arange(mb, dtype=np.int32)[None]
    k, v = rng.normal(0, 1, (2, n, 2, hd)).astype(np.float32)
    codes, s = quantize(to_pages([k], table, mb, 0))
    s[1, 0, 4, 1] = value  # token 20's second group
    out, w = attend(ctx, rng.normal(0, 1, (16, hd)), pack(codes, s, False), pack(*quantize(to_pages([v], table, mb, 0)), True), table, n)
    assert np.isnan(out[:8]).all() and np.isnan(w[0]).all()
    assert np.isfinite(out[8:]).all() and abs(w[1].sum() - 8) < 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_a_value_that_is_not_finite_costs_the_other_groups_nothing(ctx, hd, value):
    """The heaviest token of every pair of pages holds a NaN or an infinity in its
    first group and zeros elsewhere, the others, of 2^-17 of its weight, ones: they
    are what the other groups' outputs consist of, as exact as without the first
    group (test_probabilities_keep_more_than_fp16; 31 2^-17 is 2^-12)."""
    n = 512
    k, v = np.zeros((n, 1, hd), np.float32), np.ones((n, 1, hd), np.float32)
    k[::2 * PAGE, 0, 0] = 17 * np.log(2) * np.sqrt(hd)
    v[::2 * PAGE, 0] = 0
    v[::2 * PAGE, 0, 3] = value
    kp, vp, k64, v64, table = one_sequence(np.random.default_rng(hd), k, v, n // PAGE)
    q = np.zeros((1, hd))
    q[0, 0] = 1
    out, _ = attend(ctx, q, kp, vp, table, n)
    assert np.isnan(out[:, :32]).all()
    want, W, A, _ = attention(q, k64, v64)
    assert (np.abs(want[:, 32:] * 2**12 - 1) < 0.05).all()
    e = 6 * 2.0**-24 * 17 + 2.0**-19
    assert (np.abs(out - want) <= 2.0**-11 * np.abs(want) + (e + 2.0**-19) * A + n * 2.0**-33 + 2.0**-25)[:, 32:].all()


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("large", [7.5, 60.0, 700.0, 60000.0, 450000.0])
@pytest.mark.parametrize("heavy", [True, False], ids=["heavy", "light"])
def test_a_large_value_costs_the_other_groups_nothing(ctx, hd, large, heavy):
    """The same with large numbers in the first group, of the heaviest tokens or of one
    of the others.  With a scale below 2^(down + 1) the first group's products have 2^-down of
    p's factor, 2^11, so that half of fp16's smallest number, 2^-25, times a
    code of 8 is 2^(down - 33) of a token's term; p is 1 for one token of 32."""
    n = 512
    k, v = np.zeros((n, 1, hd), np.float32), np.ones((n, 1, hd), np.float32)
    k[::2 * PAGE, 0, 0] = 17 * np.log(2) * np.sqrt(hd)
    v[::2 * PAGE, 0] = 0
    v[0 if heavy else 9::2 * PAGE, 0, 3] = large
    kp, vp, k64, v64, table = one_sequence(np.random.default_rng(hd), k, v, n // PAGE)
    q = np.zeros((1, hd))
    q[0, 0] = 1
    out, w = attend(ctx, q, kp, vp, table, n)
    want, W, A, _ = attention(q, k64, v64)
    assert (np.abs(want[:, 32:] * 2**12 - 1) < 0.05).all()
    e = 6 * 2.0**-24 * 17 + 2.0**-19
    tol = 2.0**-11 * np.abs(want) + (e + 2.0**-19) * A + n * 2.0**-33 + 2.0**-25
    tol[:, :32] += 32 * 2.0**(np.floor(np.log2(large / 7)) + 1 - 33)
    past = np.abs(want) >= 65520  # (fp16 has no such number)
    assert (out[past] == np.inf).all()
    off = np.where(past, 0, np.abs(np.where(past, 0, out) - want * ~past))
    assert (off <= tol).all(), f"off by {(off / tol).max():.3g} of the bound"
    assert (np.abs(w - W) <= (e + 2.0**-22) * W + 2.0**-40).all()


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("order", [1, -1, 0], ids=["rising", "falling", "mixed"])
def test_values_of_all_magnitudes(ctx, hd, order):
    """Groups from 10^-3 to 10^4.6, in rising order, in falling and in none: a
    wavefront makes room at many of its pairs.  Beside the roundings of
    test_probabilities_keep_more_than_fp16 a token's term is off by 2^-34 of the
    largest |V| of its group, whatever its weight, and by 2^-28 of its own |V|."""
    rng = np.random.default_rng(hd + order)
    n = 4000
    mb = -(-n // PAGE)
    size = rng.uniform(-3, 4.6, (n, 1, hd // 32))
    size = size if order == 0 else np.sort(size, 0)[::order]
    v = rng.uniform(-1, 1, (n, 1, hd)) * np.repeat(10.0**size, 32, -1)
    kp, vp, k64, v64, table = one_sequence(rng, rng.normal(0, 1, (n, 1, hd)).astype(np.float32), v.astype(np.float32), mb)
    q = np.zeros((8, hd))
    q[np.arange(8), rng.integers(0, hd, 8)] = rng.choice([-2.0, -1.0, 1.0, 2.0], 8) * 8
    out, w = attend(ctx, q, kp, vp, table, n)
    want, W, A, _ = attention(q, k64, v64)
    e = 6 * 2.0**-24 * np.abs(k64[:, 0] @ q.T).max() / np.sqrt(hd) + 2.0**-19
    biggest = np.abs(v64[:, 0]).reshape(n, -1, 32).max((0, 2))  # of each group
    tol = 2.0**-11 * np.abs(want) + (e + 2.0**-19) * A + 2.0**-25 + n * 2.0**-34 * np.repeat(biggest, 32) + 2.0**-28 * np.abs(v64[:, 0]).sum(0)
    past = np.abs(want) >= 65520
    assert not past.any()
    off = np.abs(out - want)
    assert (off <= tol).all(), f"off by {(off / tol).max():.3g} of the bound"
    assert (np.abs(w - W) <= (e + 2.0**-21) * W + 2.0**-40).all()


# ------------------------------------------------------------ shared buffers --
@pytest.mark.parametrize("op", ["nx_kv_evict_f16", "nx_kv_evict_int4"])
def test_eviction_refuses_pools_that_are_another_buffer(op):
    """Both pools are written: neither may be the table, whose checked entries
    the moves go by, nor any other buffer of the call."""
    n = len(sizes(op, kvc.SHAPE))
    ids, big = list(range(1, n + 1)), [1 << 20] * n
    assert call(op, ids, kvc.SHAPE, big)[0] == 6
    for pool in (0, 1):
        for i in range(n):
            if i != pool:
                st, msg = call(op, ids[:pool] + [ids[i]] + ids[pool + 1:], kvc.SHAPE, big)
                assert st == 1 and "another buffer" in msg, (pool, i)
    # outputs in place of inputs that are given twice: the other input would change under the call
    for same, out in (((4, 3), 7), ((6, 5), 8), ((5, 6), 9)):
        twice = list(ids)
        twice[same[0]] = twice[same[1]]
        assert call(op, twice, kvc.SHAPE, big)[0] == 6  # (read alone, that is no harm)
        twice[out] = twice[same[1]]
        assert call(op, twice, kvc.SHAPE, big)[0] == 1, out


# ---------------------------------------------------------------- workspaces --
def test_reserve_refusals():
    L = kvc.nexus_amd.lib()
    L.nx_deviceless.restype = kvc.C.c_void_p
    ctx = kvc.C.c_void_p(L.nx_deviceless((kvc.C.c_size_t * 1)(1), 1))
    good = (2, 16, 4, 128, 2048)
    assert L.nx_reserve_kv_compact(ctx, *good) == 6
    assert L.nx_reserve_kv_compact(None, *good) == 1
    for i in range(5):
        for bad in (0, -1):
            assert L.nx_reserve_kv_compact(ctx, *good[:i], bad, *good[i + 1:]) == 1, i
    for bad in ((65536, 16, 4, 128, 2048), (2, 8194, 4097, 128, 2048), (2, 16, 4, 32, 2048), (2, 16, 4, 128, (1 << 26) + 1)):
        assert L.nx_reserve_kv_compact(ctx, *bad) == 4, bad
    L.nx_destroy(ctx)


@pytest.mark.gpu
def test_reserving_for_the_other_calls_takes_no_more_than_they_need(poor):
    """8 sequences of 32 heads and 131072 positions, in allocations of 64 MiB at
    most: the split records of attention are a few MiB.  (The scores of the
    calls that accumulate weights would be 128 MiB.)"""
    poor.limit(64 << 20)
    poor.check(poor.L.nx_reserve_workspace(poor.h, 8, 0, 0, 32, 8, 128, 131072), "reserve")


@pytest.mark.gpu
def test_reserved_calls_allocate_nothing(poor):
    """After nx_reserve_kv_compact every later allocation may fail: calls of
    fewer sequences, heads, kv heads, dimensions or positions run, whichever are fewer."""
    poor.check(poor.L.nx_reserve_kv_compact(poor.h, 3, 18, 18, 128, 2000), "reserve")
    rng = np.random.default_rng(3)
    cases = []
    for hq, hkv, hd, lens in ((18, 18, 128, [2000, 5, 700]), (18, 1, 128, [1999] * 3), (18, 2, 64, [40]), (9, 1, 128, [2000, 1]), (18, 6, 64, [2000] * 3)):
        for int4 in (True, False):
            B, mb = len(lens), -(-max(lens) // PAGE)
            kp, vp, k64, v64, table = kvc.cache(rng, int4, lens, hkv, hd, mb, B * mb)
            z = np.zeros((B, hkv, mb * PAGE), np.float32)
            cases.append((int4, B, hq, hkv, hd, mb, Held(
                poor, q=rng.normal(0, 1, (B, hq, hd)).astype(np.float32), kp=kp, vp=vp, table=table, lens=np.array(lens, np.int32),
                seen=np.array(lens, np.int32), out=np.zeros((B, hq, hd), np.float16), w=z, tags=z.astype(np.int32)), k64, v64, lens))
    poor.limit(64)
    for int4, B, hq, hkv, hd, mb, h, k64, v64, lens in cases:
        f = poor.attn_decode_paged_int4 if int4 else poor.attn_decode_paged_f16_acc
        f(h["q"], h["kp"], h["vp"], h["table"], h["lens"], h["out"], h["w"], B, hq, hkv, hd, mb, B * mb)
        out = h.get("out").astype(np.float64)
        for b, n in enumerate(lens):
            want, _, A, e = attention(h.a["q"][b], in_order(k64, h.a["table"][b], n), in_order(v64, h.a["table"][b], n))
            assert (np.abs(out[b] - want) <= 2.0**-11 * np.abs(want) + (e + 2.0**-18) * A + 2.0**-25).all()
        keep = max(1, max(lens) // 2)
        kvc.run_evict(poor, int4, h, B, hkv, hd, mb, B * mb, keep, 0, True)
        assert h.get("lens").tolist() == [min(n, keep) for n in lens]
    poor.limit(0)
    for c in cases:
        c[6].free()


@pytest.mark.gpu
@pytest.mark.parametrize("capture", [False, True], ids=["eager", "captured"])
def test_a_workspace_that_cannot_grow(poor, capture):
    """A call without memory fails with NX_ERR_OOM; smaller ones run on, before
    and after it, in the same token batch too."""
    rng = np.random.default_rng(9)
    small, big = [], []
    for n, to in ((100, small), (30000, big)):
        mb = -(-n // PAGE)
        kp, vp, k64, v64, table = kvc.cache(rng, True, [n], 1, 64, mb, mb)
        to += [n, mb, k64, v64, table, Held(poor, q=rng.normal(0, 1, (1, 8, 64)).astype(np.float32), kp=kp, vp=vp, table=table,
                                            lens=np.array([n], np.int32), out=np.zeros((1, 8, 64), np.float16),
                                            w=np.zeros((1, 1, mb * PAGE), np.float32))]

    def attend_to(n, mb, k64, v64, table, h):
        poor.attn_decode_paged_int4(h["q"], h["kp"], h["vp"], h["table"], h["lens"], h["out"], h["w"], 1, 8, 1, 64, mb, mb)

    attend_to(*small)
    poor.limit(1 << 16)
    if capture:
        poor.check(poor.L.nx_token_begin(poor.h), "begin")
    with pytest.raises(kvc.nexus_amd.NxError) as e:
        attend_to(*big)
    assert e.value.code == 3
    attend_to(*small)
    if capture:
        poor.check(poor.L.nx_token_end(poor.h), "end")
    n, mb, k64, v64, table, h = small
    want, W, A, e = attention(h.a["q"][0], in_order(k64, table[0], n), in_order(v64, table[0], n))
    assert (np.abs(h.get("out")[0] - want) <= 2.0**-11 * np.abs(want) + (e + 2.0**-18) * A + 2.0**-25).all()
    assert (np.abs(h.get("w")[0][:, :n] - 2 * W) <= 2 * (e + 2.0**-22) * W).all()
    poor.limit(0)
    attend_to(*big)
    assert abs(big[5].get("w").sum() - 8) < 1e-3
    for x in (small, big):
        x[5].free()


# ------------------------------------------------- a context without a device --
def test_only_the_calls_it_is_for_know_its_buffers():
    """The buffers of a context without a device are numbers, not addresses: every
    call but the compact cache's refuses them, and nothing is allocated for it."""
    L = kvc.nexus_amd.lib()
    L.nx_deviceless.restype = kvc.C.c_void_p
    ctx = kvc.C.c_void_p(L.nx_deviceless((kvc.C.c_size_t * 3)(1 << 20, 1 << 20, 1 << 20), 3))
    host = np.zeros(64, np.float32)
    size, buf = kvc.C.c_size_t(), kvc.C.c_uint64()
    for status in (L.nx_residual_add(ctx, 1, 2, 3, 16), L.nx_download(ctx, host.ctypes.data, 1, 0, 64), L.nx_upload(ctx, 1, 0, host.ctypes.data, 64),
                   L.nx_argmax(ctx, 1, 2, 16, 1), L.nx_free(ctx, 1), L.nx_buffer_size(ctx, 1, kvc.C.byref(size))):
        assert status == 1 and b"unknown buffer" in L.nx_last_error(ctx)
    assert L.nx_alloc(ctx, 64, kvc.C.byref(buf)) == 6 and buf.value == 0
    assert L.nx_token_begin(ctx) == 6 and L.nx_synchronize(ctx) == 6
    assert call("nx_kv_append_int4", [1, 2, 3, 4, 5, 6], kvc.SHAPE)[0] == 6
    L.nx_destroy(ctx)
