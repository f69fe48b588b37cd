"""Operators that keep a KV cache small, as measurable cases: 4-bit pages, attention
over them, attention that accumulates the weight every cached token gets, and
the eviction of the tokens that got least.

Where `own` is false `run` computes them from elementary torch operations,
where it is true through the library.  Shapes are the Llama-3.1-8B-shaped
configuration of the benchmark, heads of 64 as in the tests' tiny model, and
heads of 256.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

PAGE = 16


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # a decode step of a full batch writes one token per sequence: latency
        dict(name="append_step", kind="append", batch=8, tokens=1, start=1000, hkv=8, hd=128, ctx=4096),
        # short prompts of a small model, heads of 64, beginning inside a page
        dict(name="append_ragged", kind="append", batch=3, tokens=333, start=5, hkv=2, hd=64, ctx=512),
        # the cache of a long prompt, written at once
        dict(name="append_prompt", kind="append", batch=1, tokens=8192, start=0, hkv=8, hd=128, ctx=8192),
        # a tiny model's short context: every launch is latency
        dict(name="int4_tiny", kind="int4", batch=1, hq=4, hkv=2, hd=64, ctx=100, weights=False),
        # a full batch with ragged 4K contexts
        dict(name="int4_b8", kind="int4", batch=8, hq=32, hkv=8, hd=128, ctx=4096, weights=False),
        # one long conversation
        dict(name="int4_32k", kind="int4", batch=1, hq=32, hkv=8, hd=128, ctx=32768, weights=False),
        # heads of 256, accumulating weights for a later eviction
        dict(name="int4_wide_acc", kind="int4", batch=2, hq=16, hkv=2, hd=256, ctx=16384, weights=True),
        # one user's chat over fp16 pages, accumulating weights
        dict(name="f16_acc_b1", kind="f16", batch=1, hq=32, hkv=8, hd=128, ctx=4096, weights=True),
        # a full batch of the same
        dict(name="f16_acc_b8", kind="f16", batch=8, hq=32, hkv=8, hd=128, ctx=4096, weights=True),
        # a bounded chat cache of 4096 slots that ran 256 over
        dict(name="evict_f16_b1", kind="evict", pages="f16", batch=1, hkv=8, hd=128, ctx=4352, keep=4096, recent=512),
        # a full batch cut to a quarter of its context
        dict(name="evict_f16_b8", kind="evict", pages="f16", batch=8, hkv=8, hd=128, ctx=8192, keep=2048, recent=256),
        # one long conversation over 4-bit pages cut to an eighth
        dict(name="evict_int4_32k", kind="evict", pages="int4", batch=1, hkv=8, hd=128, ctx=32768, keep=4096, recent=1024),
    ]


def _log(rng, lo, hi):
    """A whole number, its logarithm uniform over [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    kind = rng.choice(["append", "int4", "int4", "f16", "evict", "evict"])
    hkv, hd = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128, 128, 256])
    batch = rng.randint(1, 8)
    unit = batch * hkv * hd
    if kind == "append":
        tokens = 1 if rng.random() < 0.25 else _log(rng, 2, 8192 * 8 * 128 // unit if unit > 1024 else 8192)
        start = rng.choice([0, _log(rng, 1, 4096)])
        return dict(kind=kind, batch=batch, tokens=tokens, start=start, hkv=hkv, hd=hd, ctx=tokens + start + rng.randint(0, 40))
    if kind in ("int4", "f16"):
        return dict(kind=kind, batch=batch, hq=hkv * rng.choice([1, 2, 3, 4, 4, 5, 8, 8, 12]), hkv=hkv, hd=hd,
                    ctx=_log(rng, 1, min(32768, 8 * 4096 * 8 * 128 // unit)), weights=kind == "f16" or rng.random() < 0.5)
    pages = rng.choice(["f16", "int4"])
    ctx = _log(rng, 64, min(32768, (8 * 8192 if pages == "f16" else 32768) * 8 * 128 // unit))
    keep = _log(rng, max(1, ctx // 16), min(ctx, 4096 * 8 * 128 // unit if pages == "int4" else ctx))
    return dict(kind=kind, pages=pages, batch=batch, hkv=hkv, hd=hd, ctx=ctx, keep=keep, recent=rng.randint(0, keep))


def _lens(case):
    """Context lengths of a batch: the longest has ctx positions, the others
    end at different points of the last quarter."""
    c = case["ctx"]
    return [max(1, c - (c * b) // (4 * case["batch"]) - (3 * b) % 16) for b in range(case["batch"])]


def _starts(case):
    """First position that each sequence of an append writes."""
    return [max(0, case["start"] - 3 * b) for b in range(case["batch"])]


def _max_blocks(case):
    return (case["ctx"] + PAGE - 1) // PAGE


# ------------------------------------------------------------------- inputs --
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 17)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _quantize(x):
    """Codes 0..15 and fp16 scales of x [..., hd], groups of 32 along hd: the
    quotient is rounded to 32 bits, then half away from zero."""
    x = x.view(*x.shape[:-1], -1, 32)
    s = (x.abs().amax(-1).double() / 7.0).float().clamp(max=65504.0).half()
    sf = s.double().unsqueeze(-1)
    r = torch.where(sf > 0, x.double() / sf, 0.0).float().double()
    q = torch.where(r < 0, -torch.floor(0.5 - r), torch.floor(r + 0.5)).clamp(-8, 7) + 8
    return q.to(torch.uint8).flatten(-2), s


def _scales_packed(s):
    """fp16 scales [nb][hkv][16][S] as the bytes of a page: four tokens of a group together."""
    nb, hkv, _, S = s.shape
    return s.view(nb, hkv, 4, 4, S).transpose(3, 4).contiguous().view(torch.uint8).view(nb, hkv, -1)


def _nibbles(q):
    return (q[..., 0::2] | (q[..., 1::2] << 4)).flatten(2)


def _pack_k(q, s):
    """K pages [nb][hkv][9 hd] from codes [nb][hkv][16][hd]: dword g S + s of a
    token's row holds dims 32 s + 8 g + j, dim j in nibble j/2 + 4 (j%2)."""
    nb, hkv, _, hd = q.shape
    w = q.view(nb, hkv, PAGE, hd // 32, 4, 4, 2).permute(0, 1, 2, 4, 3, 6, 5).reshape(nb, hkv, PAGE, -1)
    return torch.cat((_nibbles(w), _scales_packed(s)), -1)


def _pack_v(q, s):
    """V pages: dword (16 g + n) hd/32 + i holds tokens 4 g + j of dims
    32 i + 16 e + n, token j in nibble j/2 + 2 e + 4 (j%2)."""
    nb, hkv, _, hd = q.shape
    w = q.view(nb, hkv, 4, 2, 2, hd // 32, 2, PAGE).permute(0, 1, 2, 7, 5, 4, 6, 3).reshape(nb, hkv, 1, -1)
    return torch.cat((_nibbles(w), _scales_packed(s)), -1)


def _inputs(case, seed):
    """The case's inputs as plain tensors, from the seed alone."""
    g, kind = _gen(seed), case["kind"]
    B, hkv, hd, mb = case["batch"], case["hkv"], case["hd"], _max_blocks(case)
    nb, cap = B * mb, mb * PAGE
    t = dict(table=torch.randperm(nb, generator=g, device="cuda").int().view(B, mb))
    if kind == "append":
        # keys have channels of larger magnitude, as after a projection
        loud = torch.where(torch.rand(hd, generator=g, device="cuda") < 0.05, 6.0, 1.0)
        t.update(k=_randn(g, B, case["tokens"], hkv, hd) * loud, v=_randn(g, B, case["tokens"], hkv, hd),
                 start=torch.tensor(_starts(case), dtype=torch.int32, device="cuda"),
                 kpool=torch.zeros(nb, hkv, 9 * hd, dtype=torch.uint8, device="cuda"),
                 vpool=torch.zeros(nb, hkv, 9 * hd, dtype=torch.uint8, device="cuda"),
                 kout=torch.zeros(B, case["tokens"], hkv, hd, device="cuda"),
                 vout=torch.zeros(B, case["tokens"], hkv, hd, device="cuda"))
        return t
    lens = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")
    if case.get("pages", kind) == "int4":
        t.update(kpool=_pack_k(*_quantize(_randn(g, nb, hkv, PAGE, hd))),
                 vpool=_pack_v(*_quantize(_randn(g, nb, hkv, PAGE, hd))))
    else:
        t.update(kpool=_randn(g, nb, hkv, PAGE, hd).half(), vpool=_randn(g, nb, hkv, hd, PAGE).half())
    slot = torch.arange(cap, device="cuda")
    used = slot < lens[:, None, None]
    # weight that tokens gathered so far: a few have most of it, some none at all
    gathered = torch.exp(2.0 * _randn(g, B, hkv, cap)) * (torch.rand(B, hkv, cap, generator=g, device="cuda") > 0.02)
    t.update(lens=lens, weights=torch.where(used, gathered, 0.0))
    if kind != "evict":
        t.update(q=_randn(g, B, case["hq"], hd), out=torch.zeros(B, case["hq"], hd, dtype=torch.float16, device="cuda"))
        return t
    # the cache was cut before: its first three quarters hold tokens from
    # scattered positions, in no order; the rest came since
    placed = (3 * lens.long()) // 4
    seen = lens.long() + lens.long() // 2
    span = int(seen.max())
    order = torch.rand(B, hkv, span, generator=g, device="cuda")
    order = torch.where(torch.arange(span, device="cuda") < (seen - (lens - placed))[:, None, None], order, 2.0)
    pos = torch.nn.functional.pad(order.argsort(-1), (0, max(0, cap - span)))[..., :cap]
    t.update(tags=torch.where(slot < placed[:, None, None], pos + 1, 0).int(), seen=seen.int(),
             lens_out=torch.zeros(B, dtype=torch.int32, device="cuda"), weights_out=torch.zeros(B, hkv, cap, device="cuda"),
             tags_out=torch.zeros(B, hkv, cap, dtype=torch.int32, device="cuda"))
    if case["pages"] == "int4":
        t.update(first=torch.zeros(B, dtype=torch.int32, device="cuda"),
                 kout=torch.zeros(B, case["keep"], hkv, hd, device="cuda"),
                 vout=torch.zeros(B, case["keep"], hkv, hd, device="cuda"))
    return t


# -------------------------------------------------- the library and its handles --
_CTX = None


def _context():
    """The process's one context, as a program keeps it."""
    global _CTX
    if _CTX is None:
        at = str(Path(__file__).resolve().parent.parent / "nexus-inference-engine-_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        import nexus_amd
        _CTX = nexus_amd.Context(0)
    return _CTX


class State:
    """A case's tensors and, for the library, its handles to them, which end
    before the tensors do (free waits for the calls that use them)."""

    def __init__(self, case, tensors):
        self.case, self.t, self.id = case, tensors, {}

    def __del__(self):
        try:
            for b in self.id.values():
                self.ctx.free(b)
        except Exception:
            pass


def prepare(case, seed):
    s = State(case, _inputs(case, seed))
    if own:  # the library works on the tensors' own memory
        s.ctx = _context()
        for n, v in s.t.items():
            s.id[n] = s.ctx.wrap(v.data_ptr(), v.numel() * v.element_size())
        torch.cuda.synchronize()  # its stream is its own: the inputs have to be there
    return s


# -------------------------------------------------------- the library's calls --
# Queued on the context's stream, which torch's know nothing of: a program that
# goes on to read the outputs calls the context's sync() first, and one that
# queues more calls does not.
def _run_own(s):
    c, i, t, ctx = s.case, s.id, s.t, s.ctx
    B, hkv, hd, mb = c["batch"], c["hkv"], c["hd"], _max_blocks(c)
    nb = B * mb
    if c["kind"] == "append":
        ctx.kv_append_int4(i["k"], i["v"], i["kpool"], i["vpool"], i["table"], i["start"], B, c["tokens"], hkv, hd, mb, nb)
        ctx.kv_read_int4(i["kpool"], i["vpool"], i["table"], i["start"], i["kout"], i["vout"], B, c["tokens"], hkv, hd, mb, nb)
        return dict(k=t["kout"], v=t["vout"])
    if c["kind"] == "evict":
        f = ctx.kv_evict_f16 if c["pages"] == "f16" else ctx.kv_evict_int4
        f(i["kpool"], i["vpool"], i["table"], i["lens"], i["seen"], i["weights"], i["tags"], i["lens_out"],
          i["weights_out"], i["tags_out"], B, hkv, hd, mb, nb, c["keep"], c["recent"])
        y = dict(lens=t["lens_out"], weights=t["weights_out"], tags=t["tags_out"])
        if c["pages"] == "f16":
            return dict(y, k=t["kpool"], v=t["vpool"])
        ctx.kv_read_int4(i["kpool"], i["vpool"], i["table"], i["first"], i["kout"], i["vout"], B, c["keep"], hkv, hd, mb, nb)
        return dict(y, k=t["kout"], v=t["vout"])
    w = i["weights"] if c["weights"] else 0
    f = ctx.attn_decode_paged_int4 if c["kind"] == "int4" else ctx.attn_decode_paged_f16_acc
    f(i["q"], i["kpool"], i["vpool"], i["table"], i["lens"], i["out"], w, B, c["hq"], hkv, hd, mb, nb)
    return dict(out=t["out"], weights=t["weights"]) if c["weights"] else dict(out=t["out"])


# ------------------------------------------------------------- the plain forms --
def _unpack(pool, hd):
    """Codes as nibbles [nb][hkv][16 hd] and scales [nb][hkv][4][S][4] of 4-bit pages."""
    nb, hkv, _ = pool.shape
    b = pool[..., :8 * hd]
    q = torch.stack((b & 15, b >> 4), -1).view(nb, hkv, -1)
    return q, pool[..., 8 * hd:].contiguous().view(torch.float16).view(nb, hkv, 4, hd // 32, 4)


def _values_k(pool, hd):
    """K values [nb][hkv][16][hd] that 4-bit pages stand for, 32 bits."""
    q, s = _unpack(pool, hd)
    nb, hkv, S = pool.shape[0], pool.shape[1], hd // 32
    q = q.view(nb, hkv, PAGE, 4, S, 2, 4).permute(0, 1, 2, 4, 3, 6, 5).reshape(nb, hkv, PAGE, S, 32)
    s = s.transpose(3, 4).reshape(nb, hkv, PAGE, S, 1)
    return ((q.float() - 8.0) * s.float()).view(nb, hkv, PAGE, hd)


def _values_v(pool, hd):
    q, s = _unpack(pool, hd)
    nb, hkv, S = pool.shape[0], pool.shape[1], hd // 32
    q = q.view(nb, hkv, 4, 16, S, 2, 2, 2).permute(0, 1, 2, 7, 5, 4, 6, 3).reshape(nb, hkv, PAGE, S, 32)
    s = s.transpose(3, 4).reshape(nb, hkv, PAGE, S, 1)
    return ((q.float() - 8.0) * s.float()).view(nb, hkv, PAGE, hd)


def _in_order(pages, table):
    """[B][hkv][slots][hd] of pages [nb][hkv][16][hd]."""
    B, mb = table.shape
    nb, hkv, _, hd = pages.shape
    return pages[table.long()].transpose(1, 2).reshape(B, hkv, mb * PAGE, hd)


def _cached(c, t):
    """K and V of every slot in 32 bits."""
    if c.get("pages", c["kind"]) == "int4":
        return _in_order(_values_k(t["kpool"], c["hd"]), t["table"]), _in_order(_values_v(t["vpool"], c["hd"]), t["table"])
    return _in_order(t["kpool"], t["table"]).float(), _in_order(t["vpool"].transpose(2, 3), t["table"]).float()


def _plain_append(c, t):
    def values(x):
        q, s = _quantize(x)
        return ((q.view(*s.shape, 32).float() - 8.0) * s.float().unsqueeze(-1)).view(x.shape)

    return dict(k=values(t["k"]), v=values(t["v"]))


def _plain_attention(c, t):
    B, hq, hkv, hd = c["batch"], c["hq"], c["hkv"], c["hd"]
    k, v = _cached(c, t)
    slots = k.shape[2]
    q = t["q"].view(B * hkv, hq // hkv, hd)
    s = torch.bmm(q, k.view(B * hkv, slots, hd).transpose(1, 2).contiguous()).view(B, hkv, -1, slots) / math.sqrt(hd)
    s = s.masked_fill(torch.arange(slots, device="cuda") >= t["lens"][:, None, None, None], -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    out = torch.bmm(p.view(B * hkv, -1, slots), v.reshape(B * hkv, slots, hd)).view(B, hq, hd).half()
    if not c["weights"]:
        return dict(out=out)
    t["weights"] += p.sum(2)
    return dict(out=out, weights=t["weights"])


def _plain_evict(c, t):
    """Which slot's token goes where: rank the slots, then the i-th free slot
    below keep takes the i-th kept token from beyond it."""
    keep, cap = c["keep"], t["weights"].shape[-1]
    slot = torch.arange(cap, device="cuda")
    lens, seen = t["lens"].long()[:, None, None], t["seen"].long()[:, None, None]
    used = slot < lens
    pos = torch.where(t["tags"] > 0, t["tags"].long() - 1, seen - lens + slot)
    rank = torch.where(pos >= seen - c["recent"], math.inf, t["weights"])
    rank = torch.where(used, rank, -1.0).sort(dim=-1, descending=True, stable=True).indices.argsort(-1)
    kept = used & (rank < keep)
    new = lens.clamp(max=keep)
    free, far = (slot < new) & ~kept, kept & (slot >= new)
    far_in_order = (~far).long().sort(dim=-1, stable=True).indices
    nth = (free.long().cumsum(-1) - 1).clamp(min=0)
    src = torch.where(free, far_in_order.gather(-1, nth), slot.expand_as(free))
    stays = slot < new
    y = dict(lens=new.flatten().int(), weights=torch.where(stays, t["weights"].gather(-1, src), 0.0),
             tags=torch.where(stays, pos.gather(-1, src) + 1, 0).int())
    k, v = (_in_order(p, t["table"]) for p in ((t["kpool"], t["vpool"].transpose(2, 3)) if c["pages"] == "f16" else
                                               (_values_k(t["kpool"], c["hd"]), _values_v(t["vpool"], c["hd"]))))
    at = src[..., :keep, None].expand(-1, -1, -1, c["hd"])
    k, v = k.gather(2, at), v.gather(2, at)
    if c["pages"] == "int4":
        return dict(y, k=k.transpose(1, 2).contiguous(), v=v.transpose(1, 2).contiguous())
    s = slot[:keep]
    page, h = t["table"].long()[:, s // PAGE][:, None, :], torch.arange(c["hkv"], device="cuda")[:, None]
    t["kpool"][page, h, s % PAGE] = k
    t["vpool"].transpose(2, 3)[page, h, s % PAGE] = v
    return dict(y, k=t["kpool"], v=t["vpool"])


def run(s):
    if own:
        return _run_own(s)
    c = s.case
    return {"append": _plain_append, "evict": _plain_evict}.get(c["kind"], _plain_attention)(c, s.t)


# --------------------------------------------------------------------- work --
def work(case):
    B, hkv, hd = case["batch"], case["hkv"], case["hd"]
    if case["kind"] == "append":
        n = B * case["tokens"] * hkv
        # both directions: 32-bit rows and 4-bit records, each read and written once
        return dict(bytes=2 * n * (8 * hd + 2 * 9 * hd // 16), flops=2 * n * hd * 4)
    n = sum(_lens(case))
    if case["kind"] in ("int4", "f16"):
        per = 4 * hd if case["kind"] == "f16" else 2 * 9 * hd // 16
        by = n * hkv * (per + (8 if case["weights"] else 0)) + 6 * B * case["hq"] * hd
        return dict(bytes=by, flops=4 * n * case["hq"] * hd)
    # weights and tags read and written; of the kept tokens that part moves
    # which lies beyond the slots that stay (an even spread of the rest)
    moved = sum(min(case["keep"], L) * (L - min(case["keep"], L)) / L for L in _lens(case))
    cap = _max_blocks(case) * PAGE
    by = 8 * hkv * (n + B * cap) + 2 * moved * hkv * (4 * hd if case["pages"] == "f16" else 2 * 9 * hd // 16)
    if case["pages"] == "int4":
        by += B * case["keep"] * hkv * (2 * 9 * hd // 16 + 8 * hd)
    return dict(bytes=by, flops=4 * hkv * n)


# -------------------------------------------------------------------- exact --
def _exact_values(rows):
    """What 4 bits keep of rows [n][hd], in 64 bits: quotients rounded to 32
    bits as the format says, whole steps half away from zero."""
    x = rows.double().reshape(rows.shape[0], -1, 32)
    step = (x.abs().max(-1, keepdim=True).values / 7).float().clamp(max=65504.0).half().double()
    ratio = (x / step.where(step > 0, torch.ones_like(step))).float().double()
    whole = ratio.sign() * (ratio.abs() + 0.5).floor()
    return (whole.clamp(-8, 7) * step).reshape(rows.shape)


def _exact_page(record, hd, value):
    """[16][hd] in 64 bits of one head's 4-bit pages [n][9 hd], index by index."""
    dev = record.device
    tok = torch.arange(PAGE, device=dev)[:, None]
    dim = torch.arange(hd, device=dev)[None, :]
    S = hd // 32
    if value:
        word = (16 * (tok // 4) + dim % 16) * S + dim // 32
        nib = (tok % 4) // 2 + 2 * ((dim // 16) % 2) + 4 * (tok % 2)
    else:
        word = tok * (hd // 8) + ((dim // 8) % 4) * S + dim // 32
        nib = (dim % 8) // 2 + 4 * (dim % 2)
    byte = 4 * word + nib // 2
    code = (record[:, byte.expand(PAGE, hd)].long() >> (4 * (nib % 2))) & 15
    half = record[:, 8 * hd:].contiguous().view(torch.float16)
    return (code - 8).double() * half[:, ((tok // 4) * S + dim // 32) * 4 + tok % 4].double()


def exact(case, seed):
    t, kind = _inputs(case, seed), case["kind"]
    if kind == "evict":
        return None  # tokens move and are chosen: nothing is computed
    B, hkv, hd = case["batch"], case["hkv"], case["hd"]
    if kind == "append":
        return {n: _exact_values(t[n].reshape(-1, hd)).reshape(t[n].shape) for n in ("k", "v")}
    G = case["hq"] // hkv
    out, weights = torch.zeros(B, case["hq"], hd, dtype=torch.float64, device="cuda"), t["weights"].double()
    for b, n in enumerate(_lens(case)):
        pages = t["table"][b].long()
        for h in range(hkv):
            k, v = t["kpool"][pages, h], t["vpool"][pages, h]
            if kind == "int4":
                k, v = _exact_page(k, hd, False), _exact_page(v, hd, True)
            else:
                k, v = k.double(), v.double().transpose(1, 2)
            k, v = k.reshape(-1, hd)[:n], v.reshape(-1, hd)[:n]
            s = (k @ t["q"][b, h * G:(h + 1) * G].double().t().contiguous()) / math.sqrt(hd)
            p = torch.softmax(s, 0)
            out[b, h * G:(h + 1) * G] = p.t().contiguous() @ v
            weights[b, h, :n] += p.sum(1)
    return dict(out=out, weights=weights) if case["weights"] else dict(out=out)
