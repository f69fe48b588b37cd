"""nx_wrap: buffers of device memory that the caller owns.  What is refused, on
the CPU; on the GPU that calls work in the memory itself, inside its bounds,
and that the handle's end leaves it alone."""
import ctypes as C

import numpy as np
import pytest

import nexus_amd


def deviceless(*sizes):
    """A context whose buffers 1 .. n are numbers alone (it refuses nothing: no device, 6)."""
    L = nexus_amd.lib()
    L.nx_deviceless.restype = C.c_void_p
    return L, C.c_void_p(L.nx_deviceless((C.c_size_t * len(sizes))(*sizes), len(sizes)))


def test_refusals():
    L, ctx = deviceless()
    b = C.c_uint64(77)
    assert L.nx_wrap(ctx, 4096, 64, C.byref(b)) == 6  # the call itself is in order
    assert L.nx_wrap(None, 4096, 64, C.byref(b)) == 1
    assert L.nx_wrap(ctx, 4096, 64, None) == 1
    for ptr, n in ((None, 64), (4096, 0), (4096, (1 << 64) - 4096), (4104, 64), (4097, 64)):
        assert L.nx_wrap(ctx, ptr, n, C.byref(b)) == 1, (ptr, n)
    assert b.value == 77
    L.nx_destroy(ctx)


@pytest.fixture
def owner(ctx):
    """A context that stands for the memory's owner, and one that borrows."""
    with nexus_amd.Context(0) as other:
        yield ctx, other


@pytest.mark.gpu
def test_calls_work_in_the_callers_memory(owner):
    own, ctx = owner
    n = 1000
    a, b = (np.random.default_rng(i).normal(0, 1, n).astype(np.float32) for i in range(2))
    whole = own.upload(np.concatenate([a, b, np.full(2 * n, 7, np.float32)]))
    own.sync()
    ids = [ctx.wrap(whole + 4 * n * i, 4 * n) for i in range(3)]  # 4000 bytes each: 16-byte aligned parts of one allocation
    ctx.check(ctx.L.nx_residual_add(ctx.h, ids[0], ids[1], ids[2], n), "add")
    with pytest.raises(nexus_amd.NxError):  # a handle has the bytes it was given
        ctx.check(ctx.L.nx_residual_add(ctx.h, ids[0], ids[1], ids[2], n + 1), "add")
    assert np.array_equal(ctx.download(ids[2], n, np.float32), a + b)
    for i in ids:
        ctx.free(i)
    with pytest.raises(nexus_amd.NxError):
        ctx.free(ids[0])
    ids = [ctx.wrap(whole, 16 * n)]  # free again to be wrapped, as a whole
    got = own.download(whole, (4, n), np.float32)
    assert np.array_equal(got, np.stack([a, b, a + b, np.full(n, 7, np.float32)]))
    ctx.free(ids[0])
    own.free(whole)


@pytest.mark.gpu
def test_the_contexts_end_leaves_the_memory(ctx):
    x = ctx.upload(np.arange(64, dtype=np.float32))
    with nexus_amd.Context(0) as other:
        other.wrap(x, 256)
    assert np.array_equal(ctx.download(x, 64, np.float32), np.arange(64))
    ctx.free(x)


@pytest.mark.gpu
def test_what_is_no_memory_for_it(owner):
    """Host memory, bytes past an allocation's end, memory that is a buffer already."""
    own, ctx = owner
    host = np.zeros(1 << 16, np.uint8)
    mine, theirs = ctx.alloc(1 << 16), own.alloc(1 << 16)
    own.sync()
    bad = [(-(-host.ctypes.data // 16) * 16, 64), (theirs + (1 << 15), 1 << 40), (mine, 64), (mine + 64, 64), (1 << 62, 64)]
    first = ctx.wrap(theirs + 1024, 1024)
    bad += [(theirs + 1024, 1024), (theirs, 2048), (theirs + 2032, 16), (theirs + 1040, 16), (theirs, 1 << 16)]
    for ptr, n in bad:
        with pytest.raises(nexus_amd.NxError) as e:
            ctx.wrap(ptr, n)
        assert e.value.code == 1, (ptr, n)
    ok = [ctx.wrap(theirs, 1024), ctx.wrap(theirs + 2048, 1024)]  # its neighbours
    for b in [first, *ok, mine]:
        ctx.free(b)
    own.free(theirs)
    ctx.sync()


@pytest.mark.gpu
def test_not_inside_a_token_batch(owner):
    own, ctx = owner
    x, y = own.alloc(1024), ctx.alloc(1024)
    ctx.check(ctx.L.nx_token_begin(ctx.h), "begin")
    ctx.check(ctx.L.nx_residual_add(ctx.h, y, y, y, 256), "add")
    with pytest.raises(nexus_amd.NxError) as e:
        ctx.wrap(x, 1024)
    assert e.value.code == 5
    ctx.check(ctx.L.nx_token_end(ctx.h), "end")
    own.free(x)
