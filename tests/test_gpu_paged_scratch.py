"""Paged attention on a scratch that starts as something else than zeros: no part
or counter that a call has not written itself reaches its output.

u15h_create gets its scratch from hipMalloc, which hands out memory that was
freed with what it holds; so memory of that size is filled and freed before."""
import ctypes

import pytest
import torch

import paged_ref as ref
import test_gpu_paged as paged
import u15h

pytestmark = pytest.mark.gpu

SIZE = (32 << 20) + 4 * 16384               # a context's attention scratch and counters


def dirty(byte):
    """Fills and frees memory; whether memory allocated next holds it."""
    torch.zeros(1, device="cuda")
    with open("/proc/self/maps") as maps:
        path = next(line.split()[-1] for line in maps if "libamdhip64" in line)
    hip = ctypes.CDLL(path)

    def ok(status):
        assert status == 0

    def alloc():
        p = ctypes.c_void_p()
        ok(hip.hipMalloc(ctypes.byref(p), ctypes.c_size_t(SIZE)))
        return p
    p = alloc()
    ok(hip.hipMemset(p, byte, ctypes.c_size_t(SIZE)))
    ok(hip.hipDeviceSynchronize())
    ok(hip.hipFree(p))
    p = alloc()                             # what u15h_create will get
    ends = (ctypes.c_ubyte * 65536)()
    ok(hip.hipMemcpy(ends, ctypes.c_void_p(p.value + SIZE - 65536), ctypes.c_size_t(65536), 2))
    ok(hip.hipFree(p))
    return bytes(ends) == bytes([byte]) * 65536


@pytest.fixture
def filled():
    """A context whose attention scratch starts as a given byte."""
    made = []

    def make(byte):
        if not dirty(byte):
            pytest.skip("freed device memory does not keep what it holds")
        made.append(u15h.Ops(0))
        return made[-1]
    yield make
    torch.cuda.synchronize()
    for o in made:
        o.close()


@pytest.mark.parametrize("name", list(ref.PLANS))
def test_scratch_of_nan(ops, filled, name):
    """Parts and counters that start as NaN (all bits set)."""
    c, kw = paged.planned(name)
    out = c.run(filled(255), True, batch=c.batch(**kw))
    paged.check(out, c.want(True))
    assert torch.equal(paged.bits(out), paged.bits(c.run(ops, True, batch=c.batch(**kw))))


@pytest.mark.parametrize("name", ["joined", "joined_rows", "joined_narrow"])
@pytest.mark.parametrize("eager_first", [False, True])
@pytest.mark.parametrize("byte", [1, 7, 255])
def test_first_joined_call_captured(filled, name, eager_first, byte):
    """A context whose first call that counts is captured, its counters anything but
    0: replayed before any eager call, or after one that clears them too; and a
    second graph of the call, captured before the first has run."""
    o = filled(byte)
    c, kw = paged.planned(name)
    kv, b = u15h.PagedKV(c.kp.cuda(), c.vp.cuda()), c.batch(**kw)
    q = c.q.cuda()
    outs = [torch.zeros_like(q) for _ in range(3)]
    want = c.want(True)
    torch.cuda.synchronize()
    graphs = []
    for out in outs[:2]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            o.paged_attention(kv, b, q, out)
    eager = [2] if eager_first else []
    for which in eager + [1, 0, 0, 2, 1, 2, 2, 0]:
        outs[which].fill_(0)
        if which < 2:
            graphs[which].replay()
        else:
            o.paged_attention(kv, b, q, outs[which])
        torch.cuda.synchronize()
        paged.check(outs[which][:c.rows].cpu(), want)
    assert all(torch.equal(paged.bits(t), paged.bits(outs[2])) for t in outs)
    torch.cuda.synchronize()
    del graphs
