"""The fp8 tier's calls as a program combines them: outputs written over inputs
where the row or element is the writer's own, a step captured and replayed, a
stream other than the current one, a number of compute units that the chip's
eight dies do not share evenly."""
import pytest
import torch

import fp8_ref as ref
import u15h
from test_gpu_fp8_kinds import SPLIT, run

pytestmark = pytest.mark.gpu

F8, BF16, F32 = torch.float8_e4m3fn, torch.bfloat16, torch.float32


def bf16(seed, *shape, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std + mean).to(BF16).cuda()


def codes(rows, K):
    return (torch.empty(rows, K, dtype=F8, device="cuda"),
            torch.empty(ref.blocks(K), rows, device="cuda"))


def same(a, b):
    view = {1: torch.uint8, 2: torch.int16, 4: torch.int32}
    return all(torch.equal(x.view(view[x.element_size()]), y.view(view[x.element_size()]))
               for x, y in zip(a, b))


@pytest.mark.parametrize("rows,dim", [(1, 16), (5, 4096), (300, 2064), (33, 16384)])
def test_norm_over_its_inputs(ops, rows, dim):
    """y over x without a delta; with one, y over delta, or the sum over it."""
    mu = rows // 2
    x, d = bf16(dim, rows, dim, std=2.0), bf16(dim + 1, rows, dim)
    w = [bf16(i, dim, std=0.1, mean=1.0) for i in (2, 3)]

    def norm(xx, **to):
        q, s = codes(rows, dim)
        ops.mot_rms_norm_fp8(xx, mu, rows - mu, *w, q, s, **to)
        return q, s
    y, r = torch.empty_like(x), torch.empty_like(x)
    plain = (*norm(x, y=y), y)
    over = x.clone()
    assert same((*norm(over, y=over), over), plain)
    added = (*norm(x, delta=d, x_out=r, y=y), r, y)
    r2, d2 = torch.empty_like(x), d.clone()
    assert same((*norm(x, delta=d2, x_out=r2, y=d2), r2, d2), added)
    d2, y2 = d.clone(), torch.empty_like(x)
    assert same((*norm(x, delta=d2, x_out=d2, y=y2), d2, y2), added)


def test_norm_past_f32(ops):
    """A row whose squares add up past f32 is zeros, as u15h_rms_norm's."""
    x = bf16(8, 3, 400)
    x[1, 40] = 3e19
    w = torch.ones(400, dtype=BF16, device="cuda")
    q, s = codes(3, 400)
    y, other = torch.empty_like(x), torch.empty_like(x)
    ops.mot_rms_norm_fp8(x, 3, 0, w, None, q, s, y=y)
    ops.rms_norm(x, w, other)
    assert bool((y[1] == 0).all()) and bool((other[1] == 0).all())
    assert bool((q[1].float() == 0).all()) and bool((s[:, 1] == 2.0 ** -126).all())
    assert bool((y[[0, 2]] != 0).any(1).all())


@pytest.mark.parametrize("rows,inter", [(1, 16), (7, 12288), (1030, 528)])
def test_swiglu_over_its_inputs(ops, rows, inter):
    """h over gate, and over up."""
    gate, up = bf16(rows, rows, inter, std=3.0), bf16(inter, rows, inter)

    def swiglu(g, u, h):
        q, s = codes(rows, inter)
        ops.swiglu_quant_fp8(g, u, q, s, h=h)
        return q, s, h
    want = swiglu(gate, up, torch.empty_like(gate))
    g, u = gate.clone(), up.clone()
    assert same(swiglu(g, up, g), want) and same(swiglu(gate, u, u), want)


class Step:
    """A small MLP step of both groups: residual norm, gate|up, SwiGLU, down."""

    def __init__(self, mu, mg, H=512, I=1280):
        M = mu + mg
        self.size = mu, mg, H, I
        self.x, self.d = bf16(1, M, H), bf16(2, M, H)
        self.w = [bf16(i, H, std=0.1, mean=1.0) for i in (3, 4)]
        self.norm, self.act, self.out = codes(M, H), codes(M, I), codes(M, H)
        self.r = torch.empty_like(self.x)
        new = lambda n: torch.empty(M, n, dtype=BF16, device="cuda")  # noqa: E731
        self.gate_up = [self.weight(10 + 2 * i, I, H, new(I)) for i in range(2)]
        self.down = [self.weight(20, H, I, new(H))]
        torch.cuda.synchronize()

    @staticmethod
    def weight(seed, N, K, y):
        p = dict(y=y)
        for i, e in enumerate(("und", "gen")):
            wq, sw = ref.quant_blocks(bf16(seed + i, N, K, std=0.05).cpu())
            p["wq_" + e], p["sw_" + e] = wq.cuda(), sw.cuda()
        return p

    def run(self, o, stream=None):
        mu, mg, H, I = self.size
        o.mot_rms_norm_fp8(self.x, mu, mg, *self.w, *self.norm, delta=self.d, x_out=self.r,
                           stream=stream)
        o.mot_gemm_fp8(*self.norm, mu, mg, H, self.gate_up, stream=stream)
        gate, up = (p["y"] for p in self.gate_up)
        o.swiglu_quant_fp8(gate, up, *self.act, stream=stream)
        o.mot_gemm_fp8(*self.act, mu, mg, I, self.down, stream=stream)
        o.quant_rows_fp8(self.down[0]["y"], *self.out, stream=stream)

    def outputs(self):
        return (self.r, *self.norm, *[p["y"] for p in self.gate_up], *self.act,
                self.down[0]["y"], *self.out)

    def renew(self, seed):
        self.x.copy_(bf16(seed, *self.x.shape))
        self.d.copy_(bf16(seed + 50, *self.d.shape))


@pytest.mark.parametrize("mu,mg", [(1, 0), (3, 60), (40, 300)])
def test_a_step_captured_and_replayed(mu, mg):
    """Replays on new inputs, each against the same step run eagerly between them
    and by another context."""
    o, other, step = u15h.Ops(0), u15h.Ops(0), Step(mu, mg)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.run(o)
    for seed in range(100, 104):
        step.renew(seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in step.outputs()]
        for t in step.outputs():
            t.view(torch.uint8).fill_(0x55)
        step.run(other)
        torch.cuda.synchronize()
        assert same(got, step.outputs())
    del graph
    o.close()
    other.close()


def test_a_step_on_another_stream():
    o, step = u15h.Ops(0), Step(20, 150)
    step.run(o)
    torch.cuda.synchronize()
    want = [t.clone() for t in step.outputs()]
    for t in step.outputs():
        t.view(torch.uint8).fill_(0x55)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    step.run(o, stream=side)
    side.synchronize()
    assert same(step.outputs(), want)
    o.close()


@pytest.mark.parametrize("cus", ["100", "37"])
def test_units_that_eight_does_not_divide(monkeypatch, cus):
    monkeypatch.setenv("U15H_GEMM_CUS", cus)
    o = u15h.Ops(0)
    for size in SPLIT + [ref.KINDS[12][0], ref.KINDS[16][0]]:
        run(o, size)
    torch.cuda.synchronize()
    o.close()
