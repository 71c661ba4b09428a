"""The fp8 tier's product on every kernel that it chooses among (whole tiles,
shares of K, several rounds of workgroups, both groups of rows), and the tier's
calls where they meet: two graphs of one context, contexts on two streams at
once, one tensor in several places, sizes whose offsets pass 32 bits."""
import pytest
import torch

import fp8_ref as ref
import u15h

pytestmark = pytest.mark.gpu

F8, BF16, F32 = torch.float8_e4m3fn, torch.bfloat16, torch.float32


def codes(g, rows, K, exponents):
    """Random codes of magnitude 2^0 .. below 2^exponents, either sign."""
    c = torch.randint(0, 8 * exponents, (rows, K), generator=g, dtype=torch.uint8, device="cuda")
    c = (c + (7 << 3)) | (torch.randint(0, 2, (rows, K), generator=g, dtype=torch.uint8,
                                        device="cuda") << 7)
    return c.view(F8)


def operands(mu, mg, K, Ns, seed=0):
    """Codes of 4 binades against codes of 5, whose products the matrix unit
    keeps whole (multiples of 2^-13 of any group's largest binary order), and
    scales of either size."""
    g = torch.Generator(device="cuda").manual_seed(seed * 1000 + K)
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda") + 0.5  # noqa: E731
    xq, sx = codes(g, mu + mg, K, 4), rand(ref.blocks(K), mu + mg)
    projs = []
    for N in Ns:
        p = dict(y=torch.full((mu + mg, N), float("nan"), dtype=BF16, device="cuda"))
        for e, m in (("und", mu), ("gen", mg)):
            if m:
                p["wq_" + e], p["sw_" + e] = codes(g, N, K, 5), rand(ref.blocks(N), ref.blocks(K))
        projs.append(p)
    return xq, sx, projs


def check(xq, sx, projs, mu, rows=None):
    """Every output (or those of `rows`) against 64 bits, off by the additions'
    rounding and y's own at most."""
    M, K = xq.shape
    at = torch.arange(M, device="cuda") if rows is None else torch.as_tensor(rows, device="cuda")
    for p in projs:
        for e, m in (("und", at[at < mu]), ("gen", at[at >= mu])):
            if not len(m):
                continue
            x = restored(xq.view(torch.uint8)[m].view(F8), sx[:, m].t().contiguous(), 1)
            w = restored(p["wq_" + e], p["sw_" + e], 128)
            slack = x.abs() @ w.abs().t().contiguous()
            slack *= (min(K, 128) + 3 + ref.blocks(K)) * 2.0 ** -23
            ok = ref.within(p["y"][m], x @ w.t().contiguous(), slack)
            assert bool(ok.all()), (e, (~ok).nonzero()[:8].tolist(), int((~ok).sum()))


def restored(q, s, rows):
    """f64 values of codes with a scale for each `rows` x 128."""
    t = s.double().repeat_interleave(rows, 0)[:q.shape[0]]
    return q.float().double() * t.repeat_interleave(128, 1)[:, :q.shape[1]]


def run(ops, size, seed=0):
    mu, mg, K, Ns = size
    xq, sx, projs = operands(mu, mg, K, Ns, seed)
    ops.mot_gemm_fp8(xq, sx, mu, mg, K, projs)
    check(xq, sx, projs, mu)


@pytest.mark.parametrize("size,name,split,rounds", ref.KINDS, ids=str)
def test_every_kernel(ops, size, name, split, rounds):
    run(ops, size)


SPLIT = [size for size, _, split, _ in ref.KINDS if split and size[0] + size[1] < 400]


@pytest.mark.parametrize("knob,value", [("U15H_SPLIT", "0"), ("U15H_GEMM_CUS", "192")])
def test_knobs(monkeypatch, knob, value):
    """A context that splits no tiles, one whose rounds leave units free."""
    monkeypatch.setenv(knob, value)
    o = u15h.Ops(0)
    for size in SPLIT + [ref.KINDS[12][0]]:
        run(o, size)
    torch.cuda.synchronize()
    o.close()


def test_two_graphs_of_one_context():
    """Graphs that share the context's workspace, replayed in turns with eager
    calls between, each replay on new inputs."""
    o = u15h.Ops(0)
    cases, graphs = [operands(*size) for size in SPLIT[:2]], []
    for (xq, sx, projs), (mu, mg, K, _) in zip(cases, SPLIT):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o.mot_gemm_fp8(xq, sx, mu, mg, K, projs)
        graphs.append(g)
    for seed in range(1, 5):
        for g, case, (mu, mg, K, Ns) in zip(graphs, cases, SPLIT):
            xq, sx, projs = case
            new = operands(mu, mg, K, Ns, seed)
            xq.view(torch.uint8).copy_(new[0].view(torch.uint8))
            sx.copy_(new[1])
            for p in projs:
                p["y"].fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            check(xq, sx, projs, mu)
            run(o, SPLIT[2], seed)
    torch.cuda.synchronize()
    graphs.clear()
    o.close()


def test_contexts_on_two_streams():
    """Calls of two contexts in flight together, each on its stream."""
    both = [u15h.Ops(0), u15h.Ops(0)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    cases = [[operands(*size, seed) for seed in range(3)] for size in SPLIT[:2]]
    torch.cuda.synchronize()
    for turn in range(3):
        for o, st, case, (mu, mg, K, _) in zip(both, streams, cases, SPLIT):
            xq, sx, projs = case[turn]
            o.mot_gemm_fp8(xq, sx, mu, mg, K, projs, stream=st)
    torch.cuda.synchronize()
    for case, (mu, *_) in zip(cases, SPLIT):
        for xq, sx, projs in case:
            check(xq, sx, projs, mu)
    for o in both:
        o.close()


def test_one_weight_in_several_places(ops):
    """Both groups on one expert's weights, and a projection listed twice."""
    mu, mg, K, N = 60, 90, 1168, 264
    xq, sx, (p,) = operands(mu, mg, K, (N,))
    p["wq_gen"], p["sw_gen"] = p["wq_und"], p["sw_und"]
    again = dict(p, y=torch.zeros_like(p["y"]))
    ops.mot_gemm_fp8(xq, sx, mu, mg, K, [p, again])
    check(xq, sx, [p], mu)
    assert torch.equal(p["y"].view(torch.int16), again["y"].view(torch.int16))


@pytest.mark.parametrize("M", [1, 40, 200])
def test_operands_inside_larger_buffers(ops, M):
    """Views whose rows start 16 bytes, not more, into an allocation; what lies
    around the output stays."""
    K, N = 528, 136
    xq, sx, (p,) = operands(M, 0, K, (N,))

    def inside(t, pad):
        whole = torch.full((t.numel() + 2 * pad,), 3, dtype=torch.uint8, device="cuda") \
            if t.dtype is F8 else torch.full((t.numel() + 2 * pad,), 3.0, dtype=t.dtype,
                                             device="cuda")
        part = whole[pad:pad + t.numel()]
        part.copy_(t.reshape(-1).view(torch.uint8) if t.dtype is F8 else t.reshape(-1))
        return part.view(t.dtype).view(t.shape), whole
    xq, sx = inside(xq, 16)[0], inside(sx, 4)[0]
    for name, pad in (("wq_und", 16), ("sw_und", 4)):
        p[name] = inside(p[name], pad)[0]
    p["y"], whole = inside(p["y"], 8)
    ops.mot_gemm_fp8(xq, sx, M, 0, K, [p])
    check(xq, sx, [p], M)
    assert bool((whole[:8] == 3).all()) and bool((whole[-8:] == 3).all())


# ---- offsets past 32 bits -----------------------------------------------------------

def test_rows_past_32_bits(ops):
    """4.3 GB of bf16 rows: the last ones' codes are their own."""
    rows, K = 175000, 12288
    x = torch.zeros(rows, K, dtype=BF16, device="cuda")
    tail = (torch.randn(9, K, generator=torch.Generator().manual_seed(1)) * 3).to(BF16)
    x[-9:] = tail.cuda()
    q, s = torch.empty(rows, K, dtype=F8, device="cuda"), torch.empty(96, rows, device="cuda")
    ops.quant_rows_fp8(x, q, s)
    want_q, want_s = ref.quant_rows(tail)
    assert torch.equal(q[-9:].cpu().view(torch.uint8), want_q.view(torch.uint8))
    assert torch.equal(s[:, -9:].cpu(), want_s)
    assert not bool(q[:1000].view(torch.uint8).any()) and bool((s[:, :1000] == 2.0 ** -126).all())
    up = torch.ones(rows, K, dtype=BF16, device="cuda")
    ops.swiglu_quant_fp8(x, up, q, s)
    rel = float((tail.float().abs().max() * 1.45 + 6) * 2.0 ** -23)
    ref.check_codes(q[-9:].cpu(), s[:, -9:].cpu().contiguous(),
                    ref.swiglu(tail, torch.ones_like(tail)), rel)


def test_norm_past_32_bits(ops):
    rows, dim = 280000, 8208
    x = torch.zeros(rows, dim, dtype=BF16, device="cuda")
    tail = torch.randn(9, dim, generator=torch.Generator().manual_seed(2)).to(BF16)
    x[-9:] = tail.cuda()
    w = torch.ones(dim, dtype=BF16, device="cuda")
    q, s = torch.empty(rows, dim, dtype=F8, device="cuda"), torch.empty(65, rows, device="cuda")
    ops.mot_rms_norm_fp8(x, 5, rows - 5, w, w, q, s)
    _, n = ref.norm(tail, None, w.cpu(), w.cpu(), 0, 1e-6)
    # 8 additions a chunk, 4 chunks a lane, then 6 + 8, halved by the root; 6 roundings more
    ref.check_codes(q[-9:].cpu(), s[:, -9:].cpu().contiguous(), n, (46 / 2 + 6) * 2.0 ** -24)
    assert not bool(q[:1000].view(torch.uint8).any())


def test_product_past_32_bits(ops):
    """4.9 GB of outputs from 300000 rows, few, odd and last ones checked."""
    mu, mg, K, N = 7, 299993, 272, 8200
    xq, sx, projs = operands(mu, mg, K, (N,))
    ops.mot_gemm_fp8(xq, sx, mu, mg, K, projs)
    check(xq, sx, projs, mu, rows=[0, 6, 7, 8, 262143, 262144, 262150, 299998, 299999])
    assert not bool(projs[0]["y"].isnan().any())


def test_most_rows(ops):
    """2^22 rows, the most that a call takes: the last ones are as they are
    alone."""
    rows, dim = 1 << 22, 4112
    x = torch.zeros(rows, dim, dtype=BF16, device="cuda")
    tail = torch.randn(5, dim, generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
    x[-5:] = tail
    w = torch.ones(dim, dtype=BF16, device="cuda")
    q, s = torch.empty(rows, dim, dtype=F8, device="cuda"), torch.empty(33, rows, device="cuda")
    q5, s5 = torch.empty(5, dim, dtype=F8, device="cuda"), torch.empty(33, 5, device="cuda")
    for call in (lambda a, m, qq, ss: ops.mot_rms_norm_fp8(a, 0, m, None, w, qq, ss),
                 lambda a, m, qq, ss: ops.quant_rows_fp8(a, qq, ss),
                 lambda a, m, qq, ss: ops.swiglu_quant_fp8(a, a, qq, ss)):
        q.view(torch.uint8).fill_(0x55)
        call(x, rows, q, s)
        call(tail, 5, q5, s5)
        assert torch.equal(q[-5:].view(torch.uint8), q5.view(torch.uint8))
        assert torch.equal(s[:, -5:], s5)
        assert not bool(q[rows // 2:rows // 2 + 4096].view(torch.uint8).any())
        assert not bool(q[:4096].view(torch.uint8).any())
    del x, q, s
    K, N = 144, 8
    xq, sx, projs = operands(0, rows, K, (N,))
    ops.mot_gemm_fp8(xq, sx, 0, rows, K, projs)
    check(xq, sx, projs, 0, rows=[0, 1, 63, 64, 1 << 21, rows - 65, rows - 64, rows - 1])
    assert not bool(projs[0]["y"].isnan().any())
