"""The fp8 tier on the GPU: codes and scales of rows, weights, the residual
norm and SwiGLU, the grouped product over them, and a run of them together,
against the definition on the host (tests/fp8_ref.py)."""
import numpy as np
import pytest
import torch

import fp8_ref as ref
import u15h

pytestmark = pytest.mark.gpu

F8, BF16 = torch.float8_e4m3fn, torch.bfloat16


def bf16(seed, *shape, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std + mean).to(BF16)


def guarded(dtype, *shape):
    """A buffer between two guards of 256 bytes, and the whole allocation."""
    size = torch.empty(0, dtype=dtype).element_size()
    n = int(np.prod(shape)) * size
    whole = torch.full((n + 512 + (-n) % 16,), 0x5a, dtype=torch.uint8, device="cuda")
    return whole[256:256 + n].view(dtype).view(*shape), whole


def guards_kept(t, whole):
    n = t.numel() * t.element_size()
    b = whole.cpu()
    return bool((b[:256] == 0x5a).all()) and bool((b[256 + n:] == 0x5a).all())


def same_codes(q, want):
    """Equal bits, any NaN code for a NaN."""
    a, b = q.view(torch.uint8), want.view(torch.uint8)
    nan = lambda t: (t & 0x7f) == 0x7f  # noqa: E731
    return torch.equal(nan(a), nan(b)) and torch.equal(a[~nan(a)], b[~nan(b)])


def same_f32(a, b):
    return torch.equal(a.nan_to_num(nan=-1.0), b.nan_to_num(nan=-1.0))


# ---- quantisers -------------------------------------------------------------

def quant_rows(ops, x):
    rows, K = x.shape
    (q, qa), (s, sa) = guarded(F8, rows, K), guarded(torch.float32, ref.blocks(K), rows)
    ops.quant_rows_fp8(x.cuda(), q, s)
    torch.cuda.synchronize()
    assert guards_kept(q, qa) and guards_kept(s, sa)
    return q.cpu(), s.cpu()


@pytest.mark.parametrize("rows,K", [(1, 16), (1, 4096), (3, 144), (5, 1040), (31, 528), (33, 128),
                                    (129, 12288), (1024, 208), (1057, 640), (2100, 1040)])
def test_rows(ops, rows, K):
    x = bf16(rows + K, rows, K, std=3.0)
    x[:, K // 3] *= 100
    q, s = quant_rows(ops, x)
    wq, ws = ref.quant_rows(x)
    assert same_codes(q, wq) and same_f32(s, ws)


SPECIAL = [0.0, -0.0, 1.0, -448.0, 448.0, 3.3e38, -3.3e38, 1e-38, 9.2e-41, -9.2e-41,
           5.3e-36, 5.2e-36, 2.0 ** -126, float("inf"), -float("inf"), float("nan")]


def test_rows_of_special_values(ops):
    """Zeros, subnormals, the largest values, infinities and NaN, each alone in
    a block and beside ordinary values; e4m3's ties and subnormals."""
    rows = []
    for v in SPECIAL:
        alone, beside = torch.zeros(256), torch.linspace(-2, 2, 256)
        alone[7], beside[140] = v, v
        rows += [alone, beside]
    ties = torch.zeros(256)                  # every code, and every midpoint of two
    codes = torch.arange(0x7f, dtype=torch.uint8).view(F8).float()
    ties[:127] = codes
    ties[127], ties[128] = 448.0, 448.0
    ties[129:255] = (codes[1:] + codes[:-1]) / 2
    rows += [ties, -ties, ties * 2.0 ** -60]
    x = torch.stack(rows).to(BF16)
    assert torch.equal(x[-3].float(), ties)
    q, s = quant_rows(ops, x)
    wq, ws = ref.quant_rows(x)
    assert same_codes(q, wq) and same_f32(s, ws)
    bad = ~torch.isfinite(x.float())
    for b in range(2):                        # a block with a bad value restores to NaN
        cols = slice(b * 128, b * 128 + 128)
        hit = bad[:, cols].any(1)
        back = ref.restore_rows(q, s)[:, cols]
        assert bool(back[hit].isnan().all()) and bool(back[~hit].isfinite().all())


@pytest.mark.parametrize("N,K", [(1, 16), (8, 128), (130, 1040), (128, 4096), (1000, 272),
                                 (257, 129 * 16)])
def test_weights(ops, N, K):
    w = bf16(N * K, N, K, std=0.02)
    if N > 4:
        w[N // 2, K // 2] = 3.0
        w[4] = 0
    (q, qa), (s, sa) = guarded(F8, N, K), guarded(torch.float32, ref.blocks(N), ref.blocks(K))
    ops.quant_blocks_fp8(w.cuda(), q, s)
    torch.cuda.synchronize()
    assert guards_kept(q, qa) and guards_kept(s, sa)
    wq, ws = ref.quant_blocks(w)
    assert same_codes(q.cpu(), wq) and same_f32(s.cpu(), ws)


def test_weights_with_bad_values(ops):
    w = bf16(5, 256, 384)
    w[3, 5], w[200, 300], w[128:, :128] = float("nan"), float("-inf"), 0
    q, s = torch.empty(256, 384, dtype=F8, device="cuda"), torch.empty(2, 3, device="cuda")
    ops.quant_blocks_fp8(w.cuda(), q, s)
    wq, ws = ref.quant_blocks(w)
    assert same_codes(q.cpu(), wq) and same_f32(s.cpu(), ws)


# ---- the residual norm --------------------------------------------------------

# The norm's relative error: the sum of squares is off by at most one rounding
# per addition on the longest path (8 per chunk, at most 4 chunks a lane, then
# 6 + 8 partial sums), halved by the square root; the division, the addition of
# eps, the reciprocal square root (2 units) and two products add 6.
NORM_REL = (46 / 2 + 6) * 2.0 ** -24


@pytest.mark.parametrize("mu,mg,dim", [(1, 0, 4096), (0, 3, 16), (2, 5, 144), (7, 1, 2048),
                                       (3, 30, 2064), (17, 0, 6000), (5, 6, 8192), (4, 4, 8208),
                                       (3, 2, 16384), (40, 1200, 4096)])
@pytest.mark.parametrize("delta,y", [(True, False), (True, True), (False, True), (False, False)])
def test_norm(ops, mu, mg, dim, delta, y):
    M = mu + mg
    x, d = bf16(dim, M, dim, std=2.0), bf16(dim + 1, M, dim, std=0.5) if delta else None
    if M > 2:
        x[2] = 0
        if delta:
            d[2] = 0
    w_und, w_gen = bf16(1, dim, std=0.1, mean=1.0), bf16(2, dim, std=0.1, mean=-1.0)
    (q, qa), (s, sa) = guarded(F8, M, dim), guarded(torch.float32, ref.blocks(dim), M)
    x_out, xa = guarded(BF16, M, dim)
    yt, ya = guarded(BF16, M, dim)
    gx, gd = x.cuda(), d.cuda() if delta else None
    gu, gg = w_und.cuda(), w_gen.cuda()
    ops.mot_rms_norm_fp8(gx, mu, mg, gu if mu else None, gg if mg else None, q, s, delta=gd,
                         x_out=x_out if delta else None, y=yt if y else None, eps=1e-6)
    torch.cuda.synchronize()
    assert all(guards_kept(*p) for p in ((q, qa), (s, sa), (x_out, xa), (yt, ya)))
    assert torch.equal(gx.cpu(), x)
    r, n = ref.norm(x, d, w_und, w_gen, mu, 1e-6)
    if delta:
        assert torch.equal(x_out.cpu().view(torch.int16), r.view(torch.int16))
    ref.check_codes(q.cpu(), s.cpu(), n, NORM_REL)
    if y:
        off = (yt.cpu().double() - n).abs()
        assert bool((off <= n.abs() * (2.0 ** -8 + NORM_REL * 1.01)).all())
    if M > 2:
        assert bool((q[2].float() == 0).all()) and bool((s[:, 2] == 2.0 ** -126).all())
    if delta:                                   # in place: the same bits
        q2, s2 = torch.empty_like(q), torch.empty_like(s)
        ops.mot_rms_norm_fp8(gx, mu, mg, gu, gg, q2, s2, delta=gd, eps=1e-6)
        assert torch.equal(gx.view(torch.int16), x_out.view(torch.int16))
        assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s)


def test_norm_of_bad_rows(ops):
    """A row with a NaN is NaN whole; with an infinity its finite columns are
    0 (1 / sqrt(inf)) and the infinity NaN; other rows stay as they are.  eps 0
    over a row of zeros is 0 * inf."""
    x = bf16(3, 5, 400)
    x[1, 9], x[2, 300], x[3] = float("nan"), float("inf"), 0
    w = torch.ones(400, dtype=BF16)
    q, s = torch.empty(5, 400, dtype=F8, device="cuda"), torch.empty(4, 5, device="cuda")
    ops.mot_rms_norm_fp8(x.cuda(), 5, 0, w.cuda(), None, q, s, eps=0.0)
    q, s = q.cpu(), s.cpu()
    assert bool(s[:, 1].isnan().all()) and bool(s[:, 3].isnan().all())
    assert bool(s[2, 2].isnan()) and bool((s[[0, 1, 3], 2] == 2.0 ** -126).all())
    _, n = ref.norm(x[[0, 4]], None, w, w, 2, 0.0)
    ref.check_codes(q[[0, 4]], s[:, [0, 4]], n, NORM_REL)


# ---- SwiGLU -------------------------------------------------------------------

@pytest.mark.parametrize("rows,inter", [(1, 16), (1, 12288), (7, 1040), (30, 528), (1025, 272),
                                        (2050, 128)])
@pytest.mark.parametrize("h", [False, True])
def test_swiglu(ops, rows, inter, h):
    gate, up = bf16(rows, rows, inter, std=3.0), bf16(inter, rows, inter)
    (q, qa), (s, sa) = guarded(F8, rows, inter), guarded(torch.float32, ref.blocks(inter), rows)
    ht, ha = guarded(BF16, rows, inter)
    ops.swiglu_quant_fp8(gate.cuda(), up.cuda(), q, s, h=ht if h else None)
    torch.cuda.synchronize()
    assert guards_kept(q, qa) and guards_kept(s, sa) and guards_kept(ht, ha)
    v = ref.swiglu(gate, up)
    # the exponent g log2 e is rounded (off by at most |g| 1.45 2^-23, the
    # constant's rounding included), the exponential, the sum, the reciprocal
    # and the products by at most 6 units more
    rel = float((gate.abs().max() * 1.45 + 6) * 2.0 ** -23)
    ref.check_codes(q.cpu(), s.cpu(), v, rel)
    if h:
        off = (ht.cpu().double() - v).abs()
        assert bool((off <= v.abs() * (2.0 ** -8 + 1.01 * rel)).all())


def test_swiglu_of_large_gates(ops):
    """Gates whose exponential overflows or vanishes: silu(-200) is -0, silu(200)
    is 200; a NaN or infinite gate marks its block."""
    gate, up = torch.zeros(4, 128), torch.ones(4, 128)
    gate[0], gate[1], gate[2, 5], gate[3, 5] = -200.0, 200.0, float("nan"), float("inf")
    q, s = torch.empty(4, 128, dtype=F8, device="cuda"), torch.empty(1, 4, device="cuda")
    ops.swiglu_quant_fp8(gate.to(BF16).cuda(), up.to(BF16).cuda(), q, s)
    s = s.cpu()[0]
    assert float(s[0]) == 2.0 ** -126 and bool((q[0].float() == 0).all())
    assert float(s[1]) == float(torch.tensor(200.0) / 448.0) and bool((q[1].float() == 448).all())
    assert bool(s[2].isnan()) and float(s[3]) == float("inf")


# ---- the product ----------------------------------------------------------------

def weight(seed, N, K):
    return ref.quant_blocks(bf16(seed, N, K, std=0.02))


def operands(mu, mg, K, Ns, seed=0):
    M = mu + mg
    x = bf16(seed + 11, M, K)
    x[:, K // 2] *= 16
    if M > 3:
        x[3] = 0
    xq, sx = ref.quant_rows(x)
    return xq, sx, [{e: weight(seed + 7 * i + 3 * (e == "gen"), N, K)
                     for e, m in (("und", mu), ("gen", mg)) if m} for i, N in enumerate(Ns)]


def on_gpu(projs, M, Ns):
    out, wholes = [], []
    for p, N in zip(projs, Ns):
        d = {}
        for e, (wq, sw) in p.items():
            d["wq_" + e], d["sw_" + e] = wq.cuda(), sw.cuda()
        d["y"], whole = guarded(BF16, M, N)
        out.append(d)
        wholes.append(whole)
    return out, wholes


def check_product(got, xq, sx, projs, mu, exact_products=False):
    """exact_products: the operands keep every product in the matrix unit's
    window."""
    for g, p in zip(got, projs):
        y = g["y"].cpu()
        for e, rows in (("und", slice(0, mu)), ("gen", slice(mu, None))):
            if e in p:
                want, adds, window = ref.product(xq[rows], sx[:, rows], *p[e])
                ok = ref.within(y[rows], want, adds if exact_products else adds + window)
                assert bool(ok.all()), (e, (~ok).nonzero()[:8].tolist(), int((~ok).sum()))


def gemm(ops, mu, mg, K, Ns, seed=0):
    xq, sx, projs = operands(mu, mg, K, Ns, seed)
    got, wholes = on_gpu(projs, mu + mg, Ns)
    ops.mot_gemm_fp8(xq.cuda(), sx.cuda(), mu, mg, K, got)
    torch.cuda.synchronize()
    assert all(guards_kept(g["y"], w) for g, w in zip(got, wholes))
    check_product(got, xq, sx, projs, mu)
    return got


SHAPES = [
    (1, 0, 16, (8,)), (1, 0, 128, (16,)), (0, 1, 4096, (64,)), (1, 0, 4096, (512, 128, 128)),
    (2, 0, 272, (1000,)), (15, 1, 1040, (136,)), (16, 0, 12288, (128,)), (17, 0, 640, (264,)),
    (31, 33, 384, (200, 8)), (64, 0, 4096, (256,)), (65, 0, 144, (1032,)), (77, 0, 1040, (1000,)),
    (100, 0, 2048, (72, 520)), (128, 1, 512, (384,)), (129, 0, 1024, (640,)),
    (5, 200, 784, (128, 64, 64, 8)), (255, 257, 256, (264,)), (300, 0, 4096, (1024,)),
    (333, 0, 1152, (392,)), (0, 513, 400, (776,)), (128, 1024, 640, (512, 256)),
    (40, 1100, 128, (2056,)), (1300, 0, 384, (1288,)),
]


@pytest.mark.parametrize("mu,mg,K,Ns", SHAPES)
def test_product(ops, mu, mg, K, Ns):
    gemm(ops, mu, mg, K, Ns)


def narrow_codes(seed, rows, K, exponents):
    """Random codes of magnitude 2^0 .. below 2^exponents, either sign."""
    g = torch.Generator().manual_seed(seed)
    c = torch.randint(0, 8 * exponents, (rows, K), generator=g, dtype=torch.uint8) + (7 << 3)
    c |= torch.randint(0, 2, (rows, K), generator=g, dtype=torch.uint8) << 7
    return c.view(F8)


@pytest.mark.parametrize("mu,mg,K,Ns", SHAPES)
def test_exact_products(ops, mu, mg, K, Ns):
    """Codes of 4 binades against codes of 5: exponent sums spread over at most
    3 + 4 = 7, and with 6 fraction bits every product is a multiple of 2^-13 of
    2^e, so the matrix unit drops nothing and only the additions round.  A
    scale or a chunk of codes in the wrong place does not pass as rounding."""
    xq = narrow_codes(K, mu + mg, K, 4)
    g = torch.Generator().manual_seed(K + 1)
    sx = torch.rand(ref.blocks(K), mu + mg, generator=g) + 0.5
    projs = [{e: (narrow_codes(K + 5 * i + (e == "gen"), N, K, 5),
                  torch.rand(ref.blocks(N), ref.blocks(K), generator=g) + 0.5)
              for e, m in (("und", mu), ("gen", mg)) if m} for i, N in enumerate(Ns)]
    got, wholes = on_gpu(projs, mu + mg, Ns)
    ops.mot_gemm_fp8(xq.cuda(), sx.cuda(), mu, mg, K, got)
    torch.cuda.synchronize()
    assert all(guards_kept(g_["y"], w) for g_, w in zip(got, wholes))
    check_product(got, xq, sx, projs, mu, exact_products=True)


def test_product_repeats_bit_for_bit(ops):
    for args in ((1, 0, 4096, (1024,)), (77, 0, 4096, (1024,)), (333, 0, 4096, (512,)),
                 (128, 600, 1024, (512,))):
        a, b = gemm(ops, *args), gemm(ops, *args)
        for p, q in zip(a, b):
            assert torch.equal(p["y"].view(torch.int16), q["y"].view(torch.int16))


@pytest.mark.parametrize("mu,mg,N", [(3, 0, 256), (50, 30, 256), (200, 300, 384)])
def test_bad_blocks_reach_their_outputs_only(ops, mu, mg, N):
    """An activation block with an infinity turns its row NaN, a weight block
    with a NaN its 128 columns of that expert's rows; nothing else changes."""
    K, M = 512, mu + mg
    xq, sx, projs = operands(mu, mg, K, (N,))
    sx[2, 1] = float("inf")
    projs[0]["und"][1][1, 3] = float("nan")
    got, _ = on_gpu(projs, M, (N,))
    ops.mot_gemm_fp8(xq.cuda(), sx.cuda(), mu, mg, K, got)
    y = got[0]["y"].cpu()
    bad = torch.zeros(M, N, dtype=torch.bool)
    bad[1], bad[:mu, 128:256] = True, True
    assert torch.equal(~y.isfinite(), bad)
    sx[2, 1] = 1.0
    projs[0]["und"][1][1, 3] = 1.0
    for e, rows in (("und", slice(0, mu)), ("gen", slice(mu, None))):
        if e in projs[0]:
            want, adds, window = ref.product(xq[rows], sx[:, rows], *projs[0][e])
            assert bool(ref.within(y[rows], want, adds + window)[~bad[rows]].all())


def test_scales_of_any_size(ops):
    """Scales far from 1 and of either sign; blocks that differ by 2^40."""
    mu, K, N = 70, 640, 256
    xq, sx, projs = operands(mu, 0, K, (N,))
    sx[1] *= 2.0 ** 40
    sx[3] *= -2.0 ** -30
    projs[0]["und"][1][:, 1] *= 2.0 ** -38
    got, _ = on_gpu(projs, mu, (N,))
    ops.mot_gemm_fp8(xq.cuda(), sx.cuda(), mu, 0, K, got)
    check_product(got, xq, sx, projs, mu)


@pytest.mark.parametrize("mu,mg,K,Ns", [(1, 0, 4096, (1024, 256)), (90, 0, 2048, (512,)),
                                        (128, 900, 1024, (512,))])
def test_captured_and_replayed(ops, mu, mg, K, Ns):
    """A captured call replays on new inputs in the same buffers, eager calls of
    the same context between the replays."""
    M = mu + mg
    xq, sx, projs = operands(mu, mg, K, Ns)
    got, _ = on_gpu(projs, M, Ns)
    gx, gs = xq.cuda(), sx.cuda()
    o = u15h.Ops(0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o.mot_gemm_fp8(gx, gs, mu, mg, K, got)
    for seed in (1, 2, 3):
        xq, sx, _ = operands(mu, mg, K, Ns, seed)
        gx.copy_(xq)
        gs.copy_(sx)
        g.replay()
        torch.cuda.synchronize()
        check_product(got, xq, sx, projs, mu)
        gemm(o, 60, 0, 1024, (256,), seed)
    del g
    o.close()


def test_other_stream(ops):
    """Calls on a stream other than the current one, its inputs made there."""
    mu, K, N = 33, 1024, 256
    xq, sx, projs = operands(mu, 0, K, (N,))
    got, _ = on_gpu(projs, mu, (N,))
    torch.cuda.synchronize()
    side, o = torch.cuda.Stream(), u15h.Ops(0)
    with torch.cuda.stream(side):
        gx, gs = xq.cuda(non_blocking=True), sx.cuda(non_blocking=True)
    o.mot_gemm_fp8(gx, gs, mu, 0, K, got, stream=side)
    side.synchronize()
    check_product(got, xq, sx, projs, mu)
    o.close()


def test_nothing_to_do(ops):
    e = lambda dt, *sh: torch.empty(*sh, dtype=dt, device="cuda")  # noqa: E731
    ops.quant_rows_fp8(e(BF16, 0, 256), e(F8, 0, 256), e(torch.float32, 2, 0))
    ops.quant_blocks_fp8(e(BF16, 0, 256), e(F8, 0, 256), e(torch.float32, 0, 2))
    ops.swiglu_quant_fp8(e(BF16, 0, 256), e(BF16, 0, 256), e(F8, 0, 256), e(torch.float32, 2, 0))
    ops.mot_rms_norm_fp8(e(BF16, 0, 256), 0, 0, None, None, e(F8, 0, 256), e(torch.float32, 2, 0))
    ops.mot_gemm_fp8(e(F8, 0, 256), e(torch.float32, 2, 0), 0, 0, 256, [dict(y=e(BF16, 0, 8))])


# ---- refusals: nothing is launched -----------------------------------------------

def test_refusals(ops):
    e = lambda dt, *sh: torch.zeros(*sh, dtype=dt, device="cuda")  # noqa: E731
    f = torch.float32
    x, q, s = e(BF16, 4, 256), e(F8, 4, 256), e(f, 2, 4)
    w = e(BF16, 256)
    for call in (
        lambda: ops.quant_rows_fp8(e(BF16, 4, 24), e(F8, 4, 24), e(f, 1, 4)),        # width % 16
        lambda: ops.quant_blocks_fp8(e(BF16, 4, 24), e(F8, 4, 24), e(f, 1, 1)),
        lambda: ops.swiglu_quant_fp8(e(BF16, 4, 24), e(BF16, 4, 24), e(F8, 4, 24), e(f, 1, 4)),
        lambda: ops.mot_rms_norm_fp8(e(BF16, 1, 16400), 1, 0, e(BF16, 16400), None,
                                     e(F8, 1, 16400), e(f, 129, 1)),                 # dim
        lambda: ops.mot_rms_norm_fp8(x, 4, 0, w, None, q, s, eps=-1.0),
        lambda: ops.mot_rms_norm_fp8(x, 4, 0, w, None, q, s, delta=x.clone(), y=x),  # y is x_out
        lambda: ops.mot_gemm_fp8(e(F8, 2, 24), e(f, 1, 2), 2, 0, 24,
                                 [dict(wq_und=e(F8, 8, 24), sw_und=e(f, 1, 1), y=e(BF16, 2, 8))]),
        lambda: ops.mot_gemm_fp8(e(F8, 2, 32), e(f, 1, 2), 2, 0, 32,
                                 [dict(wq_und=e(F8, 12, 32), sw_und=e(f, 1, 1),
                                       y=e(BF16, 2, 12))]),                          # N % 8
    ):
        with pytest.raises(u15h.U15hError) as err:
            call()
        assert err.value.status == u15h.EINVAL
    one = dict(wq_und=e(F8, 8, 256), sw_und=e(f, 1, 2), y=e(BF16, 4, 8))
    for call, kind in (
        (lambda: ops.quant_rows_fp8(x, q, e(f, 4, 2)), ValueError),                  # row-major s
        (lambda: ops.quant_rows_fp8(x, q.view(torch.uint8), s), TypeError),
        (lambda: ops.quant_rows_fp8(x[:, ::2], q[:, ::2], s), ValueError),
        (lambda: ops.quant_rows_fp8(x.cpu(), q, s), ValueError),
        (lambda: ops.quant_rows_fp8(x[0], q[0], s), ValueError),
        (lambda: ops.mot_rms_norm_fp8(x, 3, 0, w, None, q, s), ValueError),
        (lambda: ops.mot_rms_norm_fp8(x, 4, 0, None, None, q, s), ValueError),
        (lambda: ops.mot_rms_norm_fp8(x, 4, 0, w, None, q, s, x_out=x), ValueError),
        (lambda: ops.mot_gemm_fp8(q, s, 4, 0, 256, []), ValueError),
        (lambda: ops.mot_gemm_fp8(q, s, 4, 0, 256, [one] * 5), ValueError),
        (lambda: ops.mot_gemm_fp8(q, s, 4, 0, 256, [dict(one, sw_und=e(f, 2, 1))]), ValueError),
        (lambda: ops.mot_gemm_fp8(q, s, 2, 2, 256, [one]), (KeyError, ValueError)),
    ):
        with pytest.raises(kind):
            call()


# ---- together ---------------------------------------------------------------------

def test_a_layers_projections_together(ops):
    """A layer's fp8 path as a user runs it, each step fed by the one before:
    residual norm -> q|k|v; a quantised attention output -> o; residual norm ->
    gate|up -> SwiGLU -> down.  Every step is checked against the definition on
    the inputs that it was given."""
    mu, mg, H, KV, I = 20, 150, 512, 128, 1280
    M = mu + mg
    e = lambda dt, *sh: torch.empty(*sh, dtype=dt, device="cuda")  # noqa: E731
    kb = ref.blocks

    def weights(seed, N, K):
        d, h = {}, {}
        for i, g in enumerate(("und", "gen")):
            w = bf16(seed + i, N, K, std=0.05)
            wq, sw = e(F8, N, K), e(torch.float32, kb(N), kb(K))
            ops.quant_blocks_fp8(w.cuda(), wq, sw)
            d["wq_" + g], d["sw_" + g], h[g] = wq, sw, (wq.cpu(), sw.cpu())
        d["y"] = e(BF16, M, N)
        return d, h

    def project(q, s, K, ps):
        ops.mot_gemm_fp8(q, s, mu, mg, K, [d for d, _ in ps])
        check_product([d for d, _ in ps], q.cpu(), s.cpu(), [h for _, h in ps], mu)

    x = bf16(1, M, H, std=2.0)
    gx = x.cuda()
    norms = [[bf16(10 + 2 * i + j, H, std=0.1, mean=1.0) for j in range(2)] for i in range(2)]
    q, s = e(F8, M, H), e(torch.float32, kb(H), M)

    def normed(delta, ws):
        before = gx.cpu()
        ops.mot_rms_norm_fp8(gx, mu, mg, ws[0].cuda(), ws[1].cuda(), q, s, delta=delta)
        r, n = ref.norm(before, None if delta is None else delta.cpu(), *ws, mu, 1e-6)
        assert torch.equal(gx.cpu(), r)
        ref.check_codes(q.cpu(), s.cpu(), n, NORM_REL)

    normed(None, norms[0])
    qkv = [weights(100 + 10 * i, N, H) for i, N in enumerate((H, KV, KV))]
    project(q, s, H, qkv)
    attn = qkv[0][0]["y"]                         # in attention's place
    ops.quant_rows_fp8(attn, q, s)
    wq, ws_ = ref.quant_rows(attn.cpu())
    assert same_codes(q.cpu(), wq) and same_f32(s.cpu(), ws_)
    o = weights(200, H, H)
    project(q, s, H, [o])
    normed(o[0]["y"], norms[1])
    gate_up = [weights(300 + 10 * i, I, H) for i in range(2)]
    project(q, s, H, gate_up)
    gate, up = (d["y"] for d, _ in gate_up)
    hq, hs = e(F8, M, I), e(torch.float32, kb(I), M)
    ops.swiglu_quant_fp8(gate, up, hq, hs)
    rel = float((gate.abs().max() * 1.45 + 6) * 2.0 ** -23)
    ref.check_codes(hq.cpu(), hs.cpu(), ref.swiglu(gate.cpu(), up.cpu()), rel)
    down = weights(400, H, I)
    project(hq, hs, I, [down])
