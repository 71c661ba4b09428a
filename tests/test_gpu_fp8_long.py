"""The fp8 tier at its longest K: products whose waves take more than 64 blocks
(the narrow kernel reads its weight scales again there), split and whole tiles,
and the quantisers' widest rows."""
import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu

F8, BF16, F32 = torch.float8_e4m3fn, torch.bfloat16, torch.float32


def ternary(g, rows, K):
    """Codes -1, 0 and 1."""
    return torch.randint(-1, 2, (rows, K), generator=g, device="cuda", dtype=torch.int8).float().to(F8)


def powers(g, *shape):
    """Scales 1, 2 and 4."""
    return torch.exp2(torch.randint(0, 3, shape, generator=g, device="cuda").float())


def restored(q, s, rows):
    """f32 values of codes with a scale for each `rows` x 128."""
    t = s.repeat_interleave(rows, 0)[:q.shape[0]]
    return q.float() * t.repeat_interleave(128, 1)[:, :q.shape[1]]


@pytest.mark.parametrize("size,name,split", ref.LONG, ids=str)
def test_exact_sums(ops, size, name, split):
    """Whole numbers in every step: sums of at most 128 products of +-1 a block,
    times scales of at most 16, over at most 1024 blocks stay within 2^21, which
    f32 holds exactly in any order.  So y is the exact sum rounded once, and a
    scale of the wrong block shows in it."""
    mu, mg, K, Ns = size
    M, kb = mu + mg, ref.blocks(K)
    g = torch.Generator(device="cuda").manual_seed(K + M)
    xq, sx = ternary(g, M, K), powers(g, kb, M)
    projs = []
    for N in Ns:
        p = dict(y=torch.full((M, N), float("nan"), dtype=BF16, device="cuda"))
        for e, m in (("und", mu), ("gen", mg)):
            if m:
                p["wq_" + e], p["sw_" + e] = ternary(g, N, K), powers(g, ref.blocks(N), kb)
        projs.append(p)
    ops.mot_gemm_fp8(xq, sx, mu, mg, K, projs)
    x = restored(xq, sx.t().contiguous(), 1).double()
    for p in projs:
        for e, rows in (("und", slice(0, mu)), ("gen", slice(mu, None))):
            if "wq_" + e not in p:
                continue
            w = restored(p["wq_" + e], p["sw_" + e], 128).double()
            want = x[rows] @ w.t().contiguous()
            assert float(want.abs().max()) > 1000 and torch.equal(want, want.round())
            bad = p["y"][rows] != want.to(F32).to(BF16)
            assert not bool(bad.any()), (e, bad.nonzero()[:8].tolist(), int(bad.sum()))


def test_widest_rows(ops):
    """Rows and weights of 131072 columns, and of 131056, whose last block is
    short."""
    for K in (131072, 131056):
        x = torch.randn(5, K, generator=torch.Generator().manual_seed(K)).to(BF16)
        x[:, K // 3] *= 100
        new = lambda dt, *s: torch.empty(*s, dtype=dt, device="cuda")  # noqa: E731
        q, s = new(F8, 5, K), new(F32, ref.blocks(K), 5)
        ops.quant_rows_fp8(x.cuda(), q, s)
        want_q, want_s = ref.quant_rows(x)
        assert torch.equal(q.cpu().view(torch.uint8), want_q.view(torch.uint8))
        assert torch.equal(s.cpu(), want_s)
        s = new(F32, 1, ref.blocks(K))
        ops.quant_blocks_fp8(x.cuda(), q, s)
        want_q, want_s = ref.quant_blocks(x)
        assert torch.equal(q.cpu().view(torch.uint8), want_q.view(torch.uint8))
        assert torch.equal(s.cpu(), want_s)
        up, s = x.flip(0), new(F32, ref.blocks(K), 5)
        ops.swiglu_quant_fp8(x.cuda(), up.cuda(), q, s)
        # (1.45 |g| + 6 units of 2^-23: the exponent's two roundings, the
        # exponential, the reciprocal and the products)
        rel = float((x.float().abs().max() * 1.45 + 6) * 2.0 ** -23)
        ref.check_codes(q.cpu(), s.cpu(), ref.swiglu(x, up), rel)
