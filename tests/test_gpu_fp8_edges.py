"""The fp8 tier's SwiGLU at gates whose sigmoid is below f32's normal range."""
import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu

F8, BF16 = torch.float8_e4m3fn, torch.bfloat16


def swiglu(ops, gate, up, h=False):
    rows, inter = gate.shape
    q = torch.empty(rows, inter, dtype=F8, device="cuda")
    s = torch.empty(ref.blocks(inter), rows, device="cuda")
    out = torch.empty(rows, inter, dtype=BF16, device="cuda") if h else None
    ops.swiglu_quant_fp8(gate.cuda(), up.cuda(), q, s, h=out)
    return q.cpu(), s.cpu(), out.cpu() if h else None


GATES = [-80.0, -86.5, -87.0, -87.5, -88.0, -88.5, -89.0, -90.0, -92.0, -100.0, -103.5, -120.0,
         -150.0, -174.0, -175.0, -190.0, -250.0, -348.0, -350.0, -1000.0, -3.0e38]
UPS = [1.0, -1.0, 2.0 ** -20, 2.0 ** 20, 1e10, -1e30, 3.3e38, -3.3e38]


def test_far_gates(ops):
    """silu(g) u for every far gate and up, each alone in its row, against 64
    bits.

    Off by at most (1.45 |g| + 6) 2^-23 of itself: the exponent g log2 e is
    rounded twice (the constant, the product), which the exponential turns into
    |g| 2^-23, and the exponential, reciprocal and products add 6 units at
    most (four powers of one quarter exponent: 4 and 2.5, of the 0.45 |g| >= 39
    to spare).  Below f32's normal range the last product is off by 2^-149."""
    pairs = [(g, u) for g in GATES for u in UPS]
    gate, up = torch.zeros(len(pairs), 16), torch.zeros(len(pairs), 16)
    for i, (g, u) in enumerate(pairs):
        gate[i, i % 16], up[i, i % 16] = g, u
    gate, up = gate.to(BF16), up.to(BF16)
    q, s, h = swiglu(ops, gate, up, h=True)
    # exp in 64 bits vanishes below -745; of what f32 holds nothing is lost
    v = ref.swiglu(gate, up)
    rel = (gate.double().abs() * 1.45 + 6).clamp(max=1e4) * 2.0 ** -23
    off = (h.double() - v).abs()
    assert bool((off <= v.abs() * (2.0 ** -8 + 1.01 * rel) + 2.0 ** -133).all()), \
        [pairs[i] for i in (off > v.abs() * 2.0 ** -7 + 2.0 ** -133).any(1).nonzero().flatten()]
    least = torch.tensor(2.0 ** -126, dtype=torch.float64)
    want = torch.maximum(v.abs().amax(1) / 448.0, least)
    at = rel.amax(1)
    assert bool(((s[0].double() - want).abs() <= want * (at + 2.0 ** -22)).all())
    ideal = v / want[:, None]
    most = torch.maximum(ideal.abs() * 2.0 ** -4, torch.full_like(ideal, 2.0 ** -10))
    slack = (2 * at[:, None] + 2.0 ** -21) * ideal.abs() + 2.0 ** -22
    off = (q.double() - ideal).abs()
    assert bool((off <= most + slack).all()), \
        [pairs[i] for i in (off > most + slack).any(1).nonzero().flatten()]


def test_far_gates_beside_others(ops):
    """A far gate changes no other value of its row."""
    g = torch.Generator().manual_seed(4)
    gate, up = (torch.randn(9, 400, generator=g) * 3).to(BF16), \
        torch.randn(9, 400, generator=g).to(BF16)
    gate[:, 7::8] = 0
    q, s, h = swiglu(ops, gate, up, h=True)
    far = gate.clone()
    far[:, 7::8], up[:, 7::8] = -88.0, 2.0 ** -40
    q2, s2, h2 = swiglu(ops, far, up, h=True)
    rest = torch.arange(400) % 8 != 7
    assert torch.equal(s, s2)
    assert torch.equal(q[:, rest].view(torch.uint8), q2[:, rest].view(torch.uint8))
    assert torch.equal(h[:, rest].view(torch.int16), h2[:, rest].view(torch.int16))
    assert bool((q2[:, ~rest].float() == 0).all())
