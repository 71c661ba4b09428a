"""Paged attention where scores times scale are large, in every way in which a
call is cut, against the definition in 64 bits.  Queries and keys are chosen so
that every score is exact in 32 bits: what is off is the softmax's alone."""
import math

import pytest
import torch

import paged_ref as ref
import test_gpu_paged as paged

pytestmark = pytest.mark.gpu

F64, BF16 = torch.float64, torch.bfloat16


def exact_scores(c, large):
    """Sets c's queries and keys: half the columns are 64 in both, the others -1,
    0 or 1, so scores are whole numbers of `large` near 64^2 d / 2 that differ by
    a few: products and their sums stay below 2^24 of them."""
    g = torch.Generator().manual_seed(c.rows)
    d = c.q.shape[-1]
    for t, times in ((c.q, large), (c.kp, 1.0)):
        small = torch.randint(-1, 2, t.shape, generator=g).to(torch.float32)
        small[..., :d // 2] = 64.0
        t.copy_(torch.where(torch.isnan(t), t, (small * times).to(BF16)))


def bound(c, causal, scale):
    """What the 32-bit form may be off, given exact scores: paged_ref.attend's with
    the exponents' errors as they are here.

    An exponent is (s - max) scale log2(e) with one rounding for each of scale,
    log2(e), their product and the difference's product, 4 * 2^-24 relative: of
    those above -64 (the others' weights, below 2^-64, are less than the sums'
    roundings) 2^-16.  Where the largest is below 1024 its product is rounded by
    itself, at most 2^-14, at the weight and where the maximum is raised or parts
    are added: 3 * 2^-14.  So a weight is off by less than 2^-12."""
    off = 2.0 ** -12
    q, kp = c.q[:c.rows], c.kp
    v = c.vp
    args = (kp, v, c.prefix_table, c.prefix, c.table, c.lens, c.counts, causal, scale)
    o, _ = ref.attend(q, *args)
    # sum w v^2 by the same reference, the values squared
    square, _ = ref.attend(q, kp, v.to(F64) ** 2, *args[2:])
    dev = (square - o * o).clamp(min=0).sqrt() + 1e-9 * square.sqrt()
    keys = c.prefix + max(c.lens)
    tol = (ref.HALF * (1 + 2 * ref.HALF) + 2 * off) * dev \
        + (keys / 8 + 64) * 2.0 ** -24 * square.sqrt()
    return o, tol + ref.HALF * (o.abs() + tol) + 1e-38


@pytest.mark.parametrize("name", list(ref.PLANS))
@pytest.mark.parametrize("scale", [1e-12, 1 / 8, 1.0, 1e4, 1e6, 1e8, 1e12])
def test_scales_to_the_largest(ops, name, scale):
    """The range that a call takes; from 1e4 on a row's largest scores share all
    the weight."""
    c, kw = paged.planned(name)
    exact_scores(c, 1.0)
    paged.check(c.run(ops, True, scale=scale, batch=c.batch(**kw)), bound(c, True, scale))


@pytest.mark.parametrize("name", list(ref.PLANS))
@pytest.mark.parametrize("power", [8, 20, 40, 90])
def test_large_scores(ops, name, power):
    """1 / sqrt(d) with queries of 2^power times as much, both signs of them."""
    c, kw = paged.planned(name)
    exact_scores(c, 2.0 ** power)
    c.q[::2, ::2] *= -1.0
    paged.check(c.run(ops, True, batch=c.batch(**kw)), bound(c, True, 1 / math.sqrt(c.q.shape[-1])))
