"""What the matrix unit keeps of a group of 8 neighbouring k whose products
cancel: the documented bound, and that the rounding of y is none."""
import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu

F8, BF16 = torch.float8_e4m3fn, torch.bfloat16


@pytest.mark.parametrize("M", [1, 5, 20, 40, 70, 100, 200, 1100])
def test_groups_that_cancel(ops, M):
    """Row m is zero but for one group of 8, (1, 1, 2^-7, 0..); weight rows 0 and
    1 of each 4 hold (1, -1, 2^-7) and (1, -1, 2^-6) in every group, rows 2 and 3
    the same without the first two.  The sums are 2^-14 and 2^-13 in either
    pair; next to products of 1 the unit keeps 2^-13 of them and drops 2^-14."""
    K, N = 256, 16
    x, w = torch.zeros(M, K), torch.zeros(N, K)
    for m in range(M):
        k = 8 * (m % (K // 8))
        x[m, k:k + 3] = torch.tensor([1.0, 1.0, 2.0 ** -7])
    for n in range(N):
        pair = [1.0, -1.0] if n % 4 < 2 else [0.0, 0.0]
        w[n] = torch.tensor(pair + [2.0 ** -7 if n % 2 == 0 else 2.0 ** -6] + [0.0] * 5).repeat(K // 8)
    xq, wq = x.to(F8), w.to(F8)
    assert torch.equal(xq.float(), x) and torch.equal(wq.float(), w)
    sx, sw = torch.ones(2, M), torch.ones(1, 2)
    y = torch.empty(M, N, dtype=BF16, device="cuda")
    ops.mot_gemm_fp8(xq.cuda(), sx.cuda(), M, 0, K,
                     [dict(wq_und=wq.cuda(), sw_und=sw.cuda(), y=y)])
    y = y.cpu().double()
    want, adds, window = ref.product(xq, sx, wq, sw)
    assert torch.equal(want[0, :4], torch.tensor([2.0 ** -14, 2.0 ** -13] * 2,
                                                 dtype=torch.float64))
    assert bool(ref.within(y, want, adds + window).all())
    kept = torch.tensor([0.0, 2.0 ** -13, 2.0 ** -14, 2.0 ** -13], dtype=torch.float64)
    assert torch.equal(y, kept.repeat(M, N // 4))
