"""Operands of the paged calls that may not overlap: what the Python forms look
at, on the CPU against the elements themselves, and their refusals."""
import random

import pytest
import torch

import u15h

BF16, I32, F64 = torch.bfloat16, torch.int32, torch.float64


def test_rows_that_meet():
    """Every answer against the sets of elements, equal and unequal pitches."""
    rng = random.Random(1)
    met = 0
    for _ in range(20000):
        n, wa, wb = rng.randint(0, 6), rng.randint(1, 9), rng.randint(1, 9)
        pa = wa + rng.randint(0, 12)
        pb = max(pa, wb) if rng.random() < 0.5 else wb + rng.randint(0, 12)
        if pb == max(pa, wb):
            pa = pb
        a, b = rng.randint(0, 70), rng.randint(0, 70)
        one, two = ({at + i * p + j for i in range(n) for j in range(w)}
                    for at, p, w in ((a, pa, wa), (b, pb, wb)))
        want = bool(one & two)
        met += want
        assert u15h._meet(2 * a, 2 * b, n, pa, wa, pb, wb) == want, (n, a, pa, wa, b, pb, wb)
    assert 2000 < met < 18000


@pytest.mark.gpu
def test_overlapping_operands_are_refused(ops):
    """And neighbours in one allocation are not."""
    T, hq, hkv, d = 5, 4, 2, 64
    wide = torch.zeros(T + 1, 2 * hq + 2 * hkv, d, dtype=BF16, device="cuda")
    rows, later = wide[:T], wide[1:]
    q, k, v, o = rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:hq + 2 * hkv], \
        rows[:, hq + 2 * hkv:]
    pool = torch.zeros(2, 2, hkv, 16, d, dtype=BF16, device="cuda")
    kv = u15h.PagedKV(pool[0], pool[1])
    freq, _ = u15h.rope_freqs(d, 1e4)
    rope = u15h.Rope([(freq.cuda(), 0, 0)])
    pos = torch.arange(T, dtype=I32, device="cuda")[None]
    slot = pos[0].contiguous()
    step = u15h.PagedBatch(torch.tensor([T], dtype=I32, device="cuda"),
                           torch.zeros(1, 1, dtype=I32, device="cuda"),
                           q_start=torch.tensor([0, T], dtype=I32, device="cuda"), max_q=T)
    bad = [lambda: ops.paged_attention(kv, step, q, q),
           lambda: ops.paged_attention(kv, step, q, rows[:, 2:hq + 2]),
           lambda: ops.paged_attention(kv, step, q, later[:, :hq]),
           lambda: ops.rope(q, pos, rope, rows[:, 1:hq + 1]),
           lambda: ops.rope(q, pos, rope, later[:, :hq]),
           lambda: ops.paged_append(kv, k, v, slot, pos, rope, q=q, q_out=rows[:, 1:hq + 1]),
           lambda: ops.paged_append(kv, k, v, slot, pos, rope, q=o, q_out=rows[:, hq:2 * hq]),
           lambda: ops.paged_append(kv, k, v, slot, pos, rope, q=o[:, :2], q_out=v),
           lambda: ops.paged_append(kv, k, v, slot, pos, rope, q=o, q_out=later[:, 2:hq + 2])]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError, match="overlap"):
            f()
            pytest.fail(f"refusal {i}")
    ops.paged_append(kv, k, v, slot, pos, rope, q=q, q_out=q)
    ops.paged_append(kv, k, v, slot, pos, rope, q=q, q_out=o)
    ops.paged_attention(kv, step, q, o)
    ops.rope(q, pos, rope, o)
    ops.rope(q, pos, rope, q)
    ops.rope(q.transpose(0, 1), pos[:, :hq].contiguous(), rope, o.transpose(0, 1))
    torch.cuda.synchronize()
