"""Rotary positions, the paged cache and attention behind a shared prefix on
the host, in 64 bits, with the bounds of their 32- and 16-bit forms."""
import math

import torch

F64, BF16 = torch.float64, torch.bfloat16
HALF = 2.0 ** -8                 # bf16: half a step, relative


def turn(x, pos, parts, neighbours=False, scale=1.0, inverse=False):
    """x [tokens][heads][d] turned in f64, and what its bf16 form may be off.

    The bound: half a step of bf16; and for each pair 2^-19 * (|a| + |b|): the
    angle's turn rounded to 32 bits (2^-26 turns, 2.4e-8 * 2 pi), positions to
    2^31 times frequencies of 53 bits (7e-7), cosine and sine to 4 units (2.4e-7)
    and three roundings of 2^-24, together under 2^-19.7."""
    x = x.to(F64)
    y, off = x.clone(), torch.zeros_like(x)
    for freq, start, axis in parts:
        h = freq.numel()
        angle = pos[axis].to(F64)[:, None] * freq.to(F64)
        c, s = (torch.cos(angle) * scale)[:, None], (torch.sin(angle) * scale)[:, None]
        s = -s if inverse else s
        if neighbours:
            i = slice(start, start + 2 * h, 2)
            j = slice(start + 1, start + 2 * h, 2)
        else:
            i, j = slice(start, start + h), slice(start + h, start + 2 * h)
        a, b = x[..., i], x[..., j]
        y[..., i], y[..., j] = a * c - b * s, b * c + a * s
        slack = 2.0 ** -19 * (a.abs() + b.abs()) * abs(scale)
        off[..., i], off[..., j] = slack, slack
    return y, off + HALF * (y.abs() + off) * (off > 0) + 1e-38 * (off > 0)


def gather(pool, table, n):
    """Keys [n][kv_heads][d] of a table's pages and which of them are there: a
    page number outside the pool has none."""
    pages, hkv, page, d = pool.shape
    keys = torch.zeros(n, hkv, d, dtype=F64)
    there = torch.zeros(n, dtype=torch.bool)
    for i in range(-(-n // page)):
        p, k = int(table[i]), min(page, n - i * page)
        if 0 <= p < pages:
            keys[i * page:i * page + k] = pool[p, :, :k].transpose(0, 1).to(F64)
            there[i * page:i * page + k] = True
    return keys, there


def attend(q, kp, vp, prefix_table, prefix_len, tables, lens, counts, causal, scale=0.0):
    """(out, bound) f64 [rows of all sequences][hq][d].

    With w a row's weights, s its scores and o its output, the 32-bit form rounds
      - each weight to bf16, in numerator and sum alike: 2^-8 relative, so o
        moves by at most 2^-8 sum w |v - o| <= 2^-8 dev(v) by Cauchy-Schwarz,
        over a sum that is at most 2^-8 smaller;
      - scores to (d + 4) 2^-24 sum |q k| scale, the exponent's argument and
        the exponential to 2^-21 (arguments to 2^5 matter): weights by as much;
      - sums of n terms to (n / 8 + 64) 2^-24 of sum w |v| <= rms(v): the matrix
        unit adds groups of 32 keys, the waves' shares and splits few more;
      - o to bf16, half a step."""
    d = q.shape[-1]
    scale = scale or 1.0 / math.sqrt(d)
    hq, hkv = q.shape[1], kp.shape[1]
    out, bound, at = [], [], 0
    pk, pt = gather(kp, prefix_table, prefix_len)
    pv, _ = gather(vp, prefix_table, prefix_len)
    for table, n, count in zip(tables, lens, counts):
        ok, ot = gather(kp, table, n)
        ov, _ = gather(vp, table, n)
        k = torch.cat([pk, ok]).repeat_interleave(hq // hkv, 1).permute(1, 0, 2)   # [hq][n][d]
        v = torch.cat([pv, ov]).repeat_interleave(hq // hkv, 1).permute(1, 0, 2)
        sees = torch.cat([pt, ot])[None].repeat(count, 1)
        if causal:
            last = prefix_len + n - count + torch.arange(count)[:, None]
            sees &= torch.arange(prefix_len + n)[None] <= torch.clamp(last, min=prefix_len - 1)
        qs = q[at:at + count].to(F64).transpose(0, 1)                              # [hq][c][d]
        at += count
        s = (qs @ k.transpose(1, 2) * scale).masked_fill(~sees, -math.inf)
        size = (qs.abs() @ k.abs().transpose(1, 2) * scale).masked_fill(~sees, 0.0)
        size = size.amax(-1, keepdim=True) if s.shape[-1] else torch.zeros(hq, count, 1, dtype=F64)
        if s.shape[-1] == 0:
            o = torch.zeros(hq, count, d, dtype=F64)
            tol = torch.zeros_like(o)
        else:
            top = s.amax(-1, keepdim=True).clamp(min=-1e300)
            e = torch.exp(s - top)
            total = e.sum(-1, keepdim=True)
            w = torch.where(total > 0, e / total, torch.zeros_like(e))
            o = w @ v
            square = w @ (v * v)
            dev = (square - o * o).clamp(min=0).sqrt() + 1e-9 * square.sqrt()
            ds = (d + 4) * 2.0 ** -24 * size + 2.0 ** -21
            tol = (HALF * (1 + 2 * HALF) + 2 * ds) * dev \
                + (s.shape[-1] / 8 + 64) * 2.0 ** -24 * square.sqrt()
            tol = tol + HALF * (o.abs() + tol) + 1e-38
        out.append(o.transpose(0, 1))
        bound.append(tol.transpose(0, 1))
    return torch.cat(out), torch.cat(bound)


# Batches for every way in which a call is cut: (own keys, queries, prefix, heads,
# more of Case, the plan that tests/paged_host.cc prints for 256 compute units).
PLANS = {
    "whole": ([77, 5], [1, 1], 50, (32, 8, 128), {}, r"parts=1 .*none s=1:1x.* t=0:.* nr=1"),
    "joined": ([1800], [1], 0, (8, 2, 128), {}, r"none s=1:(?!1x).* t=0.* nr=1 .*joins=1"),
    "joined_rows": ([1800, 40], [9, 3], 0, (10, 2, 64), {}, r"none s=1:(?!1x).* t=0.* nr=2 .*joins=1"),
    "joined_narrow": ([700], [2], 100, (6, 1, 32), {}, r"none s=1:(?!1x).* nr=1 .*joins=1"),
    "second_kernel": ([3000, 2500], [1, 1], 0, (8, 8, 128), dict(max_kv=50000, wide=3125),
                      r"none s=1:(?!1x).* t=0.*joins=0"),
    "prefix_streamed": ([30, 1, 500], [1, 1, 1], 2000, (6, 2, 128), {}, r"stream s=1:.* nr=1"),
    "prefix_streamed_wide": ([30, 1, 500, 7] * 2, [1] * 8, 600, (8, 2, 64), {},
                             r"stream s=1:.* nr=2"),
    "prefix_tiled": ([30, 1, 200, 7] * 6, [1] * 24, 700, (8, 2, 128), {}, r"tile s=1:.* t=0:"),
    "prefix_many_parts": ([30, 1, 90, 7] * 5, [1] * 20, 6000, (4, 1, 64), {}, r"parts=[1-9]\d .*tile"),
    "prefix_drafts": ([30, 8, 200, 7] * 2, [5, 8, 3, 7] * 2, 900, (8, 2, 64), {},
                      r"tile s=1:.* t=0:.* nr=2"),
    "prefix_beside_long": ([150, 33, 60, 200, 20], [100, 3, 60, 1, 20], 900, (8, 2, 128), {},
                           r"tile s=1:.* t=1:"),
    "long_whole": ([300, 301], [300, 17], 40, (8, 2, 128), {}, r"parts=1 .*none .* t=1:1x"),
    "long_split": ([3000], [100], 70, (8, 2, 128), {}, r"none .* t=1:(?!1x)"),
    "long_beside_split": ([700, 3000, 90, 400], [680, 1, 1, 2], 0, (32, 1, 64),
                          dict(max_kv=4096, wide=256), r"none s=1:(?!1x)"),
    "seventy": ([40, 3] * 35, [20, 1] * 35, 30, (8, 2, 32), {}, r"none .* t=1:"),
    "seventy_behind_a_prefix": ([40, 3] * 35, [20, 1] * 35, 300, (8, 2, 32), {},
                                r"tile s=1:.* t=1:"),
    "head_group_of_80_behind_a_prefix": ([30, 9, 77, 1, 5, 60], [1, 2, 1, 1, 1, 1], 900,
                                         (80, 1, 64), {}, r"tile s=0:.* t=1:"),
    "head_group_of_80": ([90, 300], [1, 3], 33, (80, 1, 64), {}, r"s=0:.* t=1:"),
}


def plan_call(name):
    """The line that asks tests/paged_host.cc for a case's plan."""
    lens, counts, prefix, (hq, hkv, d), more, _ = PLANS[name]
    most = more.get("max_kv", max(-(-n // 16) for n in lens) * 16)
    return (f"attn batch={len(lens)} tokens={sum(counts) + 2} max_q={max(counts)} max_kv={most} "
            f"prefix_len={prefix} hq={hq} heads={hkv} d={d} table_stride=9999")
