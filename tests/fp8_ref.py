"""The fp8 tier's definition on the host, for its tests: e4m3 codes with one
f32 scale for each block of 128 (activations: a row's 128 columns; weights:
128 x 128), and the product over them in 64 bits."""
import torch

BLOCK = 128
F8 = torch.float8_e4m3fn


def blocks(n):
    return -(-n // BLOCK)


def scale_of(a):
    """f32: max(a / 448, 2^-126), NaN and infinity kept."""
    return (a.float() / 448.0).clamp(min=2.0 ** -126)


def quant_rows(x):
    """Codes [rows][K], scales [blocks][rows] of x in f32, by the definition's
    own f32 steps."""
    rows, K = x.shape
    q = torch.empty(rows, K, dtype=F8)
    s = torch.empty(blocks(K), rows)
    for b in range(blocks(K)):
        v = x[:, b * BLOCK:(b + 1) * BLOCK].float()
        s[b] = scale_of(v.abs().amax(1))
        q[:, b * BLOCK:(b + 1) * BLOCK] = (v * (1.0 / s[b])[:, None]).to(F8)
    return q, s


def quant_blocks(w):
    """Codes [N][K], scales [blocks of N][blocks of K]."""
    N, K = w.shape
    q = torch.empty(N, K, dtype=F8)
    s = torch.empty(blocks(N), blocks(K))
    for i in range(blocks(N)):
        for b in range(blocks(K)):
            at = (slice(i * BLOCK, (i + 1) * BLOCK), slice(b * BLOCK, (b + 1) * BLOCK))
            v = w[at].float()
            s[i, b] = scale_of(v.abs().amax())
            q[at] = (v * (1.0 / s[i, b])).to(F8)
    return q, s


def restore_rows(q, s):
    """f64 values of activation codes."""
    return q.double() * s.t().double().repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def restore_blocks(q, s):
    """f64 values of weight codes."""
    t = s.double().repeat_interleave(BLOCK, 0)[:q.shape[0]]
    return q.double() * t.repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def product(xq, sx, wq, sw):
    """y = x . w^T in f64, and how far a kernel's f32 sums may be from it.

    Additions: a block's groups, its scale (a product of two, and the product
    with the block's sum) and the blocks before it, each off by at most 2^-23 of
    the terms' magnitudes (rounded either way).

    The matrix unit: e4m3 products are exact, but of the 8 of a group (8
    neighbouring k) it keeps each only down to 2^-13 of 2^e, e the largest sum
    of two exponents in the group, and drops the rest (measured: equal to that
    rule on every one of 5000 sums of one group).  The largest product is at
    least 2^e and keeps its 6 fraction bits, so a group is off by less than
    7 * 2^-13 of it; that is at most the group's largest |x| times its largest
    |w|."""
    x, w = restore_rows(xq, sx), restore_blocks(wq, sw)
    K = x.shape[1]
    ops = min(K, BLOCK) + 3 + blocks(K)
    slack = (x.abs() @ w.abs().t()) * ops * 2.0 ** -23
    return x @ w.t(), slack, (groups(x) @ groups(w).t()) * 7 * 2.0 ** -13


def groups(t):
    """The largest magnitude of each 8 neighbouring columns."""
    return t.abs().view(len(t), -1, 8).amax(2)


def within(y, want, slack):
    """Whether bf16 outputs are within slack and half a bf16 step (2^-8)."""
    off = (y.double() - want).abs()
    return off <= want.abs() * 2.0 ** -8 + slack * (1 + 2.0 ** -8)


def norm(x, delta, w_und, w_gen, m_und, eps):
    """(r as held in bf16, the norm in f64)."""
    r = x if delta is None else (x.float() + delta.float()).to(torch.bfloat16)
    v = r.double()
    n = v / (v.square().mean(1, keepdim=True) + eps).sqrt()
    g = torch.cat([w_und.double().expand(m_und, -1),
                   w_gen.double().expand(len(x) - m_und, -1)])
    return r, n * g


def swiglu(gate, up):
    g = gate.double()
    return g * torch.sigmoid(g) * up.double()


def check_codes(q, s, v, rel):
    """Codes and scales of f64 values v that the kernel held with a relative
    error of at most `rel`: each scale within it and a division's rounding of
    the exact one, each code within half a step (2^-4 of the value, 2^-10 below
    e4m3's normal range) of what it rounds, which is off by `rel` for the value
    and as much for the scale and its reciprocal."""
    K = v.shape[1]
    for b in range(blocks(K)):
        t = v[:, b * BLOCK:(b + 1) * BLOCK]
        want = (t.abs().amax(1) / 448.0).clamp(min=2.0 ** -126)
        assert bool(((s[b].double() - want).abs() <= want * (rel + 2.0 ** -23)).all()), b
        ideal = t / want[:, None]
        off = (q[:, b * BLOCK:(b + 1) * BLOCK].double() - ideal).abs()
        slack = (2 * rel + 2.0 ** -21) * ideal.abs()
        most = torch.maximum(ideal.abs() * 2.0 ** -4, torch.full_like(ideal, 2.0 ** -10))
        assert bool((off <= most + slack).all()), (b, float((off - most).max()))


# Sizes (M_und, M_gen, K, Ns) at which the product takes each of its kernels on
# 256 compute units: the kernel, whether shares of K are split, and whether the
# workgroups run more than one round of tiles.
KINDS = [
    ((3, 0, 528, (264,)), "narrow 16x16", False, False),
    ((1, 1, 400, (2064,)), "narrow 16x32", False, False),
    ((0, 23, 656, (40, 8)), "narrow 32x16", False, False),
    ((2, 20, 272, (680, 1464)), "narrow 32x32", False, False),
    ((35, 10, 784, (72,)), "narrow 64x16", False, False),
    ((10, 36, 144, (2128,)), "narrow 64x32", False, False),
    ((70, 0, 1040, (136,)), "narrow 96x16", False, False),
    ((98, 5, 400, (136,)), "narrow 128x16", False, False),
    ((0, 132, 144, (200,)), "tiles 64x128", False, False),
    ((132, 5, 144, (8360, 7984)), "tiles 64x128", False, True),
    ((2, 131, 2208, (8,)), "tiles 64x128", True, False),
    ((140, 2, 432, (8408,)), "tiles 128x128", False, False),
    ((35, 586, 736, (10832,)), "tiles 128x128", False, True),
    ((69, 0, 4720, (5480,)), "tiles 128x128", True, False),
    ((17, 44, 3936, (16256, 312)), "tiles 128x128", True, True),
    ((18, 321, 288, (256, 15272)), "tiles 128x256", False, False),
    ((2, 3191, 368, (4808,)), "tiles 128x256", False, True),
    ((0, 82, 8048, (1752, 15544)), "tiles 128x256", True, False),
    ((464, 10, 2368, (13320,)), "tiles 128x256", True, True),
    ((6, 3632, 272, (128, 2712)), "tiles 192x256", False, False),
    ((2771, 0, 144, (7672,)), "tiles 192x256", False, True),
    ((0, 912, 9584, (4328,)), "tiles 192x256", True, False),
    ((0, 1676, 2992, (14520,)), "tiles 192x256", True, True),
    ((3327, 25, 400, (3592, 8)), "tiles 256x256", False, False),
    ((2590, 772, 144, (6056, 1496)), "tiles 256x256", False, True),
    ((0, 392, 6448, (9736,)), "tiles 256x256", True, False),
    ((0, 1764, 1376, (9624,)), "tiles 256x256", True, True),
]

# Sizes (M_und, M_gen, K, Ns) of long K, the kernel that takes each on 256
# compute units, and whether shares of K are split.  A narrow kernel's four
# waves take more than 64 blocks each above K 32768.
LONG = [
    ((1, 0, 33280, (1024,)), "narrow 16x16", False),
    ((1, 0, 131072, (4096,)), "narrow 16x16", False),
    ((1, 1, 33040, (16384,)), "narrow 16x32", False),
    ((20, 0, 33040, (4096,)), "narrow 32x16", False),
    ((17, 0, 33040, (8192,)), "narrow 32x32", False),
    ((1, 0, 33280, (264,)), "tiles 64x128", True),
    ((300, 0, 131072, (264,)), "tiles 64x128", True),
    ((5, 200, 40976, (512,)), "tiles 64x128", True),
    ((128, 0, 33040, (8192,)), "tiles 128x128", True),
    ((600, 0, 33040, (4096,)), "tiles 128x256", True),
    ((0, 700, 33040, (2048,)), "tiles 192x256", True),
    ((2048, 0, 33040, (8192,)), "tiles 256x256", False),
]
