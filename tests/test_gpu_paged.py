"""Many requests at once on the GPU: rotary positions, the paged cache and
attention behind a shared prefix, one by one and as a step calls them, against
the definition in 64 bits on the host (tests/paged_ref.py)."""
import math

import pytest
import torch

import paged_ref as ref
import u15h

pytestmark = pytest.mark.gpu

BF16, I32, F64 = torch.bfloat16, torch.int32, torch.float64


def bf16(seed, *shape, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(BF16)


def bits(t):
    return t.contiguous().view(torch.int16)


# ---- rotary positions ---------------------------------------------------------

def rotation(parts, neighbours=False, scaling="none", theta=(5e6, 1e4, 1e4)):
    """(Rope, host parts, scale) of [(start, width, axis)]."""
    host, scale = [], 1.0
    for start, width, axis in parts:
        f, sc = u15h.rope_freqs(width, theta[axis], scaling, factor=8.0, trained=4096)
        host.append((f, start, axis))
        scale = max(scale, sc)
    return u15h.Rope([(f.cuda(), s, a) for f, s, a in host], neighbours, scale), host, scale


def positions(seed, axes, tokens, most):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-most, most, (axes, tokens), generator=g).to(I32)


ROPES = [
    # tokens, heads, d, parts, neighbours, scaling
    (1, 32, 128, [(0, 128, 0)], False, "none"),
    (1, 1, 2, [(0, 2, 0)], True, "none"),
    (3, 5, 16, [(0, 16, 0)], False, "linear"),          # one access unit a head
    (7, 8, 128, [(0, 64, 0), (64, 32, 1), (96, 32, 2)], False, "yarn"),
    (7, 3, 128, [(96, 32, 2), (0, 64, 0)], True, "bands"),
    (33, 5, 96, [(8, 54, 0)], False, "ntk"),            # 27 pairs: single columns
    (33, 5, 96, [(8, 52, 0)], False, "none"),           # 26: two columns
    (33, 2, 80, [(0, 20, 0)], True, "none"),
    (5, 2, 33, [(1, 6, 0), (9, 24, 1)], False, "none"),  # odd heads and starts
    (5, 2, 33, [(1, 6, 0), (9, 24, 1)], True, "none"),
    (1030, 2, 64, [(0, 64, 0)], False, "yarn"),         # groups of tokens, the last short
    (1027, 1, 512, [(0, 512, 0)], True, "none"),
    (2049, 3, 32, [(0, 16, 1)], False, "none"),
]


@pytest.mark.parametrize("tokens,heads,d,parts,neighbours,scaling", ROPES)
@pytest.mark.parametrize("inverse", [False, True])
def test_rope(ops, tokens, heads, d, parts, neighbours, scaling, inverse):
    rope, host, scale = rotation(parts, neighbours, scaling)
    x = bf16(tokens + d, tokens, heads, d, std=2.0)
    pos = positions(tokens, 3, tokens, 1 << 22)
    y = torch.full((tokens, heads, d), math.nan, dtype=BF16, device="cuda")
    ops.rope(x.cuda(), pos.cuda(), rope, y, inverse=inverse)
    want, off = ref.turn(x, pos, host, neighbours, scale, inverse)
    assert bool(((y.cpu().to(F64) - want).abs() <= off).all())


def test_rope_far_positions(ops):
    """The whole range of positions, with the fastest frequency."""
    rope, host, _ = rotation([(0, 128, 0)])
    pos = torch.tensor([[0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 30 + 1, 123456789]], dtype=I32)
    x = bf16(1, 7, 4, 128)
    y = torch.empty(7, 4, 128, dtype=BF16, device="cuda")
    ops.rope(x.cuda(), pos.cuda(), rope, y)
    want, off = ref.turn(x, pos, host)
    assert bool(((y.cpu().to(F64) - want).abs() <= off).all())
    assert torch.equal(bits(y[0].cpu()), bits(x[0]))


@pytest.mark.parametrize("offset", [0, 1, 2])
@pytest.mark.parametrize("layout", ["columns", "head_major", "in_place"])
def test_rope_strides(ops, layout, offset):
    """Columns of a wider matrix, [heads][tokens][d], x itself; addresses that
    keep whole, pairs of and single columns together.  The rest stays."""
    T, H, d = 9, 3, 64
    rope, host, _ = rotation([(0, 64, 0)])
    pos = positions(3, 1, T, 1000)
    whole = bf16(5, 4096).cuda()
    before = whole.clone()
    if layout == "head_major":
        x = whole[offset:offset + T * H * d].view(H, T, d).transpose(0, 1)
    else:
        pitch = H * d + (16 if offset == 0 else offset)
        x = torch.as_strided(whole, (T, H, d), (pitch, d, 1), offset)
    xh = x.cpu()
    out = torch.full((4096,), 7.0, dtype=BF16, device="cuda")
    y = x if layout == "in_place" else torch.as_strided(out, x.shape, x.stride(), offset)
    ops.rope(x, pos.cuda(), rope, y)
    want, off = ref.turn(xh, pos, host)
    assert bool(((y.cpu().to(F64) - want).abs() <= off).all())
    touched = torch.zeros(4096, dtype=torch.bool)
    torch.as_strided(touched, x.shape, x.stride(), offset).fill_(True)
    rest = whole if layout == "in_place" else out
    same = before if layout == "in_place" else torch.full_like(out, 7.0)
    assert torch.equal(bits(rest)[~touched.cuda()], bits(same)[~touched.cuda()])


def test_rope_gradient(ops):
    """The inverse is the gradient: <dy, rope(x)> moves with x as <inverse
    rope(dy), .> says, by differences of the definition and by the formula."""
    T, H, d = 5, 2, 32
    rope, host, scale = rotation([(0, 24, 0)], True, "yarn")
    pos = positions(8, 1, T, 5000)
    x, dy = bf16(1, T, H, d), bf16(2, T, H, d)
    dx = torch.empty(T, H, d, dtype=BF16, device="cuda")
    ops.rope(dy.cuda(), pos.cuda(), rope, dx, inverse=True)
    leaf = x.to(F64).requires_grad_()
    angle = pos[0].to(F64)[:, None] * host[0][0]
    c, s = (torch.cos(angle) * scale)[:, None], (torch.sin(angle) * scale)[:, None]
    a, b = leaf[..., 0:24:2], leaf[..., 1:24:2]
    y = torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), leaf[..., 24:]], -1)
    (y * dy.to(F64)).sum().backward()
    _, off = ref.turn(dy, pos, host, True, scale, True)
    assert bool(((dx.cpu().to(F64) - leaf.grad).abs() <= off).all())
    step = 2.0 ** -10
    for at in [(0, 0, 0), (2, 1, 7), (4, 0, 23), (3, 1, 30)]:
        moved = x.to(F64).clone()
        moved[at] += step
        up, _ = ref.turn(moved, pos, host, True, scale)
        down, _ = ref.turn(x, pos, host, True, scale)
        slope = ((up - down) * dy.to(F64)).sum() / step
        assert abs(float(dx[at]) - float(slope)) <= float(off[at]) + 1e-9


# ---- appending ----------------------------------------------------------------

@pytest.mark.parametrize("tokens,hq,hkv,d,page", [(1, 32, 8, 128, 16), (67, 6, 2, 64, 32),
                                                  (1030, 4, 4, 32, 256), (40, 0, 1, 128, 16),
                                                  (300, 66, 1, 64, 16)])
@pytest.mark.parametrize("parts", ["whole", "axes", "odd", None])
def test_append(ops, tokens, hq, hkv, d, page, parts):
    """Keys, values and queries from columns of one matrix into slots in any
    order, padding passed over; every other slot keeps its bits."""
    spec = {"whole": [(0, d, 0)], "axes": [(0, d // 2, 0), (d // 2, d // 4, 1),
                                           (3 * d // 4, d // 4, 2)], "odd": [(1, 14, 0)]}
    turned = parts is not None
    hq = hq if turned else 0
    rope, host, scale = rotation(spec[parts], parts == "odd") if turned else (None, [], 1.0)
    qkv = bf16(tokens, tokens, hq + 2 * hkv, d)
    dev = qkv.cuda()
    pos = positions(2, 3, tokens, 100000)
    pages = -(-tokens // page) + 2
    both = bf16(9, pages, 2, hkv, page, d).cuda()          # k and v in one allocation
    kv = u15h.PagedKV(both[:, 0], both[:, 1])
    before = both.cpu()
    slot = torch.randperm(pages * page, generator=torch.Generator().manual_seed(3))[:tokens]
    slot[5::7] = -1
    if tokens > 30:
        slot[11], slot[12], slot[13] = pages * page, 2 ** 31 - 1, -2 ** 31
    live = (slot >= 0) & (slot < pages * page)
    q_out = torch.full((tokens, max(hq, 1), d), 3.0, dtype=BF16, device="cuda")
    ops.paged_append(kv, dev[:, hq:hq + hkv], dev[:, hq + hkv:], slot.to(I32).cuda(),
                     pos=pos.cuda() if turned else None, rope=rope, q=dev[:, :hq] if hq else None,
                     q_out=q_out if hq else None)
    after = both.cpu()
    k, koff = ref.turn(qkv[:, hq:hq + hkv], pos, host, parts == "odd", scale)
    p, o = slot[live] // page, slot[live] % page
    got = after[p, 0, :, o].to(F64)
    assert bool(((got - k[live]).abs() <= koff[live]).all())
    assert torch.equal(bits(after[p, 1, :, o]), bits(qkv[live][:, hq + hkv:]))
    rest = torch.ones(pages, page, dtype=torch.bool)
    rest[p, o] = False
    i, j = rest.nonzero(as_tuple=True)
    assert torch.equal(bits(after[i, :, :, j]), bits(before[i, :, :, j]))
    if hq:
        want, off = ref.turn(qkv[:, :hq], pos, host, parts == "odd", scale)
        out = q_out.cpu()
        assert bool(((out.to(F64) - want).abs() <= off)[live].all())
        assert bool((out[~live] == 3.0).all())


def test_append_in_place(ops):
    """Queries turned where they are, padding's rows left."""
    T, H, d = 21, 4, 64
    rope, host, _ = rotation([(0, 64, 0)])
    q, kvr = bf16(1, T, H, d), bf16(2, T, 2, d)
    pos = positions(4, 1, T, 5000)
    slot = torch.arange(T)
    slot[-4:] = -1
    pool = torch.zeros(2, 2, 1, 16, d, dtype=BF16, device="cuda")
    kv = u15h.PagedKV(pool[:, 0], pool[:, 1])
    qd = q.cuda()
    ops.paged_append(kv, kvr.cuda()[:, :1], kvr.cuda()[:, 1:], slot.to(I32).cuda(), pos.cuda(),
                     rope, q=qd, q_out=qd)
    want, off = ref.turn(q, pos, host)
    assert bool(((qd.cpu().to(F64) - want).abs() <= off)[:-4].all())
    assert torch.equal(bits(qd[-4:].cpu()), bits(q[-4:]))


# ---- attention ----------------------------------------------------------------

class Case:
    """A paged cache with NaN wherever no key lies, a batch over it, queries."""

    def __init__(self, lens, counts, prefix, hq, hkv, d, page, seed=0, pad=2, std=1.5, spare=2,
                 stride=0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.counts, self.prefix, self.page = lens, counts, prefix, page
        first = -(-prefix // page)
        each = [-(-n // page) for n in lens]
        pages = first + sum(each) + spare
        order = torch.randperm(pages, generator=g)
        shape = (pages, hkv, page, d)
        self.kp = torch.full(shape, math.nan, dtype=BF16)
        self.vp = torch.full(shape, math.nan, dtype=BF16)
        self.prefix_table = order[:first].to(I32)
        width = max(each + [1]) + stride
        # entries past a sequence's pages are never read
        self.table = torch.full((len(lens), width), 2 ** 31 - 1, dtype=I32)
        at = first
        for b, n in enumerate(each):
            self.table[b, :n] = order[at:at + n].to(I32)
            at += n
        for table, n in [(self.prefix_table, prefix)] + [(t, n) for t, n in
                                                         zip(self.table, lens)]:
            for i in range(-(-n // page)):
                k = min(page, n - i * page)
                for pool in (self.kp, self.vp):
                    pool[int(table[i]), :, :k] = torch.randn(hkv, k, d, generator=g).to(BF16)
        self.rows = sum(counts)
        self.q = (torch.randn(self.rows + pad, hq, d, generator=g) * std).to(BF16)
        start = [0]
        for c in counts:
            start.append(start[-1] + c)
        self.q_start = torch.tensor(start, dtype=I32)

    def batch(self, max_q=None, max_kv=None, own_rows=True):
        some = own_rows or any(c != 1 for c in self.counts)
        return u15h.PagedBatch(torch.tensor(self.lens, dtype=I32).cuda(), self.table.cuda(),
                               q_start=self.q_start.cuda() if some else None,
                               max_q=max_q or max(self.counts + [1]),
                               max_kv=max_kv, prefix_table=self.prefix_table.cuda(),
                               prefix_len=self.prefix)

    def widen(self, pages):
        """The table with room for as many pages."""
        more = torch.full((len(self.lens), pages), -1, dtype=I32)
        more[:, :self.table.shape[1]] = self.table
        self.table = more

    def run(self, ops, causal, scale=0.0, batch=None, pad_q=0, pad_out=0, stream=None):
        """out [rows + pad][hq][d], guarded by rows of a wider matrix."""
        n, hq, d = self.q.shape
        kv = u15h.PagedKV(self.kp.cuda(), self.vp.cuda())
        wide = torch.full((n, hq + 1, d), 5.0, dtype=BF16, device="cuda")
        qw = torch.full((n, hq + pad_q, d), math.nan, dtype=BF16, device="cuda")
        qw[:, :hq] = self.q.cuda()
        ops.paged_attention(kv, batch or self.batch(), qw[:, :hq], wide[:, :hq], scale=scale,
                            causal=causal, stream=stream)
        host = wide.cpu()
        assert bool((host[:, hq] == 5.0).all()), "beside the rows"
        assert bool((host[self.rows:] == 5.0).all()), "rows of no sequence"
        return host[:self.rows, :hq]

    def want(self, causal, scale=0.0):
        return ref.attend(self.q[:self.rows], self.kp, self.vp, self.prefix_table, self.prefix,
                          self.table, self.lens, self.counts, causal, scale)


def check(out, want):
    o, bound = want
    diff = (out.to(F64) - o).abs()
    assert not bool(torch.isnan(diff).any())
    worst = (diff / bound.clamp(min=1e-38)).max() if diff.numel() else torch.zeros(())
    assert float(worst) <= 1.0, float(worst)


HEADS = [(32, 8, 128), (4, 4, 64), (6, 2, 32), (10, 1, 128), (24, 1, 64), (70, 2, 32)]
BATCHES = {
    "one": ([1], [1]),
    "tile_edges": ([15, 16, 17, 31, 32, 33], [1] * 6),
    "none": ([0, 3, 0], [1, 0, 1]),
    "more_queries_than_keys": ([5, 40], [9, 60]),
    "drafts": ([5, 77, 130, 64], [5, 5, 4, 3]),
    "chunks": ([130, 257, 1, 64, 300], [130, 33, 1, 64, 2]),
    "long": ([1500], [1]),
}


@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("name", list(BATCHES))
@pytest.mark.parametrize("prefix,page,causal", [(0, 16, True), (33, 16, True), (100, 64, False),
                                                (1, 32, True), (513, 16, False)])
def test_attention(ops, hq, hkv, d, name, prefix, page, causal):
    lens, counts = BATCHES[name]
    c = Case(lens, counts, prefix, hq, hkv, d, page, seed=prefix + hq)
    check(c.run(ops, causal), c.want(causal))


def planned(name, **more):
    lens, counts, prefix, (hq, hkv, d), kw, _ = ref.PLANS[name]
    c = Case(lens, counts, prefix, hq, hkv, d, 16, seed=len(name), **more)
    if "wide" in kw:
        c.widen(kw["wide"])
    return c, dict(max_kv=kw.get("max_kv"))


@pytest.mark.parametrize("name", list(ref.PLANS))
@pytest.mark.parametrize("causal", [True, False])
def test_attention_every_plan(ops, name, causal):
    """Every way in which a call is cut over workgroups, joined and added; twice,
    so that what one call leaves in the scratch does not reach the next."""
    c, kw = planned(name)
    want = c.want(causal)
    first = c.run(ops, causal, batch=c.batch(**kw))
    check(first, want)
    other, okw = planned("joined" if name != "joined" else "prefix_beside_long")
    other.run(ops, causal, batch=other.batch(**okw))
    assert torch.equal(bits(c.run(ops, causal, batch=c.batch(**kw))), bits(first))


@pytest.mark.parametrize("name", list(ref.PLANS))
def test_attention_bad_pages_every_plan(ops, name):
    """Holes in the prefix's and the sequences' pages."""
    c, kw = planned(name)
    if c.prefix > 16:
        c.prefix_table[1::3] = -1
    c.table[:, 0::4] = c.kp.shape[0]
    check(c.run(ops, True, batch=c.batch(**kw)), c.want(True))


@pytest.mark.parametrize("name", list(ref.PLANS))
def test_attention_nan(ops, name):
    """A NaN in a query reaches its own row and head, one in a key that a query
    sees all heads of that key's, one in a key that the mask hides nothing."""
    c, kw = planned(name)
    G = c.q.shape[1] // c.kp.shape[1]
    want = c.want(True)
    clean = c.run(ops, True, batch=c.batch(**kw))
    row = c.rows - 1
    c.q[row, 1, 5] = math.nan
    nan = torch.zeros(c.rows, c.q.shape[1], dtype=torch.bool)
    nan[row, 1] = c.prefix > 0 or c.lens[-1] > 0
    # the last key of the sequence with most queries: the last of those sees it
    b = max(range(len(c.lens)), key=lambda i: c.counts[i])
    n = c.lens[b]
    c.kp[int(c.table[b, (n - 1) // 16]), 0, (n - 1) % 16, 3] = math.nan
    nan[int(c.q_start[b + 1]) - 1, :G] = True
    out = c.run(ops, True, batch=c.batch(**kw))
    assert torch.equal(torch.isnan(out).any(-1), nan) and torch.equal(torch.isnan(out).all(-1), nan)
    assert torch.equal(bits(out[~nan]), bits(clean[~nan]))
    check(clean, want)


def test_attention_without_scratch(monkeypatch):
    """A context without the split's scratch: every sequence by itself."""
    monkeypatch.setenv("U15H_ATTN_SPLIT", "0")
    o = u15h.Ops(0)
    for name in ("joined", "prefix_tiled", "prefix_beside_long", "long_split",
                 "long_beside_split"):
        c, kw = planned(name)
        check(c.run(o, True, batch=c.batch(**kw)), c.want(True))
    torch.cuda.synchronize()
    o.close()


@pytest.mark.parametrize("names", [("joined", "prefix_tiled"), ("prefix_beside_long", "joined_rows"),
                                   ("long_beside_split", "prefix_streamed")])
def test_attention_captured(ops, names):
    """Two graphs over one context's scratch, replayed in turn with eager calls
    between, while lengths, starts and pages change under them."""
    made = []
    for name in names:
        c, kw = planned(name)
        kv = u15h.PagedKV(c.kp.cuda(), c.vp.cuda())
        kv_len, q_start = torch.tensor(c.lens, dtype=I32).cuda(), c.q_start.cuda()
        table = c.table.cuda()
        b = u15h.PagedBatch(kv_len, table, q_start=q_start, max_q=max(c.counts),
                            max_kv=kw["max_kv"], prefix_table=c.prefix_table.cuda(),
                            prefix_len=c.prefix)
        q = c.q.cuda()
        out = torch.full_like(q, 5.0)
        ops.paged_attention(kv, b, q, out)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.paged_attention(kv, b, q, out)
        made.append((c, kv, b, q, out, kv_len, q_start, table, g))
    for step in range(4):
        for c, kv, b, q, out, kv_len, q_start, table, g in made:
            lens = [max(0, n - 7 * step) for n in c.lens]
            counts = [max(0, n - step) for n in c.counts]
            start = [0]
            for n in counts:
                start.append(start[-1] + n)
            order = torch.roll(torch.arange(len(lens)), step).tolist()
            tables = c.table[order]
            lens = [lens[i] for i in order]
            kv_len.copy_(torch.tensor(lens, dtype=I32))
            q_start.copy_(torch.tensor(start, dtype=I32))
            table.copy_(tables)
            out.fill_(5.0)
            g.replay()
            got = out.clone()
            out.fill_(5.0)
            ops.paged_attention(kv, b, q, out)
            torch.cuda.synchronize()
            assert torch.equal(bits(out), bits(got)), step
            check(got[:start[-1]].cpu(),
                  ref.attend(c.q[:start[-1]], c.kp, c.vp, c.prefix_table, c.prefix, tables, lens,
                             counts, True))
            assert bool((got[start[-1]:] == 5.0).all())


def test_attention_first_call_captured():
    """A context whose first joined call is captured and runs after an eager one."""
    o = u15h.Ops(0)
    junk = torch.full((64 << 20,), 7, dtype=torch.uint8, device="cuda")     # what memory held
    c, kw = planned("joined")
    kv, b = u15h.PagedKV(c.kp.cuda(), c.vp.cuda()), c.batch(**kw)
    q = c.q.cuda()
    out, eager = torch.zeros_like(q), torch.zeros_like(q)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o.paged_attention(kv, b, q, out)
    o.paged_attention(kv, b, q, eager)
    for _ in range(3):
        out.fill_(0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(bits(out), bits(eager))
        o.paged_attention(kv, b, q, eager)
    check(eager[:c.rows].cpu(), c.want(True))
    torch.cuda.synchronize()
    del g, junk
    o.close()


def test_calls_on_another_stream(ops):
    """All three on a stream that is not the current one, in its order."""
    other = torch.cuda.Stream()
    hq, hkv, d, T = 8, 2, 128, 70
    rope, host, _ = rotation([(0, d, 0)])
    qkv = bf16(3, T, hq + 2 * hkv, d).cuda()
    pos = torch.arange(T, dtype=I32)[None].cuda()
    slot = torch.arange(T, dtype=I32).cuda()
    pool = torch.zeros(2, 5, hkv, 16, d, dtype=BF16, device="cuda")
    kv = u15h.PagedKV(pool[0], pool[1])
    q, out, y = (torch.zeros(T, hq, d, dtype=BF16, device="cuda") for _ in range(3))
    b = u15h.PagedBatch(torch.tensor([T], dtype=I32).cuda(), torch.arange(5, dtype=I32)[None].cuda(),
                        q_start=torch.tensor([0, T], dtype=I32).cuda(), max_q=T)
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        torch.cuda._sleep(20_000_000)
        ops.paged_append(kv, qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], slot, pos, rope, q=qkv[:, :hq],
                         q_out=q, stream=other)
        ops.paged_attention(kv, b, q, out, stream=other)
        ops.rope(out, pos, rope, y, inverse=True, stream=other)
    assert bool((y == 0).all())                      # not in the current stream's way
    other.synchronize()
    check(out.cpu(), ref.attend(q.cpu(), pool[0].cpu(), pool[1].cpu(), [], 0,
                                [list(range(5))], [T], [T], True))
    want, off = ref.turn(out.cpu(), pos.cpu(), host, inverse=True)
    assert bool(((y.cpu().to(F64) - want).abs() <= off).all())


def test_python_refusals(ops):
    """What the Python forms refuse before the library is asked."""
    c = Case([20], [1], 0, 8, 2, 64, 16)
    kv, b = u15h.PagedKV(c.kp.cuda(), c.vp.cuda()), c.batch()
    q = c.q[:1].cuda()
    out = torch.empty_like(q)
    rope, _, _ = rotation([(0, 64, 0)])
    pos, slot = torch.zeros(1, 1, dtype=I32).cuda(), torch.zeros(1, dtype=I32).cuda()
    k = torch.zeros(1, 2, 64, dtype=BF16, device="cuda")
    wide = torch.zeros(1, 8, 128, dtype=BF16, device="cuda")
    bad = [lambda: ops.paged_attention(kv, b, q.float(), out),
           lambda: ops.paged_attention(kv, b, q.cpu(), out),
           lambda: ops.paged_attention(kv, b, q[0], out),
           lambda: ops.paged_attention(kv, b, q, out[:, :4]),
           lambda: ops.paged_attention(kv, b, q[:, :7], out[:, :7]),
           lambda: ops.paged_attention(kv, b, wide[..., ::2], out),
           lambda: ops.paged_attention(kv, b, wide, wide.clone()),
           lambda: ops.paged_attention(kv, b, q, out, scale=-1.0),
           lambda: ops.rope(q, pos[0, :0], rope, out),
           lambda: ops.rope(q, pos.long(), rope, out),
           lambda: ops.rope(q, pos, rope, out[:, :2]),
           lambda: ops.rope(q[..., :32], pos, rope, out[..., :32]),
           lambda: ops.paged_append(kv, k, k[:, :1], slot),
           lambda: ops.paged_append(kv, k, k, slot, rope=rope),
           lambda: ops.paged_append(kv, k, k, slot.long()),
           lambda: ops.paged_append(kv, k, k, slot, pos, rope, q=q),
           lambda: ops.paged_append(kv, k, k, slot, q_out=out),
           lambda: ops.paged_append(kv, k, k, slot, q=q, q_out=out),
           lambda: u15h.PagedKV(c.kp.cuda(), c.vp.cuda()[1:]),
           lambda: u15h.PagedKV(c.kp.cuda()[:, :, ::2], c.vp.cuda()[:, :, ::2]),
           lambda: u15h.PagedKV(c.kp, c.vp),
           lambda: u15h.PagedBatch(torch.zeros(2, dtype=I32).cuda(), c.table.cuda()),
           lambda: u15h.PagedBatch(torch.zeros(1).cuda(), c.table.cuda()),
           lambda: u15h.PagedBatch(torch.zeros(1, dtype=I32).cuda(), c.table.cuda(), max_q=2),
           lambda: c.batch(max_kv=1000) and ops.paged_attention(kv, c.batch(max_kv=1000), q, out),
           lambda: u15h.Rope([]),
           lambda: u15h.Rope([(torch.zeros(4, device="cuda"), 0, 0)]),
           lambda: u15h.Rope([(torch.zeros(4, dtype=F64, device="cuda"), 0, 3)])]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, TypeError, u15h.U15hError)):
            f()
            pytest.fail(f"refusal {i}")
    ops.paged_attention(kv, b, q, out)
    ops.paged_append(kv, k, k, slot)


@pytest.mark.parametrize("batch,prefix", [(40, 700), (100, 64), (17, 2000), (3, 1000)])
def test_attention_decode(ops, batch, prefix):
    """Many sequences of one query behind a shared prefix."""
    g = torch.Generator().manual_seed(batch)
    lens = torch.randint(1, 300, (batch,), generator=g).tolist()
    c = Case(lens, [1] * batch, prefix, 8, 2, 128, 16, seed=batch)
    out = c.run(ops, True)
    check(out, c.want(True))
    alone = c.run(ops, True, batch=c.batch(own_rows=False))
    assert torch.equal(bits(alone), bits(out))            # one row each, said or not
    assert torch.equal(bits(c.run(ops, False)), bits(out))    # and no key is ahead


@pytest.mark.parametrize("count,prefix", [(200, 0), (300, 77), (129, 600)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_long_queries(ops, count, prefix, causal):
    c = Case([count + 40, count], [count, count - 1], prefix, 8, 2, 128, 64, seed=count)
    check(c.run(ops, causal), c.want(causal))


def test_attention_scale_and_peaks(ops):
    """A scale of one's own; scores far apart, so one key has all the weight."""
    c = Case([50, 700], [3, 3], 300, 8, 2, 64, 16, std=12.0)
    check(c.run(ops, True, scale=0.7), c.want(True, 0.7))
    check(c.run(ops, True, scale=1e-3), c.want(True, 1e-3))


def test_attention_rows_of_wider_matrices(ops):
    c = Case([50, 70], [2, 1], 40, 8, 2, 128, 16)
    plain = c.run(ops, True)
    check(plain, c.want(True))
    assert torch.equal(bits(c.run(ops, True, pad_q=3)), bits(plain))


def test_attention_bad_pages(ops):
    """Page numbers outside the cache, in the prefix and among own pages: their
    keys are masked, and a row that is left with none gets zeros."""
    c = Case([100, 40, 20], [2, 1, 1], 90, 8, 2, 128, 16)
    c.table[0, 1], c.table[0, 4] = -1, 2 ** 31 - 1
    c.table[1, :3] = torch.tensor([-2 ** 31, c.kp.shape[0], -5], dtype=I32)
    c.prefix_table[2] = c.kp.shape[0]
    check(c.run(ops, True), c.want(True))
    c = Case([100, 40, 20], [2, 1, 1], 0, 8, 2, 128, 16)
    c.table[1, :3] = -1
    out = c.run(ops, True)
    check(out, c.want(True))
    assert bool((out[2] == 0).all())


def test_attention_keeps_to_its_bounds(ops):
    """Lengths and starts past max_kv, max_q and the rows count as those."""
    c = Case([64, 64, 64], [4, 4, 4], 20, 4, 2, 64, 16)
    lens = torch.tensor([1000, 64, -7], dtype=I32).cuda()
    start = torch.tensor([-3, 4, 8, 100], dtype=I32).cuda()
    kv = u15h.PagedKV(c.kp.cuda(), c.vp.cuda())
    b = u15h.PagedBatch(lens, c.table.cuda(), q_start=start, max_q=4, max_kv=64,
                        prefix_table=c.prefix_table.cuda(), prefix_len=20)
    q = c.q.cuda()
    out = torch.full_like(q, 5.0)
    ops.paged_attention(kv, b, q, out, causal=False)
    c.lens = [64, 64, 0]
    check(out[:12].cpu(), c.want(False))
    assert bool((out[12:] == 5.0).all())


def test_attention_page_stride_and_offsets(ops):
    """k and v in one allocation whose later pages lie past 2^31 elements."""
    pages, hkv, page, d = 5, 1, 16, 64
    stride = (1 << 29) + 8
    whole = torch.zeros(4 * stride + 2 * hkv * page * d, dtype=BF16, device="cuda")
    size = (pages, hkv, page, d)
    k = torch.as_strided(whole, size, (stride, page * d, d, 1))
    v = torch.as_strided(whole, size, (stride, page * d, d, 1), hkv * page * d)
    c = Case([70], [1], 0, 4, 1, 64, 16, spare=0)
    k.copy_(c.kp.cuda())
    v.copy_(c.vp.cuda())
    out = torch.empty(1, 4, 64, dtype=BF16, device="cuda")
    ops.paged_attention(u15h.PagedKV(k, v), c.batch(), c.q[:1].cuda(), out)
    check(out.cpu(), c.want(True))


# ---- the largest calls ----------------------------------------------------------

@pytest.mark.parametrize("tokens,heads,d,turned", [(1 << 22, 1, 16, 16), (3, 4096, 32, 32),
                                                   (5, 4096, 512, 30), (1500, 300, 512, 500),
                                                   (1, 1, 512, 2)])
def test_rope_largest(ops, tokens, heads, d, turned):
    rope, host, _ = rotation([(0, turned, 1)])                  # theta 1e4
    g = torch.Generator(device="cuda").manual_seed(tokens)
    x = torch.randn(tokens, heads, d, device="cuda", generator=g).to(BF16)
    y = torch.full_like(x, math.nan)
    pos = torch.arange(tokens, dtype=I32, device="cuda")[None].repeat(2, 1)
    ops.rope(x, pos, rope, y)
    parts = [(f.cuda(), s, a) for f, s, a in host]
    step = max(1, (1 << 22) // (heads * d))
    for t in range(0, tokens, step):
        want, off = ref.turn(x[t:t + step], pos[:, t:t + step], parts)
        assert bool(((y[t:t + step].to(F64) - want).abs() <= off).all()), t


def test_append_4096_heads(ops):
    """As the rotation by itself, values bit for bit."""
    hq, hkv, d, T = 4096, 64, 32, 40
    rope, _, _ = rotation([(0, d, 0)])
    q, k, v = bf16(1, T, hq, d).cuda(), bf16(2, T, hkv, d).cuda(), bf16(3, T, hkv, d).cuda()
    pool = torch.zeros(2, 4, hkv, 16, d, dtype=BF16, device="cuda")
    pos = torch.arange(T, dtype=I32, device="cuda")[None]
    out, yq, yk = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k)
    ops.paged_append(u15h.PagedKV(pool[0], pool[1]), k, v, pos[0].contiguous(), pos, rope, q=q,
                     q_out=out)
    ops.rope(q, pos, rope, yq)
    ops.rope(k, pos, rope, yk)
    slots = pool.transpose(2, 3).flatten(1, 2)[:, :T]
    assert torch.equal(bits(out), bits(yq)) and torch.equal(bits(slots[0]), bits(yk))
    assert torch.equal(bits(slots[1]), bits(v))


@pytest.mark.parametrize("prefix", [0, 60])
def test_attention_20000_sequences(ops, prefix):
    """More sequences than are looked at together; the reference on the GPU in 64
    bits, within the weights' and the output's rounding of values below 6."""
    b, hq, hkv, d, most = 20000, 8, 2, 32, 40
    g = torch.Generator(device="cuda").manual_seed(prefix)
    lens = torch.randint(0, most, (b,), device="cuda", generator=g).to(I32)
    table = torch.randint(0, 500, (b, 3), device="cuda", generator=g).to(I32)
    kp, vp = (torch.randn(500, hkv, 16, d, device="cuda", generator=g).to(BF16)
              for _ in range(2))
    q = torch.randn(b, hq, d, device="cuda", generator=g).to(BF16)
    out = torch.full_like(q, math.nan)
    pt = torch.arange(40, 44, device="cuda", dtype=I32)
    ops.paged_attention(u15h.PagedKV(kp, vp),
                        u15h.PagedBatch(lens, table, max_kv=most, prefix_table=pt,
                                        prefix_len=prefix), q, out)
    both = []
    for pool in (kp, vp):
        own = pool[table.long()].transpose(2, 3).flatten(1, 2)[:, :most]
        first = pool[pt.long()].transpose(1, 2).flatten(0, 1)[:prefix].expand(b, -1, -1, -1)
        both.append(torch.cat([first, own], 1).to(F64).repeat_interleave(hq // hkv, 2))
    s = (q.to(F64)[:, None] * both[0]).sum(-1) / math.sqrt(d)
    hidden = torch.arange(prefix + most, device="cuda")[None] >= prefix + lens[:, None]
    s = s.masked_fill(hidden[..., None], -math.inf)
    w = torch.softmax(s, 1).nan_to_num(0.0)
    want = (w[..., None] * both[1]).sum(1)
    assert float(both[1].abs().max()) < 6
    assert float((out.to(F64) - want).abs().max()) <= 2.1 * 2.0 ** -8 * 6


# ---- a step -------------------------------------------------------------------

def test_step_with_the_layer_s_operators(ops):
    """Three requests behind one prompt, two steps: append the prompt, then
    each step's keys, and attend; against u15h_sdpa's caches of each request,
    and against 64 bits."""
    hq, hkv, d, page, P = 8, 2, 64, 16, 40
    rope, host, _ = rotation([(0, 64, 0)])
    pool = torch.zeros(12, 2, hkv, page, d, dtype=BF16, device="cuda")
    kv = u15h.PagedKV(pool[:, 0], pool[:, 1])
    prompt = bf16(1, P, 2 * hkv, d)
    ppos = torch.arange(P, dtype=I32)[None]
    prefix_table = torch.tensor([7, 2, 9], dtype=I32)
    slot = (prefix_table[:, None] * page + torch.arange(page)).flatten()[:P].to(I32)
    ops.paged_append(kv, prompt.cuda()[:, :hkv], prompt.cuda()[:, hkv:], slot.cuda(),
                     ppos.cuda(), rope)
    table = torch.tensor([[0, 1], [3, 4], [5, 6]], dtype=I32)
    lens, counts = [0, 0, 0], [3, 1, 14]
    rows = [[prompt], [prompt], [prompt]]
    for step in range(3):
        lens = [a + b for a, b in zip(lens, counts)]
        T = sum(counts)
        qkv = bf16(10 + step, T + 1, hq + 2 * hkv, d)
        pos, slots, at = [], [], 0
        for b, c in enumerate(counts):
            own = torch.arange(lens[b] - c, lens[b])
            pos.append(P + own)
            slots.append(table[b][own // page] * page + own % page)
            rows[b].append(qkv[at:at + c, hq:])
            at += c
        pos = torch.cat(pos + [torch.zeros(1)]).to(I32)[None]
        slots = torch.cat(slots + [-torch.ones(1)]).to(I32)
        dev = qkv.cuda()
        ops.paged_append(kv, dev[:, hq:hq + hkv], dev[:, hq + hkv:], slots.cuda(), pos.cuda(),
                         rope, q=dev[:, :hq], q_out=dev[:, :hq])
        start = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=I32)
        batch = u15h.PagedBatch(torch.tensor(lens, dtype=I32).cuda(), table.cuda(),
                                q_start=start.cuda(), max_q=max(counts),
                                prefix_table=prefix_table.cuda(), prefix_len=P)
        out = torch.zeros(T + 1, hq, d, dtype=BF16, device="cuda")
        ops.paged_attention(kv, batch, dev[:, :hq], out)
        k, v = pool[:, 0].cpu(), pool[:, 1].cpu()
        check(out[:T].cpu(), ref.attend(dev[:T, :hq].cpu(), k, v, prefix_table, P, table, lens,
                                        counts, True))
        assert bool((out[T] == 0).all())
        # the contiguous cache's operators on each request by itself
        at = 0
        for b, c in enumerate(counts):
            n = P + lens[b]
            own = torch.cat(rows[b]).cuda()
            turned = torch.empty(n, hkv, d, dtype=BF16, device="cuda")
            ops.rope(own[:, :hkv], torch.arange(n, dtype=I32)[None].cuda(), rope, turned)
            cache = turned.transpose(0, 1).contiguous()
            vals = own[:, hkv:].transpose(0, 1).contiguous()
            alone = torch.empty(c, hq * d, dtype=BF16, device="cuda")
            ops.attention_token_major(dev[at:at + c, :hq].reshape(c, hq * d).contiguous(), cache,
                                      vals, alone, hq, hkv, n, mode=1, q_offset=n - c)
            one = out[at:at + c].reshape(c, hq * d).float()
            # both within 2^-8 (weights) + 2^-8 (output) of the exact row
            assert float((one - alone.float()).abs().max()) <= 4 * 2.0 ** -8 * float(
                vals.float().abs().max())
            at += c
        counts = [1, 1, 2]
