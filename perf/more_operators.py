"""Serving many requests at once, as cases that can be timed and compared:
rotary positions, the paged key and value cache, and attention for a batch
whose sequences share a prefix, through `u15h.Ops`.

    rope    rope: pairs of columns of every head turned by position * frequency,
            in halves (i, i + width / 2) or neighbours (2 i, 2 i + 1), over the
            whole head, a part of it or several parts with axes of their own;
            frequencies as they are or scaled for long contexts
    append  paged_append: a step's keys, rotated, and its values into the slots
            of a paged cache, and its queries rotated, in one call
    attn    paged_attention: softmax(q . k * scale) . v over the shared prefix's
            pages and then the sequence's own, whose last keys are the queries'
            own positions

A cache is pages [pages][kv heads][page][head dim].  Heads are the model's (32
query heads over 8, 128 wide) and drawn ones.  Lengths within a batch are
spread evenly, in no order, by the golden ratio.
"""
import math
import os
import sys

import torch

own = False

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
THETA = (5e6, 1e4, 1e4)                    # the model's t, h and w axes
TRAINED = 4096                             # positions before the scaling
FACTOR = 8.0

_OPS = None


def _lib():
    pkg = os.path.join(os.getcwd(), "vpipe-sensenova-u1.5_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import u15h
    return u15h


def _ops():
    """The program's one context."""
    global _OPS
    if _OPS is None:
        _OPS = _lib().Ops(0)
    return _OPS


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------

FULL, MODEL = "0:128:0", "0:64:0,64:32:1,96:32:2"     # start : width : axis


def _attn(prefix, own, q, batch=1, hq=32, hkv=8, d=128, page=16, causal=True, pad=0, **more):
    return dict(kind="attn", batch=batch, prefix=prefix, own=own, queries=q, hq=hq, hkv=hkv, d=d,
                page=page, causal=causal, pad=pad, **more)


def _rope(tokens, heads=32, d=128, parts=FULL, pairs="halves", scaling="none", at=0,
          inverse=False, fused=False, **more):
    return dict(kind="rope", tokens=tokens, heads=heads, d=d, parts=parts, pairs=pairs,
                scaling=scaling, at=at, inverse=inverse, fused=fused, **more)


def _append(tokens, hq=32, hkv=8, d=128, page=16, parts=FULL, pairs="halves", scaling="none",
            at=0, pad=0, **more):
    return dict(kind="append", tokens=tokens, hq=hq, hkv=hkv, d=d, page=page, parts=parts,
                pairs=pairs, scaling=scaling, at=at, pad=min(pad, tokens - 1), **more)


def listed():
    return [
        # one token's queries
        _rope(1, at=777, name="rope_one"),
        # a context past the trained one: neighbours, half of the head, far positions
        _rope(1000, parts="0:64:0", pairs="neighbours", scaling="yarn", at=1000000, fused=True,
              name="rope_part_far"),
        # an image and its prompt turned back, as a gradient or a cache moved in time needs it
        _rope(4224, parts=MODEL, inverse=True, name="rope_image_back"),
        # a decoding step of 64 requests, a few rows of it padding
        _append(64, at=4000, pad=5, name="append_64"),
        # a 1024 x 1024 image's and its prompt's keys, queries and values
        _append(4224, page=64, parts=MODEL, name="append_image"),
        # one request's next token after a system prompt and a line of text
        _attn(128, "77:77", "1:1", name="attn_one"),
        # one request's next token after a book of its own
        _attn(0, "131072:131072", "1:1", page=256, name="attn_one_long"),
        # 64 answers over one image and its prompt
        _attn(4224, "1:1024", "1:1", batch=64, name="attn_64_answers"),
        # 256 questions on one long document
        _attn(32768, "1:512", "1:1", batch=256, page=64, name="attn_256_document"),
        # five drafted tokens of each of 16 requests checked at once, smaller heads
        _attn(8192, "5:600", "5:5", batch=16, hq=16, hkv=2, d=64, page=32,
              name="attn_16_drafts"),
        # decoding requests beside prompts that are read in chunks
        _attn(1000, "1:2500", "1:512", batch=9, page=32, pad=7, name="attn_chunks"),
        # four images drawn at once after one prompt, each seeing all of itself
        _attn(333, "1024:1024", "1024:1024", batch=4, page=64, causal=False,
              name="attn_4_images"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_parts(rng, d):
    """(parts, pairs) for heads of d."""
    pairs = rng.choice(["halves", "neighbours"])
    what = rng.choice(["whole", "whole", "part", "axes"])
    if what == "axes" and d % 64 == 0:
        return "0:%d:0,%d:%d:1,%d:%d:2" % (d // 2, d // 2, d // 4, 3 * d // 4, d // 4), pairs
    if what == "part":
        return "%d:%d:0" % (rng.choice([0, 8]), 2 * rng.randint(1, (d - 8) // 2)), pairs
    return "0:%d:0" % d, pairs


def draw(rng):
    kind = rng.choice(["rope", "append", "attn", "attn", "attn", "attn"])
    scaling = rng.choice(["none", "linear", "ntk", "yarn", "bands"])
    at = rng.choice([0, _log_int(rng, 1, 4000000)])
    if kind == "rope":
        d = rng.choice([32, 64, 80, 96, 128])
        parts, pairs = _draw_parts(rng, d)
        return _rope(_log_int(rng, 1, 4224), heads=rng.choice([1, 5, 8, 32]), d=d, parts=parts,
                     pairs=pairs, scaling=scaling, at=at, inverse=rng.random() < 0.3,
                     fused=rng.random() < 0.5)
    if kind == "append":
        d = rng.choice([32, 64, 128, 128])
        parts, pairs = _draw_parts(rng, d)
        hkv = rng.choice([1, 2, 8])
        return _append(_log_int(rng, 1, 4224), hq=hkv * rng.choice([0, 1, 4]), hkv=hkv, d=d,
                       page=rng.choice([16, 32, 64, 256]), parts=parts, pairs=pairs,
                       scaling=scaling, at=at, pad=rng.choice([0, 0, 3]))
    hq, hkv, d = rng.choice([(32, 8, 128), (32, 8, 128), (32, 8, 128), (16, 2, 64), (8, 8, 64),
                             (12, 4, 32), (10, 1, 128)])
    heads = dict(hq=hq, hkv=hkv, d=d, page=rng.choice([16, 32, 64, 256]),
                 pad=rng.choice([0, 0, 4]))
    what = rng.choice(["decode", "decode", "decode", "long", "drafts", "chunks", "images"])
    prefix = rng.choice([0, _log_int(rng, 16, 16384), _log_int(rng, 16, 16384)])
    if what == "long":
        return _attn(0, "%d:%d" % ((_log_int(rng, 4096, 131072),) * 2), "1:1", **heads)
    if what == "images":
        n = rng.randint(8, 32) * rng.randint(8, 32)
        return _attn(rng.choice([0, rng.randint(1, 500)]), "%d:%d" % (n, n), "%d:%d" % (n, n),
                     batch=rng.randint(1, 4), causal=False, **heads)
    if what == "chunks":
        return _attn(min(prefix, 2000), "1:%d" % _log_int(rng, 300, 3000),
                     "1:%d" % _log_int(rng, 8, 512), batch=rng.randint(1, 9), **heads)
    batch = _log_int(rng, 1, 128 if what == "decode" else 24)
    q = 1 if what == "decode" else rng.randint(2, 8)
    most = max(q, _log_int(rng, 1, min(4096, 131072 // batch)))
    return _attn(prefix, "%d:%d" % (q, most), "%d:%d" % (q, q), batch=batch, **heads)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _spread(text, n):
    """n whole numbers of the range "lo:hi", spread by the golden ratio."""
    lo, hi = (int(t) for t in text.split(":"))
    return [lo + int((hi - lo + 1) * ((i + 1) * 0.6180339887498949 % 1.0)) for i in range(n)]


def _lengths(case):
    """(own keys, queries) of each sequence; a query's own key is among them."""
    q = _spread(case["queries"], case["batch"])
    return [max(a, b) for a, b in zip(_spread(case["own"], case["batch"]), q)], q


def _parts(case):
    return [tuple(int(v) for v in t.split(":")) for t in case["parts"].split(",")]


def _freqs(width, theta, scaling):
    """(radians per position of each pair, what cosine and sine are times)."""
    h = width // 2
    f = [theta ** (-2.0 * i / width) for i in range(h)]
    if scaling == "linear":
        f = [v / FACTOR for v in f]
    elif scaling == "ntk":
        t = theta * FACTOR ** (width / (width - 2.0)) if width > 2 else theta
        f = [t ** (-2.0 * i / width) for i in range(h)]
    elif scaling == "yarn":
        at = [width * math.log(TRAINED / (turns * 2 * math.pi)) / (2 * math.log(theta))
              for turns in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), width - 1)
        ramp = [min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0) for i in range(h)]
        f = [v * (1 - r) + v / FACTOR * r for v, r in zip(f, ramp)]
        return f, 0.1 * math.log(FACTOR) + 1.0
    elif scaling == "bands":
        low, high = 1.0, 4.0                       # turns within the trained context
        for i, v in enumerate(f):
            turns = TRAINED * v / (2 * math.pi)
            mix = min(max((turns - low) / (high - low), 0.0), 1.0)
            f[i] = (1 - mix) * v / FACTOR + mix * v
    return f, 1.0


class _Rand:
    """Seeded values on the GPU, the same for prepare() and exact()."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def bf16(self, *shape, std=1.0):
        return torch.empty(*shape, dtype=BF16, device="cuda").normal_(0.0, std, generator=self.g)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda").to(I32)


def _positions(case, r):
    """[axes][tokens]: a text's positions, or an image's t, h and w."""
    n, axes = case["tokens"], 1 + max(a for _, _, a in _parts(case))
    pos = torch.arange(n, device="cuda") + case["at"]
    if axes == 1:
        return pos.to(I32)[None].contiguous()
    side = max(1, int(math.sqrt(n)))
    i = torch.arange(n, device="cuda")
    return torch.stack([case["at"] + i // (side * side), i // side % side, i % side]).to(I32)


def _inputs(case, seed):
    r = _Rand(seed)
    d, kind = case["d"], case["kind"]
    if kind == "rope":
        n, h = case["tokens"], case["heads"]
        x = r.bf16(n, h * d + (2 * d if case["fused"] else 0))
        return dict(x=x[:, :h * d].unflatten(1, (h, d)), pos=_positions(case, r))
    hkv, page = case["hkv"], case["page"]
    if kind == "append":
        n, hq = case["tokens"], case["hq"]
        qkv = r.bf16(n, (hq + 2 * hkv) * d).unflatten(1, (hq + 2 * hkv, d))
        pages = -(-n // page) + 3
        slot = r.order(pages)[:, None] * page + torch.arange(page, device="cuda", dtype=I32)
        slot = slot.flatten()[3:n + 3].contiguous()
        if case["pad"]:
            slot[-case["pad"]:] = -1
        return dict(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:], slot=slot,
                    pos=_positions(case, r), kp=r.bf16(pages, hkv, page, d),
                    vp=r.bf16(pages, hkv, page, d))
    lens, nq = _lengths(case)
    first = -(-case["prefix"] // page)
    each = [-(-n // page) for n in lens]
    pages = first + sum(each) + 3
    order = r.order(pages)
    table = torch.zeros(case["batch"], max(each), dtype=I32, device="cuda")
    at = first
    for b, n in enumerate(each):
        table[b, :n] = order[at:at + n]
        at += n
    start = [0]
    for n in nq:
        start.append(start[-1] + n)
    return dict(q=r.bf16(start[-1] + case["pad"], case["hq"], d, std=1.5),
                kp=r.bf16(pages, hkv, page, d), vp=r.bf16(pages, hkv, page, d),
                prefix_table=order[:first].contiguous(), table=table,
                kv_len=torch.tensor(lens, dtype=I32, device="cuda"),
                q_start=torch.tensor(start, dtype=I32, device="cuda"))


def _handles(case, s):
    """What a program keeps beside its tensors: the rotation, the cache, the
    step's batch (one for all layers)."""
    u = _lib()
    if case["kind"] != "attn":
        parts, scale = [], 1.0
        for start, width, axis in _parts(case):
            f, sc = u.rope_freqs(width, THETA[axis], case["scaling"] if axis == 0 else "none",
                                 factor=FACTOR, trained=TRAINED)
            scale = sc if axis == 0 else scale
            parts.append((f.cuda(), start, axis))
        s["rope"] = u.Rope(parts, neighbours=case["pairs"] == "neighbours", scale=scale)
    if case["kind"] != "rope":
        s["kv"] = u.PagedKV(s["kp"], s["vp"])
    if case["kind"] == "attn":
        lens, nq = _lengths(case)
        s["batch_"] = u.PagedBatch(s["kv_len"], s["table"], q_start=s["q_start"], max_q=max(nq),
                                   max_kv=max(lens), prefix_table=s["prefix_table"],
                                   prefix_len=case["prefix"])


def prepare(case, seed):
    s = dict(case, **_inputs(case, seed))
    if case["kind"] == "rope":
        s["y"] = torch.empty(case["tokens"], case["heads"], case["d"], dtype=BF16, device="cuda")
    else:
        s["out"] = torch.zeros_like(s["q"], memory_format=torch.contiguous_format)
    if case["kind"] != "attn":
        s["turn"] = []
        for start, width, axis in _parts(case):
            f, scale = _freqs(width, THETA[axis], case["scaling"] if axis == 0 else "none")
            s["turn"].append((torch.tensor(f, dtype=F64, device="cuda"), start, axis))
            s["by"] = scale if axis == 0 else s["by"]
    if own:
        _handles(case, s)
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def _turn(s, x, pos):
    """x [tokens][heads][d] with its parts turned, in f32."""
    x = x.float()
    y = x.clone()
    for f, start, axis in s["turn"]:
        h = f.numel()
        angle = pos[axis].double()[:, None] * f                     # [tokens][pairs]
        c = (torch.cos(angle) * s["by"]).float()[:, None]
        n = (torch.sin(angle) * s["by"]).float()[:, None]
        n = -n if s.get("inverse") else n
        if s["pairs"] == "halves":
            i, j = slice(start, start + h), slice(start + h, start + 2 * h)
        else:
            i, j = slice(start, start + 2 * h, 2), slice(start + 1, start + 2 * h, 2)
        a, b = x[..., i], x[..., j]
        y[..., i] = a * c - b * n
        y[..., j] = b * c + a * n
    return y.to(BF16)


def _append_plain(s):
    live = s["slot"] >= 0
    at = s["slot"][live].long()
    page, off = at // s["page"], at % s["page"]
    s["kp"][page, :, off] = _turn(s, s["k"], s["pos"])[live]
    s["vp"][page, :, off] = s["v"][live]
    if s["hq"]:
        s["out"][live] = _turn(s, s["q"], s["pos"])[live]


def _attend(s):
    hq, hkv, d, P = s["hq"], s["hkv"], s["d"], s["prefix"]
    lens, nq = _lengths(s)
    B, G, T, mq, most = s["batch"], hq // hkv, sum(nq), max(nq), max(lens)
    q = s["q"][:T].float().view(T, hkv, G, d) * (1.0 / math.sqrt(d))
    # queries padded to [sequences][most queries], and each query's place there
    start = s["q_start"].long()
    i = torch.arange(mq, device="cuda")
    count = start[1:] - start[:-1]
    token = (start[:-1, None] + i).clamp(max=T - 1)
    valid = i < count[:, None]
    place = valid.flatten().nonzero().flatten()                      # [T]
    kv = s["kv_len"].long()[:, None, None]
    key = torch.arange(most, device="cuda")
    seen = (key < kv).expand(B, mq, most)
    if s["causal"]:
        seen = seen & (key <= kv - count[:, None, None] + i[:, None])
    qp = q[token].permute(0, 2, 1, 3, 4).reshape(B, hkv, mq * G, d)

    def pages(pool, table, n):
        t = pool[table.long()]                                       # [..][np][hkv][page][d]
        return t.transpose(-4, -3).flatten(-3, -2)[..., :n, :].float()

    def rows(t):                                                     # -> [hkv][T * G][..]
        t = t.view(B, hkv, mq, G, -1).transpose(1, 2).reshape(B * mq, hkv, G, t.shape[-1])
        return t[place].transpose(0, 1).reshape(hkv, T * G, -1)

    so = qp @ pages(s["kp"], s["table"], most).transpose(-1, -2)     # [B][hkv][mq * G][most]
    so = so.masked_fill(~seen[:, None, :, None].expand(B, hkv, mq, G, most).flatten(2, 3),
                        -math.inf)
    qf = q.transpose(0, 1).reshape(hkv, T * G, d)
    m = rows(so.amax(-1, keepdim=True))
    if P:
        sp = qf @ pages(s["kp"], s["prefix_table"], P).transpose(-1, -2)
        m = torch.maximum(m, sp.amax(-1, keepdim=True))
    m = m.clamp(min=-1e30)
    mp = torch.zeros(B * mq, hkv, G, device="cuda")
    mp[place] = m.view(hkv, T, G).transpose(0, 1)
    mp = mp.view(B, mq, hkv, G).transpose(1, 2).reshape(B, hkv, mq * G, 1)
    po = torch.exp(so - mp)
    total = rows(po.sum(-1, keepdim=True))
    o = rows(po @ pages(s["vp"], s["table"], most))
    if P:
        pp = torch.exp(sp - m)
        total = total + pp.sum(-1, keepdim=True)
        o = o + pp @ pages(s["vp"], s["prefix_table"], P)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).to(BF16)
    s["out"][:T] = o.view(hkv, T, G, d).transpose(0, 1).reshape(T, hq, d)


def _run_own(s):
    o, kind = _ops(), s["kind"]
    if kind == "rope":
        o.rope(s["x"], s["pos"], s["rope"], s["y"], inverse=s["inverse"])
        return s["y"]
    if kind == "append":
        has = s["hq"] > 0
        o.paged_append(s["kv"], s["k"], s["v"], s["slot"], pos=s["pos"], rope=s["rope"],
                       q=s["q"] if has else None, q_out=s["out"] if has else None)
        return dict(k=s["kp"], v=s["vp"], q=s["out"] if has else None)
    o.paged_attention(s["kv"], s["batch_"], s["q"], s["out"], causal=s["causal"])
    return s["out"]


def run(s):
    if own:
        return _run_own(s)
    if s["kind"] == "rope":
        return _turn(s, s["x"], s["pos"])
    if s["kind"] == "append":
        _append_plain(s)
        return dict(k=s["kp"], v=s["vp"], q=s["out"] if s["hq"] else None)
    _attend(s)
    return s["out"]


# ---------------------------------------------------------------------------
# The definition in 64 bits, and the work of a pass
# ---------------------------------------------------------------------------

def _exact_turn(case, x, pos, back):
    """Every pair as a complex number, times scale * e^(i angle)."""
    out = x.to(F64)
    for start, width, axis in _parts(case):
        f, _ = _freqs(width, THETA[axis], case["scaling"] if axis == 0 else "none")
        by = _freqs(_parts(case)[0][1], THETA[0], case["scaling"])[1]
        angle = torch.outer(pos[axis].to(F64), torch.tensor(f, dtype=F64, device="cuda"))
        w = torch.polar(torch.full_like(angle, by), -angle if back else angle)[:, None]
        part = out[..., start:start + width]
        if case["pairs"] == "halves":
            z = torch.complex(part[..., :width // 2].contiguous(),
                              part[..., width // 2:].contiguous()) * w
            out[..., start:start + width] = torch.cat([z.real, z.imag], -1)
        else:
            z = torch.view_as_complex(part.unflatten(-1, (width // 2, 2)).contiguous()) * w
            out[..., start:start + width] = torch.view_as_real(z).flatten(-2)
    return out


def exact(case, seed):
    t = _inputs(case, seed)
    kind = case["kind"]
    if kind == "rope":
        return _exact_turn(case, t["x"], t["pos"], case["inverse"])
    if kind == "append":
        k, v = t["kp"].to(F64), t["vp"].to(F64)
        kr = _exact_turn(case, t["k"], t["pos"], False)
        q = torch.zeros(t["q"].shape, dtype=F64, device="cuda")
        live = (t["slot"] >= 0).nonzero().flatten()
        if case["hq"]:
            q[live] = _exact_turn(case, t["q"], t["pos"], False)[live]
        # the pools seen as one slot after the other
        for pool, new in ((k, kr), (v, t["v"].to(F64))):
            flat = pool.transpose(1, 2).flatten(0, 1).clone()
            flat[t["slot"][live].long()] = new[live]
            pool.copy_(flat.unflatten(0, (-1, case["page"])).transpose(1, 2))
        return dict(k=k, v=v, q=q if case["hq"] else None)
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    lens, nq = _lengths(case)
    out = torch.zeros(t["q"].shape, dtype=F64, device="cuda")
    first, at = t["prefix_table"].long(), 0
    for b in range(case["batch"]):
        own_pages = t["table"][b, :-(-lens[b] // page)].long()
        q = t["q"][at:at + nq[b]].to(F64)
        sees = torch.ones(nq[b], case["prefix"] + lens[b], dtype=torch.bool, device="cuda")
        if case["causal"]:
            sees = torch.tril(sees, case["prefix"] + lens[b] - nq[b])
        for h in range(hkv):
            kv = []
            for pool in (t["kp"], t["vp"]):
                kv.append(torch.cat([pool[first, h].flatten(0, 1)[:case["prefix"]],
                                     pool[own_pages, h].flatten(0, 1)[:lens[b]]]).to(F64))
            qh = q[:, h * (hq // hkv):(h + 1) * (hq // hkv)].transpose(0, 1)
            score = (qh @ kv[0].t() / math.sqrt(d)).masked_fill(~sees, -math.inf)
            out[at:at + nq[b], h * (hq // hkv):(h + 1) * (hq // hkv)] = \
                (torch.softmax(score, -1) @ kv[1]).transpose(0, 1)
        at += nq[b]
    return out


def work(case):
    d, kind = case["d"], case["kind"]
    if kind == "attn":
        lens, nq = _lengths(case)
        pairs = sum(n * (case["prefix"] + a) - (n * (n - 1) // 2 if case["causal"] else 0)
                    for a, n in zip(lens, nq))
        keys = case["prefix"] + sum(lens)
        return dict(bytes=4 * sum(nq) * case["hq"] * d + 4 * keys * case["hkv"] * d
                    + 4 * (-(-keys // case["page"])), flops=4 * case["hq"] * d * pairs)
    turned = sum(w for _, w, _ in _parts(case))
    axes = 1 + max(a for _, _, a in _parts(case))
    if kind == "rope":
        n, h = case["tokens"], case["heads"]
        return dict(bytes=4 * n * h * d + 4 * n * axes, flops=3 * n * h * turned)
    n = case["tokens"] - case["pad"]
    h = case["hq"] + case["hkv"]
    return dict(bytes=4 * n * (h + case["hkv"]) * d + 4 * n * (axes + 1), flops=3 * n * h * turned)
