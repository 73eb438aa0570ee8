"""One step of verifying drafted tokens through a decoder layer, as a serving program
calls it: the layer's new queries and keys rotated while the keys and values go into the
int8 paged cache, attention of a tree of drafted tokens over it, the accepted tokens moved
to their places, and a mixture-of-experts feed-forward with MXFP4 weights.

`listed()` holds the named cases, `draw(rng)` makes further ones of the same
ranges.  With `own` false, `run` computes an operator in elementary torch
operations; with `own` true it makes the calls of quixicore_hip.  `exact` gives
the same outputs from the definitions in 64 bits.

Kinds
  rotate   q and k of a batch rotated by their positions; q comes back, k and v go into the
           cache; the pages written to are read back
  tree     softmax(scale q k^T) v of drafted tokens: each sees its sequence's context and
           those of its drafted tokens that its mask names
  keep     the accepted ones of the drafted tokens close up behind the context; the pages
           from the context's last on are read back
  experts  y = sum_k p_k down_e(act(gate_e x) * up_e x) over the top k experts e of a router
"""
from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BASE = 10000.0


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------
def listed():
    return [
        # one decoding step of 64 requests, a token each: the usual layout of a 4096-wide layer
        {"name": "rotate_step_bf16", "kind": "rotate", "type": "bf16", "seqs": 64, "new": 1,
         "kv": 2048, "heads": 32, "kv_heads": 8, "head_dim": 128, "rotary": 128,
         "interleaved": False, "positions": 32768, "page": 64, "draft": False, "spare": 0},
        # trees of drafted tokens at their depths' positions, half of each head rotated,
        # rows behind the last sequence
        {"name": "rotate_draft_f16", "kind": "rotate", "type": "f16", "seqs": 12, "new": 33,
         "kv": 4000, "heads": 40, "kv_heads": 8, "head_dim": 128, "rotary": 64,
         "interleaved": True, "positions": 8192, "page": 16, "draft": True, "spare": 3},
        # three prompts, the longest of 4096 tokens, f32 projections
        {"name": "rotate_prompts_f32", "kind": "rotate", "type": "f32", "seqs": 3, "new": 4096,
         "kv": 6000, "heads": 32, "kv_heads": 8, "head_dim": 128, "rotary": 128,
         "interleaved": False, "positions": 8192, "page": 64, "draft": False, "spare": 0},
        # one request after a short prompt, eight drafted tokens
        {"name": "tree_one_bf16", "kind": "tree", "type": "bf16", "seqs": 1, "new": 8, "kv": 600,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 32, "window": 0, "padded": False,
         "spare": 0},
        # one request with a long context and a wide tree
        {"name": "tree_wide_bf16", "kind": "tree", "type": "bf16", "seqs": 1, "new": 64,
         "kv": 32768, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "window": 0,
         "padded": False, "spare": 0},
        # a batch of 16 requests with contexts up to 16384
        {"name": "tree_batch_f16", "kind": "tree", "type": "f16", "seqs": 16, "new": 24,
         "kv": 16384, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "window": 0,
         "padded": False, "spare": 0},
        # odd heads in a sliding window, trees padded with rows that see no drafted token
        {"name": "tree_window_f32", "kind": "tree", "type": "f32", "seqs": 5, "new": 33, "kv": 5000,
         "heads": 14, "kv_heads": 2, "head_dim": 80, "page": 16, "window": 1000, "padded": True,
         "spare": 3},
        # short drafts of a small batch: a token or two moves
        {"name": "keep_step", "kind": "keep", "type": "bf16", "seqs": 16, "new": 8, "kv": 2048,
         "kv_heads": 8, "head_dim": 128, "page": 64},
        # wide trees of many requests, paths over several pages
        {"name": "keep_wide", "kind": "keep", "type": "f16", "seqs": 64, "new": 128, "kv": 4000,
         "kv_heads": 8, "head_dim": 128, "page": 16},
        # one token through many small experts
        {"name": "experts_one_bf16", "kind": "experts", "type": "bf16", "tokens": 1, "experts": 64,
         "top": 8, "dim": 2048, "inter": 1024, "normalize": True, "gelu": False, "residual": True},
        # a short draft through no round sizes
        {"name": "experts_odd_f32", "kind": "experts", "type": "f32", "tokens": 17, "experts": 30,
         "top": 3, "dim": 2752, "inter": 1376, "normalize": False, "gelu": True,
         "residual": False},
        # the drafted tokens of a batch through few wide experts
        {"name": "experts_draft_bf16", "kind": "experts", "type": "bf16", "tokens": 64,
         "experts": 8, "top": 2, "dim": 4096, "inter": 14336, "normalize": True, "gelu": False,
         "residual": True},
    ]


def _log(rng, low, high, step=1):
    """A size whose logarithm is uniform, rounded to a multiple of step."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(step, int(round(v / step)) * step)


def draw(rng):
    kind = rng.choice(["rotate", "tree", "tree", "tree", "keep", "experts", "experts"])
    typ = rng.choice(["f32", "f16", "bf16"])
    hd = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    if kind == "rotate":
        kvh, group = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 4, 4, 7])
        draft = rng.random() < 0.4
        new = _log(rng, 2, 128) if draft else 1 if rng.random() < 0.5 else _log(rng, 2, 4096)
        seqs = _log(rng, 1, max(1, min(64, 10000 // new)))
        kv = new + _log(rng, 1, 4000)
        return {"kind": kind, "type": typ, "seqs": seqs, "new": new, "kv": kv,
                "heads": kvh * group, "kv_heads": kvh, "head_dim": hd,
                "rotary": rng.choice([hd, hd, hd // 2, hd // 4]), "interleaved": rng.random() < 0.5,
                "positions": kv + _log(rng, 1, 32768), "page": page, "draft": draft,
                "spare": rng.choice([0, 0, 5])}
    if kind == "tree":
        kvh, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 4, 7, 8, 16])
        new = _log(rng, 1, 128)
        kv = new + _log(rng, 1, 32768)
        most = min((1 << 33) // (new * kv * kvh * group * hd), (1 << 29) // (kv * kvh * hd), 64)
        return {"kind": kind, "type": typ, "seqs": _log(rng, 1, max(1, most)), "new": new, "kv": kv,
                "heads": kvh * group, "kv_heads": kvh, "head_dim": hd, "page": page,
                "window": _log(rng, 16, kv) if rng.random() < 0.25 else 0,
                "padded": rng.random() < 0.3, "spare": rng.choice([0, 0, 5])}
    if kind == "keep":
        new = _log(rng, 1, 128)
        return {"kind": kind, "type": typ, "seqs": _log(rng, 1, 64), "new": new,
                "kv": new + _log(rng, 1, 4000), "kv_heads": rng.choice([1, 2, 4, 5, 8]),
                "head_dim": hd, "page": page}
    experts = rng.choice([4, 8, 8, 30, 64, 64, 128])
    dim = _log(rng, 256, 8192, 32)
    inter = min(_log(rng, 128, 14336, 32), max(4, (1 << 29) // (experts * dim * 32)) * 32)
    top = rng.randint(1, min(8, experts))
    tokens = 1 if rng.random() < 0.25 else _log(rng, 2, 512)
    return {"kind": kind, "type": typ, "tokens": max(1, min(tokens, (1 << 32) // (top * dim * inter))),
            "experts": experts, "top": top, "dim": dim, "inter": inter,
            "normalize": rng.random() < 0.5, "gelu": rng.random() < 0.3,
            "residual": rng.random() < 0.5}


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------
class _Gen:
    """Seeded tensors of one case on the GPU."""

    def __init__(self, seed):
        self.dev = torch.device("cuda:0")
        self.g = torch.Generator(device=self.dev)
        self.g.manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device=self.dev)

    def outliers(self, *shape):
        """N(0, 1) with 0.1% of the entries 20 times larger."""
        x = self.normal(*shape)
        hit = torch.rand(*shape, generator=self.g, device=self.dev) < 0.001
        return torch.where(hit, x * 20.0, x)

    def bytes(self, *shape):
        return torch.randint(0, 256, shape, generator=self.g, device=self.dev, dtype=torch.uint8)

    def channels(self, *shape):
        """N(0, 1) times a magnitude for each of the last dimension's channels."""
        return self.normal(*shape) * torch.exp(0.5 * self.normal(shape[-1]))


def _lengths(case):
    """New and total tokens of each sequence: from a quarter of the largest, one at
    it, spread by the multiples of irrational numbers; in a batch of trees the last
    but the first sequence has no context."""
    def spread(most, step):
        return [max(1, round(most * (1.0 - 0.75 * math.modf(i * step)[0]))) for i in range(case["seqs"])]

    new = spread(case["new"], 0.6180339887)
    kv = [max(a, b) for a, b in zip(new, spread(case["kv"], 0.7548776662))]
    if case["kind"] == "tree" and case["seqs"] > 1:
        kv[-1] = new[-1]
    return new, kv


def _accepted(case):
    """How many drafted tokens of each sequence are accepted: none to half of them."""
    return [round(0.5 * n * math.modf(0.8 + i * 0.5698402910)[0]) for i, n in enumerate(_lengths(case)[0])]


def _parents(rng, n):
    """A tree of n drafted tokens: each node's parent among the few before it, -1 a root."""
    return [max(-1, i - 1 - int(rng.expovariate(0.4))) for i in range(n)]


def _cache(case, g):
    """Page table, lengths and a filled cache of a batch of sequences."""
    page, h, d = case["page"], case["kv_heads"], case["head_dim"]
    new, kv = _lengths(case)
    columns = -(-case["kv"] // page)
    pages = case["seqs"] * columns
    table = torch.randperm(pages, generator=g.g, device=g.dev).to(torch.int32)
    start = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device=g.dev)
    s = {"new": torch.tensor(new, device=g.dev), "kv": torch.tensor(kv, dtype=torch.int32, device=g.dev),
         "start": start, "table": table.view(case["seqs"], columns), "max_kv": case["kv"],
         "max_new": case["new"], "tokens": sum(new) + case.get("spare", 0),
         "status": torch.zeros(1, dtype=torch.int32, device=g.dev)}
    for name in ("k", "v"):
        x = g.channels(pages, h, page, d) if name == "k" else g.outliers(pages, h, page, d)
        scale = x.abs().amax((2, 3)) / 127.0
        s[name + "_codes"] = (x / scale[:, :, None, None]).round_().to(torch.int8)
        s[name + "_scales"] = scale
    return s


def _read_back(s, case, end):
    """A batch that spans each sequence from its first touched page's first slot to `end`."""
    new, kv = _lengths(case)
    first = [(b - a) // case["page"] * case["page"] for a, b in zip(new, kv)]
    rows = [e - f for f, e in zip(first, end)]
    dev = s["start"].device
    s["back"] = torch.tensor([0] + list(np.cumsum(rows)), dtype=torch.int32, device=dev)
    s["back_tokens"], s["back_max"] = max(1, sum(rows)), case["new"] + case["page"]


def _trees(s, case, seed):
    """The drafted tokens' parents, masks (32-bit words) and positions."""
    rng = random.Random(seed)
    new, kv = _lengths(case)
    words = -(-case["new"] // 32)
    masks, positions = [], []
    for n, length in zip(new, kv):
        parents = _parents(rng, n)
        bits, depth = [], []
        for i, p in enumerate(parents):
            bits.append((1 << i) | (bits[p] if p >= 0 else 0))
            depth.append(depth[p] + 1 if p >= 0 else 0)
        if case.get("padded"):
            # the last rows of a draft that came out short: they see no drafted token
            for i in range(n - n // 8, n):
                bits[i] = 0
        masks += bits
        positions += [length - n + d for d in depth]
    spare = s["tokens"] - len(masks)
    data = b"".join(b.to_bytes(4 * words, "little") for b in masks + [0] * spare)
    dev = s["start"].device
    s["mask"] = torch.from_numpy(np.frombuffer(data, dtype=np.int32).reshape(-1, words).copy()).to(dev)
    s["positions"] = torch.tensor(positions + [0] * spare, dtype=torch.int32, device=dev)


_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _weights(g, *shape):
    """Random MXFP4 matrices [...][k], about N(0, 0.02^2): codes of a normal value that makes
    a block's largest about 5, the even element in the low half of its byte, and biased
    exponents of each 32."""
    z = math.sqrt(2.0) * torch.erfinv(2.0 * (torch.arange(256, dtype=torch.float64) + 0.5) / 256.0 - 1.0)
    near = (z.abs()[:, None] * 2.0 - torch.tensor(_GRID, dtype=torch.float64)).abs().argmin(1)
    code = (near + 8 * (z < 0)).to(torch.uint8).to(g.dev)
    half = shape[:-1] + (shape[-1] // 2,)
    codes = torch.empty(half, dtype=torch.uint8, device=g.dev)
    for c in codes:                                # a matrix at a time
        c.copy_(code[g.bytes(*c.shape).int()] | (code[g.bytes(*c.shape).int()] << 4))
    scales = 127 - 7 + (g.bytes(*shape[:-1], shape[-1] // 32) % 3).to(torch.int16) - 1
    return codes, scales.to(torch.uint8)


def prepare(case, seed):
    g = _Gen(seed)
    kind, typ = case["kind"], TORCH[case["type"]]
    s = {"case": case}
    if kind == "experts":
        e, d, n, t = case["experts"], case["dim"], case["inter"], case["tokens"]
        s["gate_up"], s["gate_up_scales"] = _weights(g, e, 2 * n, d)
        s["down"], s["down_scales"] = _weights(g, e, d, n)
        s.update(x=g.outliers(t, d).to(typ), router=(2.5 / math.sqrt(d) * g.normal(e, d)).to(typ),
                 bias=0.5 * g.normal(e), residual=g.normal(t, d).to(typ) if case["residual"] else None)
        return s
    s.update(_cache(case, g))
    h, d, t = case["kv_heads"], case["head_dim"], s["tokens"]
    if kind == "rotate":
        # one projection's rows: q, k and v heads side by side, louder than what the pages
        # hold, so that some scales grow
        hq = case["heads"]
        rows = torch.cat([1.5 * g.normal(t, hq, d), 1.2 * g.channels(t, h, d), 1.2 * g.outliers(t, h, d)], 1)
        rows = rows.to(typ)
        s.update(q=rows[:, :hq], k=rows[:, hq: hq + h], v=rows[:, hq + h:],
                 out=torch.zeros(t, hq, d, dtype=typ, device=g.dev))
        _trees(s, case, seed)
        if not case["draft"]:
            s["positions"] = None
        p = torch.arange(case["positions"], device=g.dev, dtype=torch.float64)
        w = _BASE ** (-2.0 * torch.arange(case["rotary"] // 2, device=g.dev, dtype=torch.float64) / case["rotary"])
        angle = p[:, None] * w[None, :]
        s["cosine"], s["sine"] = angle.cos().float(), angle.sin().float()
        _read_back(s, case, _lengths(case)[1])
    elif kind == "tree":
        _trees(s, case, seed)
        s.update(q=(1.5 * g.normal(t, case["heads"], d)).to(typ),
                 out=torch.zeros(t, case["heads"], d, dtype=typ, device=g.dev))
    else:
        rng = random.Random(seed)
        paths = [sorted(rng.sample(range(n), c)) for n, c in zip(_lengths(case)[0], _accepted(case))]
        most = max(1, max(len(p) for p in paths))
        kept = torch.tensor([p + [0] * (most - len(p)) for p in paths], dtype=torch.int32)
        s.update(kept=kept.to(g.dev), count=torch.tensor(_accepted(case), dtype=torch.int32, device=g.dev))
        _read_back(s, case, [b - a + n for a, b, n in zip(*_lengths(case), _accepted(case))])
    return s


# --------------------------------------------------------------------------
# The plain forms
# --------------------------------------------------------------------------
def _places(s, start, count, kv):
    """For the tokens of ragged sequences that end at each one's length: the
    sequence, position and page of each."""
    t = torch.arange(count, device=start.device)
    seq = torch.searchsorted(start[1:].to(torch.int64), t, right=True)
    last = kv.to(torch.int64)[seq] - start[1:].to(torch.int64)[seq]
    position = last + t
    page = s["case"]["page"]
    return seq, position, s["table"].to(torch.int64)[seq, position // page], position % page


def _rotated(s, x, position):
    """Heads [tokens][heads][d] in 32 bits, turned by the tokens' positions."""
    case = s["case"]
    r = case["rotary"]
    c, n = s["cosine"][position][:, None, :], s["sine"][position][:, None, :]
    x = x.float()
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * c - b * n, b * c + a * n], dim=-1).flatten(-2)
    else:
        a, b = x[..., : r // 2], x[..., r // 2: r]
        y = torch.cat([a * c - b * n, b * c + a * n], dim=-1)
    return torch.cat([y, x[..., r:]], dim=-1)


def _back(s, kv):
    """The values of the pages written to, and all scales."""
    _, _, bp, bs = _places(s, s["back"], s["back_tokens"], kv)
    typ = TORCH[s["case"]["type"]]
    return [(s[n + "_codes"][bp, :, bs].float() * s[n + "_scales"][bp][:, :, None]).to(typ) for n in ("k", "v")] + [
        s["k_scales"], s["v_scales"]]


def _rotate_plain(s):
    case = s["case"]
    page, h = case["page"], case["kv_heads"]
    count = s["tokens"] - case["spare"]
    seq, position, pid, slot = _places(s, s["start"], count, s["kv"])
    turn = position if s["positions"] is None else s["positions"][:count].to(torch.int64)
    s["out"][:count] = _rotated(s, s["q"][:count], turn).to(s["out"].dtype)
    first = (s["kv"].to(torch.int64) - s["new"])[seq]
    touched, inverse = torch.unique(pid, return_inverse=True)
    # slots of a touched page that were full before
    full = torch.zeros(touched.numel(), dtype=torch.int64, device=pid.device)
    full[inverse] = (first - position // page * page).clamp(min=0)
    for name, x in (("k", _rotated(s, s["k"][:count], turn)), ("v", s["v"][:count].float())):
        codes, scales = s[name + "_codes"], s[name + "_scales"]
        top = torch.zeros(touched.numel(), h, device=pid.device)
        top.scatter_reduce_(0, inverse[:, None].expand(-1, h), x.abs().amax(2), "amax")
        before = torch.where(full[:, None] > 0, scales[touched], 0.0)
        scale = torch.maximum(before, top * (1.0 / 127.0))
        scale = torch.where(scale < 2.0 ** -126, 0.0, scale)
        ratio = torch.where(scale > 0, before / scale, 0.0)
        inv = torch.where(scale > 0, 1.0 / scale, 0.0)
        old = codes[touched]
        moved = (old.float() * ratio[:, :, None, None]).round().to(torch.int8)
        keep = torch.arange(page, device=pid.device)[None, :] < full[:, None]
        codes[touched] = torch.where(keep[:, None, :, None], moved, old)
        scales[touched] = scale
        codes[pid, :, slot] = (x * inv[inverse][:, :, None]).round().clamp(-127, 127).to(torch.int8)
    return [s["out"]] + _back(s, s["kv"])


def _tree_plain(s):
    case = s["case"]
    page, h, d, g = case["page"], case["kv_heads"], case["head_dim"], case["heads"] // case["kv_heads"]
    n, most, kv = case["seqs"], case["new"], case["kv"]
    table = s["table"].to(torch.int64)
    count = s["tokens"] - case["spare"]
    seq, position, _, _ = _places(s, s["start"], count, s["kv"])
    index = torch.arange(count, device=table.device) - s["start"].to(torch.int64)[seq]
    q = torch.zeros(n, most, h, g, d, device=table.device)
    q[seq, index] = s["q"][:count].float().view(count, h, g, d)
    wide = table.shape[1] * page
    k, v = [(s[m + "_codes"][table].float() * s[m + "_scales"][table][..., None, None])
            .transpose(1, 2).reshape(n, h, wide, d)[:, :, :kv] for m in ("k", "v")]
    q = q.permute(0, 2, 3, 1, 4).reshape(n, h, g * most, d) * (1.0 / math.sqrt(d))
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).view(n, h, g, most, kv)
    # a row sees the context (in its window) and the drafted tokens of its mask
    j = torch.arange(kv, device=table.device)
    context = s["kv"].to(torch.int64) - s["new"]
    seen = (j[None, :] < context[:, None])[:, None, :].expand(n, most, kv)
    if case["window"]:
        at = torch.zeros(n, most, dtype=torch.int64, device=table.device)
        at[seq, index] = s["positions"][:count].to(torch.int64)
        seen = seen & (j > at[:, :, None] - case["window"])
    seen = seen.clone()
    bit = torch.arange(most, device=table.device)
    named = torch.zeros(n, most, most, dtype=torch.bool, device=table.device)
    named[seq, index] = (s["mask"][:count][:, bit // 32] >> (bit % 32)) & 1 != 0
    drafted = context[:, None] + bit[None, :]
    there = drafted < s["kv"][:, None]
    at = torch.where(there, drafted, kv - 1)[:, None, :].expand(n, most, most)
    seen |= torch.zeros(n, most, kv, device=table.device).scatter_add_(
        2, at, (named & there[:, None, :]).float()) > 0
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p.view(n, h, g * most, kv), v.contiguous()).view(n, h, g, most, d)
    y = y / torch.where(total == 0, 1.0, total)
    s["out"][:count] = y[seq, :, :, index].reshape(count, h * g, d).to(s["out"].dtype)
    return s["out"]


def _keep_plain(s):
    case = s["case"]
    page = case["page"]
    table, kept = s["table"].to(torch.int64), s["kept"].to(torch.int64)
    context = (s["kv"].to(torch.int64) - s["new"])[:, None]
    at = torch.arange(kept.shape[1], device=kept.device)[None, :]
    there = at < s["count"][:, None]
    seq = torch.arange(case["seqs"], device=kept.device)[:, None].expand_as(kept)[there]
    source, target = (context + kept)[there], (context + at)[there]
    from_page, to_page = table[seq, source // page], table[seq, target // page]
    across = from_page != to_page
    touched, inverse = torch.unique(to_page, return_inverse=True)
    full = torch.zeros(touched.numel(), dtype=torch.int64, device=kept.device)
    full[inverse] = (context[:, 0][seq] - target // page * page).clamp(min=0)
    slots = torch.arange(page, device=kept.device)[None, :] < full[:, None]
    length = (s["kv"] - s["new"] + s["count"]).to(torch.int32)
    for name in ("k", "v"):
        codes, scales = s[name + "_codes"], s[name + "_scales"]
        h = case["kv_heads"]
        scale = scales[touched].abs()
        came = torch.where(across[:, None], scales[from_page].abs(), 0.0)
        scale = scale.scatter_reduce(0, inverse[:, None].expand(-1, h), came, "amax")
        moved = codes[from_page, :, source % page].float()
        ratio = torch.where(scale[inverse] > 0, scales[from_page] / scale[inverse], 0.0)
        held = torch.where(scale > 0, scales[touched] / scale, 0.0)
        old = codes[touched]
        turned = (old.float() * held[:, :, None, None]).round().to(torch.int8)
        codes[touched] = torch.where(slots[:, None, :, None], turned, old)
        codes[to_page, :, target % page] = (moved * ratio[:, :, None]).round().to(torch.int8)
        scales[touched] = scale
    return _back(s, length) + [length]


def _values(codes, scales, dtype):
    """The matrix that MXFP4 codes and scales stand for."""
    both = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).to(torch.int32)
    grid = torch.tensor(_GRID + tuple(-v for v in _GRID), device=codes.device, dtype=dtype)
    step = ((scales.to(torch.int64) + 896) << 52).view(torch.float64).to(dtype)
    return (grid[both].view(*scales.shape, 32) * step[..., None]).view(both.shape)


def _chosen(s):
    """Each token's experts, largest logit first, and their shares; 64 bits, so that logits
    next to each other keep their order."""
    case = s["case"]
    logits = torch.matmul(s["x"].double(), s["router"].double().T.contiguous()) + s["bias"].double()
    value, index = torch.sort(logits, dim=1, descending=True, stable=True)
    value, index = value[:, : case["top"]], index[:, : case["top"]]
    whole = (value if case["normalize"] else logits)
    p = torch.exp(value - value[:, :1]) / torch.exp(whole - value[:, :1]).sum(1, keepdim=True)
    return index, p


def _act(case, a):
    if case["gelu"]:
        return 0.5 * a * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (a + 0.044715 * a * a * a)))
    return a / (1.0 + torch.exp(-a))


def _experts_plain(s):
    case = s["case"]
    index, share = _chosen(s)
    share = share.float()
    x = s["x"].float()
    y = torch.zeros_like(x) if s["residual"] is None else s["residual"].float()
    order = torch.sort(index.flatten(), stable=True)[1]
    counts = torch.bincount(index.flatten(), minlength=case["experts"]).tolist()
    at = 0
    for e, n in enumerate(counts):
        if n == 0:
            continue
        pairs = order[at: at + n]
        at += n
        token = pairs // case["top"]
        w = _values(s["gate_up"][e], s["gate_up_scales"][e], torch.float32)
        both = torch.matmul(x[token], w.T.contiguous())
        h = _act(case, both[:, : case["inter"]]) * both[:, case["inter"]:]
        w = _values(s["down"][e], s["down_scales"][e], torch.float32)
        y.index_add_(0, token, torch.matmul(h, w.T.contiguous()) * share.flatten()[pairs, None])
    return [y.to(s["x"].dtype), index.to(torch.int32), share]


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------
_library = None


def _qc():
    global _library
    if _library is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "quixicore-cpu_amd"))
        import quixicore_hip
        _library = quixicore_hip
    return _library


def _handles(s):
    """The cache, batch and layer descriptors that a serving program keeps for its buffers."""
    if "handles" not in s:
        qc = _qc()
        if s["case"]["kind"] == "experts":
            s["handles"] = qc.Mxfp4Moe(s["router"], s["gate_up"], s["gate_up_scales"], s["down"],
                                       s["down_scales"], bias=s["bias"])
            return s["handles"]
        cache = qc.Kv8Cache(s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"])
        s["handles"] = cache, qc.Kv8Batch(s["table"], s["start"], s["kv"], s["tokens"], s["max_new"],
                                          s["max_kv"])
    return s["handles"]


def _back_own(s, kv):
    qc = _qc()
    batch = qc.Kv8Batch(s["table"], s["back"], kv, s["back_tokens"], s["back_max"], s["max_kv"])
    k, v = qc.kv8_gather(s["handles"][0], batch, dtype=TORCH[s["case"]["type"]], dev_status=s["status"])
    return [k, v, s["k_scales"], s["v_scales"]]


def _run_own(s):
    qc, case = _qc(), s["case"]
    if case["kind"] == "experts":
        return list(qc.mxfp4_moe(_handles(s), s["x"], case["top"], normalize=case["normalize"],
                                 gelu_tanh=case["gelu"], residual=s["residual"]))
    cache, batch = _handles(s)
    if case["kind"] == "rotate":
        q = qc.kv8_rope_append(cache, batch, s["q"], s["k"], s["v"], s["cosine"], s["sine"],
                               positions=s["positions"], interleaved=case["interleaved"],
                               out=s["out"], dev_status=s["status"])
        return [q] + _back_own(s, s["kv"])
    if case["kind"] == "tree":
        return qc.kv8_tree_attention(cache, batch, s["q"], s["mask"], window=case["window"],
                                     positions=s["positions"] if case["window"] else None,
                                     out=s["out"], dev_status=s["status"])
    length = qc.kv8_keep(cache, batch, s["kept"], s["count"], dev_status=s["status"])
    return _back_own(s, length) + [length]


def run(s):
    if own:
        return _run_own(s)
    return {"rotate": _rotate_plain, "tree": _tree_plain, "keep": _keep_plain,
            "experts": _experts_plain}[s["case"]["kind"]](s)


# --------------------------------------------------------------------------
# What a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    size = 4 if case["type"] == "f32" else 2
    if kind == "experts":
        t, e, d, n = case["tokens"], case["experts"], case["dim"], case["inter"]
        # experts that tokens of independent choices hit
        hit = e * (1.0 - (1.0 - case["top"] / e) ** t)
        rows = 2 + bool(case["residual"])
        return {"bytes": hit * 3 * d * n * 17 / 32 + size * (rows * t * d + e * d),
                "flops": 6 * t * case["top"] * d * n + 2 * t * e * d}
    new, kv = (np.array(v, dtype=np.float64) for v in _lengths(case))
    h, d, page = case["kv_heads"], case["head_dim"], case["page"]
    tokens = float(new.sum())
    if kind == "rotate":
        back = float((kv - np.floor((kv - new) / page) * page).sum())
        hq, r = case["heads"], case["rotary"]
        # q in and out; new rows in; the touched pages' codes out; their values read back; table rows
        return {"bytes": 2 * size * tokens * hq * d + 2 * h * d * (size * tokens + back + size * back)
                + 4 * r * min(tokens, case["positions"]),
                "flops": 3 * tokens * (hq + h) * r + 4 * tokens * h * d}
    if kind == "keep":
        # accepted codes to and fro, values read back
        kept = np.array(_accepted(case), dtype=np.float64)
        back = float((kv - new + kept - np.floor((kv - new) / page) * page).sum())
        return {"bytes": 2 * h * d * (2 * float(kept.sum()) + back + size * back), "flops": 0}
    window = case["window"] or math.inf
    seen = float((new * (np.minimum(kv - new, window) + new / 3)).sum())
    read = float(np.minimum(kv, new + window).sum())
    return {"bytes": 2 * h * d * read + 2 * size * tokens * case["heads"] * d,
            "flops": 4 * seen * case["heads"] * d}


# --------------------------------------------------------------------------
# The same outputs in 64 bits
# --------------------------------------------------------------------------
def _exact_rotated(case, s, x, position):
    d, r = case["head_dim"], case["rotary"]
    x = x.double()
    y = x.clone()
    i = torch.arange(r // 2, device=x.device)
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + r // 2)
    angle = position.double()[:, None] * _BASE ** (-2.0 * i.double() / r)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None, :]
    z = torch.complex(x[..., first], x[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_rotate(case, s):
    page, start, kv, table = case["page"], s["start"].tolist(), s["kv"].tolist(), s["table"].tolist()
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=s["out"].device)
    scales = {n: s[n + "_scales"].double() for n in ("k", "v")}
    for i, length in enumerate(kv):
        a, b = start[i], start[i + 1]
        begin = length - (b - a)
        at = torch.arange(begin, length, device=out.device)
        if s["positions"] is not None:
            at = s["positions"][a:b]
        out[a:b] = _exact_rotated(case, s, s["q"][a:b], at)
        rows = {"k": _exact_rotated(case, s, s["k"][a:b], at), "v": s["v"][a:b].double()}
        for lo in range(begin // page * page, length, page):
            x, y = max(lo, begin), min(lo + page, length)
            pid = table[i][lo // page]
            for n in ("k", "v"):
                top = rows[n][x - begin: y - begin].abs().amax((0, 2)) / 127.0
                scales[n][pid] = torch.maximum(scales[n][pid], top) if x > lo else top
    return [out, None, None, scales["k"], scales["v"]]


def _exact_tree(case, s):
    page, h, d = case["page"], case["kv_heads"], case["head_dim"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=s["out"].device)
    start, kv = s["start"].tolist(), s["kv"].tolist()
    masks, places = s["mask"].tolist(), s["positions"].tolist()
    for i, length in enumerate(kv):
        rows = start[i + 1] - start[i]
        hide = torch.ones(rows, length, dtype=torch.bool)
        for r in range(rows):
            words = masks[start[i] + r]
            hide[r, : length - rows] = False
            if case["window"]:
                hide[r, : max(0, min(length - rows, places[start[i] + r] - case["window"] + 1))] = True
            for j in range(rows):
                if words[j // 32] >> (j % 32) & 1:
                    hide[r, length - rows + j] = False
        hide = hide.to(out.device)
        ids = s["table"][i, : -(-length // page)].to(torch.int64)
        k, v = [(s[m + "_codes"][ids].double() * s[m + "_scales"][ids].double()[..., None, None])
                .permute(1, 0, 2, 3).reshape(h, -1, d)[:, :length] for m in ("k", "v")]
        q = s["q"][start[i]: start[i + 1]].double().view(rows, h, -1, d)
        for c in range(h):
            z = torch.tensordot(q[:, c], k[c], dims=([2], [1])) / math.sqrt(d)
            p = torch.softmax(z.masked_fill(hide[:, None, :], -math.inf), dim=-1)
            p = torch.where(hide.all(1)[:, None, None], torch.zeros_like(p), p)
            out[start[i]: start[i + 1]].view(rows, h, -1, d)[:, c] = torch.tensordot(p, v[c], dims=([2], [0]))
    return out


def _exact_keep(case, s):
    """The pages' scales (the codes follow from 32-bit steps)."""
    page = case["page"]
    table, start, kv = s["table"].tolist(), s["start"].tolist(), s["kv"].tolist()
    after = {}
    for i, n in enumerate(s["count"].tolist()):
        context = kv[i] - (start[i + 1] - start[i])
        for a, b in enumerate(s["kept"][i, :n].tolist()):
            pid = table[i][(context + a) // page]
            after.setdefault(pid, {pid}).add(table[i][(context + b) // page])
    both = []
    for n in ("k", "v"):
        scales = s[n + "_scales"].double()
        new = scales.clone()
        for pid, sources in after.items():
            new[pid] = scales[sorted(sources)].amax(0)
        both.append(new)
    return [None, None] + both + [None]


def _exact_experts(case, s):
    n, x = case["inter"], s["x"].double()
    logits = torch.stack([(x * r).sum(1) for r in s["router"].double()], 1) + s["bias"].double()
    index = torch.argsort(-logits, dim=1, stable=True)[:, : case["top"]]
    p = torch.softmax(logits.gather(1, index) if case["normalize"] else logits, 1)
    share = p if case["normalize"] else p.gather(1, index)
    y = torch.zeros_like(x) if s["residual"] is None else s["residual"].double()
    for e in sorted(set(index.flatten().tolist())):
        token, slot = torch.nonzero(index == e, as_tuple=True)
        z = x[token] @ _values(s["gate_up"][e], s["gate_up_scales"][e], torch.float64).T.contiguous()
        a = z[:, :n]
        a = torch.nn.functional.gelu(a, approximate="tanh") if case["gelu"] else a * torch.sigmoid(a)
        z = (a * z[:, n:]) @ _values(s["down"][e], s["down_scales"][e], torch.float64).T.contiguous()
        y[token] += z * share[token, slot][:, None]
    return [y, None, share]


def exact(case, seed):
    return {"rotate": _exact_rotate, "tree": _exact_tree, "keep": _exact_keep,
            "experts": _exact_experts}[case["kind"]](case, prepare(case, seed))
