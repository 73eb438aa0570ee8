"""The operators between a low-bit decoder layer's projections, as a serving
program calls them: rotary positions, an int8 key/value cache in pages with a
scale for each page and head, attention over it, and products of microscaled
4-bit (MXFP4) matrices.

`listed()` holds the named cases, `draw(rng)` makes further ones of the same
ranges.  With `own` false, `run` computes an operator in elementary torch
operations; with `own` true it makes the calls of quixicore_hip.  `exact` gives
the same outputs from the definitions in 64 bits.

Kinds
  rope      rotation of the heads of a batch of tokens by their positions;
            with "build", the tables of a (scaled) context are made in the call
  append    new keys and values of a batch of sequences into the cache: a page's
            scale grows to hold them and the codes in it follow
  attend    softmax(scale q k^T) v over each sequence's pages, grouped heads
  quantize  rows to MXFP4 and back to the values the codes stand for
  product   y = x w^T of two MXFP4 matrices
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------
def listed():
    return [
        # one decoding step of 16 requests: Q and K heads of a 4096-wide layer
        {"name": "rope_step_bf16", "kind": "rope", "type": "bf16", "tokens": 16, "heads": 40,
         "head_dim": 128, "rotary": 128, "interleaved": False, "scaling": "none", "factor": 1.0,
         "positions": 32768, "build": False},
        # a long prompt in a model that rotates half of each head, its context
        # stretched 16 times: tables and rotation
        {"name": "rope_long_f32", "kind": "rope", "type": "f32", "tokens": 8192, "heads": 40,
         "head_dim": 128, "rotary": 64, "interleaved": True, "scaling": "yarn", "factor": 16.0,
         "positions": 131072, "build": True},
        # one decoding step of 64 requests, a token each
        {"name": "append_step_bf16", "kind": "append", "type": "bf16", "seqs": 64, "new": 1,
         "kv": 2048, "kv_heads": 8, "head_dim": 128, "page": 64, "spare": 0},
        # prompts of odd lengths, continued in pages that are partly full
        {"name": "append_prompts_f16", "kind": "append", "type": "f16", "seqs": 7, "new": 1501,
         "kv": 4000, "kv_heads": 8, "head_dim": 128, "page": 16, "spare": 3},
        # single-stream decoding after a short prompt, f32 projections
        {"name": "attend_one_f32", "kind": "attend", "type": "f32", "seqs": 1, "new": 1, "kv": 600,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 32, "causal": True, "window": 0,
         "spare": 0},
        # decoding of 32 requests with contexts up to 16384
        {"name": "attend_batch_bf16", "kind": "attend", "type": "bf16", "seqs": 32, "new": 1,
         "kv": 16384, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "causal": True,
         "window": 0, "spare": 0},
        # prefill of one prompt of 8192 tokens
        {"name": "attend_prompt_bf16", "kind": "attend", "type": "bf16", "seqs": 1, "new": 8192,
         "kv": 8192, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "causal": True,
         "window": 0, "spare": 0},
        # the activations of a small decoding batch
        {"name": "quantize_step_bf16", "kind": "quantize", "type": "bf16", "rows": 16, "dim": 4096},
        # a weight matrix when it is loaded
        {"name": "quantize_load_f32", "kind": "quantize", "type": "f32", "rows": 14336,
         "dim": 4096},
        # one token through the wide projection
        {"name": "product_one_f32", "kind": "product", "type": "f32", "m": 1, "n": 14336, "k": 4096},
        # a short prompt through a model of no round sizes
        {"name": "product_ragged_f16", "kind": "product", "type": "f16", "m": 77, "n": 5461,
         "k": 2752},
        # prefill of many prompts through the wide projection
        {"name": "product_prompts_bf16", "kind": "product", "type": "bf16", "m": 4096, "n": 14336,
         "k": 4096},
    ]


def _log(rng, low, high, step=1):
    """A size whose logarithm is uniform, rounded to a multiple of step."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(step, int(round(v / step)) * step)


def draw(rng):
    kind = rng.choice(["rope", "append", "attend", "attend", "attend", "quantize", "product",
                       "product"])
    typ = rng.choice(["f32", "f16", "bf16"])
    hd = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    if kind == "rope":
        scaling = rng.choice(["none", "none", "linear", "ntk", "turns", "yarn"])
        return {"kind": kind, "type": typ, "tokens": _log(rng, 1, 8192), "heads": rng.randint(1, 40),
                "head_dim": hd, "rotary": rng.choice([hd, hd, hd // 2, hd // 4]),
                "interleaved": rng.random() < 0.5, "scaling": scaling,
                "factor": 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 16.0, 40.0]),
                "positions": _log(rng, 512, 131072), "build": rng.random() < 0.3}
    if kind == "append":
        kvh = rng.choice([1, 2, 4, 5, 8])
        new = 1 if rng.random() < 0.5 else _log(rng, 2, 2000)
        seqs = _log(rng, 1, 64 if new == 1 else max(1, min(32, 10000 // new)))
        return {"kind": kind, "type": typ, "seqs": seqs, "new": new, "kv": _log(rng, new, new + 4000),
                "kv_heads": kvh, "head_dim": hd, "page": page, "spare": rng.choice([0, 0, 5])}
    if kind == "attend":
        kvh, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 4, 7, 8, 16])
        heads = kvh * group
        new = 1 if rng.random() < 0.5 else _log(rng, 2, 2048)
        kv = _log(rng, max(new, 16), 16384)
        pairs = (1 << 37) // (heads * hd)        # of the prompt of 8192, half of them seen
        new = min(new, pairs // kv)
        most = min(pairs // (new * kv), (1 << 29) // (kv * kvh * hd), 64)
        seqs = _log(rng, 1, max(1, most))
        causal = rng.random() < 0.8
        return {"kind": kind, "type": typ, "seqs": seqs, "new": new, "kv": kv, "heads": heads,
                "kv_heads": kvh, "head_dim": hd, "page": page, "causal": causal,
                "window": _log(rng, 16, kv + 16) if causal and rng.random() < 0.3 else 0,
                "spare": rng.choice([0, 0, 5])}
    if kind == "quantize":
        dim = _log(rng, 32, 16384, 32)
        return {"kind": kind, "type": typ, "rows": min(_log(rng, 1, 14336), (1 << 25) // dim),
                "dim": dim}
    k = _log(rng, 256, 14336, 32)
    n = _log(rng, 256, 16384)
    m = 1 if rng.random() < 0.25 else _log(rng, 2, 4096)
    return {"kind": kind, "type": typ, "m": min(m, 4096 * 14336 * 4096 // (n * k)), "n": n, "k": k}


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

    def ints(self, low, high, n):
        """n whole numbers in [low, high]."""
        return torch.randint(low, high + 1, (n,), generator=self.g, device=self.dev)

    def channels(self, *shape):
        """N(0, 1) times a magnitude for each of the last dimension's channels."""
        return self.normal(*shape) * torch.exp(0.5 * self.normal(shape[-1]))


_BETA_FAST, _BETA_SLOW, _LOW_TURNS, _HIGH_TURNS = 32.0, 1.0, 1.0, 4.0
_BASE = 10000.0


def _magnitude(case):
    return 0.1 * math.log(case["factor"]) + 1.0 if case["scaling"] == "yarn" else 1.0


def _lengths(case):
    """New and total tokens of each sequence: from a quarter of the largest, one at
    it, spread by the multiples of irrational numbers."""
    def spread(most, step):
        return [max(1, round(most * (1.0 - 0.75 * math.modf(i * step)[0]))) for i in range(case["seqs"])]

    new = spread(case["new"], 0.6180339887)
    return new, [max(a, b) for a, b in zip(new, spread(case["kv"], 0.7548776662))]


def _cache(case, g):
    """Page table, lengths and a filled cache of a batch of sequences."""
    page, h, d = case["page"], case["kv_heads"], case["head_dim"]
    new, kv = (torch.tensor(v, device=g.dev) for v in _lengths(case))
    columns = -(-case["kv"] // page)
    pages = case["seqs"] * columns
    table = torch.randperm(pages, generator=g.g, device=g.dev).to(torch.int32)
    start = torch.zeros(case["seqs"] + 1, dtype=torch.int32, device=g.dev)
    start[1:] = new.cumsum(0)
    s = {"new": new, "kv": kv.to(torch.int32), "start": start,
         "table": table.view(case["seqs"], columns), "max_kv": case["kv"], "max_new": case["new"],
         "tokens": int(start[-1]) + case["spare"], "status": torch.zeros(1, dtype=torch.int32, device=g.dev)}
    for name in ("k", "v"):
        x = g.channels(pages, h, page, d) if name == "k" else g.outliers(pages, h, page, d)
        scale = x.abs().amax((2, 3)) / 127.0
        s[name + "_codes"] = (x / scale[:, :, None, None]).round_().to(torch.int8)
        s[name + "_scales"] = scale
    return s


def _pow2(e, dtype=torch.float32):
    """2 to the power of whole numbers, exactly."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64).to(dtype)


def _to_fp4(b):
    """Codes 0..15 and scale exponents of blocks of 32 (last dimension)."""
    top = b.abs().amax(-1, keepdim=True)
    e = (torch.frexp(top)[1] - 3).clamp(-127, 127)
    e = torch.where(top == 0, -127, e)
    a = (b * _pow2(-e)).abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5)
            + (a >= 3.5) + (a > 5.0))
    return code.to(torch.uint8) + 8 * torch.signbit(b).to(torch.uint8), e


def _packed(g, rows, k, sigma):
    """A random MXFP4 matrix: codes [rows][k/2], the even element in the low
    half of its byte, and biased scale exponents [rows][k/32]."""
    code, e = _to_fp4((g.outliers(rows, k) * sigma).view(rows, k // 32, 32))
    code = code.view(rows, k // 2, 2)
    return (code[..., 0] | (code[..., 1] << 4)).contiguous(), (e[..., 0] + 127).to(torch.uint8)


def prepare(case, seed):
    g = _Gen(seed)
    kind, typ = case["kind"], TORCH[case["type"]]
    s = {"case": case}
    if kind == "rope":
        t, h, d = case["tokens"], case["heads"], case["head_dim"]
        s.update(x=g.normal(t, h, d).to(typ), y=torch.zeros(t, h, d, dtype=typ, device=g.dev),
                 positions=g.ints(0, case["positions"] - 1, t).to(torch.int32),
                 status=torch.zeros(1, dtype=torch.int32, device=g.dev))
        if not case["build"]:
            s["tables"] = _tables(case, g.dev)
    elif kind == "append":
        s.update(_cache(case, g))
        h, d, page = case["kv_heads"], case["head_dim"], case["page"]
        # louder than what the pages hold, so that some scales grow
        s.update(k=(1.2 * g.channels(s["tokens"], h, d)).to(typ),
                 v=(1.2 * g.outliers(s["tokens"], h, d)).to(typ))
        # what is read back: the pages written to, from their first slot on
        first = (s["kv"].to(torch.int64) - s["new"]) // page * page
        back = torch.zeros_like(s["start"])
        back[1:] = (s["kv"].to(torch.int64) - first).cumsum(0)
        s.update(back=back, back_tokens=int(back[-1]), back_max=case["new"] + page)
    elif kind == "attend":
        s.update(_cache(case, g))
        h, d = case["heads"], case["head_dim"]
        s.update(q=(1.5 * g.normal(s["tokens"], h, d)).to(typ),
                 out=torch.zeros(s["tokens"], h, d, dtype=typ, device=g.dev))
    elif kind == "quantize":
        s.update(x=g.outliers(case["rows"], case["dim"]).to(typ),
                 status=torch.zeros(1, dtype=torch.int32, device=g.dev))
    else:
        s["w"], s["w_scales"] = _packed(g, case["n"], case["k"], 0.02)
        s["x"], s["x_scales"] = _packed(g, case["m"], case["k"], 1.0)
        s["y"] = torch.zeros(case["m"], case["n"], dtype=typ, device=g.dev)
    return s


# --------------------------------------------------------------------------
# The plain forms
# --------------------------------------------------------------------------
def _frequencies(case, dev):
    """Radians a position for each rotated pair."""
    d, factor, kind = case["rotary"], case["factor"], case["scaling"]
    i = torch.arange(d // 2, device=dev, dtype=torch.float64)
    f = _BASE ** (-2.0 * i / d)
    original = case["positions"] / factor
    if kind == "linear":
        return f / factor
    if kind == "ntk":
        return (_BASE * factor ** (d / (d - 2.0))) ** (-2.0 * i / d)
    if kind == "turns":
        turns = original * f / (2.0 * math.pi)
        keep = ((turns - _LOW_TURNS) / (_HIGH_TURNS - _LOW_TURNS)).clamp(0.0, 1.0)
        return keep * f + (1.0 - keep) * f / factor
    if kind == "yarn":
        low = max(math.floor(d * math.log(original / (_BETA_FAST * 2 * math.pi)) / (2 * math.log(_BASE))), 0)
        high = min(math.ceil(d * math.log(original / (_BETA_SLOW * 2 * math.pi)) / (2 * math.log(_BASE))), d - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        return (1.0 - ramp) * f + ramp * f / factor
    return f


def _tables(case, dev):
    """Cosines and sines [positions][rotary / 2]; far positions' angles need 64 bits."""
    p = torch.arange(case["positions"], device=dev, dtype=torch.float64)
    angle = p[:, None] * _frequencies(case, dev)[None, :]
    m = _magnitude(case)
    return (m * angle.cos()).float(), (m * angle.sin()).float()


def _rope_plain(s):
    case = s["case"]
    cosine, sine = s["tables"] if "tables" in s else _tables(case, s["x"].device)
    r = case["rotary"]
    p = s["positions"].to(torch.int64)
    c, n = cosine[p][:, None, :], sine[p][:, None, :]
    x = s["x"].float()
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * c - b * n, b * c + a * n], dim=-1).flatten(-2)
    else:
        a, b = x[..., : r // 2], x[..., r // 2: r]
        y = torch.cat([a * c - b * n, b * c + a * n], dim=-1)
    return torch.cat([y, x[..., r:]], dim=-1).to(s["x"].dtype)


def _places(s, start, count):
    """For the tokens of ragged sequences that end at each one's length: the
    sequence, position and page of each."""
    t = torch.arange(count, device=start.device)
    seq = torch.searchsorted(start[1:].to(torch.int64), t, right=True)
    last = s["kv"].to(torch.int64)[seq] - start[1:].to(torch.int64)[seq]
    position = last + t
    page = s["case"]["page"]
    return seq, position, s["table"].to(torch.int64)[seq, position // page], position % page


def _append_plain(s):
    case = s["case"]
    page = case["page"]
    count = s["tokens"] - case["spare"]
    seq, position, pid, slot = _places(s, s["start"], count)
    first = (s["kv"].to(torch.int64) - s["new"])[seq]
    touched, inverse = torch.unique(pid, return_inverse=True)
    # slots of a touched page that were full before
    full = torch.zeros(touched.numel(), dtype=torch.int64, device=pid.device)
    full[inverse] = (first - position // page * page).clamp(min=0)
    outs = []
    for name in ("k", "v"):
        x = s[name][:count].float()
        codes, scales = s[name + "_codes"], s[name + "_scales"]
        h = case["kv_heads"]
        top = torch.zeros(touched.numel(), h, device=pid.device)
        top.scatter_reduce_(0, inverse[:, None].expand(-1, h), x.abs().amax(2), "amax")
        before = torch.where(full[:, None] > 0, scales[touched], 0.0)
        scale = torch.maximum(before, top / 127.0)
        scale = torch.where(scale < 2.0 ** -126, 0.0, scale)
        ratio = torch.where(scale > 0, before / scale, 0.0)
        inv = torch.where(scale > 0, 1.0 / scale, 0.0)
        old = codes[touched]
        moved = (old.float() * ratio[:, :, None, None]).round().to(torch.int8)
        keep = torch.arange(page, device=pid.device)[None, :] < full[:, None]
        codes[touched] = torch.where(keep[:, None, :, None], moved, old)
        scales[touched] = scale
        codes[pid, :, slot] = (x * inv[inverse][:, :, None]).round().clamp(-127, 127).to(torch.int8)
        _, _, bp, bs = _places(s, s["back"], s["back_tokens"])
        outs.append((codes[bp, :, bs].float() * scales[bp][:, :, None]).to(s[name].dtype))
    return [outs[0], outs[1], s["k_scales"], s["v_scales"]]


def _attend_plain(s):
    case = s["case"]
    page, h, d, g = case["page"], case["kv_heads"], case["head_dim"], case["heads"] // case["kv_heads"]
    n, most, kv = case["seqs"], case["new"], case["kv"]
    table = s["table"].to(torch.int64)
    count = s["tokens"] - case["spare"]
    seq, position, _, _ = _places(s, s["start"], count)
    index = torch.arange(count, device=table.device) - s["start"].to(torch.int64)[seq]
    q = torch.zeros(n, most, h, g, d, device=table.device)
    q[seq, index] = s["q"][:count].float().view(count, h, g, d)
    at = torch.full((n, most), -1, device=table.device)
    at[seq, index] = position
    wide = table.shape[1] * page
    k, v = [(s[m + "_codes"][table].float() * s[m + "_scales"][table][..., None, None])
            .transpose(1, 2).reshape(n, h, wide, d)[:, :, :kv] for m in ("k", "v")]
    q = q.permute(0, 2, 3, 1, 4).reshape(n, h, g * most, d) * (1.0 / math.sqrt(d))
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).view(n, h, g, most, kv)
    j = torch.arange(kv, device=table.device)
    seen = (j[None, :] < s["kv"][:, None])[:, None, :]
    if case["causal"]:
        seen = seen & (j <= at[:, :, None])
    if case["window"]:
        seen = seen & (j > at[:, :, None] - case["window"])
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p.view(n, h, g * most, kv), v.contiguous()).view(n, h, g, most, d)
    y = y / torch.where(total == 0, 1.0, total)
    s["out"][:count] = y[seq, :, :, index].reshape(count, h * g, d).to(s["out"].dtype)
    return s["out"]


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _quantize_plain(s):
    x = s["x"]
    code, e = _to_fp4(x.float().view(x.shape[0], -1, 32))
    value = torch.tensor(_E2M1, device=x.device)[code.to(torch.int32)]
    return (value * _pow2(e)).view(x.shape).to(x.dtype)


def _values(codes, scales, dtype):
    """The matrix that MXFP4 codes and scales stand for."""
    both = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).to(torch.int32)
    v = torch.tensor(_E2M1, device=codes.device, dtype=dtype)[both]
    step = _pow2(scales.to(torch.int32) - 127, dtype)
    return (v.view(*scales.shape, 32) * step[..., None]).view(both.shape)


def _product_plain(s):
    w = _values(s["w"], s["w_scales"], torch.float32)
    x = _values(s["x"], s["x_scales"], torch.float32)
    return torch.matmul(x, w.T.contiguous()).to(s["y"].dtype)


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
    """The cache and batch descriptors that a serving program keeps for its buffers."""
    if "handles" not in s:
        qc = _qc()
        cache = qc.Kv8Cache(s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"])
        batch = qc.Kv8Batch(s["table"], s["start"], s["kv"], s["tokens"], s["max_new"], s["max_kv"])
        s["handles"] = cache, batch
        if "back" in s:
            s["handles"] += (qc.Kv8Batch(s["table"], s["back"], s["kv"], s["back_tokens"],
                                         s["back_max"], s["max_kv"]),)
    return s["handles"]


def _run_own(s):
    qc, case = _qc(), s["case"]
    kind = case["kind"]
    if kind == "rope":
        if "tables" in s:
            cosine, sine = s["tables"]
        else:
            cosine, sine = qc.rope_table(
                case["positions"], case["rotary"], base=_BASE, scaling=case["scaling"],
                factor=case["factor"], original_positions=case["positions"] / case["factor"],
                low_turns=_BETA_SLOW if case["scaling"] == "yarn" else _LOW_TURNS,
                high_turns=_BETA_FAST if case["scaling"] == "yarn" else _HIGH_TURNS,
                magnitude=_magnitude(case))
        return qc.rope(s["x"], cosine, sine, s["positions"], interleaved=case["interleaved"],
                       out=s["y"], dev_status=s["status"])
    if kind == "append":
        cache, batch, back = _handles(s)
        qc.kv8_append(cache, batch, s["k"], s["v"], dev_status=s["status"])
        k, v = qc.kv8_gather(cache, back, dtype=s["k"].dtype, dev_status=s["status"])
        return [k, v, s["k_scales"], s["v_scales"]]
    if kind == "attend":
        cache, batch = _handles(s)
        return qc.kv8_attention(cache, batch, s["q"], causal=case["causal"], window=case["window"],
                                out=s["out"], dev_status=s["status"])
    if kind == "quantize":
        codes, scales = qc.quantize_mxfp4(s["x"], dev_status=s["status"])
        return qc.dequantize_mxfp4(codes, scales, dtype=s["x"].dtype)
    return qc.mxfp4_gemm(s["w"], s["w_scales"], s["x"], s["x_scales"], y=s["y"])


def run(s):
    if own:
        return _run_own(s)
    return {"rope": _rope_plain, "append": _append_plain, "attend": _attend_plain,
            "quantize": _quantize_plain, "product": _product_plain}[s["case"]["kind"]](s)


# --------------------------------------------------------------------------
# What a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    size = 4 if case["type"] == "f32" else 2
    if kind == "rope":
        t, h, d, r = case["tokens"], case["heads"], case["head_dim"], case["rotary"]
        tables = 4 * r * (case["positions"] if case["build"] else min(t, case["positions"]))
        return {"bytes": 2 * size * t * h * d + tables + 4 * t, "flops": 3 * t * h * r}
    if kind in ("append", "attend"):
        new, kv = (torch.tensor(v, dtype=torch.float64) for v in _lengths(case))
        h, d, page = case["kv_heads"], case["head_dim"], case["page"]
        tokens = float(new.sum())
        if kind == "append":
            back = float((kv - torch.floor((kv - new) / page) * page).sum())
            # new rows in; the touched pages' codes out; their values read back
            return {"bytes": 2 * h * d * (size * tokens + back + size * back), "flops": 4 * tokens * h * d}
        # pairs of a query and a key that it sees
        rows = [torch.arange(int(k) - int(n), int(k), dtype=torch.float64) for n, k in zip(new, kv)]
        if not case["causal"]:
            seen = [len(r) * float(k) for r, k in zip(rows, kv)]
        else:
            w = case["window"] or math.inf
            seen = [float((r + 1).clamp(max=w).sum()) for r in rows]
        read = kv if not case["window"] else torch.minimum(kv, new + case["window"])
        return {"bytes": 2 * h * d * float(read.sum()) + 2 * size * tokens * case["heads"] * d,
                "flops": 4 * sum(seen) * case["heads"] * d}
    if kind == "quantize":
        n = case["rows"] * case["dim"]
        return {"bytes": n * (2 * size + 17 / 32), "flops": 0}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": (m + n) * k * 17 / 32 + size * m * n, "flops": 2 * m * n * k}


# --------------------------------------------------------------------------
# The same outputs in 64 bits
# --------------------------------------------------------------------------
def _exact_rope(case, s):
    d, r = case["head_dim"], case["rotary"]
    p = s["positions"].double()
    x = s["x"].double()
    y = x.clone()
    f = _frequencies(case, x.device)
    m = _magnitude(case)
    pairs = [(2 * i, 2 * i + 1) if case["interleaved"] else (i, i + r // 2) for i in range(r // 2)]
    for (a, b), w in zip(pairs, f):
        turn = torch.polar(torch.full_like(p, m), p * w)[:, None]
        z = torch.complex(x[..., a], x[..., b]) * turn
        y[..., a], y[..., b] = z.real, z.imag
    return y


def _exact_attend(case, s):
    page, h, d = case["page"], case["kv_heads"], case["head_dim"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=s["out"].device)
    start, kv = s["start"].tolist(), s["kv"].tolist()
    for i, length in enumerate(kv):
        rows = start[i + 1] - start[i]
        ids = s["table"][i, : -(-length // page)].to(torch.int64)
        k, v = [(s[m + "_codes"][ids].double() * s[m + "_scales"][ids].double()[..., None, None])
                .permute(1, 0, 2, 3).reshape(h, -1, d)[:, :length] for m in ("k", "v")]
        j = torch.arange(length, device=out.device)[None, :]
        for lo in range(0, rows, 1024):
            hi = min(rows, lo + 1024)
            at = torch.arange(length - rows + lo, length - rows + hi, device=out.device)[:, None]
            hide = torch.zeros(hi - lo, length, dtype=torch.bool, device=out.device)
            if case["causal"]:
                hide = hide | (j > at)
            if case["window"]:
                hide = hide | (j <= at - case["window"])
            q = s["q"][start[i] + lo: start[i] + hi].double().view(hi - lo, h, -1, d)
            for c in range(h):
                z = torch.tensordot(q[:, c], k[c], dims=([2], [1])) / math.sqrt(d)
                p = torch.softmax(z.masked_fill(hide[:, None, :], -math.inf), dim=-1)
                y = torch.tensordot(p, v[c], dims=([2], [0]))
                out[start[i] + lo: start[i] + hi].view(hi - lo, h, -1, d)[:, c] = y
    return out


def _exact_scales(case, s, name):
    """Every page's scale after the append (its codes follow from f32 steps)."""
    page = case["page"]
    scales = s[name + "_scales"].double()
    start, kv, table = s["start"].tolist(), s["kv"].tolist(), s["table"].tolist()
    for i, length in enumerate(kv):
        begin = length - (start[i + 1] - start[i])
        for lo in range(begin // page * page, length, page):
            a, b = max(lo, begin), min(lo + page, length)
            rows = s[name][start[i] + a - begin: start[i] + b - begin].double()
            top = rows.abs().amax((0, 2)) / 127.0
            pid = table[i][lo // page]
            scales[pid] = torch.maximum(scales[pid], top) if a > lo else top
    return scales


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rope":
        return _exact_rope(case, s)
    if kind == "append":
        return [None, None, _exact_scales(case, s, "k"), _exact_scales(case, s, "v")]
    if kind == "attend":
        return _exact_attend(case, s)
    if kind == "quantize":
        b = s["x"].double().view(s["x"].shape[0], -1, 32)
        top = b.abs().amax(-1, keepdim=True)
        step = torch.exp2(torch.floor(torch.log2(top)) - 2.0).where(top > 0, torch.ones_like(top))
        a = b.abs() / step
        # spacing 1/2 below 2, 1 up to 4, 2 above; round() takes ties to even
        grid = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
        q = ((a / grid).round() * grid).clamp(max=6.0)
        return (q * step * b.sign()).view(s["x"].shape)
    w = _values(s["w"], s["w_scales"], torch.float64)
    x = _values(s["x"], s["x_scales"], torch.float64)
    return torch.matmul(x, w.T.contiguous())
