"""GPU: rotary positions.  Tables against 64-bit angles; rotation bit for bit against
the stated f32 steps and within their error of the 64-bit formula."""
import ctypes
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

EPS = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}   # half a step


def _frequencies(d, base, kind="none", factor=1.0, original=0.0, low=1.0, high=32.0):
    w = []
    for i in range(d // 2):
        b = base * factor ** (d / (d - 2)) if kind == "ntk" else base
        f = b ** (-2.0 * i / d)
        if kind == "linear":
            f /= factor
        elif kind == "turns":
            g = min(max((original * f / (2 * math.pi) - low) / (high - low), 0.0), 1.0)
            f = g * f + (1 - g) * f / factor
        elif kind == "yarn":
            at = lambda t: d * math.log(original / (2 * math.pi * t)) / (2 * math.log(base))
            lo, hi = max(math.floor(at(high)), 0), min(math.ceil(at(low)), d - 1)
            r = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f = (1 - r) * f + r * f / factor
        w.append(f)
    return np.array(w)


@pytest.mark.parametrize("kind,d,base,factor,original,first,count", [
    ("none", 128, 1e4, 1.0, 0.0, 0, 300), ("none", 2, 1e4, 1.0, 0.0, 0, 1),
    ("linear", 64, 1e4, 4.0, 0.0, 0, 1000), ("ntk", 96, 5e5, 8.0, 0.0, 131000, 77),
    ("turns", 128, 5e5, 8.0, 8192.0, 100000, 513), ("yarn", 64, 1e4, 40.0, 4096.0, 163839, 1),
    ("yarn", 20, 1e4, 16.0, 2048.0, 5, 33), ("none", 512, 1e6, 1.0, 0.0, 1048575, 17),
    # every pair kept, every pair stretched: the blend's limits
    ("yarn", 32, 1e4, 2.0, 1e9, 0, 9), ("turns", 32, 1e4, 2.0, 0.5, 0, 9)])
def test_table(qc, kind, d, base, factor, original, first, count):
    mag = 1.25 if kind == "yarn" else 1.0
    c, s = qc.rope_table(count, d, base, kind, factor, original, magnitude=mag, first_position=first)
    angle = np.arange(first, first + count)[:, None] * _frequencies(d, base, kind, factor, original)[None]
    # a frequency off by a few 2^-53 turns an angle of 10^6 by 10^-9 at most; one rounding
    for got, want in ((c, mag * np.cos(angle)), (s, mag * np.sin(angle))):
        got = got.cpu().numpy().astype(np.float64)
        assert np.all(np.abs(got - want) <= 2.0 ** -24 * np.abs(want) + 2e-9)


def _rotate(x, c, s, pos, rd, interleaved):
    """The stated f32 steps on numpy f32 arrays."""
    y = x.copy()
    cc, ss = c[pos][:, None, :], s[pos][:, None, :]
    a, b = (x[..., 0:rd:2], x[..., 1:rd:2]) if interleaved else (x[..., :rd // 2], x[..., rd // 2:rd])
    ya, yb = a * cc - b * ss, b * cc + a * ss
    if interleaved:
        y[..., 0:rd:2], y[..., 1:rd:2] = ya, yb
    else:
        y[..., :rd // 2], y[..., rd // 2:rd] = ya, yb
    return y


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("tokens,heads,hd,rd,interleaved", [
    (1, 1, 2, 2, False), (1, 40, 128, 128, False), (3, 5, 80, 20, True), (17, 3, 64, 64, True),
    (33, 7, 96, 24, False), (5, 2, 6, 6, False), (9, 4, 10, 6, True), (64, 32, 128, 64, False),
    (257, 12, 256, 256, True), (2, 1, 130, 66, False)])
def test_rotation(qc, dev, dtype, tokens, heads, hd, rd, interleaved):
    import torch
    print(f"rope {dtype} {tokens}x{heads}x{hd} rotary {rd} interleaved {interleaved}", flush=True)
    dt = getattr(torch, dtype)
    g = torch.Generator().manual_seed(tokens * 1000 + hd)
    x = (3 * torch.randn(tokens, heads, hd, generator=g)).to(dt)
    pos = torch.randint(0, 500, (tokens,), generator=g, dtype=torch.int32)
    c, s = qc.rope_table(500, rd)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    X = x.to(dev)
    y = qc.rope(X, c, s, pos.to(dev), interleaved=interleaved, dev_status=st)
    xs, cs, ss = x.float().numpy(), c.cpu().numpy(), s.cpu().numpy()
    want = torch.from_numpy(_rotate(xs, cs, ss, pos.numpy(), rd, interleaved)).to(dt)
    assert torch.equal(y.cpu(), want) and st.item() == 0
    # the formula in 64 bits: two roundings of each product's magnitude, then the type's
    f64 = _rotate(xs.astype(np.float64), cs.astype(np.float64), ss.astype(np.float64), pos.numpy(), rd, interleaved)
    mag = _rotate(np.abs(xs).astype(np.float64), np.abs(cs).astype(np.float64), -np.abs(ss).astype(np.float64),
                  pos.numpy(), rd, interleaved)
    mag = np.maximum(np.abs(mag), np.abs(_rotate(np.abs(xs).astype(np.float64), np.abs(cs).astype(np.float64),
                                                 np.abs(ss).astype(np.float64), pos.numpy(), rd, interleaved)))
    err = np.abs(y.cpu().double().numpy() - f64)
    assert np.all(err <= 2.0 ** -23 * mag + EPS[dtype] * (1 + 2.0 ** -20) * np.abs(f64) + 2.0 ** -25)
    # in place, the blocking form
    qc.rope(X, c, s, pos.to(dev), interleaved=interleaved, out=X)
    assert torch.equal(X.cpu(), want)


def test_strided_rows_of_a_projection(qc, dev):
    """Q and K heads of fused rows [Q | K | V] in one call, in place and out of place
    into strided rows; V and everything between stay as they were.  Odd offsets too."""
    import torch
    for dt in (torch.float32, torch.bfloat16):
        for hq, hk, hd, shift in ((4, 2, 64, 0), (3, 1, 48, 1), (2, 2, 40, 3)):
            t, row = 11, (hq + 2 * hk) * hd + 5
            g = torch.Generator(device=dev).manual_seed(hd)
            buf = torch.randn(t * row + shift, generator=g, device=dev).to(dt)
            rows = buf[shift:].view(t, row)
            x = rows[:, :(hq + hk) * hd].unflatten(1, (hq + hk, hd))
            pos = torch.arange(t, dtype=torch.int32, device=dev) * 7
            c, s = qc.rope_table(128, hd)
            want = qc.rope(x.contiguous(), c, s, pos)
            before = rows.clone()
            wide = torch.full((t, hq + hk, 2 * hd + 1), 7.0, device=dev, dtype=dt)
            out = wide[:, :, 1:hd + 1]
            qc.rope(x, c, s, pos, out=out)
            assert torch.equal(out, want) and torch.all(wide[:, :, 0] == 7) and torch.all(wide[:, :, hd + 1:] == 7)
            qc.rope(x, c, s, pos, out=x)
            assert torch.equal(x, want)
            assert torch.equal(rows[:, (hq + hk) * hd:], before[:, (hq + hk) * hd:])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("tokens,heads,hd,rd,interleaved,gap", [
    (1, 5, 64, 64, False, 0), (9, 1, 64, 32, True, 0), (7, 6, 64, 64, False, 0), (33, 4, 128, 64, True, 1),
    (300, 40, 128, 128, False, 0), (5, 3, 48, 24, False, 3)])
def test_head_major_rows(qc, dev, dtype, tokens, heads, hd, rd, interleaved, gap):
    """A view [tokens][heads] of tensors that lie [heads][tokens] (rows `gap` tokens longer than
    what is rotated): out of place, into and from token-major rows, and in place."""
    import torch
    dt = getattr(torch, dtype)
    g = torch.Generator(device=dev).manual_seed(hd)
    held = torch.randn(heads, tokens + gap, hd, generator=g, device=dev).to(dt)
    x = held[:, :tokens].transpose(0, 1)
    pos = torch.arange(tokens, dtype=torch.int32, device=dev) * 3 % 128
    c, s = qc.rope_table(128, rd)
    flat = x.clone(memory_format=torch.contiguous_format)
    want = qc.rope(flat, c, s, pos, interleaved=interleaved)
    assert torch.equal(qc.rope(x, c, s, pos, interleaved=interleaved), want)
    other = torch.full_like(held, 7.0)
    out = other[:, :tokens].transpose(0, 1)
    for source in (x, flat):
        out.fill_(3.0)
        qc.rope(source, c, s, pos, interleaved=interleaved, out=out)
        assert torch.equal(out, want) and bool((other[:, tokens:] == 7).all())
    before = held.clone()
    qc.rope(x, c, s, pos, interleaved=interleaved, out=x)
    assert torch.equal(x, want) and torch.equal(held[:, tokens:], before[:, tokens:])


def test_padding_and_bad_positions(qc, dev):
    import torch
    x = torch.randn(6, 2, 32, device=dev)
    c, s = qc.rope_table(10, 32)
    pos = torch.tensor([3, -1, 9, 10, -2, 0], dtype=torch.int32, device=dev)
    out = torch.full_like(x, 5.0)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    qc.rope(x, c, s, pos, out=out, dev_status=st)
    good = torch.tensor([3, 0, 9, 0, 0, 0], dtype=torch.int32, device=dev)
    want = qc.rope(x, c, s, good)
    assert st.item() == 3
    for t, done in enumerate((1, 0, 1, 0, 0, 1)):
        assert torch.equal(out[t], want[t] if done else torch.full_like(out[t], 5.0)), t
    # the blocking form writes nothing; padding alone is no error
    out.fill_(5.0)
    with pytest.raises(qc.QcError) as e:
        qc.rope(x, c, s, pos, out=out)
    assert e.value.status == 3 and torch.all(out == 5.0)
    pos = torch.tensor([3, -1, 9, -1, -1, 0], dtype=torch.int32, device=dev)
    qc.rope(x, c, s, pos, out=out)
    assert torch.equal(out[0], want[0]) and torch.all(out[1] == 5.0)
    assert torch.all(qc.rope(x, c, s, pos)[1] == 0.0)


def test_tables_serve_the_single_token_seam(qc, oracle, dev):
    """rope of qgemv's rows = what qgemv_qkv_rope_kv stores, with the same tables."""
    import torch
    heads, kvh, hd, k, p = 4, 2, 64, 256, 41
    g = torch.Generator(device=dev).manual_seed(5)
    c, s = qc.rope_table(64, hd, scaling="linear", factor=2.0)
    pq, pk, pv = (qc.pack(0, 0.05 * torch.randn(h * hd, k, generator=g, device=dev)) for h in (heads, kvh, kvh))
    x = torch.randn(k, generator=g, device=dev)
    q = torch.empty(heads * hd, device=dev)
    kc, vc = torch.zeros(3, kvh * hd, device=dev), torch.zeros(3, kvh * hd, device=dev)
    assert qc.qgemv_qkv_rope_kv_raw(0, pq, pk, pv, x, c, s, q, kc, vc, heads, kvh, hd, k, 3, 64, p, 1) == 0
    pos = torch.tensor([p], dtype=torch.int32, device=dev)
    y = torch.cat([qc.qgemv(0, pq, x, heads * hd, k), qc.qgemv(0, pk, x, kvh * hd, k)]).view(1, heads + kvh, hd)
    qc.rope(y, c, s, pos, out=y)
    # both round the same products; the projections agree within their contract
    torch.testing.assert_close(y[0, :heads].reshape(-1), q, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(y[0, heads:].reshape(-1), kc[1], rtol=1e-5, atol=1e-5)


def test_graph_and_streams(qc, dev):
    """Captured and replayed, and on a stream of its own."""
    import torch
    x = torch.randn(50, 6, 64, device=dev)
    pos = torch.arange(50, dtype=torch.int32, device=dev)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    out = torch.empty_like(x)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    want = qc.rope(x, *qc.rope_table(64, 64, scaling="yarn", factor=4.0, original_positions=32.0), pos)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        tables = qc.rope_table(64, 64, scaling="yarn", factor=4.0, original_positions=32.0)
        qc.rope(x, *tables, pos, out=out, dev_status=st)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        qc.rope(x, *tables, pos, out=out, dev_status=st)
    for rep in range(3):
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), rep
    del graph
