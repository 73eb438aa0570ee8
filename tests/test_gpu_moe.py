"""GPU: the mixture-of-experts feed-forward with MXFP4 weights, against 64-bit arithmetic on the values that the
codes stand for, and as one step with the operators of drafted tokens."""
import numpy as np
import pytest

from test_gpu_kv8 import HALF

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]


def _weights(qc, g, dev, rows, k, sigma=0.05):
    import torch
    return qc.quantize_mxfp4(sigma * torch.randn(rows, k, generator=g, device=dev))


def _layer(qc, dev, experts, dim, inter, seed=0, router="float32", bias=True):
    """(layer, f64 values of router, bias, gate_up, down)."""
    import torch
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    guc, gus = _weights(qc, g, dev, experts * 2 * inter, dim)
    dc, ds = _weights(qc, g, dev, experts * dim, inter)
    r = (2.0 * torch.randn(experts, dim, generator=g, device=dev) / dim ** 0.5).to(getattr(torch, router))
    b = 0.5 * torch.randn(experts, generator=g, device=dev) if bias else None
    layer = qc.Mxfp4Moe(r, guc.view(experts, 2 * inter, -1), gus.view(experts, 2 * inter, -1),
                        dc.view(experts, dim, -1), ds.view(experts, dim, -1), bias=b)
    f64 = lambda t: t.double().cpu().numpy()
    values = (f64(r), f64(b) if bias else np.zeros(experts),
              f64(qc.dequantize_mxfp4(guc, gus)).reshape(experts, 2 * inter, dim),
              f64(qc.dequantize_mxfp4(dc, ds)).reshape(experts, dim, inter))
    return layer, values


def _reference(values, x, top, normalize, gelu, residual, scale, half):
    """(y, ids, weights, tolerance of y) in f64.

    A dot of K values in n terms is a chain of n K / 128 instructions of 8 sums each, whose joins round
    within 2^-23 of the sum of magnitudes S: with 16 for the last joins (n K / 16 + 16) 2^-23 S.
    A term is within 2^-4 of what was left for it, so n leave 2^-4n of a value; bf16, f16 and f32 fit x's 2, 3
    and 6.  All but the last are multiples of 2^-2 with the block's largest, m, in [2^7, 2^8): a small value keeps an
    error of 2^-3 2^-4(n-2) 2^-4 2^-7 m = 2^(-4n - 6) m, with the shares of the terms after it 1.1 times that.  In
    the last term's sums of 16 products each is cut within 2^-13 of the largest, that is 2^-4(n-1) of block's
    largest weight times m.
    act has a slope of at most 1.13 and is computed within 2^-21 of |v|; a share is within 2^-22 of itself; the sum over
    the experts and the residual rounds top + 1 times within 2^-24; y is rounded once."""
    router, bias, gu, dn = values
    inter = dn.shape[2]
    nx = {2.0 ** -24: 6, 2.0 ** -11: 3, 2.0 ** -8: 2}[half]
    nh = {2.0 ** -24: 6, 2.0 ** -11: 4, 2.0 ** -8: 3}[half]
    tops = lambda v: np.repeat(np.abs(v).reshape(*v.shape[:-1], -1, 32).max(-1), 32, -1)

    def dot_error(w, v, n):
        return (np.abs(w) @ np.abs(v) * (n * v.size / 16 + 16) * 2.0 ** -23
                + np.abs(w) @ tops(v) * 1.1 * 2.0 ** (-4 * n - 6) + tops(w) @ tops(v) * 2.0 ** (-4 * n - 9))

    logits = x @ router.T + bias
    ids = np.argsort(-logits, axis=1, kind="stable")[:, :top]
    p = np.exp(np.take_along_axis(logits, ids, 1) - logits.max(1, keepdims=True))
    p = p / (p.sum(1, keepdims=True) if normalize else np.exp(logits - logits.max(1, keepdims=True)).sum(1, keepdims=True))
    p = p * scale
    y = np.zeros_like(x) if residual is None else residual.copy()
    tol = np.abs(y) * (top + 1) * 2.0 ** -24
    for t in range(x.shape[0]):
        for s in range(top):
            w, d = gu[ids[t, s]], dn[ids[t, s]]
            z, e = w @ x[t], dot_error(w, x[t], nx)
            v, u, ev, eu = z[:inter], z[inter:], e[:inter], e[inter:]
            if gelu:
                a = 0.5 * v * (1 + np.tanh(np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)))
            else:
                a = v / (1 + np.exp(-v))
            ea = 1.13 * ev + np.abs(v) * 2.0 ** -21
            h = a * u
            eh = np.abs(u) * ea + np.abs(a) * eu + ea * eu + np.abs(h) * (2.0 ** (-4 * nh) + 2.0 ** -23)
            o, eo = d @ h, np.abs(d) @ eh + dot_error(d, h, nh)
            y[t] += p[t, s] * o
            tol[t] += abs(p[t, s]) * (eo + np.abs(o) * (2.0 ** -22 + (top + 1) * 2.0 ** -24))
    return y, ids, p, tol + half * np.abs(y) * 1.001 + (2.0 ** -25 if half == 2.0 ** -11 else 1e-38)


def _run(qc, dev, tokens, experts, top, dim, inter, dtype, normalize=True, gelu=False, residual=True, router="float32",
         bias=True, scale=1.0, seed=0, spread=1.0):
    import torch
    layer, values = _layer(qc, dev, experts, dim, inter, seed, router, bias)
    rng = np.random.default_rng(seed)
    dt = getattr(torch, dtype)
    x = torch.from_numpy(spread * rng.standard_normal((tokens, dim))).to(dt)
    r = torch.from_numpy(rng.standard_normal((tokens, dim))).to(dt) if residual else None
    y, ids, weights = qc.mxfp4_moe(layer, x.to(dev), top, normalize=normalize, gelu_tanh=gelu, weight_scale=scale,
                                   residual=None if r is None else r.to(dev))
    want, wid, wp, tol = _reference(values, x.double().numpy(), top, normalize, gelu,
                                    None if r is None else r.double().numpy(), float(np.float32(scale)), HALF[dtype])
    assert np.array_equal(ids.cpu().numpy(), wid)
    assert np.all(np.abs(weights.double().cpu().numpy() - wp) <= 2.0 ** -23 * np.abs(wp) + 1e-38)
    err = np.abs(y.double().cpu().numpy() - want)
    assert np.all(err <= tol), (float((err / tol).max()), np.argwhere(~(err <= tol))[:4].tolist())
    return layer, x, r, y, ids, weights


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,experts,top,dim,inter", [
    (1, 1, 1, 32, 32), (1, 4, 2, 64, 96), (1, 64, 8, 256, 128), (2, 3, 3, 160, 32), (5, 8, 2, 544, 288),
    (16, 30, 3, 96, 224), (17, 8, 1, 256, 64), (33, 5, 4, 128, 160), (64, 4, 2, 320, 128), (100, 128, 6, 64, 64),
    (130, 2, 1, 96, 96), (7, 1024, 64, 32, 32)])
def test_moe(qc, dev, dtype, tokens, experts, top, dim, inter):
    print(f"moe {dtype} {tokens} tokens, {top} of {experts}, {dim} x {inter}", flush=True)
    _run(qc, dev, tokens, experts, top, dim, inter, dtype, seed=tokens + experts)


@pytest.mark.parametrize("dtype,most", [("float32", 2.0 ** -19), ("float16", 2.0 ** -11), ("bfloat16", 2.0 ** -8)])
@pytest.mark.parametrize("tokens", [4, 40])
def test_moe_precision(qc, dev, tokens, dtype, most):
    """The error as a whole, where the worst case of each value says little.  Roundings of a chain of n add like
    sqrt(n): f32 sqrt(6 * 544 / 16) 2^-24 of a sum that grows to its end is 2^-20.2, the second product adds a like
    share, act 2^-22: under 2^-19.  f16 and bf16: the output's half step, 2^-11 and 2^-8, at most."""
    import torch
    layer, values = _layer(qc, dev, 8, 544, 288, 4)
    x = torch.from_numpy(np.random.default_rng(4).standard_normal((tokens, 544))).to(getattr(torch, dtype))
    y = qc.mxfp4_moe(layer, x.to(dev), 2)[0].double().cpu().numpy()
    want = _reference(values, x.double().numpy(), 2, True, False, None, 1.0, HALF[dtype])[0]
    assert np.sqrt(np.mean((y - want) ** 2) / np.mean(want ** 2)) <= most


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [2, 30])
def test_moe_outliers(qc, dev, tokens, dtype):
    """Single values far above their block's others, and blocks of very different sizes."""
    import torch
    layer, values = _layer(qc, dev, 6, 192, 160, 7)
    rng = np.random.default_rng(7)
    x = rng.standard_normal((tokens, 192)) * np.repeat(2.0 ** rng.integers(-12, 4, (tokens, 6)), 32, 1)
    x[np.arange(tokens), rng.integers(0, 192, tokens)] *= 1000
    x = torch.from_numpy(x).to(getattr(torch, dtype))
    y, ids, _ = qc.mxfp4_moe(layer, x.to(dev), 2)
    want, wid, _, tol = _reference(values, x.double().numpy(), 2, True, False, None, 1.0, HALF[dtype])
    assert np.array_equal(ids.cpu().numpy(), wid)
    got = y.double().cpu().numpy()
    # f16 ends at 65504, the values that round up from 65520 on are infinite
    past = (np.abs(want) - tol >= 65520) & (dtype == "float16")
    near = (np.abs(want) + tol >= 65520) & (dtype == "float16")
    ok = np.where(past | (near & np.isinf(got)), got == np.sign(want) * np.inf, np.abs(got - want) <= tol)
    assert ok.all(), np.argwhere(~ok)[:4].tolist()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("residual,router,bias,scale", [(True, "float32", False, 1.0), (False, "bfloat16", True, 2.5),
                                                       (False, "float16", False, -0.125)])
def test_moe_forms(qc, dev, dtype, normalize, gelu, residual, router, bias, scale):
    _run(qc, dev, 9, 6, 2, 192, 160, dtype, normalize, gelu, residual, router, bias, scale, spread=3.0)


@pytest.mark.parametrize("tokens", [511, 512, 513, 1100])
def test_moe_passes(qc, dev, tokens):
    """More tokens than a pass holds: the rows of the last ones are also right in a call of their own."""
    import torch
    layer, x, r, y, ids, weights = _run(qc, dev, tokens, 8, 2, 64, 32, "bfloat16", seed=3)
    _, values = _layer(qc, dev, 8, 64, 32, 3)
    a = tokens // 2
    part = qc.mxfp4_moe(layer, x[a:].to(dev), 2, residual=r[a:].to(dev))
    assert torch.equal(part[1], ids[a:]) and torch.equal(part[2], weights[a:])
    want, _, _, tol = _reference(values, x[a:].double().numpy(), 2, True, False, r[a:].double().numpy(), 1.0,
                                 HALF["bfloat16"])
    assert np.all(np.abs(part[0].double().cpu().numpy() - want) <= tol)


def test_moe_one_expert_takes_all(qc, dev):
    """All tokens on the same experts, and each on its own."""
    import torch
    layer, values = _layer(qc, dev, 40, 128, 96, bias=False)
    rng = np.random.default_rng(1)
    for same in (True, False):
        x = rng.standard_normal((40, 128))
        if same:
            x = x * 0.01 + values[0][7]                    # near expert 7's router row
        else:
            x = x * 0.01 + 3 * values[0][rng.permutation(40)]
        X = torch.from_numpy(x).float()
        y, ids, _ = qc.mxfp4_moe(layer, X.to(dev), 1)
        want, wid, _, tol = _reference(values, X.double().numpy(), 1, True, False, None, 1.0, HALF["float32"])
        assert np.array_equal(ids.cpu().numpy(), wid) and len(set(wid.ravel())) == (1 if same else 40)
        assert np.all(np.abs(y.double().cpu().numpy() - want) <= tol)


def test_moe_ties(qc, dev):
    """Equal logits: the lowest indexes, in order; logits apart by less than an f32 step are told apart."""
    import torch
    layer, _ = _layer(qc, dev, 12, 64, 32, bias=False)
    router = layer.tensors[0]
    router.zero_()
    x = torch.randn(5, 64, device=dev)
    y, ids, weights = qc.mxfp4_moe(layer, x, 4)
    assert ids.tolist() == [[0, 1, 2, 3]] * 5 and bool((weights == 0.25).all())
    router[9] = router[4] = 1.0
    x[:] = x.abs()
    assert [i[:2] for i in qc.mxfp4_moe(layer, x, 4)[1].tolist()] == [[4, 9]] * 5
    # 1 + 2^-30 of 64 additions of 2^-36: lost in f32
    router.zero_()
    router[3, 0], router[6, 0], router[6, 1:] = 1.0, 1.0, 2.0 ** -36
    assert qc.mxfp4_moe(layer, torch.ones(1, 64, device=dev), 2)[1].tolist() == [[6, 3]]


@pytest.mark.parametrize("dtype", TYPES)
def test_moe_nonfinite_tokens(qc, dev, dtype):
    """NaN and infinite tokens make their own rows so, no other, and their experts are experts."""
    import torch
    layer, x, r, y, ids, _ = _run(qc, dev, 20, 6, 3, 64, 96, dtype, seed=5)
    X, R = x.to(dev), r.to(dev)
    bad = [0, 7, 19]
    X[0, 3], X[7, 63], X[19, 0] = float("nan"), float("inf"), float("-inf")
    got, gid, _ = qc.mxfp4_moe(layer, X, 3, residual=R)
    rest = [t for t in range(20) if t not in bad]
    assert torch.equal(got[rest], y[rest]) and torch.equal(gid[rest], ids[rest])
    assert bool((~torch.isfinite(got[bad])).any(1).all())
    assert bool(((gid >= 0) & (gid < 6)).all())


@pytest.mark.parametrize("where", ["gate_up", "down"])
def test_moe_scale_bytes(qc, dev, where):
    """Every block scale byte that a product of bf16 can hold; 255 is NaN."""
    import torch
    dim = inter = 64
    layer, values = _layer(qc, dev, 1, dim, inter, bias=False)
    codes, scales = (layer.tensors[2], layer.tensors[3]) if where == "gate_up" else (layer.tensors[4], layer.tensors[5])
    x = torch.zeros(1, dim, device=dev)
    for byte in list(range(0, 250, 7)) + [1, 2, 3, 120, 127, 128, 250]:
        e = byte - 127
        if where == "down":
            # y is down times hidden values near 1: in range of f32
            scales.fill_(byte)
            x.copy_(torch.from_numpy(np.random.default_rng(byte).standard_normal((1, dim))))
            vals = qc.dequantize_mxfp4(codes.view(-1, inter // 2), scales.view(-1, inter // 32)).double().cpu().numpy()
            v = (values[0], values[1], values[2], vals.reshape(1, dim, inter))
        else:
            # gate rows as they are (their act near 1), up rows under the byte
            scales[:, inter:].fill_(byte)
            x.copy_(torch.from_numpy(np.random.default_rng(byte).standard_normal((1, dim))))
            vals = qc.dequantize_mxfp4(codes.view(-1, dim // 2), scales.view(-1, dim // 32)).double().cpu().numpy()
            v = (values[0], values[1], vals.reshape(1, 2 * inter, dim), values[3])
        y = qc.mxfp4_moe(layer, x, 1)[0].double().cpu().numpy()
        want, _, _, tol = _reference(v, x.double().cpu().numpy(), 1, True, False, None, 1.0, HALF["float32"])
        rows = v[2][0] @ x[0].double().cpu().numpy()
        if np.abs(rows).max() > float(np.finfo(np.float32).max):
            # the f32 sum of a row is infinite, and every output has a part of it
            assert byte >= 249 and not np.isfinite(y).any()
            continue
        # products and bf16 parts below 2^-126 may count as 0: 64 of them under a factor of 8
        assert np.all(np.abs(y - want) <= tol + 2.0 ** -117), (byte, e, float(np.abs(y - want).max()))
    scales.view(-1)[5] = 255
    assert bool(torch.isnan(qc.mxfp4_moe(layer, x, 1)[0]).any())


@pytest.mark.parametrize("dtype", TYPES)
def test_moe_strides_and_aliases(qc, dev, dtype):
    """Rows of wider arrays at any alignment; y at the residual's place and at x's."""
    import torch
    layer, x, r, y, _, _ = _run(qc, dev, 21, 7, 2, 96, 64, dtype, seed=9)
    X, R = x.to(dev), r.to(dev)
    for extra in (16, 1):
        wide = torch.zeros(21, 3 * (96 + extra), dtype=X.dtype, device=dev)
        a, b, c = (wide[:, i * (96 + extra):][:, :96] for i in range(3))
        a.copy_(X)
        b.copy_(R)
        keep = wide.clone()
        got = qc.mxfp4_moe(layer, a, 2, residual=b, out=c)[0]
        assert got is c and torch.equal(c, y)
        keep[:, 2 * (96 + extra):][:, :96] = y
        assert torch.equal(wide, keep)
    other = R.clone()
    assert torch.equal(qc.mxfp4_moe(layer, X, 2, residual=other, out=other)[0], y)
    other = X.clone()
    assert torch.equal(qc.mxfp4_moe(layer, other, 2, residual=R, out=other)[0], y)


def test_moe_helper_refusals(qc, dev):
    import torch
    layer, _ = _layer(qc, dev, 4, 64, 32)
    x = torch.zeros(3, 64, device=dev)
    with pytest.raises(ValueError):
        qc.mxfp4_moe(layer, x[:, :32], 2)
    with pytest.raises(ValueError):
        qc.mxfp4_moe(layer, x, 2, residual=x.half())
    with pytest.raises(ValueError):
        qc.mxfp4_moe(layer, x.cpu(), 2)
    with pytest.raises(TypeError):
        qc.mxfp4_moe(layer, x.double(), 2)
    with pytest.raises(qc.QcError):
        qc.mxfp4_moe(layer, x, 5)
    r, b, *w = layer.tensors
    with pytest.raises(ValueError):
        qc.Mxfp4Moe(r, w[0][:3], *w[1:])
    with pytest.raises(ValueError):
        qc.Mxfp4Moe(r, *w, bias=b.double())
    with pytest.raises(ValueError):
        qc.Mxfp4Moe(r, w[0], w[1].int(), *w[2:])


@pytest.mark.parametrize("tokens,experts,top,dim,inter", [(1, 16, 4, 256, 128), (40, 8, 2, 128, 160)])
def test_moe_repeats_and_graph(qc, dev, tokens, experts, top, dim, inter):
    """Bit for bit the same again, on another stream and replayed with tokens that change, while eager calls of
    other sizes share the stream's workspace."""
    import torch
    layer, x, r, y, ids, weights = _run(qc, dev, tokens, experts, top, dim, inter, "bfloat16", seed=2)
    other, _ = _layer(qc, dev, 5, 64, 32)
    X, R = x.to(dev), r.to(dev)
    assert torch.equal(qc.mxfp4_moe(layer, X, top, residual=R)[0], y)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        out = torch.zeros_like(X)
        qc.mxfp4_moe(layer, X, top, residual=R, out=out)
        stream.synchronize()
        assert torch.equal(out, y)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            _, gid, gw = qc.mxfp4_moe(layer, X, top, residual=R, out=out)
        for _ in range(4):
            X.copy_(torch.randn_like(X))
            qc.mxfp4_moe(other, torch.randn(9, 64, device=dev), 3)
            graph.replay()
            stream.synchronize()
            want = qc.mxfp4_moe(layer, X, top, residual=R)
            assert torch.equal(out, want[0]) and torch.equal(gid, want[1]) and torch.equal(gw, want[2])


def test_moe_from_threads(qc, dev):
    """Calls of several host threads on one stream and on their own."""
    import threading

    import torch
    layers = [_layer(qc, dev, 8, 64 * (i + 1), 96, seed=i)[0] for i in range(3)]
    xs = [torch.randn(11, 64 * (i + 1), device=dev) for i in range(3)]
    want = [qc.mxfp4_moe(a, x, 2)[0] for a, x in zip(layers, xs)]
    torch.cuda.synchronize()
    shared, wrong = torch.cuda.Stream(), []

    def work(i, stream):
        with torch.cuda.stream(stream):
            for _ in range(20):
                y = qc.mxfp4_moe(layers[i], xs[i], 2)[0]
                stream.synchronize()
                if not torch.equal(y, want[i]):
                    wrong.append(i)

    for own in (False, True):
        threads = [threading.Thread(target=work, args=(i, torch.cuda.Stream() if own else shared)) for i in range(3)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    assert not wrong


@pytest.mark.parametrize("captured", [False, True])
def test_a_verification_step(qc, dev, captured):
    """Drafted trees through a layer, their accepted tokens kept, step after step: the operators together are what the
    ones that were there give token by token on the accepted path alone -- the same values in the cache to
    its 8 bits, and attention of the path's tokens near theirs."""
    import torch
    torch.manual_seed(3)
    heads, kvh, hd, hidden, page = 8, 2, 64, 128, 16
    rows = (heads + 2 * kvh) * hd
    wc, ws = qc.quantize_mxfp4(0.08 * torch.randn(rows, hidden, device=dev))
    oc, os_ = qc.quantize_mxfp4(0.05 * torch.randn(hidden, heads * hd, device=dev))
    layer, _ = _layer(qc, dev, 6, hidden, 96)
    cosine, sine = qc.rope_table(512, hd)
    seqs, n = 3, 9
    rng = np.random.default_rng(1)
    pages = 24
    cache = qc.kv8_cache(pages, kvh, page, hd)
    table = torch.from_numpy(rng.permutation(pages).astype(np.int32).reshape(seqs, 8)).to(dev)
    start = torch.arange(0, seqs * n + 1, n, dtype=torch.int32, device=dev)
    kv = torch.full((seqs,), 0, dtype=torch.int32, device=dev)
    batch = qc.Kv8Batch(table, start, kv, seqs * n, n, 128)
    # a tree of nine tokens: 0 - 1 - 3 - 6, 1 - 4, 0 - 2 - 5 - 7 - 8
    parent = [-1, 0, 0, 1, 1, 2, 3, 5, 7]
    depth = [0, 1, 1, 2, 2, 2, 3, 3, 4]
    bits = []
    for i, p in enumerate(parent):
        bits.append((1 << i) | (bits[p] if p >= 0 else 0))
    mask = torch.tensor(bits * seqs, dtype=torch.int32, device=dev).view(-1, 1)
    deep = torch.tensor(depth, dtype=torch.int32, device=dev)
    x = torch.zeros(seqs * n, hidden, dtype=torch.bfloat16, device=dev)
    kept = torch.zeros(seqs, n, dtype=torch.int32, device=dev)
    count = torch.zeros(seqs, dtype=torch.int32, device=dev)
    length = torch.zeros(seqs, dtype=torch.int32, device=dev)
    st = torch.zeros(1, dtype=torch.int32, device=dev)

    def step():
        xc, xs = qc.quantize_mxfp4(x, dev_status=st)
        y = qc.mxfp4_gemm(wc, ws, xc, xs, dtype=torch.bfloat16).unflatten(1, (heads + 2 * kvh, hd))
        pos = ((kv - n)[:, None] + deep[None]).flatten().contiguous()
        q = qc.kv8_rope_append(cache, batch, y[:, :heads], y[:, heads:heads + kvh], y[:, heads + kvh:], cosine, sine,
                               positions=pos, dev_status=st)
        a = qc.kv8_tree_attention(cache, batch, q, mask, dev_status=st)
        ac, as_ = qc.quantize_mxfp4(a.flatten(1), dev_status=st)
        h = x + qc.mxfp4_gemm(oc, os_, ac, as_, dtype=torch.bfloat16)
        out = qc.mxfp4_moe(layer, h, 2, residual=h)[0]
        qc.kv8_keep(cache, batch, kept, count, out=length, dev_status=st)
        return y, a, out

    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph = None
        if captured:
            kv.fill_(n)
            step()                                   # sizes the workspaces
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs = step()
            for t in cache.tensors:
                t.zero_()
        plain = qc.kv8_cache(pages, kvh, page, hd)       # the accepted paths only, by the operators that were there
        held = [0, 0, 0]
        paths = [[0, 1, 3, 6], [0, 2, 5, 7, 8], [0], [], [0, 2], [0, 1, 4], [0, 1, 2, 3, 4, 5, 6, 7, 8]]
        for rep in range(6):
            chosen = [paths[(rep + 2 * s) % 6] for s in range(seqs)]
            x.copy_(torch.randn(seqs * n, hidden, device=dev))
            K = np.zeros((seqs, n), np.int32)
            for s, p in enumerate(chosen):
                K[s, :len(p)] = p
            kept.copy_(torch.from_numpy(K))
            count.copy_(torch.tensor([len(p) for p in chosen], dtype=torch.int32))
            kv.copy_(torch.tensor([h + n for h in held], dtype=torch.int32))
            stream.synchronize()
            if captured:
                graph.replay()
                y, a, out = outs
            else:
                y, a, out = step()
            stream.synchronize()
            assert length.tolist() == [h + len(p) for h, p in zip(held, chosen)]
            for s, p in enumerate(chosen):
                if not p:
                    continue
                at = torch.tensor([s * n + i for i in p], device=dev)
                pos = torch.arange(held[s], held[s] + len(p), dtype=torch.int32, device=dev)
                k = qc.rope(y[at, heads:heads + kvh].float(), cosine, sine, pos)
                q = qc.rope(y[at, :heads].contiguous(), cosine, sine, pos)
                one = qc.Kv8Batch(table[s:s + 1].contiguous(), torch.tensor([0, len(p)], dtype=torch.int32, device=dev),
                                  torch.tensor([held[s] + len(p)], dtype=torch.int32, device=dev), len(p), len(p), 128)
                qc.kv8_append(plain, one, k, y[at, heads + kvh:].float())
                want = qc.kv8_attention(plain, one, q)
                # steps of 1/127 of a page's largest value (drafted tokens that went away may have widened them):
                # a percent of a normal value, in keys and in values
                assert ((a[at].double() - want.double()).norm() / want.double().norm()).item() < 0.05
                held[s] += len(p)
            whole = qc.Kv8Batch(table, torch.tensor([0] + list(np.cumsum(held)), dtype=torch.int32, device=dev),
                                torch.tensor(held, dtype=torch.int32, device=dev), max(1, sum(held)), max(1, max(held)), 128)
            for got, want, scale in zip(qc.kv8_gather(cache, whole), qc.kv8_gather(plain, whole), cache.tensors[2:]):
                # each value has been rounded a few times to half a step of at most the cache's largest scale
                assert float((got - want).abs().max()) <= 0.5 * (rep + 3) * float(scale.max())
            assert bool(torch.isfinite(out).all())
    assert st.item() == 0



def _long_rows(qc, dev, tokens, experts, top, dim, inter=32, blocks=12):
    """A layer of long rows, run and compared at its result's ends, middle and some rows between: x is zero but for
    some blocks, so that the sums are those of 32 * blocks values.  (layer, x, y)"""
    import torch
    g = torch.Generator(device=dev)
    g.manual_seed(26)
    rng = np.random.default_rng(26)
    at = np.unique(np.concatenate([[0, 1, dim // 32 - 1, dim // 64], rng.choice(dim // 32, blocks - 4, replace=False)]))
    A = torch.from_numpy(at).to(dev)
    columns = (32 * A[:, None] + torch.arange(32, device=dev)).flatten()
    codes = lambda *shape: torch.randint(0, 256, shape, generator=g, device=dev, dtype=torch.uint8)
    guc, dc = codes(experts, 2 * inter, dim // 2), codes(experts, dim, inter // 2)
    gus, ds = (torch.full(c.shape[:2] + (c.shape[2] // 16,), 127 - 6, dtype=torch.uint8, device=dev) for c in (guc, dc))
    router = torch.zeros(experts, dim, dtype=torch.bfloat16, device=dev)
    router[:, columns] = (torch.randn(experts, columns.numel(), generator=g, device=dev) / 8).to(torch.bfloat16)
    layer = qc.Mxfp4Moe(router, guc, gus, dc, ds)
    short = torch.from_numpy(rng.standard_normal((tokens, columns.numel()))).to(torch.bfloat16)
    x = torch.zeros(tokens, dim, dtype=torch.bfloat16, device=dev)
    x[:, columns] = short.to(dev)
    out = torch.zeros_like(x)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        free = torch.cuda.mem_get_info()[0]
        y, ids, weights = qc.mxfp4_moe(layer, x, top, out=out)
        stream.synchronize()
        scratch = free - torch.cuda.mem_get_info()[0]
    rows = np.unique(np.concatenate([np.arange(512), dim // 2 + np.arange(-512, 512), dim - 512 + np.arange(512),
                                     rng.integers(0, dim, 2048)]))
    R = torch.from_numpy(rows).to(dev)
    f64 = lambda c, sc: qc.dequantize_mxfp4(c.flatten(0, 1).contiguous(), sc.flatten(0, 1).contiguous()).double().cpu().numpy()
    gu = f64(guc.unflatten(2, (dim // 32, 16))[:, :, A].flatten(2), gus[:, :, A]).reshape(experts, 2 * inter, -1)
    dn = f64(dc[:, R], ds[:, R]).reshape(experts, len(rows), inter)
    some = sorted({0, tokens // 3, tokens // 2, tokens - 1})
    values = (router[:, columns].double().cpu().numpy(), np.zeros(experts), gu, dn)
    want, wid, wp, tol = _reference(values, short[some].double().numpy(), top, True, False, np.zeros((len(some), len(rows))), 1.0,
                                    HALF["bfloat16"])
    assert np.array_equal(ids[some].cpu().numpy(), wid)
    assert np.all(np.abs(weights[some].double().cpu().numpy() - wp) <= 2.0 ** -23 * np.abs(wp))
    assert np.all(np.abs(y[some][:, R].double().cpu().numpy() - want) <= tol)
    assert bool(torch.isfinite(y).all()) and float((y == 0).float().mean()) < 0.01   # every row is written
    return scratch


def test_moe_longest_rows(qc, dev):
    """Rows of 2^26 values through one expert: 64 work-items of the pair form's last launch a value would pass 32 bits."""
    _long_rows(qc, dev, 1, 1, 1, 1 << 26)


def test_moe_scratch_of_long_rows(qc, dev):
    """200 tokens through all of 64 experts of 2^17: their pairs' outputs would be 6.7 GB, and go in passes."""
    assert _long_rows(qc, dev, 200, 64, 64, 1 << 17) <= 1.2 * (1 << 30)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,experts,top,dim,inter", [
    # the second product's K in two, four and eight parts, some beginning at odd steps, for one to four tiles of columns
    (20, 2, 1, 96, 2080), (20, 2, 1, 96, 4128), (17, 1, 1, 32, 8224), (40, 2, 1, 64, 3104), (70, 2, 1, 288, 2080),
    # pair by pair: hidden values that LDS holds in two or more parts, with and without idle waves, ...
    (5, 3, 3, 64, 1056), (10, 2, 1, 32, 1632), (1, 2, 1, 64, 16416), (3, 2, 2, 96, 5152),
    # ... and x
    (1, 2, 1, 8224, 64), (2, 3, 3, 8192 + 96, 32), (1, 4, 2, 16416, 32)])
def test_moe_wide_experts(qc, dev, dtype, tokens, experts, top, dim, inter):
    print(f"moe {dtype} {tokens} tokens, {top} of {experts}, {dim} x {inter}", flush=True)
    _run(qc, dev, tokens, experts, top, dim, inter, dtype, seed=inter + tokens)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,top,inter", [(5, 3, 96), (4, 2, 2080), (40, 1, 2080)])
def test_moe_nonfinite_tokens_alone(qc, dev, dtype, tokens, top, inter):
    """As above of few pairs, and of K in parts: the other rows keep their bits."""
    import torch
    layer, x, r, y, ids, weights = _run(qc, dev, tokens, 6, top, 64, inter, dtype, seed=5)
    X, R = x.to(dev), r.to(dev)
    X[0, 3], X[2, 63] = float("nan"), float("-inf")
    got, gid, gw = qc.mxfp4_moe(layer, X, top, residual=R)
    rest = [t for t in range(tokens) if t not in (0, 2)]
    assert torch.equal(got[rest], y[rest]) and torch.equal(gid[rest], ids[rest]) and torch.equal(gw[rest], weights[rest])
    assert bool((~torch.isfinite(got[[0, 2]])).any(1).all())
    assert bool(((gid >= 0) & (gid < 6)).all())


@pytest.mark.parametrize("where", ["gate", "up", "down"])
@pytest.mark.parametrize("tokens", [3, 40])
def test_moe_marked_blocks(qc, dev, tokens, where):
    """One block's scale byte 255: NaN in the output row that holds it (down), or in whatever goes through its expert
    (gate, up), and the same bits everywhere else."""
    import torch
    dim, inter, experts = 96, 64, 3
    layer, _ = _layer(qc, dev, experts, dim, inter, seed=11)
    x = torch.randn(tokens, dim, generator=torch.Generator(device=dev).manual_seed(3), device=dev)
    y, ids, weights = qc.mxfp4_moe(layer, x, 1)
    assert bool(torch.isfinite(y).all()) and len(ids.unique()) > 1
    e = int(ids[0, 0])
    scales = layer.tensors[5 if where == "down" else 3]
    row = {"gate": 37, "up": inter + 37, "down": 50}[where]
    scales[e, row, 1] = 255
    got, gid, gw = qc.mxfp4_moe(layer, x, 1)
    assert torch.equal(gid, ids) and torch.equal(gw, weights)
    marked = torch.zeros_like(y, dtype=torch.bool)
    if where == "down":
        marked[ids[:, 0] == e, row] = True
    else:
        marked[ids[:, 0] == e] = True
    assert torch.equal(torch.isnan(got), marked) and torch.equal(got[~marked], y[~marked])


def _kept(v, n):
    """What n terms of e4m3 hold of blocks of 32: the stated steps in f64."""
    top = np.repeat(np.abs(v).reshape(*v.shape[:-1], -1, 32).max(-1), 32, -1)
    scale = 2.0 ** (np.frexp(top)[1] - 8)
    left, sum_ = v.copy(), np.zeros_like(v)
    for i in range(n):
        t = left / scale
        if i < n - 1:
            t = np.rint(t * 4) / 4
        step = 2.0 ** np.maximum(np.frexp(t)[1] - 4, -9)     # three bits after the first
        t = np.rint(t / step) * step * scale
        sum_, left, scale = sum_ + t, left - t, scale / 16
    return sum_


def _one_value_rows(x, dtype, keep):
    """(h, what x's and h's terms may be off by, what h's n terms hold of it) of rows with one value each."""
    fits = {"float32": 6, "float16": 3, "bfloat16": 2}[dtype]
    shifted = lambda v: v[:, (np.arange(v.shape[1]) + 7) % v.shape[1]]
    tops = lambda v: np.repeat(np.abs(v).reshape(*v.shape[:-1], -1, 32).max(-1), 32, -1)
    small = lambda v, n: 1.1 * 2.0 ** (-4 * n - 6) * tops(v)
    h, ex = 32.0 * x * shifted(x), small(x, fits)
    of_x = 32.0 * (ex * shifted(x) + x * shifted(ex) + ex * shifted(ex))
    return h, of_x + 2.0 ** (-4 * keep) * h + small(h, keep)


@pytest.mark.parametrize("dtype,terms,outlier,more", [
    ("float32", 6, 1, 0.0), ("float32", 6, 4096, 0.1), ("float16", 4, 1, 0.08), ("float16", 4, 64, 0.0),
    ("bfloat16", 3, 1, 0.4), ("bfloat16", 3, 256, 0.0)])
@pytest.mark.parametrize("tokens", [3, 40])
def test_moe_terms(qc, dev, tokens, dtype, terms, outlier, more):
    """The bits that x and the hidden values are held with, where no sum hides them: every row of the weights has one
    value, act(v) = v for gates above 32, and -y as residual leaves what y's rounding lost.

    n terms hold a value within 2^-4n of itself and 1.1 2^(-4n - 6) of its block's largest (x: all of its bits, but for
    the latter); the gate's, the up's and their product's roundings, and those of six terms' sums, are 2^-24 each; y is
    rounded once.  `more`: the share of values for which hidden values of one term fewer would be further off (0: what
    x's terms, or f32 sums, may be off by hides it)."""
    import torch
    K, half = 64, HALF[dtype]
    one = lambda value, shift: torch.from_numpy(np.float32(value * np.eye(K)[(np.arange(K) + shift) % K])).to(dev)
    guc, gus = qc.quantize_mxfp4(torch.cat([one(32.0, 0), one(1.0, 7)]))
    dc, ds = qc.quantize_mxfp4(one(1.0, 0))
    layer = qc.Mxfp4Moe(torch.zeros(1, K, device=dev), guc[None], gus[None], dc[None], ds[None])
    x = np.random.default_rng(tokens).uniform(1, 2 - 2.0 ** -8, (tokens, K))
    x[:, [5, 40]] *= outlier
    x = torch.from_numpy(x).to(getattr(torch, dtype))
    want, held = _one_value_rows(x.double().numpy(), dtype, terms)
    tol = held + 10 * 2.0 ** -24 * want
    # the oracle's terms are within that, and one fewer are not
    assert np.all(np.abs(_kept(want, terms) - want) <= held)
    assert np.mean(np.abs(_kept(want, terms - 1) - want) > tol) >= more
    y = qc.mxfp4_moe(layer, x.to(dev), 1)[0]
    got = y.double().cpu().numpy()
    assert np.all(np.abs(got - want) <= tol + half * want * 1.001)
    rest = qc.mxfp4_moe(layer, x.to(dev), 1, residual=-y)[0].double().cpu().numpy()
    assert np.all(np.abs(rest - (want - got)) <= tol + half * 1.001 * (np.abs(want - got) + tol))
