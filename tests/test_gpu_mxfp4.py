"""GPU: MXFP4 quantisation bit for bit against the definition, and products
against 64-bit arithmetic."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)
EPS = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def reference(x):
    """(codes 0..15 [rows][dim], scale bytes) of f64 values, straight from the definition."""
    rows, dim = x.shape
    b = x.reshape(rows, dim // 32, 32)
    top = np.abs(b).max(2)
    e = np.where(top > 0, np.frexp(np.where(top > 0, top, 1.0))[1] - 1 - 2, -127)
    e = np.clip(e, -127, 127)
    a = np.abs(b) * np.exp2(-e.astype(np.float64))[:, :, None]
    d = np.abs(a[..., None] - GRID)
    near = d.min(-1, keepdims=True)
    hit = d == near
    first, last = hit.argmax(-1), 7 - hit[..., ::-1].argmax(-1)
    code = np.where(first % 2 == 0, first, last)        # ties: the even code
    code = code + 8 * np.signbit(b)
    return code.reshape(rows, dim), (e + 127).astype(np.uint8)


def values(codes, scales):
    c = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)
    v = np.where(c & 8, -1.0, 1.0) * GRID[c & 7]
    step = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return v * np.repeat(step, 32, axis=1)


def packed(code):
    return (code[:, 0::2] | code[:, 1::2] << 4).astype(np.uint8)


def _check(qc, dev, x, stride_pad=0):
    import torch
    rows, dim = x.shape
    X = torch.full((rows, dim + stride_pad), 3.0, dtype=x.dtype, device=dev)[:, :dim]
    X.copy_(x)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    codes, scales = qc.quantize_mxfp4(X, dev_status=st)
    want, wscale = reference(x.double().numpy())
    assert st.item() == 0
    assert np.array_equal(scales.cpu().numpy(), wscale)
    assert np.array_equal(codes.cpu().numpy(), packed(want))
    again = qc.quantize_mxfp4(X)                        # the blocking form
    assert torch.equal(again[0], codes) and torch.equal(again[1], scales)
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        got = qc.dequantize_mxfp4(codes, scales, dtype=dt)
        v = torch.from_numpy(values(codes.cpu().numpy(), scales.cpu().numpy())).float().to(dt)
        assert torch.equal(got.cpu(), v), dt


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,dim,pad", [(1, 32, 0), (3, 96, 0), (16, 4096, 0), (7, 160, 3),
                                          (130, 2752, 8), (5, 14336, 1), (1025, 64, 0)])
def test_quantize(qc, dev, dtype, rows, dim, pad):
    import torch
    print(f"mxfp4 quantize {dtype} {rows}x{dim}", flush=True)
    g = torch.Generator().manual_seed(rows + dim)
    x = torch.randn(rows, dim, generator=g)
    x[torch.rand(rows, dim, generator=g) < 0.01] *= 30
    _check(qc, dev, x.to(getattr(torch, dtype)), pad)


def test_quantize_every_border(qc, dev):
    """All borders between codes and their neighbours in f32, at scales from the smallest
    to the largest; blocks of zeros, of subnormals, signed zeros."""
    import torch
    base = np.array([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7.75], dtype=np.float32)
    near = np.concatenate([base, np.nextafter(base, np.float32(0)), np.nextafter(base, np.float32(8))])
    near = np.minimum(np.concatenate([near, -near]), np.float32(7.999))
    rows = []
    for top in (4.0, 5.5, 7.9):                         # what fixes the block's exponent
        for part in near.reshape(-1, 16):
            rows.append(np.concatenate([part, [top], np.zeros(15)]).astype(np.float32))
    rows = np.array(rows)
    for e in (-129, -127, -126, -100, -1, 0, 1, 60, 125):
        x = np.ldexp(rows.astype(np.float64), e).astype(np.float32)
        _check(qc, dev, torch.from_numpy(x))
    x = np.zeros((5, 32), np.float32)
    x[1] = -0.0
    x[2, 3] = np.float32(1e-45)
    x[3] = np.float32(-1e-40)
    x[4, 0] = np.finfo(np.float32).max
    _check(qc, dev, torch.from_numpy(x))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_quantize_nonfinite(qc, dev, dtype):
    """Blocks with NaN or infinities stay as they were; the others are done."""
    import torch
    x = torch.randn(4, 96, device=dev).to(getattr(torch, dtype))
    x[0, 40], x[2, 0], x[3, 95] = float("nan"), float("inf"), float("-inf")
    codes = torch.full((4, 48), 85, dtype=torch.uint8, device=dev)
    scales = torch.full((4, 3), 9, dtype=torch.uint8, device=dev)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    call = lambda status: qc.lib.qc_hip_quantize_mxfp4(
        x.data_ptr(), qc.STORAGE[{"float32": "f32", "float16": "f16", "bfloat16": "bf16"}[dtype]], 96,
        codes.data_ptr(), scales.data_ptr(), 4, 96, status, qc._stream(None))
    assert call(None) == 3
    assert torch.all(codes == 85) and torch.all(scales == 9)
    assert call(st.data_ptr()) == 0
    assert st.item() == 3
    want, wscale = reference(torch.where(torch.isfinite(x), x, 0).double().cpu().numpy())
    want = packed(want)
    for r in range(4):
        for b in range(3):
            bad = (r, b) in ((0, 1), (2, 0), (3, 2))
            got = codes[r, 16 * b:16 * b + 16].cpu().numpy()
            assert np.array_equal(got, np.full(16, 85) if bad else want[r, 16 * b:16 * b + 16]), (r, b)
            assert scales[r, b].item() == (9 if bad else wscale[r, b])


@pytest.fixture(params=range(8), ids=["auto", "32x32", "64x32", "64x64", "128x64", "128x128", "256x128", "256x256"])
def route(request, qc):
    """Every tile of the product at every size."""
    qc.set_mxfp4_gemm_route(request.param)
    yield request.param
    qc.set_mxfp4_gemm_route(0)


def _matrix(g, rows, k, sigma=1.0, spread=2):
    """Random codes (all 16) and scale bytes."""
    codes = g.integers(0, 256, (rows, k // 2), dtype=np.uint8)
    scales = (127 + g.integers(-spread, spread + 1, (rows, k // 32))).astype(np.uint8)
    return codes, scales


def _product(qc, dev, g, m, n, k, dtype="float32", spread=2, offset=0):
    import torch
    w, ws = _matrix(g, n, k, spread=spread)
    x, xs = _matrix(g, m, k, spread=spread)
    up = lambda a: torch.from_numpy(a).to(dev)
    y = torch.full((m, n), float("nan"), dtype=getattr(torch, dtype), device=dev)
    qc.mxfp4_gemm(up(w), up(ws), up(x), up(xs), y=y)
    W, X = values(w, ws), values(x, xs)
    want, mag = X @ W.T, np.abs(X) @ np.abs(W).T
    # products are exact; at most k / 32 + 8 additions of partial sums no larger than
    # the sum of magnitudes, then the output's rounding
    tol = (k / 32 + 8) * 2.0 ** -23 * mag + EPS[dtype] * (1 + 2.0 ** -10) * np.abs(want) + 2.0 ** -25
    err = np.abs(y.double().cpu().numpy() - want)
    assert np.all(err <= tol), (m, n, k, float(np.nanmax(err / tol)))
    return y


@pytest.mark.parametrize("m,n,k", [
    (1, 1, 32), (1, 17, 32), (2, 16, 64), (1, 300, 4096), (3, 33, 96), (4, 100, 992), (5, 64, 128),
    (8, 257, 2752), (15, 48, 512), (16, 128, 1024), (17, 129, 544), (31, 40, 480), (32, 96, 14336),
    (33, 65, 2048), (48, 130, 160), (64, 64, 256), (65, 255, 800), (77, 341, 2752), (100, 31, 4096),
    (128, 128, 512), (129, 257, 608), (200, 1000, 768), (257, 300, 32), (300, 513, 1056),
    (511, 129, 2048), (700, 1025, 320)])
def test_product_shapes(qc, dev, route, m, n, k):
    print(f"mxfp4 product {m}x{n}x{k}", flush=True)
    _product(qc, dev, np.random.default_rng(m * n + k), m, n, k)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("m,n,k", [(1, 512, 1024), (12, 200, 1056), (40, 77, 512), (300, 260, 608)])
def test_product_types(qc, dev, route, dtype, m, n, k):
    # scales that keep the sums within f16
    _product(qc, dev, np.random.default_rng(k + m), m, n, k, dtype, spread=1)


@pytest.mark.parametrize("m", [1, 9, 40, 150])
def test_product_wide_scales(qc, dev, route, m):
    """Scales over 2^+-40: a block's product is exact whatever the others are."""
    _product(qc, dev, np.random.default_rng(m), m, 70, 640, spread=20)


@pytest.mark.parametrize("at", [(1, 0), (0, 3), (2, 1)])
def test_product_scales_at_any_byte(qc, dev, route, at):
    """Scales cut out of a larger array begin at any byte; so may y's elements."""
    import torch
    g = np.random.default_rng(6)
    m, n, k = 37, 70, 384
    w, ws = _matrix(g, n, k)
    x, xs = _matrix(g, m, k)
    up = lambda a: torch.from_numpy(a).to(dev)

    def cut(a, off):
        room = torch.zeros(a.size + 8, dtype=torch.uint8, device=dev)
        view = room[off:off + a.size].view(a.shape)
        view.copy_(up(a))
        return view
    want = qc.mxfp4_gemm(up(w), up(ws), up(x), up(xs))
    y = torch.zeros(m * n + 1, device=dev)[1:].view(m, n)
    qc.mxfp4_gemm(up(w), cut(ws, at[0]), up(x), cut(xs, at[1]), y=y)
    assert torch.equal(y, want)


@pytest.mark.parametrize("m", [1, 5, 33, 140])
def test_product_special_scales(qc, dev, route, m):
    """A NaN scale of a row reaches that row's (column's) outputs only; the smallest and
    largest scales."""
    import torch
    g = np.random.default_rng(3)
    n, k = 80, 256
    w, ws = _matrix(g, n, k)
    x, xs = _matrix(g, m, k)
    ws[7, 3], xs[m // 2, 1] = 255, 255
    ws[9] = 0
    ws[11], xs[0, 0] = 230, 20
    up = lambda a: torch.from_numpy(a).to(dev)
    y = qc.mxfp4_gemm(up(w), up(ws), up(x), up(xs)).cpu().numpy()
    nan = np.zeros((m, n), bool)
    nan[:, 7] = True
    nan[m // 2] = True
    assert np.array_equal(np.isnan(y), nan)
    W, X = values(w, ws), values(x, xs)
    want, mag = X @ W.T, np.abs(X) @ np.abs(W).T
    with np.errstate(invalid="ignore"):
        ok = np.abs(y - want) <= 16 * 2.0 ** -23 * mag + 2.0 ** -126
    assert np.all(ok | nan)


def test_quantized_product_of_floats(qc, dev):
    """Activations and weights quantised on the GPU, then multiplied: the product of
    what the codes stand for, and near the unquantised product (4-bit steps: a relative
    2^-2 at most an element, normal data some 10%)."""
    import torch
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(20, 1024, generator=g, device=dev, dtype=torch.bfloat16)
    w = 0.02 * torch.randn(200, 1024, generator=g, device=dev)
    xc, xs = qc.quantize_mxfp4(x)
    wc, ws = qc.quantize_mxfp4(w)
    y = qc.mxfp4_gemm(wc, ws, xc, xs).double().cpu()
    X, W = (qc.dequantize_mxfp4(c, s).double().cpu() for c, s in ((xc, xs), (wc, ws)))
    want, mag = X @ W.T, X.abs() @ W.abs().T
    assert torch.all((y - want).abs() <= 40 * 2.0 ** -23 * mag)
    full = x.double().cpu() @ w.double().cpu().T
    assert ((y - full).norm() / full.norm()).item() < 0.25


def test_product_repeats_bit_for_bit(qc, dev, route):
    import torch
    g = np.random.default_rng(8)
    for m in (1, 24, 130):
        w, ws, x, xs = (torch.from_numpy(a).to(dev) for a in (*_matrix(g, 1500, 4096), *_matrix(g, m, 4096)))
        first = qc.mxfp4_gemm(w, ws, x, xs)
        for _ in range(3):
            assert torch.equal(qc.mxfp4_gemm(w, ws, x, xs), first)


@pytest.mark.parametrize("m,n,k", [(1, 1000, 4096), (20, 300, 2048), (260, 512, 1024)])
def test_graph_replay(qc, dev, route, m, n, k):
    """quantise + product captured, replayed with other work between on the same stream."""
    import torch
    g = torch.Generator(device=dev).manual_seed(2)
    wc, ws = qc.quantize_mxfp4(torch.randn(n, k, generator=g, device=dev))
    x = torch.randn(m, k, generator=g, device=dev)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    y, y2 = torch.empty(m, n, device=dev), torch.empty(m, n, device=dev)
    other = qc.quantize_mxfp4(torch.randn(m, k, generator=g, device=dev))
    s = torch.cuda.Stream()
    torch.cuda.synchronize()

    def call():
        xc, xs = qc.quantize_mxfp4(x, dev_status=st)
        qc.mxfp4_gemm(wc, ws, xc, xs, y=y)

    with torch.cuda.stream(s):
        call()
    torch.cuda.synchronize()
    want = y.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        call()
    for rep in range(3):
        with torch.cuda.stream(s):
            y.fill_(float("nan"))
            qc.mxfp4_gemm(wc, ws, *other, y=y2)
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), rep
    del graph
