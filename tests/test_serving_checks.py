"""CPU checks of the rotary, 8-bit cache and MXFP4 entry points: every refusal
comes before the device is touched (no GPU needed; the pointers are never read)."""
import ctypes

import pytest

P = 4096      # a 16-byte aligned address that is never read
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def q():
    import quixicore_hip
    return quixicore_hip


def _scaling(q, kind, factor=2.0, original=4096.0, low=1.0, high=32.0, magnitude=1.0):
    return ctypes.byref(q.RopeScaling(kind, factor, original, low, high, magnitude))


def test_rope_table_refusals(q):
    call = q.lib.qc_hip_rope_table

    def table(c=P, s=P, first=0, count=8, dim=64, base=1e4, scaling=None):
        return call(c, s, first, count, dim, base, scaling, None)

    for bad in (dict(count=0), dict(count=-1), dict(first=-1), dict(dim=0), dict(dim=63),
                dict(dim=514), dict(first=1 << 31, count=1), dict(count=(1 << 31) + 1),
                dict(first=(1 << 63) - 1, count=2)):
        assert table(**bad) == 1, bad
    for bad in (dict(c=None), dict(s=None), dict(base=1.0), dict(base=NAN), dict(base=INF),
                dict(base=-2.0)):
        assert table(**bad) == 3, bad
    for args in ((5,), (-1,), (1, 0.5), (1, NAN), (2, INF), (3, 2.0, 0.0), (3, 2.0, NAN),
                 (4, 2.0, 4096.0, 0.0), (4, 2.0, 4096.0, 4.0, 4.0), (3, 2.0, 4096.0, 1.0, INF),
                 (0, 1.0, 0.0, 0.0, 0.0, 0.0), (1, 2.0, 0.0, 0.0, 0.0, NAN)):
        assert table(scaling=_scaling(q, *args)) == 3, args
    assert table(dim=2, scaling=_scaling(q, 2)) == 3


def test_rope_refusals(q):
    call = q.lib.qc_hip_rope

    def rope(x=P, y=P, type=0, tokens=4, heads=2, hd=64, rd=64, xt=128, xh=64, yt=128, yh=64, c=P,
             s=P, pos=P, most=16, layout=0):
        return call(x, y, type, tokens, heads, hd, rd, xt, xh, yt, yh, c, s, pos, most, layout, P,
                    None)

    for bad in (dict(tokens=0), dict(heads=0), dict(hd=-1), dict(rd=0), dict(rd=63), dict(rd=66),
                dict(most=0), dict(xt=127), dict(xh=63), dict(yt=0), dict(yh=-64),
                dict(tokens=1 << 40), dict(most=1 << 31), dict(heads=1 << 40),
                dict(xt=(1 << 62)), dict(hd=1 << 62)):
        assert rope(**bad) == 1, bad
    assert rope(type=3) == 2
    for bad in (dict(x=None), dict(y=None), dict(c=None), dict(s=None), dict(pos=None),
                dict(layout=2), dict(layout=-1), dict(yt=256), dict(xt=256)):
        assert rope(**bad) == 3, bad


def test_rope_strides_that_overlap(q):
    """Tokens and heads in neither order apart: refused, for x and for y; the pointers are not read."""
    call = q.lib.qc_hip_rope
    for tokens, heads, token, head in ((4, 2, 64, 192), (4, 2, 127, 255), (2, 3, 128, 100), (3, 3, 64, 64),
                                       (4, 2, 63, 1024), (4, 2, 1 << 62, 64), (4, 2, 64, 1 << 62), (4, 2, 64, -256)):
        for x, y in (((token, head), (1024, 64)), ((1024, 64), (token, head))):
            assert call(P, P, 0, tokens, heads, 64, 64, *x, *y, P, P, P, 16, 0, P, None) == 1, (tokens, heads, token, head)


def _cache(q, **kw):
    f = dict(k_codes=P, v_codes=P, k_scales=P, v_scales=P, pages=8, kv_heads=2, page_tokens=16,
             head_dim=64)
    f.update(kw)
    c = q.Kv8Cache.__new__(q.Kv8Cache)
    for k, v in f.items():
        setattr(c, k, v)
    return c


def _batch(q, **kw):
    f = dict(block_table=P, seq_start=P, kv_len=P, seqs=3, columns=4, tokens=9, max_new=5,
             max_kv=60)
    f.update(kw)
    b = q.Kv8Batch.__new__(q.Kv8Batch)
    for k, v in f.items():
        setattr(b, k, v)
    return b


CACHE_SHAPES = (dict(pages=0), dict(kv_heads=0), dict(page_tokens=8), dict(page_tokens=24),
                dict(page_tokens=512), dict(head_dim=8), dict(head_dim=72), dict(head_dim=272),
                dict(head_dim=0), dict(pages=1 << 31), dict(pages=1 << 62), dict(kv_heads=1 << 30))
BATCH_SHAPES = (dict(seqs=0), dict(columns=0), dict(tokens=0), dict(max_new=0), dict(max_kv=0),
                dict(max_kv=65), dict(seqs=1 << 31), dict(tokens=1 << 31),
                dict(columns=1 << 30), dict(columns=(1 << 26) + 1), dict(seqs=1 << 62))


@pytest.mark.parametrize("entry", ["append", "gather", "attention"])
def test_kv8_refusals(q, entry):
    lib = q.lib

    def call(cache, batch, a=P, b=P, sa=None, sb=None, type=0, heads=4, scale=0.125, causal=1,
             window=0):
        row = 128 if entry != "attention" else 64 * heads
        sa, sb = sa or max(row, 1), sb or max(row, 1)
        if entry == "attention":
            return lib.qc_hip_kv8_attention(cache, batch, a, sa, b, sb, type, heads, scale, causal,
                                            window, P, None)
        if entry == "append":
            return lib.qc_hip_kv8_append(cache, batch, a, sa, b, sb, type, P, None)
        return lib.qc_hip_kv8_gather(cache, batch, a, sa, b, sb, type, 1, P, None)

    cache, batch = _cache(q), _batch(q)
    ref = ctypes.byref
    assert call(None, ref(batch)) == 3 and call(ref(cache), None) == 3
    for bad in CACHE_SHAPES:
        assert call(ref(_cache(q, **bad)), ref(batch)) == 1, bad
    for bad in BATCH_SHAPES:
        assert call(ref(cache), ref(_batch(q, **bad))) == 1, bad
    for bad in (dict(sa=127), dict(sb=127), dict(sa=1 << 62)):
        assert call(ref(cache), ref(batch), **bad) == 1, bad
    assert call(ref(cache), ref(batch), type=7) == 2
    for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
        assert call(ref(_cache(q, **{name: None})), ref(batch)) == 3, name
    for name in ("k_codes", "v_codes"):
        assert call(ref(_cache(q, **{name: P + 8})), ref(batch)) == 3, name
    for name in ("block_table", "seq_start", "kv_len"):
        assert call(ref(cache), ref(_batch(q, **{name: None}))) == 3, name
    assert call(ref(cache), ref(batch), a=None) == 3
    assert call(ref(cache), ref(batch), b=None) == 3
    if entry == "attention":
        for bad in (dict(heads=0), dict(heads=3), dict(heads=-2), dict(window=-1),
                    dict(heads=1 << 40)):
            assert call(ref(cache), ref(batch), **bad) == 1, bad
        for bad in (dict(scale=NAN), dict(scale=INF), dict(causal=0, window=4)):
            assert call(ref(cache), ref(batch), **bad) == 3, bad


def test_knobs(q):
    for f, most in ((q.lib.qc_hip_set_kv8_attention_route, 3), (q.lib.qc_hip_set_mxfp4_gemm_route, 7)):
        assert f(-1) == 3 and f(most + 1) == 3
        assert f(most) == 0 and f(0) == 0


def test_mxfp4_refusals(q):
    lib = q.lib
    quant = lambda x=P, type=0, stride=64, c=P, s=P, rows=4, dim=64: lib.qc_hip_quantize_mxfp4(
        x, type, stride, c, s, rows, dim, P, None)
    for bad in (dict(rows=0), dict(dim=0), dict(dim=48), dict(dim=-32), dict(stride=63),
                dict(rows=1 << 62), dict(stride=1 << 62)):
        assert quant(**bad) == 1, bad
    assert quant(type=-1) == 2
    for bad in (dict(x=None), dict(c=None), dict(s=None), dict(c=P + 4)):
        assert quant(**bad) == 3, bad
    deq = lambda c=P, s=P, out=P, type=0, rows=4, dim=64: lib.qc_hip_dequantize_mxfp4(
        c, s, out, type, rows, dim, None)
    for bad in (dict(rows=0), dict(dim=33), dict(rows=1 << 62)):
        assert deq(**bad) == 1, bad
    assert deq(type=4) == 2
    for bad in (dict(c=None), dict(s=None), dict(out=None), dict(c=P + 8)):
        assert deq(**bad) == 3, bad
    gemm = lambda w=P, ws=P, x=P, xs=P, y=P, type=0, m=2, n=3, k=64: lib.qc_hip_mxfp4_gemm(
        w, ws, x, xs, y, type, m, n, k, None)
    for bad in (dict(m=0), dict(n=0), dict(k=0), dict(k=31), dict(m=1 << 62), dict(n=1 << 40),
                dict(k=1 << 40), dict(m=1 << 31), dict(k=(1 << 27) + 32)):
        assert gemm(**bad) == 1, bad
    assert gemm(type=9) == 2
    for bad in (dict(w=None), dict(ws=None), dict(x=None), dict(xs=None), dict(y=None),
                dict(w=P + 2), dict(x=P + 12)):
        assert gemm(**bad) == 3, bad


def test_helpers_refuse_cpu_tensors(q):
    """No CPU fallback: the Python helpers name the device they want."""
    import torch
    if not torch.cuda.is_available():
        pytest.skip("looks up the current device")
    with pytest.raises(ValueError):
        q.quantize_mxfp4(torch.zeros(1, 32))
    with pytest.raises(ValueError):
        q.mxfp4_gemm(*[torch.zeros(1, 16, dtype=torch.uint8)] * 4)
