"""CPU checks of the entry points for drafted tokens and experts: every refusal comes
before the device is touched (no GPU needed; the pointers are never read)."""
import ctypes

import pytest

from test_serving_checks import BATCH_SHAPES, CACHE_SHAPES, INF, NAN, P, _batch, _cache, q  # noqa: F401

ref = ctypes.byref


def _common(q, call):
    """What every call over a cache and a batch refuses."""
    cache, batch = _cache(q), _batch(q)
    assert call(None, ref(batch)) == 3 and call(ref(cache), None) == 3
    for bad in CACHE_SHAPES:
        assert call(ref(_cache(q, **bad)), ref(batch)) == 1, bad
    for bad in BATCH_SHAPES:
        assert call(ref(cache), ref(_batch(q, **bad))) == 1, bad
    for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
        assert call(ref(_cache(q, **{name: None})), ref(batch)) == 3, name
    for name in ("k_codes", "v_codes"):
        assert call(ref(_cache(q, **{name: P + 8})), ref(batch)) == 3, name
    for name in ("block_table", "seq_start", "kv_len"):
        assert call(ref(cache), ref(_batch(q, **{name: None}))) == 3, name
    return lambda **kw: call(ref(cache), ref(batch), **kw)


def test_rope_append_refusals(q):  # noqa: F811
    def call(cache, batch, x=P, xs=256, y=P, ys=256, heads=4, k=P, ks=128, v=P, vs=128, type=0, c=P, s=P, pos=P,
             most=64, rotary=64, layout=0):
        return q.lib.qc_hip_kv8_rope_append(cache, batch, x, xs, y, ys, heads, k, ks, v, vs, type, c, s, pos, most,
                                            rotary, layout, P, None)

    bad = _common(q, call)
    for kw in (dict(ks=127), dict(vs=127), dict(ks=1 << 62), dict(vs=1 << 62), dict(xs=255), dict(ys=255),
               dict(xs=1 << 62), dict(ys=1 << 62), dict(heads=-1), dict(heads=1 << 40), dict(rotary=0),
               dict(rotary=63), dict(rotary=66), dict(rotary=-2), dict(most=0), dict(most=1 << 31)):
        assert bad(**kw) == 1, kw
    assert bad(type=3) == 2 and bad(type=-1) == 2
    for kw in (dict(x=None), dict(y=None), dict(k=None), dict(v=None), dict(c=None), dict(s=None), dict(layout=2),
               dict(layout=-1), dict(xs=512)):
        assert bad(**kw) == 3, kw
    # without queries theirs are not looked at: the next refusal is the layout's
    assert bad(heads=0, x=None, xs=0, y=None, ys=0, layout=5) == 3
    assert bad(heads=0, x=None, xs=0, y=None, ys=0, type=5) == 2


def test_tree_attention_refusals(q):  # noqa: F811
    def call(cache, batch, x=P, xs=256, y=P, ys=256, type=0, heads=4, scale=0.125, mask=P, words=1, pos=P, window=0):
        return q.lib.qc_hip_kv8_tree_attention(cache, batch, x, xs, y, ys, type, heads, scale, mask, words, pos,
                                               window, P, None)

    bad = _common(q, call)
    for kw in (dict(heads=0), dict(heads=3), dict(heads=-2), dict(heads=1 << 40), dict(window=-1), dict(words=0),
               dict(words=-1), dict(words=1 << 40), dict(xs=255), dict(ys=255), dict(xs=1 << 62)):
        assert bad(**kw) == 1, kw
    assert bad(type=7) == 2
    for kw in (dict(x=None), dict(y=None), dict(mask=None), dict(scale=NAN), dict(scale=INF),
               dict(window=4, pos=None)):
        assert bad(**kw) == 3, kw
    # a mask of fewer bits than a sequence may have new tokens: the smaller bound counts
    def wide(tokens, most, words):
        return call(ref(_cache(q)), ref(_batch(q, tokens=tokens, max_new=most)), words=words, type=9)
    assert wide(90, 33, 1) == 1 and wide(90, 33, 2) == 2 and wide(32, 90, 1) == 2 and wide(33, 90, 1) == 1


def test_keep_refusals(q):  # noqa: F811
    def call(cache, batch, kept=P, columns=3, count=P, out=2 * P):
        return q.lib.qc_hip_kv8_keep(cache, batch, kept, columns, count, out, P, None)

    bad = _common(q, call)
    for kw in (dict(columns=0), dict(columns=-1), dict(columns=1 << 31)):
        assert bad(**kw) == 1, kw
    for kw in (dict(kept=None), dict(count=None), dict(out=None), dict(out=P)):   # out: the batch's kv_len
        assert bad(**kw) == 3, kw


def _layer(q, **kw):
    f = dict(router=P, router_bias=None, gate_up_codes=P, gate_up_scales=P, down_codes=P, down_scales=P, router_type=0,
             experts=4, dim=64, inter=96)
    f.update(kw)
    m = q.Mxfp4Moe.__new__(q.Mxfp4Moe)
    for k, v in f.items():
        setattr(m, k, v)
    return m


def test_moe_refusals(q):  # noqa: F811
    def call(layer, x=P, xs=64, r=P, rs=64, y=2 * P, ys=64, type=0, tokens=3, top=2, scale=1.0, ids=P, weights=P):
        return q.lib.qc_hip_mxfp4_moe(layer, x, xs, r, rs, y, ys, type, tokens, top, 1, scale, 0, ids, weights, None)

    good = _layer(q)
    assert call(None) == 3
    for kw in (dict(experts=0), dict(experts=-1), dict(experts=1025), dict(dim=0), dict(dim=48), dict(inter=0),
               dict(inter=33), dict(dim=1 << 60), dict(inter=1 << 60), dict(experts=1024, dim=(1 << 17) + 32)):
        assert call(ref(_layer(q, **kw))) == 1, kw
    for kw in (dict(xs=63), dict(ys=63), dict(rs=63), dict(xs=1 << 62), dict(tokens=0), dict(tokens=-1),
               dict(tokens=1 << 31), dict(top=0), dict(top=5), dict(top=-1)):
        assert call(ref(good), **kw) == 1, kw
    assert call(ref(_layer(q, experts=100)), top=65) == 1
    assert call(ref(good), type=3) == 2 and call(ref(_layer(q, router_type=3))) == 2
    for name in ("router", "gate_up_codes", "gate_up_scales", "down_codes", "down_scales"):
        assert call(ref(_layer(q, **{name: None}))) == 3, name
    for name in ("gate_up_codes", "down_codes"):
        assert call(ref(_layer(q, **{name: P + 4}))) == 3, name
    for kw in (dict(x=None), dict(y=None), dict(ids=None), dict(weights=None), dict(scale=NAN), dict(scale=INF),
               dict(r=2 * P, rs=65), dict(x=2 * P, xs=65)):
        assert call(ref(good), **kw) == 3, kw


def test_keep_refuses_lengths_over_what_it_reads(q):  # noqa: F811
    """A head's workgroups read the paths, lengths and tables that another's would write new lengths over."""
    far = {"block_table": 2 * P, "seq_start": 3 * P, "kv_len": 4 * P}     # of 3 sequences and 4 columns
    cache, batch = _cache(q), _batch(q, **far)

    def call(out):
        return q.lib.qc_hip_kv8_keep(ref(cache), ref(batch), 5 * P, 3, 6 * P, out, P, None)

    for at, size in ((2 * P, 48), (3 * P, 16), (4 * P, 12), (5 * P, 36), (6 * P, 12)):
        for out in (at, at - 8, at + size - 4):
            assert call(out) == 3, (at, out - at)
