"""GPU: keys turned on their way into the 8-bit cache, attention of trees of drafted tokens over it, and the
accepted ones moved.  What is held in 8 bits bit for bit against the stated f32 steps; attention against 64-bit
arithmetic on the values the cache stands for."""
import numpy as np
import pytest

from test_gpu_kv8 import HALF, Ragged, _append_reference, _host, _random_cache, _same_cache

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]


def _tables(rng, positions, rotary):
    """Arbitrary f32 tables: the steps are the same whatever they hold."""
    a = rng.uniform(0, 6.3, (positions, rotary // 2))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def _turned(x, c, s, pos, interleaved):
    """Heads [t][h][d] turned in f32, each product and sum rounded."""
    x = x.astype(np.float32)
    r = 2 * c.shape[1]
    c, s = c[pos][:, None], s[pos][:, None]
    y = x.copy()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., first], x[..., second]
    with np.errstate(over="ignore", invalid="ignore"):
        y[..., first] = a * c - b * s
        y[..., second] = b * c + a * s
    return y


def _places(batch):
    """Position of each row in its sequence."""
    return np.concatenate([np.arange(k - n, k) for n, k in zip(batch.new, batch.kv)] + [[]]).astype(np.int64)


# ---- rotation and append ----------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "pairs"])
@pytest.mark.parametrize("heads,kvh,hd,rd,page,new,kv,spare", [
    (1, 1, 16, 16, 16, [1], [1], 0),
    (4, 2, 64, 64, 16, [1, 1, 1], [17, 16, 40], 0),
    (8, 8, 128, 64, 64, [1] * 9, [1, 64, 65, 128, 100, 500, 2, 63, 129], 2),
    (6, 3, 80, 20, 32, [0, 5, 33, 70], [9, 5, 64, 131], 4),
    (0, 5, 96, 48, 128, [200, 0, 1], [300, 0, 129], 0),
    (4, 2, 256, 256, 256, [257, 3], [600, 3], 1),
    (28, 4, 48, 2, 16, [100, 31, 16, 15], [100, 47, 32, 30], 7),
    (7, 1, 32, 10, 16, [1] * 70 + [150, 0, 20], [1 + 3 * i for i in range(70)] + [155, 0, 20], 3)])
def test_rope_append(qc, dev, dtype, interleaved, heads, kvh, hd, rd, page, new, kv, spare):
    import torch
    print(f"rope append {dtype} {heads}/{kvh} hd {hd} rd {rd} page {page} new {new[:6]} kv {kv[:6]}", flush=True)
    rng = np.random.default_rng(hd + rd + page + len(new))
    batch = Ragged(rng, new, kv, page, spare)
    cache = _random_cache(qc, dev, rng, batch.pages, kvh, page, hd)
    host = _host(cache)
    dt = getattr(torch, dtype)
    n, count = batch.tokens, int(batch.start[-1])
    c, s = _tables(rng, max(kv) + 50, rd)
    C, S = torch.from_numpy(c).to(dev), torch.from_numpy(s).to(dev)
    # one projection's rows, q, k, v side by side; rows of no sequence are not read
    rows = torch.from_numpy(rng.standard_normal((n, heads + 2 * kvh, hd)) * 2).to(dt)
    if spare:
        rows[count:] = float("nan")
    R = rows.to(dev)
    q, k, v = R[:, :heads], R[:, heads:heads + kvh], R[:, heads + kvh:]
    pos = _places(batch)
    given = rng.integers(0, c.shape[0], n).astype(np.int32)
    given[count:] = -9                                       # nor are their positions
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    b = batch.device(qc, dev)
    x = rows.float().numpy()

    def check(at, **kw):
        out = torch.full((n, heads, hd), 7.0, dtype=dt, device=dev)
        positions = None if at is None else torch.from_numpy(at).to(dev)
        got = qc.kv8_rope_append(cache, b, q if heads else None, k, v, C, S, positions=positions,
                                 interleaved=interleaved, out=out if heads else None, **kw)
        p = pos if at is None else at[:count]
        want = np.zeros((n, kvh, hd), np.float32)
        want[:count] = _turned(x[:count, heads:heads + kvh], c, s, p, interleaved)
        _append_reference(host, batch, want, x[:, heads + kvh:])
        _same_cache(cache, host)
        if not heads:
            assert got is None
            return
        assert got is out
        turned = torch.from_numpy(_turned(x[:count, :heads], c, s, p, interleaved)).to(dt)
        assert torch.equal(got[:count].cpu(), turned) and bool((got[count:] == 7).all())

    check(None, dev_status=st)
    check(given, dev_status=st)
    check(given)                                             # blocking
    # rows and tables that 16 bytes do not divide
    odd = torch.zeros(n * ((heads + 2 * kvh) * hd + 1) + 1, dtype=dt, device=dev)[1:].view(n, -1)[:, :(heads + 2 * kvh) * hd]
    odd.copy_(R.view(n, -1))
    odd = odd.unflatten(1, (heads + 2 * kvh, hd))
    q, k, v = odd[:, :heads], odd[:, heads:heads + kvh], odd[:, heads + kvh:]
    T = torch.zeros(2 * c.size + 1, device=dev)[1:].view(2, *c.shape)
    T[0], T[1] = C, S
    C, S = T[0], T[1]
    check(None, dev_status=st)
    # q in place; k beside it stays as it was
    if heads:
        before = k.clone()
        want = _turned(x[:count, :heads], c, s, pos, interleaved)
        got = qc.kv8_rope_append(cache, b, q, k, v, C, S, interleaved=interleaved, out=q, dev_status=st)
        assert got is q and torch.equal(got[:count].cpu(), torch.from_numpy(want).to(dt))
        assert torch.equal(torch.nan_to_num(k), torch.nan_to_num(before))
        if spare:
            assert bool(torch.isnan(q[count:]).all())
    assert st.item() == 0


def test_rope_append_is_rotation_then_append(qc, dev):
    """f32 rows: the same cache and queries as qc.rope and qc.kv8_append give."""
    import torch
    rng = np.random.default_rng(3)
    batch = Ragged(rng, [3, 70, 1], [90, 100, 40], 32, 2)
    one = _random_cache(qc, dev, rng, batch.pages, 4, 32, 64)
    two = qc.Kv8Cache(*[t.clone() for t in one.tensors])
    C, S = qc.rope_table(128, 64)
    rows = torch.from_numpy(rng.standard_normal((batch.tokens, 24, 64)).astype(np.float32)).to(dev)
    pos = torch.zeros(batch.tokens, dtype=torch.int32, device=dev)
    pos[:74] = torch.from_numpy(_places(batch).astype(np.int32)).to(dev)
    b = batch.device(qc, dev)
    q = qc.kv8_rope_append(one, b, rows[:, :16], rows[:, 16:20], rows[:, 20:], C, S)
    turned = qc.rope(rows[:, :20], C, S, pos)
    qc.kv8_append(two, b, turned[:, 16:].contiguous(), rows[:, 20:])
    assert torch.equal(q[:74], turned[:74, :16]) and bool((q[74:] == 0).all())
    for a, c in zip(one.tensors, two.tensors):
        assert torch.equal(a, c)


@pytest.mark.parametrize("bad", [-1, -2 ** 31, 64, 2 ** 31 - 1])
def test_rope_append_bad_positions(qc, dev, bad):
    """A position without a table row: its queries and the key pages that it goes to stay as they were, its
    value is written; the blocking form writes nothing."""
    import torch
    rng = np.random.default_rng(5)
    kvh, hd, page = 2, 64, 16
    batch = Ragged(rng, [3, 20, 2], [40, 36, 2], page)
    cache = _random_cache(qc, dev, rng, batch.pages, kvh, page, hd)
    host = _host(cache)
    c, s = _tables(rng, 64, hd)
    C, S = torch.from_numpy(c).to(dev), torch.from_numpy(s).to(dev)
    x = rng.standard_normal((batch.tokens, 4 + 2 * kvh, hd)).astype(np.float32)
    X = torch.from_numpy(x).to(dev)
    at = _places(batch).astype(np.int32)
    row = 3 + 7                                              # of the second sequence, position 23: page 1 of it
    at[row] = bad
    pos = torch.from_numpy(at).to(dev)
    b = batch.device(qc, dev)
    out = torch.full((batch.tokens, 4, hd), 7.0, device=dev)
    with pytest.raises(qc.QcError) as e:
        qc.kv8_rope_append(cache, b, X[:, :4], X[:, 4:6], X[:, 6:], C, S, positions=pos, out=out)
    assert e.value.status == 3 and bool((out == 7).all())
    _same_cache(cache, host)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    qc.kv8_rope_append(cache, b, X[:, :4], X[:, 4:6], X[:, 6:], C, S, positions=pos, out=out, dev_status=st)
    assert st.item() == 3
    at[row] = 0
    k, q = (_turned(x[:, lo:hi], c, s, at, False) for lo, hi in ((4, 6), (0, 4)))
    k[row] = np.nan                                          # what the reference leaves a page for
    _append_reference(host, batch, k, x[:, 6:])
    _same_cache(cache, host)
    keep = np.arange(batch.tokens) != row
    assert np.array_equal(out.cpu().numpy()[keep], q[keep]) and bool((out[row] == 7).all())


def test_rope_append_nonfinite(qc, dev):
    """NaN keys, keys that overflow once turned, infinite values; a sequence of more tokens than it is long."""
    import torch
    rng = np.random.default_rng(6)
    batch = Ragged(rng, [4, 4, 4], [20, 4, 33], 16)
    cache = _random_cache(qc, dev, rng, batch.pages, 2, 16, 32)
    host = _host(cache)
    c, s = _tables(rng, 64, 32)
    x = rng.standard_normal((12, 6, 32)).astype(np.float32)
    x[1, 2, 5] = np.nan
    x[6, 3, :] = 3.3e38                                      # finite, its turned one is not
    x[9, 4, 0] = np.inf
    X = torch.from_numpy(x).to(dev)
    C, S = torch.from_numpy(c).to(dev), torch.from_numpy(s).to(dev)
    b = batch.device(qc, dev)
    args = (X[:, :2], X[:, 2:4], X[:, 4:], C, S)
    for rows in ([1, 9], [6]):                               # each is found by the blocking form
        y = X.clone()
        for r in {1, 6, 9} - set(rows):
            y[r] = 1.0
        with pytest.raises(qc.QcError) as e:
            qc.kv8_rope_append(cache, b, y[:, :2], y[:, 2:4], y[:, 4:], C, S)
        assert e.value.status == 3
        _same_cache(cache, host)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    qc.kv8_rope_append(cache, b, *args, dev_status=st)
    assert st.item() == 3
    k = _turned(x[:, 2:4], c, s, _places(batch), False)
    assert not np.isfinite(k[6, 1]).all()
    _append_reference(host, batch, k, x[:, 4:])
    _same_cache(cache, host)
    # more new tokens than the sequence has: left alone, its queries too
    b.tensors[2][1] = 3
    st.zero_()
    out = torch.full((12, 2, 32), 7.0, device=dev)
    before = _host(cache)
    qc.kv8_rope_append(cache, b, *args, out=out, dev_status=st)
    assert st.item() == 3 and bool((out[4:8] == 7).all()) and bool((out[:4] != 7).all())
    ids = batch.table[1, :1]
    for got, want in zip(_host(cache), before):
        assert np.array_equal(got[ids], want[ids])


# ---- trees ------------------------------------------------------------------------

@pytest.fixture(params=[0, 1, 2, 3], ids=["auto", "direct16", "direct32", "tiled"])
def route(request, qc):
    """Every kernel of the attention at every size."""
    qc.set_kv8_attention_route(request.param)
    yield request.param
    qc.set_kv8_attention_route(0)


def _tree(rng, n, empty=0.0):
    """(seen [n][n], depth [n]): random parents, a share of the rows seeing nothing drafted."""
    seen, depth = np.zeros((n, n), bool), np.zeros(n, np.int64)
    for i in range(n):
        p = max(-1, i - 1 - rng.integers(0, 4))
        if p >= 0:
            seen[i], depth[i] = seen[p], depth[p] + 1
        seen[i, i] = True
    seen[rng.random(n) < empty] = False
    return seen, depth


def _bits(rng, batch, trees, words):
    """Mask words; bits past a sequence's tokens, and rows of no sequence, are set at random."""
    m = rng.random((batch.tokens, 32 * words)) < 0.5
    for s, (seen, _) in enumerate(trees):
        a, n = batch.start[s], len(seen)
        m[a:a + n, :n] = seen
    return np.packbits(m, axis=1, bitorder="little").view(np.int32)


def _tree_reference(host, batch, q, heads, scale, trees, window, half):
    """(out, tolerance) in f64.  The tolerance counts f32 dots, q and the probabilities in 11 (16-bit q) or 22
    bits, f32 sums (an addition for each 16 keys and some for the parts they are split into), one rounding to the
    output's type, and 2^-36 (f32: 2^-40) of the largest value scale times a key's codes: what f16 loses of a
    probability held relative to its row's largest."""
    kc, vc, ks, vs = host
    hd, kvh = kc.shape[3], kc.shape[1]
    g = heads // kvh
    coarse = half > 2.0 ** -24
    bits, qbits, low = (2.0 ** -11, 2.0 ** -40, 2.0 ** -36) if coarse else (2.0 ** -21, 2.0 ** -22, 2.0 ** -40)
    out = np.zeros((batch.tokens, heads, hd))
    tol = np.zeros_like(out)
    for s, (n, length) in enumerate(zip(batch.new, batch.kv)):
        if n == 0:
            continue
        c = length - n
        j = np.arange(length)
        seen = np.zeros((n, length), bool)
        seen[:, :max(c, 0)] = True
        if window:
            seen[:, :max(c, 0)] &= j[None, :max(c, 0)] > (c + trees[s][1])[:, None] - window
        seen[:, max(c, 0):] = trees[s][0][:, max(-c, 0):]
        used = seen.any(0)
        pid, slot = np.where(used, batch.table[s][j // batch.page], 0) if length else j, j % batch.page
        rows = slice(batch.start[s], batch.start[s + 1])
        for h in range(heads):
            C = np.where(used[:, None], np.abs(vc[pid, h // g, slot].astype(np.float64)), 0)
            K = np.where(used[:, None], kc[pid, h // g, slot].astype(np.float64) * ks[pid, h // g][:, None], 0)
            V = np.where(used[:, None], vc[pid, h // g, slot].astype(np.float64) * vs[pid, h // g][:, None], 0)
            Q = q[rows, h].astype(np.float64)
            z = np.where(seen, scale * (Q @ K.T), -np.inf)
            some = seen.any(1)
            top = np.where(some, z.max(1, initial=-np.inf), 0)
            p = np.exp(z - top[:, None])
            p = p / np.where(some, p.sum(1), 1)[:, None]
            o = p @ V
            size = np.where(seen, abs(scale) * (np.abs(Q) @ np.abs(K).T), 0).max(1, initial=0)
            small = abs(scale) * np.abs(Q).max(1) * np.abs(K).sum(1).max(initial=0) * 2.0 ** -38
            ds = size * ((hd + 8) * 2.0 ** -24 + qbits) + small + (np.abs(top) + size) * 2.0 ** -22
            largest = np.abs(np.where(used, vs[pid, h // g], 0)).max(initial=0)
            out[rows, h] = o
            tol[rows, h] = ((p @ np.abs(V)) * (bits + 2 * ds[:, None] + (length / 16 + 16) * 2.0 ** -23)
                            + low * largest * (seen @ C) + half * (1 + 2.0 ** -10) * np.abs(o) + 2.0 ** -25)
    return out, tol


def _attend(qc, dev, rng, new, kv, heads, kvh, hd, page, dtype, window=0, spare=0, empty=0.0, words=None,
            blocking=False, q=None, cache=None, batch=None):
    import torch
    batch = batch or Ragged(rng, new, kv, page, spare)
    cache = cache or _random_cache(qc, dev, rng, batch.pages, kvh, page, hd)
    dt = getattr(torch, dtype)
    trees = [_tree(rng, n, empty) for n in new]
    words = words or max(1, -(-batch.max_new // 32))
    mask = torch.from_numpy(_bits(rng, batch, trees, words)).to(dev)
    pos = np.full(batch.tokens, -5, np.int32)
    for s, (_, depth) in enumerate(trees):
        pos[batch.start[s]:batch.start[s + 1]] = kv[s] - new[s] + depth
    if q is None:
        q = torch.from_numpy(rng.standard_normal((batch.tokens, heads, hd))).to(dt)
    if spare:
        q[-spare:] = float("nan")
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    out = torch.full((batch.tokens, heads, hd), 7.0, dtype=dt, device=dev)
    qc.kv8_tree_attention(cache, batch.device(qc, dev), q.to(dev), mask, window=window,
                          positions=torch.from_numpy(pos).to(dev) if window else None, out=out,
                          dev_status=None if blocking else st)
    want, tol = _tree_reference(_host(cache), batch, q.float().numpy(), heads, float(np.float32(hd ** -0.5)), trees,
                                window, HALF[dtype])
    used = batch.start[-1]
    got = out.double().cpu().numpy()
    assert np.all(got[used:] == 7.0)
    err = np.abs(got[:used] - want[:used])
    assert np.all(err <= tol[:used]), (float((err / tol[:used]).max()), np.argwhere(~(err <= tol[:used]))[:4].tolist())
    assert st.item() == 0
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,kv,heads,kvh,hd,page", [
    ([1], [1], 4, 2, 64, 16),
    ([1, 2, 3], [1, 2, 40], 4, 2, 64, 16),
    ([8], [600], 8, 2, 128, 32),
    ([31, 32, 33], [100, 32, 97], 8, 2, 64, 32),
    ([64, 0, 65, 5], [500, 3, 1089, 133], 6, 2, 80, 64),
    ([16, 128], [2000, 700], 4, 1, 128, 128),
    ([24, 3], [900, 17], 16, 1, 96, 16),
    ([40], [333], 4, 4, 256, 256),
    ([97, 1], [640, 1000], 28, 4, 48, 64)])
def test_tree(qc, dev, route, dtype, new, kv, heads, kvh, hd, page):
    print(f"tree {dtype} route {route} new {new} kv {kv} {heads}/{kvh} of {hd}", flush=True)
    rng = np.random.default_rng(sum(new) + hd)
    _attend(qc, dev, rng, new, kv, heads, kvh, hd, page, dtype, spare=2)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("window", [1, 5, 33, 64, 200, 5000])
def test_tree_windows(qc, dev, route, dtype, window):
    rng = np.random.default_rng(window)
    _attend(qc, dev, rng, [33, 9, 64, 1], [1000, 9, 300, 257], 8, 2, 64, 16, dtype, window=window, blocking=True)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("new,kv", [([20, 9], [20, 9]), ([33], [20]), ([70, 2], [100, 0]), ([5], [0])])
def test_tree_rows_that_see_nothing(qc, dev, route, dtype, new, kv):
    """Empty masks without context, more drafted tokens than the sequence is long (the first are before its
    start), and an empty sequence: such rows are zeros."""
    rng = np.random.default_rng(len(new))
    _attend(qc, dev, rng, new, kv, 8, 2, 64, 16, dtype, empty=0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,kv,heads,kvh,hd,page", [
    ([64], [20600], 32, 8, 128, 64), ([33] * 65, [401] * 64 + [33], 32, 8, 128, 16), ([40, 24, 7], [9000, 8200, 7], 32, 8, 64, 32),
    ([70, 30], [9001, 5000], 8, 2, 256, 128)])
def test_tree_by_size(qc, dev, dtype, new, kv, heads, kvh, hd, page):
    """As a call of its size is worked on: one sequence's 256 rows a workgroup, 128 of many sequences', ..."""
    print(f"tree by size {dtype} {len(new)} x {max(new)} x {max(kv)}", flush=True)
    _attend(qc, dev, np.random.default_rng(hd), new, kv, heads, kvh, hd, page, dtype)


@pytest.mark.parametrize("pages", ["negative", "nan", "missing"])
def test_tree_shared_scales(qc, dev, route, pages):
    """Scales of either sign and of zero; a page that is not there, or whose scale is not finite: its keys count for
    nothing, and the status says so."""
    import torch
    rng = np.random.default_rng(17)
    new, kv, kvh, page, hd = [40, 21], [400, 333], 2, 32, 128
    batch = Ragged(rng, new, kv, page)
    cache = _random_cache(qc, dev, rng, batch.pages, kvh, page, hd)
    g = torch.Generator(device=dev).manual_seed(3)
    for s in cache.tensors[2:]:
        sign = torch.randint(-1, 2, s.shape, generator=g, device=dev).float()
        s.copy_(s * torch.where(sign == 0, torch.zeros_like(sign) if s is cache.tensors[3] else torch.ones_like(sign), sign))
    if pages == "negative":
        _attend(qc, dev, rng, new, kv, 8, kvh, hd, page, "bfloat16", cache=cache, batch=batch)
        return
    lost = int(batch.table[0][2])
    trees = [_tree(rng, n) for n in new]
    mask = torch.from_numpy(_bits(rng, batch, trees, 2)).to(dev)
    q = torch.from_numpy(rng.standard_normal((batch.tokens, 8, hd))).to(torch.bfloat16).to(dev)
    b = batch.device(qc, dev)
    if pages == "nan":
        cache.tensors[3][lost, 1] = float("nan")
    else:
        b.tensors[0][0, 2] = batch.pages + 5
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    out = qc.kv8_tree_attention(cache, b, q, mask, dev_status=st)
    assert st.item() == 3
    # the same with the page's keys out of sight: a context without them
    kc, vc, ks, vs = _host(cache)
    for s, (n, length) in enumerate(zip(new, kv)):
        for h in range(8):
            j = np.arange(length)
            pid = batch.table[s][j // page]
            seen = np.zeros((n, length), bool)
            seen[:, :length - n] = True
            seen[:, length - n:] = trees[s][0]
            if s == 0 and (pages == "missing" or h // 4 == 1):
                seen[:, 2 * page:3 * page] = False
            K = kc[pid, h // 4, j % page] * ks[pid, h // 4][:, None].astype(np.float64)
            V = np.nan_to_num(vc[pid, h // 4, j % page] * vs[pid, h // 4][:, None].astype(np.float64))
            K, V = np.nan_to_num(K), np.nan_to_num(V)
            rows, scale = slice(batch.start[s], batch.start[s + 1]), float(np.float32(hd ** -0.5))
            Q = q[rows, h].double().cpu().numpy()
            z = np.where(seen, scale * (Q @ K.T), -np.inf)
            p = np.exp(z - z.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            # as _tree_reference: what scores, probabilities, sums and the output's rounding are off by
            size = scale * (np.abs(Q) @ np.abs(K).T).max(1, keepdims=True)
            ds = size * ((hd + 8) * 2.0 ** -24 + 2.0 ** -40) + 2 * size * 2.0 ** -22 + size * hd * 2.0 ** -38
            tol = p @ np.abs(V) * (2.0 ** -11 + 2 * ds + (length / 16 + 16) * 2.0 ** -23) + np.abs(V).sum() * 2.0 ** -36
            assert np.all(np.abs(out[rows, h].double().cpu().numpy() - p @ V) <= tol + 2.0 ** -8 * 1.001 * np.abs(p @ V))


def test_tree_wide_masks_and_strides(qc, dev, route):
    """Mask rows wider than the batch needs; q and out rows of a wider array."""
    import torch
    rng = np.random.default_rng(8)
    _attend(qc, dev, rng, [3, 40], [70, 90], 8, 2, 64, 16, "float32", words=5)
    batch = Ragged(rng, [12], [300], 16)
    cache = _random_cache(qc, dev, rng, batch.pages, 2, 16, 64)
    b = batch.device(qc, dev)
    mask = torch.from_numpy(_bits(rng, batch, [_tree(rng, 12)], 1)).to(dev)
    q = torch.randn(12, 8, 64, device=dev, dtype=torch.bfloat16)
    plain = qc.kv8_tree_attention(cache, b, q, mask)
    for extra in (8, 1):
        wide = torch.zeros(12, 2 * (512 + extra), device=dev, dtype=torch.bfloat16)
        Q, O = (wide[:, i * (512 + extra):][:, :512].unflatten(1, (8, 64)) for i in range(2))
        Q.copy_(q)
        qc.kv8_tree_attention(cache, b, Q, mask, out=O)
        assert torch.equal(O, plain)


def test_a_chain_is_a_causal_prompt(qc, dev, route):
    """A tree of one path sees what qc.kv8_attention's causal rows see: within the tolerance of both."""
    import torch
    rng = np.random.default_rng(2)
    batch = Ragged(rng, [37, 4], [400, 4], 32)
    cache = _random_cache(qc, dev, rng, batch.pages, 2, 32, 128)
    b = batch.device(qc, dev)
    q = torch.randn(batch.tokens, 8, 128, device=dev)
    chain = [(np.tril(np.ones((n, n), bool)), np.arange(n)) for n in batch.new]
    mask = torch.from_numpy(_bits(rng, batch, chain, 2)).to(dev)
    got = qc.kv8_tree_attention(cache, b, q, mask)
    want = qc.kv8_attention(cache, b, q)
    _, tol = _tree_reference(_host(cache), batch, q.cpu().numpy(), 8, float(np.float32(128 ** -0.5)), chain, 0, HALF["float32"])
    assert np.all(np.abs((got - want).double().cpu().numpy()) <= 2 * tol)


def test_tree_ignores_what_it_does_not_see(qc, dev, route):
    """Infinite and NaN codes do not exist, but scales do: pages out of the window, slots past the length and rows
    of other sequences may hold anything; NaN q stays in its row."""
    import torch
    rng = np.random.default_rng(12)
    batch = Ragged(rng, [10, 4], [500, 60], 16, extra_pages=2)
    cache = _random_cache(qc, dev, rng, batch.pages, 2, 16, 64)
    b = batch.device(qc, dev)
    trees = [_tree(rng, n) for n in batch.new]
    mask = torch.from_numpy(_bits(rng, batch, trees, 1)).to(dev)
    pos = torch.from_numpy(np.concatenate([k - n + t[1] for n, k, t in zip(batch.new, batch.kv, trees)]).astype(np.int32)).to(dev)
    q = torch.randn(14, 4, 64, device=dev)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    run = lambda: qc.kv8_tree_attention(cache, b, q, mask, positions=pos, window=100, dev_status=st)
    want = run()
    first = (490 + 1 - 100) // 16
    cache.tensors[2][batch.table[0, :first].tolist()] = float("nan")
    cache.tensors[3][batch.table[0, :first].tolist()] = float("inf")
    b.tensors[0][0, :first] = 1 << 30
    unused = sorted(set(range(batch.pages)) - set(batch.table.ravel().tolist()))
    cache.tensors[2][unused] = float("nan")
    assert torch.equal(run(), want) and st.item() == 0
    q[3, 1, 7] = float("nan")
    got = run()
    assert bool(torch.isnan(got[3, 1]).all())
    got[3, 1], w = 0.0, want.clone()
    w[3, 1] = 0.0
    assert torch.equal(got, w)


def test_tree_errors(qc, dev, route):
    """Bad pages, scales and positions: told of, the other sequences done, the blocking form writes nothing."""
    import torch
    rng = np.random.default_rng(13)
    batch = Ragged(rng, [6, 7, 5], [300, 200, 77], 16)
    cache = _random_cache(qc, dev, rng, batch.pages, 2, 16, 64)
    trees = [_tree(rng, n) for n in batch.new]
    mask = torch.from_numpy(_bits(rng, batch, trees, 1)).to(dev)
    pos = np.concatenate([k - n + t[1] for n, k, t in zip(batch.new, batch.kv, trees)]).astype(np.int32)
    q = torch.randn(18, 4, 64, device=dev)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    b = batch.device(qc, dev)
    P = torch.from_numpy(pos).to(dev)
    want = qc.kv8_tree_attention(cache, b, q, mask, positions=P, window=64)
    rest = list(range(6)) + list(range(13, 18))

    def wrong(handle, positions):
        out = torch.full_like(q, 7.0)
        with pytest.raises(qc.QcError) as e:
            qc.kv8_tree_attention(cache, handle, q, mask, positions=positions, window=64, out=out)
        assert e.value.status == 3 and bool((out == 7).all())
        st.zero_()
        qc.kv8_tree_attention(cache, handle, q, mask, positions=positions, window=64, out=out, dev_status=st)
        assert st.item() == 3 and torch.equal(out[rest], want[rest])

    bad = batch.device(qc, dev)
    bad.tensors[0][1, 11] = batch.pages
    wrong(bad, P)
    bad = batch.device(qc, dev)
    bad.tensors[2][1] = batch.max_kv + 1
    wrong(bad, P)
    for value in (pos[8] - 8, 200, -1, 2 ** 31 - 1, -2 ** 31):
        p = P.clone()
        p[8] = int(value)
        wrong(b, p)
    keep = cache.tensors[3][batch.table[1, 12], 0].item()
    cache.tensors[3][batch.table[1, 12], 0] = float("nan")
    wrong(b, P)
    cache.tensors[3][batch.table[1, 12], 0] = keep
    assert torch.equal(qc.kv8_tree_attention(cache, b, q, mask, positions=P, window=64), want)


@pytest.mark.parametrize("new,kv,heads,kvh", [([8], [4000], 8, 2), ([48, 60, 9], [700, 1500, 9], 16, 4)])
def test_tree_repeats_and_graph(qc, dev, route, new, kv, heads, kvh):
    """Bit for bit the same again, on another stream and replayed, with eager calls that share the stream's
    workspace between the replays."""
    import torch
    rng = np.random.default_rng(21)
    batch = Ragged(rng, new, kv, 64)
    cache = _random_cache(qc, dev, rng, batch.pages, kvh, 64, 128)
    b = batch.device(qc, dev)
    trees = [_tree(rng, n) for n in new]
    mask = torch.from_numpy(_bits(rng, batch, trees, 2)).to(dev)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    q = torch.randn(batch.tokens, heads, 128, device=dev, dtype=torch.bfloat16)
    want = qc.kv8_tree_attention(cache, b, q, mask, dev_status=st)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = torch.zeros_like(q)
        qc.kv8_tree_attention(cache, b, q, mask, out=out, dev_status=st)
        assert torch.equal(out, want)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            qc.kv8_tree_attention(cache, b, q, mask, out=out, dev_status=st)
        for _ in range(4):
            q.copy_(torch.randn_like(q))
            other = torch.randn_like(q)
            qc.kv8_tree_attention(cache, b, other, mask, dev_status=st)
            graph.replay()
            qc.kv8_attention(cache, b, other, dev_status=st)
            stream.synchronize()
            assert torch.equal(out, qc.kv8_tree_attention(cache, b, q, mask, dev_status=st))
    assert st.item() == 0


# ---- the accepted ones ------------------------------------------------------------

def _keep_reference(host, batch, paths):
    """The stated f32 steps on the host arrays, in place; codes past the new lengths are not its business."""
    f = np.float32
    length = []
    before = [a.copy() for a in host]
    for s, path in enumerate(paths):
        c = batch.kv[s] - batch.new[s]
        length.append(c + len(path))
        moved = [(a, p) for a, p in enumerate(path) if a != p]
        for column in sorted({(c + a) // batch.page for a, _ in moved}):
            here = [(a, p) for a, p in moved if (c + a) // batch.page == column]
            pid = batch.table[s, column]
            for w in (0, 1):
                codes, scales = host[w], host[2 + w]
                for h in range(codes.shape[1]):
                    held = before[2 + w][pid, h]
                    came = [abs(before[2 + w][batch.table[s, (c + p) // batch.page], h]) for _, p in here
                            if (c + p) // batch.page != column]
                    scale = max([abs(held)] + came) if came else held
                    turn = lambda v, sc: (np.clip(np.rint(v.astype(f) * (f(sc / scale) if scale != 0 else f(0))), -127, 127)
                                          .astype(np.int8) if sc != scale else v)
                    n = c + here[0][0] - column * batch.page
                    codes[pid, h, :n] = turn(codes[pid, h, :n], held)
                    for a, p in here:
                        src = batch.table[s, (c + p) // batch.page]
                        codes[pid, h, (c + a) % batch.page] = turn(before[w][src, h, (c + p) % batch.page],
                                                                   before[2 + w][src, h])
                    scales[pid, h] = scale
    return length


def _same_kept(cache, host, batch, length):
    got = _host(cache)
    for w in (2, 3):
        assert np.array_equal(got[w].view(np.uint32), host[w].view(np.uint32))
    for s, n in enumerate(length):
        pid, slot = batch.places(s, 0, n)
        for w in (0, 1):
            assert np.array_equal(got[w][pid, :, slot], host[w][pid, :, slot]), (s, w)


@pytest.mark.parametrize("spread", [0.0, 1.0])
@pytest.mark.parametrize("heads,hd,page,new,kv,counts", [
    (1, 16, 16, [1], [1], [1]),
    (2, 64, 16, [8, 8, 8, 3], [40, 16, 30, 3], [3, 0, 8, 2]),
    (8, 128, 64, [20, 0, 33, 64], [70, 5, 33, 200], [7, 0, 20, 31]),
    (3, 80, 32, [100, 70], [131, 70], [40, 64]),
    (1, 256, 16, [128, 128], [128, 300], [90, 3]),
    (2, 32, 256, [600, 256], [700, 256], [500, 255]),
    (5, 48, 16, [300], [310], [299])])
def test_keep(qc, dev, spread, heads, hd, page, new, kv, counts):
    import torch
    print(f"keep heads {heads} hd {hd} page {page} new {new} kv {kv} counts {counts}", flush=True)
    rng = np.random.default_rng(hd + page + len(new))
    batch = Ragged(rng, new, kv, page)
    cache = _random_cache(qc, dev, rng, batch.pages, heads, page, hd, spread)
    host = _host(cache)
    for blocking in (False, True):
        paths = [sorted(rng.choice(n, c, replace=False).tolist()) for n, c in zip(new, counts)]
        kept = np.full((len(new), max(max(counts), 1) + blocking), 1 << 30, np.int32)   # past the counts: anything
        for s, p in enumerate(paths):
            kept[s, :len(p)] = p
        up = lambda a: torch.from_numpy(np.asarray(a, np.int32)).to(dev)
        st = torch.zeros(1, dtype=torch.int32, device=dev)
        b = batch.device(qc, dev)
        got = qc.kv8_keep(cache, b, up(kept), up(counts), dev_status=None if blocking else st)
        want = _keep_reference(host, batch, paths)
        assert got.tolist() == want and st.item() == 0
        assert b.tensors[2].tolist() == batch.kv
        _same_kept(cache, host, batch, want)
        host = _host(cache)


def test_keep_leaves_the_rest(qc, dev):
    """Pages that no accepted token comes to are untouched, kept prefixes move nothing at all."""
    import torch
    rng = np.random.default_rng(4)
    batch = Ragged(rng, [40, 20], [100, 60], 16)
    cache = _random_cache(qc, dev, rng, batch.pages, 2, 16, 64)
    host = _host(cache)
    up = lambda a: torch.from_numpy(np.asarray(a, np.int32)).to(dev)
    got = qc.kv8_keep(cache, batch.device(qc, dev), up([[0, 1, 2, 3], [0, 1, 5, 0]]), up([4, 3]))
    assert got.tolist() == [64, 43]
    now = _host(cache)
    touched = batch.table[1, 2]                              # position 42
    for w in range(4):
        rest = np.arange(batch.pages) != touched
        assert np.array_equal(now[w][rest], host[w][rest])


def test_keep_zero_and_negative_scales(qc, dev):
    """Scales of 0 (codes without value) and below 0 keep what they stand for."""
    import torch
    rng = np.random.default_rng(14)
    batch = Ragged(rng, [30, 30], [40, 40], 16)
    cache = _random_cache(qc, dev, rng, batch.pages, 2, 16, 32)
    for t in cache.tensors[2:]:
        t[batch.table[0, 0]] = 0.0
        t[batch.table[0, 1], 1] = 0.0
        t[batch.table[1, :2].tolist()] *= -1
    host = _host(cache)
    paths = [[3, 9, 17, 25], [1, 2, 8, 20, 29]]
    kept = np.zeros((2, 5), np.int32)
    for s, p in enumerate(paths):
        kept[s, :len(p)] = p
    up = lambda a: torch.from_numpy(np.asarray(a, np.int32)).to(dev)
    got = qc.kv8_keep(cache, batch.device(qc, dev), up(kept), up([4, 5]))
    want = _keep_reference(host, batch, paths)
    assert got.tolist() == want
    _same_kept(cache, host, batch, want)


@pytest.mark.parametrize("kept,count", [([3, 3, 5], 3), ([5, 3, 6], 3), ([-1, 2, 3], 3), ([0, 2, 20], 3), ([1, 2, 3], 4),
                                        ([1, 2, 3], -1), ([1 << 31 - 1, 2, 3], 1)])
def test_keep_bad_paths(qc, dev, kept, count):
    """The sequence and its length stay as they were, the others are done; blocking writes nothing."""
    import torch
    rng = np.random.default_rng(15)
    batch = Ragged(rng, [20, 20], [50, 50], 16)
    cache = _random_cache(qc, dev, rng, batch.pages, 2, 16, 32)
    host = _host(cache)
    up = lambda a: torch.from_numpy(np.asarray(a, np.int64).astype(np.int32)).to(dev)
    K, N = up([kept, [2, 8, 19]]), up([count, 3])
    b = batch.device(qc, dev)
    out = up([-3, -4])
    with pytest.raises(qc.QcError) as e:
        qc.kv8_keep(cache, b, K, N, out=out)
    assert e.value.status == 3 and out.tolist() == [-3, -4]
    _same_cache(cache, host)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    qc.kv8_keep(cache, b, K, N, out=out, dev_status=st)
    assert st.item() == 3 and out.tolist() == [-3, 33]
    only = Ragged(rng, batch.new, batch.kv, 16)
    only.table = batch.table
    _keep_reference(host, only, [[], [2, 8, 19]])
    _same_kept(cache, host, batch, [50, 33])


def test_keep_bad_pages_scales_and_lengths(qc, dev):
    import torch
    rng = np.random.default_rng(16)
    batch = Ragged(rng, [20, 20], [50, 50], 16)
    cache = _random_cache(qc, dev, rng, batch.pages, 2, 16, 32)
    up = lambda a: torch.from_numpy(np.asarray(a, np.int32)).to(dev)
    K, N = up([[2, 8, 19], [2, 8, 19]]), up([3, 3])
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    host = _host(cache)

    def wrong(b, want, sequences):
        before = _host(cache)
        out = up([-3, -4])
        with pytest.raises(qc.QcError) as e:
            qc.kv8_keep(cache, b, K, N, out=out)
        assert e.value.status == 3 and out.tolist() == [-3, -4]
        _same_cache(cache, before)
        st.zero_()
        qc.kv8_keep(cache, b, K, N, out=out, dev_status=st)
        assert st.item() == 3 and out.tolist() == want
        now = _host(cache)
        for s in sequences:
            for a, w in zip(now, before):
                assert np.array_equal(a[batch.table[s]].view(np.uint8), w[batch.table[s]].view(np.uint8))

    b = batch.device(qc, dev)
    b.tensors[0][0, 3] = -1                                  # position 49: where token 19 is
    wrong(b, [-3, 33], [0])
    b = batch.device(qc, dev)
    b.tensors[2][1] = 19                                     # more new tokens than it is long
    wrong(b, [33, -4], [1])
    # a scale that is not finite: that head's keys stay, the other head's and the values move
    for t, a in zip(cache.tensors, host):
        t.copy_(torch.from_numpy(a).to(dev))
    cache.tensors[2][batch.table[0, 3], 1] = float("inf")
    st.zero_()
    out = up([-3, -4])
    qc.kv8_keep(cache, batch.device(qc, dev), K, N, out=out, dev_status=st)
    assert st.item() == 3 and out.tolist() == [33, 33]
    now, want = _host(cache), [a.copy() for a in host]
    _keep_reference(want, batch, [[2, 8, 19]] * 2)
    ids = batch.table[0]
    assert np.array_equal(now[0][ids, 1], host[0][ids, 1])
    for w, h in ((0, 0), (1, 0), (1, 1)):
        pid, slot = batch.places(0, 0, 33)
        assert np.array_equal(now[w][pid, h, slot], want[w][pid, h, slot])


def test_keep_graph(qc, dev):
    """Captured, with counts and paths that change between the replays."""
    import torch
    rng = np.random.default_rng(17)
    batch = Ragged(rng, [24, 24, 24], [80, 24, 61], 16)
    cache = _random_cache(qc, dev, rng, batch.pages, 3, 16, 64)
    b = batch.device(qc, dev)
    K = torch.zeros(3, 24, dtype=torch.int32, device=dev)
    N = torch.zeros(3, dtype=torch.int32, device=dev)
    out = torch.zeros(3, dtype=torch.int32, device=dev)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            qc.kv8_keep(cache, b, K, N, out=out, dev_status=st)
        for rep in range(5):
            counts = rng.integers(0, 25, 3)
            paths = [sorted(rng.choice(24, c, replace=False).tolist()) for c in counts]
            kept = np.zeros((3, 24), np.int32)
            for s, p in enumerate(paths):
                kept[s, :len(p)] = p
            K.copy_(torch.from_numpy(kept))
            N.copy_(torch.from_numpy(counts.astype(np.int32)))
            stream.synchronize()
            host = _host(cache)
            graph.replay()
            stream.synchronize()
            want = _keep_reference(host, batch, paths)
            assert out.tolist() == want
            _same_kept(cache, host, batch, want)
    assert st.item() == 0


@pytest.mark.parametrize("dtype,hd,seqs,bound,most,longest", [
    ("bfloat16", 64, 64, 1 << 17, 128, 20000), ("float32", 64, 64, 1 << 17, 128, 9000),
    ("float16", 128, 16, 1 << 20, 128, 40000), ("bfloat16", 128, 70, 1 << 17, 60, 17000),
    ("bfloat16", 256, 4, 1 << 20, 128, 20000)])
def test_tree_partial_sums_of_a_loose_bound(qc, dev, dtype, hd, seqs, bound, most, longest):
    """Partial sums that would pass 1 GB go in passes: the scratch of many rows under a bound far above the lengths
    stays near that, and results are what they were."""
    import torch
    print(f"tree under {bound} keys, {seqs} x {most}, {dtype} heads of {hd}", flush=True)
    rng = np.random.default_rng(hd + seqs)
    new = [most] + rng.integers(1, 40, seqs - 1).tolist()
    new[seqs // 2], new[seqs - 2] = 10, 0
    kv = [n + int(k) for n, k in zip(new, rng.integers(0, 150, seqs))]
    kv[seqs // 2] = longest
    batch = Ragged(rng, new, kv, 256, spare=seqs * most - sum(new), columns=bound // 256)
    batch.max_kv = bound
    cache = _random_cache(qc, dev, rng, batch.pages, 8, 256, hd)
    q = torch.from_numpy(rng.standard_normal((batch.tokens, 64, hd)).astype(np.float32)).to(getattr(torch, dtype)).to(dev)
    out, b = torch.zeros_like(q), batch.device(qc, dev)
    mask = torch.zeros(batch.tokens, -(-most // 32), dtype=torch.int32, device=dev)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        before = torch.cuda.mem_get_info()[0]
        qc.kv8_tree_attention(cache, b, q, mask, out=out, dev_status=st)
        stream.synchronize()
        assert before - torch.cuda.mem_get_info()[0] <= 1.05 * (1 << 30) and st.item() == 0
        _attend(qc, dev, rng, new, kv, 64, 8, hd, 256, dtype, spare=batch.tokens - sum(new), cache=cache, batch=batch, q=q.cpu())


@pytest.mark.parametrize("dtype,hd", [("bfloat16", 128), ("float16", 96), ("float32", 128), ("float16", 256), ("float32", 256)])
@pytest.mark.parametrize("window", [1, 40, 300])
def test_tree_windows_of_wide_heads(qc, dev, route, dtype, hd, window):
    """Windows that begin in the context, at its end and before it, for the other sizes of heads."""
    rng = np.random.default_rng(window + hd)
    _attend(qc, dev, rng, [33, 9, 40, 1, 0], [700, 9, 300, 257, 5], 8, 2, hd, 32, dtype, window=window, spare=3, empty=0.2)
