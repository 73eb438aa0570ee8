"""GPU: the 8-bit key/value cache.  Append and gather bit for bit against the stated
f32 steps; attention against 64-bit arithmetic on the values the cache stands for."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}   # half a step


class Ragged:
    """A batch on the host: new and total tokens per sequence, a shuffled page table."""

    def __init__(self, rng, new, kv, page, spare=0, extra_pages=3, columns=None):
        self.new, self.kv, self.page = list(new), list(kv), page
        need = [-(-k // page) for k in kv]
        self.columns = columns or max(max(need), 1)
        self.pages = sum(need) + extra_pages
        ids = rng.permutation(self.pages)
        self.table = np.full((len(kv), self.columns), -7, np.int32)    # unused entries: no page
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = ids[at:at + n]
            at += n
        self.start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.tokens = int(self.start[-1]) + spare
        self.max_new, self.max_kv = max(max(new), 1), max(max(kv), 1)

    def device(self, qc, dev, **kw):
        import torch
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(dev)
        f = dict(tokens=max(self.tokens, 1), max_new=self.max_new, max_kv=self.max_kv)
        f.update(kw)
        return qc.Kv8Batch(up(self.table), up(self.start), up(self.kv), f["tokens"],
                           min(f["max_new"], f["tokens"]), f["max_kv"])

    def places(self, s, lo, hi):
        p = np.arange(lo, hi)
        return self.table[s, p // self.page], p % self.page


def _random_cache(qc, dev, rng, pages, heads, page, hd, spread=1.0):
    import torch
    codes = [rng.integers(-127, 128, (pages, heads, page, hd)).astype(np.int8) for _ in range(2)]
    scales = [(np.exp(spread * rng.standard_normal((pages, heads))) / 60).astype(np.float32) for _ in range(2)]
    up = lambda a: torch.from_numpy(a).to(dev)
    return qc.Kv8Cache(*[up(c) for c in codes], *[up(s) for s in scales])


def _host(cache):
    return [t.cpu().numpy().copy() for t in cache.tensors]


# ---- append and gather ------------------------------------------------------------

def _append_reference(host, batch, k, v):
    """The stated steps in f32 on the host arrays, in place."""
    f = np.float32
    for which, x in ((0, k), (1, v)):
        codes, scales = host[which], host[2 + which]
        for s in range(len(batch.kv)):
            begin, end = batch.kv[s] - batch.new[s], batch.kv[s]
            for c in range(begin // batch.page, -(-end // batch.page)):
                lo, hi = max(begin, c * batch.page), min(end, (c + 1) * batch.page)
                if lo >= hi:
                    continue
                pid, a, b = batch.table[s, c], lo - c * batch.page, hi - c * batch.page
                rows = x[batch.start[s] + lo - begin: batch.start[s] + hi - begin]   # [t][heads][hd]
                for h in range(codes.shape[1]):
                    r = rows[:, h].astype(f)
                    if not np.all(np.isfinite(r)):
                        continue
                    before = scales[pid, h] if a > 0 else f(0)
                    scale = max(before, f(np.abs(r).max() * f(1 / 127)))
                    if scale < f(2.0 ** -126):
                        scale = f(0)
                    inv = f(1) / scale if scale > 0 else f(0)
                    ratio = before / scale if scale > 0 else f(0)
                    codes[pid, h, :a] = np.rint(codes[pid, h, :a].astype(f) * ratio).astype(np.int8)
                    codes[pid, h, a:b] = np.clip(np.rint(r * inv), -127, 127).astype(np.int8)
                    scales[pid, h] = scale


def _same_cache(cache, host):
    for got, want in zip(_host(cache), host):
        assert np.array_equal(got.view(np.uint8), want.view(np.uint8))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,hd,page,new,kv,spare", [
    (1, 16, 16, [1], [1], 0),
    (2, 64, 16, [1, 1, 1], [17, 16, 40], 0),
    (8, 128, 64, [1] * 9, [1, 64, 65, 128, 100, 500, 2, 63, 129], 2),
    (3, 80, 32, [0, 5, 33, 70], [9, 5, 64, 131], 4),
    (5, 96, 128, [200, 0, 1], [300, 0, 129], 0),
    (2, 256, 256, [257, 3], [600, 3], 1),
    (4, 48, 16, [100, 31, 16, 15], [100, 47, 32, 30], 7),
    # one sequence far longer than the others
    (2, 32, 16, [1] * 70 + [150, 0, 20], [1 + 3 * i for i in range(70)] + [155, 0, 20], 3),
    (1, 64, 32, [400] + [0] * 9 + [3, 1], [400] + [5] * 9 + [40, 1], 1)])
def test_append_gather(qc, dev, dtype, heads, hd, page, new, kv, spare):
    import torch
    print(f"kv8 append {dtype} heads {heads} hd {hd} page {page} new {new} kv {kv}", flush=True)
    rng = np.random.default_rng(hd + page + len(new))
    batch = Ragged(rng, new, kv, page, spare)
    cache = _random_cache(qc, dev, rng, batch.pages, heads, page, hd)
    host = _host(cache)
    dt = getattr(torch, dtype)
    k, v = (torch.from_numpy(rng.standard_normal((batch.tokens, heads, hd)) * m).to(dt) for m in (1.5, 4.0))
    if spare:
        k[-spare:], v[-spare:] = float("nan"), float("inf")   # rows of no sequence are not read
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    b = batch.device(qc, dev)
    # token rows of a wider projection
    wide = torch.zeros(batch.tokens, 2 * heads * hd + 24, dtype=dt, device=dev)
    wide[:, :heads * hd] = k.view(batch.tokens, -1).to(dev)
    wide[:, heads * hd:2 * heads * hd] = v.view(batch.tokens, -1).to(dev)
    K, V = wide[:, :heads * hd], wide[:, heads * hd:2 * heads * hd]
    qc.kv8_append(cache, b, K, V, dev_status=st)
    _append_reference(host, batch, k.float().numpy(), v.float().numpy())
    assert st.item() == 0
    _same_cache(cache, host)
    # again, blocking: the codes and scales are a fixed point; other alignments
    qc.kv8_append(cache, b, k.to(dev), torch.cat([v, v])[:batch.tokens].to(dev))
    _same_cache(cache, host)
    odd = torch.zeros(batch.tokens * (heads * hd + 1) + 1, dtype=dt, device=dev)[1:].view(batch.tokens, -1)[:, :heads * hd]
    odd.copy_(k.view(batch.tokens, -1).to(dev))
    qc.kv8_append(cache, b, odd, V, dev_status=st)
    _same_cache(cache, host)
    # gather: the new tokens' values; rows of no sequence stay
    for gt in (torch.float32, dt):
        gk = torch.full((batch.tokens, heads, hd), 7.0, dtype=gt, device=dev)
        gv = torch.full((batch.tokens, heads * hd + 8), 7.0, dtype=gt, device=dev)
        qc.kv8_gather(cache, b, k=gk, v=gv[:, :heads * hd], dev_status=st)
        want = [torch.full((batch.tokens, heads, hd), 7.0, dtype=gt) for _ in range(2)]
        for s in range(len(kv)):
            pid, slot = batch.places(s, kv[s] - new[s], kv[s])
            for w in range(2):
                val = host[w][pid, :, slot].astype(np.float32) * host[2 + w][pid][:, :, None]
                want[w][batch.start[s]:batch.start[s + 1]] = torch.from_numpy(val).to(gt)
        assert torch.equal(gk.cpu(), want[0])
        assert torch.equal(gv[:, :heads * hd].cpu().view_as(want[1]), want[1]) and torch.all(gv[:, heads * hd:] == 7)
    assert st.item() == 0


def test_append_token_by_token(qc, dev):
    """A page filled one token a call, scales growing and not, ends as the steps say; zeros,
    values too small for a scale, and the largest finite ones."""
    import torch
    rng = np.random.default_rng(4)
    heads, hd, page, length = 3, 64, 16, 37
    full = Ragged(rng, [1, 1], [length, length], page)
    cache = _random_cache(qc, dev, rng, full.pages, heads, page, hd)
    host = _host(cache)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    mags = np.exp(rng.standard_normal(length) * 2)
    mags[[0, 5, 16, 17]] = [0.0, 0.0, 0.0, 1e-40]
    mags[36] = 1e37
    for t in range(length):
        step = Ragged(rng, [1, 1], [t + 1, t + 1], page, columns=full.columns)
        step.table, step.pages = full.table, full.pages
        k, v = (np.clip(rng.standard_normal((2, heads, hd)), -3, 3).astype(np.float32) * np.float32(mags[t]) for _ in range(2))
        qc.kv8_append(cache, step.device(qc, dev), torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev), dev_status=st)
        _append_reference(host, step, k, v)
        _same_cache(cache, host)
    assert st.item() == 0


def test_append_errors(qc, dev):
    """Non-finite groups, bad pages, lengths and starts: those places stay as they were,
    the rest is done; the blocking form writes nothing."""
    import torch
    rng = np.random.default_rng(9)
    heads, hd, page = 2, 32, 16
    batch = Ragged(rng, [3, 20, 2, 4], [10, 20, 2, 4], page)
    cache = _random_cache(qc, dev, rng, batch.pages, heads, page, hd)
    k, v = (rng.standard_normal((batch.tokens, heads, hd)).astype(np.float32) for _ in range(2))
    k[1, 1, 5], v[4, 0, 0] = np.nan, np.inf
    up = lambda a: torch.from_numpy(a).to(dev)

    def run(change, blocking, expect_done):
        host = _host(cache)
        b = batch.device(qc, dev, tokens=batch.tokens)
        table, start, kv = b.tensors
        change(table, start, kv)
        if blocking:
            with pytest.raises(qc.QcError) as e:
                qc.kv8_append(cache, b, up(k), up(v))
            assert e.value.status == 3
            _same_cache(cache, host)
            return
        st = torch.zeros(1, dtype=torch.int32, device=dev)
        qc.kv8_append(cache, b, up(k), up(v), dev_status=st)
        assert st.item() == 3
        sub = Ragged(rng, batch.new, batch.kv, page)
        sub.table, sub.pages = batch.table.copy(), batch.pages
        sub.new = [n if s in expect_done else 0 for s, n in enumerate(batch.new)]
        _append_reference(host, sub, k, v)
        _same_cache(cache, host)

    def bad_page(table, start, kv):
        table[2, 0] = batch.pages

    def negative_page(table, start, kv):
        table[2, 0] = -1

    def too_long(table, start, kv):
        kv[2] = batch.max_kv + 1

    def more_new_than_held(table, start, kv):
        kv[2] = 1

    def negative_length(table, start, kv):
        kv[2] = -1

    for change, done in ((lambda *a: None, (0, 1, 2, 3)), (bad_page, (0, 1, 3)), (negative_page, (0, 1, 3)),
                         (too_long, (0, 1, 3)), (more_new_than_held, (0, 1, 3)), (negative_length, (0, 1, 3))):
        run(change, True, done)
        run(change, False, done)
    # starts that run backwards or past the rows
    for at, value, done in ((3, 22, (0, 1)), (4, 1000, (0, 1, 2)), (0, -1, (1, 2, 3))):
        def starts(table, start, kv, at=at, value=value):
            start[at] = value
        run(starts, True, done)
        host = _host(cache)
        b = batch.device(qc, dev)
        b.tensors[1][at] = value
        st = torch.zeros(1, dtype=torch.int32, device=dev)
        qc.kv8_append(cache, b, up(np.abs(k)), up(np.abs(v)), dev_status=st)
        assert st.item() == 3


def test_append_of_many_sequences_and_a_long_one(qc, dev):
    """A padded grid of this batch (1024 sequences, 8193 pages each at most) would have more work-items than
    a launch may: the blocking form looks at all rows all the same, the last ones of the long sequence too."""
    import torch
    rng = np.random.default_rng(11)
    page, hd = 16, 16
    new = [1] * 500 + [131072 - 1023] + [1] * 523
    batch = Ragged(rng, new, new, page)
    cache = _random_cache(qc, dev, rng, batch.pages, 1, page, hd)
    host = _host(cache)
    k, v = (rng.standard_normal((batch.tokens, 1, hd)).astype(np.float32) for _ in range(2))
    K, V = torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev)
    b = qc.Kv8Batch(*batch.device(qc, dev).tensors, batch.tokens, batch.tokens, batch.max_kv)
    for at in (int(batch.start[500]), int(batch.start[501]) - 1, batch.tokens - 1):
        V[at, 0, 3] = float("nan")
        with pytest.raises(qc.QcError) as e:
            qc.kv8_append(cache, b, K, V)
        assert e.value.status == 3
        _same_cache(cache, host)
        V[at, 0, 3] = float(v[at, 0, 3])
    qc.kv8_append(cache, b, K, V)
    _append_reference(host, batch, k, v)
    _same_cache(cache, host)


@pytest.mark.parametrize("which", [2, 3], ids=["k", "v"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_append_errors_of_held_scales(qc, dev, which, value):
    """A scale held that is not finite: an error where the page has tokens before the new ones, and
    of no meaning where it has none.  The blocking form writes nothing; the other leaves that page and
    head and does the rest."""
    import torch
    rng = np.random.default_rng(14)
    heads, hd, page = 2, 32, 16
    batch = Ragged(rng, [3, 20, 2, 70], [10, 36, 18, 75], page)
    cache = _random_cache(qc, dev, rng, batch.pages, heads, page, hd)
    k, v = (rng.standard_normal((batch.tokens, heads, hd)).astype(np.float32) for _ in range(2))
    K, V = torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev)
    b = batch.device(qc, dev)
    touched = [(s, c) for s in range(4) for c in range((batch.kv[s] - batch.new[s]) // page, -(-batch.kv[s] // page))]
    held = [(s, c) for s, c in touched if c * page < batch.kv[s] - batch.new[s]]   # tokens before the new ones
    assert held == [(0, 0), (3, 0)]
    for s, c in held:
        keep = [t.clone() for t in cache.tensors]
        cache.tensors[which][batch.table[s, c], 1] = value
        host = _host(cache)
        with pytest.raises(qc.QcError) as e:
            qc.kv8_append(cache, b, K, V)
        assert e.value.status == 3
        _same_cache(cache, host)
        st = torch.zeros(1, dtype=torch.int32, device=dev)
        qc.kv8_append(cache, b, K, V, dev_status=st)
        assert st.item() == 3
        want = [h.copy() for h in host]
        with np.errstate(invalid="ignore"):           # (that page and head, put back below)
            _append_reference(want, batch, k, v)
        pid = batch.table[s, c]
        for w in (which - 2, which):
            want[w][pid, 1] = host[w][pid, 1]
        _same_cache(cache, want)
        for t, o in zip(cache.tensors, keep):
            t.copy_(o)
    # pages that hold nothing yet, and pages of no sequence
    unused = np.setdiff1d(np.arange(batch.pages), batch.table[batch.table >= 0])
    for pid in [batch.table[at] for at in touched if at not in held] + list(unused):
        cache.tensors[which][int(pid)] = value
    host = _host(cache)
    qc.kv8_append(cache, b, K, V)
    _append_reference(host, batch, k, v)
    _same_cache(cache, host)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("which", [2, 3], ids=["k", "v"])
@pytest.mark.parametrize("new,kv,page,hd", [([1, 1, 1], [10, 33, 16], 16, 32), ([3, 150, 0], [40, 150, 9], 16, 64),
                                            ([300, 7], [310, 500], 256, 128)])
def test_gather_errors_of_scales(qc, dev, dtype, which, new, kv, page, hd):
    """A page and head whose scale is not finite is left out (zeros in new tensors) and told
    of, the rest is read; the blocking form writes nothing.  Pages that the call does not read may hold anything."""
    import torch
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(15)
    heads = 2
    batch = Ragged(rng, new, kv, page, 2)
    cache = _random_cache(qc, dev, rng, batch.pages, heads, page, hd)
    b = batch.device(qc, dev)
    read = np.concatenate([batch.places(s, kv[s] - new[s], kv[s])[0] for s in range(len(kv))])
    cache.tensors[which][torch.from_numpy(np.setdiff1d(np.arange(batch.pages), read)).to(dev)] = float("nan")
    full = qc.kv8_gather(cache, b, dtype=dt)
    for value in (float("nan"), float("inf")):
        pid = int(read[-1])
        keep = cache.tensors[which].clone()
        cache.tensors[which][pid, 1] = value
        out = [torch.full((batch.tokens, heads, hd), 7.0, dtype=dt, device=dev) for _ in range(2)]
        with pytest.raises(qc.QcError) as e:
            qc.kv8_gather(cache, b, k=out[0], v=out[1])
        assert e.value.status == 3 and all(bool((o == 7).all()) for o in out)
        for given, rest in ((out, 7.0), (None, 0.0)):
            st = torch.zeros(1, dtype=torch.int32, device=dev)
            if given is None:
                got = qc.kv8_gather(cache, b, dtype=dt, dev_status=st)
            else:
                got = qc.kv8_gather(cache, b, k=out[0], v=out[1], dev_status=st)
            assert st.item() == 3
            for i in range(2):
                want = full[i].clone()
                want[len(read):] = rest
                if i == which - 2:
                    want[torch.from_numpy(np.flatnonzero(read == pid)).to(dev), 1] = rest
                assert torch.equal(got[i], want)
        cache.tensors[which].copy_(keep)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new,spare", [([3, 0, 20, 1, 70], 5), ([1] * 90 + [200], 130), ([64], 64), ([1], 0)])
def test_gather_into_new_tensors(qc, dev, dtype, new, spare):
    """Rows that receive nothing are zeros in tensors that the call makes: those of no sequence,
    of bad lengths (too long, fewer than the new ones), of bad starts and of bad pages."""
    import torch
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(spare)
    heads, hd, page = 3, 48, 16
    batch = Ragged(rng, new, [n + 5 for n in new], page, spare)
    cache = _random_cache(qc, dev, rng, batch.pages, heads, page, hd)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    last = len(new) - 1
    a, e = int(batch.start[last]), int(batch.start[last + 1])
    bad_page = (new[last] + 4) // page                # of the last token
    for bad in ("nothing", "long", "short", "page", "start"):
        b = batch.device(qc, dev)
        left = torch.zeros(batch.tokens, dtype=torch.bool, device=dev)
        left[e:] = True
        if bad == "long":
            b.tensors[2][last] = batch.max_kv + 1
            left[a:e] = True
        elif bad == "short":
            b.tensors[2][last] = new[last] - 1
            left[a:e] = True
        elif bad == "page":
            b.tensors[0][last, bad_page] = batch.pages
            left[e - ((new[last] + 4) % page + 1 if bad_page * page > 5 else new[last]):e] = True
        elif bad == "start":
            b.tensors[1][last + 1] = batch.tokens + 1
            left[a:] = True
        given = [torch.full((batch.tokens, heads, hd), 7.0, dtype=dt, device=dev) for _ in range(2)]
        qc.kv8_gather(cache, b, k=given[0], v=given[1], dev_status=st)
        junk = torch.full((2, batch.tokens, heads, hd), float("nan"), dtype=dt, device=dev)
        del junk                                        # what the new tensors are likely to lie on
        st.zero_()
        for got, want in zip(qc.kv8_gather(cache, b, dtype=dt, dev_status=st), given):
            assert bool((want[left] == 7).all()) and bool((got[left] == 0).all()), bad
            assert torch.equal(got[~left], want[~left])
        assert st.item() == (0 if bad == "nothing" else 3)
    one = qc.kv8_gather(cache, batch.device(qc, dev), k=given[0], dev_status=st)
    assert one[0] is given[0] and bool((one[1][e:] == 0).all())


@pytest.mark.parametrize("bound", [9, 1000, 1 << 40])
def test_loose_bound_of_new_tokens(qc, dev, bound):
    """max_new is a bound only: one above the batch's tokens changes nothing."""
    import torch
    rng = np.random.default_rng(2)
    batch = Ragged(rng, [1, 3], [17, 20], 16)
    cache = _random_cache(qc, dev, rng, batch.pages, 2, 16, 32)
    exact = batch.device(qc, dev)
    loose = qc.Kv8Batch(*exact.tensors, batch.tokens, bound, batch.max_kv)
    host = _host(cache)
    k, v = (torch.from_numpy(rng.standard_normal((batch.tokens, 2, 32)).astype(np.float32)).to(dev) for _ in range(2))
    q = torch.randn(batch.tokens, 4, 32, device=dev)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    qc.kv8_append(cache, loose, k, v, dev_status=st)
    _append_reference(host, batch, k.cpu().numpy(), v.cpu().numpy())
    _same_cache(cache, host)
    for a, b in zip(qc.kv8_gather(cache, loose, dev_status=st), qc.kv8_gather(cache, exact)):
        assert torch.equal(a, b)
    assert torch.equal(qc.kv8_attention(cache, loose, q), qc.kv8_attention(cache, exact, q))
    assert st.item() == 0


def test_errors_in_ragged_batches(qc, dev, route):
    """Bad sequences anywhere in a batch whose blocks are listed, the last one among them, are
    told of and left out; the others are done."""
    import torch
    rng = np.random.default_rng(21)
    new, kv = [150] + [1] * 130, [150] + [1 + i for i in range(130)]
    heads, hd = 2, 64
    for bad in (1, 63, 64, 130):
        batch = Ragged(rng, new, kv, 16)
        cache = _random_cache(qc, dev, rng, batch.pages, heads, 16, hd)
        k, v, q = (torch.from_numpy(rng.standard_normal((batch.tokens, n, hd)).astype(np.float32)).to(dev)
                   for n in (heads, heads, 8))
        row = int(batch.start[bad])
        rest = torch.arange(batch.tokens, device=dev) != row
        for figure in (-1, 0, batch.max_kv + 1):
            host = _host(cache)
            good = batch.device(qc, dev)
            want = qc.kv8_attention(cache, good, q)
            b = batch.device(qc, dev)
            b.tensors[2][bad] = figure
            st = torch.zeros(1, dtype=torch.int32, device=dev)
            out = torch.full_like(q, 7.0)
            qc.kv8_attention(cache, b, q, out=out, dev_status=st)
            assert torch.equal(out[rest], want[rest])
            if figure == 0:                       # no error here: a row that sees nothing
                assert st.item() == 0 and bool((out[row] == 0).all())
            else:
                assert st.item() == 3 and bool((out[row] == 7).all())
            st.zero_()
            gk = torch.full_like(k, 7.0)
            gv = torch.full_like(v, 7.0)
            qc.kv8_gather(cache, b, k=gk, v=gv, dev_status=st)
            assert st.item() == 3
            full = qc.kv8_gather(cache, good)
            assert torch.equal(gk[rest], full[0][rest]) and torch.equal(gv[rest], full[1][rest])
            assert bool((gk[row] == 7).all()) and bool((gv[row] == 7).all())
            st.zero_()
            qc.kv8_append(cache, b, k, v, dev_status=st)
            assert st.item() == 3
            sub = Ragged(rng, batch.new, batch.kv, 16)
            sub.table, sub.pages = batch.table, batch.pages
            sub.new = [n if s != bad else 0 for s, n in enumerate(batch.new)]
            _append_reference(host, sub, k.cpu().numpy(), v.cpu().numpy())
            _same_cache(cache, host)


# ---- attention --------------------------------------------------------------------

@pytest.fixture(params=[0, 1, 2, 3], ids=["auto", "direct16", "direct32", "tiled"])
def route(request, qc):
    """Every kernel of the attention at every size."""
    qc.set_kv8_attention_route(request.param)
    yield request.param
    qc.set_kv8_attention_route(0)


def _attention_reference(host, batch, q, heads, scale, causal, window, half):
    """(out, tolerance) in f64: out is softmax(scale q k^T + mask) v; the tolerance counts
    f32 dots, q and the probabilities in 11 (16-bit q) or 22 bits, f32 sums, one
    rounding to the output's type.  Sums over the keys: at most an addition for each 16
    of them and some for the parts they are split into."""
    kc, vc, ks, vs = host
    hd, kvh = kc.shape[3], kc.shape[1]
    g = heads // kvh
    bits = 2.0 ** -11 if half > 2.0 ** -24 else 2.0 ** -21
    out = np.zeros((batch.tokens, heads, hd))
    tol = np.zeros_like(out)
    for s, (n, length) in enumerate(zip(batch.new, batch.kv)):
        if n == 0:
            continue
        pos = length - n + np.arange(n)
        j = np.arange(length)
        seen = np.ones((n, length), bool)
        if causal:
            seen &= j[None] <= pos[:, None]
        if window:
            seen &= j[None] > pos[:, None] - window
        used = seen.any(0)
        pid = np.where(used, batch.table[s][j // batch.page], 0) if length else j
        slot = j % batch.page
        for h in range(heads):
            K = np.where(used[:, None], kc[pid, h // g, slot].astype(np.float64) * ks[pid, h // g][:, None], 0)
            V = np.where(used[:, None], vc[pid, h // g, slot].astype(np.float64) * vs[pid, h // g][:, None], 0)
            Q = q[batch.start[s]:batch.start[s + 1], h].astype(np.float64)
            z = np.where(seen, scale * (Q @ K.T), -np.inf)
            some = seen.any(1)
            top = np.where(some, z.max(1, initial=-np.inf), 0)
            p = np.exp(z - top[:, None])
            total = p.sum(1)
            p = p / np.where(some, total, 1)[:, None]
            o = p @ V
            # error of a score: f32 dot of hd terms, its scaling and the exponent's argument
            qbits = 2.0 ** -40 if half > 2.0 ** -24 else 2.0 ** -22
            size = np.where(seen, abs(scale) * (np.abs(Q) @ np.abs(K).T), 0).max(1, initial=0)
            # q's bits count from its row's largest element below 2^-17 of it
            small = abs(scale) * np.abs(Q).max(1) * np.abs(K).sum(1).max(initial=0) * 2.0 ** -38
            ds = size * ((hd + 8) * 2.0 ** -24 + qbits) + small + (np.abs(top) + size) * 2.0 ** -22
            spread = p @ np.abs(V)
            # a probability times its page's share of the largest value scale is held in f16
            # times 2^11 (f32 q: 2^15 and a second term): below 2^-14 the half step there is
            # 2^-25, so each key adds at most 2^-36 (2^-40) of that scale times its code
            C = np.where(used[:, None], np.abs(vc[pid, h // g, slot].astype(np.float64)), 0)
            floor = (2.0 ** -36 if half > 2.0 ** -24 else 2.0 ** -40) * np.abs(np.where(used, vs[pid, h // g], 0)).max(initial=0) * (seen @ C)
            out[batch.start[s]:batch.start[s + 1], h] = o
            tol[batch.start[s]:batch.start[s + 1], h] = (
                spread * (bits + 2 * ds[:, None] + (length / 16 + 16) * 2.0 ** -23)
                + floor + half * (1 + 2.0 ** -10) * np.abs(o) + 2.0 ** -25)
    return out, tol


def _attend(qc, dev, rng, new, kv, heads, kvh, hd, page, dtype="bfloat16", causal=True, window=0, spare=0,
            qmag=1.0, scale=None, blocking=False, spread=1.0, cache=None, batch=None, q=None):
    import torch
    batch = batch or Ragged(rng, new, kv, page, spare)
    cache = cache or _random_cache(qc, dev, rng, batch.pages, kvh, page, hd, spread)
    dt = getattr(torch, dtype)
    scale = scale if scale is not None else hd ** -0.5
    if q is None:
        q = torch.from_numpy(rng.standard_normal((batch.tokens, heads, hd)) * qmag).to(dt)
    if spare:
        q[-spare:] = float("nan")
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    out = torch.full((batch.tokens, heads, hd), 7.0, dtype=dt, device=dev)
    qc.kv8_attention(cache, batch.device(qc, dev), q.to(dev), scale=scale, causal=causal, window=window, out=out,
                     dev_status=None if blocking else st)
    want, tol = _attention_reference(_host(cache), batch, q.float().numpy(), heads, float(np.float32(scale)), causal,
                                     window, HALF[dtype])
    used = batch.start[-1]
    got = out.double().cpu().numpy()
    assert np.all(got[used:] == 7.0)
    err = np.abs(got[:used] - want[:used])
    worst = float((err / tol[:used]).max(initial=0)) if used else 0.0
    assert np.all(err <= tol[:used]), (worst, np.argwhere(~(err <= tol[:used]))[:4].tolist())
    assert st.item() == 0
    return out


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("kv", [[1], [2, 15, 16], [17, 31, 32, 33], [63, 64, 65], [127, 128, 129, 200], [600],
                                [1000, 1, 513]])
def test_attention_single_tokens(qc, dev, route, dtype, kv):
    print(f"kv8 attention {dtype} one token each, kv {kv}", flush=True)
    rng = np.random.default_rng(sum(kv))
    _attend(qc, dev, rng, [1] * len(kv), kv, 8, 2, 128, 64, dtype)
    _attend(qc, dev, rng, [1] * len(kv), kv, 4, 4, 64, 16, dtype, blocking=True)


@pytest.mark.parametrize("heads,kvh,hd,page", [
    (1, 1, 16, 16), (2, 1, 32, 16), (7, 1, 64, 32), (14, 2, 64, 128), (8, 8, 80, 64), (6, 2, 96, 16), (16, 1, 128, 64),
    (32, 2, 128, 256), (48, 2, 128, 32), (4, 2, 176, 64), (8, 1, 256, 16), (16, 1, 240, 128), (40, 1, 128, 16)])
@pytest.mark.parametrize("new,kv", [([1, 1], [150, 37]), ([5, 3, 9], [70, 3, 140])])
def test_attention_heads(qc, dev, route, heads, kvh, hd, page, new, kv):
    print(f"kv8 attention heads {heads}/{kvh} hd {hd} page {page} new {new}", flush=True)
    rng = np.random.default_rng(heads * hd + page)
    for dtype in ("bfloat16", "float32"):
        _attend(qc, dev, rng, new, kv, heads, kvh, hd, page, dtype)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("new,kv,heads,kvh,hd,page,causal,window", [
    ([64], [64], 4, 2, 64, 16, True, 0), ([65], [65], 4, 1, 128, 32, True, 0),
    ([130, 0, 1], [130, 50, 77], 8, 2, 128, 64, True, 0), ([300], [700], 2, 2, 64, 128, True, 0),
    ([100, 257], [333, 257], 4, 2, 80, 16, True, 0), ([90, 31], [200, 31], 4, 2, 96, 32, False, 0),
    ([200], [500], 4, 4, 128, 64, True, 50), ([150, 40], [150, 300], 8, 2, 64, 32, True, 1),
    ([33], [400], 8, 1, 128, 16, True, 64), ([70, 70], [70, 200], 2, 1, 256, 64, True, 0),
    ([260], [520], 16, 2, 128, 64, True, 129), ([513], [513], 2, 1, 128, 16, True, 0),
    ([40, 600], [1000, 600], 12, 4, 128, 64, True, 0)])
def test_attention_prompts(qc, dev, route, dtype, new, kv, heads, kvh, hd, page, causal, window):
    print(f"kv8 attention {dtype} new {new} kv {kv} heads {heads}/{kvh} hd {hd} page {page} {causal} {window}", flush=True)
    rng = np.random.default_rng(sum(new) + hd)
    _attend(qc, dev, rng, new, kv, heads, kvh, hd, page, dtype, causal, window, spare=2)


@pytest.mark.parametrize("dtype,new,kv,heads,kvh,hd,page,window", [
    ("bfloat16", [1] * 30 + [90] + [0, 1, 1], [200] * 30 + [120] + [0, 64, 33], 8, 2, 64, 16, 0),
    ("float32", [70] + [2] * 70, [70] + [2 + 7 * i for i in range(70)], 4, 2, 32, 16, 0),
    ("float16", [1] * 129 + [200, 0, 3], [1 + i for i in range(129)] + [210, 40, 3], 6, 1, 80, 32, 40),
    ("bfloat16", [1, 600, 0, 2, 1, 200, 90, 129, 128, 127], [700, 4200, 9, 2, 0, 200, 800, 129, 4000, 300], 32, 2, 64, 64, 0),
    ("bfloat16", [400] + [1] * 9, [9000] + [8990 - 997 * i for i in range(9)], 16, 1, 128, 128, 0),
    ("float32", [1] * 5 + [500] + [3, 130], [50] * 5 + [4500] + [4400, 2000], 16, 1, 64, 16, 0)])
def test_attention_ragged(qc, dev, route, dtype, new, kv, heads, kvh, hd, page, window):
    """Batches whose longest sequence is far longer than most: the row blocks there are
    get listed, and with 2048 rows a key head and enough work long and short go ways of their own."""
    print(f"kv8 attention ragged {dtype} {len(new)} sequences, heads {heads}/{kvh} hd {hd} {window}", flush=True)
    rng = np.random.default_rng(len(new))
    _attend(qc, dev, rng, new, kv, heads, kvh, hd, page, dtype, window=window, spare=3)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new,kv", [([5, 1, 3], [2, 0, 3]), ([200, 7], [100, 0]), ([300], [40]), ([40, 33], [0, 31])])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_rows_that_see_nothing(qc, dev, route, dtype, new, kv, causal):
    """More new tokens than the cache holds, and empty caches: rows before position 0, or
    with no key at all, are zeros."""
    print(f"kv8 attention empty rows {dtype} new {new} kv {kv} causal {causal}", flush=True)
    rng = np.random.default_rng(3)
    out = _attend(qc, dev, rng, new, kv, 4, 2, 64, 16, dtype, causal)
    if causal:
        assert bool((out[:max(new[0] - kv[0], 0)] == 0).all())


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_attention_scales_far_apart(qc, dev, route, dtype):
    """Pages' scales spread over e^+-4, sharp scores, large and small q, and scales of zero."""
    import torch
    rng = np.random.default_rng(12)
    for new, kv in (([1, 1], [300, 90]), ([70], [300])):
        _attend(qc, dev, rng, new, kv, 4, 2, 128, 16, dtype, spread=1.5, qmag=0.3)
        _attend(qc, dev, rng, new, kv, 4, 2, 64, 16, dtype, spread=0.5, qmag=3.0)
        _attend(qc, dev, rng, new, kv, 4, 2, 64, 32, dtype, spread=0.0, qmag=1e-4)
        _attend(qc, dev, rng, new, kv, 4, 2, 64, 32, dtype, spread=0.5, scale=0.0)
        _attend(qc, dev, rng, new, kv, 4, 2, 64, 32, dtype, spread=0.2, scale=-0.05)
        batch = Ragged(rng, new, kv, 16)
        cache = _random_cache(qc, dev, rng, batch.pages, 2, 16, 64)
        for i in (0, 1):                                # some pages hold zeros under a scale of zero
            zero = torch.from_numpy(rng.random((batch.pages, 2)) < 0.4).to(dev)
            cache.tensors[i][zero] = 0
            cache.tensors[2 + i][zero] = 0
        _attend(qc, dev, rng, new, kv, 4, 2, 64, 16, dtype, batch=batch, cache=cache)
        cache.tensors[3].zero_()
        cache.tensors[1].zero_()
        _attend(qc, dev, rng, new, kv, 4, 2, 64, 16, dtype, batch=batch, cache=cache)
        batch = Ragged(rng, new, kv, 16)
        cache = _random_cache(qc, dev, rng, batch.pages, 2, 16, 64)
        for i in (2, 3):                                # negative scales are scales
            cache.tensors[i][torch.from_numpy(rng.random((batch.pages, 2)) < 0.5).to(dev)] *= -1
        _attend(qc, dev, rng, new, kv, 4, 2, 64, 16, dtype, batch=batch, cache=cache)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("new,kv", [([1, 1], [300, 90]), ([70], [300]), ([1], [4000]), ([40, 3], [1500, 31])])
@pytest.mark.parametrize("down", [107, 113, 121])
def test_attention_tiny_value_scales(qc, dev, route, dtype, new, kv, down):
    """Value scales near 1e-34, 1e-36 and 2^-126 (some below it), some of them 0: outputs are those of
    scales 2^down times as large, over 2^down, to within the tolerance there and the spacing of
    the type's subnormals."""
    import torch
    print(f"kv8 attention tiny value scales {dtype} new {new} kv {kv} 2^-{down}", flush=True)
    rng = np.random.default_rng(down + len(new))
    batch = Ragged(rng, new, kv, 16)
    cache = _random_cache(qc, dev, rng, batch.pages, 2, 16, 64)
    # few bits, so that 2^-down of them is exact where it is subnormal too
    vs = rng.integers(0, 256, (batch.pages, 2)).astype(np.float32) * np.float32(2.0 ** -13)
    cache.tensors[3].copy_(torch.from_numpy(vs * np.float32(2.0 ** -down)))
    q = torch.from_numpy(rng.standard_normal((batch.tokens, 4, 64))).to(getattr(torch, dtype))
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    out = qc.kv8_attention(cache, batch.device(qc, dev), q.to(dev), dev_status=st)
    assert st.item() == 0
    if dtype == "float16":
        assert bool((out == 0).all())                 # below half of 2^-24
        return
    host = _host(cache)
    host[3] = vs
    want, tol = _attention_reference(host, batch, q.float().numpy(), 4, 0.125, True, 0, HALF[dtype])
    # half a step of subnormal outputs; the sums of at most 40 ranges are stored in f32
    tol += 2.0 ** (down - (150 if dtype == "float32" else 134)) + 40 * 2.0 ** (down - 150)
    err = np.abs(out.double().cpu().numpy() * 2.0 ** down - want)
    assert np.all(err <= tol), float((err / tol).max())


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("new", [1, 30])
@pytest.mark.parametrize("scale", [1e-34, 1e-36, 2.0 ** -126])
def test_attention_tiny_value_scales_in_some_ranges(qc, dev, route, dtype, new, scale):
    """Whole key ranges of tiny values between normal ones change nothing beyond their own share."""
    rng = np.random.default_rng(new)
    batch = Ragged(rng, [new], [4000], 16)
    cache = _random_cache(qc, dev, rng, batch.pages, 2, 16, 64)
    pid, _ = batch.places(0, 512, 2560)
    cache.tensors[3][np.unique(pid)] = scale
    _attend(qc, dev, rng, [new], [4000], 4, 2, 64, 16, dtype, batch=batch, cache=cache)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_attention_peaked_q(qc, dev, route, dtype):
    """One channel of q far above the rest where the keys hold zero: the others keep
    their bits."""
    import torch
    rng = np.random.default_rng(2)
    for new, kv in (([1, 1], [200, 77]), ([80], [200])):
        batch = Ragged(rng, new, kv, 32)
        cache = _random_cache(qc, dev, rng, batch.pages, 2, 32, 64)
        cache.tensors[0][..., 9] = 0
        q = torch.from_numpy(rng.standard_normal((batch.tokens, 4, 64))).to(getattr(torch, dtype))
        q[:, :, 9] = 1000.0
        _attend(qc, dev, rng, new, kv, 4, 2, 64, 32, dtype, batch=batch, cache=cache, q=q)


def test_attention_f32_keeps_its_second_terms(qc, dev, route):
    """Many probabilities of some size over pages of several scales, beside small scores, so that
    the bound is near 2^-18 of the values' sum: a probability whose two f16 terms do not belong together (one product rounded
    in two ways, once in some 2^13) is 2^-11 of itself off."""
    rng = np.random.default_rng(8)
    _attend(qc, dev, rng, [1] * 256, [20 + s % 31 for s in range(256)], 16, 4, 16, 16, "float32", qmag=0.3, spread=0.3)
    _attend(qc, dev, rng, [60] * 12, [60] * 12, 16, 4, 16, 16, "float32", qmag=0.3, spread=0.3)


def test_attention_nonfinite_q_stays_in_its_row(qc, dev, route):
    import torch
    rng = np.random.default_rng(6)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        for new, kv in (([1, 1, 1], [100, 40, 300]), ([70, 20], [150, 64])):
            batch = Ragged(rng, new, kv, 16)
            cache = _random_cache(qc, dev, rng, batch.pages, 2, 16, 64)
            q = torch.from_numpy(rng.standard_normal((batch.tokens, 8, 64))).to(dtype).to(dev)
            b = batch.device(qc, dev)
            clean = qc.kv8_attention(cache, b, q)
            q[1, 3, 5], q[0, 0, 0], q[2, 7, 63] = float("nan"), float("inf"), float("-inf")
            got = qc.kv8_attention(cache, b, q)
            bad = torch.zeros(batch.tokens, 8, dtype=torch.bool, device=dev)
            bad[1, 3] = bad[0, 0] = bad[2, 7] = True
            assert torch.equal(got[~bad], clean[~bad])
            assert bool(torch.isnan(got[1, 3]).all())
            assert not bool(torch.isfinite(got[0, 0]).any()) and not bool(torch.isfinite(got[2, 7]).any())


def test_attention_ignores_what_it_does_not_see(qc, dev, route):
    """Slots past the length, pages before a window and unused table entries may hold
    anything, NaN scales too."""
    import torch
    rng = np.random.default_rng(21)
    for new, kv, window in (([1, 1], [100, 33], 0), ([1, 1], [300, 290], 40), ([60, 5], [200, 70], 30), ([70], [290], 0)):
        batch = Ragged(rng, new, kv, 32, extra_pages=5)
        cache = _random_cache(qc, dev, rng, batch.pages, 2, 32, 64)
        q = torch.from_numpy(rng.standard_normal((batch.tokens, 4, 64))).to(torch.bfloat16).to(dev)
        b = batch.device(qc, dev)
        st = torch.zeros(1, dtype=torch.int32, device=dev)
        want = qc.kv8_attention(cache, b, q, window=window, dev_status=st)
        seen = np.zeros((batch.pages, 32), bool)
        for s in range(len(kv)):
            lo = max(0, kv[s] - new[s] + 1 - window) if window else 0
            pid, slot = batch.places(s, lo, kv[s])
            seen[pid, slot] = True
            if window:
                b.tensors[0][s, :lo // 32] = -1
        hide = torch.from_numpy(~seen).to(dev)
        for i in range(2):
            cache.tensors[i].masked_fill_(hide[:, None, :, None], 127)
            cache.tensors[2 + i][torch.from_numpy(~seen.any(1)).to(dev)] = float("nan")
        got = qc.kv8_attention(cache, b, q, window=window, dev_status=st)
        assert torch.equal(got, want)
        assert torch.equal(qc.kv8_attention(cache, b, q, window=window), want)
        assert st.item() == 0


def test_attention_errors(qc, dev, route):
    """A bad page or length sets the status; a sequence whose figures are wrong stays
    unwritten and the others are done."""
    import torch
    rng = np.random.default_rng(30)
    for new, kv in (([1, 1, 1], [100, 200, 50]), ([60, 70, 40], [100, 200, 50])):
        batch = Ragged(rng, new, kv, 16)
        cache = _random_cache(qc, dev, rng, batch.pages, 2, 16, 64)
        q = torch.from_numpy(rng.standard_normal((batch.tokens, 4, 64))).to(torch.float16).to(dev)
        want = qc.kv8_attention(cache, batch.device(qc, dev), q)
        a, z = int(batch.start[1]), int(batch.start[2])
        for bad in ("page", "scale", "long", "negative", "start"):
            b = batch.device(qc, dev)
            if bad == "page":
                b.tensors[0][1, 2] = batch.pages
            elif bad == "scale":
                held = cache.tensors[3].clone()
                cache.tensors[3][batch.table[1, 2], 1] = float("inf")
            elif bad == "long":
                b.tensors[2][1] = batch.max_kv + 1
            elif bad == "negative":
                b.tensors[2][1] = -5
            else:
                b.tensors[1][3] = batch.tokens + 1
            out = torch.full_like(q, 7.0)
            with pytest.raises(qc.QcError) as e:
                qc.kv8_attention(cache, b, q, out=out)
            assert e.value.status == 3 and bool((out == 7).all())
            st = torch.zeros(1, dtype=torch.int32, device=dev)
            qc.kv8_attention(cache, b, q, out=out, dev_status=st)
            assert st.item() == 3
            assert torch.equal(out[:a], want[:a])
            if bad == "start":
                assert torch.equal(out[a:z], want[a:z]) and bool((out[z:] == 7).all())
            else:
                assert torch.equal(out[z:], want[z:])
                if bad in ("page", "scale"):
                    # as if the page were not there: the same for both ways to lose it
                    assert bool(torch.isfinite(out[a:z]).all())
                else:
                    assert bool((out[a:z] == 7).all())
            if bad == "scale":
                assert torch.equal(out[a:z, :2], want[a:z, :2])      # the other key head's rows
                cache.tensors[3].copy_(held)


@pytest.mark.parametrize("new,kv,heads,kvh", [([1] * 5, [900, 1, 64, 500, 333], 8, 2), ([1], [4000], 4, 1),
                                              ([150, 40], [400, 64], 8, 2), ([20, 3], [2000, 64], 8, 2)])
def test_attention_repeats_and_graph(qc, dev, route, new, kv, heads, kvh):
    """Bit-identical reruns; captured and replayed with eager calls of other sizes on
    the same stream between."""
    import torch
    rng = np.random.default_rng(40)
    batch = Ragged(rng, new, kv, 64)
    cache = _random_cache(qc, dev, rng, batch.pages, kvh, 64, 128)
    q = torch.from_numpy(rng.standard_normal((batch.tokens, heads, 128))).to(torch.bfloat16).to(dev)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    b = batch.device(qc, dev)
    other_batch = Ragged(rng, [1, 2], [700, 90], 64)
    other_cache = _random_cache(qc, dev, rng, other_batch.pages, 2, 64, 64)
    ob = other_batch.device(qc, dev)
    oq = torch.randn(3, 8, 64, device=dev)
    out = torch.empty_like(q)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        qc.kv8_attention(other_cache, ob, oq, dev_status=st)
        want = qc.kv8_attention(cache, b, q, dev_status=st)
        for _ in range(3):
            assert torch.equal(qc.kv8_attention(cache, b, q, dev_status=st), want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        qc.kv8_attention(cache, b, q, out=out, dev_status=st)
    for rep in range(3):
        with torch.cuda.stream(s):
            out.fill_(float("nan"))
            qc.kv8_attention(other_cache, ob, oq, dev_status=st)
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), rep
    # lengths that shrink after the capture: the graph reads them
    b.tensors[2].copy_(torch.tensor([max(1, k - 5) if n == 1 else k for n, k in zip(new, kv)], dtype=torch.int32))
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, qc.kv8_attention(cache, b, q))
    assert st.item() == 0
    del graph


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new,kv,heads,kvh,window", [
    ([1], [4000], 8, 2, 0), ([1, 0, 1], [2500, 9000, 3000], 8, 2, 0), ([12, 3], [1500, 4000], 4, 2, 0),
    ([1], [9000], 4, 1, 2000), ([1] * 8, [3000 + 500 * i for i in range(8)], 8, 2, 0)])
def test_attention_under_a_loose_bound(qc, dev, dtype, new, kv, heads, kvh, window):
    """Key ranges are cut from the lengths, not from max_kv: a bound far above them gives the bits of the
    tight one where both join more than 8 ranges, as here (256 CUs).  Sequences without new tokens, and
    those of bad figures, do not count."""
    import torch
    print(f"kv8 attention loose bound {dtype} new {new} kv {kv} {window}", flush=True)
    rng = np.random.default_rng(len(new))
    columns = 131072 // 16
    batch = Ragged(rng, new, kv, 16, columns=columns)
    cache = _random_cache(qc, dev, rng, batch.pages, kvh, 16, 64)
    q = torch.from_numpy(rng.standard_normal((batch.tokens, heads, 64))).to(getattr(torch, dtype)).to(dev)
    most = max(k for n, k in zip(new, kv) if n)
    bounds = [131072] if window else [16384, 65536, 131072]
    try:
        for r in (0, 1, 2):
            qc.set_kv8_attention_route(r)
            st = torch.zeros(1, dtype=torch.int32, device=dev)
            tight = None
            if 0 not in new:
                tight = qc.kv8_attention(cache, batch.device(qc, dev, max_kv=most), q, window=window, dev_status=st)
            for bound in bounds:
                got = qc.kv8_attention(cache, batch.device(qc, dev, max_kv=bound), q, window=window, dev_status=st)
                if tight is None:                    # (the sequence without new tokens breaks the tight bound)
                    tight = got
                assert torch.equal(got, tight), (r, bound)
            assert st.item() == 0
            if 0 in new:
                b = batch.device(qc, dev, max_kv=131072)
                b.tensors[2][new.index(0)] = 1
                assert torch.equal(qc.kv8_attention(cache, b, q, window=window, dev_status=st), tight)
            if len(new) == 8:                        # the longest goes bad: the others' ranges are their own longest's
                b = batch.device(qc, dev, max_kv=131072)
                b.tensors[2][7] = 131073
                c = Ragged(rng, new[:7], kv[:7], 16, columns=columns)
                c.table = batch.table[:7]
                got = qc.kv8_attention(cache, b, q, window=window, dev_status=st)
                alone = qc.kv8_attention(cache, c.device(qc, dev, max_kv=131072), q[:7], window=window)
                assert st.item() == 3 and torch.equal(got[:7], alone)
    finally:
        qc.set_kv8_attention_route(0)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new,kv,heads,kvh", [
    ([1] * 70, [5000 - 70 * i for i in range(70)], 8, 8), ([1] * 40 + [30] + [2] * 29, [4200 - 59 * i for i in range(70)], 16, 8)])
def test_attention_of_many_sequences_under_a_loose_bound(qc, dev, dtype, new, kv, heads, kvh):
    """Blocks enough to fill the chip, and ranges besides: against 64 bits, and the tight bound's bits."""
    import torch
    rng = np.random.default_rng(heads)
    batch = Ragged(rng, new, kv, 16, spare=1, columns=32768 // 16)
    cache = _random_cache(qc, dev, rng, batch.pages, kvh, 16, 16)
    _attend(qc, dev, rng, new, kv, heads, kvh, 16, 16, dtype, spare=1, cache=cache, batch=batch)
    rng = np.random.default_rng(5)
    q = torch.from_numpy(rng.standard_normal((batch.tokens, heads, 16))).to(getattr(torch, dtype)).to(dev)
    tight = qc.kv8_attention(cache, batch.device(qc, dev), q)
    for bound in (8192, 16384, 32768):
        assert torch.equal(qc.kv8_attention(cache, batch.device(qc, dev, max_kv=bound), q), tight), bound


@pytest.mark.parametrize("new,heads,kvh", [(1, 8, 2), (5, 8, 1), (90, 4, 2)])
def test_attention_replayed_as_lengths_grow(qc, dev, route, new, heads, kvh):
    """Captured once under a bound of 65536 keys, replayed at lengths from one to 20000: each time the
    eager call's bits, and right against 64 bits."""
    import torch
    rng = np.random.default_rng(new)
    full = Ragged(rng, [new, new], [20000, 9000], 16, columns=65536 // 16)
    cache = _random_cache(qc, dev, rng, full.pages, kvh, 16, 64)
    q = torch.from_numpy(rng.standard_normal((full.tokens, heads, 64))).to(torch.bfloat16)
    Q, st = q.to(dev), torch.zeros(1, dtype=torch.int32, device=dev)
    b = full.device(qc, dev, max_kv=65536)
    out = torch.zeros_like(Q)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        qc.kv8_attention(cache, b, Q, out=out, dev_status=st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        qc.kv8_attention(cache, b, Q, out=out, dev_status=st)
    host = _host(cache)
    for kv in ([new, 0], [new + 30, new], [600, 90], [5000, 300], [20000, 9000]):
        b.tensors[2].copy_(torch.tensor(kv, dtype=torch.int32))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            out.fill_(float("nan"))
            graph.replay()
            eager = qc.kv8_attention(cache, b, Q, dev_status=st)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        at = Ragged(rng, [new, new], kv, 16, columns=full.columns)
        at.table = full.table
        want, tol = _attention_reference(host, at, q.float().numpy(), heads, 0.125, True, 0, HALF["bfloat16"])
        assert np.all(np.abs(out.double().cpu().numpy() - want) <= tol), kv
    assert st.item() == 0
    del graph


def test_attention_shared_pages(qc, dev, route):
    """Sequences that share their first pages, and a page that one sequence holds twice."""
    import torch
    rng = np.random.default_rng(33)
    batch = Ragged(rng, [1, 40, 2], [100, 90, 70], 16)
    batch.table[1, :4] = batch.table[0, :4]
    batch.table[2, :3] = batch.table[0, :3]
    batch.table[2, 3] = batch.table[2, 1]
    for dtype in ("float32", "bfloat16"):
        _attend(qc, dev, rng, batch.new, batch.kv, 8, 2, 64, 16, dtype, batch=batch)


def test_attention_from_threads(qc, dev):
    """Calls of several host threads, on one stream and on streams of their own, each with
    keys that are split and joined: every result is the lone call's."""
    import threading
    import torch
    rng = np.random.default_rng(17)
    batch = Ragged(rng, [1, 40, 1], [1500, 900, 30], 32)
    cache = _random_cache(qc, dev, rng, batch.pages, 2, 32, 64)
    b = batch.device(qc, dev)
    qs = [torch.from_numpy(rng.standard_normal((batch.tokens, 8, 64))).to(dev, torch.bfloat16) for _ in range(4)]
    want = [qc.kv8_attention(cache, b, q) for q in qs]
    torch.cuda.synchronize()
    shared, wrong = torch.cuda.Stream(), []

    def work(i):
        st = torch.zeros(1, dtype=torch.int32, device=dev)
        torch.cuda.synchronize()
        with torch.cuda.stream(shared if i < 2 else torch.cuda.Stream()):
            for _ in range(25):
                out = qc.kv8_attention(cache, b, qs[i], dev_status=st)
                if not torch.equal(out, want[i]):
                    wrong.append(i)
                    return
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_attention_without_room_for_its_sums(qc, dev):
    """A bound of keys whose ranges would take more memory than the device has is an error, with
    nothing written; the next call is none the worse."""
    import torch
    rng = np.random.default_rng(1)
    batch = Ragged(rng, [8192], [8192], 256, columns=1 << 22)
    cache = _random_cache(qc, dev, rng, batch.pages, 1, 256, 16)
    q = torch.randn(8192, 32, 16, device=dev)
    out = torch.full_like(q, 7.0)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    try:
        qc.set_kv8_attention_route(1)
        with pytest.raises(qc.QcError) as e:
            qc.kv8_attention(cache, batch.device(qc, dev, max_kv=1 << 30), q, out=out, dev_status=st)
        assert e.value.status in (4, 5)
    finally:
        qc.set_kv8_attention_route(0)
    assert bool((out == 7).all()) and st.item() == 0
    _attend(qc, dev, rng, [1, 40], [100, 700], 8, 2, 64, 16)


def test_attention_strided_rows(qc, dev, route):
    """q inside fused projection rows, out inside wider rows; odd element offsets."""
    import torch
    rng = np.random.default_rng(50)
    for dtype in (torch.float32, torch.bfloat16):
        for new, kv in (([1, 1, 1], [100, 7, 300]), ([66, 3], [100, 90])):
            batch = Ragged(rng, new, kv, 16)
            cache = _random_cache(qc, dev, rng, batch.pages, 2, 16, 48)
            q = torch.from_numpy(rng.standard_normal((batch.tokens, 6, 48))).to(dtype).to(dev)
            b = batch.device(qc, dev)
            want = qc.kv8_attention(cache, b, q)
            for pad, shift in ((8, 0), (3, 1)):
                t, row = batch.tokens, 6 * 48 + pad
                rows = torch.zeros(t * row + shift, dtype=dtype, device=dev)[shift:].view(t, row)
                rows[:, :288] = q.view(t, -1)
                wide = torch.full((t * (row + 2) + shift,), 7.0, dtype=dtype, device=dev)[shift:].view(t, row + 2)
                qc.kv8_attention(cache, b, rows[:, :288].unflatten(1, (6, 48)), out=wide[:, :288].unflatten(1, (6, 48)))
                assert torch.equal(wide[:, :288].reshape(t, 6, 48), want) and bool((wide[:, 288:] == 7).all())


def test_attention_far_into_a_large_cache(qc, dev, route):
    """Pages whose byte offsets pass 32 bits."""
    import torch
    pages, kvh, page, hd = 18000, 8, 256, 128            # 4.7 GB each of K and V
    rng = np.random.default_rng(60)
    codes = [torch.zeros(pages, kvh, page, hd, dtype=torch.int8, device=dev) for _ in range(2)]
    scales = [torch.full((pages, kvh), 0.01, device=dev) for _ in range(2)]
    cache = qc.Kv8Cache(*codes, *scales)
    batch = Ragged(rng, [1, 40], [600, 40], page)
    batch.table[0, :3] = [17999, 3, 17000]
    batch.table[1, :1] = [17500]
    b = batch.device(qc, dev)
    x = [torch.from_numpy(rng.standard_normal((600, kvh, hd))).float().to(dev) for _ in range(2)]
    one = Ragged(rng, [600, 0], [600, 40], page)
    one.table = batch.table
    qc.kv8_append(cache, one.device(qc, dev), *x)
    two = Ragged(rng, [0, 40], [600, 40], page)
    two.table = batch.table
    qc.kv8_append(cache, two.device(qc, dev), x[0][:40].contiguous(), x[1][:40].contiguous())
    q = torch.from_numpy(rng.standard_normal((41, 16, hd))).float().to(dev)
    out = qc.kv8_attention(cache, b, q)
    # the same sequences in a small cache
    small = _random_cache(qc, dev, rng, 4, kvh, page, hd)
    sb = Ragged(rng, [1, 40], [600, 40], page)
    ids = [17999, 3, 17000, 17500]
    for t, big in zip(small.tensors, cache.tensors):
        t.copy_(big[ids])
    sb.table = np.array([[0, 1, 2], [3, -7, -7]], np.int32)
    assert torch.equal(out, qc.kv8_attention(small, sb.device(qc, dev), q))
    # and against 64 bits
    want, tol = _attention_reference(_host(small), sb, q.cpu().numpy(), 16, float(np.float32(hd ** -0.5)), True, 0, HALF["float32"])
    assert np.all(np.abs(out.double().cpu().numpy() - want) <= tol)


def test_a_low_bit_layer(qc, dev, route):
    """Projections in MXFP4, rotation, append and attention of a ragged batch, step by step
    over a prompt and two decoding steps: the same as each operator alone on the values
    that the one before gave, and near full precision."""
    import torch
    torch.manual_seed(0)
    heads, kvh, hd, hidden, page = 8, 2, 64, 256, 16
    rows = (heads + 2 * kvh) * hd
    w = 0.06 * torch.randn(rows, hidden, device=dev)
    wc, ws = qc.quantize_mxfp4(w)
    W = qc.dequantize_mxfp4(wc, ws).double()
    cosine, sine = qc.rope_table(256, hd)
    cache = qc.kv8_cache(40, kvh, page, hd)
    rng = np.random.default_rng(0)
    held = [0, 0, 0]
    table = Ragged(rng, [1, 1, 1], [130, 70, 40], page, extra_pages=5)
    keys, vals = [[], [], []], [[], [], []]
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    for new in ([120, 33, 1], [1, 1, 1], [1, 0, 1]):
        held = [h + n for h, n in zip(held, new)]
        batch = Ragged(rng, new, held, page, columns=table.columns)
        batch.table = table.table
        b = batch.device(qc, dev)
        t = batch.tokens
        x = torch.randn(t, hidden, device=dev, dtype=torch.bfloat16)
        xc, xs = qc.quantize_mxfp4(x, dev_status=st)
        y = qc.mxfp4_gemm(wc, ws, xc, xs, dtype=torch.bfloat16)
        pos = torch.cat([torch.arange(h - n, h, dtype=torch.int32) for h, n in zip(held, new)]).to(dev)
        qk = y[:, :(heads + kvh) * hd].unflatten(1, (heads + kvh, hd))
        qc.rope(qk, cosine, sine, pos, out=qk, dev_status=st)
        qc.kv8_append(cache, b, y[:, heads * hd:(heads + kvh) * hd], y[:, (heads + kvh) * hd:], dev_status=st)
        out = qc.kv8_attention(cache, b, y[:, :heads * hd].unflatten(1, (heads, hd)), dev_status=st)
        # in 64 bits from the quantised activations on
        Y = qc.dequantize_mxfp4(xc, xs).double() @ W.T
        angle = pos.double()[:, None] * (10000.0 ** (-torch.arange(hd // 2, device=dev).double() * 2 / hd))[None]
        z = Y[:, :(heads + kvh) * hd].view(t, heads + kvh, 2, hd // 2)
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        rot = torch.cat([z[:, :, 0] * c - z[:, :, 1] * s, z[:, :, 1] * c + z[:, :, 0] * s], -1)
        V = Y[:, (heads + kvh) * hd:].view(t, kvh, hd)
        for i in range(3):
            a, e = batch.start[i], batch.start[i + 1]
            keys[i].append(rot[a:e, heads:])
            vals[i].append(V[a:e])
            if e == a:
                continue
            K, U = torch.cat(keys[i]), torch.cat(vals[i])
            for h in range(heads):
                sc = rot[a:e, h] @ K[:, h // 4].T / math.sqrt(hd)
                mask = torch.arange(held[i], device=dev)[None] > torch.arange(held[i] - new[i], held[i], device=dev)[:, None]
                want = torch.softmax(sc.masked_fill(mask, -math.inf), -1) @ U[:, h // 4]
                # int8 steps of a page's largest value: about 1% of a normal value each
                got = out[a:e, h].double()
                assert ((got - want).norm() / want.norm()).item() < 0.03
    assert st.item() == 0


def test_a_captured_decoding_step(qc, dev):
    """The layer's operators captured once for a batch whose lengths, positions and rows change
    between the replays; another captured batch and eager calls share the stream's workspaces.
    Every replay is the eager step's, bit for bit, cache and all."""
    import torch
    torch.manual_seed(1)
    heads, kvh, hd, hidden, page = 8, 2, 64, 224, 16
    wc, ws = qc.quantize_mxfp4(0.06 * torch.randn((heads + 2 * kvh) * hd, hidden, device=dev))
    cosine, sine = qc.rope_table(2048, hd)
    rng = np.random.default_rng(5)
    st = torch.zeros(1, dtype=torch.int32, device=dev)

    def step(cache, b, x, pos):
        xc, xs = qc.quantize_mxfp4(x, dev_status=st)
        y = qc.mxfp4_gemm(wc, ws, xc, xs, dtype=torch.bfloat16)
        qk = y[:, :(heads + kvh) * hd].unflatten(1, (heads + kvh, hd))
        qc.rope(qk, cosine, sine, pos, out=qk, dev_status=st)
        qc.kv8_append(cache, b, y[:, heads * hd:(heads + kvh) * hd], y[:, (heads + kvh) * hd:], dev_status=st)
        return qc.kv8_attention(cache, b, y[:, :heads * hd].unflatten(1, (heads, hd)), dev_status=st)

    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    runs = []
    with torch.cuda.stream(stream):
        for held in ([700, 15, 1300, 0], [40, 1, 64]):
            batch = Ragged(rng, [1] * len(held), [h + 40 for h in held], page)
            b = batch.device(qc, dev)
            b.tensors[2].copy_(torch.tensor([h + 1 for h in held], dtype=torch.int32))
            cache = _random_cache(qc, dev, rng, batch.pages, kvh, page, hd)
            x = torch.randn(len(held), hidden, device=dev, dtype=torch.bfloat16)
            pos = (b.tensors[2] - 1).clone()
            keep = [c.clone() for c in cache.tensors]
            step(cache, b, x, pos)                # sizes the workspaces
            for c, k in zip(cache.tensors, keep):
                c.copy_(k)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = step(cache, b, x, pos)
            runs.append((cache, b, x, pos, graph, out))
        for rep in range(6):
            for cache, b, x, pos, graph, out in runs:
                x.copy_(torch.randn_like(x))
                other = qc.Kv8Cache(*[c.clone() for c in cache.tensors])
                graph.replay()
                got = out.clone()
                assert torch.equal(got, step(other, b, x, pos))
                for c, o in zip(cache.tensors, other.tensors):
                    assert torch.equal(c, o)
                b.tensors[2].add_(1 + rep % 2 * 3)      # (slots between hold what they held)
                pos.copy_(b.tensors[2] - 1)
                torch.cuda.synchronize()
    assert st.item() == 0


@pytest.mark.parametrize("new,kv,route", [
    ([1] * 70, 4096, 3), ([1] * 40 + [260] + [1] * 29, 4096, 3), ([1] * 9 + [1024] * 17 + [1] * 50, 16384, 0),
    ([1, 300, 2], 40000, 3), ([700], 70000, 3)])
def test_attention_passes_of_the_layout(qc, dev, new, kv, route):
    """More keys than are laid out at a time (1 GB) or than one range holds: the same values as read
    directly, within both forms' rounding."""
    import torch
    rng = np.random.default_rng(70)
    seqs, kvh, hd = len(new), 8, 128
    batch = Ragged(rng, new, [kv - 37 * (s % 5) for s in range(seqs)], 64)
    g = torch.Generator(device=dev).manual_seed(3)
    shape = (batch.pages, kvh, 64, hd)
    codes = [torch.randint(-127, 128, shape, generator=g, device=dev, dtype=torch.int8) for _ in range(2)]
    scales = [torch.rand(batch.pages, kvh, generator=g, device=dev) / 60 for _ in range(2)]
    cache = qc.Kv8Cache(*codes, *scales)
    q = torch.randn(batch.tokens, 16, hd, generator=g, device=dev)
    b = batch.device(qc, dev)
    try:
        qc.set_kv8_attention_route(1)
        direct = qc.kv8_attention(cache, b, q)
        qc.set_kv8_attention_route(route)
        tiled = qc.kv8_attention(cache, b, q)
    finally:
        qc.set_kv8_attention_route(0)
    # f32 q: 22 bits of each operand, 64 tiles' f32 sums: 2^-18 of the values' size
    assert ((direct - tiled).abs().max() / direct.abs().max()).item() < 2.0 ** -14


@pytest.mark.parametrize("dtype,new,kv,heads,kvh,hd,window", [
    ("bfloat16", [1024, 700], [2100, 700], 16, 4, 128, 0), ("float32", [2100], [2100], 16, 4, 64, 0),
    ("float16", [513, 1000], [900, 3000], 8, 2, 256, 700), ("bfloat16", [2700], [2700], 8, 8, 80, 0)])
def test_attention_long_prompts(qc, dev, dtype, new, kv, heads, kvh, hd, window):
    """Sizes at which the tiled kernels are chosen, and splits of their keys; against 64 bits
    on the GPU, and against the other kernels."""
    import torch
    rng = np.random.default_rng(sum(kv))
    batch = Ragged(rng, new, kv, 32, 3)
    cache = _random_cache(qc, dev, rng, batch.pages, kvh, 32, hd, 0.3)
    q = torch.from_numpy(rng.standard_normal((batch.tokens, heads, hd))).to(getattr(torch, dtype)).to(dev)
    b = batch.device(qc, dev)
    want = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    size, score = torch.zeros_like(want), 0.0
    for s in range(len(kv)):
        pid, slot = (torch.from_numpy(x).to(dev) for x in batch.places(s, 0, kv[s]))
        K, V = (cache.tensors[i][pid.long(), :, slot].double() * cache.tensors[2 + i][pid.long()].double()[..., None]
                for i in range(2))
        at = torch.arange(kv[s] - new[s], kv[s], device=dev)[:, None]
        j = torch.arange(kv[s], device=dev)[None]
        hide = j > at
        if window:
            hide = hide | (j <= at - window)
        a, e = batch.start[s], batch.start[s + 1]
        for h in range(heads):
            z = (q[a:e, h].double() @ K[:, h // (heads // kvh)].T.contiguous()) * float(np.float32(hd ** -0.5))
            score = max(score, z.abs().max().item())
            p = torch.softmax(z.masked_fill(hide, -math.inf), -1)
            want[a:e, h] = p @ V[:, h // (heads // kvh)]
            size[a:e, h] = p @ V[:, h // (heads // kvh)].abs()
    # probabilities in 11 (22) bits; scores of f32 dots whose terms' magnitudes sum to a few
    # times the largest score; sums over up to 3000 keys in steps of 16; the output's rounding
    bits = 2.0 ** -11 if dtype != "float32" else 2.0 ** -21
    tol = size * (bits + 2 * 4 * score * (hd + 8) * 2.0 ** -24 + 200 * 2.0 ** -23) + HALF[dtype] * (1 + 2.0 ** -10) * want.abs() + 2.0 ** -24
    outs = []
    try:
        for r in (0, 1, 2, 3):
            qc.set_kv8_attention_route(r)
            out = qc.kv8_attention(cache, b, q, window=window)
            assert bool(((out.double() - want).abs() <= tol)[:batch.start[-1]].all()), r
            outs.append(out)
    finally:
        qc.set_kv8_attention_route(0)
    assert any(torch.equal(outs[0], o) for o in outs[1:])     # the sizes choose one of them


@pytest.mark.parametrize("dtype,long,short,kv_long,kv_short,heads,kvh,hd,window", [
    # 512 rows a key head and more are laid out, the others read directly
    ("bfloat16", [900, 128, 900], [127] + [1] * 27 + [0, 9], [1500, 2000, 900], 3000, 32, 8, 128, 0),
    ("float16", [600, 512, 700], [511] + [1] * 16 + [100, 0, 2], [2500, 512, 1800], 2400, 16, 16, 80, 700),
    ("float32", [1500, 256], [255] + [1] * 9 + [7], [3000, 1100], 2900, 6, 3, 256, 0),
    # up to 1024 keys: 256 rows and more
    ("bfloat16", [300, 64, 250], [63] + [1] * 36 + [20, 0], [300, 1000, 700], 1024, 32, 8, 64, 0),
    ("float32", [300, 260], [40] + [3] * 30, [900, 260], 1000, 32, 8, 32, 100)])
def test_attention_mixed_batches(qc, dev, dtype, long, short, kv_long, kv_short, heads, kvh, hd, window):
    """Batches of a few long prompts and many short ones at which each kind goes to a kernel of its own (checked
    against the other kernels' bits); sequences at the border, without rows and without keys; against 64 bits."""
    import torch
    print(f"kv8 attention mixed {dtype} {len(long)}+{len(short)} heads {heads}/{kvh} hd {hd} {window}", flush=True)
    rng = np.random.default_rng(len(short) + hd)
    kv_few = [max(n, kv_short - 61 * i) for i, n in enumerate(short)]
    kv_few[3] = 0                                     # one row that sees nothing
    order = rng.permutation(len(long) + len(short))
    new, kv = [(long + short)[i] for i in order], [(kv_long + kv_few)[i] for i in order]
    is_long = [bool(i < len(long)) for i in order]
    batch = Ragged(rng, new, kv, 32, 3)
    cache = _random_cache(qc, dev, rng, batch.pages, kvh, 32, hd, 0.3)
    q = torch.from_numpy(rng.standard_normal((batch.tokens, heads, hd))).to(getattr(torch, dtype)).to(dev)
    q[-3:] = float("nan")
    b = batch.device(qc, dev)
    group = heads // kvh
    want = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    size, score = torch.zeros_like(want), 0.0
    rows_long = torch.zeros(batch.tokens, dtype=torch.bool, device=dev)
    for s in range(len(kv)):
        a, e = int(batch.start[s]), int(batch.start[s + 1])
        rows_long[a:e] = is_long[s]
        if e == a or kv[s] == 0:
            continue
        pid, slot = (torch.from_numpy(x).to(dev) for x in batch.places(s, 0, kv[s]))
        K, V = (cache.tensors[i][pid.long(), :, slot].double() * cache.tensors[2 + i][pid.long()].double()[..., None]
                for i in range(2))
        at = torch.arange(kv[s] - new[s], kv[s], device=dev)[:, None]
        j = torch.arange(kv[s], device=dev)[None]
        hide = (j > at) | (j <= at - window) if window else j > at
        for h in range(heads):
            z = (q[a:e, h].double() @ K[:, h // group].T.contiguous()) * float(np.float32(hd ** -0.5))
            score = max(score, z.abs().max().item())
            p = torch.softmax(z.masked_fill(hide, -math.inf), -1)
            want[a:e, h] = p @ V[:, h // group]
            size[a:e, h] = p @ V[:, h // group].abs()
    # as in test_attention_long_prompts: probabilities in 11 (22) bits; scores of f32 dots whose terms' magnitudes sum
    # to a few times the largest score; sums over up to 3000 keys in steps of 16; the output's rounding
    bits = 2.0 ** -11 if dtype != "float32" else 2.0 ** -21
    tol = size * (bits + 2 * 4 * score * (hd + 8) * 2.0 ** -24 + 200 * 2.0 ** -23) + HALF[dtype] * (1 + 2.0 ** -10) * want.abs() + 2.0 ** -24
    used = int(batch.start[-1])
    outs = []
    try:
        for r in (0, 1, 2, 3):
            qc.set_kv8_attention_route(r)
            st = torch.zeros(1, dtype=torch.int32, device=dev)
            out = torch.full_like(q, 7.0)
            qc.kv8_attention(cache, b, q, window=window, out=out, dev_status=st)
            assert st.item() == 0 and bool((out[used:] == 7).all())
            assert bool(((out.double() - want).abs() <= tol)[:used].all()), r
            if r == 0:
                for _ in range(2):
                    again = torch.full_like(q, 7.0)
                    qc.kv8_attention(cache, b, q, window=window, out=again, dev_status=st)
                    assert torch.equal(again, out)
            outs.append(out)
    finally:
        qc.set_kv8_attention_route(0)
    short_rows = ~rows_long
    short_rows[used:] = False
    assert not torch.equal(outs[0][rows_long], outs[1][rows_long]) and not torch.equal(outs[0][rows_long], outs[2][rows_long])
    assert not torch.equal(outs[0][short_rows], outs[3][short_rows])
