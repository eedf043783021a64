"""The paged K/V cache and the draft check on the GPU against plain implementations in 64 bits: rows into and
out of the pages (every cache type, row type, page size and head_dim, ragged batches), attention over the pages
(decode, drafts and prompts; windows, soft caps, head groups, leftovers behind the sequences), drafted tokens, the
refusals, and a run of them together.

Tolerances. Cached values are compared exactly: the codes are defined by exact arithmetic. Attention is compared
normwise, |o - o64|_2 <= tol * |o64|_2 over a sequence's rows, where the inputs are N(0, 1) and scale is
1 / sqrt(head_dim), so that scores are of size 1. F32 rows: scores, weights and their sum carry 2^-20 at most each
(22-bit factors, exp and sums in 32 bits), and the weighted values the same: 2^-18 together. F16 and BF16 rows: 11-bit
factors give the scores 2 x 2^-11, the weights 2^-11, the values 2^-11, and the output is rounded once, by 2^-11
or 2^-8: 5 x 2^-11 and 2^-8 + 4 x 2^-11. No single element is off by more than 40 times that times the largest |o64|.
"""
import ctypes as C
import math
import threading

import numpy as np
import pytest

import dotnetfoundryllm_amd as F

pytestmark = pytest.mark.gpu

TYPES = {"f16": F.F16, "q8_0": F.Q8_0, "q4_0": F.Q4_0}
ACTS = {"f32": F.F32, "f16": F.F16, "bf16": F.BF16}


# ---- rows of the three element types on the host ------------------------------------------
def to_bits(x, act):
    x = np.ascontiguousarray(x, dtype=np.float32)
    if act == "f32":
        return x
    if act == "f16":
        return x.astype(np.float16)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bits(b, act):
    if act == "bf16":
        return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return b.astype(np.float64)


def dtype_of(act):
    return {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[act]


# ---- what the pages hold, in 64 bits ---------------------------------------------------
def stored(x, cache):
    """The values that the cache holds of float32 rows [.., head_dim]."""
    x = np.asarray(x, dtype=np.float64)
    if cache == "f16":
        return x.astype(np.float32).astype(np.float16).astype(np.float64)
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    at = np.abs(b).argmax(-1)  # the first of equals
    m = np.take_along_axis(b, at[..., None], -1)
    d = np.abs(m).astype(np.float32) / np.float32(127) if cache == "q8_0" else (m * -0.125).astype(np.float32)
    with np.errstate(over="ignore"):
        d = np.clip(d.astype(np.float16).astype(np.float64), -65504, 65504)
    lo, hi = (-127, 127) if cache == "q8_0" else (-8, 7)
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(d == 0, 0.0, np.clip(np.rint(b / d), lo, hi))
    out = c * d
    out = np.where(np.isfinite(b).all(-1, keepdims=True), out, np.nan)
    return out.reshape(x.shape)


class Setup:
    """Sequences over scattered pages; `garbage` fills the page array first."""

    def __init__(self, ctx, cache, kv, hd, page, new, length, seed=0, layers=2, layer=1, garbage=None, spare=3):
        self.ctx, self.cache, self.kv, self.hd, self.page, self.layer = ctx, cache, kv, hd, page, layer
        self.new, self.length = list(new), list(length)
        self.rng = np.random.default_rng(seed)
        need = [-(-n // page) for n in length]
        n_pages = sum(need) + spare
        order = self.rng.permutation(n_pages).astype(np.int32)
        self.tables = np.full((len(need), max(need + [1])), -7, dtype=np.int32)
        at = 0
        for i, n in enumerate(need):
            self.tables[i, :n] = order[at:at + n]
            at += n
        n_bytes = F.PagedKvCache.bytes_for(TYPES[cache], layers, kv, hd, page, n_pages)
        self.mem = F.DeviceBuffer(ctx, n_bytes)
        fill = self.rng.integers(0, 256, n_bytes, dtype=np.uint8) if garbage is None else np.full(n_bytes, garbage, np.uint8)
        self.mem.write(fill)
        self.pages = F.PagedKvCache(ctx, TYPES[cache], layers, kv, hd, page, n_pages, memory=self.mem)
        self.bufs = []

    def put(self, x, act, pad=0):
        """Host rows as device rows, `pad` elements between them."""
        b = to_bits(x, act)
        wide = np.zeros((b.shape[0] + 2, b.shape[1] + pad), dtype=b.dtype)
        wide[:b.shape[0], :b.shape[1]] = b
        wide.view(np.uint8)[b.shape[0]:] = 0xAB
        buf = F.DeviceBuffer(self.ctx, wide.nbytes)
        buf.write(wide)
        self.bufs.append(buf)
        r = F.Rows(buf, wide.shape[1], ACTS[act])
        r.host = (wide, b.shape[0], b.shape[1])
        return r

    def get(self, r, act):
        wide, n, w = r.host
        back = r.buf.read(wide.nbytes, dtype_of(act)).reshape(wide.shape)
        assert np.array_equal(back[n:].view(np.uint8), wide[n:].view(np.uint8)), "rows behind the last one were written"
        assert np.array_equal(back[:, w:].view(np.uint8), wide[:, w:].view(np.uint8)), "columns behind the rows were written"
        return from_bits(back[:n, :w], act)

    def batch(self, heads, window=F.NO_WINDOW, new=None, length=None):
        b = self.pages.batch(heads, window)
        b.set(self.new if new is None else new, self.length if length is None else length, self.tables)
        self.bufs.append(b)
        return b

    def fill(self, scale_k=1.0, scale_v=1.0):
        """Every position gets rows through append; what the cache holds of them, per sequence [len][kv][hd]."""
        w, n = self.kv * self.hd, sum(self.length)
        k, v = (self.rng.standard_normal((n, w)).astype(np.float32) * s for s in (scale_k, scale_v))
        b = self.batch(self.kv, new=self.length)
        b.append(self.layer, self.put(k, "f32"), self.put(v, "f32"))
        cut = np.cumsum([0] + self.length)
        part = lambda x: [stored(x[a:z], self.cache).reshape(-1, self.kv, self.hd) for a, z in zip(cut, cut[1:])]  # noqa: E731
        return part(k), part(v)

    def close(self):
        for b in self.bufs + [self.pages, self.mem]:
            b.close()


@pytest.fixture
def make(ctx):
    made = []

    def f(*a, **k):
        made.append(Setup(ctx, *a, **k))
        return made[-1]

    yield f
    for s in made:
        s.close()


def attend(q, k, v, group, pos0, window, scale, softcap):
    """64-bit attention of q [n][heads][hd] at positions pos0.. over k, v [len][kv][hd]."""
    n, heads, _ = q.shape
    o = np.zeros_like(q)
    j = np.arange(k.shape[0])
    for i in range(n):
        p = pos0 + i
        see = (j <= p) & (j > p - window)
        for h in range(heads):
            s = k[see, h // group] @ q[i, h] * scale
            if softcap > 0:
                s = softcap * np.tanh(s / softcap)
            e = np.exp(s - s.max())
            o[i, h] = (e / e.sum()) @ v[see, h // group]
    return o


# ---- rows into and out of the pages -----------------------------------------------------------
@pytest.mark.parametrize("cache", TYPES)
@pytest.mark.parametrize("act,kv,hd,page,new,length", [
    ("f32", 2, 64, 16, [1], [1]),
    ("f32", 8, 128, 64, [1, 1, 1], [64, 65, 1]),
    ("bf16", 1, 32, 16, [5, 0, 40], [17, 20, 40]),
    ("f16", 4, 96, 32, [33, 7], [95, 7]),
    ("f32", 3, 256, 128, [130, 1, 126], [257, 128, 255]),
    ("f32", 2, 160, 64, [0, 0], [0, 9]),
])
def test_append_and_read(make, cache, act, kv, hd, page, new, length):
    s = make(cache, kv, hd, page, new, length, seed=hd + page)
    k0, v0 = s.fill()
    b = s.batch(kv)
    w, n = kv * hd, sum(new)
    x = [s.rng.standard_normal((n, w)).astype(np.float32) * 10.0 ** s.rng.uniform(-3, 2, (n, 1)).astype(np.float32) for _ in (0, 1)]
    x = [from_bits(to_bits(a, act), act).astype(np.float32) for a in x]
    b.append(s.layer, s.put(x[0], act, 16), s.put(x[1], act, 8))
    want_new = [stored(a, cache) for a in x]
    out = [s.put(np.zeros((n, w)), "f32", 4) for _ in (0, 1)]
    b.read(s.layer, *out, new_only=True)
    s.ctx.sync()
    for r, want in zip(out, want_new):
        assert np.array_equal(s.get(r, "f32"), want)
    # all positions: the earlier rows are still there, the new ones stand at their places
    every = [s.put(np.zeros((sum(length), w)), a, 8) for a in ("f32", "f16")]
    b.read(s.layer, *every)
    s.ctx.sync()
    at = np.cumsum([0] + new)
    for r, old, fresh, a in zip(every, (k0, v0), want_new, ("f32", "f16")):
        rows = [np.concatenate([o.reshape(-1, w)[:ln - nn], fresh[lo:hi]]) for o, ln, nn, lo, hi in zip(old, length, new, at, at[1:])]
        want = np.concatenate(rows)
        assert np.array_equal(s.get(r, a), from_bits(to_bits(want, a), a))


@pytest.mark.parametrize("cache", TYPES)
def test_append_leaves_the_rest_of_the_pages(make, cache):
    s = make(cache, 2, 64, 32, [3, 4], [35, 20], layers=3, layer=1)
    before = s.mem.read(s.mem.n, np.uint8)
    b = s.batch(2)
    x = s.rng.standard_normal((7, 128)).astype(np.float32)
    b.append(1, s.put(x, "f32"), s.put(x, "f32"))
    s.ctx.sync()
    after = s.mem.read(s.mem.n, np.uint8)
    shape = (3, 2, -1, 2, F.PagedKvCache.bytes_for(TYPES[cache], 1, 1, 64, 32, 1) // 2)
    differ = (before != after).reshape(shape)
    assert not differ[0].any() and not differ[2].any()
    touched = {s.tables[0, 1], s.tables[1, 0]}
    for page in range(differ.shape[2]):
        assert differ[1, :, page].any() == (page in touched)
    # 7 rows: every byte of their codes and scales and no other may have changed
    assert differ.sum() <= 2 * 2 * 7 * F.type_bytes(TYPES[cache], 64)


@pytest.mark.parametrize("cache", ["q8_0", "q4_0"])
def test_append_at_the_borders_of_codes_and_scales(make, cache):
    """Quotients on and next to half steps, zeros, equal magnitudes of both signs, the smallest and the largest scales,
    and values that are no numbers."""
    rows = []
    for d in (1.0, 0.5, 2.0 ** -14, 2.0 ** -24, 3 * 2.0 ** -24, 0.0999755859375, 1000.0, 65504.0):
        d = float(np.float16(d))
        top = 127 * d if cache == "q8_0" else -8 * d
        half = (np.arange(31) - 15.5 if cache == "q8_0" else np.arange(31) / 2 - 7.5) * d
        for step in (0, 1, -1):
            x = half.astype(np.float32)
            for _ in range(abs(step)):
                x = np.nextafter(x, np.float32(step * np.inf))
            rows.append(np.concatenate([[np.float32(top)], x]))
    rows += [np.zeros(32), np.full(32, 1e-30), np.full(32, 3e38), np.tile([1.0, -1.0], 16), np.tile([-7.0, 7.0], 16),
             np.full(32, -2.0 ** -25), np.linspace(-1, 1, 32)]
    bad = []
    for v in (np.nan, np.inf, -np.inf):
        r = np.linspace(-1, 1, 32)
        r[13] = v
        bad.append(r)
    x = np.concatenate([np.stack(rows + bad).astype(np.float32)] * 2, 1)
    n = x.shape[0]
    s = make(cache, 1, 64, 16, [n], [n + 3])
    b = s.batch(1)
    b.append(1, s.put(x, "f32"), s.put(x, "f32"))
    out = [s.put(np.zeros((n, 64)), "f32") for _ in (0, 1)]
    b.read(1, *out, new_only=True)
    s.ctx.sync()
    want = stored(x, cache)
    for r in out:
        assert np.array_equal(s.get(r, "f32"), want, equal_nan=True)


# ---- attention --------------------------------------------------------------------------------
ATTENTION = [
    # kv, heads, hd, page, new, length, window, softcap
    (1, 1, 32, 16, [1], [1], None, 0.0),
    (8, 32, 128, 64, [1], [519], None, 0.0),
    (4, 28, 128, 64, [1, 1, 1], [1, 700, 64], None, 0.0),
    (2, 12, 128, 32, [1, 1], [2500, 33], None, 30.0),
    (8, 16, 256, 16, [1, 1], [300, 17], 64, 50.0),
    (2, 2, 96, 16, [2, 0, 3], [40, 5, 3], None, 0.0),
    (1, 16, 64, 128, [1, 2], [129, 2], None, 0.0),
    (1, 40, 64, 32, [1, 3], [200, 3], 7, 0.0),
    (2, 8, 128, 32, [5, 4, 1], [900, 70, 64], None, 0.0),
    (4, 28, 128, 32, [8], [1030], None, 0.0),
    (1, 4, 160, 64, [9, 33], [100, 33], 1, 0.0),
    (2, 8, 64, 16, [70], [70], None, 0.0),
    (1, 4, 128, 64, [200, 1, 37], [333, 90, 37], None, 0.0),
    (2, 4, 256, 64, [130], [391], 100, 50.0),
    (1, 7, 224, 128, [65, 129], [65, 300], 33, 0.0),
]


@pytest.mark.parametrize("cache", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: "-".join(map(str, c[:4] + (max(c[4]), max(c[5])))))
def test_attention(make, cache, act, case):
    kv, heads, hd, page, new, length, window, softcap = case
    s = make(cache, kv, hd, page, new, length, seed=heads + hd, garbage=0x7F)  # leftovers: half-precision NaNs
    k, v = s.fill()
    win = window or F.NO_WINDOW
    b = s.batch(heads, win)
    n, scale = sum(new), 1.0 / math.sqrt(hd)
    q = from_bits(to_bits(s.rng.standard_normal((n, heads * hd)), act), act)
    out = s.put(np.zeros((n, heads * hd)), act, 16)
    b.attention(s.layer, s.put(q, act, 8), out, scale, softcap)
    s.ctx.sync()
    got = s.get(out, act)
    at = np.cumsum([0] + new)
    for i, (lo, hi) in enumerate(zip(at, at[1:])):
        if lo == hi:
            continue
        qi = q[lo:hi].reshape(-1, heads, hd)
        want = attend(qi, k[i], v[i], heads // kv, length[i] - new[i], win, scale, softcap)
        tol = {"f32": 2.0 ** -18, "f16": 5 * 2.0 ** -11, "bf16": 2.0 ** -8 + 4 * 2.0 ** -11}[act]
        off = got[lo:hi].reshape(want.shape) - want
        assert np.linalg.norm(off) <= tol * np.linalg.norm(want)
        assert np.abs(off).max() <= 40 * tol * np.abs(want).max()


# ---- drafted tokens ----------------------------------------------------------------------------
def verify(target, draft, tokens, counts, ua, us):
    """The rule in 64 bits."""
    n, nd = tokens.shape
    out, kept = np.full((n, nd + 1), -1, np.int32), np.zeros(n, np.int32)
    v = target.shape[-1]
    num = lambda w: np.where(w > 0, w, 0.0)  # noqa: E731
    for i in range(n):
        c, most = 0, min(max(int(counts[i]), 0), nd)
        while c < most:
            t = tokens[i, c]
            if not 0 <= t < v:
                break
            if not float(ua[i, c]) * (1.0 if draft is None else float(draft[i, c, t])) < float(target[i, c, t]):
                break
            out[i, c] = t
            c += 1
        w = target[i, c].astype(np.float64)
        if c < most:
            if draft is None:
                less = np.zeros(v)
                if 0 <= tokens[i, c] < v:
                    less[tokens[i, c]] = 1.0
            else:
                less = draft[i, c].astype(np.float64)
            if num(w - less).sum() > 0:
                w = w - less
        w = num(w)
        run = np.cumsum(w)
        hit = np.flatnonzero((run > float(us[i]) * run[-1]) & (w > 0))
        out[i, c] = hit[0] if hit.size else v - 1
        kept[i] = c
    return out, kept


def run_verify(ctx, target, draft, tokens, counts, ua, us, ld=None, skew=0):
    n, nd = tokens.shape
    v = target.shape[-1]
    ld = ld or v
    bufs = []

    def put(x, dtype):
        x = np.ascontiguousarray(x, dtype=dtype)
        b = F.DeviceBuffer(ctx, max(x.nbytes, 4))
        if x.nbytes:
            b.write(x)
        bufs.append(b)
        return b

    def rows(x):
        wide = np.full((x.shape[0] * x.shape[1], ld), np.nan, np.float32)
        wide[:, :v] = x.reshape(-1, v)
        return F.Rows(put(np.concatenate([np.full(skew, np.nan, np.float32), wide.reshape(-1)]), np.float32), ld, F.F32, 4 * skew)

    out, kept = put(np.full((n, nd + 1), 77), np.int32), put(np.full(n, 77), np.int32)
    F.draft_verify(ctx, n, nd, v, rows(target), put(tokens, np.int32), put(ua, np.float32), put(us, np.float32), out, kept,
                   draft=None if draft is None else rows(draft), counts=None if counts is None else put(counts, np.int32))
    ctx.sync()
    got = out.read(4 * n * (nd + 1), np.int32).reshape(n, nd + 1), kept.read(4 * n, np.int32)
    for b in bufs:
        b.close()
    return got


@pytest.mark.parametrize("n,nd,v,greedy,ld,skew", [
    (1, 4, 128256, False, 0, 0), (3, 1, 1, False, 0, 0), (5, 8, 5, False, 9, 1), (40, 5, 1000, True, 0, 2),
    (7, 3, 4097, False, 4099, 3), (2, 0, 333, False, 0, 0), (130, 2, 64, False, 0, 0), (2, 6, 152064, True, 152065, 1),
    (1, 1, 1 << 20, False, 0, 0), (12, 1, 70001, False, 0, 1), (1, 70, 40, False, 0, 0), (3, 130, 9, True, 0, 0),
])
def test_draft_verify(ctx, n, nd, v, greedy, ld, skew):
    rng = np.random.default_rng(v + n)
    logit = rng.standard_normal((n, nd + 1, v)) * 2
    soft = lambda x: (np.exp(x - x.max(-1, keepdims=True)) / np.exp(x - x.max(-1, keepdims=True)).sum(-1, keepdims=True)).astype(np.float32)  # noqa: E731
    target = soft(logit)
    near = soft(logit[:, :nd] + 0.5 * rng.standard_normal((n, nd, v)))
    target[rng.random(target.shape) < 0.2] = 0  # as top-p leaves zeros
    draft = None if greedy else near
    tokens = near.argmax(-1) if greedy else (near.astype(np.float64).cumsum(-1) < rng.random((n, nd, 1))).sum(-1).clip(0, v - 1)
    counts = rng.integers(0, nd + 1, n)
    counts[0] = nd
    ua, us = rng.random((n, nd), dtype=np.float32), rng.random(n, dtype=np.float32)
    got = run_verify(ctx, target, draft, tokens, counts, ua, us, ld, skew)
    want = verify(target, draft, tokens, counts, ua, us)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_draft_verify_at_the_edges(ctx):
    v, nd = 300, 2
    p = np.zeros((8, nd + 1, v), np.float32)
    q = np.zeros((8, nd, v), np.float32)
    tok, ua, us = np.full((8, nd), 7), np.full((8, nd), 0.5, np.float32), np.zeros(8, np.float32)
    counts = np.full(8, nd)
    p[0, :, 7], q[0, :, 7] = 1, 1                       # the same distribution: all kept
    p[1, :, 9], q[1, :, 7] = 1, 1                       # nothing in common: refused at once, 9 drawn
    p[2, :, 7], q[2, :, 7], ua[2] = 0.5, 1, 0.5         # u q == p is refused
    p[3, :, 20:30], q[3, :, 20:30], us[3] = 0.1, 0.1, 1 - 2.0 ** -24  # token of no weight, nothing left: target itself
    tok[4, 0], p[4, :, 11], q[4, :, 11] = v, 1, 0.5     # an id behind the vocabulary
    tok[5, 1], p[5, :, 7], q[5, :, 7] = -3, 1, 1        # one before it
    p[6] = 0                                            # no weight at all
    p[7, :, ::2], p[7, 0, 4], p[7, 0, 6], counts[7] = 0.01, np.nan, -1, -5  # what is no weight; a negative count
    us[7] = 0.02
    got = run_verify(ctx, p, q, tok, counts, ua, us)
    want = verify(p, q, tok, counts, ua, us)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    assert list(got[1]) == [2, 0, 0, 0, 0, 1, 0, 0]
    assert got[0][1, 0] == 9 and got[0][6, 0] == v - 1
    got = run_verify(ctx, p, None, tok, None, ua, us)
    want = verify(p, None, tok, np.full(8, nd), ua, us)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


# ---- refusals -----------------------------------------------------------------------------------
def test_pages_and_batches_refuse(ctx):
    for bad in [(F.Q4_K, 1, 1, 64, 16, 4)]:
        with pytest.raises(F.NotSupportedException):
            F.PagedKvCache(ctx, *bad)
    for bad in [(F.F16, 1, 1, 48, 16, 4), (F.F16, 1, 1, 288, 16, 4), (F.F16, 1, 1, 64, 24, 4), (F.F16, 0, 1, 64, 16, 4),
                (F.F16, 1, 1, 64, 16, 0)]:
        with pytest.raises(F.ArgumentException):
            F.PagedKvCache(ctx, *bad)
    small = F.DeviceBuffer(ctx, 1024)
    with pytest.raises(F.ArgumentException):
        F.PagedKvCache(ctx, F.F16, 1, 1, 64, 16, 4, memory=small)
    with pytest.raises(F.ArgumentNullException):
        F.DeviceBuffer.wrap(ctx, None, 16)
    p = F.PagedKvCache(ctx, F.Q8_0, 2, 2, 64, 16, 4)
    with pytest.raises(F.ArgumentException):
        p.batch(3)
    with pytest.raises(F.ArgumentOutOfRangeException):
        p.batch(4, 0)
    b = p.batch(4, 20)
    for new, length, table, err in [
            ([2], [1], [[0]], F.ArgumentOutOfRangeException), ([-1], [1], [[0]], F.ArgumentOutOfRangeException),
            ([1], [17], [[0]], F.ArgumentException), ([1], [17], [[0, 4]], F.ArgumentOutOfRangeException),
            ([1], [17], [[-1, 1]], F.ArgumentOutOfRangeException), ([1, 1], [3, 3], [[2], [2]], F.ArgumentException),
            ([1, 0], [17, 5], [[0, 1], [1, 0]], F.ArgumentException), ([17], [32], [[3, 3]], F.ArgumentException)]:
        with pytest.raises(err):
            b.set(new, length, table)
    b.set([1, 1], [17, 18], [[0, 1], [0, 2]])  # a shared page that is only read
    b.set([1], [60], [[-1, -1, 2, 3]])         # pages before the window given back
    rows = F.DeviceBuffer(ctx, 60 * 128 * 4)
    ok = F.Rows(rows, 128)
    with pytest.raises(F.InvalidOperationException):
        b.read(0, ok)
    b.read(0, ok, new_only=True)
    with pytest.raises(F.ArgumentOutOfRangeException):
        b.append(2, ok, ok)
    with pytest.raises(F.ArgumentOutOfRangeException):
        b.append(-1, ok, ok)
    with pytest.raises(F.ArgumentNullException):
        b.read(0)
    for bad in (F.Rows(rows, 64), F.Rows(rows, 130), F.Rows(rows, 128, F.F32, 8), F.Rows(rows, 128, F.F32, 60 * 512 - 256)):
        with pytest.raises(F.ArgumentException):
            b.append(0, ok, bad)
    with pytest.raises(F.NotSupportedException):
        b.append(0, F.Rows(rows, 128, F.Q8_0), ok)
    q, out = F.Rows(rows, 256), F.Rows(rows, 256, F.F32, 4096)
    b.attention(0, q, out, 0.1)
    with pytest.raises(F.ArgumentException):
        b.attention(0, q, q, 0.1)
    for scale, cap in ((math.nan, 0.0), (math.inf, 0.0), (1.0, -1.0), (1.0, math.inf)):
        with pytest.raises(F.ArgumentOutOfRangeException):
            b.attention(0, q, out, scale, cap)
    other = F.Context(0)
    theirs = F.DeviceBuffer(other, 4096)
    with pytest.raises(F.ArgumentException):
        b.append(0, F.Rows(theirs, 128), ok)
    with pytest.raises(F.ArgumentException):
        F.PagedKvCache(ctx, F.F16, 1, 1, 32, 16, 1, memory=theirs)
    theirs.close()
    other.close()
    # a refused set leaves an empty batch: calls do nothing
    with pytest.raises(F.ArgumentOutOfRangeException):
        b.set([1], [1], [[9]])
    rows.write(np.full(60 * 128, 3.0, np.float32))
    b.attention(0, q, out, 0.1)
    b.read(0, ok)
    ctx.sync()
    assert (rows.read(60 * 128 * 4) == 3.0).all()
    b.set([], [], np.zeros((0, 0)))
    b.append(0, ok, ok)
    p.close()
    with pytest.raises(F.ObjectDisposedException):
        b.append(0, ok, ok)
    with pytest.raises(F.ObjectDisposedException):
        b.set([1], [1], [[0]])
    b.close()
    with pytest.raises(F.ObjectDisposedException):
        b.append(0, ok, ok)
    for x in (rows, small):
        x.close()


def test_draft_verify_refuses(ctx):
    b = F.DeviceBuffer(ctx, 4 * 64)
    r = F.Rows(b, 8)
    ok = dict(target=r, tokens=b, u_accept=b, u_sample=b, out_tokens=b, out_counts=b)
    for n, nd, v, more, err in [
            (-1, 1, 8, {}, F.ArgumentOutOfRangeException), (1, -1, 8, {}, F.ArgumentOutOfRangeException),
            (1, 1, 0, {}, F.ArgumentOutOfRangeException), (1, 1, 9, {}, F.ArgumentException), (5, 1, 8, {}, F.ArgumentException),
            (1, 1, 8, {"draft": F.Rows(b, 4)}, F.ArgumentException), (1, 1, 8, {"tokens": None}, F.ArgumentNullException),
            (1, 1, 8, {"target": F.Rows(b, 8, F.F16)}, F.NotSupportedException), (1, 1, (1 << 20) + 1, {}, F.NotSupportedException),
            (1, 1, 8, {"target": F.Rows(b, 8, F.F32, 2)}, F.ArgumentException)]:
        with pytest.raises(err):
            F.draft_verify(ctx, n, nd, v, **{**ok, **more})
    tiny = F.DeviceBuffer(ctx, 4)
    with pytest.raises(F.ArgumentException):
        F.draft_verify(ctx, 1, 1, 8, **{**ok, "out_tokens": tiny})
    F.draft_verify(ctx, 0, 1, 8, **ok)
    ids, kept = F.DeviceBuffer(ctx, 64), F.DeviceBuffer(ctx, 64)
    b.write(np.zeros(64, np.float32))
    for same in ({"out_tokens": b}, {"out_counts": b}, {"out_counts": ids}):  # outputs that are read or written elsewhere too
        with pytest.raises(F.ArgumentException):
            F.draft_verify(ctx, 1, 1, 8, **{**ok, "out_tokens": ids, "out_counts": kept, **same})
    F.draft_verify(ctx, 1, 1, 8, **{**ok, "out_tokens": ids, "out_counts": kept})
    ctx.sync()
    assert list(ids.read(8, np.int32)) == [7, -1] and list(kept.read(4, np.int32)) == [0]
    for x in (b, tiny, ids, kept):
        x.close()


@pytest.mark.parametrize("cache", TYPES)
def test_operands_that_are_columns_of_one_matrix(make, cache):
    """q, k and v, the rows read back and the outputs as columns of one matrix; what shares memory is refused."""
    kv, heads, hd = 2, 4, 64
    s = make(cache, kv, hd, 32, [3, 50], [40, 50], seed=11)
    k, v = s.fill()
    b, w, wq, n = s.batch(heads), kv * hd, heads * hd, 53
    ld = 2 * (w + wq)
    x = s.rng.standard_normal((n, ld)).astype(np.float32)
    buf = F.DeviceBuffer(s.ctx, x.nbytes)
    s.bufs.append(buf)
    buf.write(x)
    part = lambda at: F.Rows(buf, ld, F.F32, 4 * at)  # noqa: E731
    b.append(1, part(wq), part(wq + w))
    b.attention(1, part(0), part(wq + 2 * w), 0.125)
    b.read(1, part(wq), part(wq + w), new_only=True)
    s.ctx.sync()
    got = buf.read(x.nbytes).reshape(n, ld)
    assert np.array_equal(got[:, :wq], x[:, :wq])
    fresh = [stored(x[:, a:a + w].reshape(n, kv, hd), cache) for a in (wq, wq + w)]
    for a, f in zip((wq, wq + w), fresh):
        assert np.array_equal(got[:, a:a + w], f.reshape(n, w).astype(np.float32))
    for lo, hi, i, pos0 in ((0, 3, 0, 37), (3, 53, 1, 0)):
        ki, vi = (np.concatenate([old[i][:pos0], f[lo:hi]]) for old, f in zip((k, v), fresh))
        want = attend(x[lo:hi, :wq].reshape(-1, heads, hd).astype(np.float64), ki, vi, 2, pos0, F.NO_WINDOW, 0.125, 0.0)
        check(got[lo:hi, wq + 2 * w:].astype(np.float64), want, "f32")
    for at in (0, 4, wq - 4, ld - 4):
        if at + wq <= ld or at == ld - 4:
            with pytest.raises(F.ArgumentException):
                b.attention(1, part(0), part(at), 0.125)
    with pytest.raises(F.ArgumentException):
        b.read(1, part(0), part(w - 4), new_only=True)
    inside = F.Rows(s.mem, wq)
    for call in (lambda: b.append(1, inside, part(0)), lambda: b.append(1, part(0), inside), lambda: b.read(1, inside, None, new_only=True),
                 lambda: b.attention(1, inside, part(0), 1.0), lambda: b.attention(1, part(0), inside, 1.0)):
        with pytest.raises(F.ArgumentException):
            call()


def test_one_long_prompt_among_many_decoding_sequences(make):
    """Sequences of very different lengths in one batch, empty ones among them: rows in, rows out, attention."""
    new = [1, 0, 700, 1, 1, 0, 0, 1] + [1, 0] * 40
    length = [3, 0, 5000, 40, 16, 0, 17, 900] + [5, 0] * 40
    s = make("q8_0", 2, 64, 16, new, length, seed=13)
    k, v = s.fill()
    out = [s.put(np.zeros((sum(length), 128)), "f32") for _ in (0, 1)]
    b = s.batch(4)
    b.read(1, *out)
    fresh = [s.put(np.zeros((sum(new), 128)), "f32") for _ in (0, 1)]
    b.read(1, *fresh, new_only=True)
    s.ctx.sync()
    for x, r, f in zip((k, v), out, fresh):
        assert np.array_equal(s.get(r, "f32"), np.concatenate(x).reshape(-1, 128))
        assert np.array_equal(s.get(f, "f32"), np.concatenate([a[len(a) - n:] for a, n in zip(x, new)]).reshape(-1, 128))
    for got, want in attention_of(s, k, v, 4, batch=b):
        check(got, want, "f32")


def test_a_failed_allocation_is_forgotten(ctx):
    """Memory that cannot be had is refused, and the next calls are not blamed for it."""
    with pytest.raises(F.OutOfMemoryException):
        F.PagedKvCache(ctx, F.F16, 1024, 1024, 256, 128, 1 << 20)  # 2^57 bytes
    with F.PagedKvCache(ctx, F.F16, 1, 1, 32, 16, 2) as p, p.batch(1) as b:
        b.set([1], [1], [[1]])
        x = F.DeviceBuffer(ctx, 128)
        x.write(np.ones(32, np.float32))
        b.append(0, F.Rows(x, 32), F.Rows(x, 32))
        ctx.sync()
        x.close()


def test_closed_buffers_are_refused(ctx):
    mem = F.DeviceBuffer(ctx, F.PagedKvCache.bytes_for(F.F16, 1, 1, 32, 16, 2))
    p, x = F.PagedKvCache(ctx, F.F16, 1, 1, 32, 16, 2, memory=mem), F.DeviceBuffer(ctx, 128)
    b, r = p.batch(1), F.Rows(x, 32)
    b.set([1], [1], [[1]])
    x.close()
    with pytest.raises(F.ArgumentNullException):
        b.append(0, r, r)
    mem.close()
    with pytest.raises(F.ObjectDisposedException):
        b.set([1], [1], [[1]])
    b.close()
    p.close()


def test_batches_reuse_memory_of_destroyed_ones(make):
    """Batches that come and go while calls on them are under way."""
    s = make("f16", 1, 64, 16, [1, 20], [500, 60], seed=12)
    k, v = s.fill()
    q = s.put(s.rng.standard_normal((21, 256)), "f32")
    host = from_bits(q.host[0][:21, :256], "f32")
    outs = [s.put(np.zeros((21, 256)), "f32") for _ in range(30)]
    for i, o in enumerate(outs):
        length = [500 - i, 60 - i]
        b = s.pages.batch(4)
        b.set(s.new, length, s.tables)
        b.attention(1, q, o, 0.125)
        b.close()
    s.ctx.sync()
    for i in (0, 1, 14, 29):
        got = s.get(outs[i], "f32")
        for lo, hi, j in ((0, 1, 0), (1, 21, 1)):
            ln = (500 - i, 60 - i)[j]
            check(got[lo:hi], attend(host[lo:hi].reshape(-1, 4, 64), k[j][:ln], v[j][:ln], 4, ln - (hi - lo), F.NO_WINDOW, 0.125, 0.0), "f32")


def test_wrapped_buffers(ctx):
    """A buffer over part of another one: the same memory; the GEMV's reads past a matrix stay inside."""
    hip = C.CDLL("libamdhip64.so.7")  # the runtime that the library has loaded
    base = C.c_void_p()
    assert hip.hipMalloc(C.byref(base), C.c_size_t(4096)) == 0
    whole = F.DeviceBuffer.wrap(ctx, base.value, 4096)
    whole.write(np.arange(1024, dtype=np.float32))
    w = F.DeviceBuffer.wrap(ctx, base.value + 64, 1024)
    assert np.array_equal(w.read(1024), np.arange(16, 272, dtype=np.float32))
    w.write(np.full(4, 9.0, np.float32), 16)
    assert list(whole.read(24, offset=76)) == [19, 9, 9, 9, 9, 24]
    with pytest.raises(F.ArgumentException):
        F.DeviceBuffer.wrap(ctx, base.value + 4, 16)
    host = np.zeros(64, np.float32)
    with pytest.raises(F.ArgumentException):
        F.DeviceBuffer.wrap(ctx, (host.ctypes.data + 15) // 16 * 16, 16)
    x, y = F.DeviceBuffer(ctx, 128), F.DeviceBuffer(ctx, 128)
    with pytest.raises(F.ArgumentException):  # 8 x 32 floats fill it: nothing behind them
        F.gemv(ctx, F.F32, w, 8, 32, x, y)
    x.write(np.ones(32, np.float32))
    F.gemv(ctx, F.F32, w, 4, 32, x, y)
    ctx.sync()
    assert np.allclose(y.read(16), w.read(512).reshape(4, 32).sum(1))
    for b in (w, whole, x, y):
        b.close()
    assert hip.hipFree(base) == 0


# ---- longer, wider, larger ------------------------------------------------------------------------
def check(got, want, act, more=1.0):
    tol = more * {"f32": 2.0 ** -18, "f16": 5 * 2.0 ** -11, "bf16": 2.0 ** -8 + 4 * 2.0 ** -11}[act]
    off = got.reshape(want.shape) - want
    assert np.linalg.norm(off) <= tol * np.linalg.norm(want)
    assert np.abs(off).max() <= 40 * tol * np.abs(want).max()


def attention_of(s, k, v, heads, act="f32", window=F.NO_WINDOW, scale=None, softcap=0.0, batch=None, new=None, length=None, q=None):
    """One call's rows and what they should be, a sequence each."""
    new, length = new or s.new, length or s.length
    b = batch or s.batch(heads, window, new, length)
    n, hd, scale = sum(new), s.hd, 1.0 / math.sqrt(s.hd) if scale is None else scale
    q = s.rng.standard_normal((n, heads * hd)) if q is None else q
    q = from_bits(to_bits(q, act), act)
    out = s.put(np.zeros((n, heads * hd)), act)
    b.attention(s.layer, s.put(q, act), out, scale, softcap)
    s.ctx.sync()
    got, at = s.get(out, act), np.cumsum([0] + new)
    for i, (lo, hi) in enumerate(zip(at, at[1:])):
        if hi > lo:
            yield got[lo:hi], attend(q[lo:hi].reshape(-1, heads, hd), k[i], v[i], heads // s.kv, length[i] - new[i], window, scale, softcap)


@pytest.mark.parametrize("cache", TYPES)
@pytest.mark.parametrize("kv,heads,hd,page,new,length,window,softcap", [
    (1, 4, 256, 64, [111, 3], [500, 90], None, 0.0),      # wide heads, many rows beside few
    (2, 6, 192, 16, [150], [163], 40, 20.0),              # tiles whose window leaves parts of their steps
    (1, 8, 64, 32, [130, 120], [1000, 120], None, 0.0),   # pages shorter than a step, two sequences
    (1, 4, 128, 128, [97], [9000], None, 0.0),            # few tiles over long keys: cut and joined
    (1, 2, 256, 128, [65], [6000], None, 0.0),
    (1, 1, 128, 64, [1], [70000], None, 0.0),             # one row over very many keys
    (1, 16, 32, 16, [1, 1], [20000, 31], 19990, 0.0),
    (1, 8, 256, 64, [120], [361], 150, 50.0),             # 960 rows and more: a quantised cache's keys turned once
    (1, 9, 192, 16, [101, 2], [130, 77], None, 0.0),
    (2, 20, 128, 128, [100], [700], None, 0.0),
    (1, 12, 96, 32, [80, 77], [80, 400], 99, 0.0),
    (1, 32, 128, 64, [2], [4000], None, 0.0),
])
def test_attention_over_longer_ranges(make, cache, kv, heads, hd, page, new, length, window, softcap):
    for act in ("f32", "bf16"):
        s = make(cache, kv, hd, page, new, length, seed=hd, garbage=0x7F)
        for got, want in attention_of(s, *s.fill(), heads, act, window or F.NO_WINDOW, None, softcap):
            check(got, want, act)


@pytest.mark.parametrize("cache", TYPES)
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("new,length", [([1, 3], [300, 40]), ([140], [150])])
def test_attention_of_other_magnitudes(make, cache, act, new, length):
    """Scores' scales of any sign and zero, values near the ends of half precision, rows of q of any size. The tolerances
    are relative to the outputs; scores stay of size 1."""
    for scale, of_k, of_v, of_q in ((-0.125, 1, 1, 1), (0.0, 1, 1, 1), (0.125, 1, 2.0 ** -18, 1), (0.125, 1, 10000, 1),
                                    (0.125 * 2.0 ** 12, 2.0 ** -12, 1, 1), (0.125 * 2.0 ** -90, 1, 1, 2.0 ** 90),
                                    (0.125 * 2.0 ** 90, 1, 1, 2.0 ** -90), (1.0, 0, 1, 2.0 ** 120)):
        s = make(cache, 2, 64, 32, new, length, seed=5)
        k, v = s.fill(of_k, of_v)
        q = s.rng.standard_normal((sum(new), 6 * 64)) * of_q
        q[0, :64] = 0.0
        for softcap in (0.0, 2.0):
            for got, want in attention_of(s, k, v, 6, act, scale=scale, softcap=softcap, q=q):
                check(got, want, act)


@pytest.mark.parametrize("cache", TYPES)
def test_attention_with_pages_given_back(make, cache):
    """A page before the window may go to another sequence, whose rows then stand in it."""
    s = make(cache, 2, 64, 32, [2, 40], [300, 250], seed=3)
    k, v = s.fill()
    s.tables[0, :5] = -1  # 300 - 2 - 100 + 1 = 199: keys from page 6 on
    s.tables[1, :3] = -1  # 250 - 40 - 100 + 1 = 111
    for got, want in attention_of(s, k, v, 8, window=100):
        check(got, want, "f32")


@pytest.mark.parametrize("cache", TYPES)
def test_attention_over_a_shared_prefix(make, cache):
    s = make(cache, 2, 64, 16, [3, 3, 70], [70, 75, 134], seed=4)
    s.tables[1:, :4] = s.tables[0, :4]
    w = 128
    x = [s.rng.standard_normal((64 + 6 + 11 + 70, w)).astype(np.float32) for _ in (0, 1)]
    b = s.batch(2, new=[0, 0, 0], length=[64, 64, 64])
    b.set([64], [64], s.tables[:1])  # a page that is written belongs to one sequence
    b.append(1, *(s.put(a[:64], "f32") for a in x))
    b.set([6, 11, 70], [70, 75, 134], s.tables)
    b.append(1, *(s.put(a[64:], "f32") for a in x))
    part = [[np.concatenate([a[:64], a[lo:hi]]) for lo, hi in ((64, 70), (70, 81), (81, 151))] for a in x]
    k, v = ([stored(a, cache).reshape(-1, 2, 64) for a in p] for p in part)
    for got, want in attention_of(s, k, v, 4):
        check(got, want, "f32")


@pytest.mark.parametrize("cache,new,length", [("f16", 1, 50), ("q8_0", 1, 50), ("q8_0", 100, 100), ("q4_0", 500, 500)])
def test_attention_of_far_scores(make, cache, new, length):
    """Scores of -1e34 and less are scores: the largest of them has the weight."""
    s = make(cache, 1, 32, 16, [new], [length], seed=9)
    k, v = s.fill()
    down = np.full((length, 32), -1.0, np.float32) * (1 + np.arange(length)[::-1, None] // 16).astype(np.float32)  # -n in page n from the end
    b = s.batch(1, new=[length])
    b.append(1, s.put(down, "f32"), s.put(v[0].reshape(length, 32), "f32"))
    v = [stored(v[0].reshape(length, 32).astype(np.float32), cache).reshape(length, 1, 32)]
    q = np.full((new, 32), 2.0 ** 114)
    for got, want in attention_of(s, [stored(down, cache).reshape(length, 1, 32)], v, 1, scale=1.0, q=q):
        check(got, want, "f32")


@pytest.mark.parametrize("cache", TYPES)
@pytest.mark.parametrize("kv,heads,hd,new", [(2, 8, 64, 5), (1, 2, 128, 100), (1, 12, 128, 100), (1, 10, 256, 100)])
def test_a_key_that_is_no_number_is_its_own_querys_matter(make, cache, kv, heads, hd, new):
    """The last token's key is NaN: the tokens before it do not see it; itself and nobody else gets NaN."""
    s = make(cache, kv, hd, 32, [new], [new + 20], seed=14)
    k, v = s.fill()
    b, n = s.batch(kv), new
    x = [np.concatenate([a[0][20:]]).reshape(n, kv * hd).astype(np.float32) for a in (k, v)]
    x[0][-1, 7] = np.nan
    b.append(1, s.put(x[0], "f32"), s.put(x[1], "f32"))
    k, v = ([np.concatenate([a[0][:20], stored(y, cache).reshape(n, kv, hd)])] for a, y in zip((k, v), x))
    for scale, softcap in ((0.1, 0.0), (0.1, 30.0), (1e10, 1e-30)):
        for got, want in attention_of(s, k, v, heads, scale=scale, softcap=softcap):
            check(got[:-1], want[:-1], "f32")
            group = heads // kv
            assert np.isnan(got[-1].reshape(heads, hd)[:group]).all()


@pytest.mark.parametrize("cache,act", [("f16", "f32"), ("q8_0", "bf16"), ("q4_0", "f32")])
def test_the_same_call_gives_the_same_bits(make, cache, act):
    s = make(cache, 2, 128, 64, [1, 5, 100], [3000, 700, 400], seed=6)
    s.fill()
    b, n = s.batch(8), 106
    q = s.put(s.rng.standard_normal((n, 1024)), act)
    outs = [s.put(np.zeros((n, 1024)), act) for _ in range(6)]
    for o in outs:
        b.attention(1, q, o, 0.1)
    s.ctx.sync()
    for o in outs[1:]:
        assert np.array_equal(s.get(outs[0], act), s.get(o, act))


def test_pages_beyond_four_gigabytes(ctx):
    """Cells and rows whose offsets pass 32 bits: pages at the end of a large array, rows far apart."""
    kv, hd, page, n_pages = 8, 256, 128, 9000
    for cache in ("f16", "q8_0"):
        p = F.PagedKvCache(ctx, TYPES[cache], 1, kv, hd, page, n_pages)
        b = p.batch(kv)
        b.set([150], [150], [[n_pages - 1, n_pages - 2]])
        rng = np.random.default_rng(1)
        x = [rng.standard_normal((150, kv * hd)).astype(np.float32) for _ in (0, 1)]
        ld = 1 << 24
        far = F.DeviceBuffer(ctx, 149 * 4 * ld + 4 * kv * hd)  # 10 GB
        for i, row in enumerate(x[0]):
            far.write(row, 4 * ld * i)
        near = F.DeviceBuffer(ctx, x[1].nbytes)
        near.write(x[1])
        b.append(0, F.Rows(far, ld), F.Rows(near, kv * hd))
        far.write(np.zeros(kv * hd, np.float32), 4 * ld * 140)
        b.read(0, F.Rows(far, ld), F.Rows(near, kv * hd))
        ctx.sync()
        k, v = (stored(a.reshape(150, kv, hd), cache) for a in x)
        assert np.array_equal(far.read(4 * kv * hd, offset=4 * ld * 140), k[140].reshape(-1).astype(np.float32))
        assert np.array_equal(near.read(x[1].nbytes).reshape(150, kv, hd), v.astype(np.float32))
        q = rng.standard_normal((150, kv * hd)).astype(np.float32)
        for i, row in enumerate(q):
            far.write(row, 4 * ld * i)
        for new in (150, 2):  # many rows, few rows
            b.set([new], [150], [[n_pages - 1, n_pages - 2]])
            b.attention(0, F.Rows(far, ld, F.F32, 4 * ld * (150 - new)), F.Rows(near, kv * hd), 1 / 16)
            ctx.sync()
            got = near.read(4 * new * kv * hd).reshape(new, kv, hd).astype(np.float64)
            check(got, attend(q[150 - new:].reshape(new, kv, hd).astype(np.float64), k, v, 1, 150 - new, F.NO_WINDOW, 1 / 16, 0.0), "f32")
        for x in (b, p, far, near):
            x.close()


def test_two_threads_on_one_context(make):
    """Calls of two threads share the context's stream and workspace."""
    s = make("q8_0", 2, 64, 32, [1, 2, 90], [4000, 300, 260], seed=8)
    s.fill()
    sets = [([1, 2, 90], s.batch(8)), ([1, 0, 0], s.batch(8, new=[1, 0, 0])), ([0, 2, 0], s.batch(8, new=[0, 2, 0]))]
    jobs = []
    for new, b in sets:
        q = s.put(s.rng.standard_normal((sum(new), 512)), "f32")
        outs = [s.put(np.zeros((sum(new), 512)), "f32") for _ in range(12)]
        b.attention(1, q, outs[0], 0.1)
        jobs.append((b, q, outs))
    s.ctx.sync()
    failed = []

    def work(b, q, outs):
        try:
            for o in outs[1:]:
                b.attention(1, q, o, 0.1)
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    s.ctx.sync()
    assert not failed
    for _, _, outs in jobs:
        first = s.get(outs[0], "f32")
        assert first.any()
        for o in outs[1:]:
            assert np.array_equal(s.get(o, "f32"), first)


# ---- together ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("cache", TYPES)
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 64)])
def test_serving_with_drafts(ctx, cache, hd, page):
    """Three requests through two layers as a server has them: prompts in, then steps of up to three drafted tokens behind
    the last one, each checked against the target; what was refused is overwritten by the next step. A dense model of the
    same layers in 64 bits, without pages, drafts or steps, gives the same rows."""
    kv, heads, vocab, layers, drafts = 2, 6, 301, 2, 3
    rng = np.random.default_rng(hd)
    lens, n_pages = [37, 5, 70], 60
    tables = rng.permutation(n_pages).astype(np.int32)[:3 * 15].reshape(3, 15)
    w, wq = kv * hd, heads * hd
    embed = rng.standard_normal((layers, 2, vocab, w)).astype(np.float32)   # a token's k and v in each layer
    query = rng.standard_normal((layers, vocab, wq)).astype(np.float32)
    tokens = [list(rng.integers(0, vocab, n)) for n in lens]
    p = F.PagedKvCache(ctx, TYPES[cache], layers, kv, hd, page, n_pages)
    b, bufs = p.batch(heads), []

    def put(x):
        x = np.ascontiguousarray(x)
        buf = F.DeviceBuffer(ctx, max(x.nbytes, 16))
        buf.write(x)
        bufs.append(buf)
        return buf

    def step(new):
        """New tokens of each request through both layers: the rows of the last one."""
        ids = np.concatenate([np.asarray(t, np.int64) for t in new])
        b.set([len(t) for t in new], [len(t) + len(n) for t, n in zip(tokens, new)], tables)
        outs = []
        for layer in range(layers):
            b.append(layer, F.Rows(put(embed[layer, 0, ids]), w), F.Rows(put(embed[layer, 1, ids]), w))
            out = put(np.zeros((len(ids), wq), np.float32))
            b.attention(layer, F.Rows(put(query[layer, ids]), wq), F.Rows(out, wq), 0.1)
            outs.append(out)
        ctx.sync()
        return [o.read(4 * len(ids) * wq).reshape(len(ids), heads, hd).astype(np.float64) for o in outs], [len(t) for t in new]

    def dense(i, layer, ids, pos0):
        k, v = (stored(embed[layer, j, np.asarray(ids)].reshape(-1, kv, hd), cache) for j in (0, 1))
        q = query[layer, np.asarray(ids)[pos0:]].reshape(-1, heads, hd).astype(np.float64)
        return attend(q, k, v, heads // kv, pos0, F.NO_WINDOW, 0.1, 0.0)

    def compare(outs, counts, new):
        at = np.cumsum([0] + counts)
        for layer in range(layers):
            for i in range(3):
                check(outs[layer][at[i]:at[i + 1]], dense(i, layer, tokens[i] + list(new[i]), len(tokens[i])), "f32")

    prompts, tokens = tokens, [[], [], []]
    outs, counts = step(prompts)
    compare(outs, counts, prompts)
    tokens = [list(t) for t in prompts]
    soft = lambda x: (np.exp(x) / np.exp(x).sum(-1, keepdims=True)).astype(np.float32)  # noqa: E731
    lasts = [int(rng.integers(0, vocab)) for _ in range(3)]
    refused = 0
    for _ in range(6):
        n_draft = np.array([drafts, int(rng.integers(0, drafts + 1)), 1])
        q = soft(3 * rng.standard_normal((3, drafts, vocab)))
        t = soft(3 * rng.standard_normal((3, drafts + 1, vocab)))
        t[:, :drafts] = 0.6 * t[:, :drafts] + 0.4 * q
        drafted = np.array([[rng.choice(vocab, p=r.astype(np.float64) / r.sum(dtype=np.float64)) for r in rows] for rows in q])
        new = [[lasts[i]] + list(drafted[i, :n_draft[i]]) for i in range(3)]
        outs, counts = step(new)
        compare(outs, counts, new)
        ua, us = rng.random((3, drafts), dtype=np.float32), rng.random(3, dtype=np.float32)
        ids, kept = put(np.zeros((3, drafts + 1), np.int32)), put(np.zeros(3, np.int32))
        F.draft_verify(ctx, 3, drafts, vocab, F.Rows(put(t.reshape(-1, vocab)), vocab), put(drafted.astype(np.int32)), put(ua), put(us),
                       ids, kept, draft=F.Rows(put(q.reshape(-1, vocab)), vocab), counts=put(n_draft.astype(np.int32)))
        ctx.sync()
        got = ids.read(48, np.int32).reshape(3, drafts + 1), kept.read(12, np.int32)
        want = verify(t, q, drafted, n_draft, ua, us)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        for i in range(3):
            c = got[1][i]
            refused += n_draft[i] - c
            tokens[i] += new[i][:1 + c]
            lasts[i] = int(got[0][i, c])
    assert refused > 0
    b.set([0, 0, 0], [len(t) for t in tokens], tables)
    n = sum(len(t) for t in tokens)
    k, v = put(np.zeros((n, w), np.float32)), put(np.zeros((n, w), np.float32))
    b.read(1, F.Rows(k, w), F.Rows(v, w))
    ctx.sync()
    ids = np.concatenate([np.asarray(t) for t in tokens])
    for j, x in enumerate((k, v)):
        assert np.array_equal(x.read(4 * n * w).reshape(n, kv, hd), stored(embed[1, j, ids].reshape(-1, kv, hd), cache).astype(np.float32))
    for x in bufs + [b, p]:
        x.close()
