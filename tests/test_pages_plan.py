"""CPU tests of the paged cache's planner (csrc/pages_plan.hpp, compiled here by itself): what it refuses, and that
the attention's items cover every row and every key that the row sees once, inside the tables and the partial rows."""
import ctypes as C
import os
import random
import subprocess

import numpy as np
import pytest

import dotnetfoundryllm_amd._native as N

HERE = os.path.dirname(os.path.abspath(__file__))
NO_WINDOW = 0x7FFFFFFF
TILE, SPLIT = (4, 8, 16, 32, 128, 128), (128, 128, 128, 128, 32, 32)  # rows of the item classes, most items of a tile
STEP = 64


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("plan") / "plan.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-o", out,
                    os.path.join(HERE, "pages_plan_shim.cpp")], check=True)
    so = C.CDLL(out)
    so.plan_items.restype = so.plan_part_rows.restype = so.plan_images.restype = C.c_int64
    so.plan_error.restype = C.c_char_p
    return so


def plan(so, new, length, tables, heads=4, kv=2, hd=64, page=16, n_pages=1000, window=NO_WINDOW, cus=256, kind=N.Q8_0):
    i32 = lambda a: np.ascontiguousarray(a, dtype=np.int32)  # noqa: E731
    new, length, tables = i32(new), i32(length), i32(tables)
    p = lambda a: a.ctypes.data_as(C.c_void_p)  # noqa: E731
    d = N.PagesDesc(kind, 1, kv, hd, page, n_pages)
    return so.plan_set(C.byref(d), heads, window, cus, len(new), p(new), p(length), p(tables),
                       C.c_int64(tables.shape[1] if tables.ndim == 2 else 0))


def items(so):
    out = []
    for c in range(len(TILE)):
        n = so.plan_items(c, None)
        a = np.zeros((n, 16), np.int32)
        so.plan_items(c, a.ctypes.data_as(C.c_void_p))
        out.append(a)
    return out


def sizes(so):
    a = np.zeros(8, np.int32)
    so.plan_sizes(a.ctypes.data_as(C.c_void_p))
    return dict(zip(("seqs", "rows", "pos", "pages", "tiles", "first", "max_new", "holes"), a.tolist()))


def test_refusals(lib):
    for new, length, table, more, code in [
            ([2], [1], [[0]], {}, N.E_ARG_RANGE), ([-1], [4], [[0]], {}, N.E_ARG_RANGE), ([0], [-1], [[0]], {}, N.E_ARG_RANGE),
            ([1], [(1 << 30) + 1], [[0]], {}, N.E_ARG_RANGE), ([1], [17], [[0]], {}, N.E_ARG),
            ([1], [17], [[0, 1000]], {}, N.E_ARG_RANGE), ([1], [17], [[-2, 1]], {}, N.E_ARG_RANGE),
            ([1], [17], [[-1, 1]], {}, N.E_ARG_RANGE), ([1], [17], [[-1, 1]], {"window": 2}, N.E_ARG_RANGE),
            ([1], [33], [[0, 1, -1]], {"window": 1}, N.E_ARG_RANGE),
            ([1, 1], [3, 3], [[2], [2]], {}, N.E_ARG), ([1, 0], [17, 5], [[0, 1], [1, 0]], {}, N.E_ARG),
            ([17], [32], [[3, 3]], {}, N.E_ARG), ([1], [32], [[3, 3]], {}, N.E_ARG)]:
        assert plan(lib, new, length, table, **more) == code, (new, length, table, more)
        assert lib.plan_error()
    ok = [([1], [17], [[-1, 1]], {"window": 1}), ([1, 1], [17, 18], [[0, 1], [0, 2]], {}), ([0, 0], [16, 16], [[5], [5]], {}),
          ([0], [0], [[-9]], {}), ([], [], np.zeros((0, 0)), {}), ([1], [16], [[0, -5, 2000]], {})]
    for new, length, table, more in ok:
        assert plan(lib, new, length, table, **more) == 0, (new, length, table, lib.plan_error())
    assert plan(lib, [1], [17], [[-1, 1]], window=1) == 0 and sizes(lib)["holes"] == 1


def test_descriptions(lib):
    n = C.c_uint64()
    desc = lambda *a: lib.plan_desc(C.byref(N.PagesDesc(*a)), C.byref(n))  # noqa: E731
    for kind, cell in ((N.F16, 64 * 128 * 2), (N.Q8_0, 64 * 128 // 32 * 34), (N.Q4_0, 64 * 128 // 32 * 18)):
        assert desc(kind, 3, 8, 128, 64, 10) == 0 and n.value == 3 * 2 * 10 * 8 * cell
    assert desc(N.Q8_0, 1 << 20, 1024, 256, 128, 1 << 30) == N.E_ARG  # beyond 2^63 bytes
    for a in ((N.F32, 1, 1, 64, 16, 1), (N.BF16, 1, 1, 64, 16, 1), (N.Q4_K, 1, 1, 64, 16, 1)):
        assert desc(*a) == N.E_NOT_SUPPORTED
    for a in ((N.F16, 1, 1, 0, 16, 1), (N.F16, 1, 1, 33, 16, 1), (N.F16, 1, 1, 288, 16, 1), (N.F16, 1, 1, 64, 0, 1),
              (N.F16, 1, 1, 64, 256, 1), (N.F16, 0, 1, 64, 16, 1), (N.F16, 1, 0, 64, 16, 1), (N.F16, 1, 1, 64, 16, 0),
              (N.F16, 1, 1025, 64, 16, 1)):
        assert desc(*a) == N.E_ARG


def check(so, new, length, heads, kv, window):
    group = heads // kv
    seen = {}      # (sequence, row) -> ranges
    parts = set()  # partial rows in use
    limit, first = so.plan_part_rows(), np.zeros(len(new) + 1, np.int32)
    so.plan_first(first.ctypes.data_as(C.c_void_p))
    for c, list_ in enumerate(items(so)):
        for seq, row0, nrows, k0, k1, part, split, nsplit, tok0, pos0, ln, table in list_[:, :12].tolist():  # noqa: E741
            assert 0 <= seq < len(new) and 0 <= row0 and 1 <= nrows <= TILE[c] and row0 + nrows <= new[seq] * group
            assert 0 <= k0 < k1 <= length[seq] and k0 % STEP == 0 and 0 <= split < nsplit <= SPLIT[c]
            assert k1 % STEP == 0 or split == nsplit - 1
            assert (tok0, pos0, ln, table) == (sum(new[:seq]), length[seq] - new[seq], length[seq], first[seq])
            for r in range(row0, row0 + nrows):
                seen.setdefault((seq, r), []).append((k0, k1))
            if nsplit > 1:
                rows = range(part + split * nrows, part + (split + 1) * nrows)
                assert rows[-1] < limit and not parts.intersection(rows)
                parts.update(rows)
    assert len(parts) == limit
    # images: every key step of the last class's items has one, made once, in order, for its own sequence
    total = C.c_int64()
    n = so.plan_images(None, C.byref(total))
    a = np.zeros((n, 8), np.int32)
    so.plan_images(a.ctypes.data_as(C.c_void_p), C.byref(total))
    made = {}
    for tab, ln, lo, k0, n, image, _, _ in a.tolist():
        assert n >= 1 and k0 % STEP == 0 and k0 + n * STEP < ln + STEP and 0 <= lo < ln
        for k in range(n):
            assert 0 <= image + k < total.value and image + k not in made
            made[image + k] = (tab, k0 + k * STEP, lo)
    assert len(made) == total.value
    for row in items(so)[-1].tolist():
        seq, row0, k0, k1, image = row[0], row[1], row[3], row[4], row[12]
        for k in range(k0 // STEP, -(-k1 // STEP)):
            tab, at, lo = made[image + k]
            assert (tab, at) == (first[seq], k * STEP)
            assert lo <= max(0, length[seq] - new[seq] + row0 // group - window + 1)
    for i, (n, ln) in enumerate(zip(new, length)):
        for r in range(n * group):
            got = sorted(seen.pop((i, r)))
            p = ln - n + r // group
            assert all(a[1] == b[0] for a, b in zip(got, got[1:]))
            assert got[0][0] <= max(0, p - window + 1) and got[-1][1] >= p + 1
    assert not seen


def test_items_cover_every_row_and_key_once(lib):
    rng = random.Random(5)
    for _ in range(150):
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4, 7, 8, 20])
        page = rng.choice([16, 32, 64, 128])
        window = rng.choice([NO_WINDOW, NO_WINDOW, 1, 63, 64, 65, rng.randint(1, 5000)])
        n = rng.randint(1, 9)
        length = [rng.choice([0, 1, 63, 64, 65, rng.randint(0, 200), rng.randint(0, 9000)]) for _ in range(n)]
        new = [min(ln, rng.choice([0, 1, 1, 1, 2, 5, 16, 33, 200, ln])) for ln in length]
        new = [min(x, 600) for x in new]
        need = [-(-ln // page) for ln in length]
        table = np.full((n, max(need + [1])), -3)
        order = list(range(sum(need)))
        rng.shuffle(order)
        for i, k in enumerate(need):
            table[i, :k] = [order.pop() for _ in range(k)]
        assert plan(lib, new, length, table, heads, kv, rng.choice([64, 256]), page, max(1, sum(need)), window, rng.choice([1, 64, 256]),
                    rng.choice([N.F16, N.Q8_0, N.Q4_0])) == 0
        s = sizes(lib)
        assert (s["rows"], s["pos"], s["pages"], s["max_new"]) == (sum(new), sum(length), sum(need), max(new))
        pages, first, tiles = np.zeros(sum(need), np.int32), np.zeros(n + 1, np.int32), np.zeros((s["tiles"], 4), np.int32)
        for name, a in (("tables", pages), ("first", first), ("tiles", tiles)):
            getattr(lib, "plan_" + name)(a.ctypes.data_as(C.c_void_p))
        assert s["first"] == n + 1 and first.tolist() == np.cumsum([0] + need).tolist()
        assert pages.tolist() == [x for row, k in zip(table, need) for x in row[:k]]
        rows = 0  # the tiles are the new tokens in order, a page each
        tiles = tiles.tolist()
        for i, (x, ln) in enumerate(zip(new, length)):
            at = ln - x
            while at < ln:
                off, m, row, pg = tiles.pop(0)
                assert (off, row, pg) == (at % page, rows, table[i, at // page]) and m == min(page - off, ln - at)
                at, rows = at + m, rows + m
        assert not tiles
        check(lib, new, length, heads, kv, window)


def test_long_sequences(lib):
    n = 1 << 27
    table = np.arange(n // 128, dtype=np.int32)[None]
    assert plan(lib, [1], [n], table, 32, 8, 128, 128, n // 128) == 0
    got = np.concatenate(items(lib))
    assert got[:, 4].max() == n and got[:, 3].min() == 0
    check(lib, [1], [n], 32, 8, NO_WINDOW)
    # rows and positions past 2^31 in all are refused
    assert plan(lib, [1] * 20, [n] * 20, np.repeat(table, 20, 0), 32, 8, 128, 128, n // 128) == N.E_ARG


def test_images(lib):
    """A quantised cache's keys are turned once for sequences of many rows, unless the images would be too large."""
    def images(new, length, kind=N.Q8_0, hd=128, kv=8, window=NO_WINDOW):
        n = -(-length // 128)
        assert plan(lib, [new], [length], np.arange(n, dtype=np.int32)[None], 4 * kv, kv, hd, 128, n, window, kind=kind) == 0
        check(lib, [new], [length], 4 * kv, kv, window)
        total = C.c_int64()
        lib.plan_images(None, C.byref(total))
        return total.value

    assert images(224, 4000) == 0 and images(225, 4000) == 63  # 7 tiles of 128 rows and one more
    assert images(400, 4000, N.F16) == 0
    assert images(300, 4000, window=500) == 63 - (4000 - 300 - 499) // STEP
    per = 128 * STEP * 2 * 2 * 2 * 8  # bytes of a key step
    most = (4 << 30) // per * STEP
    assert images(225, most) == most // STEP and images(225, most + 1) == 0


def test_a_join_is_worth_its_steps(lib):
    """Few rows over a middling length: items of at least sqrt(steps rows / 16) steps once that is 4."""
    def steps(length, heads, kv):
        n = -(-length // 64)
        assert plan(lib, [1], [length], np.arange(n, dtype=np.int32)[None], heads, kv, 128, 64, n) == 0
        check(lib, [1], [length], heads, kv, NO_WINDOW)
        a = np.concatenate(items(lib))
        return max(-(-k1 // STEP) - k0 // STEP for k0, k1 in a[:, 3:5].tolist())

    assert [steps(n, 32, 8) for n in (518, 2048, 4096, 8192)] == [2, 2, 4, 6]
    assert steps(131071, 32, 8) > 8
