"""How paged attention through a window deals its work out, by the kernels' own functions (csrc/paged.cuh) compiled for the host: every key that a token sees is some
run's, once; units that no token of a tile sees are left out; no page that may be gone is asked for; nothing in lengths or starts leads out of bounds."""
import ctypes as C
import os
import random
import subprocess

import numpy as np
import pytest

import __graft_entry__ as entry
from helpers import ROOT

# tile rows, units of keys, units worth a run, runs: f32 (8, 32, 64 rows), single tokens, chunks
LAUNCHES = [(8, 5, 1, 40), (32, 5, 1, 60), (64, 5, 1, 30), (16, 6, 1, 100), (256, 7, 4, 20)]
MOST = 1 << 30   # keys that a window may have, and first keys
WILD = [-2 ** 31, -1, 0, 1, 3, 17, 64, 2 ** 31 - 1]


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    build = entry._load_build_module()
    out = str(tmp_path_factory.mktemp("plan") / "plan.so")
    r = subprocess.run([build._nvcc(), *build.NVCC_FLAGS, "-shared", os.path.join(ROOT, "tests", "paged_window_host.cu"), "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    lib = C.CDLL(out)
    lib.units.restype, lib.units.argtypes = C.c_longlong, [C.c_int, C.c_longlong, C.c_int, C.c_int, C.c_int, C.c_int, C.POINTER(C.c_longlong)]
    return lib


def deal(lib, lens, starts, tokens, width, page_shift, kv_heads, group, launch, cutting, window, sinks, room=20000):
    tile_rows, key_shift, least, ctas = launch
    lens = np.asarray(lens, np.int32)
    starts = None if starts is None else np.asarray(starts, np.int32)
    pieces, status = np.zeros((room, 12), np.int32), np.zeros(1, np.int32)
    at = lambda x: None if x is None else x.ctypes.data_as(C.c_void_p)  # noqa: E731
    n = lib.plan(at(lens), at(starts), len(lens), tokens, width, page_shift, kv_heads, group, ctas, tile_rows, key_shift, least, int(cutting), window, sinks, at(pieces), room, at(status))
    assert n >= 0
    return pieces[:n], int(status[0])


def test_units_of_tiles_add_up(lib):
    rng = random.Random(2)
    for _ in range(4000):
        base, n, ts, ks = rng.choice([-300, -17, -1, 0, 1, 5, 64, 127, 128, rng.randint(0, 70000)]), rng.randint(0, 60), rng.randint(0, 8), rng.choice([5, 6, 7])
        window, sinks, by_tile = rng.choice([1, 2, 31, 64, 128, 129, 1000, rng.randint(1, 5000), MOST]), rng.choice([0, 1, 4, 64, 65, rng.randint(0, 600), MOST]), C.c_longlong()
        assert lib.units(base, n, ts, ks, window, sinks, by_tile) == by_tile.value


@pytest.mark.parametrize("launch", LAUNCHES)
@pytest.mark.parametrize("cutting", [True, False])
def test_every_key_in_sight_is_looked_at_once(lib, launch, cutting):
    rng = random.Random(3)
    tile_rows, key_shift, _, ctas = launch
    unit = 1 << key_shift
    for trial in range(60):
        rows, kv_heads = rng.choice([1, 2, 5, 20]), rng.randint(1, 3)
        group = rng.choice([g for g in (1, 2, 3, 4, 8, 16) if g <= tile_rows])
        window, sinks = rng.choice([1, 2, 31, 32, 64, 100, 128, 129, rng.randint(1, 600), MOST]), rng.choice([0, 0, 1, 4, unit, unit + 1, rng.randint(0, 300), MOST])
        lens = [rng.choice([0, 1, 31, 32, 33, 64, 65, 127, 129, rng.randint(0, 1500)]) for _ in range(rows)]
        new = [rng.choice([0, 1, 1, min(n, 4), min(n, 5), n // 2, n, n + 3, n + rng.randint(0, 700)]) for n in lens]
        starts = np.concatenate([[0], np.cumsum(new)])
        pieces, status = deal(lib, lens, starts, int(starts[-1]), 100, 4, kv_heads, group, launch, cutting, window, sinks)
        assert status == 0
        tile = 1 << (tile_rows // group).bit_length() - 1
        seen, units = {}, {}
        for c, row, head, t0, ntok, lo, hi, gap, jump, k0, k1, kt in pieces.tolist():
            virtual = np.arange(lo, max(lo, hi))
            keys = np.where(virtual >= jump, virtual + gap, virtual)
            assert (keys >= 0).all() and (keys < max(lens[row], 1)).all() or lens[row] == 0 and not len(keys)
            for t in range(t0, t0 + ntok):
                pos = lens[row] - new[row] + t
                mine = keys[(keys <= pos) & ((keys < sinks) | (keys > pos - window))]
                seen.setdefault((row, head, t), []).extend(mine.tolist())
            units[row, head, t0] = kt
            assert not (k0 and not cutting)
            first = lens[row] - new[row] + t0   # position of the tile's first token
            for page in {int(k) // 16 for k in keys}:
                held = range(16 * page, 16 * page + 16)
                assert lib.hidden(lens[row] - new[row], t0, window, sinks, 16 * page, 16) == all(sinks <= k <= first - window for k in held)
        for row in range(rows):
            for t in range(new[row]):
                pos = lens[row] - new[row] + t
                want = [k for k in range(pos + 1) if k < sinks or k > pos - window]
                for head in range(kv_heads):
                    assert sorted(seen[row, head, t]) == want, (row, t)
        if cutting:   # the units of a tile: those that its keys lie in, one more at most on each side of what is left out, and what a whole tile of tokens would see
            for (row, head, t0), kt in units.items():
                base = lens[row] - new[row]
                if base < 0:   # tokens without a place: their keys are counted as those of tokens that have one
                    continue
                assert kt <= -(-(base + t0 + tile) // unit) and kt <= -(-sinks // unit) + -(-(window + tile) // unit) + 1 or window > base + t0 + tile


def test_no_length_or_start_leads_out_of_bounds(lib):
    rng = random.Random(5)
    for trial in range(600):
        launch = rng.choice(LAUNCHES)
        rows, tokens, width, shift, group = rng.randint(1, 9), rng.randint(0, 40), rng.randint(1, 5), rng.choice([4, 6]), rng.choice([1, 3, 8])
        starts = [rng.choice(WILD + [rng.randint(0, 40)]) for _ in range(rows + 1)] if rng.random() < 0.8 else None
        if starts is None:
            tokens = rows
        lens = [rng.choice(WILD + [rng.randint(0, 99)]) for _ in range(rows)]
        window, sinks = rng.choice([1, 7, 64, MOST]), rng.choice([0, 1, 70, MOST])
        pieces, status = deal(lib, lens, starts, tokens, width, shift, 2, group, launch, True, window, sinks)
        for c, row, head, t0, ntok, lo, hi, gap, jump, *_ in pieces.tolist():
            assert 0 <= row < rows and 0 <= head < 2 and ntok > 0 and 0 <= t0 and t0 + ntok <= tokens
            assert 0 <= lo and gap >= 0 and (hi <= lo or hi + (gap if hi > jump else 0) <= width << shift)


def test_the_longest_rows(lib):
    """2^30 tokens of a row: through a window of 1000 each takes the units of the sinks and of the window, at keys far behind."""
    for launch in LAUNCHES:
        unit, tile = 1 << launch[1], 1 << (launch[0] // 4).bit_length() - 1
        pieces, status = deal(lib, [(1 << 30) - 1] * 6, list(range(7)), 6, 1 << 22, 8, 8, 4, launch, True, 1000, 5)
        assert status == 0
        seen = {}
        for c, row, head, t0, ntok, lo, hi, gap, jump, *_ in pieces.tolist():
            virtual = np.arange(lo, hi)
            keys = np.where(virtual >= jump, virtual.astype(np.int64) + gap, virtual)
            seen.setdefault((row, head), []).extend(keys[(keys < 5) | (keys > (1 << 30) - 2 - 1000)].tolist())
        assert len(seen) == 48 and all(sorted(k) == [*range(5), *range((1 << 30) - 1001, (1 << 30) - 1)] for k in seen.values())
        assert sum(p[10] - p[9] for p in pieces.tolist()) <= 48 * (1 + -(-(1000 + tile) // unit) + 1)
