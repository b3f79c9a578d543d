"""How paged attention deals its work out, by the kernels' own functions (csrc/paged.cuh) compiled for the host: every key that a token sees is some
run's, once; cut items are finished from the slots that their pieces lie in; nothing in lengths or starts leads out of bounds."""
import ctypes as C
import os
import random
import subprocess

import numpy as np
import pytest

import __graft_entry__ as entry
from helpers import ROOT

# tile rows, units of keys, units worth a run, runs: f32 (8, 32, 64 rows), single tokens, chunks
LAUNCHES = [(8, 5, 1, 296), (32, 5, 1, 592), (64, 5, 1, 444), (8, 6, 1, 1184), (16, 6, 1, 1184), (256, 7, 4, 148)]
EVERY = 0x7fffffff


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    build = entry._load_build_module()
    out = str(tmp_path_factory.mktemp("plan") / "plan.so")
    r = subprocess.run([build._nvcc(), *build.NVCC_FLAGS, "-shared", os.path.join(ROOT, "tests", "paged_plan_host.cu"), "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    lib = C.CDLL(out)
    lib.units.restype, lib.units.argtypes = C.c_longlong, [C.c_int, C.c_longlong, C.c_int, C.c_int, C.c_int]
    return lib


def deal(lib, lens, starts, tokens, width, page_shift, kv_heads, group, above, most, launch, cutting, room=200000):
    tile_rows, key_shift, least, ctas = launch
    lens, rows = np.asarray(lens, np.int32), len(lens)
    starts = None if starts is None else np.asarray(starts, np.int32)
    cut, pieces, status = np.zeros((ctas, 4), np.int32), np.zeros((room, 12), np.int32), np.zeros(1, np.int32)
    at = lambda x: None if x is None else x.ctypes.data_as(C.c_void_p)  # noqa: E731
    n = lib.plan(at(lens), at(starts), rows, tokens, width, page_shift, kv_heads, group, above, most, ctas, tile_rows, key_shift, least, int(cutting), at(cut), at(pieces), room, at(status))
    assert n >= 0
    return pieces[:n], cut, int(status[0])


def test_units_are_the_keys_that_a_tile_of_queries_sees(lib):
    rng = random.Random(2)
    for _ in range(2000):
        base, n, ts, ks = rng.choice([0, 1, 5, 64, 127, 128, rng.randint(0, 70000)]), rng.randint(0, 60), rng.randint(0, 8), rng.choice([5, 6, 7])
        assert lib.units(base, n, ts, ks, 0) == sum(-(-(base + ((i + 1) << ts)) // (1 << ks)) for i in range(n))
        assert lib.units(base, n, ts, ks, 1) == n


def test_rows_of_a_tile_are_tokens_times_heads(lib):
    for group in range(1, 33):
        for row in range(256):
            assert lib.token(group, row) == row // group


@pytest.mark.parametrize("launch", LAUNCHES)
@pytest.mark.parametrize("cutting", [True, False])
def test_every_key_in_sight_is_looked_at_once(lib, launch, cutting):
    rng = random.Random(3)
    tile_rows, key_shift, _, ctas = launch
    for trial in range(60):
        rows = rng.choice([1, 2, 5, 33, 70, 500]) if trial % 4 else rng.randint(380, 800)
        group, kv_heads = rng.choice([g for g in (1, 2, 3, 4, 8, 16, 20, 32) if g <= tile_rows]), rng.randint(1, 8 if rows < 50 else 2)
        above, most = rng.choice([(0, EVERY), (16, EVERY), (0, 16)])
        longest = 4000 if rows < 50 else 300
        lens = [rng.choice([0, 1, 31, 32, 33, 63, 64, 65, 127, 129, rng.randint(0, longest)]) for _ in range(rows)]
        new = [rng.choice([0, 1, 1, min(n, 4), min(n, 5), n // 2, n, n + 3]) for n in lens]
        one_each = rng.random() < 0.2
        if one_each:
            new = [1] * rows
        starts = np.concatenate([[0], np.cumsum(new)])
        tokens = int(starts[-1])
        pieces, cut, status = deal(lib, lens, None if one_each else starts, tokens, 1 + longest // 16 + 1, 4, kv_heads, group, above, most, launch, cutting)
        assert status == 0
        tile = 1 << (tile_rows // group).bit_length() - 1
        asked = {}    # (row, head, tile of queries) -> units looked at
        slots = {}
        for c, row, head, q, k0, k1, kt, first, ntok, lo, hi, slot in pieces.tolist():
            item, base = (row, head, q), lens[row] - new[row]
            assert above < new[row] * group <= most and 0 <= head < kv_heads and 0 <= k0 < k1 <= kt
            assert first == starts[row] + q * tile and ntok == min(tile, new[row] - q * tile) > 0
            last = base + q * tile + ntok   # behind the last key that the item's tokens see
            assert lo == (0 if not cutting else k0 << key_shift) and hi == (last if not cutting else min(last, k1 << key_shift))
            done = asked.setdefault(item, [])
            assert not set(done) & set(range(k0, k1))
            done += range(k0, k1)
            if (k0, k1) != (0, kt):
                assert cutting and slot not in slots
                slots[slot] = item
            if k1 == kt:
                assert not cutting or k1 << key_shift >= max(last, 0)
        want = {(r, h, q) for r in range(rows) if above < new[r] * group <= most for h in range(kv_heads) for q in range(-(-new[r] // tile))}
        assert set(asked) == want
        for (row, head, q), done in asked.items():
            assert sorted(done) == list(range(len(done)))
            keys = lens[row] - new[row] + min((q + 1) * tile, new[row])
            assert not cutting or len(done) << key_shift >= keys
        merged = []
        for c in range(ctas):
            first, ntok, head, to = cut[c].tolist()
            if ntok == 0:
                continue
            item = slots[2 * c + 1]
            assert item[1] == head and first == starts[item[0]] + item[2] * tile and c < to < ctas
            mine = [2 * j + (j == c) for j in range(c, to + 1)]
            assert all(slots[s] == item for s in mine)
            merged += mine
        assert sorted(merged) == sorted(slots)


def test_no_length_or_start_leads_out_of_bounds(lib):
    rng = random.Random(5)
    wild = [-2 ** 31, -1, 0, 1, 3, 17, 64, 2 ** 31 - 1]
    for trial in range(400):
        launch = rng.choice(LAUNCHES)
        rows, tokens, width, shift, group = rng.randint(1, 9), rng.randint(0, 40), rng.randint(1, 5), rng.choice([4, 6]), rng.choice([1, 3, 8])
        starts = [rng.choice(wild + [rng.randint(0, 40)]) for _ in range(rows + 1)] if rng.random() < 0.8 else None
        if starts is None:
            tokens = rows
        lens = [rng.choice(wild + [rng.randint(0, 99)]) for _ in range(rows)]
        pieces, _, status = deal(lib, lens, starts, tokens, width, shift, 2, group, 0, EVERY, launch, True)
        for c, row, head, q, k0, k1, kt, first, ntok, lo, hi, slot in pieces.tolist():
            assert 0 <= row < rows and 0 <= head < 2 and ntok > 0 and 0 <= first and first + ntok <= tokens
            assert 0 <= lo and hi <= width << shift
        fine = all(0 <= n <= width << shift for n in lens) and (starts is None or (0 <= starts[0] and starts[-1] <= tokens and all(a <= b for a, b in zip(starts, starts[1:]))))
        assert (status == 0) == fine


def test_the_longest_rows(lib):
    """2^30 tokens of a row, several of them: units and runs are counted in 64 bits."""
    for launch in LAUNCHES:
        pieces, _, status = deal(lib, [1 << 30] * 6, list(range(7)), 6, 1 << 22, 8, 8, 4, 0, EVERY, launch, True)
        assert status == 0
        seen = {}
        for c, row, head, q, k0, k1, *_ in pieces.tolist():
            seen[row, head] = seen.get((row, head), 0) + k1 - k0
        tile = 1 << (launch[0] // 4).bit_length() - 1   # a unit's keys are counted to the end of a whole tile of tokens: the last unit may hold none
        assert len(seen) == 48 and set(seen.values()) == {-(-((1 << 30) - 1 + tile) // (1 << launch[1]))}
        runs = np.bincount(pieces[:, 0], weights=pieces[:, 5] - pieces[:, 4], minlength=launch[3])
        assert runs.max() - runs.min() <= 1
