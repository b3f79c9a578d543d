"""Paged caches without a GPU: who holds which page, what the entry points refuse, how the attention's work is dealt out, and that
no table, length or start can lead a kernel out of its buffers."""
import ctypes as C
import random

import pytest
import torch

from helpers import pkg


def cache(pages=20, page=16, batch=4, **kw):
    return pkg().PagedKVCache(pages, page, 2, 64, batch, device="cpu", **kw)


def test_pages_are_taken_given_back_and_never_shared():
    c, rng = cache(), random.Random(1)
    for _ in range(300):
        if rng.random() < 0.6:
            rows = rng.sample(range(4), rng.randint(1, 4))
            new = [rng.choice([0, 1, 1, 5, 40]) for _ in rows]
            free = c.free_pages()
            try:
                s = c.step(rows, new)
            except pkg().Ab2Error as e:
                assert e.status == -4 and c.free_pages() == free
                continue
            assert s.tokens == sum(new) and s.lens.tolist() == [c.seq_len(r) + n for r, n in zip(rows, new)]
            assert s.starts.tolist() == [sum(new[:i]) for i in range(len(new) + 1)]
            for i, r in enumerate(rows):
                need = -(-s.lens[i].item() // 16)
                assert s.table[i, :need].tolist() == c._pages[r][:need]
            c.commit(s)
        else:
            r = rng.randrange(4)
            c.truncate(rng.randint(0, c.seq_len(r)), r)
        held = [p for row in c._pages for p in row]
        assert len(held) == len(set(held)) and sorted(held + c._free) == list(range(20))
        for r in range(4):
            assert len(c._pages[r]) * 16 >= c.seq_len(r)
    c.clear()
    assert c.free_pages() == 20


def test_a_step_written_anew_keeps_its_place():
    c = cache()
    s = c.step([0, 2], [10, 1], room=100)
    at = s.packed.data_ptr()
    c.commit(s)
    for _ in range(40):
        again = c.step([0, 2], [1, 1], into=s)
        assert again is s and s.packed.data_ptr() == at and s.tokens == 11 and s.starts.tolist() == [0, 1, 2]
        c.commit(s)
    assert c.seq_len(0) == 50 and c.seq_len(2) == 41
    with pytest.raises(pkg().Ab2Error):
        c.step([0], [1], into=s)
    with pytest.raises(pkg().Ab2Error):
        c.step([0, 2], [60, 1], into=s)
    assert c.seq_len(0) == 50 and c.free_pages() == 20 - 4 - 3


def test_refusals_of_the_cache():
    p = pkg()
    for kw in (dict(page=8), dict(page=24), dict(pages=0), dict(dtype="int8"), dict(batch=0)):
        with pytest.raises(p.Ab2Error):
            cache(**kw)
    c = cache()
    for rows, new in (([4], [1]), ([-1], [1]), ([0, 0], [1, 1]), ([0], [-1]), ([], []), ([0], [1, 2])):
        with pytest.raises(p.Ab2Error):
            c.step(rows, new)
    with pytest.raises(p.Ab2Error):
        c.truncate(1, 0)
    assert c.free_pages() == 20


def test_entry_points_refuse_before_any_device_work():
    """Bad arguments are answered on a machine without a GPU as well."""
    p = pkg()
    lib = p.lib
    good = dict(k_pages=1 << 20, v_pages=1 << 21, table=1 << 22, lens=1 << 23, starts=1 << 24, pages=4, page_size=16, kv_heads=2, head_dim=64, table_width=3, rows=2, tokens=5, table_stride=3)

    def paged(**kw):
        return p._lib.Paged(**{**good, **kw})

    def attention(c, q=1 << 25, qs=512, heads=8, out=1 << 26, os=512, max_new=3, dtype=2, work=None):
        return lib.ab2_paged_attention(C.byref(c) if c else None, q, qs, heads, out, os, max_new, 1.0, work, 0, dtype, None)

    assert attention(None) == -7
    for kw, code in ((dict(k_pages=None), -7), (dict(v_pages=None), -7), (dict(table=None), -7), (dict(lens=None), -7), (dict(page_size=24), -8), (dict(page_size=8), -8), (dict(page_size=512), -8),
                     (dict(head_dim=96), -8), (dict(pages=0), -1), (dict(rows=0), -1), (dict(tokens=-1), -1), (dict(table_width=0), -1), (dict(table_stride=2), -1), (dict(kv_heads=0), -1),
                     (dict(starts=None), -1), (dict(k_pages=(1 << 20) + 8), -2), (dict(table_width=(1 << 26) + 1, table_stride=1 << 28), -1)):
        assert attention(paged(**kw)) == code, kw
        assert lib.ab2_paged_append(C.byref(paged(**kw)), 1 << 25, 128, 1 << 26, 128, None, 0, 0, None, 0, None, 0, 0, 1.0, 2, None) == code, kw
    for kw, code in ((dict(q=None), -7), (dict(out=None), -7), (dict(heads=7), -1), (dict(heads=0), -1), (dict(heads=66), -1), (dict(out=1 << 25), -7), (dict(max_new=0), -1), (dict(qs=511), -1), (dict(os=100), -1),
                     (dict(qs=513), -2), (dict(q=(1 << 25) + 2), -2), (dict(dtype=1), -3), (dict(dtype=9), -3), (dict(work=(1 << 25) + 8), -2)):
        assert attention(paged(), **kw) == code, kw
    assert attention(paged(tokens=0)) == 0
    rot = lambda **kw: lib.ab2_rotary_apply(*{**dict(q=1 << 20, qs=256, h=4, k=1 << 21, ks=128, kv=2, d=64, pos=1 << 22, p64=0, n=3, f=1 << 23, rot=64, layout=0, m=1.0,  # noqa: E731
                                                     qo=1 << 24, qos=256, ko=1 << 25, kos=128, dtype=0, s=None), **kw}.values())
    for kw, code in ((dict(q=None), -7), (dict(k=None), -7), (dict(pos=None), -7), (dict(f=None), -7), (dict(qo=None), -7), (dict(layout=2), -7), (dict(rot=65), -1), (dict(rot=66), -1), (dict(rot=-2), -1),
                     (dict(d=63), -1), (dict(n=-1), -1), (dict(h=0, kv=0), -1), (dict(h=-1), -1), (dict(qs=255), -1), (dict(kos=1), -1), (dict(dtype=3), -3), (dict(q=(1 << 20) + 2), -2)):
        assert rot(**kw) == code, kw
    assert rot(n=0) == 0
    adj = lambda **kw: lib.ab2_adjust_logits(*{**dict(z=1 << 20, st=100, rows=2, vocab=100, h=1 << 21, hs=5, hw=5, n=None, r=1 << 22, bi=None, bv=None, nb=0, al=None, out=1 << 23, dtype=0, s=None),  # noqa: E731
                                               **kw}.values())
    for kw, code in ((dict(z=None), -7), (dict(out=None), -7), (dict(h=None), -7), (dict(r=None), -7), (dict(hs=4), -7), (dict(nb=3), -7), (dict(st=99), -1), (dict(vocab=0), -1), (dict(rows=-1), -1),
                     (dict(rows=70000), -1), (dict(hw=-1), -1), (dict(nb=-1), -1), (dict(dtype=5), -3), (dict(out=(1 << 23) + 1), -2)):
        assert adj(**kw) == code, kw
    assert adj(rows=0) == 0


def test_cpu_tensors_are_refused():
    """A kernel given host memory would fault: no operator lets one through, alone or among others."""
    p = pkg()
    d, z = p.dispatch, torch.zeros
    q, pages, i32 = z(2, 2, 64), z(3, 2, 16, 64), lambda *s: z(*s, dtype=torch.int32)  # noqa: E731
    calls = [lambda: d.rotary_apply(q, None, i32(2), z(4, dtype=torch.float64)), lambda: d.rotary_apply(q, q, i32(2), z(4, dtype=torch.float64), out=(q, q)),
             lambda: d.paged_append(pages, pages, q, q, i32(2, 2), i32(2)), lambda: d.paged_append(pages, pages, q, q, i32(2, 2), i32(2), i32(3), q=q, out=q),
             lambda: d.attention_paged(q, pages, pages, i32(2, 2), i32(2), 1.0), lambda: d.attention_paged(q, pages, pages, i32(2, 2), i32(2), 1.0, i32(3), 1, q),
             lambda: d.adjust_logits(z(2, 9)), lambda: d.adjust_logits(z(2, 9), i32(2, 3), i32(2), z(2, 3), i32(2, 1), z(2, 1), i32(2, 1), z(2, 9))]
    for call in calls:
        with pytest.raises(p.Ab2Error) as e:
            call()
        assert e.value.status == -7 and "CUDA device" in str(e.value)


# -- how the attention's work is dealt out: the arithmetic of paged.cuh, restated -----------------------

def bounded(starts, lens, b, tokens, capacity):
    s0, s1 = (starts[b], starts[b + 1]) if starts else (b, b + 1)
    first = min(max(s0, 0), tokens)
    return first, min(max(s1, first), tokens) - first, min(max(lens[b], 0), capacity)


def units(base, n, ts, ks, whole):
    """paged_units: its closed forms."""
    if whole:
        return n
    s = ks - ts
    if s <= 0:
        return n * ((base + (1 << ks) - 1) >> ks) + ((n * (n + 1) // 2) << -s)
    c = ((base + (1 << ts) - 1) >> ts) + (1 << s)
    floors = lambda y: (((y >> s) * ((y >> s) - 1) // 2) << s) + (y >> s) * (y & ((1 << s) - 1))  # noqa: E731
    return floors(c + n) - floors(c)


def test_units_are_the_keys_that_a_tile_of_queries_sees():
    rng = random.Random(2)
    for _ in range(2000):
        base, n, ts, ks = rng.choice([0, 1, 5, 64, 127, 128, rng.randint(0, 70000)]), rng.randint(0, 60), rng.randint(0, 8), rng.choice([5, 6, 7])
        assert units(base, n, ts, ks, False) == sum(-(-(base + ((i + 1) << ts)) // (1 << ks)) for i in range(n))


@pytest.mark.parametrize("whole", [False, True])
def test_every_unit_of_work_is_done_once_and_cut_items_are_finished(whole):
    rng = random.Random(3)
    for trial in range(400):
        rows, kv_heads, most_ctas, group = rng.randint(1, 9), rng.randint(1, 4), rng.choice([2, 7, 296]), rng.choice([1, 3, 4, 8])
        ts, ks, least = rng.choice([(0, 6, 1), (1, 6, 2), (3, 6, 1), (6, 7, 4), (8, 7, 4)])
        above, most = rng.choice([(0, 2 ** 31 - 1), (32, 2 ** 31 - 1), (0, 32)])
        least = 1 if whole else least
        lens = [rng.choice([0, 1, 63, 64, 65, 500, 4000]) for _ in range(rows)]
        new = [rng.choice([0, 1, min(2, n), n // 2, n]) if n else 0 for n in lens]
        tiles = [-(-c // (1 << ts)) if above < c * group <= most else 0 for c in new]
        per = [units(n - c, q, ts, ks, whole) for n, c, q in zip(lens, new, tiles)]
        total = kv_heads * sum(per)
        ctas = max(1, min(most_ctas, total // least))
        begin = [total * min(c, ctas) // ctas for c in range(most_ctas + 1)]
        done, slots, merged = {}, {}, []
        for c in range(most_ctas):
            u, last = begin[c], None
            if u < begin[c + 1]:   # where the run begins
                before, row = 0, 0
                while u >= before + per[row] * kv_heads:
                    before += per[row] * kv_heads
                    row += 1
                head, at = divmod(u - before, per[row])
                lo, hi = 0, tiles[row] - 1
                while lo < hi:
                    mid = (lo + hi + 1) // 2
                    lo, hi = (mid, hi) if units(lens[row] - new[row], mid, ts, ks, whole) <= at else (lo, mid - 1)
                k = at - units(lens[row] - new[row], lo, ts, ks, whole)
                keys = lambda: 1 if whole else (lens[row] - new[row] + ((lo + 1) << ts) + (1 << ks) - 1) >> ks  # noqa: E731
                kt = keys()
            while u < begin[c + 1]:
                if k == kt:   # the next item
                    k, lo = 0, lo + 1
                    if lo == tiles[row]:
                        lo, head = 0, head + 1
                        if head == kv_heads:
                            head, row = 0, row + 1
                            while tiles[row] == 0:
                                row += 1
                    kt = keys()
                k0, k1 = k, min(kt, k + begin[c + 1] - u)
                assert head < kv_heads and lo << ts < new[row] and 0 <= k0 < k1 <= kt
                for i in range(k0, k1):
                    assert done.setdefault((row, head, lo, i), c) == c
                if (k0, k1) != (0, kt):
                    assert not whole
                    slot = 2 * c + (k0 == 0)
                    assert slot not in slots
                    slots[slot] = (row, head, lo)
                u += k1 - k0
                k = k1
                last = (row, head, lo, k0, k1, kt, u + kt - k1)
            if last and last[3] == 0 and last[4] < last[5]:
                assert c < most_ctas - 1
                to = min(ctas - 1, (last[6] * ctas - 1) // total)
                assert begin[to] < last[6] <= begin[to + 1]
                merged.append((last[:3], [2 * j + (j == c) for j in range(c, to + 1)]))
        assert len(done) == total
        assert sorted(s for _, m in merged for s in m) == sorted(slots)
        assert all(slots[s] == item for item, m in merged for s in m)
        want = {(r, h, i, k) for r in range(rows) for h in range(kv_heads) for i in range(tiles[r])
                for k in range(1 if whole else -(-(lens[r] - new[r] + ((i + 1) << ts)) // (1 << ks)))}
        assert want == set(done)


def test_no_table_length_or_start_leads_out_of_the_buffers():
    rng = random.Random(5)
    wild = [-2 ** 31, -1, 0, 1, 3, 17, 64, 2 ** 31 - 1]
    for _ in range(3000):
        rows, tokens, width, shift = rng.randint(1, 5), rng.randint(0, 40), rng.randint(1, 5), rng.choice([4, 6])
        starts = [rng.choice(wild + [rng.randint(0, 40)]) for _ in range(rows + 1)] if rng.random() < 0.8 else None
        if not starts:
            tokens = rows
        lens = [rng.choice(wild + [rng.randint(0, 99)]) for _ in range(rows)]
        for b in range(rows):
            first, count, length = bounded(starts, lens, b, tokens, width << shift)
            assert 0 <= first and count >= 0 and first + count <= tokens and 0 <= length <= width << shift
            for i in range(count):   # a token's last key, when it sees any, lies in the table
                pos = length - count + i
                assert pos < length and (pos < 0 or pos >> shift < width)
        for t in range(tokens):   # the row that the append finds for a token
            row = sum(s <= t for s in starts[1:]) if starts else t
            if row < rows:
                first, count, length = bounded(starts, lens, row, tokens, width << shift)
                pos = length - (first + count) + t
                if first <= t < first + count and pos >= 0:
                    assert pos >> shift < width
