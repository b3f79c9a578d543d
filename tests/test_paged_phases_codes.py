"""The barriers of the tensor-memory kernel over pages of 8 bits, restated: a producer of codes (values, then keys), the warps that make values f16 in the ring's slots, and
the issue of the products and the softmax of two tiles of rows as over bf16 (``test_paged_phases``)."""
import itertools
import random

import pytest

from test_paged_phases import LISTS, Barrier, WrongPhase

WARPS = 4


def roles(pieces, slots, raws):
    full, empty = [Barrier(1 + WARPS) for _ in range(slots)], [Barrier(2) for _ in range(slots)]
    rfull, rempty = [Barrier(1) for _ in range(raws)], [Barrier(WARPS) for _ in range(raws)]
    qfull, sfull, sfree, pfull, odone = ([Barrier(1), Barrier(1)] for _ in range(5))
    tiles = sum(max(p) for p in pieces)

    def producer():
        for n in range(tiles + 1):   # the last is the end
            yield rempty[n % raws], n // raws - 1
            rfull[n % raws].arrive()
            if n < tiles:
                yield empty[n % slots], n // slots - 1
                full[n % slots].arrive()

    def values():
        for n in range(tiles + 1):
            yield rfull[n % raws], n // raws
            if n < tiles:
                yield empty[n % slots], n // slots - 1
                full[n % slots].arrive()
                rempty[n % raws].arrive()

    def products(g):
        n = scored = done = asked = 0

        def scores(n):
            nonlocal scored
            yield full[n % slots], n // slots
            if scored:
                yield sfree[g], scored - 1
            sfull[g].arrive()
            scored += 1
        for piece in pieces:
            if piece[g]:
                yield qfull[g], asked
                asked += 1
                yield from scores(n)
            for j in range(max(piece)):
                if j + 1 < piece[g]:
                    yield from scores(n + 1)
                if j >= piece[g]:
                    yield full[n % slots], n // slots
                else:
                    yield pfull[g], done
                    done += 1
                    odone[g].arrive()
                empty[n % slots].arrive()
                n += 1

    def softmax(g):
        scored = 0
        for piece in pieces:
            if piece[g]:
                qfull[g].arrive()
            for j in range(piece[g]):
                yield sfull[g], scored
                sfree[g].arrive()
                if j:
                    yield odone[g], scored - 1
                pfull[g].arrive()
                scored += 1
            if piece[g]:
                yield odone[g], scored - 1

    return [producer(), *(values() for _ in range(WARPS)), products(0), products(1), softmax(0), softmax(1)]


def comes_to_an_end(pieces, slots, raws, pick):
    live = {i: (r, None) for i, r in enumerate(roles(pieces, slots, raws))}
    while live:
        ready = [i for i, (_, w) in live.items() if w is None or w[0].passed(w[1])]
        if not ready:
            return False
        i = pick(ready)
        if live[i][1] and live[i][1][0].phase != live[i][1][1] + 1:
            raise WrongPhase(pieces)
        try:
            live[i] = live[i][0], next(live[i][0])
        except StopIteration:
            del live[i]
    return True


@pytest.mark.parametrize("slots,raws", [(4, 2), (8, 2), (3, 3)])
def test_every_order_of_the_roles_ends(slots, raws):
    rng = random.Random(7)
    orders = list(itertools.permutations(range(9)))
    for pieces in LISTS:
        for order in rng.sample(orders, 40):   # each role as far as it can go before the next one
            assert comes_to_an_end(pieces, slots, raws, lambda ready: min(ready, key=order.index)), (pieces, order)
    for _ in range(300):
        pieces = []
        for _ in range(rng.randint(1, 9)):
            second = rng.choice([0, 1, 1, 2, 3, 9])
            pieces.append((max(0, second - rng.choice([0, 0, 1])) if second else rng.choice([0, 1, 1, 2, 6]), second))
        assert comes_to_an_end(pieces, slots, raws, rng.choice)
