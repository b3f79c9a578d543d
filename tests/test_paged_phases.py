"""The barriers of the tensor-memory kernel of paged attention (csrc/attention_paged_tc.cu), restated: a producer of tiles of keys, the issue of the
products and the softmax of two tiles of rows.  A barrier is known by the parity of its phase alone, so a role that comes late or early may take one phase for
another; every order of the roles has to come to the end, and no wait may end in another phase than the one it means."""
import itertools
import random

import pytest

SLOTS = (4, 5, 8)


class Barrier:
    def __init__(self, count):
        self.count = self.left = count
        self.phase = 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.left, self.phase = self.count, self.phase + 1

    def passed(self, meant):
        """What a wait for the end of phase `meant` sees: the parity."""
        return (self.phase & 1) != (meant & 1)


def as_it_is(n, j, first):
    """Whether the producer, having passed its n-th slot, tile j of its piece, waits for the first queries."""
    return n == 2 and j == 1 and first > 1


def at_any_piece(n, j, first):
    return n == 2 and first > 0


LONG = "a row is computed again"


def roles(pieces, slots, waits, cleared="behind scores", again=None):
    """Generators that yield the (barrier, phase) they wait for.  A piece: tiles of keys that either tile of rows looks at, the last of them partial.  The
    softmax clears what lies behind a partial tile's keys in its slot of the ring, `cleared` "behind scores" or "ahead of scores".  `again`: where the first
    tile's softmax stays for as long as it takes, "in its piece" (the first) or "behind all"."""
    full, empty = [Barrier(1) for _ in range(slots)], [Barrier(2) for _ in range(slots)]
    qfull, sfull, sfree, pfull, odone = ([Barrier(1), Barrier(1)] for _ in range(5))

    def producer():
        n = 0
        for piece in pieces:
            for j in range(max(piece)):
                slot = n % slots
                yield empty[slot], n // slots - 1
                n += 1
                if waits(n, j, piece[0]):
                    yield qfull[0], 0
                full[slot].arrive()

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
            tiles = piece[g]
            if tiles:
                yield qfull[g], asked
                asked += 1
                yield from scores(n)
            for j in range(max(piece)):
                if j + 1 < tiles:
                    yield from scores(n + 1)
                if j >= tiles:
                    yield full[n % slots], n // slots
                else:
                    yield pfull[g], done
                    done += 1
                    odone[g].arrive()
                empty[n % slots].arrive()
                n += 1

    def softmax(g):
        scored = n = 0
        for piece in pieces:
            if piece[g]:
                qfull[g].arrive()
            for j in range(piece[g]):
                partial, slot = j == max(piece) - 1, n + j
                if partial and cleared == "ahead of scores":
                    yield full[slot % slots], slot // slots
                yield sfull[g], scored
                if partial and cleared == "behind scores":
                    yield full[slot % slots], slot // slots
                sfree[g].arrive()
                if j:
                    yield odone[g], scored - 1
                pfull[g].arrive()
                scored += 1
            if piece[g]:
                yield odone[g], scored - 1
            n += max(piece)
            if g == 0 and again == "in its piece":
                yield LONG
        if g == 0 and again == "behind all":
            yield LONG

    return [producer(), products(0), products(1), softmax(0), softmax(1)]


class WrongPhase(Exception):
    pass


def comes_to_an_end(pieces, slots, waits, pick, **kw):
    """Runs the roles, `pick` choosing among those that can go on, until all are done (True) or none can."""
    live = {i: (r, None) for i, r in enumerate(roles(pieces, slots, waits, **kw))}
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
            continue
        if live[i][1] == LONG:   # for good, as far as the others' bounded waits go
            del live[i]
    return True


LISTS = [[(1, 1), (1, 1), (2, 2)], [(1, 0)] * 9, [(1, 2), (3, 3)], [(1, 0), (1, 0), (1, 1)], [(0, 1), (1, 1), (1, 1)], [(0, 0), (3, 4), (2, 0)], [(0, 2), (1, 1), (1, 1)], [(7, 9), (7, 9)], [(2, 2)] * 4,
         [(0, 0), (1, 1), (0, 1), (0, 0), (5, 5)], [(2, 0)] * 7 + [(1, 1)], [(0, 3), (0, 3), (0, 5), (1, 1)], [(1, 1), (0, 0), (1, 1), (1, 1)]]


@pytest.mark.parametrize("slots", SLOTS)
def test_every_order_of_the_roles_ends(slots):
    for pieces in LISTS:
        for order in itertools.permutations(range(5)):   # each role as far as it can go before the next one
            assert comes_to_an_end(pieces, slots, as_it_is, lambda ready: min(ready, key=order.index)), (pieces, order)
    rng = random.Random(7)
    for _ in range(400):
        pieces = []
        for _ in range(rng.randint(1, 9)):
            second = rng.choice([0, 1, 1, 2, 3, 9])
            pieces.append((max(0, second - rng.choice([0, 0, 1])) if second else rng.choice([0, 1, 1, 2, 6]), second))
        assert comes_to_an_end(pieces, slots, as_it_is, rng.choice)


def test_a_wait_at_any_piece_would_not():
    """What the condition is for: waited for at whichever piece the second slot is of, the queries' barrier may be two phases on."""
    late = lambda ready: max(ready)  # noqa: E731: the producer goes on only where no other can
    assert not comes_to_an_end([(1, 1), (1, 1), (2, 2)], 4, at_any_piece, late)
    assert not comes_to_an_end([(1, 2), (3, 3)], 4, at_any_piece, late)
    assert comes_to_an_end([(1, 1), (1, 1), (2, 2)], 4, as_it_is, late)


def test_a_slot_cleared_ahead_of_its_scores_would_be_another():
    """The softmax of the second tile passes over pieces without rows of its own; eight slots later a barrier of the ring has the same parity."""
    ahead = lambda ready: max(ready)  # noqa: E731: the softmax of the second tile as far as it can go
    for pieces in ([(2, 0)] * 7 + [(1, 1)], [(4, 0), (4, 0), (1, 1)]):
        with pytest.raises(WrongPhase):
            comes_to_an_end(pieces, 4, as_it_is, ahead, cleared="ahead of scores")
        assert comes_to_an_end(pieces, 4, as_it_is, ahead)


def test_no_role_waits_for_a_row_that_is_computed_again():
    for pieces in LISTS:
        assert comes_to_an_end(pieces, 4, as_it_is, max, again="behind all")
    assert not comes_to_an_end([(2, 2)] * 4, 4, as_it_is, max, again="in its piece")
