"""Turns of two query tiles with the exponentials: a model of the waits of prompt attention, whose barriers are counted as the kernels
count them (host arithmetic, no GPU).  Every actor is a warp's role; a pass in which none can go on is a kernel that would wait forever."""

import random

import pytest

from nkipy_b200.ops import _lib


class Barrier:
    def __init__(self, count=1):
        self.count, self.left, self.phase = count, count, 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.left, self.phase = self.count, self.phase + 1

    def passed(self, parity):
        return self.phase & 1 != parity & 1


def runs(actors, rng):
    """Whether all actors (generators of (barrier, parity) to wait for) come to their end, in a random order."""
    waits = {a: None for a in actors}
    while waits:
        went = False
        for a in rng.sample(list(waits), len(waits)):
            w = waits[a]
            while w is None or w[0].passed(w[1]):
                went = True
                w = next(a, False)
                if w is False:
                    del waits[a]
                    break
                waits[a] = w
                if rng.random() < 0.3:
                    break
        if not went:
            return False
    return True


def bars(n, count=1):
    return [Barrier(count) for _ in range(n)]


def first_visible(pos, window, chunk):
    lo = pos - window + 1 if window > 0 and pos >= window else 0
    return max(lo, pos - pos % chunk) if chunk > 0 and pos >= 0 else lo


def tiles_of(row0, all_rows, group, q_len, ctx, causal, window, chunk, tile):
    """Key tiles [lo, hi) of 128 rows from row0 on, and how many rows there are."""
    if row0 >= all_rows:
        return 0, 0, 0
    rows = min(128, all_rows - row0)
    first, last = ctx - q_len + row0 // group, ctx - q_len + (row0 + rows - 1) // group
    hi = -(-max(ctx, 0) // tile)
    if causal:
        hi = min(hi, max(last + tile, 0) // tile)
    lo = first_visible(first, window, chunk) // tile
    return lo, max(hi, lo), rows


def by_key_tile(t0, t1):
    """attn_prefill.cu's rule, as it is compiled: key tile -> turn, or -1."""
    lib = _lib.lib()
    b = t1[:2] if t1[2] else (0, 0)
    return lambda t, at: lib.nkb_query_turn(t, t0[0], t0[1], *b, at)


def from_the_first(t0, t1):
    """attn_q8_prefill.cu's."""
    n = _lib.lib().nkb_query_turns_from_first(*t0[:2], *t1[:2]) if t1[2] else 0
    return lambda t, at: at - (t0, t1)[t][0] if at - (t0, t1)[t][0] < n else -1


def by_own_count(t0, t1):
    """Counted from each query tile's own first key tile, which chunks part."""
    n = min(t0[1] - t0[0], t1[1] - t1[0]) if t1[2] else 0
    return lambda t, at: at - (t0, t1)[t][0] if at - (t0, t1)[t][0] < n else -1


def pages16(t0, t1, stages, kept, rule):
    """attn_prefill.cu: one pair of query tiles, behind `kept` key tiles that both see."""
    two = t1[2] > 0
    u_lo = t0[0]
    n = kept + (max(t0[1], t1[1]) if two else t0[1]) - u_lo
    kv_full, kv_empty = bars(stages), bars(stages, 2 if two else 1)
    s_full, s_empty, p_full, o_full, turn = (bars(2) for _ in range(5))
    rule = rule(t0, t1)

    def load():
        for i in range(2 * n):
            yield kv_empty[i % stages], i // stages + 1
            kv_full[i % stages].arrive()

    def issue(t):
        a_lo, a_hi = (kept + (t0, t1)[t][j] - u_lo for j in (0, 1))
        item = 0
        for is_v, x in order(n):
            yield kv_full[item % stages], item // stages
            if x < kept or a_lo <= x < a_hi:
                own = x if x < kept else x - a_lo + kept
                if is_v:
                    yield p_full[t], own
                    o_full[t].arrive()
                else:
                    yield s_empty[t], own + 1
                    s_full[t].arrive()
            kv_empty[item % stages].arrive()
            item += 1

    def softmax(t):
        lo, hi, _ = (t0, t1)[t]
        for it in range(kept + hi - lo):
            yield s_full[t], it
            s_empty[t].arrive()
            if it:
                yield o_full[t], it - 1
            if it < kept:
                at = it if two else -1
            else:
                at = rule(t, lo + it - kept)
                at += kept if at >= 0 else 0
            if at >= 1 - t:
                yield turn[t], at - 1 + t
            if at >= 0:
                turn[1 - t].arrive()
            p_full[t].arrive()
        if kept + hi - lo:
            yield o_full[t], kept + hi - lo - 1

    return [load(), issue(0), softmax(0)] + ([issue(1), softmax(1)] if two else [])


def order(n):
    """Ring items: K(0), then K(u + 1), V(u)."""
    items = [(False, 0)] if n else []
    for u in range(n):
        items += ([(False, u + 1)] if u + 1 < n else []) + [(True, u)]
    return items


def pages8(works, stages, rule):
    """attn_q8_prefill.cu: the works of a CTA, each the ranges of two query tiles, the first key tile of the walk and how many there are."""
    kWorks, kSlots, kLead = 3, 8, 4
    raw_full, raw_empty, kv_full = (bars(stages) for _ in range(3))
    kv_empty, e_full, e_empty = bars(stages, 2), bars(kSlots), bars(kSlots)
    s_full, s_empty, p_full, o_full, o_empty, q_full, turn = (bars(2) for _ in range(7))
    w_full, w_empty = bars(kWorks), bars(kWorks, 6)
    ring = [None] * kWorks
    u_lo, union = (lambda w: w[2]), (lambda w: w[3])                         # noqa: E731

    def fetch():
        item = 0
        for n, w in enumerate(works + [None]):
            yield w_empty[n % kWorks], n // kWorks + 1
            ring[n % kWorks] = w
            w_full[n % kWorks].arrive()
            for _ in range(2 * union(w) if w else 0):
                yield raw_empty[item % stages], item // stages + 1
                raw_full[item % stages].arrive()
                item += 1

    def works_of(step):
        """A reader's works, one behind another; step(w): what it does with one."""
        n = 0
        while True:
            yield w_full[n % kWorks], n // kWorks
            w = ring[n % kWorks]
            w_empty[n % kWorks].arrive()
            n += 1
            if w is None:
                return
            yield from step(w)

    def scales():
        tiles = 0

        def one(w):
            nonlocal tiles
            for _ in range(union(w)):
                if tiles >= kLead:
                    yield e_empty[(tiles - kLead) % kSlots], (tiles - kLead) // kSlots
                e_full[tiles % kSlots].arrive()
                tiles += 1
        return works_of(one)

    def convert():
        item = tiles = 0

        def one(w):
            nonlocal item, tiles
            for is_v, x in order(union(w)):
                st, slot = item % stages, (tiles + x) % kSlots
                if not is_v:
                    yield e_full[slot], (tiles + x) // kSlots
                yield raw_full[st], item // stages
                yield kv_empty[st], item // stages + 1
                kv_full[st].arrive()
                raw_empty[st].arrive()
                if is_v:
                    e_empty[slot].arrive()
                item += 1
            tiles += union(w)
        return works_of(one)

    def issue(t):
        item = tiles = results = 0

        def one(w):
            nonlocal item, tiles, results
            lo, hi = ((w[t][j] - u_lo(w)) for j in (0, 1)) if w[t][1] > w[t][0] else (0, 0)
            if hi > lo:
                yield q_full[t], results
            for is_v, x in order(union(w)):
                yield kv_full[item % stages], item // stages
                if lo <= x < hi:
                    if is_v:
                        if x == lo:
                            yield o_empty[t], results + 1
                        yield p_full[t], tiles + x - lo
                        o_full[t].arrive()
                    else:
                        yield s_empty[t], tiles + x - lo + 1
                        s_full[t].arrive()
                kv_empty[item % stages].arrive()
                item += 1
            tiles += hi - lo
            results += hi > lo
        return works_of(one)

    def softmax(t):
        seen = done = pairs = 0
        cur = None

        def finish():
            nonlocal done, pairs
            if cur is None:
                return
            w, tiles0, at_turn = cur
            lo, hi, _ = w[t]
            if hi > lo:
                yield o_full[t], done + hi - lo - 1
                o_empty[t].arrive()
            done += hi - lo
            pairs += sum(at_turn(t, x) >= 0 for x in range(lo, hi))

        def loop():
            w, tiles0, at_turn = cur
            lo, hi, _ = w[t]
            for it in range(hi - lo):
                x = tiles0 + lo - u_lo(w) + it
                yield e_full[x % kSlots], x // kSlots
                yield s_full[t], done + it
                s_empty[t].arrive()
                if it:
                    yield o_full[t], done + it - 1
                at = at_turn(t, lo + it)
                if at >= 0 and (t == 1 or pairs + at > 0):
                    yield turn[t], pairs + at - (t == 0)
                if at >= 0:
                    turn[1 - t].arrive()
                p_full[t].arrive()

        def one(w):
            """Queries of the next work are taken ahead of the result of the one before."""
            nonlocal seen, cur
            tiles0, seen = seen, seen + union(w)
            if w[t][2] == 0:
                return
            if w[t][1] > w[t][0]:
                q_full[t].arrive()
            yield from finish()
            cur = w, tiles0, rule(w[0], w[1])
            yield from loop()

        yield from works_of(one)
        yield from finish()

    return [fetch(), scales(), convert(), issue(0), issue(1), softmax(0), softmax(1)]


def random_masks(rng, chunks):
    masks = dict(causal=rng.random() < 0.8, window=0, chunk=0)
    if rng.random() < 0.5:
        masks["window"] = rng.choice([1, 50, 128, 129, 500, 700, 1500])
    if chunks and rng.random() < 0.9:
        masks["chunk"] = rng.choice([70, 128, 200, 300, 511, 512, 700, 1024, 1500, 2048])
    return masks


def random_pairs(rng, chunks, tile, groups):
    """Ranges of the pairs of query tiles of one prompt."""
    q_len, cached = rng.choice([1, 100, 129, 300, 1000, 2000]), rng.choice([0, 1, 100, 200, 333, 1000, 3000])
    group, masks = rng.choice(groups), random_masks(rng, chunks)
    rows = q_len * group
    return [tuple(tiles_of(r, rows, group, q_len, cached + q_len, masks["causal"], masks["window"], masks["chunk"], tile) for r in (row0, row0 + 128))
            for row0 in range(0, rows, 256)]


def parts_of(pair, parts=1):
    """Works of a pair of query tiles, whose walk is divided."""
    t0, t1 = pair
    lo, n = t0[0], (max(t0[1], t1[1]) if t1[2] else t0[1]) - t0[0]
    if n < 4:
        parts = 1
    parts = max(min(parts, n), 1)
    for part in range(parts):
        a, b = (lo + n * (part + i) // parts for i in (0, 1))
        cut = (t if parts == 1 else (max(t[0], a), max(min(t[1], b), t[0], a), t[2]) for t in (t0, t1))
        yield (*cut, a, b - a)


@pytest.mark.parametrize("chunks", [False, True])
@pytest.mark.parametrize("tile,stages", [(128, 3), (128, 4), (64, 4)])
def test_bf16_pages_come_to_an_end(tile, stages, chunks):
    rng = random.Random(tile + stages + chunks)
    for _ in range(60):
        for t0, t1 in random_pairs(rng, chunks, tile, [1])[:6]:
            kept = rng.choice([0, 0, 1, 2]) if not chunks else 0
            if kept > t0[0]:
                kept = t0[0]
                t1 = (min(t0[0], t1[1]), *t1[1:]) if t1[2] else t1
            assert runs(pages16(t0, t1, stages, kept, by_key_tile), rng), (t0, t1, kept)


@pytest.mark.parametrize("chunks", [False, True])
@pytest.mark.parametrize("stages", [2, 4])
def test_8_bit_pages_come_to_an_end(stages, chunks):
    rng = random.Random(stages + chunks)
    for _ in range(60):
        works = [w for _ in range(rng.choice([1, 3])) for pair in random_pairs(rng, chunks, 128, [1, 2, 4, 5, 16]) for w in parts_of(pair)]
        works = rng.sample(works, min(len(works), 6))
        assert runs(pages8(works, stages, from_the_first), rng), works


def test_the_model_finds_waits_without_an_end():
    """Turns that go by each one's own count: a chunk that begins between the two query tiles' first positions."""
    t0, t1 = (tiles_of(r, 2000, 1, 2000, 2200, True, 0, 512, 128) for r in (256, 384))
    assert (t0, t1) == ((0, 5, 128), (4, 6, 128))
    works = list(parts_of((t0, t1)))
    assert not runs(pages8(works, 2, by_own_count), random.Random(1)) and runs(pages8(works, 2, from_the_first), random.Random(1))
    assert not runs(pages16(t0, t1, 3, 0, by_own_count), random.Random(1)) and runs(pages16(t0, t1, 3, 0, by_key_tile), random.Random(1))


def test_parts_of_a_walk_come_to_an_end():
    """Works that are a part of the key tiles of their rows: one query tile may have none of them."""
    rng = random.Random(9)
    for _ in range(60):
        works = [part for pair in random_pairs(rng, True, 128, [1, 4])[:3] for part in parts_of(pair, rng.choice([1, 2, 5, 16]))]
        assert runs(pages8(works, 2, from_the_first), rng), works
