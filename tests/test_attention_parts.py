"""How attention's work is cut, in the arithmetic of lt_attention.hip and lt_attention_wide.hip, on the CPU: every block
once, places of parts that no two parts share, and as many as the workspace has."""
import math
import random

import numpy as np
import pytest

JOIN = 16


def thin_splits(blocks, share, least):
    if blocks <= 3 * least:
        return 1
    n = blocks // share if share > least else -(-blocks // share)
    return min(max(n, 1), JOIN * JOIN - 1)


@pytest.mark.parametrize("target,least", [(512, 8), (256, 8), (256, 4)])
def test_few_row_parts_fit_grid_and_workspace(target, least):
    r = random.Random(target + least)
    for _ in range(400):
        heads = r.choice([1, 2, 3, 4, 8, 17, 64, 256])
        top = r.choice([4, 30, 100, 5000, 200000])
        rows = [(r.randint(0, 32), r.randint(1, top)) for _ in range(r.choice([1, 1, 3, 64, 300]))]
        width = max(b for _, b in rows) + r.randint(0, 9)
        total = sum(t * b for t, b in rows)
        share = max(least, math.ceil(total * heads / target))
        splits = [thin_splits(b, share, least) for _, b in rows]
        slots = 2 * (target // heads + 1) + 2
        assert sum(t * s for (t, _), s in zip(rows, splits) if s > 1) <= slots
        tiles = sum(t for t, _ in rows)
        grid = min(tiles + target // heads + 1, tiles * -(-width // least))
        assert sum(t * s for (t, _), s in zip(rows, splits)) <= max(grid, 0)
        assert 2 * slots * heads <= 8192  # counters
        for (_, b), s in zip(rows, splits):
            cuts = [b * i // s for i in range(s + 1)]
            assert cuts[0] == 0 and cuts[-1] == b and all(x < y for x, y in zip(cuts, cuts[1:]))
            for hands in (1, 2, 4, 32):
                each = s if s <= JOIN or s <= 8 * hands else math.ceil(math.sqrt(s))
                groups = -(-s // each)
                assert each * groups >= s and (groups == 1 or groups <= JOIN and each <= JOIN)


def test_tokens_of_rows_by_a_product():
    f = np.float32
    for group in range(1, 600):
        rows = np.arange(512 + 16)
        assert np.array_equal(((rows.astype(f) + f(0.5)) * (f(1) / f(group))).astype(np.uint32), rows // group)


def test_many_row_pieces_cover_every_tile_once():
    r = random.Random(5)
    for _ in range(100):
        heads, fit = r.choice([1, 2, 4, 8]), r.choice([256, 512, 768])
        tiles = [r.randint(1, r.choice([2, 40, 3000])) for _ in range(r.choice([1, 2, 9, 100, 400]))]
        line = sum(tiles)
        total = line * heads
        pieces = max(1, min(fit, total // 8))
        seen, places, counters = {}, {}, set()
        order = [i % 8 * (pieces // 8) + i // 8 if pieces == fit and pieces % 8 == 0 else i for i in range(fit)]
        assert sorted(p for p in order if p < pieces) == list(range(pieces))
        firsts = [sum(tiles[:i]) for i in range(len(tiles))]
        for piece in range(pieces):
            u, u1 = total * piece // pieces, total * (piece + 1) // pieces
            while u < u1:
                h, at = divmod(u, line)
                t = max(i for i, f in enumerate(firsts) if f <= at)
                first = h * line + firsts[t]
                end = first + tiles[t]
                nxt = min(end, u1)
                seen[h, t] = seen.get((h, t), 0) + nxt - u
                if u != first or nxt != end:
                    f, g = first * pieces // total, (end - 1) * pieces // total
                    while f + 1 < pieces and total * (f + 1) // pieces <= first:
                        f += 1
                    while g + 1 < pieces and total * (g + 1) // pieces <= end - 1:
                        g += 1
                    assert f <= piece <= g
                    place = 2 * piece + (piece == f)
                    assert place not in places and place < 2 * fit
                    places[place] = (h, t)
                    parts = g - f + 1
                    groups = -(-parts // JOIN)
                    each = -(-parts // groups)
                    assert each <= JOIN and -(-parts // each) <= groups
                    counters.add((2 * fit + f, h, t))
                u = nxt
        assert all(seen[h, t] == b for h in range(heads) for t, b in enumerate(tiles))
        assert len({c for c, _, _ in counters}) == len(counters)  # a tile that is cut has a counter of its own
        assert all(c < 3 * fit <= 8192 for c, _, _ in counters)
