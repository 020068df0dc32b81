"""The work table of chunk attention over the 8-bit cache: every row's visible blocks belong to one item, once; parts and joins agree."""
import random

import numpy as np
import pytest

from arctic_platform_b200.ops.kv_fp8 import _work

CASES = [([5] * 16, [1500 - 61 * i for i in range(16)], 32, 8), ([512], [16896], 32, 8), ([3000, 1, 17], [4096, 9000, 17], 16, 8),
         ([1], [1], 1, 1), ([1], [0], 4, 2), ([7], [3], 4, 2), ([0, 0], [5, 0], 4, 2), ([16], [36864], 32, 4), ([2000], [2000], 5, 1),
         ([9, 300], [40000, 300], 200, 1), ([3], [700], 256, 2), ([1] * 40, [901] * 40, 8, 1)]


def _random():
    r = random.Random(3)
    for _ in range(60):
        lengths = [r.choice([0, 1, 127, 128, 129, r.randint(0, 30000)]) for _ in range(r.randint(1, 9))]
        yield [r.choice([0, 1, 2, 17, 64, 65, min(n, 2000)]) for n in lengths], lengths, *r.choice([(16, 8), (32, 4), (14, 2), (5, 1), (130, 1)])


@pytest.mark.parametrize("sms", [1, 5, 148])
def test_every_visible_block_once(sms):
    for new, lengths, Hq, H in [*CASES, *_random()]:
        w = _work(np.array(new), np.array(lengths), Hq, H, sms)
        R, starts = Hq // H, np.concatenate([[0], np.cumsum(new)])
        hp = min(R, 128)
        tp = 128 // hp
        ranges, scratch = {}, set()
        for row0, tokens, s, kvh, head0, heads, pos0, length, b0, blocks, part, _ in w.items.tolist():
            assert 0 < tokens <= 2 * tp and starts[s] <= row0 and row0 + tokens <= starts[s + 1]
            assert pos0 == lengths[s] - new[s] + row0 - starts[s] and length == lengths[s]
            assert kvh * R <= head0 and head0 + heads <= (kvh + 1) * R and 0 < heads <= hp
            ranges.setdefault((row0, tokens, head0, heads), []).append((b0, blocks, part, max(0, min(length, pos0 + tokens))))
            for g in range(2 if tokens > tp else 1) if part >= 0 else ():
                assert 0 <= part + g < w.part_tiles and part + g not in scratch
                scratch.add(part + g)
        assert sum(tokens * heads for _, tokens, _, heads in ranges) == sum(new) * Hq
        for pieces in ranges.values():
            pieces.sort()
            at = 0
            for b0, blocks, part, _ in pieces:
                assert b0 == at and (blocks > 0 or len(pieces) == 1) and (part >= 0) == (len(pieces) > 1)
                at += blocks
            assert at == -(-pieces[0][3] // 128)
        assert len(scratch) == w.part_tiles
        joined = [part + k * step for _, _, _, _, part, parts, step, _ in w.joins.tolist() for k in range(parts)]
        assert sorted(joined) == sorted(scratch)
        assert w.one_tile == all(m <= tp for m in new)
        assert w.ctas <= sms and len(w.first) == w.ctas + 1 and (not w.ctas or (w.first[0] == 0 and w.first[-1] == len(w.items)))
        assert (np.diff(w.first) >= 0).all()


def test_shares_of_a_long_conversation_are_even():
    """Blocks of the slowest CTA against the mean of all: fewer items than CTAs would leave some idle."""
    w = _work(np.array([512]), np.array([16896]), 32, 8, 148)
    load = [w.items[a:b, 9].sum() for a, b in zip(w.first, w.first[1:])]
    assert len(load) == 148 and max(load) <= 1.2 * sum(load) / 148


@pytest.mark.parametrize("sms", [2, 5, 148])
def test_pairs_see_every_block_once(sms):
    """Pairs of CTAs take tiles of twice the tokens; the joins leave out tiles that no token fills."""
    seen = 0
    for new, lengths, Hq, H in [*CASES, *_random()]:
        hp = min(Hq // H, 128)
        tp = 128 // hp
        assert (_work(np.array(new), np.array(lengths), Hq, H, sms, 128).form == 1) == all(m <= tp for m in new)
        if all(m <= tp for m in new):
            continue
        w = _work(np.array(new), np.array(lengths), Hq, H, sms, 128, form=2)
        assert w.form == 2
        seen += 1
        assert w.ctas <= sms // 2 and len(w.first) == w.ctas + 1 and w.first[-1] == len(w.items) and (np.diff(w.first) >= 0).all()
        ranges, scratch, filled = {}, set(), set()
        for row0, tokens, s, kvh, head0, heads, pos0, length, b0, blocks, part, _ in w.items.tolist():
            assert 0 < tokens <= 4 * tp
            ranges.setdefault((row0, tokens, head0, heads), []).append((b0, blocks, part, max(0, min(length, pos0 + tokens))))
            for g in range(4 if tokens > 2 * tp else 2) if part >= 0 else ():
                assert part + g < w.part_tiles and part + g not in scratch
                scratch.add(part + g)
                if g * tp < tokens:
                    filled.add(part + g)
        assert sum(tokens * heads for _, tokens, _, heads in ranges) == sum(new) * Hq
        for pieces in ranges.values():
            at = 0
            for b0, blocks, part, _ in sorted(pieces):
                assert b0 == at and (part >= 0) == (len(pieces) > 1)
                at += blocks
            assert at == -(-pieces[0][3] // 128)
        joined = [part + k * step for _, _, _, _, part, parts, step, _ in w.joins.tolist() for k in range(parts)]
        assert sorted(joined) == sorted(filled) and len(scratch) == w.part_tiles
    assert seen > 3
