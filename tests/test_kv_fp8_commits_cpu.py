"""The end of chunk attention over the 8-bit cache (csrc/kv_fp8_chunk.cu): commits of the tensor core arrive at a block's barriers by
themselves, some time after the products that they follow, and in pairs at the partner's too.  Nobody may have left by then.

The roles and their order are those of the walk through the barriers; here the arrivals of commits are on their way by themselves, to each
block in the order of issue."""
import random

import pytest
from tests.test_kv_fp8_protocol_cpu import Kernel

ITEMS = [[(2, 5)], [(1, 1)], [(2, 1)] * 6, [(1, 2), (2, 3), (1, 0), (2, 1), (1, 1), (1, 4)], [(2, 0)], [(2, 2), (1, 1), (1, 1), (2, 9)]]


class Late(Kernel):
    """``drained``: the roles wait for the last arrivals, as the kernel's do."""

    def __init__(self, form, items, rng, drained):
        super().__init__(form, items, rng)
        self.drained, self.on_their_way, self.left = drained, [[] for _ in range(self.ctas)], [False] * self.ctas

    def tensor(self):
        """Products in the order of issue, and commits that start out behind them."""
        while not self.issued or self.queue or any(self.on_their_way):
            yield None
            under_way = [c for c in range(self.ctas) if self.on_their_way[c]]
            if under_way and (not self.queue or self.rng.random() < 0.5):
                c = self.rng.choice(under_way)
                assert not self.left[c], "an arrival at a block that has left"
                self.on_their_way[c].pop(0).arrive()
            elif self.queue:
                op = self.queue.pop(0)
                if op[0] == "commit":
                    for c, b in enumerate(op[1]):
                        self.on_their_way[c].append(b)
                else:
                    self.product(op)

    def product(self, op):
        for c in range(self.ctas):
            if op[0] == "S":
                self.s[c][op[1]] = op[3:]
            else:
                _, g, h, _, i, j, _ = op
                self.o[c][g], self.p[c][2 * g + h] = (i, j, h), None

    # the roles of a block: what they do and then, at the end, wait for
    def turn(self, c, w):
        yield from super().turn(c, w)
        if self.drained:
            blocks = sum(b for _, b in self.items)
            for slot in range(self.ring):
                yield self.kv_empty[c][slot], len(range(slot, 2 * blocks, self.ring)) - 1

    def copies(self, c):
        yield from super().copies(c)
        if self.drained:
            yield self.q_empty[c][0], sum(b > 0 for _, b in self.items) - 1

    def softmax(self, c, g):
        yield from super().softmax(c, g)
        if self.drained and self.halves == 2:
            blocks = sum((b + 1 - g) // 2 if self.form == "dual" else b if g == 0 or t == 2 else 0 for t, b in self.items)
            yield self.o_full[c][g * 2], blocks - 1

    def run(self):
        C = range(self.ctas)
        roles = {c: [self.copies(c), *(self.turn(c, w) for w in range(2)), *(self.softmax(c, g) for g in range(2))] for c in C}
        agents = [self.issue(), self.tensor(), *(a for c in C for a in roles[c])]
        at = {a: next(a, "end") for a in agents}
        for _ in range(10 ** 6):
            if all(v == "end" for v in at.values()):
                return
            # a pair's blocks leave together (a barrier of the cluster), when the threads of both are done
            if at[agents[0]] == "end" and all(at[a] == "end" for c in C for a in roles[c]):
                self.left = [True] * self.ctas
            ready = [a for a in agents if at[a] != "end" and (at[a] is None or at[a][0].passes(at[a][1]))]
            assert ready, "nobody can go on"
            a = self.rng.choice(ready)
            for _ in range(self.rng.choice([1, 1, 3, 40])):
                at[a] = next(a, "end")
                if at[a] == "end" or (at[a] is not None and not at[a][0].passes(at[a][1])):
                    break
        raise AssertionError("nobody comes to an end")


def _runs(form, drained):
    rng = random.Random(5)
    for items in ITEMS + [[(rng.randint(1, 2), rng.randint(0, 4)) for _ in range(rng.randint(1, 6))] for _ in range(12)]:
        for _ in range(10):
            Late(form, [(1, b) for _, b in items] if form == "dual" else items, rng, drained).run()


@pytest.mark.parametrize("form", ["two", "dual", "pair"])
def test_no_commit_arrives_at_a_block_that_has_left(form):
    _runs(form, True)


@pytest.mark.parametrize("form", ["two", "dual", "pair"])
def test_without_the_last_waits_one_does(form):
    with pytest.raises(AssertionError, match="has left"):
        _runs(form, False)
