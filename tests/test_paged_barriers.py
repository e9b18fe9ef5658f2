"""The barriers of the tensor-core prompt kernel (jx_paged_prompt.cu), modelled on the CPU.

Every wait and arrival of the kernel's roles in a random order: each wait has to end, and on the
phase that it means.  Ring stages and the period of the partial sums are read from the source."""
import os
import random
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "jxai_b200", "csrc",
                      "jx_paged_prompt.cu")


def constant(name, hd):
    """`name = HD == 64 ? a : b` of the kernel's configuration."""
    with open(SOURCE) as fh:
        a, b = re.search(rf"int {name} = HD == 64 \? (\d+) : (\d+);", fh.read()).groups()
    return int(a) if hd == 64 else int(b)


class Run:
    """Roles as generators of waits (barrier, phase that has to be complete); a wait names its phase
    by the parity alone, as the kernel's do."""

    let_on = True  # a tile without rows has a commit of its own, too

    def __init__(self, items, stages, drain):
        self.items, self.stages, self.drain = items, stages, drain
        self.done = {}      # barrier -> completed phases
        self.commits = []   # of the tensor cores, in order
        self.copies = []    # on their way, in order

    def arrive(self, bar):
        self.done[bar] = self.done.get(bar, 0) + 1

    def producer(self):
        n = 0
        for item in self.items:
            for _ in range(2 * max(item)):
                if n >= self.stages:
                    yield ("free", n % self.stages), n // self.stages
                self.copies.append(("full", n % self.stages))
                n += 1

    def issuer(self):
        base, weights = 0, [0, 0]

        def tile(n):
            return ("full", n % self.stages), n // self.stages + 1
        for i, item in enumerate(self.items):
            for x in (0, 1):
                yield ("q", x), i + 1
                if item[x]:
                    if weights[x]:
                        yield ("pv", x), weights[x]
                    yield tile(base)
                if item[x] or self.let_on:
                    self.commits.append(("s", x))
            if max(item):
                self.commits.append(("free", base % self.stages))
            for t in range(max(item)):
                for x in (0, 1):
                    if t >= item[x]:
                        continue
                    weights[x] += 1
                    yield ("p", x), weights[x]
                    if t == 0 and i:
                        yield ("o", x), i
                    yield tile(base + 2 * t + 1)
                    self.commits.append(("pv", x))
                    if t + 1 < item[x]:
                        yield ("pv", x), weights[x]
                        yield tile(base + 2 * t + 2)
                        self.commits.append(("s", x))
                self.commits.append(("free", (base + 2 * t + 1) % self.stages))
                if t + 1 < max(item):
                    self.commits.append(("free", (base + 2 * t + 2) % self.stages))
            base += 2 * max(item)

    def softmax(self, x):
        scores = weights = 0
        self.arrive(("q", x))
        for i, item in enumerate(self.items):
            for t in range(item[x]):
                if t and t % self.drain == 0:
                    yield ("pv", x), weights
                scores += 1
                yield ("s", x), scores
                self.arrive(("p", x))
                weights += 1
            if not item[x]:
                scores += 1
                yield ("s", x), scores
            if i + 1 < len(self.items):
                self.arrive(("q", x))
            if item[x]:
                yield ("pv", x), weights
            self.arrive(("o", x))

    def go(self, rng):
        roles = [self.producer(), self.issuer(), self.softmax(0), self.softmax(1)]
        waits = [next(r, None) for r in roles]
        while any(w is not None for w in waits):
            # a wait passes when the phase of its parity is complete: done and phase alike, mod 2
            ready = [i for i, w in enumerate(waits) if w is not None and (self.done.get(w[0], 0) - w[1]) % 2 == 0]
            acts = ready + ["commit"] * bool(self.commits) + ["copy"] * bool(self.copies)
            assert acts, "a wait never ends"
            act = rng.choice(acts)
            if act == "commit":
                self.arrive(self.commits.pop(0))
            elif act == "copy":
                self.arrive(self.copies.pop(0))
            else:
                bar, phase = waits[act]
                assert self.done.get(bar, 0) == phase, f"the wait for {bar} ends on another phase"
                waits[act] = next(roles[act], None)


@pytest.mark.parametrize("hd", [64, 128])
def test_every_wait_ends_on_its_phase(hd):
    stages, drain = constant("NS", hd), constant("DRAIN", hd)
    rng = random.Random(hd)
    for _ in range(500):
        items = []
        for _ in range(rng.randint(1, 6)):
            a = rng.randint(1, 3 * drain + 1)
            items.append((a, rng.choice([0, a, a + 1, max(1, a - 1)])))
        Run(items, stages, drain).go(rng)


def test_the_model_finds_a_tile_that_runs_ahead():
    """Without the commit that lets a tile without rows on, its softmax would wait for good."""
    class Without(Run):
        let_on = False
    with pytest.raises(AssertionError):
        Without([(3, 0), (3, 3)], 8, 4).go(random.Random(0))
