"""What the slots of a cache are said to share: ids and lengths after forks, forks of forks and releases.  No GPU is touched."""

import random

import pytest
import torch

from tests.test_host_step import cache_of, launches  # noqa: F401  (a fixture)

P = 16


class Lines:
    """A cache and the tokens of each slot, by name."""

    def __init__(self, slots=60, n_pages=6000, columns=400):
        self.cache = cache_of(slots, n_pages, P=P, columns=columns, prefix_sharing=True)
        self.tokens: dict[int, list[int]] = {}
        self.named = 0

    def new(self, n):
        slot = self.cache.allocate()
        self.tokens[slot] = []
        self.extend(slot, n)
        return slot

    def extend(self, slot, more):
        old = len(self.tokens[slot])
        self.cache.step_tables([slot], [old], [old + more])
        self.tokens[slot] += range(self.named, self.named + more)
        self.named += more

    def fork(self, parent, n, count=1):
        slots = self.cache.fork(parent, n, count)
        for slot in slots:
            self.tokens[slot] = self.tokens[parent][:n]
        return slots

    def erase(self, slot):
        self.cache.erase(slot)
        del self.tokens[slot]

    def said(self, *slots):
        return [(int(self.cache.prefix_ids[s]), int(self.cache.prefix_lens[s])) for s in slots]

    def check(self):
        ids, lens = self.cache.prefix_ids.tolist(), self.cache.prefix_lens.tolist()
        for a in range(len(ids)):
            if a not in self.tokens:
                assert ids[a] == 0
            for b in range(a):
                if ids[a] == ids[b] > 0:
                    n = min(lens[a], lens[b])
                    assert n <= len(self.tokens[a]) and self.tokens[a][:n] == self.tokens[b][:n]


def test_one_line(launches):
    s = Lines()
    cat, dog = s.new(133), s.new(40)
    assert s.said(cat, dog) == [(0, 0), (0, 0)]
    a = s.fork(cat, 133, 3)
    assert s.said(cat, *a) == [(1, 133)] * 4
    b = s.fork(cat, 64, 2)
    assert s.said(cat, *b) == [(1, 133), (1, 64), (1, 64)]
    s.extend(cat, 100)
    c = s.fork(cat, 233)
    assert s.said(cat, *a, *b, *c) == [(1, 233)] + [(1, 133)] * 3 + [(1, 64)] * 2 + [(1, 233)]
    d = s.fork(dog, 40, 1)
    assert s.said(dog, *d) == [(2, 40)] * 2
    s.erase(cat)
    assert s.said(cat, *a) == [(0, 233)] + [(1, 133)] * 3
    again = s.new(10)
    assert again == cat and s.said(again)[0][0] == 0
    s.check()


def test_questions_about_pictures_behind_one_system_prompt(launches):
    """All forks of a picture share the picture, not the system prompt alone."""
    s = Lines()
    system = s.new(500)
    pictures = s.fork(system, 500, 3)
    for p in pictures:
        s.extend(p, 4000)
    asked = [s.fork(p, 4500, 8) for p in pictures[:2]]
    asked.append([s.fork(pictures[2], 4500)[0] for _ in range(8)])  # one at a time
    for p, forks in zip(pictures, asked):
        (line,) = set(s.said(p, *forks))
        assert line[1] == 4500
    assert len({i for i, _ in s.said(system, *pictures)}) == 4
    s.check()


def test_a_fork_that_goes_on_a_little_stays_in_its_line(launches):
    s = Lines()
    cat = s.new(1000)
    beams = s.fork(cat, 1000, 6)
    for b in beams:
        s.extend(b, 20)
    twice = [s.fork(b, 1020)[0] for b in beams]
    assert set(s.said(cat, *beams, *twice)) == {(1, 1000)}
    # 41 forks of one of them, 20 tokens behind the line: 820 tokens that they do not share with each other, below the line's 1000
    more = [s.fork(beams[0], 1020)[0] for _ in range(40)]
    assert set(s.said(*more)) == {(1, 1000)}
    s.extend(beams[0], 300)
    late = s.fork(beams[0], 1320)
    assert s.said(beams[0], *late) == [(2, 1320)] * 2 and set(s.said(cat, *beams[1:], *more)) == {(1, 1000)}
    s.check()


@pytest.mark.parametrize("seed", range(12))
def test_what_slots_are_said_to_share_they_share(launches, seed):
    rng = random.Random(seed)
    s = Lines()
    for _ in range(120):
        what = rng.random()
        if not s.tokens or (what < 0.15 and len(s.tokens) < 50):
            s.new(rng.randrange(1, 700))
        elif what < 0.4:
            s.extend(rng.choice(list(s.tokens)), rng.randrange(1, 90))
        elif what < 0.8 and len(s.tokens) < 50:
            parent = rng.choice(list(s.tokens))
            s.fork(parent, rng.randrange(1, len(s.tokens[parent]) + 1), rng.randrange(1, 4))
        elif what >= 0.8:
            s.erase(rng.choice(list(s.tokens)))
        s.check()
    for slot in list(s.tokens):
        s.erase(slot)
    assert not s.cache._prefixes and not s.cache._page_slots and not s.cache.prefix_ids.any()
    assert sorted(s.cache.free_pages) == list(range(1, 6000))
