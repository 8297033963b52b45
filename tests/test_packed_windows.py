"""The search of the packed attention's scheduler warp (csrc/packed_attn.cu, packed_attn_kernel, warp 19) for the sequence
and the pair of query tiles of a window, restated step for step with its 32-bit unsigned arithmetic: whatever blocks a CTA
is given, and in whatever order, each window of the batch is found exactly once and no other. Blocks past the last window
(the grid is an upper bound) are passed over."""
import random

import pytest

M32 = (1 << 32) - 1


class Search:
    """One CTA's search; it keeps its place from window to window. forward: it never starts again, and ends with the first
    block that holds no window."""

    def __init__(self, lens, rows, forward=False):
        self.lens, self.rows, self.forward, self.over = lens, rows, forward, False   # rows: query tokens of a pair of tiles
        self.b_at, self.loaded, self.before = 0, -1, 0

    def _load(self):
        """32 sequences, those with most keys first (here: as many keys as queries), their windows and sums."""
        part = [(self.lens[b] if b < len(self.lens) else 0, b) for b in range(self.b_at, self.b_at + 32)]
        part = [part[i] for i in sorted(range(32), key=lambda i: (-part[i][0], i))]
        self.seq = [b for _, b in part]
        self.own = [-(-n // self.rows) for n, _ in part]
        self.upto, total = [], 0
        for n in self.own:
            total = (total + n) & M32
            self.upto.append(total)
        self.loaded = self.b_at

    def find(self, pair):
        """(sequence, pair of tiles), or None past the last window."""
        if self.over:
            return None
        if not self.forward and pair < self.before:
            self.b_at = self.before = 0
        while self.b_at < len(self.lens):
            if self.loaded != self.b_at:
                self._load()
            hit = [i for i in range(32) if (self.before + self.upto[i]) & M32 > pair]
            if hit:
                at = hit[0]
                skipped = (self.upto[at] - self.own[at]) & M32
                place = min((pair - self.before - skipped) & M32, (self.own[at] - 1) & M32)
                return self.seq[at], (self.own[at] - 1 - place) & M32
            self.before = (self.before + self.upto[31]) & M32
            self.b_at += 32
        self.over = self.forward
        return None


def _cover(seed, forward):
    """All blocks of a grid dealt to a few CTAs, in the grid's order, nearly so, or in none."""
    rng = random.Random(seed)
    rows = rng.choice([4, 32, 256])
    lens = [rng.choice([0, 1, rows, rng.randint(1, 5 * rows)]) for _ in range(rng.choice([1, 20, 33, 100, 200]))]
    blocks = list(range(sum(lens) // rows + len(lens)))             # the host's upper bound
    want = sorted((b, i) for b, n in enumerate(lens) for i in range(-(-n // rows)))
    if seed % 3:
        key = {i: i + rng.uniform(0, 40 if seed % 3 == 1 else 1e6) for i in blocks}
        blocks.sort(key=key.get)
    ctas = [Search(lens, rows, forward) for _ in range(rng.choice([1, 3, 16]))]
    found = [rng.choice(ctas).find(i) for i in blocks]
    return sorted(f for f in found if f is not None) == want


@pytest.mark.parametrize("seed", range(60))
def test_every_window_is_found_once_in_any_order_of_blocks(seed):
    assert _cover(seed, forward=False)


def test_a_search_that_only_goes_forward_depends_on_the_order():
    assert all(_cover(seed, forward=True) for seed in range(0, 60, 3))           # in the grid's order
    assert not all(_cover(seed, forward=True) for seed in range(60))
