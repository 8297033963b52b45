"""The barrier protocol of the persistent packed attention (csrc/packed_attn.cu, packed_attn_kernel) in the
discrete-event model of protocol_model: random windows (with and without a second tile, with none and few key tiles),
random latencies, and every warp late by up to several microseconds anywhere, as one whose instructions are not in the
cache yet is.

  scheduler  per window: (from the second on) want_next, ask and get the next block; win_empty[slot]; publish; win_full
  producer   per window: win_full, win_empty; per key tile: (last one: want_next) k_empty, K; (first one: q_empty, Q);
             v_empty, V
  issuer     per window: win_full, win_empty; q_full, K(first); S of both tiles; then per key tile as the chunk attention;
             q_empty behind the window's last S, o_done[i] behind the last P V of each tile
  watcher    per key tile: V landed, next K of the window landed -> p_ready[0]; that phase complete
  softmax i  two agents, one per half of a tile's keys; per window with tile i, per key tile: s_full[i]; maxima exchanged
             (written, pair barrier, read); P; where the maximum has grown O rescaled by both, pair barrier; p_ready[i];
             then o_done[i]; sums exchanged between two pair barriers; O read; win_empty (windows without tile i: at once)
Hazards: S complete when read; P V only after P and V; P over S only after the P V that read it; O read when complete and
overwritten only after it was read; ring and Q slots refilled only after every MMA that read them; no wait lapped."""
import random

import pytest

from protocol_model import Bar, Model


def packed(m, windows, lateness, watch_first_k=False):
    """windows: [(n_p, n_s, two)]; an invalid one ends the list."""
    q_full, q_empty = Bar("q_full"), Bar("q_empty")
    k_full, k_empty = [Bar(f"k_full{s}") for s in range(2)], [Bar(f"k_empty{s}") for s in range(2)]
    v_full, v_empty = [Bar(f"v_full{s}") for s in range(2)], [Bar(f"v_empty{s}") for s in range(2)]
    s_full, o_done = [Bar(f"s_full{i}") for i in range(2)], [Bar(f"o_done{i}") for i in range(2)]
    p_ready = [Bar(f"p_ready{i}", 8 + (i == 0)) for i in range(2)]
    win_full, win_empty = [Bar(f"win_full{s}") for s in range(2)], [Bar(f"win_empty{s}", 7) for s in range(2)]
    pair = [Bar(f"pair{i}", 2) for i in range(2)]
    exchanged = {}                               # (tile, half) -> what the other half reads next
    want, steal = Bar("want_next"), Bar("steal")
    MMA_S, MMA_PV = 512, 256
    slots = [None, None]
    p_written, o_read, rescaled = {}, set(), {}
    late = lambda: ("work", m.rng.choice([0.0, 0.0, 0.0, m.rng.uniform(0, lateness)]))  # noqa: E731

    def scheduler():
        for i, w in enumerate([*windows, None]):
            yield late()
            if i > 0:
                yield ("wait", want, i)
                yield ("tma", steal, ("steal", i))
                yield ("wait", steal, i)
            yield ("wait", win_empty[i & 1], i >> 1)
            slots[i & 1] = (i, w)
            yield ("arrive", win_full[i & 1])

    def window(i):
        at, w = slots[i & 1]
        assert at == i, "window overwritten while read"
        return w

    def producer():
        j = loads = 0
        for i in range(len(windows) + 1):
            yield late()
            yield ("wait", win_full[i & 1], (i >> 1) + 1)
            w = window(i)
            yield ("arrive", win_empty[i & 1])
            if w is None:
                return
            if w[0] == 0:
                yield ("arrive", want)
            for t in range(w[0]):
                if t + 1 == w[0]:
                    yield ("arrive", want)
                yield late()
                yield ("wait", k_empty[j & 1], j >> 1)
                if j >= 2:
                    assert all(m.complete(tag) for tag in m.issued if tag[0] == "S" and tag[2] == j - 2), "K slot refilled"
                yield ("tma", k_full[j & 1], ("K", j))
                if t == 0:
                    yield ("wait", q_empty, loads)
                    assert all(m.complete(tag) for tag in m.issued if tag[0] == "S"), "Q refilled while read"
                    yield ("tma", q_full, ("Q", i))
                    loads += 1
                yield ("wait", v_empty[j & 1], j >> 1)
                if j >= 2:
                    assert all(m.complete(tag) for tag in m.issued if tag[0] == "PV" and tag[3] == j - 2), "V slot refilled"
                yield ("tma", v_full[j & 1], ("V", j))
                j += 1

    def issuer():
        jp, js, loads = 0, 0, 0
        for i in range(len(windows) + 1):
            yield late()
            yield ("wait", win_full[i & 1], (i >> 1) + 1)
            w = window(i)
            yield ("arrive", win_empty[i & 1])
            if w is None:
                return
            n_p, n_s, _ = w
            if n_p == 0:
                continue
            loads += 1
            yield ("wait", q_full, loads)
            yield ("wait", k_full[jp & 1], (jp >> 1) + 1)
            assert ("Q", i) in m.loaded and ("K", jp) in m.loaded
            for t in range(2 if n_s else 1):
                yield ("mma", ("S", t, jp), MMA_S)
                yield ("commit", s_full[t])
            yield ("commit", k_empty[jp & 1])
            if n_p == 1:
                yield ("commit", q_empty)
            for j in range(n_p):
                s, more = jp & 1, j + 1 < n_p
                yield late()
                yield ("wait", p_ready[0], jp + 1)
                assert p_written.get((0, jp), 0) == 8 and ("V", jp) in m.loaded, "P V before P / V"
                if j == 0:
                    assert all((0, k, g) in o_read for k in range(i) if windows[k][0] for g in range(2)), "O overwritten"
                yield ("mma", ("PV", 0, 0, jp), MMA_PV)
                if more:
                    assert ("K", jp + 1) in m.loaded, "S before K"
                    yield ("mma", ("S", 0, jp + 1), MMA_S)
                    yield ("commit", s_full[0])
                else:
                    yield ("commit", o_done[0])
                if j < n_s:
                    yield ("wait", p_ready[1], js + 1)
                    assert p_written.get((1, jp), 0) == 8, "P V before P"
                    if j == 0:
                        assert all((1, k, g) in o_read for k in range(i) if windows[k][1] for g in range(2)), "O overwritten"
                    yield ("mma", ("PV", 1, 0, jp), MMA_PV)
                    js += 1
                yield ("commit", v_empty[s])
                if j + 1 < n_s:
                    yield ("mma", ("S", 1, jp + 1), MMA_S)
                    yield ("commit", s_full[1])
                elif j + 1 == n_s:
                    yield ("commit", o_done[1])
                if more:
                    yield ("commit", k_empty[s ^ 1])
                if j + 2 == n_p:
                    yield ("commit", q_empty)
                jp += 1

    def watcher():
        jp = 0
        for i in range(len(windows) + 1):
            yield ("wait", win_full[i & 1], (i >> 1) + 1)
            w = window(i)
            yield ("arrive", win_empty[i & 1])
            if w is None:
                return
            yield late()
            if watch_first_k and w[0]:
                yield ("wait", k_full[jp & 1], (jp >> 1) + 1)
            for j in range(w[0]):
                yield late()
                yield ("wait", v_full[jp & 1], (jp >> 1) + 1)
                yield late()
                if j + 1 < w[0]:
                    yield ("wait", k_full[(jp + 1) & 1], ((jp + 1) >> 1) + 1)
                assert p_ready[0].k == jp
                yield ("arrive", p_ready[0])
                yield late()
                yield ("wait", p_ready[0], jp + 1)
                jp += 1

    def softmax(wg, half):
        jp, jt, done, meets = 0, 0, 0, 0   # key tiles of the primary, of this tile, windows of this tile, pair barriers

        def meet():
            nonlocal meets
            meets += 1
            yield ("arrive", pair[wg])
            yield ("wait", pair[wg], meets)

        def exchange(value, then=None):
            exchanged[(wg, half)] = value
            yield from meet()
            yield late()
            assert exchanged[(wg, half ^ 1)] == value, "the other half's value was overwritten before it was read"

        for i in range(len(windows) + 1):
            yield late()
            yield ("wait", win_full[i & 1], (i >> 1) + 1)
            yield from meet()
            w = window(i)
            if w is None:
                return
            n = w[wg]
            for j in range(n if w[2] or wg == 0 else 0):
                yield ("wait", s_full[wg], jt + 1)
                assert m.complete(("S", wg, jp + j)), "S read before it was complete"
                for tag in m.issued:
                    if tag[0] == "PV" and tag[1] == wg:
                        assert m.complete(tag), "P overwritten while read"
                yield ("work", m.rng.uniform(50, 600))
                yield from exchange(("max", jt))
                yield ("work", m.rng.uniform(150, 1300))
                if random.Random(jt * 2 + wg).random() < 0.3 and j:
                    for tag in m.issued:
                        if tag[0] == "PV" and tag[1] == wg:
                            assert m.complete(tag), "O rescaled while a P V runs"
                    yield ("work", m.rng.uniform(100, 500))
                    rescaled.setdefault((wg, jt), set()).add(half)
                    yield from meet()
                    assert len(rescaled[(wg, jt)]) == 2
                for _ in range(4):
                    p_written[(wg, jp + j)] = p_written.get((wg, jp + j), 0) + 1
                    assert p_ready[wg].k == jt, "softmax arrival in another phase"
                    yield ("arrive", p_ready[wg])
                jt += 1
            if wg == 0 or w[2]:
                if n:
                    done += 1
                    yield ("wait", o_done[wg], done)
                    assert all(m.complete(tag) for tag in m.issued if tag[0] == "PV" and tag[1] == wg)
                yield from exchange(("sum", i))
                yield from meet()
                if n:
                    yield ("work", m.rng.uniform(100, 1500))
                    o_read.add((wg, i, half))
            assert slots[i & 1][0] == i
            yield ("arrive", win_empty[i & 1])
            jp += w[0]

    for gen in (scheduler, producer, issuer, watcher):
        m.spawn(gen(), gen.__name__)
    for wg in range(2):
        for half in range(2):
            m.spawn(softmax(wg, half), f"softmax{wg}{half}")


def _windows(rng):
    out = []
    for _ in range(rng.randint(1, 6)):
        n_p = rng.choice([0, 1, 1, 2, 3, 5])
        two = rng.random() < 0.6
        out.append((n_p, rng.randint(max(0, n_p - 2), n_p) if two else 0, two))
    return out


@pytest.mark.parametrize("jitter", [0.0, 300.0, 3000.0])
@pytest.mark.parametrize("lateness", [0.0, 1000.0, 6000.0])
def test_packed_attention_protocol(jitter, lateness):
    for seed in range(200):
        m = Model(seed, commit_jitter=jitter)
        packed(m, _windows(random.Random(seed)), lateness)
        m.run()


def test_watching_the_first_key_tile_can_be_lapped():
    """A watcher that waits for a window's first K, which nothing holds back, misses it when it is late by a tile."""
    caught = 0
    for seed in range(100):
        m = Model(seed)
        packed(m, _windows(random.Random(seed)), 6000.0, watch_first_k=True)
        try:
            m.run()
        except AssertionError:
            caught += 1
    assert caught > 0
