"""Event-driven CPU model of the mbarrier protocol of the 8-bit prefill kernel (csrc/paged_prefill_q8.cu), on the simulator of
test_prefill_barrier_protocol.py.

Roles: item records, TMA producer (K bytes; what a tile is, into a ring of records), two MMA issuers, two softmax warpgroups, a
warpgroup that splits Q and writes V in fp16.  Beside what the simulator checks by itself (deadlock, parity aliases, too many
arrivals), under randomised latencies:

  * nobody reads a ring's entry (item, tile record, K slot, V slot, Q and its factors) that holds another item or tile, at the
    beginning of its use and at the end;
  * scores are not written over before all warps have taken them, nor probabilities before P.V has read them;
  * a warp that rescales O does so between the P.V in front and its own step's.
"""
import random
from collections import namedtuple

import pytest

from test_prefill_barrier_protocol import Bar, ProtocolError, Sim

K_SLOTS, V_SLOTS, ITEM_RING = 4, 3, 2
ITEM_READERS = 15

# steps of 64 keys of Q tile A / B (0: no such tile), live rows of either; rescale: how often a warp finds a larger maximum
Item = namedtuple("Item", "steps live rescale")


def run_cta(items, seed=0, jitter=0.0, infos=8, early_k=False, last_two=True, factors=2, qk_first=False):
    sim = Sim(seed, jitter)
    item_full = [Bar(f"item_full{s}", 1) for s in range(ITEM_RING)]
    item_empty = [Bar(f"item_empty{s}", ITEM_READERS) for s in range(ITEM_RING)]
    q_full, q_empty = Bar("q_full", 4), Bar("q_empty", 2)
    factor_full = [Bar(f"factor_full{s}", 4) for s in range(2)]
    k_full, k_empty = [Bar(f"k_full{s}", 1) for s in range(K_SLOTS)], [Bar(f"k_empty{s}", 2) for s in range(K_SLOTS)]
    v_full, v_empty = [Bar(f"v_full{s}", 4) for s in range(V_SLOTS)], [Bar(f"v_empty{s}", 2) for s in range(V_SLOTS)]
    info_full = [Bar(f"info_full{s}", 1) for s in range(infos)]
    s_full = [[Bar(f"s_full{x}{b}", 1) for b in range(2)] for x in range(2)]
    p_full = [[Bar(f"p_full{x}{b}", 4) for b in range(2)] for x in range(2)]
    o_done = [[Bar(f"o_done{x}{b}", 1) for b in range(2)] for x in range(2)]
    o_empty = [Bar(f"o_empty{x}", 4) for x in range(2)]
    ring, info, k_slot, v_slot = [None] * ITEM_RING, [None] * infos, [None] * K_SLOTS, [[None] * 4 for _ in range(V_SLOTS)]
    q_rows, q_factor = [None] * 4, [[None] * 4 for _ in range(2)]  # a converting warp's share each
    scores = [[None] * 2 for _ in range(2)]  # step whose scores a buffer holds
    probs = [[set() for _ in range(2)] for _ in range(2)]  # warps that have written theirs over them
    products = [0, 0]  # P.V of a Q tile that are complete, over all items

    def expect(what, got, want):
        if got != want:
            raise ProtocolError(f"{what} holds {got}, not {want}")

    def n_kv(it):
        return max((s + 1) // 2 for s in it.steps)

    def records():
        for k in range(len(items) + 1):
            if k >= ITEM_RING:
                yield ("wait", item_empty[k % ITEM_RING], k // ITEM_RING - 1)
            yield ("delay", 1400)
            ring[k % ITEM_RING] = k
            yield ("arrive", item_full[k % ITEM_RING])

    def next_item(k):
        yield ("wait", item_full[k % ITEM_RING], k // ITEM_RING)
        expect("item ring", ring[k % ITEM_RING], k)
        return items[k] if k < len(items) else None

    def producer():
        t = i = 0
        while (it := (yield from next_item(i))) is not None:
            yield ("arrive", item_empty[i % ITEM_RING])
            yield ("delay", 700)
            for _ in range(n_kv(it)):
                if t >= K_SLOTS:
                    yield ("wait", k_empty[t % K_SLOTS], t // K_SLOTS - 1)
                info[t % infos] = t
                yield ("arrive", info_full[t % infos])
                k_slot[t % K_SLOTS] = t
                yield ("tma", k_full[t % K_SLOTS])
                t += 1
            i += 1

    def issuer(x):
        kt = g = used = i = 0

        def qk(h, steps):
            t, b = kt + h // 2, (g + h) & 1
            if h & 1 == 0:
                yield ("wait", k_full[t % K_SLOTS], t // K_SLOTS)
            expect("K slot", k_slot[t % K_SLOTS], t)
            if len(probs[x][b]) not in (0, 4):
                raise ProtocolError(f"scores of step {g + h} written over {len(probs[x][b])} warps' probabilities")
            if scores[x][b] is not None and not probs[x][b]:
                raise ProtocolError(f"scores of step {scores[x][b]} written over before they were read")
            scores[x][b] = g + h
            probs[x][b] = set()
            yield ("mma", 384, [s_full[x][b]] + ([q_empty] if h + 1 == steps else []))
            expect("K slot, when Q.K^T has been issued,", k_slot[t % K_SLOTS], t)

        while (it := (yield from next_item(i))) is not None:
            yield ("arrive", item_empty[i % ITEM_RING])
            steps = it.steps[x]
            yield ("wait", q_full, i)
            expect("Q", q_rows, [i] * 4)
            if steps == 0:
                yield ("arrive", q_empty)
            for h in range(min(2, steps)):
                yield from qk(h, steps)
            for h in range(steps):
                t, b = kt + h // 2, (g + h) & 1
                if h & 1 == 0:
                    yield ("wait", v_full[t % V_SLOTS], t // V_SLOTS)
                expect("V slot", v_slot[t % V_SLOTS], [t] * 4)
                if h == 0 and used > 0:
                    yield ("wait", o_empty[x], used - 1)
                yield ("wait", p_full[x][b], (g + h) // 2)
                expect("probabilities", (scores[x][b], len(probs[x][b])), (g + h, 4))
                commits = []
                if last_two and (h + 2 == steps or steps == 1):
                    commits.append(o_done[x][0])
                if h + 1 == steps:
                    commits.append(o_done[x][1])
                if h & 1 or h + 1 == steps:
                    commits.append(v_empty[t % V_SLOTS])
                if qk_first and h + 2 < steps:
                    yield from qk(h + 2, steps)
                yield ("mma", 256, [Counter(x)] + commits)
                if h + 2 < steps and not qk_first:
                    yield from qk(h + 2, steps)
            for j in range((steps + 1) // 2, n_kv(it)):
                t = kt + j
                yield ("wait", k_full[t % K_SLOTS], t // K_SLOTS)
                yield ("arrive", k_empty[t % K_SLOTS])
                yield ("wait", v_full[t % V_SLOTS], t // V_SLOTS)
                yield ("arrive", v_empty[t % V_SLOTS])
            g += steps
            used += steps > 0
            kt += n_kv(it)
            i += 1

    class Counter(Bar):  # an arrival on it is a P.V of Q tile x that is complete
        def __init__(self, x):
            super().__init__(f"count{x}", 1)
            self.x = x

        @property
        def pending(self):
            return self._pending

        @pending.setter
        def pending(self, value):
            self._pending = value
            if value == 0:
                products[self.x] += 1

    def softmax(x, warp):
        rng = random.Random(seed * 100 + x * 10 + warp)
        g = kt = used = k = 0
        while (it := (yield from next_item(k))) is not None:
            steps, g0, kt0, i = it.steps[x], g, kt, k
            kt, g, k = kt + n_kv(it), g + steps, k + 1
            if steps == 0:
                yield ("arrive", item_empty[i % ITEM_RING])
                continue
            yield ("delay", rng.choice([0, 0, 0, 6000]))  # a warp that is held up
            yield ("wait", factor_full[i & 1], i // 2)
            expect("factors of Q", q_factor[i % factors], [i] * 4)
            dead = 32 * warp >= it.live[x]
            for h in range(steps):
                t, b = kt0 + h // 2, (g0 + h) & 1
                if not dead and h & 1 == 0:
                    yield ("wait", info_full[t % infos], t // infos)
                    expect("tile record", info[t % infos], t)
                if early_k and h & 1 == 0 and warp == 0:
                    yield ("arrive", k_empty[t % K_SLOTS])
                yield ("wait", s_full[x][b], (g0 + h) // 2)
                expect("scores", scores[x][b], g0 + h)
                if not early_k and (h & 1 or h + 1 == steps) and warp == 0:
                    yield ("arrive", k_empty[t % K_SLOTS])
                if not dead:
                    yield ("delay", 200)
                    if h > 0 and rng.random() < it.rescale:
                        if h + 1 < steps:
                            yield ("wait", s_full[x][b ^ 1], (g0 + h + 1) // 2)
                        elif last_two:
                            yield ("wait", o_done[x][0], used)
                        if products[x] != g0 + h:
                            raise ProtocolError(f"O rescaled in front of step {g0 + h} after {products[x]} P.V")
                        yield ("delay", 400)
                        expect("P.V complete, after the rescaling,", products[x], g0 + h)
                    yield ("delay", 700)
                expect("scores, until the probabilities are there,", scores[x][b], g0 + h)
                probs[x][b].add(warp)
                yield ("arrive", p_full[x][b])
            yield ("wait", o_done[x][1], used)
            expect("P.V complete, at the end,", products[x], g)
            used += 1
            if not dead:
                yield ("delay", 900)
            expect("P.V complete, behind the epilogue,", products[x], g)
            yield ("arrive", o_empty[x])
            yield ("arrive", item_empty[i % ITEM_RING])

    def convert(w):
        t = k = 0
        while (it := (yield from next_item(k))) is not None:
            yield ("arrive", item_empty[k % ITEM_RING])
            if k > 0:
                yield ("wait", q_empty, k - 1)
            yield ("delay", 1500)
            q_rows[w] = k
            q_factor[k % factors][w] = k
            yield ("arrive", factor_full[k & 1])
            yield ("arrive", q_full)
            for j in range(n_kv(it)):
                yield ("wait", info_full[t % infos], t // infos)
                expect("tile record, for V,", info[t % infos], t)
                yield ("delay", 800)
                if t >= V_SLOTS:
                    yield ("wait", v_empty[t % V_SLOTS], t // V_SLOTS - 1)
                v_slot[t % V_SLOTS][w] = t
                yield ("delay", 300)
                yield ("arrive", v_full[t % V_SLOTS])
                t += 1
            k += 1

    sim.spawn("records", records())
    sim.spawn("producer", producer())
    for x in range(2):
        sim.spawn(f"issuer{x}", issuer(x))
        for warp in range(4):
            sim.spawn(f"softmax{x}{warp}", softmax(x, warp))
    for w in range(4):
        sim.spawn(f"convert{w}", convert(w))
    sim.run()
    return sim.t


def random_items(rng, count):
    items = []
    for _ in range(count):
        a = rng.choice([1, 1, 2, 3, 4, 5, 8, 13, 24])
        b = rng.choice([0, a, a, a + 1, a + 2, max(1, a - 1), 1])
        items.append(Item((a, b), (rng.choice([1, 40, 128]), rng.choice([1, 70, 128])), rng.choice([0.0, 0.1, 1.0])))
    return items


def test_single_items():
    for a in range(1, 12):
        for b in (0, a, a + 1, a + 2, a + 9):
            for rescale in (0.0, 1.0):
                for live in (1, 128):
                    run_cta([Item((a, b), (live, live), rescale)])


@pytest.mark.parametrize("seed", range(40))
def test_random_item_lists_under_random_latencies(seed):
    rng = random.Random(seed)
    items = random_items(rng, rng.randint(1, 14))
    for jitter in (0.0, 0.4, 0.95):
        run_cta(items, seed=seed, jitter=jitter)


def broken(**how):
    for seed in range(60):
        rng = random.Random(seed)
        run_cta(random_items(rng, 12), seed=seed, jitter=0.95, **how)


def test_model_catches_broken_protocols():
    with pytest.raises(ProtocolError):  # a K slot given back before its scores are there
        broken(early_k=True)
    with pytest.raises(ProtocolError):  # records of only as many tiles as there are K slots
        broken(infos=4)
    with pytest.raises(ProtocolError, match="rescaled|P.V"):  # an item's last rescaling does not wait for the P.V in front
        broken(last_two=False)
    with pytest.raises(ProtocolError, match="factors"):  # factors of one item at a time
        broken(factors=1)
    with pytest.raises(ProtocolError):  # the next scores issued in front of the P.V whose probabilities they replace
        broken(qk_first=True)
