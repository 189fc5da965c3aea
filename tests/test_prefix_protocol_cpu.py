"""A CPU model of the barrier protocol of kv_prefix_kernel (qraf_b200/csrc/kv_prefix.cuh): the two
softmax warpgroups, the warps that make K and V tiles, and the MMA warp with its asynchronous MMAs and
commits, each written as the kernel runs it over several stretches, interleaved at random and with
roles of very different speeds.

The model checks what the GPU's timing hides:
  * every parity wait that passes passes for the phase it means (not two phases early, nor lapped);
  * no tile, score buffer, scale or maximum is read before it is there or overwritten while it is needed;
  * O is read, scaled and left only while no MMA into it is in flight;
  * every role finishes."""
from __future__ import annotations

import random

import pytest


class Bar:
    """mbarrier: `count` arrivals complete a phase."""

    def __init__(self, count):
        self.count, self.pending, self.completed = count, count, 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.completed += 1
            self.pending = self.count

    def passes(self, phase):
        """try_wait.parity for the completion of phase `phase` (0-based), as the hardware answers it."""
        if (self.completed ^ phase) & 1 == 0:
            assert self.completed <= phase, "a wait that its phase has left behind"
            return False
        assert self.completed == phase + 1, "a wait passed for another phase than its own"
        return True


class Sync:
    """__syncthreads or a named barrier over `count` warps."""

    def __init__(self, count):
        self.count, self.here, self.round = count, 0, 0

    def wait(self):
        mine = self.round
        self.here += 1
        if self.here == self.count:
            self.here, self.round = 0, self.round + 1
        while self.round == mine:
            yield


def run_model(stretches, term, seed, last_wait="o_ready"):
    """One CTA over stretches of so many tiles; O starts anew every `term` tiles."""
    rng = random.Random(seed)
    k_ready, s_ready, p_ready = ([Bar(c) for _ in range(3)] for c in (4, 1, 4))
    v_ready, pv_done = ([Bar(c) for _ in range(2)] for c in (4, 1))
    m_ready = [[Bar(1) for _ in range(4)] for _ in range(2)]
    q_ready, o_ready = Bar(8), Bar(1)
    everyone, all_v = Sync(17), Sync(4)
    queue = []             # MMAs and commits in their order, not yet complete
    done = set()           # ("S", x) and ("PV", x) that are
    k_tile, v_tile = [None] * 4, [[None] * 4 for _ in range(2)]      # by the warps that write them: the tile's x
    scales, scores = [[None] * 4 for _ in range(3)], [[None] * 4 for _ in range(3)]   # scores: ("S" or "P", x) by warp's rows
    maxima = [[None] * 4 for _ in range(2)]
    queries = [None] * 8
    read = set()           # (x, w): the maximum of tile x has been read by the next tile's warp

    def wait(bar, phase):
        while not bar.passes(phase):
            yield

    def in_flight(kind, x=None):
        return any(op[0] == kind and (x is None or op[1] == x) for op in queue)

    def softmax(wg, w):
        x0 = 0
        for stretch, n in enumerate(stretches):
            assert not in_flight("S") and not in_flight("PV"), "queries overwritten under an MMA"
            queries[4 * wg + w] = stretch
            q_ready.arrive()
            yield
            for t in range(wg, n, 2):
                x = x0 + t
                b = x % 3
                yield from wait(k_ready[b], x // 3)
                yield from wait(s_ready[b], x // 3)
                assert scales[b] == [x] * 4 and scores[b][w] == ("S", x)
                yield
                alpha = False
                if t > 0:
                    px = x - 1
                    yield from wait(m_ready[px & 1][w], px >> 1)
                    assert maxima[px & 1][w] == px
                    read.add((px, w))
                    alpha = t % term != 0 and rng.random() < 0.4
                assert t < 2 or (x - 2, w) in read, "a maximum overwritten before it was read"
                maxima[x & 1][w] = x
                m_ready[x & 1][w].arrive()
                yield
                if alpha or t > 0 and t % term == 0:   # scale O, or let its term go
                    yield from wait(pv_done[(x - 1) & 1], (x - 1) >> 1)
                    for _ in range(2):
                        assert ("PV", x - 1) in done and not in_flight("PV") and ("PV", x) not in done
                        yield
                assert scales[b] == [x] * 4
                scores[b][w] = ("P", x)
                yield
                p_ready[b].arrive()
            x0 += n
            last = x0 - 1
            if last_wait == "o_ready":
                yield from wait(o_ready, stretch)
            else:
                yield from wait(pv_done[last & 1], last >> 1)
            yield from everyone.wait()
            for _ in range(2):
                assert ("PV", last) in done and not queue, "O left before its last MMA"
                yield
            yield from everyone.wait()
            if stretch + 1 < len(stretches):
                yield from everyone.wait()

    def make_k(w):
        x0 = 0
        for stretch, n in enumerate(stretches):
            for t in range(n):
                x = x0 + t
                b = x % 3
                if x > 0:
                    yield from wait(s_ready[(x - 1) % 3], (x - 1) // 3)
                if x > 2:
                    yield from wait(p_ready[b], x // 3 - 1)
                assert x == 0 or ("S", x - 1) in done, "K overwritten under an MMA"
                assert x < 3 or scores[b] == [("P", x - 3)] * 4, "scales overwritten before they were read"
                k_tile[w] = scales[b][w] = x
                yield
                k_ready[b].arrive()
                yield
            x0 += n
            yield from everyone.wait()
            yield from everyone.wait()
            if stretch + 1 < len(stretches):
                yield from everyone.wait()

    def make_v(w):
        x0 = 0
        for stretch, n in enumerate(stretches):
            for t in range(n):
                x = x0 + t
                yield from all_v.wait()
                if x > 1:
                    yield from wait(pv_done[x & 1], x // 2 - 1)
                assert x < 2 or ("PV", x - 2) in done, "V overwritten under an MMA"
                v_tile[x & 1][w] = x
                yield
                v_ready[x & 1].arrive()
                yield from all_v.wait()
            x0 += n
            yield from everyone.wait()
            yield from everyone.wait()
            if stretch + 1 < len(stretches):
                yield from everyone.wait()

    def mma():
        x0 = 0
        for stretch, n in enumerate(stretches):
            def scores_of(t, other, phase):
                x = x0 + t
                yield from wait(k_ready[x % 3], x // 3)
                yield from wait(other, phase)
                assert k_tile == [x] * 4 and queries == [stretch] * 8
                assert t < 3 or ("PV", x - 3) in done, "scores over weights that are still read"
                queue.extend([("S", x), ("commit", s_ready[x % 3])])

            for t in range(min(3, n)):
                yield from scores_of(t, q_ready, stretch)
                yield
            for t in range(n):
                x = x0 + t
                b, sl = x % 3, x & 1
                yield from wait(p_ready[b], x // 3)
                yield from wait(v_ready[sl], x >> 1)
                assert scores[b] == [("P", x)] * 4 and v_tile[sl] == [x] * 4
                queue.extend([("PV", x), ("commit", pv_done[sl])])
                if t + 1 == n:
                    queue.append(("commit", o_ready))
                yield
                if t + 3 < n:
                    yield from scores_of(t + 3, pv_done[sl], x >> 1)
            x0 += n
            yield from everyone.wait()
            yield from everyone.wait()
            if stretch + 1 < len(stretches):
                yield from everyone.wait()
        assert not queue, "TMEM freed under an MMA"

    def tensor_cores():
        while True:
            if queue:
                kind, what = queue.pop(0)
                if kind == "commit":
                    what.arrive()
                else:
                    done.add((kind, what))
                    if kind == "S":
                        scores[what % 3][:] = [("S", what)] * 4
            yield

    roles = [softmax(wg, w) for wg in range(2) for w in range(4)] + [make_k(w) for w in range(4)] + [make_v(w) for w in range(4)]
    roles += [mma(), tensor_cores()]
    kinds = [0] * 4 + [1] * 4 + [2] * 4 + [3] * 4 + [4, 5]
    speed = [10.0 ** rng.uniform(-1.5, 0) for _ in range(6)]
    weight = [speed[k] * rng.uniform(0.5, 1) for k in kinds]
    alive = list(range(len(roles)))
    for _ in range(400000):
        if alive == [len(roles) - 1]:
            return
        i = rng.choices(alive, [weight[j] for j in alive])[0]
        try:
            next(roles[i])
        except StopIteration:
            alive.remove(i)
    raise AssertionError("a role never finished")


STRETCHES = [(1,), (2,), (3,), (16,), (17,), (1, 6), (7, 7), (2, 1, 3), (5, 1, 1, 4), (34,)]


@pytest.mark.parametrize("term", [2, 8])
@pytest.mark.parametrize("stretches", STRETCHES, ids=str)
def test_every_wait_means_its_phase(stretches, term):
    for seed in range(12):
        run_model(stretches, term, seed)


def test_a_wait_for_the_last_tiles_parity_is_caught():
    """The end of a stretch waited for by the last tile's own barrier: where V tiles come slowly a warp
    gets there before the tile two before the last is in O, and that one's parity lets it pass."""
    caught = 0
    for seed in range(60):
        try:
            run_model((16,), 8, seed, last_wait="pv_done")
        except AssertionError as e:
            assert "another phase" in str(e) or "O left" in str(e), e
            caught += 1
    assert caught > 0
