"""Barrier protocol of the chunk attention tiles (csrc/chunk.cu), checked on the CPU.

The four loader warps (one ring slot each), the MMA issuer (V(j) and the next K
awaited ahead of P, the wait for a tile shared by two row streams made once) and
the two streams' softmax warps are restated as coroutines over mbarriers with the
hardware's parity rule, as the query-tile kernel's are.  Copies land in any order,
MMAs and commits complete in issue order.  No run may stall, no parity wait may be
evaluated outside its phase or the one after, no ring slot or query slot may be
rewritten while an MMA reads it, S(u + 1) may not be issued over a P(u) that has
not been read, and O may not be read before its last product.
"""
import random

import pytest

from tests.test_tc_protocol import Bar

WARPS = 4                                # softmax warps of a stream


class Cta:
    """``ntiles`` key tiles for two row streams (``two``) or two key streams of one row tile."""

    def __init__(self, ntiles, two, rng, late_release=False):
        self.n, self.two, self.rng, self.late_release = ntiles, two, rng, late_release
        b = lambda name, count=1: Bar(name, count)           # noqa: E731
        pair = lambda name, count=1: [b(f"{name}{i}", count) for i in range(2)]   # noqa: E731
        self.k_full, self.k_empty, self.v_full, self.v_empty = map(pair, ("KF", "KE", "VF", "VE"))
        self.s_full, self.pv_done = pair("S"), pair("PV")
        self.p_full, self.q_full = pair("P", WARPS), pair("Q", WARPS)
        self.count = [ntiles, ntiles] if two else [(ntiles + 1) // 2, ntiles // 2]
        self.copies, self.pipe = [], []
        self.ring = {"K": [None, None], "V": [None, None]}
        self.reading = {"K": [0, 0], "V": [0, 0], "Q": [0, 0]}
        self.products = [0, 0]           # P.V completed per stream
        self.p_ready = [-1, -1]          # last P written per stream
        self.s_written = [-1, -1]        # last S completed per stream
        self.finished = 0

    def tile(self, t, u):
        return u if self.two else 2 * u + t

    def parity_ok(self, bar, phase):
        assert bar.done in (phase, phase + 1), f"{bar.name}: waiting for phase {phase} at {bar.done}"
        return bar.done % 2 != phase % 2

    # -- roles -----------------------------------------------------------------------
    def loader(self, ring, slot):
        full = (self.k_full if ring == "K" else self.v_full)[slot]
        empty = (self.k_empty if ring == "K" else self.v_empty)[slot]
        last = None
        for j in range(slot, self.n, 2):
            if j >= 2:
                yield ("wait", empty, j // 2 - 1)
            assert self.reading[ring][slot] == 0, f"{ring} slot refilled while an MMA reads it"
            self.ring[ring][slot] = None
            self.copies.append((full, ring, slot, j))
            last = j
            yield ("step",)
        if last is not None:
            yield ("wait", full, last // 2)

    def issue_s(self, t, u):
        j = self.tile(t, u)
        q = t if self.two else 0
        assert self.ring["K"][j % 2] == j, f"S reads K({j}) from a slot holding {self.ring['K'][j % 2]}"
        self.reading["K"][j % 2] += 1
        self.reading["Q"][q] += 1
        self.pipe.append(("s", t, u, j % 2, q))
        self.pipe.append(("commit", self.s_full[t]))
        if not self.two or t == 1 or self.late_release:
            self.pipe.append(("commit", self.k_empty[j % 2]))

    def issue_pv(self, t, u):
        j = self.tile(t, u)
        assert self.ring["V"][j % 2] == j and self.p_ready[t] == u
        self.reading["V"][j % 2] += 1
        self.pipe.append(("pv", t, u, j % 2))
        if u == self.count[t] - 1:
            self.pipe.append(("commit", self.pv_done[t]))
        if not self.two or t == 1:
            self.pipe.append(("commit", self.v_empty[j % 2]))

    def inputs(self, t, u):
        if self.two and t == 1:
            return
        j = self.tile(t, u)
        yield ("wait", self.v_full[j % 2], j // 2)
        if u + 1 < self.count[t]:
            k = self.tile(t, u + 1)
            yield ("wait", self.k_full[k % 2], k // 2)

    def issuer(self):
        for t in range(2):
            if self.count[t]:
                j = self.tile(t, 0)
                yield ("wait", self.q_full[t if self.two else 0], 0)
                yield ("wait", self.k_full[j % 2], j // 2)
                self.issue_s(t, 0)
        yield from self.inputs(0, 0)
        for u in range(self.count[0]):
            for t in range(2):
                if u >= self.count[t]:
                    continue
                yield ("wait", self.p_full[t], u)
                self.issue_pv(t, u)
                if u + 1 < self.count[t]:
                    self.issue_s(t, u + 1)
                yield ("step",)
                nt, nu = (1, u) if t == 0 and u < self.count[1] else (0, u + 1)
                if nu < self.count[nt]:
                    yield from self.inputs(nt, nu)
        for j in range(max(0, self.n - 2), self.n):
            yield ("wait", self.k_empty[j % 2], j // 2)
            yield ("wait", self.v_empty[j % 2], j // 2)

    def softmax(self, t):
        if self.two or t == 0:
            for _ in range(WARPS):
                self.q_full[t].arrive()
        for u in range(self.count[t]):
            yield ("wait", self.s_full[t], u)
            assert self.s_written[t] == u and self.products[t] == u, "S seen before the product ahead of it"
            self.p_ready[t] = u
            for _ in range(WARPS):
                self.p_full[t].arrive()
            yield ("step",)
        if self.count[t]:
            yield ("wait", self.pv_done[t], 0)
        joined = not self.two and self.n > 1
        if joined and t == 0:
            yield ("wait", self.pv_done[1], 0)
        assert self.products[t] == self.count[t]
        if self.two or t == 0:           # rows leave through the query slot
            assert self.reading["Q"][t] == 0, "the epilogue stages over queries an MMA reads"
            if joined:
                assert self.products[1] == self.count[1]
        self.finished += 1

    # -- scheduler -------------------------------------------------------------------
    def complete(self):
        op = self.pipe.pop(0)
        if op[0] == "commit":
            op[1].arrive()
        elif op[0] == "s":
            _, t, u, slot, q = op
            assert self.products[t] == u, "S overwrites a P that has not been read"
            self.s_written[t] = u
            self.reading["K"][slot] -= 1
            self.reading["Q"][q] -= 1
        else:
            _, t, u, slot = op
            self.products[t] += 1
            self.reading["V"][slot] -= 1

    def run(self):
        agents = [self.loader(r, s) for r in "KV" for s in range(2)] + [self.issuer(), self.softmax(0), self.softmax(1)]
        waits = [("step",)] * len(agents)
        live = list(range(len(agents)))
        speed = {i: self.rng.choice([0.02, 1.0, 1.0, 8.0]) for i in [*live, "copy", "pipe"]}
        for _ in range(100000):
            ready = [i for i in live if waits[i][0] == "step" or self.parity_ok(*waits[i][1:])]
            ready += ["copy"] * bool(self.copies) + ["pipe"] * bool(self.pipe)
            if not ready:
                assert not live, f"deadlock: {[waits[i] for i in live]}"
                return
            i = self.rng.choices(ready, weights=[speed[r] for r in ready])[0]
            if i == "copy":
                bar, ring, slot, tile = self.copies.pop(self.rng.randrange(len(self.copies)))
                self.ring[ring][slot] = tile
                bar.arrive()
            elif i == "pipe":
                self.complete()
            else:
                try:
                    waits[i] = next(agents[i])
                except StopIteration:
                    live.remove(i)
        raise AssertionError("no progress bound reached")


@pytest.mark.parametrize("two", [False, True], ids=["key streams", "row streams"])
@pytest.mark.parametrize("ntiles", [1, 2, 3, 4, 5, 9])
def test_chunk_barrier_protocol(ntiles, two):
    for seed in range(300):
        cta = Cta(ntiles, two, random.Random(seed * 100 + ntiles))
        cta.run()
        assert cta.finished == 2


def test_the_model_catches_an_early_release():
    """A K slot released by the first of two row streams is refilled, or counted, too early."""
    caught = 0
    for seed in range(100):
        try:
            Cta(5, True, random.Random(seed), late_release=True).run()
        except AssertionError:
            caught += 1
    assert caught > 50
