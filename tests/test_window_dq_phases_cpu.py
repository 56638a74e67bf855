"""The hand-over of a unit's query and dO rows in the window's dQ kernel, played through on the CPU.

A wait by parity tells two neighbouring phases apart and no more: who waits has to have seen the phase before.  Two pairs of warpgroups take a
unit's items in turn, the pair with the first item moves the unit's rows out of shared memory, and a unit of one item leaves the other
pair without any sign of it.  So units use two barriers in turn.  Here the loading warp, the issuing warp, the tensor core, TMA and the two
pairs are agents that run in any order; how many barriers there are and how they are waited for is read off the kernel's source."""
import random
import re

import pytest

from test_dependent_launch_cpu import functions, read


class Barrier:
    def __init__(self, count):
        self.count, self.left, self.phase = count, count, 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.left, self.phase = self.count, self.phase + 1

    def passes(self, parity):
        return (self.phase & 1) != parity


def play(totals, sets, seed):
    """Runs the units through; returns the faults seen (rows read that are not the unit's, agents that never end)."""
    rng, faults = random.Random(seed), []
    bar = {n: Barrier(c) for n, c in dict(qdo_full0=1, qdo_full1=1, ops_ready=1, ops_free0=1, ops_free1=1, rows_read=1, s_full0=1, s_full1=1, s_free0=1, s_free1=1, dp_full0=1,
                                          dp_full1=1, ds_ready0=1, ds_ready1=1, acc_full0=1, acc_full1=1, acc_empty=1).items()}
    rows, flights, tensor = [None], [], []            # what the tile in shared memory holds; loads under way; commits in issue order
    wait = lambda name, parity: (name, parity)        # noqa: E731

    def of_unit(name, u):                             # barrier and parity of unit u's phase, of `sets` barriers in turn
        return f"{name}{u % sets}", (u // sets) & 1

    def loads():
        for u in range(len(totals)):
            yield wait("rows_read", (u & 1) ^ 1)
            rows[0] = ("on its way", u)
            flights.append(u)
            yield None

    def issue():
        items = [(u, i, n) for u, n in enumerate(totals) for i in range(n)]

        def s(j):
            u, i, _ = items[j]
            if j >= 2:
                yield wait(f"s_free{j % 2}", ((j // 2) & 1) ^ 1)
            if i == 0:
                yield wait("ops_ready", u & 1)
            tensor.append(f"s_full{j % 2}")

        def dp(j):
            u, i, n = items[j]
            tensor.append(f"dp_full{j % 2}")
            if i == n - 1:
                tensor.append(of_unit("ops_free", u)[0])
        for j in range(min(2, len(items))):
            yield from s(j)
            dp(j)
        for it, (u, i, n) in enumerate(items):
            early = it + 2 < len(items) and items[it + 2][1] > 0
            if early:
                yield from s(it + 2)
            if i == 0:
                yield wait("acc_empty", (u & 1) ^ 1)
            yield wait(f"ds_ready{it % 2}", (it // 2) & 1)
            if i == n - 1:
                tensor.append(f"acc_full{it & 1}")
            if it + 2 < len(items):
                if not early:
                    yield from s(it + 2)
                dp(it + 2)

    def pair(p):
        it0 = drains = 0
        pending = False
        for u, total in enumerate(totals):
            mover = p == (it0 & 1)
            if mover:
                yield wait(*of_unit("qdo_full", u))
                if u > 0:
                    yield wait(*of_unit("ops_free", u - 1))
                if rows[0] != ("there", u):
                    faults.append((u, rows[0]))
                yield None
                if rows[0] != ("there", u):
                    faults.append((u, rows[0]))
                bar["ops_ready"].arrive()
                bar["rows_read"].arrive()
            if pending:
                yield wait(f"acc_full{p}", drains & 1)
                drains += 1
                bar["acc_empty"].arrive()
                pending = False
            for i in range((it0 + p) & 1, total, 2):
                it = it0 + i
                yield wait(f"s_full{it % 2}", (it // 2) & 1)
                bar[f"s_free{it % 2}"].arrive()
                yield wait(f"dp_full{it % 2}", (it // 2) & 1)
                bar[f"ds_ready{it % 2}"].arrive()
            it0 += total
            pending = p == ((it0 - 1) & 1)
        if pending:
            yield wait(f"acc_full{p}", drains & 1)

    agents = {"loads": loads(), "issue": issue(), "pair 0": pair(0), "pair 1": pair(1)}
    speed = {n: rng.choice([1, 1, 8]) for n in (*agents, "tma", "tensor")}
    at = {n: None for n in agents}
    for _ in range(20000):
        ready = [n for n in agents if at[n] is None or bar[at[n][0]].passes(at[n][1])]
        ready += ["tma"] * bool(flights) + ["tensor"] * bool(tensor)
        if not ready:
            break
        n = rng.choices(ready, [speed[x] for x in ready])[0]
        if n == "tma":
            rows[0] = ("there", flights.pop(0))
            bar[of_unit("qdo_full", rows[0][1])[0]].arrive()
        elif n == "tensor":
            bar[tensor.pop(0)].arrive()
        else:
            try:
                at[n] = next(agents[n])
            except StopIteration:
                del agents[n]
    return faults + [("never ends", n) for n in agents]


def sets_in_the_source():
    (_, body), = functions(read("window_sm100.cu"))[0]["window_dq_sm100_kernel"]
    two = ["mbar_wait(smem_u32(&sm->qdo_full[u & 1]), (u >> 1) & 1,", "mbar_wait(smem_u32(&sm->ops_free[(u - 1) & 1]), ((u - 1) >> 1) & 1,",
           "qb = smem_u32(&sm->qdo_full[u & 1]);", "mma_commit(smem_u32(&sm->ops_free[c.u & 1]));"]
    assert len(re.findall(r"mbar_wait\(smem_u32\(&sm->(?:qdo_full|ops_free)", body)) == 2
    return 2 if all(body.count(x) == 1 for x in two) else 1


def cases():
    rng = random.Random(1)
    return [[1] * 9, [1, 1, 1, 2, 1, 1, 3, 1, 1], [2] * 6, [3] * 6, [5, 1, 1, 1, 4, 1, 1]] + [[rng.choice([1, 1, 2, 3, 4]) for _ in range(8)] for _ in range(5)]


@pytest.mark.parametrize("totals", cases())
def test_every_unit_is_computed_from_its_own_rows(totals):
    sets = sets_in_the_source()
    for seed in range(300):
        assert play(totals, sets, seed) == [], seed


def test_the_play_shows_what_one_barrier_does():
    assert any(play([1] * 9, 1, seed) for seed in range(300))
    assert not any(play([2] * 6, 1, seed) for seed in range(300))
