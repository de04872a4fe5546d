"""The attention kernel's ring of K and V tiles as a model (CPU): barriers with phases, read by
parity as the device reads them, copies that land in any order, and roles that run in any
interleaving.

fu_attention.cu: warp 8 loads K_0, V_0, K_1, V_1, .. into a ring of STAGES; warp 9 issues the
products, S(j + 1) behind O(j), and gives a stage back when a product is through with it; warps 10
and 11 look at the V tiles that lie at a mask's edge.  Whether they too give the stages back is read
from the source: the barrier's count is 1 without them, 3 with them.  Checked: every role finds in a
stage the tile that it waited for, a tile at an edge is multiplied only when both warps have been
through it, and everything ends."""

import random
import re
from pathlib import Path

import pytest

SOURCE = (Path(__file__).resolve().parent.parent / "flash_ulysses_b200" / "csrc"
          / "fu_attention.cu").read_text()
STAGES = int(re.search(r"constexpr int STAGES = (\d+);", SOURCE).group(1))
EMPTY_COUNT = int(re.search(r"mbar_init\(b\.kv_empty \+ 8 \* s, (\d+)\);", SOURCE).group(1))
CLEANERS = 2


class Fault(Exception):
    pass


class Barrier:
    """Phases that complete after `count` arrivals; passed() is a wait on a phase's parity."""

    def __init__(self, count):
        self.count, self.left, self.phase = count, count, 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.left, self.phase = self.count, self.phase + 1

    def passed(self, parity):
        return self.phase & 1 != parity


class Ring:
    def __init__(self, tiles, edges, empty_count):
        self.tiles, self.edges = tiles, edges
        self.gives_back = empty_count == 1 + CLEANERS
        self.full = [Barrier(1) for _ in range(STAGES)]
        self.empty = [Barrier(empty_count) for _ in range(STAGES)]
        self.clean = [Barrier(CLEANERS) for _ in range(STAGES)]
        self.holds = [None] * STAGES          # the load whose bytes are in a stage
        self.been = {}                        # V tile -> cleaning warps that went through it
        self.flying = []                      # loads that have not landed

    def expect(self, load, who):
        if self.holds[load % STAGES] != load:
            raise Fault(f"{who} finds {self.holds[load % STAGES]} where it waited for {load}")

    def loader(self):
        for load in range(2 * self.tiles):
            s = load % STAGES
            yield lambda s=s, load=load: self.empty[s].passed((load // STAGES & 1) ^ 1)
            self.holds[s] = None
            self.flying.append(load)

    def memory(self, rnd):
        for _ in range(2 * self.tiles):
            yield lambda: bool(self.flying)
            load = self.flying.pop(rnd.randrange(len(self.flying)))
            self.holds[load % STAGES] = load
            self.full[load % STAGES].arrive()

    def mma(self):
        def full(load):
            return lambda: self.full[load % STAGES].passed(load // STAGES & 1)

        yield full(0)
        self.expect(0, "S 0")
        self.empty[0].arrive()
        for j in range(self.tiles):
            v, k = 2 * j + 1, 2 * j + 2
            if j in self.edges:
                yield lambda j=j: self.clean[j % STAGES].passed(j // STAGES & 1)
                if self.been.get(j) != CLEANERS:
                    raise Fault(f"tile {j} multiplied after {self.been.get(j)} cleaning warps")
            else:
                yield full(v)
            self.expect(v, f"O {j}")
            yield lambda: True
            self.expect(v, f"O {j}")
            self.empty[v % STAGES].arrive()
            if j + 1 < self.tiles:
                yield full(k)
                self.expect(k, f"S {j + 1}")
                self.empty[k % STAGES].arrive()

    def cleaner(self):
        for j in range(self.tiles):
            for load in (2 * j, 2 * j + 1):
                if load == 2 * j and not self.gives_back:
                    continue
                s = load % STAGES
                yield lambda s=s, load=load: self.full[s].passed(load // STAGES & 1)
                if load == 2 * j + 1:
                    self.expect(load, "a cleaning warp")
                    if j in self.edges:
                        yield lambda: True            # it takes a while
                        self.expect(load, "a cleaning warp")
                    self.been[j] = self.been.get(j, 0) + 1
                    self.clean[j % STAGES].arrive()
                if self.gives_back:
                    self.empty[s].arrive()


def run(seed, empty_count):
    """One interleaving; every role runs at a pace of its own, some hardly ever."""
    rnd = random.Random(seed)
    tiles = rnd.choice([1, 2, 3, 4, 5, 9, 20, 41])
    edges = {j for j in range(tiles) if rnd.random() < rnd.choice([0.0, 0.1, 0.5, 1.0])}
    edges.add(tiles - 1)
    ring = Ring(tiles, edges, empty_count)
    roles = [ring.loader(), ring.memory(rnd), ring.mma()]
    roles += [ring.cleaner() for _ in range(CLEANERS)]
    pace = [rnd.choice([1.0, 0.3, 0.05, 0.01]) for _ in roles]
    waits = [next(r, None) for r in roles]
    while any(w is not None for w in waits):
        ready = [i for i, w in enumerate(waits) if w is not None and w()]
        if not ready:
            raise Fault(f"stuck: {[i for i, w in enumerate(waits) if w is not None]}")
        i = rnd.choices(ready, [pace[i] for i in ready])[0]
        waits[i] = next(roles[i], None)
    assert ring.been == {j: CLEANERS for j in range(tiles)}


def test_every_role_gets_the_tile_that_it_waits_for():
    for seed in range(3000):
        run(seed, EMPTY_COUNT)


@pytest.mark.parametrize("what", ["stuck", "finds", "multiplied"])
def test_model_detects_cleaning_warps_that_do_not_give_stages_back(what):
    """Each way in which it went wrong where the products alone gave a stage back: the call that
    never ends, a warp that looks at another tile, and a product with a tile not looked at."""
    for seed in range(20000):
        try:
            run(seed, 1)
        except Fault as fault:
            if what in str(fault):
                return
    raise AssertionError("not found")
