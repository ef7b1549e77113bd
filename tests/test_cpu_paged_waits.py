"""The ring of the paged attention (voxgen_b200/csrc/paged_attention.cuh) played through on the CPU, with bounded waits that run
out at any time: no stage is filled while a copy into it is in flight, no warp reads a stage that has not landed, every warp
comes to its end, and no copy is in flight when the block ends."""
import random

import pytest

from voxgen_b200._build import CSRC


class Broken(Exception):
    pass


class Barrier:
    """An mbarrier: a phase completes when its arrivals and its copies' bytes are in."""

    def __init__(self, count):
        self.count, self.left, self.copies, self.phase, self.early = count, count, 0, 0, False

    def _check(self):
        if self.left == 0 and self.copies == 0:
            self.left, self.phase = self.count, self.phase + 1

    def arrive(self, n=1, copies=0):
        if n > self.left:
            raise Broken("more arrivals than a phase takes")
        self.left -= n
        self.copies += copies
        self._check()

    def land(self):
        self.copies -= 1
        self._check()

    def passed(self, parity):
        return self.phase & 1 != parity


class Block:
    """One CTA: W consumer warps, W copying lanes (each has its own stages), pieces of (blocks, tiles)."""

    def __init__(self, rng, warps, stages, pieces, risk, mended):
        self.rng, self.W, self.S, self.pieces, self.risk, self.mended = rng, warps, stages, pieces, risk, mended
        self.full = [Barrier(1) for _ in range(stages)]
        self.empty = [Barrier(warps) for _ in range(stages)]
        self.holds = [None] * stages          # the number whose copy has landed there
        self.flying = {}                      # stage: number
        self.gave_up = False
        self.late = False                     # a wait for copies in flight ran out
        self.names = [0] * warps              # named barriers passed by each consumer
        self.rounds = [-(-b // warps) * warps for b, _ in pieces]

    def wait(self, bar, parity):
        """Yields until the phase has passed; may run out whenever it has not."""
        while not bar.passed(parity):
            if self.rng.random() < self.risk or self.stuck:
                return False
            yield
        return True

    def lane(self, lane):
        """A copying lane; all of them leave a round together."""
        n0, issued = 0, lane
        for piece, (blocks, _) in enumerate(self.pieces):
            for r in range(0, self.rounds[piece], self.W):
                n = n0 + r + lane
                stage, turn = n % self.S, n // self.S
                ok = True
                if turn:
                    ok = yield from self.wait(self.empty[stage], (turn - 1) & 1)
                if ok:
                    if stage in self.flying:
                        raise Broken("a stage is filled while a copy into it is in flight")
                    copy = r + lane < blocks
                    self.holds[stage] = n if not copy else None
                    if copy:
                        self.flying[stage] = n
                    self.full[stage].arrive(1, int(copy))
                    issued = n + self.W
                self.votes.setdefault((piece, r), []).append(ok)
                while len(self.votes[piece, r]) < self.W:
                    yield
                if not all(self.votes[piece, r]):
                    self.gave_up = True
                    yield from self.drain(issued)
                    return
                yield
            n0 += self.rounds[piece]
        yield from self.drain(issued)

    def drain(self, issued):
        if self.mended:
            for k in range(1, self.S // self.W + 1):
                n = issued - k * self.W
                if n >= 0 and not (yield from self.wait(self.full[n % self.S], n // self.S & 1)):
                    self.late = True
                    return

    def meet(self, warp):
        self.names[warp] += 1
        while min(self.names) < self.names[warp]:
            yield

    def consumer(self, warp):
        n0, stopped = 0, False
        for piece, (blocks, tiles) in enumerate(self.pieces):
            teams = self.W // tiles
            yield from self.meet(warp)
            stopped |= self.gave_up
            for b in range(warp // tiles, self.rounds[piece], teams):
                n = n0 + b
                stage = n % self.S
                if not stopped and not (yield from self.wait(self.full[stage], n // self.S & 1)):
                    stopped = self.gave_up = True
                if not stopped:
                    if self.holds[stage] != n:
                        raise Broken("a stage is read that has not landed")
                    yield
                    if self.holds[stage] != n or stage in self.flying:
                        raise Broken("a stage changes while it is read")
                if not (self.mended and stopped):
                    self.empty[stage].arrive(teams)
                yield
            n0 += self.rounds[piece]
            yield from self.meet(warp)
        if stopped and not self.mended:
            for n in range(n0 - min(n0, self.S), n0):
                if not (yield from self.wait(self.full[n % self.S], n // self.S & 1)):
                    self.late = True
                    return

    def run(self):
        self.votes, self.stuck, self.speed = {}, False, self.rng.choice([0.02, 0.1, 0.5])
        live = [self.lane(i) for i in range(self.W)] + [self.consumer(i) for i in range(self.W)]
        idle = 0
        while live:
            before = (self.names[:], [b.phase for b in self.full + self.empty], len(live))
            for x in self.rng.sample(live, len(live)):
                if self.rng.random() < 0.7:
                    try:
                        next(x)
                    except StopIteration:
                        live.remove(x)
            for stage in list(self.flying):
                if self.rng.random() < self.speed:
                    self.holds[stage] = self.flying.pop(stage)
                    self.full[stage].land()
            idle = idle + 1 if before == (self.names[:], [b.phase for b in self.full + self.empty], len(live)) else 0
            self.stuck = idle > 50            # nothing moves but waits: their time runs out
            if idle > 500:
                raise Broken("a warp waits for good")
        if self.flying and not self.late:
            raise Broken("a copy is in flight when the block ends")
        return self.gave_up


def play(seed, mended):
    rng = random.Random(seed)
    warps, stages = rng.choice([(12, 24), (12, 48), (4, 4), (4, 8)])
    pieces = [(rng.randint(1, 3 * stages), rng.choice([1, 2, 4])) for _ in range(rng.randint(1, 4))]
    return Block(rng, warps, stages, pieces, rng.choice([0, 0.001, 0.01, 0.1]), mended).run()


def test_the_ring_where_waits_run_out():
    gave_up = sum(play(seed, True) for seed in range(300))
    assert gave_up > 100


def test_releases_of_stages_that_were_not_awaited_are_found():
    """The play has teeth: with consumers that go on releasing stages after a wait ran out, it finds the faults of that."""
    broken = 0
    for seed in range(300):
        try:
            play(seed, False)
        except Broken:
            broken += 1
    assert broken > 10


def test_the_kernel_keeps_the_rules_of_the_play():
    text = (CSRC / "paged_attention.cuh").read_text()
    assert text.count("mbar_arrive_count(&empty[stage], teams)") == 1
    assert "if (lane == 0 && !stopped) mbar_arrive_count(&empty[stage], teams)" in text
    assert text.count("mbar_wait_bounded(&full[") == 2      # a consumer's, and the copying warp's at its end
    assert "const uint32_t n = issued - k * W;" in text and "issued = n + W;" in text
    assert text.count("mbar_wait_bounded") == 3


@pytest.mark.parametrize("warps,stages", [(12, 24), (12, 48), (4, 4), (4, 8)])
def test_a_lane_has_its_own_stages(warps, stages):
    """Numbers lane, lane + W, ... fall on stages that no other lane's do, kStages / W of them."""
    for lane in range(warps):
        mine = {n % stages for n in range(lane, 10 * stages, warps)}
        assert len(mine) == stages // warps and all(s % warps == lane for s in mine)
