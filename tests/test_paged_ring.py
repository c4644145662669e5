"""The few-rows kernel's ring of tiles, and the many-rows kernel's last product, as models on the CPU: which tile a team of warps finds in a stage, for copies that land in
any order.  The number of stages and the parities that a team waits for are read from the kernel's source."""
import os
import random
import re

import pytest

SOURCE = os.path.join(os.path.dirname(__file__), "..", "saetta_macqwen_b200", "csrc", "paged_attend.cu")


class Barrier:
    """An mbarrier seen by its waiters: a wait for a parity holds while the phase under way is of the other one."""

    def __init__(self):
        self.phase = 0

    def passed(self, parity):
        return self.phase & 1 != parity


def kernel():
    text = open(SOURCE).read()
    stages = int(re.search(r"kStages = (\d+);", text).group(1))
    loop = text[text.index("if ((g & 1) != team) continue;"):text.index("const int32_t key0 = int32_t(kt * kTile + sub")]
    own = "mbar_wait(&full[g % L::kFull], (g / L::kFull) & 1, abort_flag)" in loop
    return stages, int(re.search(r"kFull = (\d+) \* kStages;", text).group(1)) if own else 1


def stale_reads(stages, per_stage, tiles, seed, slow):
    """Runs producer, copies and two teams in a random order of steps; `slow` is the tile whose copy lands only when nothing else can move.
    per_stage: barriers of landed tiles that a stage's uses go round."""
    rng = random.Random(seed)
    bars = stages * per_stage
    full, empty = [Barrier() for _ in range(bars)], [Barrier() for _ in range(stages)]
    holds = [None] * stages  # the tile whose bytes are whole in a stage
    issued, flying, at = 0, [], [0, 1]
    while min(at) < tiles:
        moves = []
        if issued < tiles and empty[issued % stages].passed((issued // stages & 1) ^ 1):
            moves.append(("issue", issued))
        moves += [("land", g) for g in flying if g != slow]
        moves += [("read", team) for team, g in enumerate(at) if g < tiles and full[g % bars].passed(g // bars & 1)]
        if not moves:
            moves = [("land", g) for g in flying]
        if not moves:
            return "stuck"
        what, i = rng.choice(moves)
        if what == "issue":
            holds[i % stages] = None
            flying.append(i)
            issued += 1
        elif what == "land":
            flying.remove(i)
            holds[i % stages] = i
            full[i % bars].phase += 1
        else:
            g = at[i]
            if holds[g % stages] != g:
                return g, holds[g % stages]
            empty[g % stages].phase += 1
            at[i] += 2
    return None


@pytest.mark.parametrize("slow", range(12))
def test_no_team_reads_a_tile_before_it_landed(slow):
    stages, per_stage = kernel()
    for seed in range(200):
        assert stale_reads(stages, per_stage, 31, seed, slow) is None, (stages, per_stage, seed)


def test_the_model_finds_a_missed_use_of_a_stage():
    """With one barrier for a stage and an odd number of stages, a team returns to a stage by the same parity."""
    assert any(stale_reads(5, 1, 31, seed, 5) for seed in range(200))
    assert not any(stale_reads(4, 1, 31, seed, slow) for seed in range(50) for slow in range(8))


PREFILL = os.path.join(os.path.dirname(SOURCE), "paged_prefill.cu")


def early_ends(order, tiles, seed):
    """The many-rows kernel's barrier for a row tile's last product (two arrivals: the issuing warp's and the products' own, which comes late), for items of
    the given numbers of tiles.  `order`: whether the warp arrives before or after it waited for the item before to be read.  Returns the items whose
    output is read before their products are done."""
    rng = random.Random(seed)
    count, phase, done, read = 0, 0, 0, 0  # of the barrier; products done and outputs read, in items
    pending, early = [], []  # commits under way
    steps = []
    for i, n in enumerate(tiles):
        for t in range(n):
            last, first = t + 1 == n, t == 0
            if last and order == "before":
                steps.append(("arrive", i))
            if first:
                steps.append(("wait read", i))
            if last and order == "after":
                steps.append(("arrive", i))
        steps.append(("commit", i))
    at = 0
    while read < len(tiles):
        moves = ["land"] * bool(pending)
        if at < len(steps) and (steps[at][0] != "wait read" or read >= steps[at][1]):
            moves.append("warp")
        if phase > read:
            moves.append("read")
        assert moves, "stuck"
        move = rng.choice(moves)
        if move == "warp":
            what, i = steps[at]
            at += 1
            if what == "commit":
                pending.append(i)
            count += what == "arrive"
        elif move == "land":
            done = pending.pop(0) + 1
            count += 1
        else:
            early += [read] * (done <= read)
            read += 1
        if count == 2:
            count, phase = 0, phase + 1
    return early


def test_a_row_tile_is_read_after_its_last_product():
    text = open(PREFILL).read()
    value_products = text[text.index("---- value products"):]
    order = "before" if value_products.index("mbar_arrive(o_final)") < value_products.index("PP_WAIT(o_empty") else "after"
    for seed in range(200):
        tiles = [random.Random(seed + 1000).choice((1, 1, 2, 5)) for _ in range(12)]
        assert not early_ends(order, tiles, seed), (order, seed)


def test_the_model_finds_an_arrival_that_comes_too_early():
    assert any(early_ends("before", [1, 1, 1, 2, 1], seed) for seed in range(200))
