"""The tcgen05 GEMV's waits for its stages, with loads that land in any order: a model of its roles over
barriers that, as the hardware's, show a waiter the parity of their phase and nothing else."""
import os
import random
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flashbfp_b200", "csrc", "gemv_tc.cu")


class Barrier:
    def __init__(self):
        self.done = 0                                  # phases completed

    def passes(self, parity):                          # mbarrier.try_wait.parity
        return (self.done & 1) != parity


def _constants():
    text = open(SOURCE).read()
    stages, dq = (int(re.search(rf"constexpr int {n} = (\d+);", text).group(1)) for n in ("kStages", "kDqPerQuarter"))
    full = re.search(r"constexpr int kFull = ([^;]+);", text)
    return stages, dq, eval(full.group(1), {"kStages": stages, "kDqPerQuarter": dq}) if full else stages


def run(stages, dq, full, units, seed):
    """Units that a role read before they had landed."""
    rng = random.Random(seed)
    bars = [Barrier() for _ in range(full)]
    issued, landed = 0, set()
    at = list(range(dq))                               # each dequantiser's next unit (of one lane quarter)
    reading, stored, outliers, mma = [None] * dq, set(), 0, 0
    early = []
    slow = {i: rng.random() < 0.2 for i in range(units)}
    while mma < units or outliers < units:
        do = rng.randrange(4 + dq)
        if do == 0 and issued < units:                 # the producer: a stage is free when all roles are done with it
            old = issued - stages
            if old < 0 or (old in stored and old < mma and old < outliers):
                issued += 1
        elif do == 1:                                  # a load lands
            flying = [i for i in range(issued) if i not in landed]
            if flying:
                i = rng.choice(flying)
                if not slow[i] or rng.random() < 0.05:
                    landed.add(i)
                    bars[i % full].done += 1
        elif do == 2 and mma in stored:
            mma += 1
        elif do == 3 and outliers < units and bars[outliers % full].passes(outliers // full & 1):
            if outliers not in landed:
                early.append(("outliers", outliers))
            outliers += 1
        elif do >= 4:
            d = do - 4
            if reading[d] is None:
                if at[d] < units and bars[at[d] % full].passes(at[d] // full & 1):
                    if at[d] not in landed:
                        early.append(("dequantiser", at[d]))
                    reading[d] = at[d]
            elif reading[d] < dq or reading[d] - dq < mma:          # its tensor-memory slots are free
                stored.add(reading[d])
                reading[d], at[d] = None, at[d] + dq
        if early:
            break
    return early


def test_no_unit_is_read_before_it_has_landed():
    stages, dq, full = _constants()
    for seed in range(60):
        assert not run(stages, dq, full, 60, seed), seed


def test_a_barrier_per_stage_is_not_enough():
    """The model tells: five barriers for three dequantisers that take turns."""
    assert any(run(5, 3, 5, 60, seed) for seed in range(60))
    assert not any(run(6, 3, 6, 60, seed) for seed in range(30))
