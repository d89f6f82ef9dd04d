"""The waits of the prompts' attention for its ring of keys and values (heads of 136 to 256 values), with loads
that land in any order: a model of its roles over barriers that, as the hardware's, show a waiter the parity
of their phase and nothing else. What a role reads has to have landed."""
import os
import random
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flashbfp_b200", "csrc", "prompt_attn.cu")
SLOTS, PER = 10, 4


def _source():
    """Whether the values' role waits for a step's scores first, and how many barriers tell that values are here."""
    text = open(SOURCE).read()
    values = text[text.index("if (of_scores) {"):text.index("} else if (warp >= kMma) {")].split("} else {")[1]
    after_scores = values.find("ctl.s_full[0][g & 1]") in range(0, values.find("ctl.full[slot]"))
    return after_scores, 2 if re.search(r"\bv_here\[2\]\[2\]", text) else 1


def run(after_scores, here, tiles, seed, looks=0.4):
    """The first reads that came before their unit; ``looks``: the share of steps whose values the softmax looks at."""
    rng = random.Random(seed)
    order, where, g = [], {}, 0                        # units as they are loaded: (kind, step, part)
    for blocks in tiles:
        k = min(2, blocks)
        seq = [("k", j) for j in range(k)]
        for j in range(blocks):
            seq.append(("v", j))
            if j + 2 < blocks:
                seq.append(("k", j + 2))
        for kind, j in seq:
            for p in range(PER):
                where[kind, g + j, p] = len(order)
                order.append((kind, g + j, p))
        g += blocks
    steps = g
    cut = [rng.random() < looks for _ in range(steps)]
    done = {}                                          # phases completed, by barrier
    landed, released, early = set(), set(), []

    def wait(name, phase):
        return lambda: (done.get(name, 0) & 1) != (phase & 1)

    def full(u):
        return wait(("full", u % SLOTS), u // SLOTS)

    def arrive(name):
        done[name] = done.get(name, 0) + 1

    def read(who, u):
        if u not in landed:
            early.append((who, order[u]))

    def scores():
        for g in range(steps):
            if g >= 2:
                yield wait(("o", g & 1), (g >> 1) - 1)
            for p in range(PER):
                u = where["k", g, p]
                yield full(u)
                read("scores", u)
                released.add(u)
            arrive(("s", g & 1))

    def values():
        for g in range(steps):
            if after_scores:
                yield wait(("s", g & 1), g >> 1)
            yield full(where["v", g, 0])
            arrive(("here", g % here))
            yield wait(("p", g & 1), g >> 1)
            for p in range(PER):
                u = where["v", g, p]
                if p:
                    yield full(u)
                read("values", u)
                released.add(u)
            arrive(("o", g & 1))

    def softmax():
        for g in range(steps):
            yield wait(("s", g & 1), g >> 1)
            if cut[g]:
                yield wait(("here", g % here), g // here)
                for p in range(PER):
                    yield full(where["v", g, p])
                    read("softmax", where["v", g, p])
            arrive(("p", g & 1))
        for b in (0, 1):
            if steps > b:
                yield wait(("o", b), (steps - 1 - b) >> 1)

    roles = [f() for f in (scores, values, softmax)]
    waits = [next(r) for r in roles]
    issued = 0
    slow = rng.random() * 0.3
    late = [rng.random() < slow for _ in order]
    for _ in range(200000):
        if all(w is None for w in waits) or early:
            return early
        do = rng.randrange(5)
        if do == 0:
            if issued < len(order) and (issued < SLOTS or issued - SLOTS in released):
                issued += 1
        elif do == 1:
            flying = [u for u in range(max(0, issued - SLOTS), issued) if u not in landed]
            if flying:
                u = rng.choice(flying)
                if not late[u] or rng.random() < 0.05:
                    landed.add(u)
                    arrive(("full", u % SLOTS))
        elif waits[do - 2] is not None and waits[do - 2]():
            waits[do - 2] = next(roles[do - 2], None)
    raise AssertionError("a role waits for good")


TILES = ([1], [2, 1], [16], [1, 1, 5, 2, 1, 9], [10, 10, 3])


def test_products_take_what_has_landed():
    after_scores, here = _source()
    for tiles in TILES:
        for seed in range(80):
            early = run(after_scores, here, tiles, seed, looks=0.0)
            assert not early, (tiles, seed, early)


def test_softmax_looks_at_what_has_landed():
    after_scores, here = _source()
    for tiles in TILES:
        for seed in range(80):
            early = run(after_scores, here, tiles, seed)
            assert not early, (tiles, seed, early)


def test_the_model_tells():
    """Values waited for without their step's scores, or one barrier that the softmax looks at now and then."""
    assert any(run(False, 2, TILES[2], seed, looks=0.0) for seed in range(300))
    assert any(run(True, 1, TILES[2], seed) for seed in range(300))
