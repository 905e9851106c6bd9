"""The stages of the fp8 product's few-rows kernel, on the host: their number,
and its barriers in a model that runs the threads in random orders."""
import ctypes
import random

import pytest

SIZES = (16, 32, 64, 96, 128)
ACC = 4  # accumulators


def all_stages(sampler_lib):
    f = sampler_lib.lib().bm_detail_fp8_stages
    f.argtypes = [ctypes.c_int, ctypes.c_int]
    return {(nb, kb): f(nb, kb) for nb in SIZES for kb in range(1, 129)}


def test_stages_are_even_and_fit(sampler_lib):
    """Tiles of 128 + nb rows of 128 bytes, the scales of kb blocks and 256
    bytes of barriers in 220 KB, whatever d up to 16384; the sums that a
    cluster exchanges (nb * 512 bytes) over the stages."""
    for (nb, kb), n in all_stages(sampler_lib).items():
        stage = (128 + nb) * 128
        assert n % 2 == 0 and 2 <= n <= 12, (nb, kb, n)
        assert n * stage + 1024 + 256 + kb * nb * 4 <= 220 * 1024, (nb, kb, n)
        assert nb * 512 <= n * stage


class Barrier:
    """Phases completed; a wait for a parity passes when the phase before the
    current one has it."""

    def __init__(self):
        self.phases = 0

    def passes(self, parity):
        return (self.phases - 1) % 2 == parity % 2


def overwrites(stages, blocks, rng):
    """Runs two copying threads, two MMA threads and the promotion in a random
    order with random delays; True where a copy goes to a stage whose block
    has not been read, or an MMA reads a block that is not there."""
    full, empty = [Barrier() for _ in range(stages)], [Barrier() for _ in range(stages)]
    accf, acce = [Barrier() for _ in range(ACC)], [Barrier() for _ in range(ACC)]
    holds = [None] * stages   # the block that lies in a stage, unread
    landed = [None] * stages
    flights = []

    def copier(first):
        for j in range(first, blocks, 2):
            s, use = j % stages, j // stages
            while not empty[s].passes(use + 1):
                yield "waits"
            if holds[s] is not None:
                yield "bad"
            holds[s] = j
            flights.append([j, s])
            yield "ran"

    def mma(first):
        for j in range(first, blocks, 2):
            s, use, b, turn = j % stages, j // stages, j % ACC, j // ACC
            while not acce[b].passes(turn + 1):
                yield "waits"
            while not full[s].passes(use):
                yield "waits"
            if landed[s] != j:
                yield "bad"
            yield "ran"
            holds[s] = None
            empty[s].phases += 1
            accf[b].phases += 1
            yield "ran"

    def promotion():
        for j in range(blocks):
            b = j % ACC
            while not accf[b].passes(j // ACC):
                yield "waits"
            yield "ran"
            acce[b].phases += 1
            yield "ran"

    def copies():
        while True:
            if flights:
                # one block's copies may be far slower than the next ones'
                j, s = flights.pop(rng.randrange(len(flights)) if rng.random() < 0.2 else -1)
                landed[s] = j
                full[s].phases += 1
                yield "ran"
            else:
                yield "waits"

    threads = [copier(0), copier(1), mma(0), mma(1), promotion(), copies()]
    idle = 0
    while len(threads) > 1:
        t = rng.choice(threads)
        for _ in range(rng.choice((1, 1, 4, 20))):
            state = next(t, "done")
            if state == "bad":
                return True
            if state == "done":
                threads.remove(t)
                break
            idle = idle + 1 if state == "waits" else 0
            if idle > 5000:
                return True  # (nobody goes on)
    return False


def test_the_model_sees_five_stages_fail():
    rng = random.Random(1)
    assert any(overwrites(5, 120, rng) for _ in range(40))


def test_no_stage_is_overwritten(sampler_lib):
    for stages in sorted(set(all_stages(sampler_lib).values())):
        rng = random.Random(stages)
        for _ in range(60):
            assert not overwrites(stages, 120, rng), stages
