"""The bounded barrier waits of the tensor-core kernels, on CPU.

A wait that runs out must end the kernel, not hang it.  Where a whole warp waits, each lane polls for itself; lanes that left
with different answers would meet again only in instructions that need all of them (elect.sync, warp barriers, tcgen05 loads,
stores and allocations), and stand there.  So the kernels wait per lane only where a single lane walks the loop, and
with a vote (`mbar_wait_warp`, `mbar_wait_cluster_warp`) everywhere else."""

import random
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "cute-kernels_b200" / "csrc"
KERNELS = ["gemm_tc.cu", "gemm_tc2.cu", "gemm_fp8.cu", "gemm_wgrad.cu", "fp8_few.cu"]


def _enclosing(text: str, at: int) -> list[str]:
    """What stands before the braces that are open at `at`."""
    heads, start = [], 0
    for i in range(at):
        if text[i] == "{":
            heads.append(text[start:i])
            start = i + 1
        elif text[i] == "}":
            heads.pop()
            start = i + 1
        elif text[i] == ";":
            start = i + 1
    return heads


@pytest.mark.parametrize("name", KERNELS)
def test_waits_of_single_lanes_stand_where_a_single_lane_runs(name):
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    calls = [m for m in re.finditer(r"\bmbar_wait(_cluster)?(_warp)?\(", text)]
    assert calls
    for call in calls:
        single = any(re.search(r"\blane == 0\b|\btid == 0\b", head) for head in _enclosing(text, call.start()))
        whole_warp = call.group(2) is not None
        line = text[text.rfind("\n", 0, call.start()) + 1 : text.find("\n", call.start())].strip()
        assert single != whole_warp, f"{name}: {line}"


def test_wrappers_vote():
    for name, of in (("gemm_tc.cuh", "mbar_wait"), ("gemm_pair.cuh", "mbar_wait_cluster")):
        text = (CSRC / name).read_text()
        body = text[text.index(f"bool {of}_warp(") :]
        assert f"return __all_sync(0xffffffffu, {of}(bar, parity, abort_flag, status));" in body[: body.index("}")]


def _poll(lanes: int, completes: int, limit: int, rng: random.Random) -> list[bool]:
    """mbar_wait of each lane, on a common clock: the lanes poll at times of their own, and the first to pass the limit
    sets the abort flag."""
    answers: list[bool | None] = [None] * lanes
    abort, clock = False, 0
    while None in answers:
        clock += 1
        order = [i for i in range(lanes) if answers[i] is None and rng.random() < 0.5]
        rng.shuffle(order)
        for i in order:
            if clock >= completes:
                answers[i] = True
            elif abort or clock > limit:
                abort, answers[i] = True, False
    return [bool(a) for a in answers]


def test_lanes_can_part_and_the_vote_keeps_them_together():
    rng = random.Random(0)
    parted = 0
    for _ in range(200):
        answers = _poll(32, completes=13, limit=10, rng=rng)
        parted += len(set(answers)) > 1
        together = [all(answers)] * 32  # what __all_sync gives each lane
        assert len(set(together)) == 1 and (not together[0] or all(answers))
    assert parted > 0  # why the vote is there
    assert all(_poll(32, completes=5, limit=10, rng=rng)) and not any(_poll(32, completes=10**6, limit=10, rng=rng))
