"""The hand-overs between the warps of attention's dq kernel, on the CPU: every order of events is gone through."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("hand_over") / "model")
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-o", exe, os.path.join(HERE, "hand_over.cpp")])
    return lambda turns: subprocess.run([exe, str(turns)], capture_output=True, text=True, timeout=300)


def test_every_order_of_events_ends(model):
    run = model(3)
    assert run.returncode == 0, run.stdout


@pytest.mark.parametrize("turns", [1, 2], ids=["sums_on_one_barrier", "rows_on_one_barrier"])
def test_a_single_barrier_is_told_from_its_last_time_by_luck(model, turns):
    """The model tells: with one barrier a warp that looks late waits for a phase that never comes."""
    run = model(turns)
    assert run.returncode == 1, run.stdout


def test_every_wait_of_a_role_is_bounded():
    """A warp that gives up leaves its group: no role may wait for the others in a way that has no limit.  What is left of
    the CTA's own barriers stands in front of the roles, and behind them, where every warp comes."""
    csrc = os.path.join(HERE, os.pardir, "cswap_b200", "csrc")
    text = "".join(open(os.path.join(csrc, f)).read() for f in ("attention_kernels.cu", "tensor_core.cuh"))
    code = "\n".join(line.split("//")[0] for line in text.splitlines())
    assert "bar.sync" not in code and "barrier.sync" not in code and "barrier.cta" not in code
    kernels = code.count("__global__") - 1  # the one that adds up parts has no roles
    assert kernels == 3 and code.count("__syncthreads()") == kernels + 1  # and once in what they all end with
