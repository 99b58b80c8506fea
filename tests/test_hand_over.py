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
