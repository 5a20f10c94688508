"""Sliding-window attention, the parts that need no GPU: the geometry the kernels walk, and the refusals of the host."""

import os
import shutil
import subprocess

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


@pytest.mark.skipif(shutil.which("nvcc") is None, reason="needs nvcc to build the host program")
def test_tile_ranges_hold_every_visible_pair(tmp_path):
    exe = str(tmp_path / "window_tiles_check")
    build = subprocess.run(
        ["nvcc", "-std=c++17", "-O2", "-gencode", "arch=compute_100a,code=sm_100a", "-o", exe,
         os.path.join(HERE, "host_checks", "window_tiles_check.cu")],
        capture_output=True, text=True, timeout=600)
    assert build.returncode == 0, build.stderr[-2000:]
    run = subprocess.run([exe], capture_output=True, text=True, timeout=600)
    assert run.returncode == 0, run.stdout[-2000:]
    assert run.stdout.startswith("ok ") and int(run.stdout.split()[1]) > 1_000_000_000


@pytest.mark.parametrize("arguments", (dict(window=0), dict(window=-3), dict(window=2.0), dict(window=True),
                                       dict(window=None), dict(window=4, sinks=-1), dict(window=4, sinks=1.5),
                                       dict(window=4, query_start=-1), dict(window=4, query_start=2**31),
                                       dict(window=4, query_start=torch.zeros(2, dtype=torch.int64)),
                                       dict(window=4, query_start=torch.zeros(3, dtype=torch.int32)),
                                       dict(window=4, query_start=torch.zeros(2, 1, dtype=torch.int32))))
def test_window_arguments_are_refused(arguments):
    from kohakufa_cute import api

    values = dict(dict(sinks=0, query_start=0), **arguments)
    with pytest.raises(ValueError, match="sliding_window_attention"):
        api._window_arguments("sliding_window_attention", 2, torch.device("cpu"), **values)


def test_window_arguments_are_taken():
    from kohakufa_cute import api

    starts = torch.arange(4, dtype=torch.int32)[::2]
    taken, start = api._window_arguments("f", 2, torch.device("cpu"), 7, 0, starts)
    assert start == 0 and taken.is_contiguous() and taken.tolist() == [0, 2]
    assert api._window_arguments("f", 2, torch.device("cpu"), 7, 3, 5) == (None, 5)
    assert api._resolved_scale("f", None, 64) == 0.125
    for scale in (float("nan"), float("inf"), 1e39):
        with pytest.raises(ValueError, match="finite"):
            api._resolved_scale("f", scale, 64)


def test_operands_off_the_gpu_are_refused():
    import kohakufa_cute

    q = torch.zeros(1, 1, 4, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        kohakufa_cute.sliding_window_attention(q, q, q, window=2)
