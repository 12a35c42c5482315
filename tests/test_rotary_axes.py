"""Copies of ``RotaryAxes``: a module that holds its axes is deep-copied, pickled and sent to other processes."""
from __future__ import annotations

import copy
import ctypes
import gc
import pickle
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from min_fa3_demo_b200 import _cabi, rotary

SECTIONS = (16, 24, 24)


def make():
    return rotary.RotaryAxes.from_sections(SECTIONS, 1e6, adjacent=True)


def is_whole(axes):
    """What the library would read through the address, which has to be the object's own memory."""
    assert axes._at == ctypes.addressof(axes._c)
    there = _cabi.RotaryAxes.from_address(axes._at)
    return (list(there.turn) == [rotary._turn(1e6 ** (-i / 64)) for i in range(64)] and there.pairs == axes.pairs == 64
            and list(there.axis) == [a for a, n in enumerate(SECTIONS) for _ in range(n)] and there.axes == axes.axes == 3 and there.adjacent == 1)


class Holder(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.axes = make()


@pytest.mark.parametrize("how", ["copy", "deepcopy", "pickle", "module"])
def test_copies_have_memory_of_their_own(how):
    axes = make()
    if how == "module":
        holder = Holder()
        other = copy.deepcopy(holder).axes
        del holder
    else:
        other = {"copy": copy.copy, "deepcopy": copy.deepcopy, "pickle": lambda a: pickle.loads(pickle.dumps(a))}[how](axes)
    assert type(other) is rotary.RotaryAxes and is_whole(axes)
    del axes
    gc.collect()
    others = [rotary.RotaryAxes([0.5] * 8) for _ in range(50)]     # whatever takes the original's place
    assert is_whole(other) and len(others) == 50


def test_another_process():
    code = ("import ctypes, pickle, sys; a = pickle.loads(sys.stdin.buffer.read());"
            "assert a._at == ctypes.addressof(a._c); print(list(a._c.turn)[63], a.pairs, a.axes)")
    root = Path(__file__).resolve().parents[1]
    done = subprocess.run([sys.executable, "-c", code], input=pickle.dumps(make()), capture_output=True, cwd=root, timeout=300)
    assert done.returncode == 0, done.stderr.decode()[-500:]
    assert done.stdout.decode().split() == [str(rotary._turn(1e6 ** (-63 / 64))), "64", "3"]
