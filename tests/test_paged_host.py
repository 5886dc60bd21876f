"""CPU checks of the paged batch: refusals, index rules and launch plan (paged_check.cpp, with g++
and its sanitizers), and the entry points before llmp_init."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from llmplayer_amd import _lib
from tests import paged_cases as pc

HERE = os.path.dirname(os.path.abspath(__file__))


def test_host_side(tmp_path):
    exe = str(tmp_path / "paged_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=address,undefined",
                    "-fno-sanitize-recover=all", "-I", os.path.join(HERE, "..", "include"),
                    os.path.join(HERE, "paged_check.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


def test_calls_before_init():
    h = C.c_uint64()
    calls = {"llmp_paged_create": (1, 4, 16, 64, 1, 64, 0, C.byref(h)), "llmp_paged_bytes": (1, C.byref(h)),
             "llmp_paged_bind": (1, 256), "llmp_paged_planes": (1, 0, None, None, None, None),
             "llmp_paged_tables": (1, 1, 0, 1) + (4,) * 11 + (0,),
             "llmp_paged_append": (1, 0, 1, 4, 4, 0, 4, 64, 4, 64, 4, 64, 4, 64, 0),
             "llmp_paged_attn": (1, 0, 1, 1, 0, 0, 4, 4, 4, 16, 64, 0, 16, 64, 0)}
    for name, args in calls.items():
        assert _lib.status(name, *args) == 3, name   # LLMP_ERR_NOT_INIT


def test_reference_tables_by_hand():
    """The tests' own reference on a step small enough to follow: pages of 16, sequences of 16, 5, 40
    and 0 rows that take 1, 3, end, and 17."""
    blocks = np.full((4, 4), -1, np.int32)
    blocks[0, :1], blocks[1, :1], blocks[2, :3] = 7, 8, [9, 3, 4]
    free = np.array([5, 6, 0, 1, -1, -1, -1, -1, -1, -1], np.int32)
    r = pc.reference_tables([16, 5, 40, 0], [1, 3, -1, 17], free, 4, blocks, 16, 64, 1, 25, 10)
    # returned: 3, 4 (the shared block 9 stays); popped from the top: 4, then 3 and 1
    assert r["status"] == 0 and r["n_free"] == 3
    assert r["free"][:6].tolist() == [5, 6, 0, 1, 3, 4]
    assert r["blocks"][0].tolist() == [7, 4, -1, -1] and r["blocks"][3].tolist() == [3, 1, -1, -1]
    assert r["len"].tolist() == [17, 8, 0, 17] and r["seq_start"].tolist() == [0, 1, 4, 4, 21]
    assert r["positions"].tolist() == [16, 5, 6, 7] + list(range(17)) + [-1] * 4
    assert r["slots"].tolist() == [64, 133, 134, 135] + list(range(48, 64)) + [16] + [-1] * 4


@pytest.mark.parametrize("change,status", [({"len": [70, 5, 40, 0]}, -1), ({"len": [-1, 5, 40, 0]}, -1),
                                           ({"grow": [60, 3, -1, 17]}, -1), ({"tokens": 20}, -2), ({"n_free": 0}, 1)])
def test_reference_tables_refuse(change, status):
    a = {"len": [16, 5, 40, 0], "grow": [1, 3, -1, 17], "tokens": 25, "n_free": 4, **change}
    blocks, free = np.zeros((4, 4), np.int32), np.arange(10, dtype=np.int32)
    r = pc.reference_tables(a["len"], a["grow"], free, a["n_free"], blocks, 16, 64, 1, a["tokens"], 10)
    assert r["status"] == status and not r["seq_start"].any() and (r["positions"] == -1).all()
    assert r["len"].tolist() == a["len"] and np.array_equal(r["blocks"], blocks) and r["n_free"] == a["n_free"]
