"""Beam search's floor for a wave's vectors of logits, the code that the kernel runs, on the host: whatever the logits, no
more vectors are put beside each other than there is room for, and the best logits are in them."""

import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOM = 128  # vectors of a wave that there is room for
HERE = Path(__file__).resolve().parent


@pytest.fixture(scope="module")
def choose(tmp_path_factory):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no host compiler")
    out = tmp_path_factory.mktemp("beam_floor") / "beam_floor_host.so"
    subprocess.run([compiler, "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", str(HERE / "beam_floor_host.cpp"), "-o", str(out)],
                   check=True)
    f = ctypes.CDLL(str(out)).beam_floor_host
    f.restype = ctypes.c_int
    f.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_uint32, ctypes.c_uint32, ctypes.c_int, ctypes.c_int,
                  ctypes.POINTER(ctypes.c_uint32), ctypes.POINTER(ctypes.c_int)]

    def call(tops, lowest, highest, most):
        least, count = ctypes.c_uint32(), ctypes.c_int()
        tops = np.ascontiguousarray(tops)
        place = f(tops.ctypes.data, tops.shape[0], int(lowest), int(highest), most, ROOM, ctypes.byref(least), ctypes.byref(count))
        return least.value, count.value, place
    return call


def ordered(x):
    """The order of fp32 as whole numbers, -0 as 0."""
    u = (np.asarray(x, np.float32) + np.float32(0)).view(np.uint32)
    return np.where(u >> 31, ~u, u | np.uint32(0x80000000)).astype(np.uint32)


def wave_logits(shape, rng, vectors):
    """[vectors of a lane][64 lanes][8], as the kernel's wave has them."""
    n = (vectors, 64, 8)
    flat = np.zeros(n, np.float32)
    if shape == "normal":
        return rng.standard_normal(n).astype(np.float32)
    if shape == "rounded":
        return np.round(3 * rng.standard_normal(n)).astype(np.float32)
    if shape == "comb":  # the largest all in a few lanes
        return (4.0 * (np.arange(64) == rng.integers(64))[None, :, None] + rng.random(n)).astype(np.float32)
    if shape == "alike":
        return flat
    kind, count = shape
    where = rng.permutation(flat.size)[:count]
    if kind == "allowed":  # all others -inf
        flat[:] = -np.inf
        flat.ravel()[where] = rng.standard_normal(count)
    elif kind == "filled":  # all others a large negative number
        flat[:] = -1.0e4
        flat.ravel()[where] = rng.standard_normal(count)
    elif kind == "above":  # alike, but for a few
        flat.ravel()[where] = 1.0 + rng.integers(0, 3, count)
    return flat


SHAPES = ["normal", "rounded", "comb", "alike"] + [(kind, count) for kind in ("allowed", "filled", "above") for count in (0, 1, 3, 12, 60, 63, 64, 200)]


@pytest.mark.parametrize("vectors", [1, 2, 4, 8])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_no_more_than_there_is_room_for(choose, shape, vectors):
    rng = np.random.default_rng(vectors)
    for most in (1, 2, 3, 5, 8, 16, 33, 63, 64):
        for _ in range(4):
            x = ordered(wave_logits(shape, rng, vectors))
            tops = x.max(2)
            lanes = np.sort(tops.max(0))[::-1]
            lowest = lanes[most - 1]  # as many lanes reach it
            least, count, place = choose(tops, lowest, tops.max(), most)
            assert count == int((tops >= least).sum())
            assert least >= lowest and place < ROOM
            if count > ROOM:  # none is put anywhere, the wave's logits are looked through from the lowest floor on
                assert place == -1 and least == lowest
            else:
                assert place == count - 1 and count >= most
                assert int((x >= least).sum()) >= most  # so the best `most` are among them
