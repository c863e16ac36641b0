"""What the operators on rows refuse of buffers that lie upon each other, without a GPU: no call here names a device that exists, so
one that is not refused ends with PSKV_EHIP, and nothing is ever launched."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from conftest import REPO


NOWHERE = -1  # a device that does not exist
AT = [(i + 1) << 40 for i in range(8)]
p = ctypes.c_void_p


def refused(capi, code):
    assert code in (capi.EINVAL, capi.EHIP)
    return code == capi.EINVAL


# --- tokens by expert --------------------------------------------------------------------------------------------

T, CHOICES, K, ROWS = 10, 2, 16, 20  # float32: 10 rows of 64 bytes, 80 bytes of places or weights, 20 sorted rows


def rows(capi, x=AT[0], place=AT[1], to=AT[2], to_stride=K):
    return refused(capi, capi.load().pskv_route_rows(NOWHERE, None, 0, p(x), K, T, K, p(place), CHOICES, p(to), to_stride, ROWS))


@pytest.mark.parametrize("offset", [-76, 0, 64, 20 * 64 - 4])
def test_rows_refuse_their_places(capi, offset):
    assert rows(capi, place=AT[2] + offset)


@pytest.mark.parametrize("offset", [-80, 20 * 64])
def test_rows_beside_their_places(capi, offset):
    assert not rows(capi, place=AT[2] + offset)
    # 80 bytes of places between rows 160 bytes apart
    assert not rows(capi, place=AT[2] + 64, to_stride=40) and rows(capi, place=AT[2] + 60, to_stride=40) and rows(capi, place=AT[2] + 84, to_stride=40)


def back(capi, answers=AT[0], place=AT[1], weights=AT[2], to=AT[3], to_stride=K):
    return refused(capi, capi.load().pskv_route_sum(NOWHERE, None, 0, p(answers), K, ROWS, p(place), p(weights), CHOICES, p(to), to_stride, T, K))


@pytest.mark.parametrize("what", ["place", "weights"])
@pytest.mark.parametrize("offset", [-76, 0, 64, 10 * 64 - 4])
def test_sum_refuses_its_places_and_weights(capi, what, offset):
    assert back(capi, **{what: AT[3] + offset})


@pytest.mark.parametrize("what", ["place", "weights"])
def test_sum_beside_its_places_and_weights(capi, what):
    assert not back(capi, **{what: AT[3] - 80}) and not back(capi, **{what: AT[3] + 640})
    assert not back(capi, to_stride=40, **{what: AT[3] + 64}) and not back(capi, weights=None) and not back(capi, place=AT[2])


GRAD = dict(grad=AT[0], answers=AT[1], place=AT[2], weights=AT[3], grad_rows=AT[4], grad_weights=AT[5], stride=K)


def back_grad(capi, **change):
    a = dict(GRAD, **change)
    return refused(capi, capi.load().pskv_route_sum_grad(NOWHERE, None, 0, p(a["grad"]), K, T, K, p(a["answers"]), K, ROWS, p(a["place"]),
                                                         p(a["weights"]), CHOICES, p(a["grad_rows"]), a["stride"], p(a["grad_weights"])))


@pytest.mark.parametrize("what,size", [("place", 80), ("weights", 80), ("grad", 640), ("answers", 1280)])
@pytest.mark.parametrize("written,room", [("grad_rows", 1280), ("grad_weights", 80)])
def test_gradients_refuse_what_they_read(capi, what, size, written, room):
    for offset in (4 - size, 0, 64, room - 4):
        assert back_grad(capi, **{what: GRAD[written] + offset})
    for offset in (-size, room):
        assert not back_grad(capi, **{what: GRAD[written] + offset})


def test_gradients_refuse_each_other(capi):
    for offset in (-76, 0, 1276):
        assert back_grad(capi, grad_weights=AT[4] + offset)
    for offset in (-80, 1280):
        assert not back_grad(capi, grad_weights=AT[4] + offset)
    # between rows 160 bytes apart
    for what in ("place", "weights", "grad_weights"):
        assert not back_grad(capi, stride=40, **{what: AT[4] + 64}) and back_grad(capi, stride=40, **{what: AT[4] + 60})


# --- dropout -----------------------------------------------------------------------------------------------------

def dropout(capi, x=AT[0], out=AT[1], keys=None, step=None, stride=16):
    """10 rows of 16 float32."""
    return refused(capi, capi.load().pskv_dropout(NOWHERE, None, 0, p(x), stride, p(out), stride, 10, 16, 0.5, 1, p(step), p(keys), 0))


@pytest.mark.parametrize("what,size", [("keys", 80), ("step", 8)])
def test_dropout_refuses_its_keys_and_step(capi, what, size):
    for offset in (8 - size, 0, 64, 632):
        assert dropout(capi, **{what: AT[1] + offset})
        assert dropout(capi, x=AT[1], **{what: AT[1] + offset})  # in place, too
    for offset in (-size, 640):
        assert not dropout(capi, **{what: AT[1] + offset})
    assert not dropout(capi, stride=40, **{what: AT[1] + 64})  # between rows 160 bytes apart
    assert not dropout(capi, **{what: AT[0]})                  # both are read


# --- the gradient of the position bias ---------------------------------------------------------------------------

@pytest.fixture(scope="module")
def entry(tmp_path_factory):
    folder = tmp_path_factory.mktemp("entry")
    exe, obj = str(folder / "entry_check"), str(folder / "entry_check.o")
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    subprocess.run([hipcc, "-x", "hip", "--offload-arch=gfx950", "--offload-host-only", "-O0", "-std=c++17", "-I" + os.path.join(REPO, "include"),
                    "-c", os.path.join(REPO, "tests", "entry_check.cc"), "-o", obj], check=True, capture_output=True)
    # (there is no code for a device to be found)
    subprocess.run(["g++", "-no-pie", obj, "-Wl,--unresolved-symbols=ignore-all", "-o", exe], check=True)
    return exe


@pytest.mark.parametrize("shape", [(0, 10, 10), (2, 0, 10), (2, 10, 0)])
def test_empty_gradient_with_working_memory(capi, entry, shape):
    """A gradient of nothing has no strides to be looked at."""
    done = subprocess.run([entry] + [str(x) for x in shape], capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout.split() == [str(capi.EHIP)], done


def strides(*by):
    return (ctypes.c_int64 * 3)(*by)


BIAS_GRAD = dict(grad=AT[0], by=(400, 100, 10), at=None, B=2, Q=10, K=10, table=AT[1], work=AT[2], size=4)


def bias_grad(capi, **change):
    """4 heads, 32 buckets: a gradient of 512 bytes."""
    a = dict(BIAS_GRAD, **change)
    types = {4: 0, 2: 1}
    return refused(capi, capi.load().pskv_relbias_grad(NOWHERE, None, types[a["size"]], p(a["grad"]), strides(*a["by"]), 32, 4, 128, 1, 0, 0, p(a["at"]),
                                                       a["B"], a["Q"], a["K"], p(a["table"]), p(a["work"]), 1 << 20))


def test_bias_gradient_refuses_what_it_reads(capi):
    size = 2 * 400 * 4
    for offset in (-508, 0, 1600, size - 4):
        assert bias_grad(capi, table=AT[0] + offset)
    for offset in (-512, size):
        assert not bias_grad(capi, table=AT[0] + offset)
    for offset in (-8, 0, 504):  # 16 bytes of positions
        assert bias_grad(capi, at=AT[1] + offset)
    for offset in (-16, 512):
        assert not bias_grad(capi, at=AT[1] + offset)


def test_bias_gradient_and_its_working_memory(capi):
    lib = capi.load()
    many = dict(B=40)  # takes working memory, with positions and without
    room = lib.pskv_relbias_grad_room(32, 4, 40, 10, 10, 1)
    assert room >= 512
    for offset in (-312, 0, room - 8):  # 320 bytes of positions
        assert bias_grad(capi, at=AT[2] + offset, **many)
    for offset in (-320, room):
        assert not bias_grad(capi, at=AT[2] + offset, **many)


def test_bias_gradient_beside_what_it_reads(capi):
    """512 bytes between the sequences, heads or queries of a gradient, whose dimensions lie in any order."""
    rng = np.random.default_rng(5)
    for _ in range(3000):
        B, Q, K, size = int(rng.integers(1, 4)), int(rng.integers(1, 4)), int(rng.integers(1, 40)), int(rng.choice([2, 4]))
        n, by, reach = {0: B, 1: 4, 2: Q}, [0, 0, 0], K
        for d in rng.permutation(3):
            by[d] = int(reach + rng.choice([0, 3, 700]))
            reach = (n[d] - 1) * by[d] + reach
        if rng.random() < 0.2:
            by[int(rng.integers(0, 3))] = 0  # (of a gradient that is expanded)
        starts = np.add.outer(np.add.outer(np.arange(B) * by[0], np.arange(4) * by[1]), np.arange(Q) * by[2]).ravel() * size
        offset = 4 * int(rng.integers(-140, reach * size // 4 + 10))
        share = bool(np.any((starts < offset + 512) & (starts + K * size > offset)))
        got = bias_grad(capi, B=B, Q=Q, K=K, size=size, by=by, table=AT[0] + offset)
        assert got == share, (B, Q, K, size, by, offset)
