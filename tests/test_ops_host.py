"""The operators on rows (ps-lite_amd/ops.py) without a GPU: what they refuse, the buckets of the relative position bias against
whole numbers of any length, the generator of the dropout against its published answers, where rows overlap."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from conftest import REPO

AT = [ctypes.c_void_p((i + 1) << 40) for i in range(8)]  # addresses that nothing may be read from: every call is refused


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("ops") / "ops_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-Wno-unknown-pragmas", "-fsanitize=undefined",
                    "-fno-sanitize-recover", os.path.join(REPO, "tests", "ops_check.cc"), "-o", exe], check=True)

    def ask(lines):
        return subprocess.run([exe], input="\n".join(lines) + "\n", capture_output=True, text=True, check=True).stdout.splitlines()
    return ask


# --- buckets -----------------------------------------------------------------------------------------------------

def bucket(rel, buckets, far, two_sided):
    side = buckets // 2 if two_sided else buckets
    d = abs(rel) if two_sided else max(-rel, 0)
    near = side // 2
    n = side - near
    row = d
    if d >= near:
        row = near
        while row < side - 1 and d ** n >= near ** (n - (row + 1 - near)) * far ** (row + 1 - near):
            row += 1
    return side + row if two_sided and rel > 0 else row


@pytest.mark.parametrize("buckets,far,two_sided", [(32, 128, True), (32, 128, False), (2, 2, False), (4, 2, True), (5, 3, True),
                                                   (8, 1000, False), (64, 65, False), (256, 2000, False), (256, 129, True),
                                                   (255, 128, False), (7, 64, False), (16, 1 << 30, True)])
def test_buckets(capi, buckets, far, two_sided):
    ops = _ops()
    reach = list(range(0, min(far, 2000) + 3)) + [1 << 20, (1 << 30) - 1, 1 << 30, 1 << 40, (1 << 63) - 1]
    for d in reach:
        for rel in (d, -d):
            assert ops.relbias_bucket(rel, buckets, far, two_sided) == bucket(rel, buckets, far, two_sided), rel
    assert ops.relbias_bucket(-(1 << 63), buckets, far, two_sided) == bucket(-(1 << 30), buckets, far, two_sided)


def test_borders_that_are_whole_numbers(check):
    # a ratio of 2^4 over 8 steps: every second border is a power of two; of 2^8 over 8: every one
    got = check(["border 32 128 1", "border 16 1024 0", "border 256 1073741824 0", "border 6 192 0"])
    assert got[0].split() == ["12", "16", "23", "32", "46", "64", "91"]
    assert got[1].split() == [str(8 * 2 ** c) if (c * 7) % 8 == 0 else str(int(np.ceil(8 * 2 ** (7 * c / 8)))) for c in range(1, 8)]
    near, far, n = 128, 1 << 30, 128
    for c, d in enumerate(map(int, got[2].split()), 1):
        bound = near ** (n - c) * far ** c
        assert d ** n >= bound > (d - 1) ** n
    assert got[3].split() == ["12", "48"]  # 3 * 4^c


def _ops():
    import __graft_entry__ as graft
    return graft.load_package().ops


@pytest.mark.parametrize("buckets,far,two_sided", [(0, 128, True), (1, 128, False), (3, 128, True), (257, 1000, False), (32, 8, True),
                                                   (32, 16, False), (32, 0, True), (32, (1 << 30) + 1, True)])
def test_settings_without_buckets(capi, buckets, far, two_sided):
    with pytest.raises(capi.PskvError) as e:
        _ops().relbias_bucket(1, buckets, far, two_sided)
    assert e.value.code == capi.EINVAL


# --- the generator -----------------------------------------------------------------------------------------------

def test_published_answers(check):
    """The known answers of Philox4x32-10 that its authors publish with it."""
    got = check(["philox 0 0 0 0 0 0", "philox " + " ".join(["ffffffff"] * 6),
                 "philox 243f6a88 85a308d3 13198a2e 03707344 a4093822 299f31d0"])
    assert got == ["6627e8d5 e169c58d bc57ac4c 9b00dbd8", "408f276d 41c83b0e a20bc7c6 6d5451fd",
                   "d16cfe09 94fdcceb 5001e420 24126ea1"]


# --- where rows overlap ------------------------------------------------------------------------------------------

def test_rows_overlap(check):
    rng = np.random.default_rng(3)
    lines, want = [], []
    for _ in range(4000):
        spans = []
        common = int(rng.integers(1, 9))
        for _ in range(2):
            n, k, size = int(rng.integers(0, 5)), int(rng.integers(0, 5)), int(rng.choice([2, 4]))
            stride = common if rng.random() < 0.7 else int(rng.integers(0, 9))
            spans.append((int(rng.integers(0, 60)) + 100, n, k, stride, size))
        if rng.random() < 0.7:
            spans[1] = spans[1][:4] + spans[0][4:]
        used = [{at + (r * stride + c) * size + byte for r in range(n) for c in range(k) for byte in range(size)}
                for at, n, k, stride, size in spans]
        same_step = spans[0][3] * spans[0][4] == spans[1][3] * spans[1][4]
        lines.append("overlap " + " ".join(str(x) for s in spans for x in s))
        want.append((bool(used[0] & used[1]), same_step and spans[0][3] * spans[0][4] > 0
                     and all(s[3] >= s[2] for s in spans)))
    for line, got, (share, decided) in zip(lines, check(lines), want):
        if share:
            assert got == "1", line  # what shares a byte is never let through
        elif decided:
            assert got == "0", line  # columns of one matrix are not refused


# --- refusals ----------------------------------------------------------------------------------------------------

SORT = dict(bits=64, n=100, E=8, experts=AT[0], order=AT[1], place=AT[2], offsets=AT[3], work=None, room=0)


@pytest.mark.parametrize("change", [dict(bits=16), dict(E=0), dict(E=2049), dict(n=1 << 31), dict(experts=None), dict(order=None),
                                    dict(place=None), dict(offsets=None), dict(n=10000), dict(n=10000, work=AT[4], room=8),
                                    dict(n=10000, work=ctypes.c_void_p((1 << 40) + 2), room=1 << 20), dict(order=AT[0]),
                                    dict(place=ctypes.c_void_p(AT[0].value + 796)), dict(place=AT[1]), dict(offsets=AT[2]),
                                    dict(n=10000, work=AT[3], room=1 << 20)])
def test_sort_refuses(capi, change):
    a = dict(SORT, **change)
    assert capi.load().pskv_route_sort(0, None, a["experts"], a["bits"], a["n"], a["E"], a["order"], a["place"], a["offsets"],
                                       a["work"], a["room"]) == capi.EINVAL
    assert capi.load().pskv_last_error()


def test_rooms(capi):
    ops, lib = _ops(), capi.load()
    assert ops.route_room(0, 8) == 0 and ops.route_room(4096, 2048) == 0
    assert ops.route_room(4097, 8) >= 5 * 9 * 4
    assert lib.pskv_relbias_grad_room(32, 4, 0, 5, 5, 0) == 0 and lib.pskv_relbias_grad_room(32, 4, 1, 5, 5, 0) == 0
    assert lib.pskv_relbias_grad_room(32, 4, 80, 5, 5, 1) > lib.pskv_relbias_grad_room(32, 4, 1, 5, 5, 1)


ROWS = dict(type=0, x=AT[0], x_stride=16, tokens=10, k=16, place=AT[1], choices=2, rows=AT[2], rows_stride=16, n=20, weights=AT[3],
            grad_rows=AT[4], grad_weights=AT[5], grad_stride=16)
BAD_ROWS = [dict(type=3), dict(type=-1), dict(choices=0), dict(k=0), dict(k=(1 << 30) + 1), dict(tokens=1 << 31),
            dict(tokens=1 << 30, choices=2), dict(n=1 << 31), dict(place=None), dict(x=None), dict(x_stride=(1 << 40) + 1)]


def _rows_call(capi, which, a):
    lib = capi.load()
    if which == "rows":
        return lib.pskv_route_rows(0, None, a["type"], a["x"], a["x_stride"], a["tokens"], a["k"], a["place"], a["choices"],
                                   a["rows"], a["rows_stride"], a["n"])
    if which == "sum":
        return lib.pskv_route_sum(0, None, a["type"], a["rows"], a["rows_stride"], a["n"], a["place"], a["weights"], a["choices"],
                                  a["x"], a["x_stride"], a["tokens"], a["k"])
    return lib.pskv_route_sum_grad(0, None, a["type"], a["x"], a["x_stride"], a["tokens"], a["k"], a["rows"], a["rows_stride"],
                                   a["n"], a["place"], a["weights"], a["choices"], a["grad_rows"], a["grad_stride"],
                                   a["grad_weights"])


@pytest.mark.parametrize("which", ["rows", "sum", "grad"])
@pytest.mark.parametrize("change", BAD_ROWS)
def test_rows_refuse(capi, which, change):
    assert _rows_call(capi, which, dict(ROWS, **change)) == capi.EINVAL


@pytest.mark.parametrize("which,change", [
    ("rows", dict(rows=None)), ("rows", dict(rows_stride=15)), ("rows", dict(rows=AT[0])),
    ("rows", dict(rows=ctypes.c_void_p(AT[0].value + 10 * 64 - 4))), ("sum", dict(rows=None)), ("sum", dict(x_stride=15)),
    ("sum", dict(x=AT[2])), ("grad", dict(weights=None)), ("grad", dict(grad_weights=None)), ("grad", dict(grad_rows=None)),
    ("grad", dict(grad_weights=AT[3])), ("grad", dict(grad_stride=15)), ("grad", dict(grad_rows=AT[0])), ("grad", dict(grad_rows=AT[2]))])
def test_rows_refuse_what_they_write(capi, which, change):
    assert _rows_call(capi, which, dict(ROWS, **change)) == capi.EINVAL


def _strides(*by):
    return (ctypes.c_int64 * 3)(*by)


BIAS = dict(type=0, table=AT[0], buckets=32, H=4, far=128, q_first=0, k_first=0, scores=AT[1], in_by=_strides(400, 100, 10), out=AT[2],
            out_by=_strides(400, 100, 10), B=2, Q=10, K=10, grad_table=AT[3], work=AT[4], room=1 << 20)
# a gradient that takes working memory
LARGE = dict(B=40, Q=10, K=10)
BAD_BIAS = [dict(type=7), dict(H=0), dict(H=65536), dict(buckets=1), dict(buckets=300), dict(far=8), dict(q_first=(1 << 60) + 1),
            dict(k_first=-(1 << 60) - 1), dict(B=(1 << 20) + 1), dict(Q=(1 << 20) + 1), dict(K=(1 << 30) + 1),
            dict(in_by=None), dict(in_by=_strides(-1, 100, 10))]


def _bias_call(capi, grad, a):
    lib = capi.load()
    if grad:
        return lib.pskv_relbias_grad(0, None, a["type"], a["scores"], a["in_by"], a["buckets"], a["H"], a["far"], 1, a["q_first"],
                                     a["k_first"], None, a["B"], a["Q"], a["K"], a["grad_table"], a["work"], a["room"])
    return lib.pskv_relbias(0, None, a["type"], a["table"], a["buckets"], a["H"], a["far"], 1, a["q_first"], a["k_first"], None,
                            a["scores"], a["in_by"], a["out"], a["out_by"], a["B"], a["Q"], a["K"])


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("change", BAD_BIAS)
def test_bias_refuses(capi, grad, change):
    assert _bias_call(capi, grad, dict(BIAS, **change)) == capi.EINVAL


@pytest.mark.parametrize("grad,change", [
    (False, dict(table=None)), (False, dict(out=AT[0])), (False, dict(out=None)), (True, dict(LARGE, work=AT[3])), (True, dict(LARGE, work=AT[1])), (False, dict(out_by=None)), (False, dict(out_by=_strides(0, 100, 10))),
    (False, dict(out_by=_strides(400, 100, 9))), (False, dict(out_by=_strides(400, 99, 10))), (False, dict(out_by=_strides(400, 100, 0))),
    (False, dict(out=ctypes.c_void_p(AT[1].value + 4))), (False, dict(out=AT[1], in_by=_strides(0, 100, 10))),
    (True, dict(scores=None)), (True, dict(grad_table=None)), (True, dict(LARGE, work=None)), (True, dict(LARGE, room=100)),
    (True, dict(LARGE, work=ctypes.c_void_p(AT[4].value + 2)))])
def test_bias_refuses_what_it_writes(capi, grad, change):
    assert _bias_call(capi, grad, dict(BIAS, **change)) == capi.EINVAL


DROP = dict(type=1, x=AT[0], x_stride=10, out=AT[1], out_stride=10, n=10, k=10, p=0.5, keys=None, first=0)


@pytest.mark.parametrize("change", [dict(type=9), dict(p=-0.1), dict(p=1.1), dict(p=float("nan")), dict(x=None), dict(out=None),
                                    dict(out_stride=9), dict(k=(1 << 30) + 1), dict(n=(1 << 40) + 1), dict(n=1 << 40, k=8),
                                    dict(keys=AT[2], first=1), dict(out=AT[0], out_stride=11),
                                    dict(out=ctypes.c_void_p(AT[0].value + 2)), dict(x_stride=(1 << 40) + 1)])
def test_dropout_refuses(capi, change):
    a = dict(DROP, **change)
    assert capi.load().pskv_dropout(0, None, a["type"], a["x"], a["x_stride"], a["out"], a["out_stride"], a["n"], a["k"], a["p"], 1,
                                    None, a["keys"], a["first"]) == capi.EINVAL


def test_tensors_that_are_not_on_a_gpu(capi):
    import torch
    ops = _ops()
    x, place, w = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    rows, i32 = torch.zeros(8, 8), dict(dtype=torch.int32)
    calls = [lambda: ops.route_sort(place, 4, torch.zeros(8, **i32), torch.zeros(8, **i32), torch.zeros(5, **i32)),
             lambda: ops.route_rows(x, place, rows), lambda: ops.route_sum(rows, place, x, w),
             lambda: ops.route_sum_grad(x, rows, place, w, rows.clone(), w.clone()),
             lambda: ops.relbias(torch.zeros(32, 2), torch.zeros(2, 4, 4), 128),
             lambda: ops.relbias_grad(torch.zeros(2, 4, 4), torch.zeros(32, 2), 128), lambda: ops.dropout(x, x, 0.5, 1)]
    for call in calls:
        with pytest.raises(ValueError):
            call()
    for call in [lambda: ops.route_rows(np.zeros((4, 8)), place, rows), lambda: ops.dropout(None, x, 0.5, 1)]:
        with pytest.raises(TypeError):
            call()
