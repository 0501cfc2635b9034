"""The training operators without a GPU: the 64-bit references against differences and torch's own
types, the refusals that happen before any device work, and the build's view of the new sources."""
import ctypes
import inspect

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from kernelforge_b200 import binding as B
from kernelforge_b200 import train
from tests import train_reference as R

vp, i32, i64, sz, f32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_size_t, ctypes.c_float
NULL = vp(0)
SOME = vp(256)   # never dereferenced: the calls below are refused first


def _ids(t, k, g, masked=0.25):
    ids = torch.stack([torch.randperm(256, generator=g)[:k] for _ in range(t)]).to(torch.int32)
    ids[torch.rand(t, generator=g) < masked] = -1
    return ids


# ------------------------------------------------------------- the references --


@pytest.mark.parametrize("align,cut", [(1, 0), (8, 0), (16, 32)])
def test_reference_order_is_a_stable_sort_in_both_directions(align, cut):
    g = torch.Generator().manual_seed(align)
    ids = _ids(37, 5, g)
    experts, offset = 40, 100
    rows = R.worst_rows(37, 5, experts, align) - cut
    pair_row, row_pair, counts, starts = R.order(ids, experts, offset, align, rows)
    local = (ids >= offset) & (ids < offset + experts)
    assert int(counts.sum()) == int(local.sum())
    assert (pair_row[~local] == -1).all()
    for p, r in enumerate(pair_row.reshape(-1).tolist()):
        if r >= 0:
            assert int(row_pair[r]) == p
    assert int((row_pair >= 0).sum()) == int((pair_row >= 0).sum())
    if not cut:
        assert (pair_row[local] >= 0).all()
    for e in range(experts):
        mine = pair_row[ids == e + offset]
        mine = mine[mine >= 0]
        assert (mine[1:] == mine[:-1] + 1).all() and starts[e] % align == 0
        assert not mine.numel() or int(mine[0]) == int(starts[e])


def test_reference_gradients_agree_with_differences():
    g = torch.Generator().manual_seed(3)
    ids = _ids(6, 3, g)
    pair_row, row_pair, _, _ = R.order(ids, 256, 0, 4, R.worst_rows(6, 3, 256, 4))
    rows = torch.randn(row_pair.numel(), 5, generator=g, dtype=torch.float64)
    w = torch.rand(6, 3, generator=g, dtype=torch.float64)
    dout = torch.randn(6, 5, generator=g, dtype=torch.float64)
    drows, dw, _ = R.combine_grads(dout, rows, pair_row, row_pair, w)
    for a, da in ((rows, drows), (w, dw)):
        for i in range(a.numel()):
            step = torch.zeros_like(a)
            step.reshape(-1)[i] = 1e-3

            def f(sign):
                r2, w2 = (rows + sign * step, w) if a is rows else (rows, w + sign * step)
                return float((R.combine(r2, pair_row, w2)[0] * dout).sum())

            assert abs((f(1) - f(-1)) / 2e-3 - float(da.reshape(-1)[i])) < 1e-9   # the sum is linear in each
    u, gate, d = (torch.randn(4, 7, generator=g, dtype=torch.float64) for _ in range(3))
    du, dg, _, _ = R.swiglu_grads(u, gate, d)
    h = 1e-5   # central differences: the third derivative times h^2 / 6, some 1e-10
    assert (du - d * (R.swiglu(u + h, gate) - R.swiglu(u - h, gate)) / (2 * h)).abs().max() < 1e-8
    assert (dg - d * (R.swiglu(u, gate + h) - R.swiglu(u, gate - h)) / (2 * h)).abs().max() < 1e-8
    logits = torch.randn(3, 256, generator=g, dtype=torch.float64)
    ids = _ids(3, 8, g, 0.0)
    ids[1, 2] = -1
    gw = torch.randn(3, 8, generator=g, dtype=torch.float64)
    dl, _ = R.route_grad(logits, ids, gw, 2.5)
    for t in range(3):
        for e in ids[t].tolist() + [int(x) for x in torch.randperm(256, generator=g)[:4]]:
            if e < 0:
                continue
            step = torch.zeros_like(logits)
            step[t, e] = h
            num = ((R.route_weights(logits + step, ids, 2.5) - R.route_weights(logits - step, ids, 2.5)) * gw).sum() / (2 * h)
            assert abs(float(num) - float(dl[t, e])) < 1e-8


def test_reference_8_bit_values_are_within_half_a_step():
    g = torch.Generator().manual_seed(5)
    x = (torch.randn(9, 300, generator=g) * torch.exp(3 * torch.randn(9, 300, generator=g))).to(torch.bfloat16)
    v, e = R.to_8_bits(x)
    for b in range(3):
        c = slice(128 * b, 128 * b + 128)
        err = (v[:, c] - x[:, c].double()).abs()
        assert (err <= torch.maximum(x[:, c].double().abs() * 2.0 ** -4, torch.exp2(e[:, b:b + 1] - 10))).all()


# ------------------------------------------------------------------ refusals --


def _sort(**kw):
    a = dict(x=SOME, dtype=0, stride=64, ids=SOME, T=4, K=2, H=64, E=8, off=0, align=1, R=8, rows=SOME, pr=SOME, rp=SOME,
             cnt=SOME, st=SOME, ws=SOME, wsb=1 << 20)
    a.update(kw)
    f = B.library().kf_sort_tokens
    f.argtypes = [vp, i32, i64, vp, i32, i32, i32, i32, i32, i32, i32, vp, vp, vp, vp, vp, vp, sz, vp]
    return f(a["x"], a["dtype"], a["stride"], a["ids"], a["T"], a["K"], a["H"], a["E"], a["off"], a["align"], a["R"],
             a["rows"], a["pr"], a["rp"], a["cnt"], a["st"], a["ws"], a["wsb"], NULL)


@pytest.mark.parametrize("bad", [dict(T=-1), dict(T=(1 << 24) + 1), dict(K=0), dict(K=17), dict(H=0), dict(H=(1 << 20) + 1),
                                 dict(E=0), dict(E=257), dict(off=-1), dict(off=249), dict(off=2 ** 31 - 1), dict(align=0), dict(align=1025),
                                 dict(align=16, R=24), dict(R=-1), dict(R=(1 << 30) + 1), dict(dtype=3), dict(dtype=-1), dict(stride=-1),
                                 dict(x=NULL), dict(x=vp(257)), dict(rows=vp(258), dtype=2), dict(ids=NULL), dict(rows=NULL), dict(pr=NULL), dict(rp=NULL),
                                 dict(cnt=NULL), dict(st=NULL), dict(T=65536, R=65536 * 2, ws=NULL)])
def test_sort_refuses_bad_arguments_before_device_work(bad):
    assert _sort(**bad) == 1


def test_sort_refuses_a_small_workspace_and_sizes_it():
    lib = B.library()
    lib.kf_sort_workspace_bytes.restype = sz
    lib.kf_sort_workspace_bytes.argtypes = [i32, i32, i32]
    assert lib.kf_sort_workspace_bytes(16, 8, 256) == 0 < lib.kf_sort_workspace_bytes(4096, 8, 256) < lib.kf_sort_workspace_bytes(65536, 8, 256)
    assert lib.kf_sort_workspace_bytes(1, 0, 1) == lib.kf_sort_workspace_bytes(1, 17, 1) == 0
    assert lib.kf_sort_workspace_bytes(1, 1, 257) == lib.kf_sort_workspace_bytes(-1, 1, 1) == 0
    assert _sort(T=65536, K=8, R=65536 * 8, wsb=16) == 2


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_sort_refuses_a_workspace_off_its_alignment(offset):
    assert _sort(T=65536, K=8, R=65536 * 8, ws=vp(256 + offset)) == 1


@pytest.mark.parametrize("bad", [dict(T=-1), dict(K=0), dict(K=17), dict(H=0), dict(dtype=5), dict(R=-1), dict(pr=NULL),
                                 dict(out=NULL), dict(out=vp(257)), dict(rows=NULL), dict(rows=vp(1)), dict(stride=-3)])
def test_combine_refuses_bad_arguments_before_device_work(bad):
    a = dict(rows=SOME, dtype=0, stride=64, R=8, pr=SOME, w=NULL, T=4, K=2, H=64, out=SOME)
    a.update(bad)
    f = B.library().kf_combine_tokens
    f.argtypes = [vp, i32, i64, i32, vp, vp, i32, i32, i32, vp, vp]
    assert f(a["rows"], a["dtype"], a["stride"], a["R"], a["pr"], a["w"], a["T"], a["K"], a["H"], a["out"], NULL) == 1


@pytest.mark.parametrize("bad", [dict(T=-1), dict(K=17), dict(H=0), dict(dtype=-2), dict(R=-1), dict(g=NULL), dict(pr=NULL),
                                 dict(rows=NULL), dict(rp=NULL), dict(stride=-1)])
def test_combine_backward_refuses_bad_arguments_before_device_work(bad):
    a = dict(g=SOME, rows=SOME, dtype=0, stride=64, R=8, pr=SOME, rp=SOME, w=SOME, T=4, K=2, H=64, dr=SOME, dw=SOME)
    a.update(bad)
    f = B.library().kf_combine_backward
    f.argtypes = [vp, vp, i32, i64, i32, vp, vp, vp, i32, i32, i32, vp, vp, vp]
    assert f(a["g"], a["rows"], a["dtype"], a["stride"], a["R"], a["pr"], a["rp"], a["w"], a["T"], a["K"], a["H"], a["dr"],
             a["dw"], NULL) == 1


def test_the_8_bit_entry_points_refuse_bad_arguments_before_device_work():
    lib = B.library()
    lib.kf_pack8.argtypes = [vp, i32, i64, i32, i32, vp, vp, vp]
    lib.kf_restore8.argtypes = [vp, vp, i32, i32, i32, vp, vp, i32, i32, vp, vp]
    lib.kf_swiglu_pack8.argtypes = [vp, i32, i64, i32, i32, vp, vp, vp, vp]
    lib.kf_swiglu_backward8.argtypes = [vp, vp, vp, i32, i64, i32, i32, vp, vp, vp]
    ok = (SOME, 0, 64, 4, 64, SOME, SOME, NULL)
    for i, v in ((0, NULL), (0, vp(33)), (1, 3), (2, -1), (3, -1), (4, 0), (4, (1 << 20) + 1), (5, NULL), (6, NULL)):
        assert lib.kf_pack8(*(v if j == i else a for j, a in enumerate(ok))) == 1
    ok = (SOME, SOME, 0, 4, 64, SOME, SOME, 2, 8, SOME, NULL)
    for i, v in ((0, NULL), (1, NULL), (2, 9), (3, -1), (3, (1 << 24) + 1), (4, 0), (5, NULL), (6, NULL), (7, 0), (7, -1), (7, 17), (8, -1), (9, NULL)):
        assert lib.kf_restore8(*(v if j == i else a for j, a in enumerate(ok))) == 1
    assert lib.kf_restore8(SOME, SOME, 0, 4, 64, NULL, NULL, 0, 5, SOME, NULL) == 1   # without an order the rows stay as many
    ok = (SOME, 0, 128, 4, 64, SOME, SOME, SOME, NULL)
    for i, v in ((0, NULL), (1, -1), (2, -1), (3, -1), (4, 0), (5, NULL), (6, NULL), (7, NULL)):
        assert lib.kf_swiglu_pack8(*(v if j == i else a for j, a in enumerate(ok))) == 1
    ok = (SOME, SOME, SOME, 0, 64, 4, 64, SOME, SOME, NULL)
    for i, v in ((0, NULL), (1, NULL), (2, NULL), (3, 3), (4, -1), (5, -1), (6, 0), (7, NULL)):
        assert lib.kf_swiglu_backward8(*(v if j == i else a for j, a in enumerate(ok))) == 1
    lib.kf_moe_route_backward.argtypes = [vp, vp, vp, i32, f32, vp, vp]
    ok = (SOME, SOME, SOME, 4, 2.5, SOME, NULL)
    for i, v in ((0, NULL), (1, NULL), (2, NULL), (3, -1), (3, (1 << 24) + 1), (5, NULL), (5, vp(8))):
        assert lib.kf_moe_route_backward(*(v if j == i else a for j, a in enumerate(ok))) == 1


def test_cpu_tensors_are_refused():
    x, ids = torch.zeros(2, 16), torch.zeros(2, 1, dtype=torch.int32)
    order = train.TokenOrder(ids, torch.zeros(2, dtype=torch.int32), ids, ids)
    kept = train.Rows8(torch.zeros(2, 16, dtype=torch.float8_e4m3fn), torch.zeros(2, 1, dtype=torch.uint8), torch.float32)
    calls = [lambda: train.route(torch.zeros(2, 256), torch.zeros(256, dtype=torch.bfloat16), 1.0),
             lambda: train.route_backward(torch.zeros(2, 256), ids, torch.zeros(2, 8), 1.0),
             lambda: train.sort_tokens(x, ids, 4), lambda: train.sort_tokens_backward(x, order),
             lambda: train.combine_tokens(x, order), lambda: train.combine_tokens_backward(x, x, order, x),
             lambda: train.pack8(x), lambda: train.restore8(kept), lambda: train.swiglu(x), lambda: train.swiglu_pack8(x),
             lambda: train.swiglu_backward8(kept, x)]
    for call in calls:
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


@pytest.mark.parametrize("n", [1, 64, 100, 128, 129, 384])
def test_rows_in_8_bits_kept_the_other_way_are_refused(n):
    """SwiGLU's blocks begin at each half's first column; where that is elsewhere, the other way's rows are refused."""
    codes = torch.zeros(3, 2 * n, dtype=torch.float8_e4m3fn)
    whole = train.WholeRows8(codes, torch.zeros(3, -(-2 * n // 128), dtype=torch.uint8), torch.float32)
    halves = train.HalvesRows8(codes, torch.zeros(3, 2 * -(-n // 128), dtype=torch.uint8), torch.float32)
    message = "no CPU fallback" if n % 128 == 0 else "begin elsewhere"
    for kept in (halves, halves._replace(dtype=torch.bfloat16)):
        with pytest.raises(RuntimeError, match=message):
            train.restore8(kept)
    with pytest.raises(RuntimeError, match=message):
        train.swiglu_backward8(whole, torch.zeros(3, n))
    for call in (lambda: train.restore8(whole), lambda: train.swiglu_backward8(halves, torch.zeros(3, n)),
                 lambda: train.restore8(train.Rows8(*halves)), lambda: train.swiglu_backward8(train.Rows8(*whole), torch.zeros(3, n))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_tangents_are_refused_before_any_other_check():
    """No operator has a forward-mode rule, so none takes a tensor with a tangent and loses it."""
    x, ids = torch.zeros(2, 16), torch.zeros(2, 1, dtype=torch.int32)
    w, bias, logits = torch.zeros(2, 1), torch.zeros(256, dtype=torch.bfloat16), torch.zeros(2, 256)
    order = train.TokenOrder(ids, torch.zeros(2, dtype=torch.int32), ids, ids)
    kept = train.Rows8(torch.zeros(2, 32, dtype=torch.float8_e4m3fn), torch.zeros(2, 2, dtype=torch.uint8), torch.float32)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        calls = [lambda: train.route(dual(logits), bias, 1.0), lambda: train.route_backward(dual(logits), ids, x, 1.0),
                 lambda: train.route_backward(logits, ids, dual(x), 1.0), lambda: train.sort_tokens(dual(x), ids, 4),
                 lambda: train.sort_tokens_backward(dual(x), order), lambda: train.combine_tokens(dual(x), order),
                 lambda: train.combine_tokens(x, order, dual(w)), lambda: train.combine_tokens_backward(dual(x), x, order, w),
                 lambda: train.combine_tokens_backward(x, dual(x), order, w), lambda: train.combine_tokens_backward(x, x, order, dual(w)),
                 lambda: train.swiglu(dual(x)), lambda: train.swiglu_backward8(kept, dual(x))]
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_every_operator_is_documented():
    for name in ("route", "route_backward", "sort_tokens", "sort_tokens_backward", "combine_tokens",
                 "combine_tokens_backward", "pack8", "restore8", "swiglu", "swiglu_pack8", "swiglu_backward8"):
        assert inspect.getdoc(getattr(train, name)), name
        assert callable(getattr(B.extension(), name)), name
