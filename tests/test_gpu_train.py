"""The training operators on a B200 against their definitions in 64 bits (``train_reference``).

Tolerances.  A result is one fp32 computation rounded once to its type: half a step of the type
(``R.half_step``) on top of the fp32 operations' own 2^-24 each.  A sum of n terms is off by at
most n * 2^-24 times the sum of their magnitudes; a dot product over the width passes every term
through at most 8 additions per 256 columns of one warp, 5 in the warp and 16 across warps.  A
sigmoid from expf (2 ulp), an addition and a division is within 2^-21, and the products around
it add a few 2^-24: 2^-20 of the magnitudes in all.  For 16-bit types e^-g is 2^y of the rounded
y = -g log2 e: an error of half an ulp in y, |g| log2 e 2^-24, is one of |g| 2^-24 in e^-g, which the
sigmoid passes on at most whole.  Where e^-g leaves fp32's normal numbers
(g below -87.3, 1 + e^-g above 2^126) the sigmoid, at most 2^-126, may come out as zero: FAR of
the magnitudes around it.
"""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from kernelforge_b200 import binding as B
from kernelforge_b200 import train
from tests import train_reference as R
from tests.helpers import gpu_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a B200")]

U = 2.0 ** -24
FAR = 2.0 ** -126
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _ids(t, k, g, masked=0.0, experts=256):
    """Distinct experts per token, some more popular than others; masked tokens have none."""
    score = torch.randn(t, 256, generator=g) + torch.randn(256, generator=g)
    ids = score.topk(k, dim=1).indices.to(torch.int32)
    ids[torch.rand(t, generator=g) < masked] = -1
    return ids


def _sigmoid_slack(gate, dtype):
    """Relative slack of products with a sigmoid of ``gate``."""
    return 2.0 ** -20 + (0.0 if dtype == torch.float32 else U * gate.abs())


def _dot_slack(h):
    return (8 * ((h + 255) // 256) + 21) * U


def _order(case, ids):
    t, k = ids.shape
    rows = case.get("max_rows") or R.worst_rows(t, k, case["experts"], case["align"])
    return R.order(ids, case["experts"], case["offset"], case["align"], rows), rows


def _same_order(order, ref):
    for got, want in zip(order, ref):
        assert got.dtype == torch.int32 and torch.equal(got.cpu(), want)


SORT_CASES = [
    # tokens, k, hidden, experts, offset, align, masked share, bound on the rows
    dict(t=1, k=1, h=64, experts=256, offset=0, align=1, masked=0.0),
    dict(t=1, k=8, h=7168, experts=256, offset=0, align=1, masked=0.0),
    dict(t=5, k=16, h=1, experts=256, offset=0, align=1, masked=0.3),
    dict(t=16, k=8, h=7168, experts=32, offset=96, align=128, masked=0.0),
    dict(t=33, k=3, h=1031, experts=100, offset=156, align=8, masked=0.3),
    dict(t=129, k=2, h=520, experts=1, offset=7, align=16, masked=0.0),
    dict(t=300, k=8, h=264, experts=256, offset=0, align=1, masked=0.5),
    dict(t=513, k=7, h=200, experts=64, offset=64, align=1024, masked=0.0),
    dict(t=1000, k=8, h=96, experts=256, offset=0, align=16, masked=0.1, max_rows=4000),
    dict(t=64, k=4, h=136, experts=256, offset=0, align=1, masked=0.0, max_rows=1),
    dict(t=7000, k=8, h=24, experts=256, offset=0, align=8, masked=0.0),
    dict(t=40, k=8, h=80, experts=256, offset=0, align=4, masked=1.0),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", SORT_CASES, ids=lambda c: "-".join(str(v) for v in c.values()))
def test_sort_and_its_gradient(case, dtype):
    g = torch.Generator().manual_seed(case["t"] * 31 + case["k"])
    t, k, h = case["t"], case["k"], case["h"]
    ids = _ids(t, k, g, case["masked"])
    ref, rows = _order(case, ids)
    x = torch.randn(t, h, generator=g).to(dtype)
    xg = x.cuda().requires_grad_(True)
    out, order = train.sort_tokens(xg, ids.cuda(), case["experts"], case["offset"], row_align=case["align"],
                                   max_rows=case.get("max_rows"))
    _same_order(order, ref)
    assert out.dtype == dtype and torch.equal(out.detach().cpu(), R.gather(x, ref[1], k))
    grad = torch.randn(rows, h, generator=g).to(dtype)
    grad[ref[1] < 0] = float("nan")          # rows of no pair must not be read
    dx, = torch.autograd.grad(out, xg, grad.cuda())
    want, mag = R.combine(grad, ref[0])
    R.close(dx, want, dtype, k * U * mag)
    assert torch.equal(train.sort_tokens_backward(grad.cuda(), order), dx)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", SORT_CASES, ids=lambda c: "-".join(str(v) for v in c.values()))
def test_combine_and_its_gradients(case, dtype):
    g = torch.Generator().manual_seed(case["t"] * 17 + case["k"])
    t, k, h = case["t"], case["k"], case["h"]
    ids = _ids(t, k, g, case["masked"])
    ref, rows = _order(case, ids)
    order = train.TokenOrder(*(a.cuda() for a in ref))
    y = torch.randn(rows, h, generator=g).to(dtype)
    y[ref[1] < 0] = float("inf")
    w = torch.randn(t, k, generator=g)
    w[ref[0] < 0] = float("nan")             # weights of pairs without a row are not used
    dout = torch.randn(t, h, generator=g).to(dtype)
    yg, wg = y.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    out = train.combine_tokens(yg, order, wg)
    want, mag = R.combine(y, ref[0], w)
    R.close(out.detach(), want, dtype, (k + 1) * U * mag)
    dy, dw = torch.autograd.grad(out, (yg, wg), dout.cuda())
    want_rows, want_w, mag_w = R.combine_grads(dout, y, ref[0], ref[1], w)
    R.close(dy, want_rows, dtype, U * want_rows.abs())
    R.close(dw, want_w, torch.float32, _dot_slack(h) * mag_w)
    both = train.combine_tokens_backward(dout.cuda(), y.cuda(), order, w.cuda())
    assert torch.equal(both[0], dy) and torch.equal(both[1], dw)
    # one gradient alone, and no weights
    yg2 = y.cuda().requires_grad_(True)
    dy2, = torch.autograd.grad(train.combine_tokens(yg2, order, w.cuda()), yg2, dout.cuda())
    assert torch.equal(dy2, dy)
    wg2 = w.cuda().requires_grad_(True)
    dw2, = torch.autograd.grad(train.combine_tokens(y.cuda(), order, wg2), wg2, dout.cuda())
    assert torch.equal(dw2, dw)
    plain, mag = R.combine(y, ref[0])
    yg3 = y.cuda().requires_grad_(True)
    out3 = train.combine_tokens(yg3, order)
    R.close(out3.detach(), plain, dtype, k * U * mag)
    dy3, = torch.autograd.grad(out3, yg3, dout.cuda())
    assert torch.equal(dy3.cpu(), R.gather(dout, ref[1], k))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("h", [264, 131])
def test_rows_in_place_of_other_layouts(h, dtype):
    """Strided rows, rows off a 16-byte boundary, transposed rows, and expanded gradients."""
    g = torch.Generator().manual_seed(h)
    t, k = 50, 4
    ids = _ids(t, k, g)
    big = torch.randn(t, 2 * h + 3, generator=g).to(dtype).cuda()
    case = dict(experts=256, offset=0, align=8)
    ref, rows = _order(case, ids)
    for x in (big[:, :h], big[:, 3:3 + h], big[:, 8:8 + h], torch.randn(h, t, generator=g).to(dtype).cuda().t(),
              big[:1, :h].expand(t, h)):
        out, order = train.sort_tokens(x, ids.cuda(), 256, row_align=8)
        assert torch.equal(out.cpu(), R.gather(x.cpu(), ref[1], k))
        kept = train.pack8(x)
        same = train.pack8(x.contiguous())
        assert torch.equal(kept.codes.view(torch.uint8), same.codes.view(torch.uint8)) and torch.equal(kept.exponents, same.exponents)
    wide = torch.randn(rows, h + 5, generator=g).to(dtype).cuda()
    order = train.TokenOrder(*(a.cuda() for a in ref))
    w = torch.rand(t, k, generator=g)
    want, mag = R.combine(wide[:, 2:2 + h].cpu(), ref[0], w)
    y = wide[:, 2:2 + h].detach().requires_grad_(True)
    out = train.combine_tokens(y, order, w.t().contiguous().t().cuda())
    R.close(out.detach(), want, dtype, (k + 1) * U * mag)
    dy, = torch.autograd.grad(out.sum(), y)      # an expanded gradient
    R.close(dy, R.combine_grads(torch.ones(t, h), wide[:, 2:2 + h].cpu(), ref[0], ref[1], w)[0], dtype, 0.0)


def test_gradients_of_broadcast_inputs():
    """One row for every token and one weight row for all: torch sums what the operators return."""
    g = torch.Generator().manual_seed(4)
    t, k, h = 30, 4, 72
    ids = _ids(t, k, g)
    row = torch.randn(1, h, generator=g).cuda().requires_grad_(True)
    rows, order = train.sort_tokens(row.expand(t, h), ids.cuda(), 256)
    grad = torch.randn(t * k, h, generator=g)
    d, = torch.autograd.grad(rows, row, grad.cuda())
    R.close(d, grad.double().sum(0, keepdim=True), torch.float32, t * k * U * grad.double().abs().sum(0, keepdim=True))
    w = torch.rand(1, k, generator=g).cuda().requires_grad_(True)
    dout = torch.randn(t, h, generator=g)
    dw, = torch.autograd.grad(train.combine_tokens(rows.detach(), order, w.expand(t, k)), w, dout.cuda())
    _, want, mag = R.combine_grads(dout, rows.detach().cpu(), order.pair_row.cpu(), order.row_pair.cpu(), w.detach().cpu().expand(t, k))
    R.close(dw, want.sum(0, keepdim=True), torch.float32, (_dot_slack(h) + t * U) * mag.sum(0, keepdim=True))


def test_sort_of_repeated_and_foreign_ids():
    ids = torch.tensor([[3, 3, 3], [300, -5, 3], [2 ** 31 - 1, -2 ** 31, 255], [0, 255, 0]], dtype=torch.int32)
    x = torch.randn(4, 16)
    ref = R.order(ids, 256, 0, 2, R.worst_rows(4, 3, 256, 2))
    out, order = train.sort_tokens(x.cuda(), ids.cuda(), 256, row_align=2)
    _same_order(order, ref)
    assert torch.equal(out.cpu(), R.gather(x, ref[1], 3))
    shifted, order = train.sort_tokens(x.cuda(), ids.cuda(), 200, 56)
    _same_order(order, R.order(ids, 200, 56, 1, 12))


def test_sort_without_tokens_or_rows():
    out, order = train.sort_tokens(torch.empty(0, 32).cuda(), torch.empty(0, 8, dtype=torch.int32).cuda(), 12)
    assert out.shape == (0, 32) and order.pair_row.shape == (0, 8) and order.row_pair.shape == (0,)
    assert not order.counts.any() and not order.starts.any()
    out, order = train.sort_tokens(torch.empty(0, 32).cuda(), torch.empty(0, 8, dtype=torch.int32).cuda(), 12, row_align=4, max_rows=8)
    assert not out.any() and (order.row_pair == -1).all() and out.shape == (8, 32)
    x = torch.randn(3, 32).cuda()
    ids = torch.zeros(3, 2, dtype=torch.int32).cuda()
    out, order = train.sort_tokens(x, ids, 12, max_rows=0)
    assert out.shape == (0, 32) and (order.pair_row == -1).all() and int(order.counts[0]) == 6
    assert not train.combine_tokens(out, order, torch.ones(3, 2).cuda()).any()
    assert train.restore8(train.pack8(x), order).shape == (0, 32)
    xg, yg, wg = x.clone().requires_grad_(True), out.clone().requires_grad_(True), torch.ones(3, 2).cuda().requires_grad_(True)
    assert not torch.autograd.grad(train.sort_tokens(xg, ids, 12, max_rows=0)[0], xg, out)[0].any()
    dy, dw = torch.autograd.grad(train.combine_tokens(yg, order, wg), (yg, wg), x)
    assert dy.shape == (0, 32) and not dw.any()
    none = train.sort_tokens(x[:0], ids[:0], 12, row_align=4, max_rows=8)[1]
    assert not train.restore8(train.pack8(x[:0]), none).any() and not train.combine_tokens_backward(
        x[:0], torch.ones(8, 32).cuda(), none, torch.ones(0, 2).cuda())[0].any()
    assert train.combine_tokens(torch.empty(0, 32).cuda(), train.TokenOrder(
        torch.empty(0, 2, dtype=torch.int32).cuda(), torch.empty(0, dtype=torch.int32).cuda(), order.counts, order.starts)).shape == (0, 32)
    assert train.pack8(torch.empty(0, 32).cuda()).codes.shape == (0, 32)
    assert train.swiglu(torch.empty(0, 32).cuda()).shape == (0, 16)


def test_an_order_that_does_not_fit_is_harmless():
    """Rows or pairs out of range in a caller's order count as none (no read or write out of range)."""
    pair_row = torch.tensor([[0, 7], [2 ** 31 - 1, -9]], dtype=torch.int32).cuda()
    row_pair = torch.tensor([0, 99, -7, 2 ** 31 - 1], dtype=torch.int32).cuda()
    order = train.TokenOrder(pair_row, row_pair, pair_row[0], pair_row[0])
    y = torch.randn(4, 40).cuda()
    w = torch.ones(2, 2).cuda()
    out = train.combine_tokens(y, order, w)
    assert torch.equal(out[0], y[0]) and not out[1].any()
    dr, dw = train.combine_tokens_backward(torch.ones(2, 40).cuda(), y, order, w)
    assert (dr[0] == 1).all() and not dr[1:].any() and not dw[1].any() and dw[0, 1] == 0
    back = train.restore8(train.pack8(y[:2].contiguous()), order)
    assert not back[1:].any()


# ---------------------------------------------------------------------- route --


@pytest.mark.parametrize("t", [1, 7, 64, 1000])
def test_route_and_its_gradient(t):
    g = torch.Generator().manual_seed(t)
    logits = torch.randn(t, 256, generator=g)
    bias = (0.02 * torch.randn(256, generator=g)).to(torch.bfloat16)
    lg = logits.cuda().requires_grad_(True)
    idx, w = train.route(lg, bias.cuda(), 2.5)
    idx0, w0 = B.route(logits.cuda(), bias.cuda(), 2.5)
    assert torch.equal(idx, idx0) and torch.equal(w.detach(), w0)
    gw = torch.randn(t, 8, generator=g)
    dl, = torch.autograd.grad(w, lg, gw.cuda())
    want, mag = R.route_grad(logits, idx.cpu(), gw, 2.5)
    R.close(dl, want, torch.float32, 2.0 ** -19 * mag)
    assert torch.equal(dl, train.route_backward(logits.cuda(), idx, gw.cuda(), 2.5))


def test_route_gradient_at_the_ends():
    """Saturated logits, ids of no choice and a token without any."""
    g = torch.Generator().manual_seed(1)
    logits = 30 * torch.randn(40, 256, generator=g)
    ids = torch.stack([torch.randperm(256, generator=g)[:8] for _ in range(40)]).to(torch.int32)
    ids[3] = -1
    ids[4, ::2] = 256
    gw = torch.randn(40, 8, generator=g)
    gw[3] = float("nan")
    dl = train.route_backward(logits.cuda(), ids.cuda(), gw.cuda(), 1.5)
    want, mag = R.route_grad(logits, ids, torch.nan_to_num(gw), 1.5)
    # sigmoids down to e^-100 lose their last bits as fp32 subnormals: what they weigh is below 1e-30
    R.close(dl, want, torch.float32, 2.0 ** -19 * mag + 1e-30)
    assert not dl[3].any()


def test_route_gradient_of_repeated_ids():
    """A repeated id (outside the routing's contract) gets the sum of its choices' gradients."""
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(9, 256, generator=g)
    ids = torch.stack([torch.randperm(256, generator=g)[:8] for _ in range(9)]).to(torch.int32)
    ids[1, 3] = ids[1, 6]
    ids[2] = 255
    ids[5, :4] = ids[5, 4:]
    gw = torch.randn(9, 8, generator=g)
    want, mag = R.route_grad(logits, ids, gw, 2.5)
    R.close(train.route_backward(logits.cuda(), ids.cuda(), gw.cuda(), 2.5), want, torch.float32, 2.0 ** -19 * mag)


# --------------------------------------------------------------------- 8 bits --


def _rows(r, w, dtype, g):
    x = torch.randn(r, w, generator=g) * torch.exp(2 * torch.randn(r, 1, generator=g))
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("r,w", [(1, 1), (3, 127), (2, 128), (5, 136), (4, 1000), (17, 257), (64, 7168), (9, 2047)])
def test_rows_in_8_bits_and_back(r, w, dtype):
    g = torch.Generator().manual_seed(r + w)
    x = _rows(r, w, dtype, g)
    kept = train.pack8(x.cuda())
    want, e = R.to_8_bits(x)
    assert kept.dtype == dtype and torch.equal(kept.exponents.cpu().double() - 127, e)
    back = train.restore8(kept)
    assert back.dtype == dtype and torch.equal(back.cpu().double(), want.to(dtype).double())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("w", [256, 131])
def test_rows_in_8_bits_at_the_ends(w, dtype):
    """Zeros, the type's largest and smallest values, values next to a border, and values that are not finite."""
    info = torch.finfo(dtype)
    rows = [torch.zeros(w), torch.full((w,), info.max), torch.full((w,), -info.max), torch.full((w,), info.tiny),
            torch.linspace(-1, 1, w) * info.max, torch.linspace(-448, 448, w), torch.linspace(-1, 1, w) * 449,
            torch.linspace(-17.5, 17.5, w), 2.0 ** torch.linspace(-24, 15, w), torch.linspace(0, 2.0 ** -9, w),
            torch.linspace(-1, 1, w) * info.tiny, torch.linspace(0, 1, w) * info.tiny / 4]
    odd = torch.linspace(-3, 3, w)
    odd[5], odd[7], odd[w - 1] = float("inf"), float("nan"), float("-inf")
    rows += [odd, torch.full((w,), float("nan")), torch.full((w,), float("inf"))]
    x = torch.stack(rows).to(dtype)
    want, e = R.to_8_bits(x)
    kept = train.pack8(x.cuda())
    assert torch.equal(kept.exponents.cpu().double() - 127, e)
    back = train.restore8(kept).cpu()
    finite = torch.isfinite(x)
    assert torch.isnan(back[~finite]).all() and torch.isfinite(back[finite]).all()
    assert torch.equal(back[finite].double(), want.to(dtype)[finite].double())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", SORT_CASES[1:9], ids=lambda c: "-".join(str(v) for v in c.values()))
def test_rows_in_8_bits_in_expert_order(case, dtype):
    g = torch.Generator().manual_seed(case["t"])
    ids = _ids(case["t"], case["k"], g, case["masked"])
    ref, _ = _order(case, ids)
    x = _rows(case["t"], case["h"], dtype, g)
    back = train.restore8(train.pack8(x.cuda()), train.TokenOrder(*(a.cuda() for a in ref)))
    assert torch.equal(back.cpu(), R.gather(R.to_8_bits(x)[0].to(dtype), ref[1], case["k"]))


MANY_CHOICES = [
    # more than eight choices: two batches of rows per slice, in the 16-byte and in the plain forms
    dict(t=37, k=9, h=264, experts=256, offset=0, align=8, masked=0.2),
    dict(t=3000, k=16, h=72, experts=64, offset=32, align=1, masked=0.0),
    dict(t=20, k=12, h=7168, experts=256, offset=0, align=16, masked=0.0),
    dict(t=21, k=13, h=1031, experts=200, offset=0, align=1, masked=0.3),
    dict(t=90, k=16, h=520, experts=256, offset=0, align=1, masked=0.0, max_rows=900),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", MANY_CHOICES, ids=lambda c: "-".join(str(v) for v in c.values()))
def test_more_than_eight_choices(case, dtype):
    test_sort_and_its_gradient(case, dtype)
    test_combine_and_its_gradients(case, dtype)
    test_rows_in_8_bits_in_expert_order(case, dtype)


MANY_STEPS = [
    # more tokens than blocks that stay, and several steps per warp and token: the load stream is a step ahead of the sum
    dict(t=400, k=3, h=7168, experts=256, offset=0, align=1, masked=0.2),
    dict(t=400, k=8, h=7168, experts=128, offset=64, align=8, masked=0.2),
    dict(t=400, k=2, h=7168, experts=256, offset=0, align=1, masked=0.2),
    dict(t=400, k=11, h=7168, experts=256, offset=0, align=1, masked=0.2),
    dict(t=600, k=8, h=2056, experts=256, offset=0, align=1, masked=0.2),
    dict(t=500, k=4, h=3848, experts=256, offset=0, align=1, masked=0.2),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", MANY_STEPS, ids=lambda c: "-".join(str(v) for v in c.values()))
def test_several_tokens_a_block_and_steps_a_warp(case, dtype):
    """Random weights and rows of their own per pair: a step summed with another token's or choice's weight or row fails."""
    test_combine_and_its_gradients(case, dtype)


def test_combine_past_32_bit_offsets_tells_weights_and_rows_apart():
    """More than 2^31 elements of rows, each row and weight its own, against sums in 64 bits at some of the tokens."""
    t, h, k = 40960, 7168, 8
    g = torch.Generator(device="cuda").manual_seed(10)
    ids = torch.randn(t, 256, generator=g, device="cuda").topk(k, dim=1).indices.to(torch.int32)
    _, order = train.sort_tokens(torch.zeros(t, 1, dtype=torch.bfloat16, device="cuda"), ids, 256)
    rows = torch.randn(t * k, h, generator=g, device="cuda", dtype=torch.bfloat16)
    assert rows.numel() > 2 ** 31 and int(order.pair_row.max()) == t * k - 1
    w = torch.rand(t, k, generator=g, device="cuda") + 0.1
    dout = torch.randn(t, h, generator=g, device="cuda", dtype=torch.bfloat16)
    out = train.combine_tokens(rows, order, w)
    drows, dw = train.combine_tokens_backward(dout, rows, order, w)
    last = order.row_pair[-200:].long() // k          # the tokens of the last rows
    pick = torch.cat([torch.arange(50, device="cuda"), torch.randint(0, t, (250,), device="cuda", generator=g), last])
    at = order.pair_row[pick].long()
    picked = rows[at.reshape(-1)].double().reshape(pick.numel(), k, h)
    terms = picked * w[pick, :, None].double()
    R.close(out[pick], terms.sum(1).cpu(), torch.bfloat16, (k + 1) * U * terms.abs().sum(1).cpu())
    prod = picked * dout[pick, None].double()
    R.close(dw[pick], prod.sum(2).cpu(), torch.float32, _dot_slack(h) * prod.abs().sum(2).cpu())
    want = (dout[pick, None].double() * w[pick, :, None].double()).reshape(-1, h).cpu()
    R.close(drows[at.reshape(-1)], want, torch.bfloat16, U * want.abs())


# --------------------------------------------------------------------- swiglu --


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("r,n", [(1, 1), (1, 128), (3, 131), (7, 1368), (33, 2048), (130, 264)])
def test_swiglu_and_its_gradient(r, n, dtype):
    g = torch.Generator().manual_seed(r * n)
    h = _rows(r, 2 * n, dtype, g)
    d = torch.randn(r, n, generator=g).to(dtype)
    act, kept = train.swiglu_pack8(h.cuda())
    u, gate = h[:, :n].double(), h[:, n:].double()
    R.close(act, R.swiglu(u, gate), dtype, _sigmoid_slack(gate, dtype) * R.swiglu(u, gate).abs() + FAR * (u * gate).abs())
    (ku, eu), (kg, eg) = R.to_8_bits(h[:, :n]), R.to_8_bits(h[:, n:])
    assert torch.equal(kept.exponents.cpu().double() - 127, torch.cat([eu, eg], 1))
    dh, again = train.swiglu_backward8(kept, d.cuda())
    du, dg, a, mag = R.swiglu_grads(ku, kg, d.double())
    dd = d.double()
    near = _sigmoid_slack(kg, dtype)
    R.close(again, a, dtype, near * a.abs() + FAR * (ku * kg).abs())
    R.close(dh[:, :n], du, dtype, near * du.abs() + FAR * (dd * kg).abs())
    R.close(dh[:, n:], dg, dtype, near * mag + FAR * (dd * ku).abs() * (1 + kg.abs()))
    hg = h.cuda().requires_grad_(True)
    out = train.swiglu(hg)
    dh2, = torch.autograd.grad(out, hg, d.cuda())
    assert torch.equal(out.detach(), act) and torch.equal(dh2, dh)
    assert torch.equal(train.swiglu(h.cuda()), act)
    only, none = train.swiglu_backward8(kept, d.cuda(), need_act=False)
    assert none is None and torch.equal(only, dh)


@pytest.mark.parametrize("dtype", TYPES)
def test_swiglu_of_far_gates(dtype):
    gate = torch.tensor([-60000.0, -1000, -90, -88, -40, -20, -1e-6, 0, 1e-6, 20, 90, 1000, 60000]).to(dtype)
    h = torch.cat([torch.ones_like(gate), gate])[None]
    n = gate.numel()
    act, kept = train.swiglu_pack8(h.cuda())
    # a sigmoid below fp32's smallest normal value may come out as zero: |gate| * 2^-126
    R.close(act, R.swiglu(h[:, :n].double(), h[:, n:].double()), dtype, 2.0 ** -18 * R.swiglu(h[:, :n].double(), h[:, n:].double()).abs() + 1e-33)
    dh, again = train.swiglu_backward8(kept, torch.ones(1, n).to(dtype).cuda())
    assert torch.isfinite(dh).all() and torch.isfinite(again).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_swiglu_gradient_of_large_values(dtype):
    """A gate gradient d u (s + g s (1 - s)) whose product d u alone is beyond fp32, and one whose product u (s + ..) is."""
    big = 60000.0 if dtype == torch.float16 else 1e20
    pairs = [(big, big), (-big, big), (big, -big)]
    pairs += [] if dtype == torch.float16 else [(3e38, 0.1), (0.1, 3e38), (3e38, 3e38), (3e38, -2.0), (1e30, 1e9)]
    gates = [-1000.0, -90, -86, -60, -50, -30, -10, -1, -1e-3, 0, 1e-3, 1, 2.4, 10, 1000]
    # one value a block: each is kept on its own scale
    u, d, gate = (torch.tensor(v) for v in zip(*[(a, b, g) for a, b in pairs for g in gates]))
    u, d, gate = u[:, None].to(dtype), d[:, None].to(dtype), gate[:, None].to(dtype)
    _, kept = train.swiglu_pack8(torch.cat([u, gate], 1).cuda())
    ku, kg, dd = R.to_8_bits(u)[0], R.to_8_bits(gate)[0], d.double()
    dh, act = train.swiglu_backward8(kept, d.cuda())
    du, dg, a, mag = R.swiglu_grads(ku, kg, dd)
    near = _sigmoid_slack(kg, dtype)
    R.close(act, a, dtype, near * a.abs() + FAR * (ku * kg).abs())
    R.close(dh[:, :1], du, dtype, near * du.abs() + FAR * (dd * kg).abs())
    R.close(dh[:, 1:], dg, dtype, near * mag + FAR * (dd * ku).abs() * (1 + kg.abs()))
    # a gradient that is no number hides no neighbour's product
    row = torch.full((1, 8), 1.0).to(dtype)
    row[0, 3] = float("nan")
    d = torch.full((1, 8), big).to(dtype)
    d[0, 5] = float("nan")
    _, kept = train.swiglu_pack8(torch.cat([row * big, torch.full((1, 8), -50.0).to(dtype)], 1).cuda())
    dg = train.swiglu_backward8(kept, d.cuda())[0][:, 8:].cpu()
    assert torch.equal(torch.isnan(dg[0]), torch.tensor([i in (3, 5) for i in range(8)]))
    fine = torch.tensor([0, 1, 2, 4, 6, 7])
    ku, dd = R.to_8_bits(row * big)[0][:, fine], d[:, fine].double()
    kg = R.to_8_bits(torch.full((1, 8), -50.0).to(dtype))[0][:, fine]
    _, want, _, mag = R.swiglu_grads(ku, kg, dd)
    R.close(dg[:, fine], want, dtype, _sigmoid_slack(kg, dtype) * mag)


@pytest.mark.parametrize("n", [70, 96, 100, 127, 128, 256])
def test_rows_in_8_bits_know_where_their_blocks_begin(n):
    """SwiGLU's blocks begin at each half's first column: rows kept one way are not read the other way unless both agree."""
    g = torch.Generator().manual_seed(n)
    h = torch.randn(6, 2 * n, generator=g)
    h[:, n:] *= 1000                                  # a half's scale would not fit the other's values
    d = torch.randn(6, n, generator=g).cuda()
    whole, (_, halves) = train.pack8(h.cuda()), train.swiglu_pack8(h.cuda())
    want = train.swiglu_backward8(halves, d)[0]
    again = train.Rows8(halves.codes, halves.exponents, halves.dtype)      # as a caller's autograd function puts it together
    assert torch.equal(train.swiglu_backward8(again, d)[0], want)
    assert isinstance(whole, train.Rows8) and isinstance(halves, train.Rows8) and len(halves) == 3
    if n % 128:
        with pytest.raises(RuntimeError, match="restore8"):
            train.restore8(halves)
        with pytest.raises(RuntimeError, match="swiglu_backward8"):
            train.swiglu_backward8(whole, d)
    else:
        assert torch.equal(train.restore8(halves).cpu().double(), R.to_8_bits(h)[0])
        assert torch.equal(train.swiglu_backward8(whole, d)[0], want)


# ------------------------------------------------------------------- together --


def test_refusals_on_the_gpu():
    x, ids = torch.zeros(4, 32).cuda(), torch.zeros(4, 2, dtype=torch.int32).cuda()
    _, order = train.sort_tokens(x, ids, 8)
    w = torch.ones(4, 2).cuda()
    kept = train.pack8(x)
    bad = [lambda: train.sort_tokens(x.double(), ids, 8), lambda: train.sort_tokens(x[0], ids, 8),
           lambda: train.sort_tokens(x, ids.long(), 8), lambda: train.sort_tokens(x, ids[:3], 8),
           lambda: train.sort_tokens(x, ids.cpu(), 8), lambda: train.sort_tokens(x, ids, 0),
           lambda: train.sort_tokens(x, ids, 257), lambda: train.sort_tokens(x, ids, 8, 250),
           lambda: train.sort_tokens(x, ids, 8, -1), lambda: train.sort_tokens(x, ids, 8, row_align=0),
           lambda: train.sort_tokens(x, ids, 8, row_align=2000), lambda: train.sort_tokens(x, ids, 8, row_align=8, max_rows=12),
           lambda: train.sort_tokens(x, ids, 8, max_rows=-1), lambda: train.sort_tokens(x, ids, 8, max_rows=2 ** 31),
           lambda: train.sort_tokens(x[:, :0], ids, 8), lambda: train.sort_tokens(x, ids.expand(4, 2).repeat(1, 9), 8),
           lambda: train.combine_tokens(x, order, w), lambda: train.combine_tokens(torch.zeros(8, 32).cuda(), order, w.double()),
           lambda: train.combine_tokens(torch.zeros(8, 32).cuda(), order, w[:, :1]),
           lambda: train.combine_tokens(torch.zeros(8, 32).cuda().long(), order, w),
           lambda: train.sort_tokens_backward(x, order),
           lambda: train.combine_tokens_backward(x, torch.zeros(8, 16).cuda(), order, w),
           lambda: train.combine_tokens_backward(x[:3], torch.zeros(8, 32).cuda(), order, w),
           lambda: train.restore8(kept._replace(exponents=kept.exponents[:3])), lambda: train.restore8(kept._replace(dtype=torch.int32)),
           lambda: train.restore8(train.pack8(x[:3]), order), lambda: train.swiglu(x[:, :31]),
           lambda: train.swiglu_backward8(kept, x), lambda: train.swiglu_backward8(train.swiglu_pack8(x)[1], x),
           lambda: train.route_backward(torch.zeros(4, 256).cuda(), ids, w, 1.0),
           lambda: train.route(torch.zeros(4, 255).cuda(), torch.zeros(255, dtype=torch.bfloat16).cuda(), 1.0)]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was accepted")


def test_no_second_derivative():
    x = torch.randn(4, 32).cuda().requires_grad_(True)
    rows, order = train.sort_tokens(x, torch.zeros(4, 2, dtype=torch.int32).cuda(), 8)
    for out in (rows, train.swiglu(x), train.combine_tokens(rows, order)):
        with pytest.raises(RuntimeError, match="not twice differentiable"):
            torch.autograd.grad(out.sum(), x, create_graph=True)


def test_forward_mode_derivatives_are_refused():
    """No operator has a forward-mode rule: a tangent raises, in the forward and in the backward pass, instead of getting lost."""
    g = torch.Generator().manual_seed(21)
    x, ids = torch.randn(4, 32, generator=g).cuda(), torch.tensor([[0, 1]] * 4, dtype=torch.int32).cuda()
    logits, bias = torch.randn(4, 256, generator=g).cuda(), torch.zeros(256, dtype=torch.bfloat16).cuda()
    w = torch.ones(4, 2).cuda()
    rows, order = train.sort_tokens(x, ids, 8)
    act, kept = train.swiglu_pack8(x)
    leaves = [a.clone().requires_grad_(True) for a in (x, rows, w, logits)]
    outs = [(train.sort_tokens(leaves[0], ids, 8)[0], leaves[0]), (train.swiglu(leaves[0]), leaves[0]),
            (train.combine_tokens(leaves[1], order, w), leaves[1]), (train.combine_tokens(rows, order, leaves[2]), leaves[2]),
            (train.route(leaves[3], bias, 2.5)[1], leaves[3])]
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t.detach(), torch.ones_like(t))

        calls = [lambda: train.route(dual(logits), bias, 2.5), lambda: train.sort_tokens(dual(x), ids, 8),
                 lambda: train.combine_tokens(dual(rows), order, w), lambda: train.combine_tokens(rows, order, dual(w)),
                 lambda: train.combine_tokens(dual(rows), order), lambda: train.swiglu(dual(x)),
                 lambda: train.sort_tokens_backward(dual(rows), order), lambda: train.combine_tokens_backward(dual(x), rows, order, w),
                 lambda: train.combine_tokens_backward(x, rows, order, dual(w)), lambda: train.swiglu_backward8(kept, dual(act)),
                 lambda: train.route_backward(logits, ids.repeat(1, 4), dual(w.repeat(1, 4)), 2.5)]
        calls += [lambda out=out, leaf=leaf: torch.autograd.grad(out, leaf, dual(out)) for out, leaf in outs]
        for i, call in enumerate(calls):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
                pytest.fail(f"call {i} was accepted")
        assert torch.equal(train.swiglu(x), act)      # without a tangent, inside the level too
    for out, leaf in outs:                            # and the reverse mode as ever
        assert torch.isfinite(torch.autograd.grad(out, leaf, torch.ones_like(out))[0]).all()


def _layer(x, logits, bias, w13, w2, products):
    """An MoE layer with the caller's own expert products."""
    idx, weight = train.route(logits, bias, 2.5)
    rows, order = train.sort_tokens(x, idx, w13.shape[0], row_align=8)
    h = products(rows, order, w13)
    y = products(train.swiglu(h), order, w2)
    return train.combine_tokens(y, order, weight), order, idx


def _products(rows, order, w):
    """Each expert's rows times its matrix, a segment at a time (fp32)."""
    starts = order.starts.tolist()
    parts = [rows[starts[e]:starts[e + 1]] @ w[e].t() for e in range(w.shape[0])]
    return torch.cat(parts + [rows.new_zeros(rows.shape[0] - starts[-1], w.shape[1])])


def test_the_operators_together_as_a_layer():
    """A whole fp32 layer, forward and every gradient, against the same layer in 64 bits.

    The 64-bit layer's backward pass takes SwiGLU's input as the 8-bit form keeps it, as the operator
    documents.  fp32 products over 48 and 32 columns and the operators' own sums: 200 roundings of 2^-24 of
    the largest magnitudes at most, against outputs and gradients compared at their largest value; 1e-4 of
    it is that with a factor of 8 for cancellation inside the sums.  A kept value may fall on the other side of an
    e4m3 border than the 64-bit one (h differs by fp32 rounding): the 64-bit layer keeps the fp32 h's values.
    """
    g = torch.Generator().manual_seed(11)
    t, h, n, experts = 70, 48, 32, 256
    x = torch.randn(t, h, generator=g)
    logits = torch.randn(t, 256, generator=g)
    bias = (0.02 * torch.randn(256, generator=g)).to(torch.bfloat16)
    w13 = 0.2 * torch.randn(experts, 2 * n, h, generator=g)
    w2 = 0.2 * torch.randn(experts, h, n, generator=g)
    dout = torch.randn(t, h, generator=g)
    leaves = [a.cuda().requires_grad_(True) for a in (x, logits, w13, w2)]
    kept = {}

    def products(rows, order, w):
        out = _products(rows, order, w)
        kept.setdefault("h", out.detach().cpu())
        return out

    torch.backends.cuda.matmul.allow_tf32 = False
    out, order, idx = _layer(leaves[0], leaves[1], bias.cuda(), leaves[2], leaves[3], products)
    grads = torch.autograd.grad(out, leaves, dout.cuda())

    xd, ld, w13d, w2d = (a.double().requires_grad_(True) for a in (x, logits, w13, w2))
    idx, pair_row, row_pair = idx.cpu(), order.pair_row.cpu(), order.row_pair.cpu()
    s = torch.sigmoid(ld.gather(1, idx.long()))
    weight = 2.5 * s / (s.sum(1, keepdim=True) + 1e-20)
    q = torch.cat([R.to_8_bits(kept["h"][:, :n])[0], R.to_8_bits(kept["h"][:, n:])[0]], 1)
    want = torch.zeros(t, h, dtype=torch.float64)
    for tok in range(t):
        for k in range(8):
            e = int(idx[tok, k])
            hh = w13d[e] @ xd[tok]
            exact_act = R.swiglu(hh[:n], hh[n:])
            kq = q[int(pair_row[tok, k])] + (hh - hh.detach())        # the kept value, with h's gradient
            act = R.swiglu(kq[:n], kq[n:])
            act = exact_act.detach() + (act - act.detach())           # the forward value, the kept value's gradient
            want[tok] = want[tok] + weight[tok, k] * (w2d[e] @ act)
    wants = torch.autograd.grad(want, (xd, ld, w13d, w2d), dout.double())
    for got, ref in zip((out.detach(),) + grads, (want.detach(),) + wants):
        assert (got.double().cpu() - ref).abs().max() <= 1e-4 * ref.abs().max()


def _training_calls(x, ids, w, dout, d8):
    rows, order = train.sort_tokens(x, ids, 256, row_align=8)
    out = train.combine_tokens(rows, order, w)
    drows, dw = train.combine_tokens_backward(dout, rows, order, w)
    dx = train.sort_tokens_backward(drows, order)
    act, kept = train.swiglu_pack8(rows)
    dh, again = train.swiglu_backward8(kept, d8)
    back = train.restore8(train.pack8(x), order)
    return (rows, *order, out, drows, dw, dx, act, dh, again, back)


def _inputs(seed, t=200, h=320, k=8):
    g = torch.Generator().manual_seed(seed)
    rows = R.worst_rows(t, k, 256, 8)
    return [a.cuda() for a in (torch.randn(t, h, generator=g).to(torch.bfloat16), _ids(t, k, g, 0.1),
                               torch.rand(t, k, generator=g), torch.randn(t, h, generator=g).to(torch.bfloat16),
                               torch.randn(rows, h // 2, generator=g).to(torch.bfloat16))]


@pytest.mark.parametrize("t", [3, 200, 6000])
def test_captured_and_replayed(t):
    """Two graphs captured one after the other and replayed in turn on new inputs give the direct calls' bits."""
    a, b = _inputs(1, t), _inputs(2, t)
    want = [[o.clone() for o in _training_calls(*i)] for i in (a, b)]
    torch.cuda.synchronize()
    graphs, static, outs = [], [], []
    for i in (a, b):
        static.append([torch.zeros_like(v) for v in i])
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(_training_calls(*static[-1]))
        graphs.append(gr)
    for _ in range(2):
        for i, gr, s in ((a, graphs[0], static[0]), (b, graphs[1], static[1])):
            for dst, src in zip(s, i):
                dst.copy_(src)
            gr.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(x.nan_to_num(), y.nan_to_num()) for x, y in zip(o, w))


def test_gradients_captured_and_replayed():
    """Forward and backward through autograd in one capture, replayed on new inputs."""
    def step(x, ids, w, dout):
        rows, order = train.sort_tokens(x, ids, 256, row_align=8)
        out = train.combine_tokens(train.swiglu(torch.cat([rows, rows], 1)), order, w)
        return (out.detach(),) + torch.autograd.grad(out, (x, w), dout)

    i = _inputs(8, 300)
    x, ids, w, dout = i[0].requires_grad_(True), i[1], i[2].requires_grad_(True), i[3]
    want = [o.clone() for o in step(x, ids, w, dout)]
    static = [torch.zeros_like(x).requires_grad_(True), torch.zeros_like(ids), torch.zeros_like(w).requires_grad_(True),
              torch.zeros_like(dout)]
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        outs = step(*static)
    with torch.no_grad():
        for dst, src in zip(static, (x, ids, w, dout)):
            dst.copy_(src)
    gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, v) for o, v in zip(outs, want))


def test_capture_with_an_eager_graph_of_the_same_leaf_is_refused():
    x = torch.randn(8, 64, device="cuda", requires_grad=True)
    ids = torch.zeros(8, 1, dtype=torch.int32, device="cuda")
    eager, order = train.sort_tokens(x, ids, 4)        # alive, on the default stream
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    w = torch.ones(8, 1, device="cuda", requires_grad=True)
    also = train.combine_tokens(eager.detach(), order, w)
    logits = torch.randn(8, 256, device="cuda", requires_grad=True)
    bias = torch.zeros(256, dtype=torch.bfloat16, device="cuda")
    fourth = train.route(logits, bias, 1.0)
    for call in (lambda: train.sort_tokens(x, ids, 4), lambda: train.swiglu(x), lambda: train.combine_tokens(x, order),
                 lambda: train.combine_tokens(eager.detach(), order, w), lambda: train.route(logits, bias, 1.0)):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            gr.capture_begin()
            try:
                with pytest.raises(RuntimeError, match="eager autograd graph is still alive"):
                    call()
            finally:
                gr.capture_end()
    torch.cuda.synchronize()
    dx, = torch.autograd.grad(eager, x, torch.ones_like(eager))
    assert (dx == 1).all() and also.requires_grad and fourth[1].requires_grad


@pytest.mark.parametrize("backward", [True, False], ids=["backward", "grad"])
def test_capture_with_a_graph_of_the_same_leaf_on_a_side_stream(backward):
    """Warm-up on a side stream whose graph still lives, then a capture: that stream joins the capture."""
    g = torch.Generator().manual_seed(31)
    x, w, logits = (torch.randn(8, n, generator=g).cuda().requires_grad_(True) for n in (64, 1, 256))
    bias, ids = torch.zeros(256, dtype=torch.bfloat16).cuda(), torch.zeros(8, 1, dtype=torch.int32).cuda()
    douts = [torch.randn(8, n, generator=g).cuda() for n in (64, 8, 32)]
    leaves = (x, w, logits)

    def step():
        rows, order = train.sort_tokens(x, ids, 4)
        return train.combine_tokens(rows, order, w), train.route(logits, bias, 2.5)[1], train.swiglu(x)

    def gradients(outs):
        if not backward:
            return torch.autograd.grad(outs, leaves, douts, retain_graph=True)
        for leaf in leaves:
            leaf.grad = None
        torch.autograd.backward(outs, douts, retain_graph=True)
        return [leaf.grad for leaf in leaves]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = step()                                # lives through the capture
        want = [a.clone() for a in gradients(alive)]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for leaf in leaves:
        leaf.grad = None
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = gradients(step())
    for a in got:
        a.detach().zero_()
    gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and len(alive) == 3


def test_a_factor_on_the_gpu_is_refused_in_a_capture():
    """Reading it back would end the capture; the refusal leaves the capture whole.  Outside it is read."""
    logits, bias = torch.randn(8, 256).cuda(), torch.zeros(256, dtype=torch.bfloat16).cuda()
    factor = torch.tensor(2.5).cuda()
    ids, w = train.route(logits, bias, 2.5)
    assert torch.equal(train.route(logits, bias, factor)[1], w)
    want = train.route_backward(logits, ids, w, 2.5)
    assert torch.equal(train.route_backward(logits, ids, w, factor), want)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        for call in (lambda: train.route(logits, bias, factor), lambda: train.route_backward(logits, ids, w, factor)):
            with pytest.raises(RuntimeError, match="pass a number"):
                call()
        again = train.route(logits, bias, torch.tensor(2.5))[1]      # on the host it may be a tensor
        grad = train.route_backward(logits, ids, w, 2.5)
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, w) and torch.equal(grad, want)


def test_two_streams_at_once():
    """Calls in flight on two streams share nothing."""
    inputs = [_inputs(3, 6000), _inputs(4, 6000)]
    want = [[o.clone() for o in _training_calls(*i)] for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    got = [None, None]
    for _ in range(3):
        for n, (s, i) in enumerate(zip(streams, inputs)):
            with torch.cuda.stream(s):
                got[n] = _training_calls(*i)
    torch.cuda.synchronize()
    for o, w in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(o, w))


def test_equal_inputs_give_equal_bits():
    i = _inputs(5, 3000)
    first = [o.clone() for o in _training_calls(*i)]
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, _training_calls(*i)))


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_on_a_device_that_is_not_current():
    i = _inputs(6)
    want = _training_calls(*i)
    got = _training_calls(*(v.to("cuda:1") for v in i))
    assert all(o.device.index == 1 and torch.equal(o.cpu(), w.cpu()) for o, w in zip(got, want))


class _Guarded:
    """Output buffers inside larger ones whose other bytes must stay as they are."""

    def __init__(self):
        self.all = []

    def __call__(self, nbytes, offset=0):
        big = torch.full((nbytes + 1024 + offset,), 0xA5, dtype=torch.uint8, device="cuda")
        self.all.append((big, 512 + offset, nbytes))
        return ctypes.c_void_p(big.data_ptr() + 512 + offset)

    def check(self):
        for big, at, n in self.all:
            assert (big[:at] == 0xA5).all() and (big[at + n:] == 0xA5).all()


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("t,k,h,align,rows", [(1, 1, 1, 1, 1), (5, 3, 257, 8, 40), (40, 8, 1031, 1, 320), (3, 16, 8, 128, 1024),
                                              (33, 2, 264, 16, 32), (2000, 8, 24, 8, 17600), (130, 5, 130, 1, 0)])
def test_nothing_outside_the_outputs_is_written(t, k, h, align, rows, dtype):
    """The C entry points on buffers between guards, also of elements off 16-byte boundaries."""
    lib, null, es = B.library(), ctypes.c_void_p(0), 4 if dtype == 2 else 2
    vp, i32, i64, sz = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_size_t
    lib.kf_sort_tokens.argtypes = [vp, i32, i64, vp, i32, i32, i32, i32, i32, i32, i32, vp, vp, vp, vp, vp, vp, sz, vp]
    lib.kf_sort_workspace_bytes.restype = sz
    lib.kf_combine_tokens.argtypes = [vp, i32, i64, i32, vp, vp, i32, i32, i32, vp, vp]
    lib.kf_combine_backward.argtypes = [vp, vp, i32, i64, i32, vp, vp, vp, i32, i32, i32, vp, vp, vp]
    lib.kf_pack8.argtypes = [vp, i32, i64, i32, i32, vp, vp, vp]
    lib.kf_restore8.argtypes = [vp, vp, i32, i32, i32, vp, vp, i32, i32, vp, vp]
    lib.kf_swiglu_pack8.argtypes = [vp, i32, i64, i32, i32, vp, vp, vp, vp]
    lib.kf_swiglu_backward8.argtypes = [vp, vp, vp, i32, i64, i32, i32, vp, vp, vp]
    torch.cuda.synchronize()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for offset in (0, es, 8 * es):
        new = _Guarded()
        src = torch.zeros(2 * t * h + 64, dtype=torch.float32, device="cuda")
        x = vp(src.data_ptr() + offset)
        ids = torch.randint(0, 256, (t, k), device="cuda", dtype=torch.int32)
        w = torch.ones(t, k, device="cuda")
        pr, rp, counts, starts, out = new(4 * t * k), new(4 * rows), new(1024), new(1028), new(rows * h * es, offset)
        need = lib.kf_sort_workspace_bytes(t, k, 256)
        assert lib.kf_sort_tokens(x, dtype, h, vp(ids.data_ptr()), t, k, h, 256, 0, align, rows, out, pr, rp, counts, starts,
                                  new(need), need, stream) == 0
        y, dr, dw = new(t * h * es, offset), new(rows * h * es, offset), new(4 * t * k)
        wp = vp(w.data_ptr())
        assert lib.kf_combine_tokens(out, dtype, h, rows, pr, wp, t, k, h, y, stream) == 0
        assert lib.kf_combine_backward(x, out, dtype, h, rows, pr, rp, wp, t, k, h, dr, dw, stream) == 0
        assert lib.kf_combine_backward(x, null, dtype, h, rows, pr, rp, wp, t, k, h, dr, null, stream) == 0
        assert lib.kf_combine_backward(x, out, dtype, h, rows, pr, rp, wp, t, k, h, null, dw, stream) == 0
        nb = (h + 127) // 128
        codes, exps = new(t * h, offset // es), new(t * nb)
        assert lib.kf_pack8(x, dtype, h, t, h, codes, exps, stream) == 0
        assert lib.kf_restore8(codes, exps, dtype, t, h, null, null, 0, t, new(t * h * es, offset), stream) == 0
        assert lib.kf_restore8(codes, exps, dtype, t, h, pr, rp, k, rows, out, stream) == 0
        act, codes, exps = new(t * h * es, offset), new(2 * t * h, offset // es), new(2 * t * nb)
        assert lib.kf_swiglu_pack8(x, dtype, 2 * h, t, h, act, codes, exps, stream) == 0
        assert lib.kf_swiglu_pack8(x, dtype, 2 * h, t, h, act, null, null, stream) == 0
        assert lib.kf_swiglu_backward8(codes, exps, x, dtype, h, t, h, new(2 * t * h * es, offset), act, stream) == 0
        torch.cuda.synchronize()
        new.check()


def test_rows_past_32_bit_offsets():
    """A buffer of more than 2^31 elements: the last segment's rows lie past 32-bit offsets."""
    t, h, k = 40960, 7168, 8          # 327680 rows of 7168: 2.35e9 elements
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(t, h, generator=g, device="cuda").to(torch.bfloat16)
    ids = torch.randn(t, 256, generator=g, device="cuda").topk(k, dim=1).indices.to(torch.int32)
    rows, order = train.sort_tokens(x, ids, 256)
    assert rows.numel() > 2 ** 31
    pick = torch.cat([torch.arange(3), torch.randint(0, rows.shape[0], (2000,), device="cuda", generator=g).cpu(),
                      torch.arange(rows.shape[0] - 3, rows.shape[0])]).cuda()
    pair = order.row_pair[pick].long()
    assert torch.equal(rows[pick], x[pair // k])
    assert torch.equal(order.pair_row.reshape(-1)[pair].long(), pick)
    w = torch.full((t, k), 0.125, device="cuda")
    assert torch.equal(train.combine_tokens(rows, order, w), x)       # eight equal rows times 1/8: exact
    drows, dw = train.combine_tokens_backward(x, rows, order, w)
    assert torch.equal(drows[pick], (x[pair // k].float() * 0.125).to(torch.bfloat16))
    want = (x[:64].double() ** 2).sum(1, keepdim=True)
    assert ((dw[:64].double() - want).abs() <= _dot_slack(h) * want).all()
    back = train.restore8(train.pack8(x), order)
    assert torch.equal(back[pick], train.restore8(train.pack8(x))[pair // k])
