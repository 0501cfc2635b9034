"""The training operators in 64 bits, plainly, on the CPU; and the tolerances of a kernel against them.

A kernel's result is one fp32 computation rounded once to its type.  A rounding to a type is
off by at most half a step, ``finfo(t).eps / 2`` of the value (and half the smallest subnormal
step near zero); every fp32 operation adds 2^-24 of its own result.
"""
import torch

BLOCK = 128


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half the step between the subnormals of a type: what rounding costs next to zero."""
    return torch.finfo(dtype).smallest_normal * half_step(dtype)


def close(got, ref, dtype, slack):
    """Every element within one rounding to ``dtype`` of a value within ``slack`` of ``ref``.

    A value of at least the largest number and half a step rounds to infinity, of the value's sign.
    """
    got, ref = got.double().cpu(), ref.double()
    beyond = torch.finfo(dtype).max * (1 + half_step(dtype) / 2)
    far = ref.abs() + slack >= beyond                       # may be infinite
    assert (got[far & (ref.abs() - slack >= beyond)].isinf()).all()
    inf = far & got.isinf() & (got.sign() == ref.sign())
    got = torch.where(inf, ref, got)
    limit = slack + half_step(dtype) * (ref.abs() + slack) + smallest(dtype)
    bad = ~((got - ref).abs() <= limit)
    assert not bad.any(), (int(bad.sum()), float(((got - ref).abs() / limit).nan_to_num(1e30).max()))


def order(ids, experts, offset, align, rows):
    """(pair_row, row_pair, counts, starts) by one pass over the pairs per expert."""
    t, k = ids.shape
    flat = ids.reshape(-1).tolist()
    pair_row, row_pair = [-1] * (t * k), [-1] * rows
    counts, starts, at = [], [0], 0
    for e in range(offset, offset + experts):
        mine = [p for p, i in enumerate(flat) if i == e]
        for j, p in enumerate(mine):
            if at + j < rows:
                pair_row[p] = at + j
                row_pair[at + j] = p
        counts.append(len(mine))
        at = (at + len(mine) + align - 1) // align * align
        starts.append(min(at, rows))
    i32 = torch.int32
    return (torch.tensor(pair_row, dtype=i32).reshape(t, k), torch.tensor(row_pair, dtype=i32),
            torch.tensor(counts, dtype=i32), torch.tensor(starts, dtype=i32))


def worst_rows(t, k, experts, align):
    return (t * k + min(t * k, experts) * (align - 1)) // align * align


def gather(x, row_pair, k):
    out = torch.zeros(row_pair.numel(), x.shape[1], dtype=x.dtype)
    has = row_pair >= 0
    out[has] = x[(row_pair[has] // k).long()]
    return out


def combine(rows, pair_row, weight=None):
    """(out, sum of the terms' magnitudes), both f64."""
    t, k = pair_row.shape
    out = torch.zeros(t, rows.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(out)
    for j in range(k):
        has = pair_row[:, j] >= 0
        term = rows[pair_row[has, j].long()].double()
        if weight is not None:
            term = term * weight[has, j, None].double()
        out[has] += term
        mag[has] += term.abs()
    return out, mag


def combine_grads(dout, rows, pair_row, row_pair, weight):
    """(drows, dweight, sum of the magnitudes in each dweight), all f64."""
    t, k = pair_row.shape
    g, w = dout.double(), weight.double()
    drows = torch.zeros(row_pair.numel(), dout.shape[1], dtype=torch.float64)
    dw = torch.zeros(t, k, dtype=torch.float64)
    mag = torch.zeros_like(dw)
    for j in range(k):
        has = pair_row[:, j] >= 0
        at = pair_row[has, j].long()
        drows[at] = g[has] * w[has, j, None]
        prod = g[has] * rows[at].double()
        dw[has, j], mag[has, j] = prod.sum(1), prod.abs().sum(1)
    return drows, dw, mag


def to_8_bits(x):
    """(values f64, exponents): e4m3 codes times 2^e per row and 128 columns; values not finite become NaN."""
    r, width = x.shape
    top = 8 if x.dtype == torch.float16 else 120
    out = torch.empty(r, width, dtype=torch.float64)
    exps = []
    for c in range(0, width, BLOCK):
        b = x[:, c:c + BLOCK].double()
        fine = torch.isfinite(b)
        amax = torch.where(fine, b.abs(), torch.zeros_like(b)).amax(1)
        e = torch.full((r,), -126, dtype=torch.float64)
        for _ in range(250):                    # the smallest exponent, by search
            e = torch.where(amax > 448.0 * torch.exp2(e), e + 1, e)
        v = b * torch.exp2(-e)[:, None]         # exact
        limit = torch.where(e == top, 240.0, 448.0)[:, None].double()
        v = torch.where(fine, torch.maximum(torch.minimum(v, limit), -limit), torch.zeros_like(v))
        q = v.float().to(torch.float8_e4m3fn).double() * torch.exp2(e)[:, None]
        out[:, c:c + BLOCK] = torch.where(fine, q, torch.full_like(q, float("nan")))
        exps.append(e)
    return out, torch.stack(exps, 1)


def swiglu(u, g):
    return u * g * torch.sigmoid(g)


def swiglu_grads(u, g, d):
    """(du, dg, act, magnitude behind dg) of kept f64 values and dL/dact."""
    s = torch.sigmoid(g)
    return (d * g * s, d * u * s * (1 + g * (1 - s)), u * g * s, (d * u * s).abs() * (1 + g.abs() * (1 - s)))


def route_weights(logits, ids, factor):
    """The routing weights of chosen experts, f64 (ids outside [0, 256) count as no choice)."""
    has = (ids >= 0) & (ids < 256)
    s = torch.where(has, torch.sigmoid(logits.double().gather(1, ids.clamp(0, 255).long())), torch.zeros((), dtype=torch.float64))
    return factor * s / (s.sum(1, keepdim=True) + 1e-20)


def route_grad(logits, ids, g, factor):
    """(gradient [T, 256], magnitude behind each element), f64."""
    has = (ids >= 0) & (ids < 256)
    at = ids.clamp(0, 255).long()
    x = logits.double().gather(1, at)
    s = torch.where(has, torch.sigmoid(x), torch.zeros_like(x))
    p = s / (s.sum(1, keepdim=True) + 1e-20)
    g = torch.where(has, g.double(), torch.zeros_like(x))
    scale = factor * p * torch.sigmoid(-x)
    d = scale * (g - (g * p).sum(1, keepdim=True))
    m = scale.abs() * (g.abs() + (g * p).abs().sum(1, keepdim=True))
    zero = torch.zeros(logits.shape, dtype=torch.float64)
    return zero.scatter_add(1, at, d), zero.scatter_add(1, at, m)
