"""64-bit restatement of the products and norms around the expert FFN, with a bound on what a kernel that sums in fp32 and
rounds once may be off, element by element.  Test infrastructure only.

The bounds count roundings.  ``U32`` = 2^-24 is half a step of fp32.  A sum of n products in fp32, in any order and with
additions that may cut instead of round (2 U32 each), is off by at most n * 2 U32 * sum |a b|.  A final rounding to type t is
off by ``half(t)`` = eps / 2 of the value, or half of the smallest subnormal."""

import torch

U32 = 2.0 ** -24
SUBNORMAL_HALF = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def half(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(ref, err, dtype):
    """Bound after a value that is off by ``err`` is rounded to ``dtype``."""
    return err + half(dtype) * (ref.abs() + err) + SUBNORMAL_HALF[dtype]


def activation(name, z):
    """act(z) and act'(z)."""
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z), (z > 0).to(z.dtype)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * torch.sigmoid(-z)
    if name == "gelu":
        c = 0.5 * torch.special.erfc(-z * 0.5 ** 0.5)
        return z * c, c + z * torch.exp(-0.5 * z * z) * (2 * torch.pi) ** -0.5
    if name == "gelu_tanh":
        a = (2 / torch.pi) ** 0.5
        c = torch.sigmoid(2 * a * (z + 0.044715 * z ** 3))
        return z * c, c + 2 * z * c * (1 - c) * a * (1 + 3 * 0.044715 * z * z)
    assert name == "none"
    return z, torch.ones_like(z)


def linear(x, w, bias, act, residual, out_dtype):
    """(y, bound of y, slope, bound of slope)"""
    xd, wd = x.double(), w.double()
    z = xd @ wd.t()
    err = 2 * x.shape[1] * U32 * (xd.abs() @ wd.abs().t())
    if bias is not None:
        z = z + bias.double()
        err = err + U32 * (z.abs() + err)
    y, slope = activation(act, z)
    y_err, s_err = err, torch.zeros_like(err)
    if act != "none":
        # |act'| <= 1.13; exp, erf and the quotient are good to a few units: 16 U32 of terms not larger than |z| and 1
        y_err = 1.13 * err + 16 * U32 * z.abs()
        # |act''| < 1
        s_err = err + 32 * U32 * (1 + z.abs())
    if act == "relu":
        s_err = (z.abs() <= err).double()  # either side of the jump
    if residual is not None:
        y = y + residual.double()
        y_err = y_err + U32 * (y.abs() + y_err)
    return y, rounded(y, y_err, out_dtype), slope, rounded(slope, s_err, x.dtype)


def _product(a, a_err, b, dtype):
    """a @ b for operands where a is known to a_err, and its bound."""
    ref = a @ b
    err = a_err @ b.abs() + 2 * a.shape[1] * U32 * ((a.abs() + a_err) @ b.abs())
    return ref, rounded(ref, err, dtype)


def linear_backward(dy, x, w, slope, dw_dtype):
    """((dx, bound), (dw, bound), (db, bound))"""
    dz = dy.double() if slope is None else dy.double() * slope.double()
    exactly = slope is None and dy.dtype == x.dtype
    dz_err = torch.zeros_like(dz) if exactly else rounded(dz, U32 * dz.abs(), x.dtype)
    dx = _product(dz, dz_err, w.double(), x.dtype)
    dw = _product(dz.t(), dz_err.t(), x.double(), dw_dtype)
    return dx, dw, (dz.sum(0), (dz.shape[0] + 1) * U32 * dz.abs().sum(0) + 2.0 ** -140)


def grouped_linear(x, w, sizes):
    parts, bounds, begin = [], [], 0
    for e, size in enumerate(sizes):
        y, b = _product(x[begin : begin + size].double(), torch.zeros(size, x.shape[1], dtype=torch.float64, device=x.device),
                        w[e].double().t(), x.dtype)
        parts.append(y)
        bounds.append(b)
        begin += size
    return torch.cat(parts), torch.cat(bounds)


def grouped_linear_backward(dy, x, w, sizes, dw_dtype):
    dx, dxb, dw, dwb, begin = [], [], [], [], 0
    for e, size in enumerate(sizes):
        rows = slice(begin, begin + size)
        begin += size
        a, b, _ = linear_backward(dy[rows], x[rows], w[e], None, dw_dtype)
        dx.append(a[0])
        dxb.append(a[1])
        dw.append(b[0])
        dwb.append(b[1])
    return (torch.cat(dx), torch.cat(dxb)), (torch.stack(dw), torch.stack(dwb))


def _row_sum(v, hidden):
    """Bound of a sum over a row by at least 32 partial sums that are then joined."""
    return (hidden / 32 + 34) * U32 * v.abs().sum(1, keepdim=True)


def layer_norm(x, weight, bias, eps):
    """((y, bound), (mean, bound), (rstd, bound))"""
    h = x.shape[1]
    xd = x.double()
    mean = xd.mean(1, keepdim=True)
    mean_err = _row_sum(xd, h) / h + 2 * U32 * mean.abs()
    d = xd - mean
    var = d.square().mean(1, keepdim=True)
    d_err = mean_err + U32 * d.abs()
    var_err = (2 * d.abs() * d_err + d_err.square()).mean(1, keepdim=True) + _row_sum(d.square(), h) / h + 3 * U32 * var
    rstd = (var + eps) ** -0.5
    # eps itself is rounded to fp32; the bound of 1/sqrt is its slope over the whole interval
    low = (var + eps - var_err - U32 * (var + 2 * eps)).clamp(min=eps / 2)
    rstd_err = 0.5 * (var_err + U32 * (var + 2 * eps)) * low ** -1.5 + 4 * U32 * rstd
    n = d * rstd
    n_err = d_err * (rstd + rstd_err) + d.abs() * rstd_err + U32 * n.abs()
    y, y_err = n, n_err
    if weight is not None:
        y_err = n_err * weight.double().abs() + U32 * (n * weight.double()).abs()
        y = n * weight.double()
    if bias is not None:
        y = y + bias.double()
        y_err = y_err + U32 * (y.abs() + y_err)
    return (y, rounded(y, y_err, x.dtype)), (mean[:, 0], mean_err[:, 0]), (rstd[:, 0], rstd_err[:, 0])


def layer_norm_backward(dy, x, mean, rstd, weight):
    """((dx, bound), (dweight, bound), (dbias, bound)), mean and rstd as given"""
    rows, hidden = x.shape
    d, m, r = dy.double(), mean.double()[:, None], rstd.double()[:, None]
    h = (x.double() - m) * r
    g = d if weight is None else d * weight.double()
    mg, mgh = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    mg_err = _row_sum(g, hidden) / hidden + 3 * U32 * g.abs().mean(1, keepdim=True)
    mgh_err = _row_sum(g * h, hidden) / hidden + 6 * U32 * (g * h).abs().mean(1, keepdim=True)
    dx = r * (g - mg - h * mgh)
    dx_err = r * (8 * U32 * (g.abs() + mg.abs() + (h * mgh).abs()) + mg_err + h.abs() * mgh_err)
    dw_err = (rows + 6) * U32 * (d * h).abs().sum(0) + 2.0 ** -140
    return (dx, rounded(dx, dx_err, x.dtype)), ((d * h).sum(0), dw_err), (d.sum(0), (rows + 2) * U32 * d.abs().sum(0) + 2.0 ** -140)


def inside(got, ref, bound):
    """None, or what is wrong: the worst element against its bound."""
    if got.shape != ref.shape:
        return f"shape {tuple(got.shape)} instead of {tuple(ref.shape)}"
    off = (got.double() - ref).abs() / bound
    off = torch.where(torch.isnan(off), torch.full_like(off, float("inf")), off)
    if off.numel() and off.max() > 1:
        i = int(off.argmax())
        return f"{int((off > 1).sum())} of {off.numel()} elements past the bound, the worst at {i}: {got.reshape(-1)[i].item()} for {ref.reshape(-1)[i].item()}, {off.max().item():.3g} times the bound"
    return None
