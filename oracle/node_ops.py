"""Node-wise operators in float64: embedding and its gradient, residual dropout, the gated feed-forward block, the
root-mean-square norm, dense layers. No counterpart in the reference; stated from the formulas."""

import math

import numpy as np
import torch


def embedding(ids, table, scale):
    """scale * table[ids]; rows of NaN for ids outside the table."""
    t = table.double()
    ok = (ids >= 0) & (ids < t.shape[0])
    out = t[ids.clamp(0, t.shape[0] - 1)] * scale
    return torch.where(ok.unsqueeze(-1), out, torch.full_like(out, math.nan))


def embedding_grad(grad, ids, rows, scale, padding=None):
    """(gradient of the table, the same sum of absolute values, tokens per row)."""
    ids, g = ids.reshape(-1), grad.double().reshape(-1, grad.shape[-1])
    live = (ids >= 0) & (ids < rows)
    if padding is not None:
        live &= ids != padding
    ids, g = ids[live], g[live]
    zero = torch.zeros(rows, g.shape[1], dtype=torch.float64)
    return (zero.index_add(0, ids, g) * scale, zero.index_add(0, ids, g.abs()) * abs(scale),
            torch.bincount(ids, minlength=rows))


def philox4x32(counter, key):
    """Ten rounds of Philox4x32 (Salmon et al., 2011): counter (n, 4) and key (2) of numbers below 2^32, as (n, 4)."""
    c = [np.asarray(counter)[:, k].astype(np.uint64) for k in range(4)]
    k0, k1 = int(key[0]), int(key[1])
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ np.uint64(k0), b & low, (a >> half) ^ c[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, axis=1)


def dropout_keep(n, p, seed, offset, first=0):
    """Which of the elements first .. first + n - 1 are kept."""
    b0 = first // 4
    blocks = np.arange(b0, (first + n + 3) // 4, dtype=np.uint64)
    offset, seed = offset % 2 ** 64, seed % 2 ** 64
    counter = np.stack([blocks & np.uint64(0xFFFFFFFF), blocks >> np.uint64(32),
                        np.full_like(blocks, offset & 0xFFFFFFFF), np.full_like(blocks, offset >> 32)], axis=1)
    words = philox4x32(counter, (seed & 0xFFFFFFFF, seed >> 32)).reshape(-1)[first - 4 * b0:][:n]
    return torch.from_numpy(words >= math.floor(p * 2 ** 32))


def dropout_add(x, residual, p, seed, offset):
    keep = dropout_keep(x.numel(), p, seed, offset).view(x.shape)
    kept = torch.where(keep, x.double() / (1 - p) if p < 1 else x.double(), torch.zeros((), dtype=torch.float64))
    return kept if residual is None else residual.double() + kept


def activation(g, act):
    """act(g) and its derivative; "gelu" in the erf form."""
    if act == "gelu":
        cdf = 0.5 * torch.erfc(-g * math.sqrt(0.5))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(g)
    return (s, s * (1 - s)) if act == "sigmoid" else (g * s, s * (1 + g * (1 - s)))


def gated_feed_forward(x, w_in, w_out, act, c, s_in, s_out, grad=None, mid=0.0, end=0.0, kept=0.0, tiny=0.0):
    """{name: (value, bound)} of y and, with ``grad``, of the gradients dx, dw_in, dw_out, by the formulas in float64.

    The bound is what a float32 evaluation may be off that rounds the hidden values and the gradients of gate and up by
    ``mid`` relative to them, the outputs by ``end``, and the factors a, b that the backward pass keeps by ``kept``;
    ``tiny``: half the smallest step of the operator's type. It takes |act'| <= 1.13, |act''| <= 0.8 and 16 roundings
    for the activation's evaluation."""
    f = 2.0 ** -24
    x, w_in, w_out = x.double(), w_in.double(), w_out.double()
    width, hidden, n = x.shape[1], w_out.shape[1], x.shape[0]
    pre = s_in * (x @ w_in.t())
    e_pre = (width + 3) * f * abs(s_in) * (x.abs() @ w_in.abs().t())
    (gate, up), (e_g, e_u) = pre.chunk(2, 1), e_pre.chunk(2, 1)
    a, d = activation(gate, act)
    a, d = c * a, c * d
    b, h = d * up, a * up
    e_a = c * (1.13 * e_g + 16 * f * (1 + gate.abs()))
    e_b = c * (0.8 * e_g + 16 * f * (1 + gate.abs())) * (up.abs() + e_u) + d.abs() * e_u
    e_h = e_a * (up.abs() + e_u) + a.abs() * e_u + mid * h.abs() + tiny
    y = s_out * (h @ w_out.t())

    def bound(value, size):
        return end * value.abs() + size + tiny

    res = {"y": (y, bound(y, abs(s_out) * ((e_h + (hidden + 3) * f * h.abs()) @ w_out.abs().t())))}
    if grad is None:
        return res
    g = grad.double()
    dh = s_out * (g @ w_out)
    e_dh = (width + 3) * f * abs(s_out) * (g.abs() @ w_out.abs())
    dpre = torch.cat([dh * b, dh * a], 1)
    e_d = torch.cat([dh.abs() * (e_b + kept * b.abs()) + e_dh * (b.abs() + e_b),
                     dh.abs() * (e_a + kept * a.abs()) + e_dh * (a.abs() + e_a)], 1) + mid * dpre.abs() + tiny
    dx, dwi, dwo = s_in * (dpre @ w_in), s_in * (dpre.t() @ x), s_out * (g.t() @ h)
    res["dx"] = (dx, bound(dx, abs(s_in) * ((e_d + (2 * hidden + 3) * f * dpre.abs()) @ w_in.abs())))
    res["dw_in"] = (dwi, bound(dwi, abs(s_in) * ((e_d + (n + 3) * f * dpre.abs()).t() @ x.abs())))
    res["dw_out"] = (dwo, bound(dwo, abs(s_out) * (g.abs().t() @ (e_h + (n + 3) * f * h.abs()))))
    return res


def rms_norm_add(x, residual, weight, eps, grad=None, grad_total=None, end=0.0, tiny=0.0):
    """{name: (value, bound)} of the total (as it is stored, in x's type), y, and with ``grad`` the gradients dx and dw.

    The bound is what a float32 evaluation may be off: y is a product of three factors whose square sum has relative error
    (width / 2 + 2) 2^-24 at most, halved by the root; ``end`` and ``tiny`` as in ``gated_feed_forward``."""
    f = 2.0 ** -24
    n, width = x.shape
    total = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    t = total.double()
    w = t.new_ones(width) if weight is None else weight.double()
    r = 1 / torch.sqrt((t * t).mean(1, keepdim=True) + eps)
    e_r = (0.5 * (width / 2 + 2) + 4) * f
    y = t * r * w
    res = {"total": (t, torch.zeros_like(t)), "y": (y, (end + e_r + 2 * f) * y.abs() + tiny)}
    if grad is None:
        return res
    g, xhat = grad.double(), t * r
    gw = g * w
    mean, size = (gw * xhat).mean(1, keepdim=True), (gw * xhat).abs().mean(1, keepdim=True)
    dx = r * (gw - xhat * mean)
    e_dx = r * (((e_r + 4 * f) * (gw.abs() + 2 * xhat.abs() * mean.abs())) + xhat.abs() * (width + e_r / f) * f * size)
    if grad_total is not None:
        dx = dx + grad_total.double()
    res["dx"] = (dx, (end + f) * dx.abs() + e_dx + tiny)
    terms = g * xhat
    res["dw"] = (terms.sum(0), end * terms.sum(0).abs() + ((e_r + (n + 2) * f) * terms.abs()).sum(0) + tiny)
    return res


def e4m3_rows(y):
    """(values of the 8-bit numbers, scale) of rows of float64 values: the nearest of the e4m3 numbers, ties to even."""
    scale = y.abs().amax(1).clamp_min(2.0 ** -100) / 448
    v = y / scale[:, None]
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448), scale


def dense(x, weight, bias, residual, act, c, s, grad=None, mid=0.0, end=0.0, kept=0.0, tiny=0.0):
    """{name: (value, bound)} of y and, with ``grad``, of dx, dw and db. Roundings as in ``gated_feed_forward``."""
    f = 2.0 ** -24
    x, w = x.double(), weight.double()
    n, (out, width) = x.shape[0], w.shape
    z = s * (x @ w.t())
    e_z = (width + 3) * f * abs(s) * (x.abs() @ w.abs().t())
    if bias is not None:
        z = z + bias.double()
    e_z = e_z + f * z.abs()
    if act is None:
        a, d, e_a, e_d = z, torch.ones_like(z), e_z, torch.zeros_like(z)
    else:
        a, d = activation(z, act)
        e_a, e_d = 1.13 * e_z + 16 * f * (1 + z.abs()), 0.8 * e_z + 16 * f * (1 + z.abs())
    y, e_y = c * a, abs(c) * (e_a + 2 * f * a.abs())
    if residual is not None:
        y = y + residual.double()
        e_y = e_y + f * y.abs()
    res = {"y": (y, end * y.abs() + e_y + tiny)}
    if grad is None:
        return res
    g = grad.double()
    dz = c * g * d
    e_dz = (c * g).abs() * (e_d + (kept if act else 0.0) * d.abs() + 3 * f * d.abs())
    m_dz = e_dz + mid * dz.abs() + tiny  # as an operand
    dx, dw, db = s * (dz @ w), s * (dz.t() @ x), dz.sum(0)

    def bound(value, size):
        return end * value.abs() + size + tiny

    res["dx"] = (dx, bound(dx, abs(s) * ((m_dz + (out + 3) * f * dz.abs()) @ w.abs())))
    res["dw"] = (dw, bound(dw, abs(s) * ((m_dz + (n + 3) * f * dz.abs()).t() @ x.abs())))
    res["db"] = (db, bound(db, (e_dz + (n + 3) * f * dz.abs()).sum(0)))
    return res


def group_rows(offsets, rows):
    """The [first, end) rows of each group: offsets inside the rows, none smaller than one before it."""
    ends, last = [], 0
    for v in offsets.tolist():
        last = max(last, min(max(v, 0), rows))
        ends.append(last)
    return list(zip(ends, ends[1:]))


def grouped_dense(x, weight, offsets, bias, act, c, s, grad=None, **roundings):
    """``dense`` group by group; rows of no group are zero in y and dx."""
    rows, (groups, out, width) = x.shape[0], weight.shape
    shapes = {"y": (rows, out), "dx": (rows, width), "dw": (groups, out, width), "db": (groups, out)}
    res = {k: tuple(torch.zeros(v, dtype=torch.float64) for _ in range(2))
           for k, v in shapes.items() if k == "y" or grad is not None}
    for e, (a, b) in enumerate(group_rows(offsets, rows)):
        part = dense(x[a:b], weight[e], None if bias is None else bias[e], None, act, c, s,
                     None if grad is None else grad[a:b], **roundings)
        for k, v in part.items():
            at = slice(a, b) if k in ("y", "dx") else e
            for to, value in zip(res[k], v):
                to[at] = value
    return res
