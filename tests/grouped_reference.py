"""Plain 64-bit forms of the operators on grouped rows, for their tests: on the
CPU, in numpy / torch float64, from the definitions in include/qlinear.h."""
import numpy as np
import torch

BF16, F32, I32, FP8, I8, F16 = 0, 1, 2, 3, 4, 5
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}


def group(ids, groups):
    """order, slots, offsets of flat ids by plain loops."""
    ids = np.asarray(ids).reshape(-1)
    order, slots, offsets = [], np.full(ids.size, -1, np.int32), [0]
    for g in range(groups):
        for i in np.nonzero(ids == g)[0]:
            slots[i] = len(order)
            order.append(i)
        offsets.append(len(order))
    order = np.array(order + [-1] * (ids.size - len(order)), np.int32)
    return order, slots, np.array(offsets, np.int32)


def route(logits, top_k, normalize):
    """ids, weights (float64) of float64 logits [tokens, experts]."""
    tokens, _ = logits.shape
    ids = np.full((tokens, top_k), -1, np.int32)
    weights = np.zeros((tokens, top_k))
    for t in range(tokens):
        row = logits[t]
        live = [e for e in range(row.size) if row[e] > -np.inf]  # NaN compares false
        if not live:
            continue
        best = sorted(live, key=lambda e: (-row[e], e))[:top_k]
        peak = row[best[0]]
        p = {e: 1.0 if row[e] == peak else float(np.exp(row[e] - peak)) for e in live}
        total = sum(p[e] for e in (best if normalize else live))
        for j, e in enumerate(best):
            ids[t, j], weights[t, j] = e, p[e] / total
    return ids, weights


def code_values(codes, fmt):
    """uint8 codes -> float64 values."""
    t = torch.as_tensor(codes)
    return t.view(torch.int8 if fmt == I8 else torch.float8_e4m3fn).to(torch.float32).double()


def expert_rows(x, sx, w, sw, fmt, group, out_dtype):
    """One expert's y [rows, N] in out_dtype (INT8 per channel: the exact bits)
    or (y64, bound): the 64-bit result and how far the kernel may be off."""
    xv, wv = code_values(x, fmt), code_values(w, fmt)
    K = xv.shape[1]
    if fmt == I8 and not group:
        acc = (xv @ wv.t()).float()  # integers below 2^31: the kernel's int -> fp32 rounding
        return ((acc * sx[:, None]) * sw[None, :]).to(out_dtype)
    if group:
        at = torch.arange(K) // group
        xv, wv = xv * sx.double().t()[:, at], wv * sw.double().t()[:, at]
    else:
        xv, wv = xv * sx.double()[:, None], wv * sw.double()[:, None]
    y = xv @ wv.t()
    # Each of K products enters a sum once; every addition (and the scales' few
    # products) is off by at most one unit 2^-23 of a partial sum of magnitudes.
    bound = (K + 6) * 2.0 ** -23 * (xv.abs() @ wv.abs().t())
    if fmt == FP8:
        # The FP8 matrix instruction adds the products of eight consecutive K in units
        # of 2^-13 of the largest of them, dropping what is below (measured: beside
        # products of 2^16 that cancel, one of 2^3 is kept and one of 2^2 lost, in any
        # two places of the same eight; in other eights 2^-8 is kept). The largest is
        # at most the product of both operands' largest in those eight.
        most = lambda v: torch.nn.functional.pad(v.abs(), (0, -K % 8)).unflatten(1, (-1, 8)).amax(2)
        bound = bound + 8 * 2.0 ** -13 * (most(xv) @ most(wv).t())
    return y, bound + HALF_STEP[out_dtype] * (y.abs() + bound) + 1e-38


def adapter_rows(x, a, b, base, scale):
    """y64 and its bound for rows x of one adapter (a [r, K], b [N, r] cut to its rank)."""
    dtype, (r, K) = x.dtype, a.shape
    xd, ad, bd = x.double(), a.double(), b.double()
    t = xd @ ad.t()
    y = base.double() + scale * (t @ bd.t())
    unit = 2.0 ** -23
    split = HALF_STEP[dtype] ** 2  # hi is off by half a step of t, lo by half a step of that
    mags = (xd.abs() @ ad.abs().t()) @ bd.abs().t()
    bound = abs(scale) * ((K + 1) * unit * mags + (split + (2 * r + 4) * unit) * (t.abs() @ bd.abs().t()))
    bound = bound + 2 * unit * base.double().abs() + HALF_STEP[dtype] * y.abs()
    return y, bound + HALF_STEP[dtype] * bound + torch.finfo(dtype).tiny
