"""Plain 64-bit forms of the operators of language models (RMSNorm, distillation from a teacher's
top logits, verification of drafted tokens), and the error bounds their tests use.

Bounds are in units of the roundings a result passes through. U[t] is half a step of type t
relative to the value; U32 (U64 for float64 tensors) is the rounding of the accumulator. DEPTH is
the most additions any term of a row's sum passes through: up to 64 per thread (rows of up to
65536 elements on 1024 threads), 6 across a wavefront, 16 across wavefronts, and 10 for
the products around them."""

import numpy as np
import torch

U = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24, "float64": 2.0 ** -53}
# half of the smallest subnormal: what a value near zero is off by at most
TINY = {"float16": 2.0 ** -25, "bfloat16": 2.0 ** -134, "float32": 2.0 ** -150, "float64": 0.0}
DEPTH = 96
E4M3_MAX = 448.0


def u_acc(dtype):
    return U["float64"] if dtype == "float64" else U["float32"]


def acc_dtype(dtype):
    return torch.float64 if dtype == "float64" else torch.float32


def f64(t):
    return t.detach().cpu().double().numpy()


def assert_close(got, want, bound, what=""):
    """Elementwise |got - want| <= bound, NaN and infinities in the same places."""
    got, want, bound = np.broadcast_arrays(np.asarray(got, np.float64), want, bound)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what + ": NaN elsewhere"
    rest = ~fine & ~np.isnan(want)
    assert np.array_equal(got[rest], want[rest]), what + ": infinities elsewhere"
    off = np.abs(got[fine] - want[fine])
    bad = ~(off <= bound[fine])
    if bad.any():
        i = int(np.argmax(np.where(bad, off - bound[fine], -1)))
        raise AssertionError("%s: %d of %d off, worst %g against %g where a bound of %g holds" % (
            what, bad.sum(), bad.size, got[fine][i], want[fine][i], bound[fine][i]))


# ---------------------------------------------------------------- RMSNorm

def rms_norm(x, residual, gamma, eps):
    """(h, rsig, y) of float64 arrays [N, C]."""
    s = x if residual is None else x + residual
    rsig = 1.0 / np.sqrt((s * s).mean(1) + eps)
    return s, rsig, s * rsig[:, None] * gamma


def rms_norm_bounds(dtype, s, rsig, y):
    u, ua = U[dtype], u_acc(dtype)
    # rsig: half the relative error of the mean, and the square root and quotient
    stat = (DEPTH / 2 + 3) * ua
    return ((u + ua) * np.abs(s) + TINY[dtype], stat * rsig,
            (u + stat + 4 * ua) * np.abs(y) + TINY[dtype])


def quant(y, group):
    """(scale [N, groups], y / scale) of a float64 array."""
    n, c = y.shape
    width = group or c
    groups = -(-c // width)
    scale = np.empty((n, groups))
    v = np.empty_like(y)
    for g in range(groups):
        part = y[:, g * width:(g + 1) * width]
        scale[:, g] = np.maximum(np.fmax.reduce(np.abs(part), 1), 1e-30) / E4M3_MAX
        v[:, g * width:(g + 1) * width] = part / scale[:, g:g + 1]
    return scale, v


def e4m3(v):
    """Nearest e4m3 value of a float64 array within +-448 (through float32: its rounding is far
    inside the margins the callers leave)."""
    return torch.from_numpy(v).float().to(torch.float8_e4m3fn).double().numpy()


def rms_norm_grad(h, rsig, gamma, dy, dh):
    z = dy * gamma
    c = (z * h).mean(1, keepdims=True) * rsig[:, None] ** 2
    dx = rsig[:, None] * (z - h * c)
    if dh is not None:
        dx = dx + dh
    return dx, (dy * h * rsig[:, None]).sum(0)


def rms_norm_grad_bounds(dtype, h, rsig, gamma, dy, dh, dx):
    u, ua = U[dtype], u_acc(dtype)
    rs = rsig[:, None]
    z = np.abs(dy * gamma)
    spread = (z * np.abs(h)).mean(1, keepdims=True) * rs ** 2  # what the mean's terms add up to
    terms = 8 * rs * (z + np.abs(h) * spread) + (0 if dh is None else np.abs(dh))
    bound_dx = u * np.abs(dx) + ua * (terms + (DEPTH + 8) * rs * np.abs(h) * spread) + TINY[dtype]
    # a column's sum: at most one addition per row and a chain of joins no longer than that
    bound_dgamma = (len(h) + 40) * ua * (np.abs(dy * h) * rs).sum(0)
    return bound_dx, bound_dgamma


# ---------------------------------------------------------------- distillation

def teacher_shares(C, temperature, index, teacher):
    """listed [N, K], and p and log p over the listed entries (0 elsewhere)."""
    listed = (index >= 0) & (index < C) & ~(teacher == -np.inf)
    z = np.where(listed, teacher / temperature, -np.inf)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        top = np.where(listed.any(1), np.max(z, 1), 0.0)[:, None]
        e = np.where(listed, np.exp(z - top), 0.0)
        total = e.sum(1, keepdims=True)
        p = np.where(listed, e / total, 0.0)
        logp = np.where(listed, z - top - np.log(total), 0.0)
    return listed, p, logp


def log_sum_exp(x):
    top = x.max(1)
    with np.errstate(invalid="ignore", divide="ignore"):
        out = top + np.log(np.exp(x - top[:, None]).sum(1))
    return np.where(np.isneginf(top), np.nan, out)


def divisor_of(reduction, counted):
    return {"NONE": 1.0, "SUM": 1.0, "MEAN": float(len(counted)), "BATCH_MEAN": float(len(counted)),
            "VALID": float(counted.sum())}[reduction]


def distill_forward(temperature, reduction, x, index, teacher):
    """(stats [N + 1], loss per row [N], loss as the reduction gives it)."""
    n, c = x.shape
    listed, p, logp = teacher_shares(c, temperature, index, teacher)
    counted = listed.any(1)
    x = x / temperature
    lse = log_sum_exp(x)
    xk = np.take_along_axis(x, np.where(listed, index, 0), 1)
    with np.errstate(invalid="ignore"):
        terms = np.where(p != 0, p * (logp - xk + lse[:, None]), 0.0)
    rows = np.where(counted, terms.sum(1) * temperature ** 2, 0.0)
    divisor = divisor_of(reduction, counted)
    stats = np.concatenate([np.where(counted, lse, np.inf), [divisor]])
    return stats, rows, rows if reduction == "NONE" else np.array([rows.sum() / max(divisor, 1.0)])


def _largest(x):
    """Per row the largest |logit| among those that take part. One that is 800 and more below the row's
    maximum has an exponential of exactly 0 in every type (the smallest 64-bit value is exp(-745)), whatever
    parts in 10^7 its argument is off by: it adds no error, and its size (the type's lowest value, say) no bound."""
    top = np.where(np.isfinite(x), x, -np.inf).max(1)
    with np.errstate(over="ignore", invalid="ignore"):
        near = np.isfinite(x) & (x > (np.where(np.isfinite(top), top, 0.0) - 800)[:, None])
    return np.abs(np.where(near, x, 0.0)).max(1)


def distill_bounds(dtype, temperature, x, index, teacher):
    """(lse bound [N], loss bound [N]) where the logits are finite or -inf.
    lse: a sum of positive terms (DEPTH roundings), each an exponential of an argument that is off
    by 4 roundings of the largest logit r, and the final sum. loss: the shares are off by 4
    roundings of the largest teacher logit, the exponential and K additions, times the
    largest factor behind a share; the factor by that of the lse."""
    ua = u_acc(dtype)
    c, k = x.shape[1], index.shape[1]
    listed, p, logp = teacher_shares(c, temperature, index, teacher)
    xs = np.where(np.isfinite(x), x, 0.0) / temperature
    r = _largest(x / temperature)
    z = np.abs(np.where(listed, teacher / temperature, 0.0)).max(1)
    lse = log_sum_exp(x / temperature)
    b_lse = ua * (DEPTH + 20 + 8 * r + 2 * np.abs(np.nan_to_num(lse, posinf=0.0)))
    xk = np.take_along_axis(xs, np.where(listed, index, 0), 1)
    factor = np.abs(np.where(p > 0, logp - xk + np.nan_to_num(lse)[:, None], 0.0)).max(1)
    b_loss = temperature ** 2 * (b_lse + ua * ((4 * z + 30 + k) * factor + 4 * (z + r + 20)))
    return b_lse, b_loss


def distill_backward(temperature, reduction, x, index, teacher, stats, dl):
    """dx, and its share by the softmax and by the teacher, both without sign and weight."""
    n, c = x.shape
    listed, p, _ = teacher_shares(c, temperature, index, teacher)
    lse = stats[:n, None]
    ignored = np.isposinf(lse[:, 0])
    with np.errstate(invalid="ignore"):
        s = np.exp(x / temperature - lse)
    t = np.zeros_like(s)
    rows = np.repeat(np.arange(n)[:, None], index.shape[1], 1)
    np.add.at(t, (rows[listed], index[listed]), p[listed])
    s[ignored], t[ignored] = 0.0, 0.0
    w = (dl if reduction == "NONE" else np.full(n, dl[0])) * temperature / max(stats[n], 0.5)
    w = np.where(ignored, 0.0, w)[:, None]
    return w * (s - t), np.abs(w) * s, np.abs(w) * t


def distill_grad_bound(dtype, temperature, x, teacher, index, stats, dx, s, t):
    u, ua = U[dtype], u_acc(dtype)
    n = len(x)
    r = _largest(x / temperature)
    z = np.abs(np.where(np.isfinite(teacher), teacher, 0.0)).max(1) / temperature
    lse = np.abs(np.where(np.isfinite(stats[:n]), stats[:n], 0.0))
    return u * np.abs(dx) + TINY[dtype] + ua * (
        s * (20 + 8 * r + 2 * lse)[:, None] + t * (30 + 4 * z + index.shape[1])[:, None])


# ---------------------------------------------------------------- drafted tokens

def weight(p):
    return np.where((p > 0) & np.isfinite(p), p, 0.0)


def draft_verify(target, draft, drafted, lengths, u_accept, u_sample):
    """(tokens [B, K + 1], accepted [B]); target [B, K + 1, C], draft [B, K, C] or None."""
    b, places, c = target.shape
    k = places - 1
    tokens, accepted = np.full((b, places), -1, np.int64), np.zeros(b, np.int64)
    for i in range(b):
        length = k if lengths is None else min(max(int(lengths[i]), 0), k)
        n = 0
        while n < length:
            d = int(drafted[i, n])
            if not 0 <= d < c:
                break
            q = 1.0 if draft is None else float(weight(draft[i, n, d]))
            if not float(u_accept[i, n]) * q < float(weight(target[i, n, d])):
                break
            n += 1
        tokens[i, :n] = drafted[i, :n]
        accepted[i] = n
        p = weight(target[i, n])
        r = p
        if n < length:
            d = int(drafted[i, n])
            if draft is not None:
                r = np.maximum(p - weight(draft[i, n]), 0.0)
            elif 0 <= d < c:
                r = p.copy()
                r[d] = 0.0
        if not r.sum() > 0:
            r = p
        cdf = np.cumsum(r)
        u = float(u_sample[i])
        level = u * cdf[-1] if u > 0 else 0.0
        hit = np.nonzero((cdf > level) & (r > 0))[0]
        held = np.nonzero(r > 0)[0]
        tokens[i, n] = hit[0] if len(hit) else (held[-1] if len(held) else -1)
    return tokens, accepted
