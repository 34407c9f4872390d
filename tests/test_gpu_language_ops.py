"""The operators of language models on the GPU against their plain 64-bit forms (language_ops.py),
elementwise within bounds that count roundings."""

import numpy as np
import pytest
import torch

from tests import language_ops as L

pytestmark = pytest.mark.gpu

DTYPES = ["float16", "bfloat16", "float32", "float64"]


def _K():
    from dragon_amd import kernels
    return kernels


def _make(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * scale).to(getattr(torch, dtype)).cuda()


def _odd(t, lead=1):
    """The same values, contiguous, `lead` elements behind an allocation's start."""
    flat = torch.empty(t.numel() + lead, dtype=t.dtype, device=t.device)
    out = flat[lead:].view(t.shape)
    out.copy_(t)
    return out


# ---------------------------------------------------------------- RMSNorm forward

ROWS = [(1, 1), (3, 7), (2, 64), (5, 100), (1, 4096), (130, 257), (70, 512), (33, 1000), (9, 2048), (1025, 520),
        (7, 5003), (4, 8192), (3, 16384), (2, 20001), (2, 65536)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", ROWS)
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm(shape, dtype, residual):
    N, C = shape
    x, r = _make(shape, dtype, 1), _make(shape, dtype, 2, 3.0) if residual else None
    gamma = (1 + _make((C,), "float64", 3, 0.3)).to(L.acc_dtype(dtype))
    h, y = torch.empty_like(x), torch.empty_like(x)
    rsig = torch.empty(N, dtype=gamma.dtype, device="cuda")
    _K().rms_norm(N, C, 1e-5, x, r, gamma, h, rsig, y)
    s, rs, want = L.rms_norm(L.f64(x), None if r is None else L.f64(r), L.f64(gamma), float(np.float32(1e-5)))
    bh, brs, by = L.rms_norm_bounds(dtype, s, rs, want)
    L.assert_close(L.f64(h), s, bh, "h")
    L.assert_close(L.f64(rsig), rs, brs, "rsig")
    L.assert_close(L.f64(y), want, by, "y")


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("shape", [(40, 1024), (3, 4096), (6, 33), (2, 20000), (5, 8192)])
def test_rms_norm_odd_addresses_and_optional_outputs_change_no_bit(shape, dtype):
    """The sums' order may differ with the alignment, so values are compared within the bounds; with
    the alignment given, leaving an output out or laying it on an input changes nothing."""
    N, C = shape
    x, r = _make(shape, dtype, 4), _make(shape, dtype, 5)
    gamma = torch.rand(C, device="cuda") + 0.5
    s, rs, want = L.rms_norm(L.f64(x), L.f64(r), L.f64(gamma), float(np.float32(1e-6)))
    bh, brs, by = L.rms_norm_bounds(dtype, s, rs, want)
    K = _K()
    h, y, rsig = torch.empty_like(x), torch.empty_like(x), torch.empty(N, device="cuda")
    K.rms_norm(N, C, 1e-6, x, r, gamma, h, rsig, y)
    xo, ro, go, ho, yo = _odd(x), _odd(r, 3), _odd(gamma), _odd(h, 5), _odd(y, 2)
    ho.zero_(), yo.zero_()
    K.rms_norm(N, C, 1e-6, xo, ro, go, ho, rsig, yo)
    L.assert_close(L.f64(ho), s, bh, "h")
    L.assert_close(L.f64(yo), want, by, "y")
    bare = torch.empty_like(y)
    K.rms_norm(N, C, 1e-6, x, r, gamma, None, None, bare)
    assert torch.equal(bare, y)
    # the residual stream and the input updated in place, either way round
    for first in (True, False):
        x2, r2 = x.clone(), r.clone()
        K.rms_norm(N, C, 1e-6, x2, r2, gamma, r2 if first else x2, rsig, x2 if first else r2)
        assert torch.equal(r2 if first else x2, h) and torch.equal(x2 if first else r2, y)


def test_rms_norm_zero_rows_and_values_that_are_not_finite():
    K = _K()
    N, C = 6, 300
    for dtype in DTYPES:
        x = _make((N, C), dtype, 6)
        x[1] = 0
        x[2, 5], x[3, 7], x[4, 9] = float("nan"), float("inf"), float("-inf")
        gamma = torch.ones(C, dtype=L.acc_dtype(dtype), device="cuda")
        y, h, rsig = torch.empty_like(x), torch.empty_like(x), torch.empty(N, dtype=gamma.dtype, device="cuda")
        K.rms_norm(N, C, 1e-5, x, None, gamma, h, rsig, y)
        with np.errstate(invalid="ignore"):
            s, rs, want = L.rms_norm(L.f64(x), None, L.f64(gamma), float(np.float32(1e-5)))
            bh, brs, by = L.rms_norm_bounds(dtype, s, rs, want)
        L.assert_close(L.f64(y), want, by, "y")
        L.assert_close(L.f64(rsig), rs, brs, "rsig")
        assert torch.equal(h.nan_to_num(7), x.nan_to_num(7))


def test_rms_norm_nothing_behind_the_last_row_is_written():
    K = _K()
    for N, C, dtype in ((3, 1000, torch.bfloat16), (5, 33, torch.float32), (1, 4099, torch.float16)):
        x = torch.randn(N, C, device="cuda").to(dtype)
        gamma = torch.ones(C, device="cuda")
        y, h = (torch.full((N * C + 64,), 7.0, dtype=dtype, device="cuda") for _ in range(2))
        q = torch.full((N * C + 64,), 7, dtype=torch.uint8, device="cuda")
        rsig, scale = (torch.full((N * (C // 32 + 1) + 8,), 7.0, device="cuda") for _ in range(2))
        K.rms_norm(N, C, 1e-5, x, x, gamma, h, rsig, y)
        assert (y[N * C:] == 7).all() and (h[N * C:] == 7).all() and (rsig[N:] == 7).all()
        K.rms_norm_quant(N, C, 32, 1e-5, x, x, gamma, h, rsig, q, scale)
        assert (q[N * C:] == 7).all() and (h[N * C:] == 7).all() and (rsig[N:] == 7).all()
        assert (scale[N * -(-C // 32):] == 7).all()


def test_rms_norm_offsets_beyond_32_bits():
    """More than 2^32 elements: rows are addressed with 64 bits. Checked on the last rows."""
    K = _K()
    C = 8192
    N = (1 << 32) // C + 3
    x = torch.empty((N, C), dtype=torch.bfloat16, device="cuda").normal_()
    gamma = torch.rand(C, device="cuda") + 0.5
    y = torch.empty_like(x)
    K.rms_norm(N, C, 1e-5, x, None, gamma, None, None, y)
    s, rs, want = L.rms_norm(L.f64(x[-4:]), None, L.f64(gamma), float(np.float32(1e-5)))
    L.assert_close(L.f64(y[-4:]), want, L.rms_norm_bounds("bfloat16", s, rs, want)[2], "y")


# ---------------------------------------------------------------- RMSNorm in 8 bits

@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (1, 4096), (70, 512), (33, 1000), (9, 2050), (1025, 520),
                                   (7, 5003), (4, 8192), (2, 20001), (300, 96), (65, 256)])
@pytest.mark.parametrize("group", [0, 32, 128, 256])
def test_rms_norm_quant(shape, dtype, group):
    N, C = shape
    x, r = _make(shape, dtype, 11), _make(shape, dtype, 12, 2.0)
    gamma = 1 + _make((C,), "float32", 13, 0.3)
    h = torch.empty_like(x)
    q = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
    groups = -(-C // group) if group else 1
    scale, rsig = torch.empty((N, groups), device="cuda"), torch.empty(N, device="cuda")
    _K().rms_norm_quant(N, C, group, 1e-5, x, r, gamma, h, rsig, q, scale)
    _check_quant(dtype, group, x, r, gamma, h, rsig, q, scale)


def _check_quant(dtype, group, x, r, gamma, h, rsig, q, scale):
    s, rs, y = L.rms_norm(L.f64(x), L.f64(r), L.f64(gamma), float(np.float32(1e-5)))
    bh, brs, _ = L.rms_norm_bounds(dtype, s, rs, y)
    L.assert_close(L.f64(h), s, bh, "h")
    L.assert_close(L.f64(rsig), rs, brs, "rsig")
    want_scale, v = L.quant(y, group)
    # y's own roundings in the accumulator (statistic, two products), and a quotient
    rel = (L.DEPTH / 2 + 8) * L.U["float32"]
    L.assert_close(L.f64(scale), want_scale, rel * want_scale, "scale")
    # the code is the nearest one of a value that is off by those of y and of the scale
    got = q.cpu().float().double().numpy()
    lo, hi = L.e4m3(v * (1 - 2 * rel)), L.e4m3(np.clip(v * (1 + 2 * rel), -448, 448))
    assert ((got >= np.minimum(lo, hi)) & (got <= np.maximum(lo, hi))).all()


@pytest.mark.parametrize("group", [0, 64])
def test_rms_norm_quant_odd_addresses_in_place_and_zero_rows(group):
    K = _K()
    for dtype in ("bfloat16", "float32"):
        for N, C in ((6, 1000), (5, 4096), (3, 30000)):
            x, r = _make((N, C), dtype, 21), _make((N, C), dtype, 22)
            x[1], r[1] = 0, 0
            gamma = torch.rand(C, device="cuda") + 0.5
            groups = -(-C // group) if group else 1
            q = torch.empty((N, C), dtype=torch.uint8, device="cuda")
            h, scale, rsig = torch.empty_like(x), torch.empty((N, groups), device="cuda"), torch.empty(N, device="cuda")
            K.rms_norm_quant(N, C, group, 1e-5, x, r, gamma, h, rsig, q, scale)
            _check_quant(dtype, group, x, r, gamma, h, rsig, q.view(torch.float8_e4m3fn), scale)
            assert (q[1] & 127 == 0).all() and torch.equal(scale[1], torch.full_like(scale[1], np.float32(1e-30) / np.float32(448)))
            xo, ro, go, qo = _odd(x), _odd(r, 3), _odd(gamma), _odd(q, 1)
            K.rms_norm_quant(N, C, group, 1e-5, xo, ro, go, ro, rsig, qo, scale)
            _check_quant(dtype, group, x, r, gamma, ro, rsig, qo.view(torch.float8_e4m3fn), scale)


def test_rms_norm_quant_nan_keeps_its_code_and_spares_the_other_groups():
    K = _K()
    N, C = 3, 512
    x = _make((N, C), "float32", 23)
    gamma = torch.ones(C, device="cuda")
    gamma[70] = float("nan")
    q, scale = torch.empty((N, C), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((N, 8), device="cuda")
    K.rms_norm_quant(N, C, 64, 1e-5, x, None, gamma, None, None, q, scale)
    nan = q.float().isnan()
    assert nan[:, 70].all() and int(nan.sum()) == N and scale.isfinite().all()
    x[1, 3] = float("nan")  # the whole row has no norm
    K.rms_norm_quant(N, C, 64, 1e-5, x, None, gamma, None, None, q, scale)
    assert q[1].float().isnan().all() and not q[0, :64].float().isnan().any()


# ---------------------------------------------------------------- RMSNorm gradient

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (1, 4096), (700, 512), (33, 1000), (9, 2050), (1025, 520),
                                   (7, 5003), (40, 8192), (300, 1001), (3, 40000), (2049, 96), (600, 4096)])
@pytest.mark.parametrize("through_h", [False, True])
def test_rms_norm_grad(shape, dtype, through_h):
    N, C = shape
    h, dy = _make(shape, dtype, 31, 2.0), _make(shape, dtype, 32)
    dh = _make(shape, dtype, 33) if through_h else None
    gamma = (1 + _make((C,), "float64", 34, 0.3)).to(L.acc_dtype(dtype))
    _, rs, _ = L.rms_norm(L.f64(h), None, L.f64(gamma), 1e-5)
    rsig = torch.from_numpy(rs).to(gamma.dtype).cuda()
    dgamma, dx = torch.full_like(gamma, 9.0), torch.empty_like(h)
    _K().rms_norm_grad(N, C, h, rsig, gamma, dy, dh, dgamma, dx)
    _check_grad(dtype, h, rsig, gamma, dy, dh, dgamma, dx)


def _check_grad(dtype, h, rsig, gamma, dy, dh, dgamma, dx):
    args = (L.f64(h), L.f64(rsig), L.f64(gamma), L.f64(dy), None if dh is None else L.f64(dh))
    want, want_g = L.rms_norm_grad(*args)
    bx, bg = L.rms_norm_grad_bounds(dtype, *args, want)
    L.assert_close(L.f64(dx), want, bx, "dx")
    L.assert_close(L.f64(dgamma), want_g, bg, "dgamma")


def test_rms_norm_grad_against_differences():
    """d sum(y * dy + h * dh) / dx and / dgamma by central differences of the plain form in 64 bits."""
    rng = np.random.default_rng(0)
    N, C, step = 3, 20, 1e-6
    x, r, dy, dh = (rng.standard_normal((N, C)) for _ in range(4))
    gamma = rng.uniform(0.5, 1.5, C)

    def value(x, gamma):
        s, _, y = L.rms_norm(x, r, gamma, 1e-5)
        return (y * dy + s * dh).sum()

    s, rs, _ = L.rms_norm(x, r, gamma, 1e-5)
    t = [torch.from_numpy(a).cuda() for a in (s, rs, gamma, dy, dh)]
    dgamma, dx = torch.empty(C, dtype=torch.float64, device="cuda"), torch.empty(N, C, dtype=torch.float64, device="cuda")
    _K().rms_norm_grad(N, C, *t, dgamma, dx)
    for i in range(N):
        for j in range(C):
            d = np.zeros((N, C))
            d[i, j] = step
            slope = (value(x + d, gamma) - value(x - d, gamma)) / (2 * step)
            # second differences of order step^2, and 64-bit roundings of a value of order 100 over the step
            assert abs(slope - float(dx[i, j])) < 1e-7
    for j in range(C):
        d = np.zeros(C)
        d[j] = step
        assert abs((value(x, gamma + d) - value(x, gamma - d)) / (2 * step) - float(dgamma[j])) < 1e-7


@pytest.mark.parametrize("shape", [(50, 1000), (300, 4096), (4, 50000), (2100, 520)])
def test_rms_norm_grad_in_place_odd_addresses_and_equal_bits(shape):
    K = _K()
    N, C = shape
    for dtype in ("bfloat16", "float32"):
        h, dy, dh = (_make(shape, dtype, 41 + i) for i in range(3))
        gamma, rsig = torch.rand(C, device="cuda") + 0.5, torch.rand(N, device="cuda") + 0.5
        dgamma, dx = torch.empty(C, device="cuda"), torch.empty_like(h)
        K.rms_norm_grad(N, C, h, rsig, gamma, dy, dh, dgamma, dx)
        _check_grad(dtype, h, rsig, gamma, dy, dh, dgamma, dx)
        for target in (0, 1):
            dy2, dh2, dg2 = dy.clone(), dh.clone(), torch.empty_like(dgamma)
            out = dy2 if target == 0 else dh2
            K.rms_norm_grad(N, C, h, rsig, gamma, dy2, dh2, dg2, out)
            assert torch.equal(out, dx) and torch.equal(dg2, dgamma)
        odd = [_odd(t, i + 1) for i, t in enumerate((h, rsig, gamma, dy, dh, dgamma, dx))]
        K.rms_norm_grad(N, C, *odd)
        _check_grad(dtype, h, rsig, gamma, dy, dh, odd[5], odd[6])


def test_rms_norm_grad_of_no_rows_is_zero():
    dgamma = torch.full((64,), 3.0, device="cuda")
    e = torch.empty((0, 64), device="cuda")
    _K().rms_norm_grad(0, 64, e, torch.empty(0, device="cuda"), torch.ones(64, device="cuda"), e, None, dgamma, e)
    assert (dgamma == 0).all()


# ---------------------------------------------------------------- distillation

def _distill_case(N, C, K, dtype, index_dtype, seed, scale=3.0):
    """Logits, classes (some absent, some twice, some rows without any) and a teacher's logits."""
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((N, C)) * scale)
    index = rng.integers(0, C, (N, K))
    index[rng.random((N, K)) < 0.15] = -1
    if K > 1:
        twice = rng.random(N) < 0.3
        index[twice, 1] = index[twice, 0]
    if N > 2:
        index[rng.integers(0, N)] = -1
        index[rng.integers(0, N), 0] = C  # behind the vocabulary
    teacher = rng.standard_normal((N, K)) * 2 + 5
    teacher[rng.random((N, K)) < 0.05] = -np.inf
    return (torch.from_numpy(x).to(getattr(torch, dtype)).cuda(), torch.from_numpy(index).to(index_dtype).cuda(),
            torch.from_numpy(teacher).to(L.acc_dtype(dtype)).cuda())


def _run_distill(x, index, teacher, temperature, reduction, dl, in_place=False):
    K = _K()
    N, C = x.shape
    k = index.shape[1]
    acc = teacher.dtype
    stats = torch.full((N + 1,), 9.0, dtype=acc, device="cuda")
    loss = torch.full((N if reduction == "NONE" else 1,), 9.0, dtype=acc, device="cuda")
    K.topk_distillation_loss_forward(N, C, k, temperature, reduction, x, index, teacher, stats, loss)
    dx = x.clone() if in_place else torch.empty_like(x)
    K.topk_distillation_loss_backward(N, C, k, temperature, reduction, dx if in_place else x, index, teacher, stats,
                                      dl, dx)
    return stats, loss, dx


def _check_distill(dtype, x, index, teacher, temperature, reduction, dl, stats, loss, dx):
    a = (L.f64(x), index.cpu().numpy().astype(np.int64), L.f64(teacher))
    N = len(a[0])
    ws, rows, wl = L.distill_forward(temperature, reduction, *a)
    b_lse, b_rows = L.distill_bounds(dtype, temperature, *a)
    L.assert_close(L.f64(stats)[:N], ws[:N], b_lse, "lse")
    assert float(stats[N]) == ws[N]
    ua = L.u_acc(dtype)
    if reduction == "NONE":
        L.assert_close(L.f64(loss), wl, b_rows, "loss")
    else:
        counted = np.isfinite(ws[:N])
        # the rows' own bounds, and N additions at most of what they add up to
        bound = (b_rows[counted].sum() + (N + 8) * ua * np.abs(rows).sum()) / max(ws[N], 1.0)
        L.assert_close(L.f64(loss), wl, bound, "loss")
    if dx is not None:
        # the gradient as the formula of what it is given: its own statistics
        got_stats = L.f64(stats)
        want, s, t = L.distill_backward(temperature, reduction, *a, got_stats, L.f64(dl))
        L.assert_close(L.f64(dx), want, L.distill_grad_bound(dtype, temperature, a[0], a[2], a[1], got_stats, want, s, t),
                       "dx")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1), (4, 10, 3), (1, 32000, 20), (37, 1000, 64), (130, 257, 5), (3, 50257, 32),
                                   (5, 8192, 1024), (2, 200001, 33), (600, 2000, 8), (12, 131072, 20)])
@pytest.mark.parametrize("reduction", ["VALID", "NONE", "MEAN"])
def test_distillation(shape, dtype, reduction):
    N, C, k = shape
    index_dtype = torch.int32 if (N + k) % 2 else torch.int64
    x, index, teacher = _distill_case(N, C, k, dtype, index_dtype, N + C)
    dl = (torch.rand(N if reduction == "NONE" else 1, device="cuda") + 0.5).to(teacher.dtype)
    temperature = 1.0 if C % 2 else 2.0
    stats, loss, dx = _run_distill(x, index, teacher, temperature, reduction, dl)
    _check_distill(dtype, x, index, teacher, temperature, reduction, dl, stats, loss, dx)


@pytest.mark.parametrize("shape", [(6, 1000, 7), (3, 32000, 64), (2, 100003, 16)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_distillation_in_place_odd_addresses_and_equal_bits(shape, dtype):
    N, C, k = shape
    x, index, teacher = _distill_case(N, C, k, dtype, torch.int64, 5)
    dl = torch.full((1,), 0.7, device="cuda")
    first = _run_distill(x, index, teacher, 1.5, "SUM", dl)
    for again in (_run_distill(x, index, teacher, 1.5, "SUM", dl), _run_distill(x, index, teacher, 1.5, "SUM", dl, True)):
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    xo, io, to = _odd(x, 1), _odd(index, 1), _odd(teacher, 1)
    stats, loss, dx = _run_distill(xo, io, to, 1.5, "SUM", _odd(dl))
    _check_distill(dtype, x, index, teacher, 1.5, "SUM", dl, stats, loss, dx)


def test_distillation_masked_vocabulary_empty_rows_and_values_that_are_not_finite():
    N, C, k = 9, 500, 6
    inf, nan = float("inf"), float("nan")
    for dtype in DTYPES:
        x, index, teacher = _distill_case(N, C, k, dtype, torch.int32, 77)
        index.copy_(torch.arange(k).expand(N, k))
        teacher.copy_(torch.arange(k).expand(N, k).to(teacher.dtype))
        low = torch.finfo(x.dtype).min
        x[0, 100:] = -inf                        # a masked vocabulary
        x[1, 100:] = low                         # the same with the type's lowest value
        x[2], index[2] = nan, -1                 # an ignored row of garbage
        x[3], teacher[3] = inf, -inf             # another, by its teacher
        x[4] = -inf                              # no distribution
        x[5, 499] = nan
        x[6, 499] = inf
        x[7, 2] = -inf                           # a class the teacher gives weight
        teacher[8, 3] = nan
        dl = torch.full((N,), 0.5, dtype=teacher.dtype, device="cuda")
        stats, loss, dx = _run_distill(x, index, teacher, 1.0, "NONE", dl)
        got, st, grad = L.f64(loss), L.f64(stats), L.f64(dx)
        assert np.isfinite(got[[0, 1]]).all() and np.isfinite(grad[[0, 1]]).all()
        assert (grad[0, 100:] == 0).all() and (grad[1, 100:] == 0).all()
        for i in (2, 3):
            assert got[i] == 0 and (grad[i] == 0).all() and np.isposinf(st[i])
        for i in (4, 5, 6):
            assert np.isnan(got[i]) and np.isnan(grad[i]).all()
        assert np.isposinf(got[7]) and np.isfinite(grad[7]).all()
        assert np.isnan(got[8])
        # the same rows in place, and what remains of them by the bounds
        keep = [0, 1, 2, 3]
        part = _run_distill(x[keep], index[keep], teacher[keep], 1.0, "VALID", dl[:1])
        assert float(part[0][4]) == 2.0
        xs = x[keep].clone()
        xs[2:] = 0  # what an ignored row holds does not matter
        _check_distill(dtype, xs, index[keep], teacher[keep], 1.0, "VALID", dl[:1], *part)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(6, 130, 3), (6, 4200, 300), (6, 9001, 5), (6, 70001, 9)])
@pytest.mark.parametrize("temperature", [0.75, 1.0, 1.5, 2.0])
def test_distillation_of_rows_masked_all_over_and_of_logits_far_from_zero(dtype, shape, temperature):
    """Loss and gradient depend on differences of logits alone, so the plain form is that of the rows
    less their largest logit (exact in 64 bits: they are on one grid), with its bounds. Its log-sum is
    that of the rows less largest / t, two roundings of it and clipped to the type's range."""
    N, C, k = shape
    x, index, teacher = _distill_case(N, C, k, dtype, torch.int32, 5, 2.0)
    g = torch.Generator().manual_seed(3)
    index.copy_(torch.randint(0, C // 3, (N, k), generator=g))
    teacher.nan_to_num_(neginf=0.0)
    low = torch.finfo(x.dtype).min
    x[0] = low
    x[1] = low
    x[1, C // 2:] = -float("inf")
    x[2] += 30000
    x[3] -= 30000
    x[4, C // 3:] = low  # a masked tail: an ordinary row
    x[5] = low
    x[5, C - 1] = low / 2  # one class is left, far from zero itself
    index[5] = C - 1
    dl = torch.rand(N, generator=g).to(teacher.dtype).cuda()
    stats, loss, dx = _run_distill(x, index, teacher, temperature, "NONE", dl)
    a = [L.f64(x), index.cpu().numpy().astype(np.int64), L.f64(teacher)]
    top = a[0].max(1)
    top[4] = 0.0
    with np.errstate(over="ignore"):
        a[0] -= top[:, None]
    ws, rows, _ = L.distill_forward(temperature, "NONE", *a)
    b_lse, b_rows = L.distill_bounds(dtype, temperature, *a)
    ua = L.u_acc(dtype)
    most = float(torch.finfo(teacher.dtype).max)
    with np.errstate(over="ignore"):
        lse = np.clip(top / temperature + ws[:N], -most, most)
    L.assert_close(L.f64(stats)[:N], lse, b_lse + 4 * ua * np.abs(lse), "lse")
    L.assert_close(L.f64(loss), rows, b_rows, "loss")
    # the ordinary row's gradient is that of its own statistics
    ws[4] = float(stats[4])
    want, s, t = L.distill_backward(temperature, "NONE", *a, ws, L.f64(dl))
    L.assert_close(L.f64(dx), want, L.distill_grad_bound(dtype, temperature, a[0], a[2], a[1], ws, want, s, t), "dx")
    again = _run_distill(x, index, teacher, temperature, "NONE", dl, in_place=True)
    assert torch.equal(again[2], dx) and torch.equal(again[0], stats) and torch.equal(again[1], loss)


@pytest.mark.parametrize("dtype", ["bfloat16", "float64"])
@pytest.mark.parametrize("N", [1, 2, 15, 16, 17])
@pytest.mark.parametrize("C,k", [(1000, 40), (2100, 200), (40001, 40), (70000, 200)])
def test_distillation_reduced_by_the_launch_that_finishes_the_rows(dtype, N, C, k):
    for reduction in ("VALID", "MEAN", "SUM"):
        x, index, teacher = _distill_case(N, C, k, dtype, torch.int64, N + k)
        dl = torch.full((1,), 0.75, dtype=teacher.dtype, device="cuda")
        _check_distill(dtype, x, index, teacher, 1.5, reduction, dl, *_run_distill(x, index, teacher, 1.5, reduction, dl))


@pytest.mark.parametrize("dtype", DTYPES)
def test_distillation_of_a_listed_class_that_is_masked_by_the_lowest_value(dtype):
    N, C, k = 3, 300, 4
    x, index, teacher = _distill_case(N, C, k, dtype, torch.int64, 8)
    index.copy_(torch.arange(k).expand(N, k))
    teacher.copy_(torch.tensor([0.0, 1.0, 2.0, 3.0]).expand(N, k))  # shares of 0.03 to 0.64
    x[1, 2] = torch.finfo(x.dtype).min
    dl = torch.ones(N, dtype=teacher.dtype, device="cuda")
    _check_distill(dtype, x, index, teacher, 1.0, "NONE", dl, *_run_distill(x, index, teacher, 1.0, "NONE", dl))


def test_distillation_of_rows_that_list_nothing_and_of_no_rows():
    for N in (0, 3):
        x = torch.randn(N, 100, device="cuda")
        index, teacher = torch.full((N, 4), -1, device="cuda"), torch.zeros(N, 4, device="cuda")
        for reduction in ("VALID", "MEAN", "SUM", "NONE"):
            dl = torch.ones(N if reduction == "NONE" else 1, device="cuda")
            stats, loss, dx = _run_distill(x, index, teacher, 1.0, reduction, dl)
            assert (loss == 0).all() and (dx == 0).all() and stats[:N].isposinf().all()
            assert float(stats[N]) == {"VALID": 0, "MEAN": max(N, 1), "SUM": 1, "NONE": 1}[reduction]


def test_distillation_gradient_against_differences():
    rng = np.random.default_rng(1)
    N, C, k, temperature, step = 3, 40, 5, 1.5, 1e-5
    x, teacher = rng.standard_normal((N, C)) * 2, rng.standard_normal((N, k))
    index = rng.integers(0, C, (N, k))
    index[0, 1] = index[0, 0]
    index[2] = -1
    dev = [torch.from_numpy(a).cuda() for a in (x, index, teacher)]
    _, _, dx = _run_distill(*dev, temperature, "VALID", torch.ones(1, dtype=torch.float64, device="cuda"))
    for i in range(N):
        for j in range(C):
            d = np.zeros((N, C))
            d[i, j] = step
            up, down = (L.distill_forward(temperature, "VALID", v, index, teacher)[2][0] for v in (x + d, x - d))
            # third derivatives of order 1 times step^2, and 64-bit roundings over the step
            assert abs((up - down) / (2 * step) - float(dx[i, j])) < 1e-9


def test_distillation_offsets_beyond_32_bits():
    K = _K()
    C, k = 131072, 4
    N = (1 << 32) // C + 2
    x = torch.empty((N, C), dtype=torch.bfloat16, device="cuda").normal_()
    index = torch.full((N, k), -1, dtype=torch.int64, device="cuda")
    teacher = torch.zeros((N, k), device="cuda")
    index[-2:] = torch.arange(k, device="cuda") * 1000
    stats, loss = torch.empty(N + 1, device="cuda"), torch.empty(N, device="cuda")
    K.topk_distillation_loss_forward(N, C, k, 1.0, "NONE", x, index, teacher, stats, loss)
    tail = x[-2:].clone()
    dl = torch.ones(N, device="cuda")
    K.topk_distillation_loss_backward(N, C, k, 1.0, "NONE", x, index, teacher, stats, dl, x)
    _check_distill("bfloat16", tail, index[-2:], teacher[-2:], 1.0, "NONE", dl[-2:],
                   torch.cat([stats[N - 2:N], stats[N:]]), loss[-2:], x[-2:])
    assert float(loss[:-2].abs().max()) == 0


def test_calls_of_several_threads_on_one_stream():
    """Each call's launches use scratch that no other thread's call writes in between."""
    import threading
    K = _K()
    cases = []
    for seed in range(4):
        x, index, teacher = _distill_case(40, 70001, 20, "float32", torch.int32, seed)
        h, dy = _make((300, 2048), "float32", seed), _make((300, 2048), "float32", seed + 9)
        cases.append((x, index, teacher, h, dy, torch.rand(300, device="cuda"), torch.rand(2048, device="cuda")))

    def call(case):
        x, index, teacher, h, dy, rsig, gamma = case
        stats, loss = torch.empty(41, device="cuda"), torch.empty(1, device="cuda")
        K.topk_distillation_loss_forward(40, 70001, 20, 1.0, "MEAN", x, index, teacher, stats, loss)
        dgamma, dx = torch.empty(2048, device="cuda"), torch.empty_like(h)
        K.rms_norm_grad(300, 2048, h, rsig, gamma, dy, None, dgamma, dx)
        return stats, loss, dgamma, dx

    want = [call(c) for c in cases]
    torch.cuda.synchronize()
    got, start = [[] for _ in cases], threading.Barrier(len(cases))

    def work(i):
        start.wait()
        for _ in range(50):
            got[i].append(call(cases[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i, calls in enumerate(got):
        assert len(calls) == 50
        for outputs in calls:
            assert all(torch.equal(a, b) for a, b in zip(outputs, want[i]))


# ---------------------------------------------------------------- drafted tokens

def _verify_case(B, k, C, dtype, index_dtype, sampled, seed):
    rng = np.random.default_rng(seed)
    logits = rng.standard_normal((B, k + 1, C)) * 3
    p = np.exp(logits - logits.max(2, keepdims=True))
    p /= p.sum(2, keepdims=True)
    other = np.exp(rng.standard_normal((B, k, C)) * 2)
    q = 0.6 * p[:, :k] + 0.4 * other / other.sum(2, keepdims=True)
    drafted = np.array([[rng.choice(C, p=q[b, i] / q[b, i].sum()) for i in range(k)] for b in range(B)]).reshape(B, k)
    td = getattr(torch, dtype)
    t = {"target": torch.from_numpy(p).to(td).cuda(), "draft": torch.from_numpy(q).to(td).cuda() if sampled else None,
         "drafted": torch.from_numpy(drafted).to(index_dtype).cuda(),
         "lengths": torch.from_numpy(rng.integers(0, k + 1, B)).to(index_dtype).cuda(),
         "u_accept": torch.from_numpy(rng.random((B, k))).float().clamp(max=1 - 2 ** -24).cuda(),
         "u_sample": torch.from_numpy(rng.random(B)).float().clamp(max=1 - 2 ** -24).cuda()}
    return t


def _run_verify(t, k=None):
    B, places, C = t["target"].shape
    it = t["drafted"].dtype
    tokens = torch.full((B, places), 99, dtype=it, device="cuda")
    accepted = torch.full((B,), 99, dtype=it, device="cuda")
    _K().draft_verify(B, places - 1, C, t["target"], t["draft"], t["drafted"], t["lengths"], t["u_accept"],
                      t["u_sample"], tokens, accepted)
    return tokens, accepted


def _check_verify(t):
    tokens, accepted = _run_verify(t)
    lengths = None if t["lengths"] is None else t["lengths"].cpu().numpy()
    want, n = L.draft_verify(L.f64(t["target"]), None if t["draft"] is None else L.f64(t["draft"]),
                             t["drafted"].cpu().numpy(), lengths, L.f64(t["u_accept"]), L.f64(t["u_sample"]))
    assert np.array_equal(accepted.cpu().numpy(), n)
    assert np.array_equal(tokens.cpu().numpy(), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1), (7, 3, 10), (1, 4, 32000), (5, 4, 1000), (40, 2, 257), (3, 8, 50257),
                                   (300, 1, 64), (2, 3, 200001), (2, 70, 130)])
@pytest.mark.parametrize("sampled", [True, False])
def test_draft_verify(shape, dtype, sampled):
    B, k, C = shape
    index_dtype = torch.int32 if (B + C) % 2 else torch.int64
    t = _verify_case(B, k, C, dtype, index_dtype, sampled, B + C)
    _check_verify(t)
    t["lengths"] = None
    t["u_accept"].mul_(0.3)  # more of them pass
    _check_verify(t)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_draft_verify_odd_addresses(dtype):
    for C in (33, 1000, 32000, 70001):
        t = _verify_case(4, 3, C, dtype, torch.int64, True, C)
        _check_verify({k: v if v is None else _odd(v, 1) for k, v in t.items()})


def test_draft_verify_without_drafts():
    for B, C in ((1, 1), (3, 50000), (130, 100)):
        t = _verify_case(B, 1, C, "float32", torch.int32, False, C)
        target = t["target"][:, :1].contiguous()
        tokens = torch.full((B, 1), 99, dtype=torch.int32, device="cuda")
        accepted = torch.full((B,), 99, dtype=torch.int32, device="cuda")
        _K().draft_verify(B, 0, C, target, None, None, None, None, t["u_sample"], tokens, accepted)
        want, n = L.draft_verify(L.f64(target), None, np.zeros((B, 0), np.int64), None, np.zeros((B, 0)),
                                 L.f64(t["u_sample"]))
        assert np.array_equal(tokens.cpu().numpy(), want) and not accepted.any()


def test_draft_verify_corners():
    """One-hot rows, equal distributions, rows without weight, garbage in them, tokens outside the vocabulary,
    lengths outside the drafts, random numbers at and beyond their ends."""
    inf, nan = float("inf"), float("nan")
    k, C = 3, 5000
    t = _verify_case(14, k, C, "float32", torch.int64, True, 9)
    t["lengths"].fill_(k)
    p, q = t["target"], t["draft"]
    p[0] = 0
    p[0, :, 4321] = 1                                # one-hot target
    q[1] = p[1, :k]
    t["u_accept"][1] = 1.0                           # equal distributions refused: no residual, the target decides
    p[2] = 0                                         # no weight anywhere
    q[3], p[3] = nan, nan                            # garbage everywhere
    p[4, :, ::7], q[4, :, ::11] = nan, inf           # and here and there
    p[4, :, 3], p[4, :, 4] = -1.0, -inf
    t["drafted"][5] = torch.tensor([C, -1, 2 ** 40])
    t["drafted"][6, 0] = -5
    t["lengths"][7], t["lengths"][8] = -3, 99
    t["u_sample"][9], t["u_accept"][9] = 0.0, 0.0
    t["u_sample"][10], t["u_accept"][10] = 1.0, 1.5
    t["u_sample"][11] = 2.0
    p[12, :, 100:] = 0                               # all of the weight in the first packets
    p[13, :, :-1] = 0                                # and in the last element
    q[13] = 0
    _check_verify(t)
    t["draft"] = None
    _check_verify(t)
    t["u_sample"][0], t["u_accept"][1] = nan, nan    # NaN draws the first class, and refuses
    t["u_sample"][2] = -1.0
    _check_verify(t)


def test_draft_verify_offsets_beyond_32_bits():
    B, k, C = 9000, 3, 131072  # 4.7e9 probabilities of the target
    target = torch.zeros((B, k + 1, C), dtype=torch.bfloat16, device="cuda")
    at = torch.arange(B, device="cuda") * 13 % C
    rows = torch.arange(B, device="cuda")
    for i in range(k + 1):
        target[rows, i, (at + i) % C] = 1.0
    drafted = torch.stack([(at + i) % C for i in range(k)], 1)
    drafted[::2, 1] = 0
    drafted = drafted.contiguous()
    tokens, accepted = torch.empty((B, k + 1), dtype=torch.int64, device="cuda"), torch.empty(B, dtype=torch.int64, device="cuda")
    u, us = torch.full((B, k), 0.5, device="cuda"), torch.full((B,), 0.5, device="cuda")
    _K().draft_verify(B, k, C, target, None, drafted, None, u, us, tokens, accepted)
    want = torch.stack([(at + i) % C for i in range(k + 1)], 1)
    refused = (drafted != want[:, :k]).any(1)
    assert torch.equal(accepted, torch.where(refused, 1, k))
    assert torch.equal(tokens[~refused], want[~refused])
    assert torch.equal(tokens[refused][:, :2], want[refused][:, :2]) and (tokens[refused][:, 2:] == -1).all()


# ---------------------------------------------------------------- together

def test_a_training_step_of_a_student_block():
    """Residual norm, a product with the vocabulary's weights, the distillation loss and all gradients back to
    the residual stream and gamma, in float64 against torch's derivatives of the definitions."""
    K = _K()
    N, C, V, k, temperature, eps = 24, 96, 500, 8, 2.0, 1e-5
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.float64)
    x, r, gamma, w = rand(N, C), rand(N, C), 1 + 0.1 * rand(C), rand(C, V) * 0.3
    teacher = rand(N, k) + 4
    index = torch.stack([torch.randperm(V, generator=g, device="cuda")[:k] for _ in range(N)])
    index[-3:] = -1
    h, y, rsig = torch.empty_like(x), torch.empty_like(x), torch.empty(N, device="cuda", dtype=torch.float64)
    K.rms_norm(N, C, eps, x, r, gamma, h, rsig, y)
    logits = (y @ w).contiguous()
    stats, loss = torch.empty(N + 1, dtype=torch.float64, device="cuda"), torch.empty(1, dtype=torch.float64, device="cuda")
    K.topk_distillation_loss_forward(N, V, k, temperature, "VALID", logits, index, teacher, stats, loss)
    dlogits, dl = torch.empty_like(logits), torch.ones(1, dtype=torch.float64, device="cuda")
    K.topk_distillation_loss_backward(N, V, k, temperature, "VALID", logits, index, teacher, stats, dl, dlogits)
    dy = (dlogits @ w.t().contiguous()).contiguous()
    dgamma, dx = torch.empty_like(gamma), torch.empty_like(x)
    K.rms_norm_grad(N, C, h, rsig, gamma, dy, h, dgamma, dx)  # with d(sum h^2 / 2) along the stream

    xa, ga = x.clone().requires_grad_(), gamma.clone().requires_grad_()
    s = xa + r
    out = s / torch.sqrt(s.square().mean(1, keepdim=True) + float(np.float32(eps))) * ga
    logp = torch.log_softmax(out @ w / temperature, 1)
    t = torch.softmax(teacher / temperature, 1)
    rows = (t * (t.log() - logp.gather(1, index.clamp(min=0)))).sum(1) * temperature ** 2
    want = rows[:-3].sum() / (N - 3)
    (want + s.square().sum() / 2).backward()
    # chains of a few hundred 64-bit roundings on values of order 1 to 10
    assert abs(float(loss) - float(want.detach())) < 1e-12
    assert float((dx - xa.grad).abs().max()) < 1e-11 and float((dgamma - ga.grad).abs().max()) < 1e-11


def test_a_served_step_quantised_norm_softmax_and_verification():
    """An 8-bit norm feeds two heads, Softmax makes their probabilities and the drafted tokens are verified."""
    K = _K()
    B, k, C, V = 6, 3, 256, 4001
    rows = B * (k + 1)
    x, r = _make((rows, C), "bfloat16", 50), _make((rows, C), "bfloat16", 51)
    gamma = torch.rand(C, device="cuda") + 0.5
    q = torch.empty((rows, C), dtype=torch.float8_e4m3fn, device="cuda")
    h, scale = torch.empty_like(x), torch.empty((rows, 2), device="cuda")
    K.rms_norm_quant(rows, C, 128, 1e-5, x, r, gamma, h, None, q, scale)
    y = (q.float().view(rows, 2, 128) * scale[:, :, None]).view(rows, C)
    _, _, want = L.rms_norm(L.f64(x), L.f64(r), L.f64(gamma), 1e-5)
    # half a step of e4m3, or of its subnormals against the group's largest value
    top = np.abs(want).reshape(rows, 2, 128).max(2).repeat(128, 1)
    L.assert_close(L.f64(y), want, 1.001 * (2.0 ** -4 * np.abs(want) + 2.0 ** -10 * top / 448) + 1e-6 * top, "y")
    w = _make((C, V), "float32", 52, 0.4)
    logits = (y @ w).contiguous()
    p, d = torch.empty_like(logits), torch.empty_like(logits)
    K.softmax(rows, 1, V, logits, p)
    K.softmax(rows, 1, V, (logits * 0.7).contiguous(), d)
    target, draft = p.view(B, k + 1, V), d.view(B, k + 1, V)[:, :k].contiguous()
    g = torch.Generator(device="cuda").manual_seed(4)
    drafted = torch.multinomial(draft.view(-1, V), 1, generator=g).view(B, k)
    _check_verify({"target": target, "draft": draft, "drafted": drafted, "lengths": None,
                   "u_accept": torch.rand(B, k, generator=g, device="cuda"),
                   "u_sample": torch.rand(B, generator=g, device="cuda")})


def _everything(K, t):
    N, C = t["x"].shape
    K.rms_norm(N, C, 1e-5, t["x"], t["r"], t["g"], t["h"], t["rsig"], t["y"])
    K.rms_norm_quant(N, C, 128, 1e-5, t["x"], t["r"], t["g"], None, None, t["q"], t["scale"])
    K.rms_norm_grad(N, C, t["h"], t["rsig"], t["g"], t["y"], t["r"], t["dg"], t["dx"])
    V, k = t["logits"].shape[1], t["index"].shape[1]
    K.topk_distillation_loss_forward(len(t["logits"]), V, k, 2.0, "VALID", t["logits"], t["index"], t["teacher"],
                                     t["stats"], t["loss"])
    K.topk_distillation_loss_backward(len(t["logits"]), V, k, 2.0, "VALID", t["logits"], t["index"], t["teacher"],
                                      t["stats"], t["dl"], t["dlogits"])
    B, places, V = t["target"].shape
    K.draft_verify(B, places - 1, V, t["target"], t["draft"], t["drafted"], t["lengths"], t["u_accept"], t["u_sample"],
                   t["tokens"], t["accepted"])


OUTPUTS = ("h", "rsig", "y", "q", "scale", "dg", "dx", "stats", "loss", "dlogits", "tokens", "accepted")


def _everything_tensors(seed, N=70, C=1024, V=60000, rows=5):
    t = {"x": _make((N, C), "bfloat16", seed), "r": _make((N, C), "bfloat16", seed + 1), "g": torch.rand(C, device="cuda")}
    t["h"], t["y"], t["dx"] = (torch.empty_like(t["x"]) for _ in range(3))
    t["rsig"], t["dg"] = torch.empty(N, device="cuda"), torch.empty(C, device="cuda")
    t["q"], t["scale"] = torch.empty((N, C), dtype=torch.uint8, device="cuda"), torch.empty((N, C // 128), device="cuda")
    t["logits"], t["index"], t["teacher"] = _distill_case(rows, V, 16, "bfloat16", torch.int64, seed)
    t["stats"], t["loss"], t["dl"] = torch.empty(rows + 1, device="cuda"), torch.empty(1, device="cuda"), torch.ones(1, device="cuda")
    t["dlogits"] = torch.empty_like(t["logits"])
    t.update(_verify_case(3, 2, V, "float32", torch.int64, True, seed))
    t["tokens"], t["accepted"] = torch.empty((3, 3), dtype=torch.int64, device="cuda"), torch.empty(3, dtype=torch.int64, device="cuda")
    return t


def test_replayed_graphs_that_were_captured_side_by_side():
    """Two graphs of all entry points, captured one after the other and replayed in turn with eager work of
    larger sizes between: each replay equals the eager result on the same inputs, bit for bit."""
    K = _K()
    sets = [_everything_tensors(100), _everything_tensors(200)]
    fresh = [_everything_tensors(300), _everything_tensors(400)]
    graphs = []
    for t in sets:
        _everything(K, t)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _everything(K, t)
        graphs.append(graph)
    large = _everything_tensors(500, N=3000, C=4096, V=100000, rows=40)
    inputs = [k for k in sets[0] if k not in OUTPUTS]
    for step in range(3):
        source = fresh[step % 2]
        for t, graph in zip(sets, graphs):
            for name in inputs:
                t[name].copy_(source[name])
            for name in OUTPUTS:
                t[name].fill_(3)
        _everything(K, large)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        _everything(K, source)
        torch.cuda.synchronize()
        for t in sets:
            for name in OUTPUTS:
                assert torch.equal(t[name].view(torch.uint8), source[name].view(torch.uint8)), (step, name)


def test_two_streams_at_once():
    K = _K()
    streams = [torch.cuda.Stream() for _ in range(2)]
    sets = [_everything_tensors(600 + i, V=30000 + 8 * i) for i in range(2)]
    want = []
    for t in sets:
        _everything(K, t)
        torch.cuda.synchronize()
        want.append({n: t[n].clone() for n in OUTPUTS})
        for n in OUTPUTS:
            t[n].fill_(3)
    torch.cuda.synchronize()
    for _ in range(5):
        for t, s in zip(sets, streams):
            with torch.cuda.stream(s):
                _everything(K, t)
    torch.cuda.synchronize()
    for t, w in zip(sets, want):
        for n in OUTPUTS:
            assert torch.equal(t[n].view(torch.uint8), w[n].view(torch.uint8)), n


# ---------------------------------------------------------------- sizes at which the launchers change kernels

@pytest.mark.parametrize("dtype,vec", [("bfloat16", 8), ("float32", 4), ("float64", 2)])
def test_rms_norm_at_the_seams(dtype, vec):
    """Rows of one packet more or less, and one element more or less, than the tiles hold; groups of rows that
    are partly filled."""
    K = _K()
    for packets in (1, 2, 8, 16, 32, 64, 128, 256, 512, 1024, 2048, 4096):
        for extra in (-1, 0, 1, vec):
            C = packets * vec + extra
            for N in (1, 67 if packets < 64 else 5):
                x, r, dy = (_make((N, C), dtype, packets + i) for i in range(3))
                gamma = (1 + _make((C,), "float64", 9, 0.3)).to(L.acc_dtype(dtype))
                h, y, rsig = torch.empty_like(x), torch.empty_like(x), torch.empty(N, dtype=gamma.dtype, device="cuda")
                K.rms_norm(N, C, 1e-5, x, r, gamma, h, rsig, y)
                s, rs, want = L.rms_norm(L.f64(x), L.f64(r), L.f64(gamma), float(np.float32(1e-5)))
                bh, brs, by = L.rms_norm_bounds(dtype, s, rs, want)
                L.assert_close(L.f64(h), s, bh, "h %d" % C)
                L.assert_close(L.f64(rsig), rs, brs, "rsig %d" % C)
                L.assert_close(L.f64(y), want, by, "y %d" % C)
                dgamma, dx = torch.empty_like(gamma), torch.empty_like(x)
                K.rms_norm_grad(N, C, h, rsig, gamma, dy, r, dgamma, dx)
                _check_grad(dtype, h, rsig, gamma, dy, r, dgamma, dx)
                if dtype != "float64":
                    for group in (0, 64):
                        q = torch.empty((N, C), dtype=torch.float8_e4m3fn, device="cuda")
                        scale = torch.empty((N, -(-C // group) if group else 1), device="cuda")
                        K.rms_norm_quant(N, C, group, 1e-5, x, r, gamma, h, rsig, q, scale)
                        _check_quant(dtype, group, x, r, gamma, h, rsig, q, scale)


@pytest.mark.parametrize("dtype,vec", [("bfloat16", 8), ("float32", 4)])
@pytest.mark.parametrize("packets", [40, 144, 320, 896, 1025, 1279, 1280, 1281, 1535, 1536, 1537])
def test_rms_norm_of_rows_that_leave_slots_empty(dtype, vec, packets):
    """Tiles of 640 and 768 threads and those beside them; rows more than the workgroups, so that they walk."""
    K = _K()
    for C, N in ((packets * vec, 1100), (packets * vec - 1, 5), (packets * vec + 1, 530)):
        x, r, dy = (_make((N, C), dtype, packets + i) for i in range(3))
        gamma = (1 + _make((C,), "float64", 9, 0.3)).float()
        h, y, rsig = torch.empty_like(x), torch.empty_like(x), torch.empty(N, device="cuda")
        K.rms_norm(N, C, 1e-5, x, r, gamma, h, rsig, y)
        s, rs, want = L.rms_norm(L.f64(x), L.f64(r), L.f64(gamma), float(np.float32(1e-5)))
        bh, brs, by = L.rms_norm_bounds(dtype, s, rs, want)
        L.assert_close(L.f64(h), s, bh, "h %d" % C)
        L.assert_close(L.f64(rsig), rs, brs, "rsig %d" % C)
        L.assert_close(L.f64(y), want, by, "y %d" % C)
        dgamma, dx = torch.empty_like(gamma), torch.empty_like(x)
        K.rms_norm_grad(N, C, h, rsig, gamma, dy, r, dgamma, dx)
        _check_grad(dtype, h, rsig, gamma, dy, r, dgamma, dx)
        for group in (0, 32, 128, 256):
            q = torch.empty((N, C), dtype=torch.float8_e4m3fn, device="cuda")
            scale = torch.empty((N, -(-C // group) if group else 1), device="cuda")
            K.rms_norm_quant(N, C, group, 1e-5, x, r, gamma, h, rsig, q, scale)
            _check_quant(dtype, group, x, r, gamma, h, rsig, q, scale)


@pytest.mark.parametrize("dtype,vec", [("bfloat16", 8), ("float32", 4)])
def test_distillation_at_the_seams(dtype, vec):
    for packets in (256, 512, 1024, 2048, 2600):
        for extra in (-1, 0, 1):
            C = packets * vec + extra
            for k in (64, 65, 256, 257):
                x, index, teacher = _distill_case(5, C, k, dtype, torch.int32, C + k)
                dl = torch.ones(1, device="cuda")
                _check_distill(dtype, x, index, teacher, 2.0, "VALID", dl, *_run_distill(x, index, teacher, 2.0, "VALID", dl))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32", "float64"])
def test_draft_verify_at_the_seams(dtype):
    """Rows that end inside a packet, inside a run of 64 packets and behind one, on both sides of the size from which
    rows are cut; drafts of 64 positions and more."""
    for B, k, C in ((3, 2, 7), (3, 2, 8), (3, 2, 511), (3, 2, 513), (2, 2, 32767), (2, 2, 32768), (2, 2, 32769), (2, 1, 65537),
                    (2, 64, 300), (2, 65, 300), (2, 1, 262145)):
        for sampled in (True, False):
            t = _verify_case(B, k, C, dtype, torch.int32, sampled, C + k)
            if C % 2:
                t["u_accept"].fill_(0.999)  # refused early
            _check_verify(t)
            t["u_sample"].fill_(1 - 2.0 ** -24)
            t["lengths"].fill_(k)
            _check_verify(t)


def test_arguments_are_checked():
    K = _K()
    from dragon_amd import _lib
    x, g, y = torch.ones(4, 64, device="cuda"), torch.ones(64, device="cuda"), torch.empty(4, 64, device="cuda")
    with pytest.raises(ValueError, match="elements"):
        K.rms_norm(5, 64, 1e-5, x, None, g, None, None, y)
    with pytest.raises(ValueError, match="memory"):
        K.rms_norm(4, 64, 1e-5, x, None, g.cpu(), None, None, y)
    with pytest.raises(ValueError, match="contiguous"):
        K.rms_norm(4, 32, 1e-5, x[:, ::2], None, g, None, None, y)
    with pytest.raises(ValueError, match="missing"):
        K.rms_norm(4, 64, 1e-5, x, None, None, None, None, y)
    with pytest.raises(TypeError):
        K.rms_norm(4, 64, 1e-5, x, None, g.half(), None, None, y)
    with pytest.raises(TypeError):
        K.rms_norm(4, 64, 1e-5, x, x.half(), g, None, None, y)
    with pytest.raises(ValueError, match="negative"):
        K.rms_norm(-1, 64, 1e-5, x, None, g, None, None, y)
    with pytest.raises(_lib.DragonHipError) as e:
        K.rms_norm(4, 64, 1e-5, x, x, g, y, None, y)
    assert e.value.status == -1
    q, scale = torch.empty(4, 64, dtype=torch.uint8, device="cuda"), torch.empty(4, 8, device="cuda")
    with pytest.raises(_lib.DragonHipError):
        K.rms_norm_quant(4, 64, 48, 1e-5, x, None, g, None, None, q, scale)
    with pytest.raises(_lib.DragonHipError) as e:
        K.rms_norm_quant(4, 64, 32, 1e-5, x.double(), None, g.double(), None, None, q, scale)
    assert e.value.status == -2
    with pytest.raises(TypeError):
        K.rms_norm_quant(4, 64, 32, 1e-5, x, None, g, None, None, y, scale)
    index, teacher, stats, loss = (torch.zeros(4, 3, dtype=torch.int64, device="cuda"), torch.zeros(4, 3, device="cuda"),
                                   torch.empty(5, device="cuda"), torch.empty(1, device="cuda"))
    for k, temperature in ((0, 1.0), (1025, 1.0), (3, 0.0), (3, -1.0), (3, float("nan")), (3, float("inf"))):
        wide = torch.zeros(4, max(k, 1), dtype=torch.int64, device="cuda")
        with pytest.raises(_lib.DragonHipError):
            K.topk_distillation_loss_forward(4, 64, k, temperature, "MEAN", x, wide, wide.float(), stats, loss)
        with pytest.raises(_lib.DragonHipError):
            K.topk_distillation_loss_backward(4, 64, k, temperature, "MEAN", x, wide, wide.float(), stats, loss, y)
    with pytest.raises(TypeError):
        K.topk_distillation_loss_forward(4, 64, 3, 1.0, "MEAN", x, index.short(), teacher, stats, loss)
    with pytest.raises(ValueError, match="elements"):
        K.topk_distillation_loss_forward(4, 64, 3, 1.0, "MEAN", x, index, teacher, stats[:4], loss)
    with pytest.raises(KeyError):
        K.topk_distillation_loss_forward(4, 64, 3, 1.0, "SOME", x, index, teacher, stats, loss)
    tokens, accepted = torch.empty(1, 4, dtype=torch.int64, device="cuda"), torch.empty(1, dtype=torch.int64, device="cuda")
    u = torch.rand(1, 3, device="cuda")
    with pytest.raises(TypeError):
        K.draft_verify(1, 3, 64, x, None, tokens[:, :3].int().contiguous(), None, u, u, tokens, accepted)
    with pytest.raises(ValueError, match="missing"):
        K.draft_verify(1, 3, 64, x, None, None, None, u, u, tokens, accepted)


# ---------------------------------------------------------------- the operators of the host layer

@pytest.fixture()
def ws():
    from dragon_amd import runtime
    w = runtime.Workspace("language_ops_test")
    yield w
    w.close()


def test_operator_rms_norm_and_its_gradient(ws):
    from dragon_amd import runtime as rt
    rng = np.random.default_rng(5)
    x, r, dy, dh = (rng.standard_normal((2, 6, 40)) for _ in range(4))
    w = rng.uniform(0.5, 1.5, 40)
    names = [ws.feed(n, a) for n, a in (("x", x), ("w", w), ("r", r), ("dy", dy), ("dh", dh))]
    flat = lambda a: a.reshape(12, 40)
    eps = float(np.float32(1e-3))
    # without a residual
    tape = rt.Tape(ws)
    y = rt.rms_norm(tape, names[:2], epsilon=1e-3)
    dx, dw = tape.gradient(y, names[:2], output_gradient="dy")
    _, rs, want = L.rms_norm(flat(x), None, w, eps)
    gx, gw = L.rms_norm_grad(flat(x), rs, w, flat(dy), None)
    for got, ref in ((y, want), (dx, gx), (dw, gw)):
        assert np.allclose(ws.fetch(got).reshape(ref.shape), ref, rtol=1e-12, atol=1e-13)
    # with one, and a gradient through the sum
    tape = rt.Tape(ws)
    y, h = rt.rms_norm(tape, names[:3], epsilon=1e-3)
    s, rs, want = L.rms_norm(flat(x), flat(r), w, eps)
    assert np.array_equal(ws.fetch(h).reshape(s.shape), s) and np.allclose(ws.fetch(y).reshape(s.shape), want, rtol=1e-12)
    forward = tape.records[-1][0]
    for through in (True, False):
        defs, grads = ws.gradient_defs(forward, ["dy", "dh" if through else "NULL"])
        for d in defs:
            ws.run_operator(d)
        gx, gw = L.rms_norm_grad(s, rs, w, flat(dy), flat(dh) if through else None)
        for name, ref in zip(grads, (gx, gw, gx)):
            assert np.allclose(ws.fetch(name).reshape(ref.shape), ref, rtol=1e-12, atol=1e-13)
    # two axes normalised as one
    tape = rt.Tape(ws)
    ws.feed("w2", np.ones((240,)))
    y = rt.rms_norm(tape, ["x", "w2"], axis=1)
    assert np.allclose(ws.fetch(y).reshape(2, 240), L.rms_norm(x.reshape(2, 240), None, 1.0, float(np.float32(1e-5)))[2], rtol=1e-12)
    with pytest.raises(rt.DragonError, match="second output"):
        ws.run_operator(rt.make_def("RMSNorm", names[:3], ["y"]))
    with pytest.raises(rt.DragonError, match="dimensions"):
        ws.run_operator(rt.make_def("RMSNorm", ["x", "w2"], ["y"]))
    with pytest.raises(rt.DragonError, match="type"):
        ws.feed("r32", r.astype(np.float32))
        ws.run_operator(rt.make_def("RMSNorm", ["x", "w", "r32"], ["y", "h"]))


def test_operator_rms_norm_quant(ws):
    from dragon_amd import runtime as rt
    rng = np.random.default_rng(6)
    x, r = (rng.standard_normal((3, 5, 200)).astype(np.float32) for _ in range(2))
    w = rng.uniform(0.5, 1.5, 200).astype(np.float32)
    names = [ws.feed(n, a) for n, a in (("x", x), ("w", w), ("r", r))]
    for group, groups in ((0, 1), (64, 4)):
        tape = rt.Tape(ws)
        q, s, h = rt.rms_norm_quant(tape, names, group_size=group)
        assert ws.info(q) == ("uint8", (3, 5, 200)) and ws.info(s) == ("float32", (3, 5, groups))
        _, _, y = L.rms_norm(x.reshape(15, 200).astype(np.float64), r.reshape(15, 200).astype(np.float64), w.astype(np.float64), 1e-5)
        want_scale, v = L.quant(y, group)
        assert np.allclose(ws.fetch(s).reshape(15, groups), want_scale, rtol=1e-5)
        codes = torch.from_numpy(ws.fetch(q)).view(torch.float8_e4m3fn).double().numpy().reshape(15, 200)
        assert (np.abs(codes - v) <= 1.001 * (2.0 ** -4 * np.abs(v) + 2.0 ** -10)).all()
        assert np.array_equal(ws.fetch(h), x + r)
    with pytest.raises(rt.DragonError, match="Unsupported type"):
        ws.feed("x64", x.astype(np.float64))
        ws.run_operator(rt.make_def("RMSNormQuant", ["x64", "w"], ["q", "s"]))
    with pytest.raises(rt.DragonError):
        ws.run_operator(rt.make_def("RMSNormQuant", ["x", "w"], ["q", "s"], group_size=48))


@pytest.mark.parametrize("reduction", ["valid", "none", "mean", "sum", "batch_mean"])
def test_operator_topk_distillation_loss_and_its_gradient(ws, reduction):
    from dragon_amd import runtime as rt
    rng = np.random.default_rng(7)
    x, t = rng.standard_normal((2, 5, 50)) * 2, rng.standard_normal((2, 5, 4))
    i = rng.integers(0, 50, (2, 5, 4))
    i[1, 4] = -1
    names = [ws.feed(n, a) for n, a in (("x", x), ("i", i), ("t", t))]
    dl = rng.random((2, 5)) if reduction == "none" else np.array(0.5)
    ws.feed("dl", dl)
    tape = rt.Tape(ws)
    loss = rt.topk_distillation_loss(tape, names, temperature=2.0, reduction=reduction)
    (dx,) = tape.gradient(loss, ["x"], output_gradient="dl")
    a = (x.reshape(10, 50), i.reshape(10, 4), t.reshape(10, 4))
    by = "SUM" if reduction == "batch_mean" else reduction.upper()
    stats, _, want = L.distill_forward(2.0, by, *a)
    grad, _, _ = L.distill_backward(2.0, by, *a, stats, dl.reshape(-1))
    over = 2.0 if reduction == "batch_mean" else 1.0  # the leading extent
    assert ws.info(loss)[1] == ((2, 5) if reduction == "none" else ())
    assert np.allclose(ws.fetch(loss).reshape(-1), want / over, rtol=1e-12)
    assert np.allclose(ws.fetch(dx).reshape(10, 50), grad / over, rtol=1e-12, atol=1e-15)


def test_operator_draft_verify_after_softmax(ws):
    from dragon_amd import runtime as rt
    rng = np.random.default_rng(8)
    B, k, C = 4, 3, 300
    zp, zq = rng.standard_normal((B, k + 1, C)).astype(np.float32) * 2, rng.standard_normal((B, k, C)).astype(np.float32)
    drafted, lengths = rng.integers(0, C, (B, k)), np.array([3, 2, 0, 3])
    ua, us = rng.random((B, k)).astype(np.float32) * 0.1, rng.random(B).astype(np.float32)
    for n, a in (("zp", zp), ("zq", zq), ("d", drafted), ("n", lengths), ("ua", ua), ("us", us)):
        ws.feed(n, a)
    tape = rt.Tape(ws)
    p, q = rt.softmax(tape, ["zp"]), rt.softmax(tape, ["zq"])
    for draft in (True, False):
        tokens, accepted = rt.draft_verify(tape, [p, "d", "n", "ua", "us"] + ([q] if draft else []))
        want, n = L.draft_verify(ws.fetch(p).astype(np.float64), ws.fetch(q).astype(np.float64) if draft else None, drafted,
                                 lengths, ua.astype(np.float64), us.astype(np.float64))
        assert np.array_equal(ws.fetch(tokens), want) and np.array_equal(ws.fetch(accepted), n)
    with pytest.raises(rt.DragonError, match="type"):
        ws.run_operator(rt.make_def("DraftVerify", [p, "d", "us", "ua", "us"], ["tok", "acc"]))
    with pytest.raises(rt.DragonError, match="dimensions"):
        ws.run_operator(rt.make_def("DraftVerify", [p, "d", "n", "us", "us"], ["tok", "acc"]))
