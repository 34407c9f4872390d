"""The operators of language models at the edges of their ranges: logits and probabilities at which roundings decide,
tensors and extents beyond 31 bits, gradients that reach an operator by one of its outputs alone."""

import numpy as np
import pytest
import torch

from tests import language_ops as L
from tests.test_gpu_language_ops import DTYPES, _distill_case, _run_distill, _run_verify, ws  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(7, 130, 3), (7, 4200, 300), (7, 9001, 5), (7, 70001, 9)])
@pytest.mark.parametrize("temperature", [0.5, 0.75, 1.5])
def test_distillation_of_teachers_far_from_zero(dtype, shape, temperature):
    """The teacher's shares depend on differences of its logits alone, so the plain form is that of the rows less
    their largest listed logit (exact in 64 bits), with its bounds; entries that are 800 and more below it have
    a share of exactly 0 in every type and are not listed there."""
    N, C, k = shape
    x, index, teacher = _distill_case(N, C, k, dtype, torch.int32, 21, 2.0)
    g = torch.Generator().manual_seed(4)
    index.copy_(torch.randint(0, C, (N, k), generator=g))
    teacher.copy_(torch.randn((N, k), generator=g, dtype=torch.float64) * 2)
    low = torch.finfo(teacher.dtype).min
    teacher[0] += 30000
    teacher[1] -= 30000
    teacher[2] = low                  # nothing but the type's lowest value: equal shares
    teacher[3] = low                  # one entry is left
    teacher[3, k - 1] = 1.0
    teacher[4] = -low / 2             # far above zero
    teacher[4, 0] = low
    teacher[5, 0] = -float("inf")     # not listed
    teacher[5, 1:] += 1e6
    dl = torch.rand(N, generator=g).to(teacher.dtype).cuda()
    stats, loss, dx = _run_distill(x, index, teacher, temperature, "NONE", dl)
    t = L.f64(teacher)
    with np.errstate(over="ignore"):
        shifted = t - t.max(1, keepdims=True)
        near = shifted / temperature > -800
    plain = (L.f64(x), np.where(near, index.cpu().numpy().astype(np.int64), -1), np.where(near, shifted, 0.0))
    ws_, rows, _ = L.distill_forward(temperature, "NONE", *plain)
    b_lse, b_rows = L.distill_bounds(dtype, temperature, *plain)
    L.assert_close(L.f64(loss), rows, b_rows, "loss")
    L.assert_close(L.f64(stats)[:N], ws_[:N], b_lse, "lse")
    got_stats = L.f64(stats)
    want, s, sh = L.distill_backward(temperature, "NONE", *plain, got_stats, L.f64(dl))
    L.assert_close(L.f64(dx), want, L.distill_grad_bound(dtype, temperature, plain[0], plain[2], plain[1], got_stats, want,
                                                         s, sh), "dx")


@pytest.mark.parametrize("reduction", ["batch_mean", "mean", "valid"])
def test_operator_topk_distillation_loss_of_one_row_of_logits(ws, reduction):
    """Logits [C] without leading axes are one row."""
    from dragon_amd import runtime as rt
    rng = np.random.default_rng(9)
    x, t, i = rng.standard_normal(50), rng.standard_normal(4), rng.integers(0, 50, 4)
    for n, a in (("x", x), ("i", i), ("t", t), ("dl", np.array(0.5))):
        ws.feed(n, a)
    tape = rt.Tape(ws)
    loss = rt.topk_distillation_loss(tape, ["x", "i", "t"], temperature=2.0, reduction=reduction)
    (dx,) = tape.gradient(loss, ["x"], output_gradient="dl")
    stats, _, want = L.distill_forward(2.0, "MEAN", x[None], i[None], t[None])
    grad, _, _ = L.distill_backward(2.0, "MEAN", x[None], i[None], t[None], stats, np.array([0.5]))
    assert ws.info(loss)[1] == () and np.allclose(ws.fetch(loss), want, rtol=1e-12)
    assert np.allclose(ws.fetch(dx), grad[0], rtol=1e-12, atol=1e-15)


def test_operator_rms_norm_gradient_of_more_than_2_31_elements(ws):
    """With a residual: its gradient is in a tensor of its own, equal to that of X to the last row."""
    from dragon_amd import runtime as rt
    C = 4096
    N = (1 << 31) // C + 5
    rng = np.random.default_rng(3)
    bits = lambda shape, seed: torch.randn(shape, generator=torch.Generator().manual_seed(seed)).bfloat16().view(torch.uint16).numpy()
    at = np.array([0, 1, N - 6, N - 5, N - 2, N - 1])
    parts = {}
    for i, n in enumerate(("x", "r", "dy")):
        a = np.zeros((N, C), np.uint16)
        parts[n] = bits((len(at), C), i)
        a[at] = parts[n]
        ws.feed(n, a, dtype="bfloat16", device=("hip", 0))
        del a
    w = rng.uniform(0.5, 1.5, C).astype(np.float32)
    ws.feed("w", w)
    tape = rt.Tape(ws)
    y, h = rt.rms_norm(tape, ["x", "w", "r"])
    dx, dw, dr = tape.gradient(y, ["x", "w", "r"], output_gradient="dy")
    f = {n: torch.from_numpy(v).view(torch.bfloat16).double().numpy() for n, v in parts.items()}
    got = ws.fetch(dr)
    assert got.shape == (N, C)
    rest = np.ones(N, bool)
    rest[at] = False
    assert not got[:2000][rest[:2000]].any() and not got[-2000:][rest[-2000:]].any()
    tail = got[at].copy()
    del got
    assert np.array_equal(ws.fetch(dx)[at], tail)
    hs = torch.from_numpy(ws.fetch(h)[at]).view(torch.bfloat16).double().numpy()
    _, rs, _ = L.rms_norm(f["x"] + f["r"], None, w.astype(np.float64), float(np.float32(1e-5)))
    args = (hs, rs, w.astype(np.float64), f["dy"], None)
    want, want_g = L.rms_norm_grad(*args)
    bx, _ = L.rms_norm_grad_bounds("bfloat16", *args, want)
    # rsig is the kernel's own, off by (DEPTH / 2 + 3) roundings; dx holds its third power at most
    L.assert_close(torch.from_numpy(tail).view(torch.bfloat16).double().numpy(), want,
                   bx + 3 * (L.DEPTH / 2 + 3) * 2.0 ** -24 * (np.abs(want) + np.abs(f["dy"] * w) * rs[:, None]), "dx")


def test_operator_rms_norm_gradients_through_a_chain(ws):
    """Two residual norms with Softmax between them, the stream through both: Tape.gradient from the last norm, from
    the last sum and from the first sum against torch's derivatives in float64."""
    from dragon_amd import runtime as rt
    rng = np.random.default_rng(11)
    a = {n: rng.standard_normal((2, 5, 24)) for n in ("x", "r")}
    a.update({n: rng.uniform(0.5, 1.5, 24) for n in ("w1", "w2")})
    d = rng.standard_normal((2, 5, 24))
    for n in a:
        ws.feed(n, a[n])
    ws.feed("d", d)
    t = {n: torch.from_numpy(v).requires_grad_() for n, v in a.items()}
    eps = float(np.float32(1e-5))
    norm = lambda s, w: s / torch.sqrt(s.square().mean(-1, keepdim=True) + eps) * w
    h1 = t["x"] + t["r"]
    m = torch.softmax(norm(h1, t["w1"]), -1)
    h2 = m + h1
    y2 = norm(h2, t["w2"])

    tape = rt.Tape(ws)
    o1, s1 = rt.rms_norm(tape, ["x", "w1", "r"])
    mid = rt.softmax(tape, [o1])
    o2, s2 = rt.rms_norm(tape, [mid, "w2", s1])
    sources = ["x", "w1", "r", "w2"]
    for target, value, reached in ((o2, y2, sources), (s2, h2, sources), (s1, h1, ["x", "w1", "r"])):
        want = torch.autograd.grad((value * torch.from_numpy(d)).sum(), [t[n] for n in reached], retain_graph=True,
                                   allow_unused=True)
        got = tape.gradient(target, reached, output_gradient="d")
        for n, g, w in zip(reached, got, want):
            w = np.zeros_like(a[n]) if w is None else w.numpy()
            # chains of a hundred roundings in 64 bits on values of order 1 to 10
            assert np.abs(ws.fetch(g) - w).max() < 1e-13, (target, n)


@pytest.mark.parametrize("dtype", DTYPES)
def test_operator_rms_norm_gradient_through_the_sum_alone(ws, dtype):
    """dX and dR are dH, bit for bit, and dW is zero."""
    from dragon_amd import runtime as rt
    raw = {"bfloat16": "bfloat16", "float16": "float16"}.get(dtype)
    acc = np.float64 if dtype == "float64" else np.float32
    def feed(name, shape, seed):
        v = torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(getattr(torch, dtype))
        ws.feed(name, v.view(torch.uint16).numpy() if raw else v.numpy(), dtype=raw)
    for shape in ((3, 7, 50), (0, 50)):
        for i, n in enumerate(("x", "r", "dh")):
            feed(n, shape, i)
        ws.feed("w", np.ones(50, acc))
        tape = rt.Tape(ws)
        y, h = rt.rms_norm(tape, ["x", "w", "r"])
        dx, dw, dr = tape.gradient(h, ["x", "w", "r"], output_gradient="dh")
        want = ws.fetch("dh", raw=True)
        for g in (dx, dr):
            assert ws.info(g) == (dtype, shape) and np.array_equal(ws.fetch(g, raw=True), want)
        assert ws.info(dw)[1] == (50,) and not ws.fetch(dw).any()


def test_operators_refuse_extents_that_their_kernels_do_not_count(ws):
    from dragon_amd import runtime as rt
    huge = (1 << 32) + 3  # 3 rows, were it cut to 32 bits
    ws.feed("x", np.zeros((huge, 1), np.float16))
    ws.feed("w", np.zeros(1, np.float32))
    with pytest.raises(rt.DragonError, match="2147483647"):
        ws.run_operator(rt.make_def("RMSNorm", ["x", "w"], ["y"]))


@pytest.mark.parametrize("op,inputs,outputs", [("RMSNorm", "xw", 1), ("RMSNormQuant", "xw", 2), ("RMSNormGradient", "xwx", 2),
                                               ("TopKDistillationLoss", "xit", 1), ("TopKDistillationLossGradient", "xitw", 1),
                                               ("DraftVerify", "pintw", 2)])
def test_operators_name_the_extents_they_refuse(ws, op, inputs, outputs):
    """Without elements, so without memory."""
    from dragon_amd import runtime as rt
    huge = (1 << 32) + 3
    for n, shape, dtype in (("x", (huge, 0), np.float32), ("w", (0,), np.float32), ("i", (huge, 0), np.int64), ("n", (0,), np.int64),
                            ("t", (huge, 0), np.float32), ("p", (huge, 1, 0), np.float32)):
        ws.feed(n, np.zeros(shape, dtype))
    with pytest.raises(rt.DragonError, match="2147483647"):
        ws.run_operator(rt.make_def(op, list(inputs), ["o%d" % i for i in range(outputs)]))
    if op == "RMSNormQuant":
        ws.feed("x", np.zeros((2, 64), np.float32))
        ws.feed("w", np.zeros(64, np.float32))
        with pytest.raises(rt.DragonError, match="2147483647"):  # groups of 32, were it cut
            ws.run_operator(rt.make_def(op, ["x", "w"], ["q", "s"], group_size=(1 << 32) + 32))


def test_operators_of_empty_batches_and_without_drafts(ws):
    from dragon_amd import runtime as rt
    f = lambda *s: np.zeros(s, np.float32)
    for n, a in (("x", f(0, 8)), ("w", f(8)), ("i", np.zeros((0, 2), np.int64)), ("t", f(0, 2)), ("dy", f(0, 8)), ("one", np.ones((), np.float32))):
        ws.feed(n, a)
    tape = rt.Tape(ws)
    y, h = rt.rms_norm(tape, ["x", "w", "x"])
    assert ws.info(y)[1] == (0, 8)
    y = rt.rms_norm(tape, ["x", "w"])
    dx, dw = tape.gradient(y, ["x", "w"], output_gradient="dy")
    assert ws.info(dx)[1] == (0, 8) and not ws.fetch(dw).any()
    loss = rt.topk_distillation_loss(tape, ["x", "i", "t"])
    assert float(ws.fetch(loss)) == 0
    (dx,) = tape.gradient(loss, ["x"], output_gradient="one")
    assert ws.info(dx)[1] == (0, 8)
    p = np.random.default_rng(1).random((3, 1, 9)).astype(np.float32)
    for n, a in (("p", p), ("d", np.zeros((3, 0), np.int64)), ("n", np.zeros(3, np.int64)), ("ua", f(3, 0)), ("us", f(3)), ("q", f(3, 0, 9))):
        ws.feed(n, a)
    for inputs in (["p", "d", "n", "ua", "us"], ["p", "d", "n", "ua", "us", "q"]):
        tokens, accepted = rt.draft_verify(tape, inputs)
        assert not ws.fetch(accepted).any() and not ws.fetch(tokens).any()  # u = 0: the first class


def test_operator_rms_norm_gradient_of_other_rows_than_the_forward_saw(ws):
    """The kept reciprocal roots are as many as the rows: more rows would read behind them."""
    from dragon_amd import runtime as rt
    f = lambda *s: np.ones(s, np.float32)
    for n, a in (("x", f(2, 8)), ("w", f(8)), ("more", f(2000, 8)), ("less", f(1, 8))):
        ws.feed(n, a)
    tape = rt.Tape(ws)
    rt.rms_norm(tape, ["x", "w"])
    (text,), _ = ws.gradient_defs(tape.records[-1][0], ["x"])
    ws.run_operator(text)
    for other in ("more", "less"):
        with pytest.raises(rt.DragonError, match="other rows"):
            ws.run_operator(text.replace('input: "x"', 'input: "%s"' % other))


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("C", [700, 32000, 70001])
def test_draft_verify_at_the_end_of_the_running_sum(dtype, C):
    """u = 1 and more draw the last class of non-zero weight, however the sums round: the last weights here are far
    below half a step of the total."""
    B = 64
    rng = np.random.default_rng(C)
    p = rng.random((B, 1, C)) ** 4
    p[:, :, C - 40:] = 0
    p[:, :, C - 3] = 1e-25
    for u in (1.0, 1.5, np.inf):
        t = {"target": torch.from_numpy(p).to(getattr(torch, dtype)).cuda(), "draft": None,
             "drafted": torch.zeros((B, 0), dtype=torch.int64, device="cuda"), "lengths": None,
             "u_accept": torch.zeros((B, 0), device="cuda"), "u_sample": torch.full((B,), u, device="cuda")}
        tokens, accepted = _run_verify(t)
        assert (tokens == C - 3).all() and not accepted.any(), u


def test_operator_rms_norm_of_a_tensor_that_is_its_own_residual(ws):
    """The sum is right; its gradient would be two shares in one tensor, and is refused."""
    from dragon_amd import runtime as rt
    ws.feed("x", np.arange(8, dtype=np.float32).reshape(2, 4))
    ws.feed("w", np.ones(4, np.float32))
    tape = rt.Tape(ws)
    y, h = rt.rms_norm(tape, ["x", "w", "x"])
    assert np.array_equal(ws.fetch(h), 2 * ws.fetch("x"))
    with pytest.raises(rt.DragonError, match=r"Output\(2\) is the tensor of Output\(0\)"):
        tape.gradient(y, ["x"], output_gradient=h)


def test_tensors_side_by_side_are_taken():
    """Outputs that end where inputs begin, and the other way round, share nothing."""
    from dragon_amd import kernels as K
    flat = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    at = 0
    def carve(shape, dtype):
        nonlocal at
        n = int(np.prod(shape)) * torch.empty((), dtype=dtype).element_size()
        t = flat[at:at + n].view(dtype).view(shape)
        at += n
        return t
    f, b, i64 = torch.float32, torch.bfloat16, torch.int64
    N, C = 4, 64
    x, h, r, y = carve((N, C), f), carve((N, C), f), carve((N, C), f), carve((N, C), f)
    g, rsig, dg = carve((C,), f), carve((N,), f), carve((C,), f)
    q, scale = carve((N, C), torch.uint8), carve((N, 2), f)
    x.normal_(), r.normal_(), g.fill_(1)
    K.rms_norm(N, C, 1e-5, x, r, g, h, rsig, y)
    K.rms_norm_quant(N, C, 32, 1e-5, x, r, g, h, rsig, q, scale)
    K.rms_norm_grad(N, C, h, rsig, g, x, r, dg, y)
    at = (at + 7) // 8 * 8
    index, teacher, stats, loss, dl = carve((N, 2), i64), carve((N, 2), f), carve((N + 1,), f), carve((1,), f), carve((1,), f)
    K.topk_distillation_loss_forward(N, C, 2, 1.0, "MEAN", x, index, teacher, stats, loss)
    K.topk_distillation_loss_backward(N, C, 2, 1.0, "MEAN", x, index, teacher, stats, dl, h)
    at = (at + 7) // 8 * 8
    B, k = 2, 3
    target, tokens, draft = carve((B, k + 1, 16), f), carve((B, k + 1), i64), carve((B, k, 16), f)
    accepted, drafted, lengths = carve((B,), i64), carve((B, k), i64), carve((B,), i64)
    ua, us = carve((B, k), f), carve((B,), f)
    target.fill_(1 / 16)
    K.draft_verify(B, k, 16, target, draft, drafted, lengths, ua, us, tokens, accepted)
    torch.cuda.synchronize()
    assert torch.isfinite(flat[:at // 4 * 4].view(f)[:4 * N * C]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C,k", [(130, 4), (9001, 70), (70001, 5)])
def test_distillation_of_teacher_logits_that_are_not_finite(dtype, C, k):
    """NaN or +inf among a row's listed teacher logits: no loss, and no gradient at the listed classes; the other
    classes' and the other rows' are those of a teacher without it."""
    x, _, teacher = _distill_case(4, C, k, dtype, torch.int64, 6)
    teacher.nan_to_num_(neginf=0.0)
    index = torch.stack([torch.randperm(C)[:k] for _ in range(4)]).cuda()
    dl = torch.full((4,), 0.5, dtype=teacher.dtype, device="cuda")
    stats, loss, dx = _run_distill(x, index, teacher, 1.5, "NONE", dl)
    teacher[1, 2], teacher[3, k - 1] = float("nan"), float("inf")
    got = _run_distill(x, index, teacher, 1.5, "NONE", dl)
    assert torch.equal(got[0], stats) and torch.equal(got[1][::2], loss[::2]) and got[1][1::2].isnan().all()
    listed = torch.zeros((4, C), dtype=torch.bool, device="cuda").scatter_(1, index, True)
    listed[::2] = False
    assert got[2][listed].isnan().all() and torch.equal(got[2][~listed], dx[~listed])
