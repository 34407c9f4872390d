"""The operators of language models without a GPU: what the entry points refuse before anything is
enqueued, the scratch they ask for, and the plain forms the GPU tests compare with."""

import ctypes

import numpy as np
import pytest
import torch

from dragon_amd import _lib, kernels as K
from tests import language_ops as L

P = [ctypes.c_void_p((i + 1) << 32) for i in range(12)]  # distinct, never read
EINVAL, EDTYPE, ESCRATCH = -1, -2, -3
BIG = 1 << 40


def test_rms_norm_refusals():
    f = _lib.lib().dragon_hip_rms_norm
    call = lambda dtype=1, N=4, C=8, x=P[0], r=P[1], g=P[2], h=P[3], rs=P[4], y=P[5]: f(
        dtype, N, C, 1e-5, x, r, g, h, rs, y, None)
    assert call(N=-1) == EINVAL and call(C=0) == EINVAL and call(C=1 << 31) == EINVAL and call(N=1 << 31) == EINVAL
    assert call(x=None) == EINVAL and call(g=None) == EINVAL and call(y=None) == EINVAL
    assert call(y=P[3]) == EINVAL  # y and h in one buffer
    assert call(dtype=4) == EDTYPE and call(dtype=-1) == EDTYPE
    assert call(N=0, x=None, y=None) == 0


def test_rms_norm_quant_refusals():
    f = _lib.lib().dragon_hip_rms_norm_quant
    call = lambda dtype=1, N=4, C=8, group=0, x=P[0], q=P[5], s=P[6]: f(
        dtype, N, C, group, 1e-5, x, P[1], P[2], P[3], P[4], q, s, None)
    assert call(dtype=3) == EDTYPE and call(dtype=9) == EDTYPE
    for group in (-1, 1, 16, 48, 512):
        assert call(group=group) == EINVAL
    assert call(x=None) == EINVAL and call(q=None) == EINVAL and call(s=None) == EINVAL
    assert call(N=-1) == EINVAL and call(C=0) == EINVAL and call(C=1 << 31) == EINVAL
    assert call(N=0) == 0


def test_rms_norm_grad_refusals():
    lib = _lib.lib()
    call = lambda dtype=1, N=4, C=8, h=P[0], dg=P[5], dx=P[6], ws=P[7], nbytes=BIG: lib.dragon_hip_rms_norm_grad(
        dtype, N, C, h, P[1], P[2], P[3], P[4], dg, dx, ws, nbytes, None)
    need = lib.dragon_hip_rms_norm_grad_scratch_bytes(1, 4, 8)
    assert need > 0
    assert call(ws=None) == ESCRATCH and call(nbytes=need - 1) == ESCRATCH
    assert call(h=None) == EINVAL and call(dg=None) == EINVAL and call(dx=None) == EINVAL and call(dx=P[0]) == EINVAL
    assert call(N=-1) == EINVAL and call(C=0) == EINVAL and call(C=1 << 31) == EINVAL and call(N=1 << 31) == EINVAL
    assert call(dtype=5) == EDTYPE
    assert lib.dragon_hip_rms_norm_grad_scratch_bytes(1, 0, 8) == 0
    assert lib.dragon_hip_rms_norm_grad_scratch_bytes(7, 4, 8) == 0


def test_outputs_that_lie_across_inputs_are_refused():
    """Shifted by one element, or of another width: whatever is read after it is written would be lost."""
    lib = _lib.lib()
    at = lambda p, shift: ctypes.c_void_p(p.value + shift)
    norm = lambda x=P[0], r=P[1], h=P[3], y=P[5]: lib.dragon_hip_rms_norm(1, 4, 8, 1e-5, x, r, P[2], h, P[4], y, None)
    for shift in (2, -2, 62, -62):
        assert norm(y=at(P[0], shift)) == EINVAL and norm(y=at(P[1], shift)) == EINVAL
        assert norm(h=at(P[0], shift)) == EINVAL and norm(h=at(P[1], shift)) == EINVAL
        assert norm(y=at(P[3], shift)) == EINVAL
    quant = lambda h=P[3], q=P[5]: lib.dragon_hip_rms_norm_quant(1, 4, 8, 0, 1e-5, P[0], P[1], P[2], h, P[4], q, P[6], None)
    for other in (P[0], P[1], P[3]):
        assert quant(q=other) == EINVAL and quant(q=at(other, 63)) == EINVAL and quant(q=at(other, -31)) == EINVAL
    assert quant(h=at(P[0], 4)) == EINVAL
    grad = lambda dx: lib.dragon_hip_rms_norm_grad(2, 4, 8, P[0], P[1], P[2], P[3], P[4], P[5], dx, P[7], BIG, None)
    for shift in (4, -4, 124):
        assert grad(at(P[0], shift)) == EINVAL and grad(at(P[3], shift)) == EINVAL and grad(at(P[4], shift)) == EINVAL
    loss = lambda dx: lib.dragon_hip_topk_distillation_loss_backward(3, 5, 4, 8, 2, 1.0, -1.0, P[0], P[1], P[2], P[3], P[4],
                                                                     dx, None)
    assert loss(at(P[0], 8)) == EINVAL and loss(at(P[0], -248)) == EINVAL
    verify = lambda tok=P[6], acc=P[7]: lib.dragon_hip_draft_verify(2, 5, 2, 3, 8, P[0], P[1], P[2], P[3], P[4], P[5], tok, acc,
                                                                    P[8], BIG, None)
    assert verify(tok=at(P[2], 40)) == EINVAL and verify(tok=at(P[2], -56)) == EINVAL and verify(tok=at(P[3], -8)) == EINVAL
    assert verify(acc=at(P[2], 8)) == EINVAL and verify(acc=at(P[6], 56)) == EINVAL


def _shared(call, tensors, outputs, very=()):
    """Lays each output over every other tensor: on its first byte, on its last, with its own last byte on the
    first. (output, input) pairs in `very` may be one buffer. tensors: name -> bytes."""
    at = {n: (i + 1) << 32 for i, n in enumerate(tensors)}
    for out in outputs:
        for other in tensors:
            if other == out:
                continue
            for shift in (0, tensors[other] - 1, 1 - tensors[out]):
                if shift == 0 and ((out, other) in very or (other, out) in very):
                    continue
                place = dict(at, **{out: at[other] + shift})
                assert call(*[ctypes.c_void_p(place[n]) for n in tensors]) == EINVAL, (out, other, shift)


def test_no_output_shares_memory_with_another_tensor():
    """Every output against every other tensor of the call, scratch among them."""
    lib = _lib.lib()
    N, C, k = 6, 40, 3
    for dtype, e, a in ((1, 2, 4), (2, 4, 4), (3, 8, 8)):
        n = N * C * e
        _shared(lambda x, r, g, h, rs, y: lib.dragon_hip_rms_norm(dtype, N, C, 1e-5, x, r, g, h, rs, y, None),
                dict(x=n, r=n, g=C * a, h=n, rs=N * a, y=n), ("h", "rs", "y"), [(o, i) for o in "hy" for i in "xr"])
        if dtype != 3:
            for group, groups in ((0, 1), (32, 2)):
                _shared(lambda x, r, g, h, rs, q, s: lib.dragon_hip_rms_norm_quant(dtype, N, C, group, 1e-5, x, r, g, h, rs, q, s, None),
                        dict(x=n, r=n, g=C * a, h=n, rs=N * a, q=N * C, s=N * groups * 4), ("h", "rs", "q", "s"), [("h", "x"), ("h", "r")])
        need = lib.dragon_hip_rms_norm_grad_scratch_bytes(dtype, N, C)
        _shared(lambda h, rs, g, dy, dh, dg, dx, ws: lib.dragon_hip_rms_norm_grad(dtype, N, C, h, rs, g, dy, dh, dg, dx, ws, need, None),
                dict(h=n, rs=N * a, g=C * a, dy=n, dh=n, dg=C * a, dx=n, ws=need), ("dg", "dx", "ws"), [("dx", "dy"), ("dx", "dh")])
        for it, one in ((4, 4), (5, 8)):
            for norm, losses in ((0.0, N), (-1.0, 1)):
                need = lib.dragon_hip_topk_distillation_loss_scratch_bytes(dtype, N, C)
                _shared(lambda x, i, t, st, l, ws: lib.dragon_hip_topk_distillation_loss_forward(
                            dtype, it, N, C, k, 1.0, norm, x, i, t, st, l, ws, need, None),
                        dict(x=n, i=N * k * one, t=N * k * a, st=(N + 1) * a, l=losses * a, ws=need), ("st", "l", "ws"))
                _shared(lambda x, i, t, st, dl, dx: lib.dragon_hip_topk_distillation_loss_backward(
                            dtype, it, N, C, k, 1.0, norm, x, i, t, st, dl, dx, None),
                        dict(x=n, i=N * k * one, t=N * k * a, st=(N + 1) * a, dl=losses * a, dx=n), ("dx",), [("dx", "x")])
            for B, V in ((2, 40), (2, 40000)):  # in one launch, and in two with scratch
                need = lib.dragon_hip_draft_verify_scratch_bytes(dtype, B, k, V)
                assert (need > 0) == (V > 32768)
                sizes = dict(p=B * (k + 1) * V * e, q=B * k * V * e, d=B * k * one, n=B * one, ua=B * k * 4, us=B * 4,
                             tok=B * (k + 1) * one, acc=B * one)
                if need:
                    sizes["ws"] = need
                call = lambda p, q, d, n, ua, us, tok, acc, ws=None: lib.dragon_hip_draft_verify(
                    dtype, it, B, k, V, p, q, d, n, ua, us, tok, acc, ws, need, None)
                _shared(call, sizes, ("tok", "acc") + (("ws",) if need else ()))


def test_distillation_refusals():
    lib = _lib.lib()
    fwd = lambda dtype=1, it=5, N=4, C=8, k=2, t=1.0, norm=-1.0, x=P[0], st=P[3], loss=P[4], ws=P[5], nbytes=BIG: \
        lib.dragon_hip_topk_distillation_loss_forward(dtype, it, N, C, k, t, norm, x, P[1], P[2], st, loss, ws, nbytes, None)
    bwd = lambda dtype=1, it=5, N=4, C=8, k=2, t=1.0, norm=-1.0, x=P[0], st=P[3], dl=P[4], dx=P[5]: \
        lib.dragon_hip_topk_distillation_loss_backward(dtype, it, N, C, k, t, norm, x, P[1], P[2], st, dl, dx, None)
    for f in (fwd, bwd):
        assert f(dtype=4) == EDTYPE and f(it=2) == EDTYPE
        for bad in (dict(N=-1), dict(C=0), dict(k=0), dict(k=1025), dict(t=0.0), dict(t=-2.0), dict(t=float("nan")),
                    dict(t=float("inf")), dict(t=1e-20), dict(t=1e20), dict(norm=float("nan")), dict(x=None), dict(st=None), dict(C=1 << 31),
                    dict(N=(1 << 31) - 1)):
            assert f(**bad) == EINVAL, bad
    assert fwd(loss=None) == EINVAL and bwd(dl=None) == EINVAL and bwd(dx=None) == EINVAL
    assert fwd(ws=None) == ESCRATCH
    assert fwd(nbytes=lib.dragon_hip_topk_distillation_loss_scratch_bytes(1, 4, 8) - 1) == ESCRATCH
    assert bwd(N=0) == 0


def test_draft_verify_refusals():
    lib = _lib.lib()
    call = lambda dtype=2, it=5, B=2, k=3, C=8, t=P[0], d=P[2], ua=P[4], us=P[5], tok=P[6], acc=P[7]: \
        lib.dragon_hip_draft_verify(dtype, it, B, k, C, t, P[1], d, P[3], ua, us, tok, acc, P[8], BIG, None)
    assert call(dtype=4) == EDTYPE and call(it=1) == EDTYPE
    for bad in (dict(B=-1), dict(k=-1), dict(C=0), dict(C=1 << 31), dict(t=None), dict(d=None), dict(ua=None),
                dict(us=None), dict(tok=None), dict(acc=None)):
        assert call(**bad) == EINVAL, bad
    for bad in (dict(acc=P[3]), dict(acc=P[2]), dict(tok=P[2]), dict(tok=P[3]), dict(tok=P[7])):  # outputs on inputs
        assert call(**bad) == EINVAL, bad
    assert call(B=0) == 0


def test_every_operator_has_a_plan():
    for op, dims in (("rms_norm", (8, 4096)), ("rms_norm_quant", (8, 4096, 128)), ("rms_norm_grad", (8, 4096)),
                     ("topk_distillation_loss_forward", (8, 32000, 16)),
                     ("topk_distillation_loss_backward", (8, 32000, 16)), ("draft_verify", (2, 4, 32000))):
        assert "[" in K.plan_name(op, "bfloat16", dims)
        with pytest.raises(ValueError):
            K.plan_name(op, "bfloat16", (4, -1, 0))


def test_plans_by_size():
    """Which kernels sizes take: rows in registers up to 4096 packets, wavefront rows, segments and parts."""
    plan = lambda op, dims, dtype="bfloat16": K.plan_name(op, dtype, dims)
    assert plan("rms_norm", (8, 4096)).startswith("threads_per_row=256:packets=2:rms_norm_rows<")
    assert plan("rms_norm", (8, 64)).startswith("threads_per_row=8:packets=1:")
    assert plan("rms_norm", (8, 32768)).startswith("threads_per_row=1024:packets=4:")
    for columns, threads in ((8192, 512), (8200, 640), (10240, 640), (10248, 768), (12288, 768), (12296, 1024)):
        assert plan("rms_norm", (8, columns)).startswith("threads_per_row=%d:packets=2:" % threads)
        assert "grad_rows<T,%d,2" % threads in plan("rms_norm_grad", (8, columns))
    assert "rms_norm_rows_looped" in plan("rms_norm", (8, 32769)) and "looped" in plan("rms_norm", (8, 7))
    assert "rms_norm_rows_looped" in plan("rms_norm_quant", (8, 40000, 128))
    assert "grad_rows" in plan("rms_norm_grad", (8, 16384)) and "grad_dots" in plan("rms_norm_grad", (8, 16392))
    assert "grad_rows" in plan("rms_norm_grad", (8, 16384), "float32")
    f, b = "topk_distillation_loss_forward", "topk_distillation_loss_backward"
    assert "IndexT,64,1,true" in plan(f, (2048, 16384, 64)) and "IndexT,256,1,true" in plan(f, (2047, 16384, 64))
    assert "IndexT,256,1,true" in plan(f, (2048, 65536, 64)) and "IndexT,256,1,false" in plan(f, (2048, 65544, 64))
    assert "IndexT,256,1,true" in plan(f, (512, 32768, 64)) and "IndexT,256,1,false" in plan(f, (511, 32768, 64))
    # up to 16 rows that wavefronts finish are reduced by the same launch
    assert plan(f, (16, 4096, 64)).count("[") == 1 and plan(f, (17, 4096, 64)).count("[") == 2
    assert plan(f, (16, 131072, 200)).count("[") == 2 and plan(f, (17, 131072, 200)).count("[") == 3
    assert plan(f, (16, 131072, 257)).count("[") == 3 and plan(f, (1, 16384, 64)).count("[") == 2
    assert "IndexT,64,1,true" in plan(f, (100, 4096, 64)) and "IndexT,64,4,true" in plan(f, (100, 4096, 256))
    assert "IndexT,256,4,true" in plan(f, (100, 4096, 257)) and "IndexT,256,1,true" in plan(f, (100, 16384, 64))
    assert "IndexT,256,1,false" in plan(f, (100, 16392, 64)) and "distill_forward_join<T,IndexT,64,1>" in plan(f, (100, 16392, 64))
    assert "distill_forward_join<T,IndexT,256,4>" in plan(f, (100, 131072, 1024))
    assert "IndexT,64,4,1" in plan(b, (100, 2048, 64)) and "IndexT,64,8,4" in plan(b, (100, 4096, 65))
    assert "IndexT,256,2,1" in plan(b, (100, 131072, 64)) and "IndexT,256,4,4" in plan(b, (100, 131072, 300))
    assert "draft_verify_rows" in plan("draft_verify", (1, 4, 32768), "float32")
    assert "draft_verify_runs" in plan("draft_verify", (1, 4, 32769), "float32")
    assert "draft_verify_rows" in plan("draft_verify", (512, 4, 131072), "float32")
    assert "draft_verify_runs" in plan("draft_verify", (512, 4, 1 << 20), "float32")


# ---------------------------------------------------------------- the operators of the host layer

@pytest.fixture()
def ws():
    from dragon_amd import runtime
    w = runtime.Workspace("language_ops_host_test")
    yield w
    w.close()


def test_gradient_definitions_of_rms_norm_by_what_arrives(ws):
    """A definition names no tensor that does not exist: neither "NULL" nor "" is an input of its own."""
    from dragon_amd import runtime as rt
    forward = rt.make_def("RMSNorm", ["x", "w", "r"], ["y", "h"], name="n", axis=-1, epsilon=1e-3)
    grads = ["x_grad", "w_grad", "r_grad"]
    for none in ("NULL", ""):
        for arriving, op, inputs in ((["dy", "dh"], "RMSNormGradient", ["h", "w", "dy", "dh"]),
                                     (["dy", none], "RMSNormGradient", ["h", "w", "dy"]),
                                     ([none, "dh"], "RMSNormSumGradient", ["dh", "w"])):
            (text,), names = ws.gradient_defs(forward, arriving)
            assert names == grads and 'type: "%s"' % op in text
            assert [p.split('"')[1] for p in text.split("input: ")[1:]] == inputs
            assert [p.split('"')[1] for p in text.split("output: ")[1:]] == grads
        with pytest.raises(rt.DragonError, match="No gradient"):
            ws.gradient_defs(forward, [none, none])
    assert "RMSNormSumGradient" in rt.registered_operators()


@pytest.mark.parametrize("op,inputs,outputs", [
    ("RMSNorm", "xwr", "yy"), ("RMSNormQuant", "xw", "qq"), ("RMSNormQuant", "xwr", "qsq"), ("RMSNormGradient", "xwr", "aa"),
    ("RMSNormGradient", "xwr", "aba"), ("RMSNormSumGradient", "xw", "aba"), ("DraftVerify", "xiirr", "tt")])
def test_operators_refuse_one_tensor_for_two_outputs(ws, op, inputs, outputs):
    """They differ in type or size: the second would free the memory that was taken for the first. Refused before
    the device is looked at."""
    from dragon_amd import runtime as rt
    for n, dtype in (("x", np.float32), ("w", np.float32), ("r", np.float32), ("i", np.int64)):
        ws.feed(n, np.zeros(8, dtype))
    with pytest.raises(rt.DragonError, match=r"Output\(\d\) is the tensor of Output\(0\)"):
        ws.run_operator(rt.make_def(op, list(inputs), list(outputs)))


@pytest.mark.parametrize("op,inputs,outputs", [("RMSNorm", "xw", "y"), ("RMSNormQuant", "xw", "qs"), ("RMSNormSumGradient", "xw", "abc"),
                                               ("TopKDistillationLoss", "xir", "l"), ("DraftVerify", "xiirr", "ta")])
def test_cached_operators_refuse_an_input_for_an_output(ws, op, inputs, outputs):
    """The schema refuses it of a new operator; one that is rebound to other tensors says so too."""
    from dragon_amd import runtime as rt
    for n, dtype in (("x", np.float32), ("w", np.float32), ("r", np.float32), ("i", np.int64)):
        ws.feed(n, np.zeros(8, dtype))
    define = lambda out: rt.make_def(op, list(inputs), out, cache_key="k")
    try:
        ws.run_operator(define(list(outputs)))
    except rt.DragonError:
        pass  # it is created; without a device, or with shapes that do not fit, it does not run
    with pytest.raises(rt.DragonError, match=r"Output\(0\) is the tensor of Input\(0\)"):
        ws.run_operator(define([inputs[0]] + list(outputs[1:])))


# ---------------------------------------------------------------- the plain forms themselves

def test_plain_distillation_is_the_divergence_of_torch():
    g = torch.Generator().manual_seed(0)
    n, c, k, t = 5, 30, 4, 1.7
    x = torch.randn(n, c, generator=g, dtype=torch.float64)
    teacher = torch.randn(n, k, generator=g, dtype=torch.float64)
    index = torch.stack([torch.randperm(c, generator=g)[:k] for _ in range(n)])
    p = torch.softmax(teacher / t, 1)
    want = (p * (p.log() - torch.log_softmax(x / t, 1).gather(1, index))).sum(1) * t * t
    stats, rows, loss = L.distill_forward(t, "MEAN", x.numpy(), index.numpy(), teacher.numpy())
    assert np.allclose(rows, want.numpy(), rtol=1e-13) and np.allclose(loss, want.mean().item(), rtol=1e-13)
    x.requires_grad_()
    p = torch.softmax(teacher / t, 1)
    ((p * (p.log() - torch.log_softmax(x / t, 1).gather(1, index))).sum(1) * t * t).mean().backward()
    dx, _, _ = L.distill_backward(t, "MEAN", x.detach().numpy(), index.numpy(), teacher.numpy(), stats, np.ones(1))
    assert np.allclose(dx, x.grad.numpy(), rtol=1e-12, atol=1e-15)


def test_plain_rms_norm_gradient_is_that_of_torch():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 9, generator=g, dtype=torch.float64, requires_grad=True)
    gamma = (torch.rand(9, generator=g, dtype=torch.float64) + 0.5).requires_grad_()
    dy, dh = torch.randn(4, 9, generator=g, dtype=torch.float64), torch.randn(4, 9, generator=g, dtype=torch.float64)
    y = x / torch.sqrt(x.square().mean(1, keepdim=True) + 1e-5) * gamma
    ((y * dy).sum() + (x * dh).sum()).backward()
    _, rs, want = L.rms_norm(x.detach().numpy(), None, gamma.detach().numpy(), 1e-5)
    assert np.allclose(want, y.detach().numpy(), rtol=1e-13)
    dx, dg = L.rms_norm_grad(x.detach().numpy(), rs, gamma.detach().numpy(), dy.numpy(), dh.numpy())
    assert np.allclose(dx, x.grad.numpy(), rtol=1e-12, atol=1e-14) and np.allclose(dg, gamma.grad.numpy(), rtol=1e-12)


def test_plain_verification_follows_the_target():
    """Accepted and drawn first tokens together have the target's distribution: 40000 draws, five classes. A
    class's share is off by more than 5 standard deviations (at most 0.0125) about once in a million."""
    rng = np.random.default_rng(2)
    p, q = np.array([0.4, 0.3, 0.2, 0.1, 0.0]), np.array([0.1, 0.2, 0.3, 0.2, 0.2])
    B = 40000
    drafted = rng.choice(5, (B, 1), p=q)
    target = np.broadcast_to(np.stack([p, p]), (B, 2, 5))
    tokens, n = L.draft_verify(target, np.broadcast_to(q, (B, 1, 5)), drafted, None, rng.random((B, 1)), rng.random(B))
    share = np.bincount(tokens[:, 0], minlength=5) / B
    assert np.abs(share - p).max() < 0.0125 and share[4] == 0
