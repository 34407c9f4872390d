"""The operators of language models that the package offers beside LayerNorm, Softmax and the
softmax cross-entropy loss, as cases to be measured and compared:

  rms_norm          residual addition and root-mean-square norm, 16- or 32-bit output
  rms_norm_quant    the same with an e4m3 output and a scale per row or per group of columns
  rms_norm_grad     its gradient, with the gradient that arrives along the residual stream
  distill_forward   loss of a student against a teacher's top logits
  distill_backward  its gradient with respect to the student's logits
  draft_verify      verification of drafted tokens against the target's probabilities

``run`` computes each in plain torch operations where ``own`` is false and calls
``dragon_amd.kernels`` where it is true.
"""

import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
INTS = {"i32": torch.int32, "i64": torch.int64}
EPS = 1e-5
FP8_MAX = 448.0     # the largest e4m3 value
AMAX_FLOOR = 1e-30  # keeps the scale of a group of zeros a normal number


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one new token of a served model: the whole cost is launching and one row's latency
        {"name": "rms_norm_token", "op": "rms_norm", "dtype": "bf16", "rows": 1, "cols": 4096, "residual": True},
        # a training step's tokens through a wide model
        {"name": "rms_norm_step", "op": "rms_norm", "dtype": "bf16", "rows": 8192, "cols": 8192, "residual": True},
        # a decode batch whose next product runs in 8 bits, one scale per token
        {"name": "rms_norm_quant_batch", "op": "rms_norm_quant", "dtype": "bf16", "rows": 64, "cols": 5120,
         "residual": True, "group": 0},
        # a long prompt with scales per 128 columns
        {"name": "rms_norm_quant_prompt", "op": "rms_norm_quant", "dtype": "bf16", "rows": 16384, "cols": 4096,
         "residual": True, "group": 128},
        # the gradient of a training step's norm
        {"name": "rms_norm_grad_step", "op": "rms_norm_grad", "dtype": "bf16", "rows": 8192, "cols": 4096,
         "residual": True},
        # an odd width in 32 bits, without a residual stream (a final norm)
        {"name": "rms_norm_grad_odd", "op": "rms_norm_grad", "dtype": "f32", "rows": 2051, "cols": 1001,
         "residual": False},
        # a large vocabulary, every token of a micro-batch
        {"name": "distill_forward_large", "op": "distill_forward", "dtype": "bf16", "rows": 4096, "cols": 131072,
         "k": 64, "temperature": 2.0, "reduction": "VALID", "index": "i32"},
        # few rows of a large vocabulary, a loss for each: the tail of a sequence
        {"name": "distill_forward_few", "op": "distill_forward", "dtype": "f32", "rows": 12, "cols": 131072,
         "k": 20, "temperature": 1.0, "reduction": "NONE", "index": "i64"},
        {"name": "distill_backward_large", "op": "distill_backward", "dtype": "bf16", "rows": 4096, "cols": 131072,
         "k": 64, "temperature": 2.0, "reduction": "VALID", "index": "i32"},
        # an odd vocabulary, where hardly a row starts on a packet, and a weight for each row's gradient
        {"name": "distill_backward_odd", "op": "distill_backward", "dtype": "bf16", "rows": 1000, "cols": 50257,
         "k": 32, "temperature": 1.5, "reduction": "NONE", "index": "i64"},
        # one conversation, four drafted tokens: latency alone
        {"name": "draft_verify_one", "op": "draft_verify", "dtype": "f32", "batch": 1, "drafts": 4, "cols": 32000,
         "sampled": True, "index": "i64"},
        # a served batch over a large vocabulary
        {"name": "draft_verify_batch", "op": "draft_verify", "dtype": "f32", "batch": 192, "drafts": 5,
         "cols": 131072, "sampled": True, "index": "i32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rms_norm", "rms_norm_quant", "rms_norm_grad", "distill_forward", "distill_backward",
                     "draft_verify"])
    dtype = rng.choice(["f16", "bf16", "bf16", "f32"])
    if op.startswith("rms_norm"):
        cols = _log(rng, 64, 16384)
        if rng.random() < 0.7:
            cols = max(64, cols // 64 * 64)
        rows = _log(rng, 1, min(32768, (1 << 25) // cols))
        case = {"op": op, "dtype": dtype, "rows": rows, "cols": cols, "residual": rng.random() < 0.7}
        if op == "rms_norm_quant":
            case["group"] = rng.choice([0, 0, 32, 64, 128, 256])
        return case
    if op.startswith("distill"):
        cols = _log(rng, 1000, 200000)
        if rng.random() < 0.6:
            cols = cols // 64 * 64
        rows = _log(rng, 1, min(8192, (1 << 28) // cols))
        return {"op": op, "dtype": dtype, "rows": rows, "cols": cols, "k": _log(rng, 1, 256),
                "temperature": rng.choice([1.0, 1.5, 2.0, 4.0]),
                "reduction": rng.choice(["VALID", "VALID", "MEAN", "NONE"]), "index": rng.choice(["i32", "i64"])}
    cols = _log(rng, 1000, 200000)
    if rng.random() < 0.6:
        cols = cols // 64 * 64
    drafts = rng.randint(1, 8)
    batch = _log(rng, 1, min(256, (1 << 26) // (cols * drafts)))
    return {"op": op, "dtype": dtype, "batch": batch, "drafts": drafts, "cols": cols,
            "sampled": rng.random() < 0.75, "index": rng.choice(["i32", "i64"])}


# ---------------------------------------------------------------- inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, shape, scale=1.0):
    return torch.empty(shape, device="cuda").normal_(0.0, scale, generator=g)


def _prepare_rms(case, g):
    dt = DTYPES[case["dtype"]]
    n, c = case["rows"], case["cols"]
    # activations: unit scale with a few channels that are many times larger, as residual streams have
    spread = 1.0 + 20.0 * (torch.rand(c, device="cuda", generator=g) < 0.004).float()
    s = {"case": case}
    s["gamma"] = 1.0 + _normal(g, (c,), 0.2)
    residual = case["residual"]
    if case["op"] == "rms_norm_grad":
        s["h"] = (_normal(g, (n, c), 2.0) * spread).to(dt)  # what the forward kept of x + residual
        s["rsig"] = (s["h"].float().square().mean(1) + EPS).rsqrt()
        s["dy"] = _normal(g, (n, c), 0.1).to(dt)
        s["dh"] = _normal(g, (n, c), 0.1).to(dt) if residual else None
        s["dgamma"] = torch.empty(c, device="cuda")
        s["dx"] = torch.empty((n, c), dtype=dt, device="cuda")
        return s
    s["x"] = _normal(g, (n, c)).to(dt)
    s["residual"] = (_normal(g, (n, c), 2.0) * spread).to(dt) if residual else None
    s["h"] = torch.empty((n, c), dtype=dt, device="cuda") if residual else None
    if case["op"] == "rms_norm":
        s["rsig"] = torch.empty(n, device="cuda")
        s["y"] = torch.empty((n, c), dtype=dt, device="cuda")
    else:
        group = case["group"] or c
        s["q"] = torch.empty((n, c), dtype=torch.float8_e4m3fn, device="cuda")
        s["scale"] = torch.empty((n, -(-c // group)), device="cuda")
    return s


def _prepare_distill(case, g):
    dt, it = DTYPES[case["dtype"]], INTS[case["index"]]
    n, c, k = case["rows"], case["cols"], case["k"]
    # distinct classes per row: a start and a stride that does not come round
    start = torch.randint(0, c, (n, 1), device="cuda", generator=g)
    stride = torch.randint(1, max(2, c // k), (n, 1), device="cuda", generator=g)
    index = (start + stride * torch.arange(k, device="cuda")) % c
    teacher = torch.sort(_normal(g, (n, k), 2.0) + 9.0, dim=1, descending=True).values
    x = torch.empty((n, c), dtype=dt, device="cuda").normal_(0.0, 2.0, generator=g)
    # a student that agrees with its teacher roughly
    x.scatter_(1, index, (teacher + _normal(g, (n, k), 1.0)).to(dt))
    # a tenth of the rows is padding, and some rows list fewer classes than k
    padded = torch.rand((n, 1), device="cuda", generator=g) < 0.1
    kept = torch.randint(max(1, k // 2), k + 1, (n, 1), device="cuda", generator=g)
    index = torch.where(padded | (torch.arange(k, device="cuda") >= kept), -1, index)
    s = {"case": case, "x": x, "index": index.to(it), "teacher": teacher}
    if case["op"] == "distill_forward":
        s["stats"] = torch.empty(n + 1, device="cuda")
        s["loss"] = torch.empty(n if case["reduction"] == "NONE" else 1, device="cuda")
        return s
    # what the forward leaves for the gradient: the log-sum-exp of each row, +inf where nothing is
    # listed, and the divisor of the reduction
    lse = torch.logsumexp(x.float() / case["temperature"], 1)
    counted = (s["index"] >= 0).any(1)
    lse = torch.where(counted, lse, math.inf)
    divisor = {"VALID": counted.sum().float(), "MEAN": torch.tensor(float(n), device="cuda"),
               "NONE": torch.tensor(1.0, device="cuda")}[case["reduction"]]
    s["stats"] = torch.cat([lse, divisor.view(1)])
    if case["reduction"] == "NONE":
        s["dloss"] = torch.rand(n, device="cuda", generator=g)
    else:
        s["dloss"] = torch.full((1,), 0.5, device="cuda")
    s["dx"] = torch.empty_like(x)
    return s


def _prepare_verify(case, g):
    dt, it = DTYPES[case["dtype"]], INTS[case["index"]]
    b, k, c = case["batch"], case["drafts"], case["cols"]

    def logits(rows, peak):
        return _normal(g, (rows, c), 3.0).scatter_(1, peak, 16.0)

    peak = torch.randint(0, c, (b * (k + 1), 1), device="cuda", generator=g)
    p = torch.softmax(logits(b * (k + 1), peak), 1).view(b, k + 1, c)
    # the draft: half the target, half another distribution with the same favourite
    q = p[:, :k].clone().mul_(0.5)
    q += torch.softmax(logits(b * k, peak.view(b, k + 1, 1)[:, :k].reshape(b * k, 1)), 1).view(b, k, c) * 0.5
    drafted = torch.multinomial(q.view(b * k, c), 1, generator=g).view(b, k)
    s = {"case": case, "target": p.to(dt), "draft": q.to(dt) if case["sampled"] else None}
    s["drafted"] = drafted.to(it)
    s["lengths"] = torch.where(torch.rand(b, device="cuda", generator=g) < 0.8, k,
                               torch.randint(0, k + 1, (b,), device="cuda", generator=g)).to(it)
    s["u_accept"] = torch.rand((b, k), device="cuda", generator=g)
    s["u_sample"] = torch.rand(b, device="cuda", generator=g)
    s["tokens"] = torch.empty((b, k + 1), dtype=it, device="cuda")
    s["accepted"] = torch.empty(b, dtype=it, device="cuda")
    return s


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op.startswith("rms_norm"):
        return _prepare_rms(case, g)
    if op.startswith("distill"):
        return _prepare_distill(case, g)
    return _prepare_verify(case, g)


# ---------------------------------------------------------------- the package's calls

def _own(s):
    from dragon_amd import kernels as K
    case = s["case"]
    op = case["op"]
    if op == "rms_norm":
        K.rms_norm(case["rows"], case["cols"], EPS, s["x"], s["residual"], s["gamma"], s["h"], s["rsig"], s["y"])
        return {"y": s["y"], "h": s["h"], "rsig": s["rsig"]}
    if op == "rms_norm_quant":
        K.rms_norm_quant(case["rows"], case["cols"], case["group"], EPS, s["x"], s["residual"], s["gamma"], s["h"],
                         None, s["q"], s["scale"])
        return {"q": s["q"], "scale": s["scale"], "h": s["h"]}
    if op == "rms_norm_grad":
        K.rms_norm_grad(case["rows"], case["cols"], s["h"], s["rsig"], s["gamma"], s["dy"], s["dh"], s["dgamma"],
                        s["dx"])
        return {"dx": s["dx"], "dgamma": s["dgamma"]}
    if op == "distill_forward":
        K.topk_distillation_loss_forward(case["rows"], case["cols"], case["k"], case["temperature"], case["reduction"],
                                         s["x"], s["index"], s["teacher"], s["stats"], s["loss"])
        return {"loss": s["loss"], "stats": s["stats"]}
    if op == "distill_backward":
        K.topk_distillation_loss_backward(case["rows"], case["cols"], case["k"], case["temperature"], case["reduction"],
                                          s["x"], s["index"], s["teacher"], s["stats"], s["dloss"], s["dx"])
        return {"dx": s["dx"]}
    K.draft_verify(case["batch"], case["drafts"], case["cols"], s["target"], s["draft"], s["drafted"], s["lengths"],
                   s["u_accept"], s["u_sample"], s["tokens"], s["accepted"])
    return {"tokens": s["tokens"], "accepted": s["accepted"]}


# ---------------------------------------------------------------- the plain forms

def _plain_rms(s):
    t = s["x"].float()
    if s["residual"] is not None:
        t = t + s["residual"].float()
    rsig = 1.0 / torch.sqrt(t.square().mean(1) + EPS)
    return t, rsig, t * rsig[:, None] * s["gamma"]


def _plain_rms_norm(s):
    t, rsig, y = _plain_rms(s)
    dt = s["x"].dtype
    return {"y": y.to(dt), "h": t.to(dt) if s["residual"] is not None else None, "rsig": rsig}


def _plain_rms_norm_quant(s):
    t, rsig, y = _plain_rms(s)
    n, c = y.shape
    group = s["case"]["group"] or c
    groups = -(-c // group)
    if groups * group != c:
        y = torch.cat([y, y.new_zeros((n, groups * group - c))], 1)
    y = y.view(n, groups, group)
    scale = y.abs().amax(2).clamp(min=AMAX_FLOOR) / FP8_MAX
    q = (y / scale[:, :, None]).view(n, groups * group)[:, :c].to(torch.float8_e4m3fn)
    return {"q": q, "scale": scale, "h": t.to(s["x"].dtype) if s["residual"] is not None else None}


def _plain_rms_norm_grad(s):
    h, dy, rsig = s["h"].float(), s["dy"].float(), s["rsig"][:, None]
    z = dy * s["gamma"]
    dx = rsig * (z - h * (rsig.square() * (z * h).mean(1, keepdim=True)))
    if s["dh"] is not None:
        dx = dx + s["dh"].float()
    return {"dx": dx.to(s["h"].dtype), "dgamma": (dy * h * rsig).sum(0)}


def _plain_teacher(s):
    """Which entries count, their classes, and the teacher's probabilities over them and their logarithms."""
    c, temperature = s["case"]["cols"], s["case"]["temperature"]
    index = s["index"].long()
    listed_ = (index >= 0) & (index < c)
    z = torch.where(listed_, s["teacher"] / temperature, -math.inf)
    top = z.amax(1, keepdim=True)
    z = z - torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = z.exp()
    total = e.sum(1, keepdim=True)
    total = torch.where(total > 0, total, torch.ones_like(total))
    return listed_, torch.where(listed_, index, 0), e / total, torch.where(listed_, z - total.log(), 0.0)


def _plain_distill_forward(s):
    temperature = s["case"]["temperature"]
    x = s["x"].float() / temperature
    top = x.amax(1, keepdim=True)
    lse = (x - top).exp().sum(1, keepdim=True).log() + top
    on, index, t, log_t = _plain_teacher(s)
    rows = (t * (log_t - x.gather(1, index) + lse)).sum(1) * temperature ** 2
    counted = on.any(1)
    divisor = counted.sum().float()
    if s["case"]["reduction"] != "VALID":
        divisor = torch.full_like(divisor, s["case"]["rows"] if s["case"]["reduction"] == "MEAN" else 1.0)
    rows = torch.where(counted, rows, 0.0)
    loss = rows if s["case"]["reduction"] == "NONE" else (rows.sum() / torch.clamp(divisor, min=1.0)).view(1)
    lse = torch.where(counted, lse[:, 0], math.inf)
    return {"loss": loss, "stats": torch.cat([lse, divisor.view(1)])}


def _plain_distill_backward(s):
    temperature = s["case"]["temperature"]
    n = s["case"]["rows"]
    g = (s["x"].float() / temperature - s["stats"][:n, None]).exp()
    on, index, t, _ = _plain_teacher(s)
    g = g.scatter_add(1, index, -t)
    w = s["dloss"] / torch.clamp(s["stats"][n:], min=0.5) * temperature
    return {"dx": (g * w[:, None]).to(s["x"].dtype)}


def _plain_draft_verify(s):
    case = s["case"]
    b, k, c = case["batch"], case["drafts"], case["cols"]
    it = s["drafted"].dtype
    drafted = s["drafted"].long()
    lengths = s["lengths"].long()
    rows = torch.arange(b, device="cuda")
    places = torch.arange(k + 1, device="cuda")
    p_d = s["target"][:, :k].gather(2, drafted[:, :, None])[:, :, 0].double()
    if s["draft"] is not None:
        q_d = s["draft"].gather(2, drafted[:, :, None])[:, :, 0].double()
    else:
        q_d = torch.ones_like(p_d)
    ok = (s["u_accept"].double() * q_d < p_d) & (places[:k] < lengths[:, None])
    n = ok.long().cumprod(1).sum(1)
    refused = n < lengths
    at = n.clamp(max=k - 1)
    r = s["target"][rows, n].double()
    if s["draft"] is not None:
        r = torch.where(refused[:, None], (r - s["draft"][rows, at].double()).clamp(min=0.0), r)
    else:
        r = r.scatter(1, drafted[rows, at][:, None],
                      torch.where(refused, 0.0, r.gather(1, drafted[rows, at][:, None])[:, 0])[:, None])
    cdf = r.cumsum(1)
    token = (cdf <= s["u_sample"].double()[:, None] * cdf[:, -1:]).sum(1).clamp(max=c - 1)
    full = torch.cat([drafted, drafted.new_zeros((b, 1))], 1)
    out = torch.where(places < n[:, None], full, torch.where(places == n[:, None], token[:, None], -1))
    return {"tokens": out.to(it), "accepted": n.to(it)}


_PLAIN = {
    "rms_norm": _plain_rms_norm,
    "rms_norm_quant": _plain_rms_norm_quant,
    "rms_norm_grad": _plain_rms_norm_grad,
    "distill_forward": _plain_distill_forward,
    "distill_backward": _plain_distill_backward,
    "draft_verify": _plain_draft_verify,
}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    op, e = case["op"], BYTES[case["dtype"]]
    if op.startswith("rms_norm"):
        n, c = case["rows"], case["cols"]
        streams = 2 if case["residual"] else 1
        if op == "rms_norm":  # x and residual in, h and y out, gamma, rsig
            return {"bytes": 2 * streams * n * c * e + 4 * c + 4 * n, "flops": 5 * n * c}
        if op == "rms_norm_quant":  # the same with one byte per element of y and the scales
            groups = -(-c // (case["group"] or c))
            return {"bytes": (2 * streams - 1) * n * c * e + n * c + 4 * c + 4 * n * groups, "flops": 7 * n * c}
        # h and dy (and dh) in, dx out, gamma in, dgamma out
        return {"bytes": (2 + streams) * n * c * e + 8 * c + 4 * n, "flops": 9 * n * c}
    ints = 4 if case["index"] == "i32" else 8
    if op.startswith("distill"):
        n, c, k = case["rows"], case["cols"], case["k"]
        side = n * k * (4 + ints) + 4 * n
        # a padded row (one in ten) is not read; its gradient is written all the same
        if op == "distill_forward":
            return {"bytes": 0.9 * n * c * e + side, "flops": 4 * n * c}
        return {"bytes": 1.9 * n * c * e + side, "flops": 4 * n * c}
    b, k, c = case["batch"], case["drafts"], case["cols"]
    # one row of the target per sequence, and one of the draft where a token is refused: a drafted
    # token passes about three times in four
    refused = 1.0 - 0.75 ** k if case["sampled"] else 0.0
    return {"bytes": b * c * e * (1.0 + refused) + b * k * (2 * ints + 4 + 2 * e), "flops": 3 * b * c}


# ---------------------------------------------------------------- from the definitions, in 64 bits

def exact(case, seed):
    op = case["op"]
    if op == "draft_verify":
        return None  # whole numbers
    s = prepare(case, seed)
    if op in ("rms_norm", "rms_norm_quant"):
        a = s["x"].double()
        if s["residual"] is not None:
            a += s["residual"].double()
        n, c = a.shape
        inv = (torch.linalg.vector_norm(a, dim=1).pow(2) / c + EPS).pow(-0.5)
        kept = a.clone() if s["residual"] is not None else None
        a *= inv.view(n, 1)
        a *= s["gamma"].double()
        if op == "rms_norm":
            return {"y": a, "h": kept, "rsig": inv}
        scales = []
        width = case["group"] or c
        for lo in range(0, c, width):
            part = a[:, lo:lo + width]
            scale = torch.maximum(part.max(1).values, -part.min(1).values).clamp(min=AMAX_FLOOR) / FP8_MAX
            part /= scale.view(n, 1)
            scales.append(scale)
        return {"q": a, "scale": torch.stack(scales, 1), "h": kept}
    if op == "rms_norm_grad":
        h, dy, rs, gamma = s["h"].double(), s["dy"].double(), s["rsig"].double(), s["gamma"].double()
        n, c = h.shape
        unit = h * rs.view(n, 1)  # the normalised rows
        into = dy * gamma
        along = torch.linalg.vecdot(into, unit) / c
        dx = (into - unit * along.view(n, 1)) * rs.view(n, 1)
        if s["dh"] is not None:
            dx += s["dh"].double()
        return {"dx": dx, "dgamma": torch.linalg.vecdot(dy, unit, dim=0)}
    n, c, temperature = case["rows"], case["cols"], case["temperature"]
    on = (s["index"] >= 0) & (s["index"] < c)
    teacher = torch.where(on, s["teacher"].double() / temperature, -torch.inf)
    counted = on.any(1)
    t = torch.softmax(torch.where(counted.view(n, 1), teacher, 0.0), 1) * on
    step = max(1, (1 << 26) // c)
    divisor = {"VALID": float(counted.sum()), "MEAN": float(n), "NONE": 1.0}[case["reduction"]]
    if op == "distill_forward":
        losses, lses = [], []
        for lo in range(0, n, step):
            rows = slice(lo, lo + step)
            x = s["x"][rows].double() / temperature
            lse = torch.logsumexp(x, 1)
            chosen = torch.gather(x, 1, s["index"][rows].long().clamp(0, c - 1)) - lse.view(-1, 1)
            losses.append((torch.xlogy(t[rows], t[rows]) - t[rows] * chosen).sum(1))
            lses.append(lse)
        loss = torch.cat(losses).masked_fill(~counted, 0.0) * (temperature * temperature)
        if case["reduction"] != "NONE":
            loss = loss.sum().view(1) / max(divisor, 1.0)
        lse = torch.cat(lses).masked_fill(~counted, torch.inf)
        return {"loss": loss, "stats": torch.cat([lse, lse.new_tensor([divisor])])}
    scale = (s["dloss"].double() * (temperature / max(float(s["stats"][n]), 0.5))).expand(n)
    dx = torch.empty((n, c), dtype=torch.float64, device="cuda")
    for lo in range(0, n, step):
        rows = slice(lo, min(lo + step, n))
        part = torch.exp(s["x"][rows].double() / temperature - s["stats"][:n][rows].double().view(-1, 1))
        where_ = s["index"][rows].long().clamp(0, c - 1)
        part.scatter_add_(1, where_, -t[rows])
        dx[rows] = part * scale[rows].view(-1, 1)
    return {"dx": dx}
