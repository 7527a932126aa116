"""Cases for group norm with an activation, a teacher's top logits and the distillation loss on them.

``run`` computes the operators in plain torch operations, or with the framework's kernels where ``own`` is true; ``exact``
gives the same results in 64 bits."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5

# the most bytes of the main input of a drawn case: half of what the largest listed case of its operator has
GN_MAX = 400 * 56 * 56 * 256
DISTILL_MAX = 8192 * 131072
TOP_MAX = 4096 * 131072


def _gn(name, n, h, w, c, groups, dtype, act, residual, train):
    return {"name": name, "op": "group_norm", "n": n, "h": h, "w": w, "c": c, "groups": groups, "dtype": dtype, "act": act,
            "residual": residual, "train": train}


def _distill(name, rows, classes, k, dtype, temperature, rest, ragged, mean, train):
    return {"name": name, "op": "distill", "rows": rows, "classes": classes, "k": k, "dtype": dtype,
            "temperature": temperature, "rest": rest, "ragged": ragged, "mean": mean, "train": train}


def _top(name, rows, classes, k, dtype, temperature):
    return {"name": name, "op": "top", "rows": rows, "classes": classes, "k": k, "dtype": dtype,
            "temperature": temperature}


def listed():
    return [
        # one image at inference: the last stage of a ResNet, where the latency of the call counts
        _gn("gn_one_image", 1, 7, 7, 2048, 32, "fp16", "relu", True, False),
        # first stage of a ResNet-18 on 32x32 images at the default batch: thousands of small samples
        _gn("gn_small_images", 3200, 8, 8, 64, 32, "fp32", "relu", True, True),
        # block output of the first stage of a ResNet-50 at the benchmark's batch: the largest tensors of a step
        _gn("gn_block_output", 400, 56, 56, 256, 32, "fp16", "relu", True, True),
        # stem output: few channels a group, many positions, a smooth activation
        _gn("gn_stem_silu", 128, 112, 112, 64, 32, "bf16", "silu", False, True),
        # a branch of a ShuffleNet: channels that fill no whole vectors, 29 of them a group, a clipped activation
        _gn("gn_odd_channels", 128, 28, 28, 116, 4, "fp16", "relu6", False, True),
        # the smallest training call: a short batch over few stored entries
        _distill("distill_short", 32, 1000, 5, "fp32", 1.0, False, False, True, True),
        # the benchmark's batch of image classes against stored top entries and their remainder
        _distill("distill_classes", 400, 1000, 32, "fp16", 4.0, True, False, True, True),
        # tokens over an odd vocabulary, some without entries, each with a weight of its own
        _distill("distill_tokens_odd", 2047, 50001, 50, "bf16", 1.0, False, True, False, True),
        # the largest: a long batch of tokens over a large vocabulary
        _distill("distill_tokens", 8192, 131072, 64, "bf16", 2.0, True, True, True, True),
        # a teacher that scores one token
        _top("top_one_token", 1, 131072, 64, "fp16", 2.0),
        # a teacher that labels a batch of images
        _top("top_classes", 400, 1000, 10, "fp32", 4.0),
        # a teacher that labels a batch of tokens
        _top("top_tokens", 4096, 131072, 64, "bf16", 2.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("group_norm", "group_norm", "distill", "distill", "top"))
    dtype = rng.choice(tuple(DTYPES))
    if op == "group_norm":
        groups = rng.choice((1, 2, 4, 8, 16, 32, 32))
        c = groups * _log_int(rng, 1, 64)
        h = _log_int(rng, 1, 112)
        w = h if rng.random() < 0.7 else _log_int(rng, 1, 112)
        n = _log_int(rng, 1, max(1, min(512, GN_MAX // (4 if dtype == "fp32" else 2) // (h * w * c))))
        return _gn(None, n, h, w, c, groups, dtype, rng.choice(("none", "relu", "relu6", "silu")), rng.random() < 0.5,
                   rng.random() < 0.8)
    classes = _log_int(rng, 16, 131072)
    most = (DISTILL_MAX if op == "distill" else TOP_MAX) // (4 if dtype == "fp32" else 2)
    rows = _log_int(rng, 1, max(1, min(8192, most // classes)))
    k = _log_int(rng, 1, min(classes - 1, 128))
    temperature = rng.choice((1.0, 2.0, 4.0, round(rng.uniform(0.5, 8.0), 2)))
    if op == "distill":
        return _distill(None, rows, classes, k, dtype, temperature, rng.random() < 0.5, rng.random() < 0.5,
                        rng.random() < 0.5, rng.random() < 0.8)
    return _top(None, rows, classes, k, dtype, temperature)


def _blocks(rows, classes):
    """Row ranges of about 64 million elements."""
    step = max(1, (1 << 26) // classes)
    return [(r, min(rows, r + step)) for r in range(0, rows, step)]


def _logits(rows, classes, dtype, gen):
    z = torch.empty((rows, classes), device="cuda", dtype=dtype)
    for a, b in _blocks(rows, classes):
        z[a:b] = torch.randn((b - a, classes), device="cuda", generator=gen) * 3.0
    return z


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    st = dict(case)
    if case["op"] == "group_norm":
        n, h, w, c = case["n"], case["h"], case["w"], case["c"]

        def rand(*shape):
            return torch.randn(shape, device="cuda", generator=gen)

        # a convolution's output: every channel has its own scale and offset
        x = (rand(n, h, w, c) * (0.5 + rand(c).abs()) + 0.5 * rand(c)).to(dtype)
        st["x"] = x.requires_grad_(case["train"])
        st["gamma"] = (1.0 + 0.2 * rand(c)).requires_grad_(case["train"])
        st["beta"] = (0.2 * rand(c)).requires_grad_(case["train"])
        st["res"] = rand(n, h, w, c).clamp_min_(0.0).to(dtype).requires_grad_(case["train"]) if case["residual"] else None
        st["dout"] = (0.1 * rand(n, h, w, c)).to(dtype) if case["train"] else None
        return st
    rows, classes, k, t = case["rows"], case["classes"], case["k"], case["temperature"]
    z = _logits(rows, classes, dtype, gen)
    st["z"] = z
    if case["op"] == "top":
        return st
    # the teacher agrees with the student in part
    values = torch.empty((rows, k), device="cuda", dtype=torch.float32)
    indices = torch.empty((rows, k), device="cuda", dtype=torch.int64)
    rest = torch.empty((rows,), device="cuda", dtype=torch.float32)
    for a, b in _blocks(rows, classes):
        teacher = z[a:b].float() * 0.8 + torch.randn((b - a, classes), device="cuda", generator=gen)
        values[a:b], indices[a:b] = torch.topk(teacher, k, dim=1)
        u = (teacher / t).scatter_(1, indices[a:b], -math.inf)
        rest[a:b] = torch.logsumexp(u, dim=1)
    if case["ragged"]:
        # rows of padding have no entries, others fewer than k
        length = torch.randint(1, k + 1, (rows, 1), device="cuda", generator=gen)
        length = torch.where(torch.rand((rows, 1), device="cuda", generator=gen) < 0.15, 0, length)
        indices.masked_fill_(torch.arange(k, device="cuda") >= length, -1)
    st["values"], st["indices"], st["rest"] = values.to(dtype), indices, rest if case["rest"] else None
    st["z"] = z.requires_grad_(case["train"])
    # what arrives from above: a weight for each row, and the loss scale that half precision is trained with
    scale = 1024.0 if case["dtype"] == "fp16" else 1.0
    if case["mean"]:
        st["weight"] = torch.tensor(scale * 2.0 ** round(math.log2(rows)) if scale != 1.0 else 1.0, device="cuda")
    else:
        st["weight"] = scale * torch.rand((rows,), device="cuda", generator=gen)
    return st


def run(state):
    if state["op"] == "group_norm":
        return _own_group_norm(state) if own else _plain_group_norm(state)
    if state["op"] == "distill":
        return _own_distill(state) if own else _plain_distill(state)
    return _own_top(state) if own else _plain_top(state)


def _own_group_norm(st):
    from pytorch_distributed_amd import ops
    act = {"none": False, "relu": True, "relu6": 6.0, "silu": "silu"}[st["act"]]
    out = ops.group_norm_act(st["x"], st["groups"], st["gamma"], st["beta"], st["res"], act, EPS)
    if not st["train"]:
        return {"out": out}
    wrt = [st["x"], st["gamma"], st["beta"]] + ([st["res"]] if st["res"] is not None else [])
    grads = torch.autograd.grad(out, wrt, st["dout"])
    r = {"out": out.detach(), "dx": grads[0], "dgamma": grads[1], "dbeta": grads[2]}
    if st["res"] is not None:
        r["dres"] = grads[3]
    return r


def _own_distill(st):
    from pytorch_distributed_amd import ops
    loss = ops.distill_loss(st["z"], st["values"], st["indices"], st["rest"], st["temperature"],
                            "mean" if st["mean"] else "none")
    if not st["train"]:
        return {"loss": loss}
    return {"loss": loss.detach(), "dz": torch.autograd.grad(loss, st["z"], st["weight"])[0]}


def _own_top(st):
    from pytorch_distributed_amd import ops
    values, indices, rest = ops.top_logits(st["z"], st["k"], st["temperature"])
    return {"values": values, "indices": indices, "rest": rest}


def _plain_group_norm(st):
    with torch.no_grad():
        x, res = st["x"], st["res"]
        n, h, w, c = x.shape
        groups = st["groups"]
        m = h * w * (c // groups)
        shape = (n, h * w, groups, c // groups)
        gamma, beta = st["gamma"].view(1, 1, groups, -1), st["beta"].view(1, 1, groups, -1)
        xv = x.reshape(shape)
        # the statistics are long sums, and z is compared with the borders of the activation: both in 64 bits
        mean = xv.sum((1, 3), keepdim=True, dtype=torch.float64) / m
        xh = xv.double() - mean
        rstd = ((xh * xh).sum((1, 3), keepdim=True) / m + EPS).rsqrt()
        xh = xh * rstd
        z = xh * gamma.double() + beta.double()
        if res is not None:
            z += res.reshape(shape)
        if st["act"] in ("relu", "relu6"):
            cap = 6.0 if st["act"] == "relu6" else math.inf
            slope = ((z > 0) & (z < cap)).float()
            z = z.float().clamp(0.0, cap)
            out = z
        else:
            z = z.float()
            slope = torch.ones_like(z)
            out = z
            if st["act"] == "silu":
                sig = 1.0 / (1.0 + torch.exp(-z))
                out = z * sig
                slope = sig * (1.0 + z * (1.0 - sig))
        out = out.to(x.dtype).view(n, h, w, c)
        if not st["train"]:
            return {"out": out}
        xh = xh.float()
        g = st["dout"].reshape(shape).float() * slope
        gx = g * xh
        r = {"out": out}
        r["dbeta"] = g.sum((0, 1), dtype=torch.float64).float().reshape(-1)
        r["dgamma"] = gx.sum((0, 1), dtype=torch.float64).float().reshape(-1)
        a = ((g.sum(1, keepdim=True) * gamma).sum(3, keepdim=True)) / m
        b = ((gx.sum(1, keepdim=True) * gamma).sum(3, keepdim=True)) / m
        r["dx"] = (rstd.float() * (g * gamma - a - xh * b)).to(x.dtype).view(n, h, w, c)
        if res is not None:
            r["dres"] = g.to(x.dtype).view(n, h, w, c)
        return r


def _plain_distill(st):
    with torch.no_grad():
        z, idx, t = st["z"], st["indices"], st["temperature"]
        rows, classes = z.shape
        valid = (idx >= 0) & (idx < classes)
        some = valid.any(1)
        slot = torch.where(valid, idx, classes)
        u = z.float() / t
        most = z.amax(1, keepdim=True)
        u -= most.float() / t
        e = u.exp()
        # the loss is a difference of nearly equal logarithms where student and teacher agree: the few numbers of a row that
        # it is made of are held in 64 bits
        total = e.sum(1, keepdim=True, dtype=torch.float64)
        logq = (z.gather(1, idx.clamp_min(0)).double() - most.double()) / t - total.log()
        logq = torch.where(valid, logq, 0.0)
        tau = torch.where(valid, st["values"].double() / t, -math.inf)
        bound = tau.amax(1, keepdim=True)
        if st["rest"] is not None:
            bound = torch.maximum(bound, st["rest"][:, None].double())
        bound = torch.where(some[:, None], bound, 0.0)
        mass = (tau - bound).exp()
        norm = mass.sum(1, keepdim=True)
        if st["rest"] is not None:
            rest = (st["rest"][:, None].double() - bound).exp()
            norm = norm + rest
        norm = torch.where(some[:, None], norm, 1.0)
        p = mass / norm
        logp = torch.where(p > 0, tau - bound - norm.log(), 0.0)
        loss = (p * (logp - logq)).sum(1)
        factor = torch.ones_like(loss, dtype=torch.float32)
        top = torch.zeros((rows, classes + 1), device=z.device, dtype=torch.bool).scatter_(1, slot, True)[:, :classes]
        if st["rest"] is not None:
            pr = rest[:, 0] / norm[:, 0]
            left = torch.where(top, 0.0, e).sum(1, dtype=torch.float64)
            qr = left / total[:, 0]
            loss = loss + pr * (pr.log() - left.log() + total[:, 0].log())
            factor = (1.0 - pr / qr).float()
        loss = torch.where(some, loss, 0.0) * (t * t)
        r = {"loss": (loss.mean() if st["mean"] else loss).float()}
        if not st["train"]:
            return r
        weight = (st["weight"] / rows).expand(rows) if st["mean"] else st["weight"]
        weight = weight * t
        weight = torch.where(some, weight, 0.0)[:, None]
        q = e / total.float()
        dz = torch.where(top, q, q * factor[:, None])
        dz.scatter_add_(1, torch.where(valid, idx, 0), torch.where(valid, -p, 0.0).float())
        r["dz"] = (dz * weight).to(z.dtype)
        return r


def _plain_top(st):
    z, k, t = st["z"], st["k"], st["temperature"]
    classes = z.shape[1]
    # one whole number orders by value first, then by the lower class
    bits = (z.float() + 0.0).view(torch.int32)
    key = bits ^ ((bits >> 31) & 0x7fffffff)
    key = torch.where(torch.isnan(z), 0x7fffffff, key).long()
    key = (key << 32) + (classes - 1 - torch.arange(classes, device=z.device))
    best = torch.topk(key, k, dim=1).values
    indices = classes - 1 - (best & 0xffffffff)
    u = (z.float() / t).scatter_(1, indices, -math.inf)
    m = u.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    rest = ((u - m).exp().sum(1, dtype=torch.float64).log() + m[:, 0]).float()
    return {"values": z.gather(1, indices), "indices": indices, "rest": rest}


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "group_norm":
        elements = case["n"] * case["h"] * case["w"] * case["c"]
        tensors = 2 + case["residual"] + (2 + case["residual"] if case["train"] else 0)
        return {"bytes": elements * size * tensors + 4 * case["c"] * (4 if case["train"] else 2),
                "flops": elements * (35 if case["train"] else 10)}
    rows, classes, k = case["rows"], case["classes"], case["k"]
    if case["op"] == "distill":
        return {"bytes": rows * classes * size * (2 if case["train"] else 1) + rows * (k * (size + 8) + 8),
                "flops": rows * classes * (8 if case["train"] else 4)}
    return {"bytes": rows * classes * size + rows * (k * (size + 8) + 4), "flops": rows * classes * 5}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "group_norm":
        return _exact_group_norm(st)
    if case["op"] == "distill":
        return _exact_distill(st)
    values, indices, rest = [], [], []
    for a, b in _blocks(case["rows"], case["classes"]):
        z = st["z"][a:b].double()
        s, i = torch.sort(z, dim=1, descending=True, stable=True)
        values.append(s[:, :case["k"]].clone())
        indices.append(i[:, :case["k"]].clone())
        rest.append(torch.logsumexp(s[:, case["k"]:] / case["temperature"], dim=1))
    return {"values": torch.cat(values), "indices": torch.cat(indices), "rest": torch.cat(rest)}


def _exact_group_norm(st):
    """Channels first, a block of samples at a time, the gradients by differentiation."""
    n, h, w, c = st["x"].shape
    groups = st["groups"]
    gamma = st["gamma"].detach().double().requires_grad_(st["train"])
    beta = st["beta"].detach().double().requires_grad_(st["train"])
    parts = {"out": [], "dx": [], "dres": []}
    dgamma, dbeta = torch.zeros_like(gamma), torch.zeros_like(beta)
    step = max(1, (1 << 25) // (h * w * c))
    for a in range(0, n, step):
        def part(t):
            return t[a:a + step].detach().double().permute(0, 3, 1, 2)

        x = part(st["x"]).requires_grad_(st["train"])
        res = part(st["res"]).requires_grad_(st["train"]) if st["res"] is not None else None
        flat = x.reshape(x.shape[0], groups, -1)
        var, mean = torch.var_mean(flat, dim=2, unbiased=False, keepdim=True)
        y = ((flat - mean) / torch.sqrt(var + EPS)).reshape(x.shape)
        y = y * gamma.view(1, c, 1, 1) + beta.view(1, c, 1, 1)
        y = y if res is None else y + res
        if st["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif st["act"] != "none":
            y = y.clamp(0.0, 6.0 if st["act"] == "relu6" else math.inf)
        parts["out"].append(y.detach().permute(0, 2, 3, 1))
        if not st["train"]:
            continue
        wrt = [x, gamma, beta] + ([res] if res is not None else [])
        grads = torch.autograd.grad(y, wrt, part(st["dout"]))
        parts["dx"].append(grads[0].permute(0, 2, 3, 1))
        dgamma += grads[1]
        dbeta += grads[2]
        if res is not None:
            parts["dres"].append(grads[3].permute(0, 2, 3, 1))
    r = {"out": torch.cat(parts["out"])}
    if st["train"]:
        r.update(dx=torch.cat(parts["dx"]), dgamma=dgamma.detach(), dbeta=dbeta.detach())
        if st["res"] is not None:
            r["dres"] = torch.cat(parts["dres"])
    return r


def _exact_distill(st):
    """Kullback-Leibler divergence between the two distributions over the entries' classes (and the remainder), a block of
    rows at a time, the gradient by differentiation."""
    t = st["temperature"]
    rows, classes = st["z"].shape
    losses, grads = [], []
    for a, b in _blocks(rows, classes * 4):
        z = st["z"][a:b].detach().double().requires_grad_(st["train"])
        idx = st["indices"][a:b]
        valid = (idx >= 0) & (idx < classes)
        some = valid.any(1, keepdim=True)
        logq = torch.log_softmax(z / t, dim=1)
        student = logq.gather(1, idx.clamp_min(0))
        teacher = (st["values"][a:b].double() / t).masked_fill(~valid, -math.inf)
        if st["rest"] is not None:
            taken = torch.zeros((b - a, classes + 1), device=z.device, dtype=torch.bool)
            taken = taken.scatter(1, torch.where(valid, idx, classes), True)[:, :classes]
            student = torch.cat([student, torch.logsumexp(logq.masked_fill(taken, -math.inf), 1, keepdim=True)], 1)
            teacher = torch.cat([teacher, st["rest"][a:b, None].double()], 1)
        teacher = torch.log_softmax(torch.where(some, teacher, 0.0), dim=1)
        p = teacher.exp()
        terms = torch.where(p > 0, p * (torch.where(p > 0, teacher, 0.0) - student), 0.0)
        loss = torch.where(some[:, 0], terms.sum(1), 0.0) * t * t
        losses.append(loss.detach())
        if st["train"]:
            weight = st["weight"].double()
            weight = (weight / rows).expand(b - a) if st["mean"] else weight[a:b]
            grads.append(torch.autograd.grad(loss, z, weight)[0])
    loss = torch.cat(losses)
    r = {"loss": loss.mean() if st["mean"] else loss}
    if st["train"]:
        r["dz"] = torch.cat(grads)
    return r
