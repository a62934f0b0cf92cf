"""The operators of a training step around the compressed gradient exchange, as measurable cases.

A case is a dict of plain values: ``op`` names the operator, ``pass`` what one call does (``forward``, or
``train``: forward and gradients), the other keys its sizes and types.

  layer_norm       rows normalised, scaled and shifted; gradients of the rows, the scale and the shift
  linear           activation(x W^T + b) + residual; gradients of x, W and b
  token_logprobs   log probability of a given token per row of logits, the row's entropy and its most likely
                   tokens; gradient of the logits for both numbers
  orthogonalize    the Newton-Schulz iteration that makes a momentum matrix nearly orthogonal

Where ``own`` is false the operators are computed from elementary torch operations in 32 bits.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-5
NS = (3.4445, -4.7750, 2.0315)
NS_EPS = 1e-7
NS_STEPS = 5
IGNORED = -100


def listed():
    return [
        # the last norm of the GPT-2-shaped model for one new token: nothing but latency
        {"name": "norm_one_token", "op": "layer_norm", "pass": "forward", "rows": 1, "width": 768, "type": "fp32", "out": "bf16"},
        # one norm of the trainer's model at batch 8, sequence 1024: fp32 residual stream in, bf16 out
        {"name": "norm_train_8192x768", "op": "layer_norm", "pass": "train", "rows": 8192, "width": 768, "type": "fp32", "out": "bf16"},
        # a wide model in bf16 throughout, with a width that no vector load divides
        {"name": "norm_train_6001x5003", "op": "layer_norm", "pass": "train", "rows": 6001, "width": 5003, "type": "bf16", "out": "bf16"},
        # query, key and value projection of one new token
        {"name": "linear_one_token", "op": "linear", "pass": "forward", "rows": 1, "inner": 768, "width": 2304, "type": "bf16", "activation": "none", "bias": True, "residual": "none"},
        # the same projection in a training step
        {"name": "linear_train_qkv", "op": "linear", "pass": "train", "rows": 8192, "inner": 768, "width": 2304, "type": "bf16", "activation": "none", "bias": True, "residual": "none"},
        # first half of a feed-forward block with its activation, over packed sequences of a ragged total length
        {"name": "linear_train_gelu_ragged", "op": "linear", "pass": "train", "rows": 4109, "inner": 1600, "width": 6400, "type": "fp16", "activation": "gelu_tanh", "bias": True, "residual": "none"},
        # second half of a large feed-forward block, added to the fp32 residual stream (a prompt of 8192 tokens)
        {"name": "linear_down_residual", "op": "linear", "pass": "forward", "rows": 8192, "inner": 8192, "width": 4096, "type": "bf16", "activation": "none", "bias": True, "residual": "fp32"},
        # one new token over the model's vocabulary, with the five most likely tokens
        {"name": "logprobs_one_token", "op": "token_logprobs", "pass": "forward", "rows": 1, "vocab": 50257, "type": "bf16", "top": 5, "masked": False},
        # the loss of the trainer's model: all rows of a batch, with the gradient of the logits
        {"name": "logprobs_train_8192", "op": "token_logprobs", "pass": "train", "rows": 8192, "vocab": 50257, "type": "bf16", "top": 0, "masked": False},
        # the small model's two layers
        {"name": "muon_2x192x64", "op": "orthogonalize", "pass": "forward", "batch": 2, "height": 192, "width": 64, "type": "fp32"},
        # query, key and value weights of all twelve layers of the trainer's model at once
        {"name": "muon_12x2304x768", "op": "orthogonalize", "pass": "forward", "batch": 12, "height": 2304, "width": 768, "type": "fp32"},
        # one matrix of a large model
        {"name": "muon_4096x8192", "op": "orthogonalize", "pass": "forward", "batch": 1, "height": 4096, "width": 8192, "type": "bf16"},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm; one in three is rounded to a multiple of 8."""
    v = min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return max(8, v // 8 * 8) if v >= 8 and rng.random() < 0.34 else v


def draw(rng):
    op = rng.choice(["layer_norm", "linear", "linear", "token_logprobs", "orthogonalize"])
    if op == "layer_norm":
        kind = rng.choice(["fp32", "bf16", "fp16"])
        case = {"op": op, "pass": rng.choice(["forward", "train", "train"]), "rows": _spread(rng, 1, 16384), "width": _spread(rng, 32, 8192),
                "type": kind, "out": rng.choice(["bf16", "fp32"]) if kind == "fp32" else kind}
        case["rows"] = min(case["rows"], max(1, 6001 * 5003 // case["width"]))
    elif op == "linear":
        case = {"op": op, "pass": rng.choice(["forward", "train"]), "rows": _spread(rng, 1, 16384), "inner": _spread(rng, 64, 8192), "width": _spread(rng, 64, 8192),
                "type": rng.choice(["bf16", "bf16", "fp16"]), "activation": rng.choice(["none", "gelu_tanh", "relu", "silu"]), "bias": rng.random() < 0.7}
        case["residual"] = rng.choice(["none", "fp32", "same"]) if case["activation"] == "none" else "none"
        most = 8192 * 8192 * 4096 // (3 if case["pass"] == "train" else 1)
        case["rows"] = min(case["rows"], max(1, most // (case["inner"] * case["width"])))
    elif op == "token_logprobs":
        case = {"op": op, "pass": rng.choice(["forward", "train"]), "rows": _spread(rng, 1, 16384), "vocab": _spread(rng, 257, 131072),
                "type": rng.choice(["bf16", "fp32", "fp16"]), "masked": rng.random() < 0.5}
        case["rows"] = min(case["rows"], max(1, 8192 * 50257 // (2 * case["vocab"])))
        case["top"] = rng.choice([0, 1, 5, 20]) if case["pass"] == "forward" else 0
    else:
        case = {"op": op, "pass": "forward", "batch": _spread(rng, 1, 16), "height": _spread(rng, 32, 4096), "width": _spread(rng, 32, 4096), "type": rng.choice(["fp32", "bf16"])}
        case["batch"] = min(case["batch"], max(1, 4096 * 8192 // (case["height"] * case["width"])))
    return case


def _random(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    g = _random(seed)
    t = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    s = dict(case)
    if case["op"] == "layer_norm":
        d = case["width"]
        # activations have an offset and a few channels that are much larger than the others
        scale = torch.where(torch.rand(d, device="cuda", generator=g) < 0.01, 20.0, 1.0)
        s["x"] = (normal(case["rows"], d) * scale + 0.3 * normal(d)).to(t)
        s["weight"], s["bias"] = 1 + 0.2 * normal(d), 0.1 * normal(d)
        s["grad"] = normal(case["rows"], d).to(TYPES[case["out"]])
    elif case["op"] == "linear":
        m, k, n = case["rows"], case["inner"], case["width"]
        s["x"] = normal(m, k).to(t)
        s["weight"] = (normal(n, k) / math.sqrt(k)).to(t)
        s["bias"] = (0.2 * normal(n)).to(t) if case["bias"] else None
        s["residual"] = None if case["residual"] == "none" else normal(m, n).to(TYPES["fp32"] if case["residual"] == "fp32" else t)
        s["grad"] = normal(m, n).to(t if s["residual"] is None else s["residual"].dtype) if case["pass"] == "train" else None
    elif case["op"] == "token_logprobs":
        m, v = case["rows"], case["vocab"]
        logits = normal(m, v).mul_(2.5)
        tokens = torch.randint(0, v, (m,), device="cuda", generator=g)
        sure = torch.rand(m, device="cuda", generator=g) < 0.5  # rows whose token the model has learnt
        logits[torch.arange(m, device="cuda"), tokens] += torch.where(sure, 12.0, 0.0)
        if case["masked"]:  # tokens that a grammar or a padded vocabulary forbids
            banned = torch.rand(v, device="cuda", generator=g) < 0.2
            logits[:, banned] = -math.inf
            logits[torch.arange(m, device="cuda"), tokens] = 3.0
        padded = torch.rand(m, device="cuda", generator=g) < 0.03
        padded[0] = False
        s["logits"], s["tokens"] = logits.to(t), torch.where(padded, IGNORED, tokens)
        s["grad"], s["grad_entropy"] = normal(m), -0.01 * torch.ones(m, device="cuda")
    else:
        b, m, n = case["batch"], case["height"], case["width"]
        # momentum of a weight: a falling spectrum over a floor of noise
        r = min(m, n, 64)
        falling = 1 / torch.arange(1, r + 1, device="cuda")
        s["update"] = (1e-3 * ((normal(b, m, r) * falling) @ normal(b, r, n) + 0.05 * normal(b, m, n))).to(t)
    return s


def _activation(z, kind):
    """The activation and its derivative, elementwise."""
    if kind == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if kind == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p * (1 + z * (1 - p))
    if kind == "relu":
        return torch.clamp(z, min=0), (z > 0).to(z.dtype)
    return z, None


def _layer_norm(s):
    x, w, out = s["x"].float(), s["weight"], TYPES[s["out"]]
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
    h = c * rstd
    y = (h * w + s["bias"]).to(out)
    if s["pass"] == "forward":
        return {"y": y}
    g = s["grad"].float()
    gw = g * w
    dx = rstd * (gw - gw.mean(1, keepdim=True) - h * (gw * h).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dweight": (g * h).sum(0), "dbias": g.sum(0)}


def _linear(s):
    t = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y, slope = _activation(z, s["activation"])
    y = y.to(t) if s["residual"] is None else (y + s["residual"].float()).to(s["residual"].dtype)
    if s["grad"] is None:
        return {"y": y}
    g = s["grad"].float()
    if slope is not None:
        g = g * slope
    grads = {"y": y, "dx": (g @ w).to(t), "dweight": (g.t() @ x).to(t)}
    if s["bias"] is not None:
        grads["dbias"] = g.sum(0).to(s["bias"].dtype)
    return grads


def _token_logprobs(s):
    x = s["logits"].float()
    kept = s["tokens"] != IGNORED
    at = torch.where(kept, s["tokens"], 0)[:, None]
    top = x.max(1, keepdim=True).values
    logp = x - top
    logp = logp - torch.log(torch.exp(logp).sum(1, keepdim=True))
    p = torch.exp(logp)
    out = {"logprobs": torch.where(kept, logp.gather(1, at)[:, 0], 0.0),
           "entropy": torch.where(kept, -torch.where(p > 0, p * logp, 0.0).sum(1), 0.0)}
    if s["top"]:
        # largest first, the lowest index first among equals: value and index in one whole number
        bits = (x + 0.0).view(torch.int32)
        bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        key = (bits << 32) - torch.arange(x.shape[1], device=x.device)
        best = key.topk(s["top"], 1).values
        i = (-best) & 0xFFFFFFFF
        out["top_tokens"] = torch.where(kept[:, None], i, -1)
        out["top_logprobs"] = torch.where(kept[:, None], logp.gather(1, i), 0.0)
    if s["pass"] == "train":
        a = torch.where(kept, s["grad"], 0.0)[:, None]
        b = torch.where(kept, s["grad_entropy"], 0.0)[:, None]
        d = -a * p - b * torch.where(p > 0, p * (logp + out["entropy"][:, None]), 0.0)
        d.scatter_add_(1, at, a)
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


def _orthogonalize(s):
    a, b, c = NS
    x = s["update"].float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.mT
    x = x / (torch.sqrt((x * x).sum((1, 2), keepdim=True)) + NS_EPS)
    for _ in range(NS_STEPS):
        q = x @ x.mT
        x = a * x + (b * q + c * (q @ q)) @ x
    return {"update": (x.mT if tall else x).to(torch.bfloat16)}


def _own(s):
    from tirocinio_triennale_b200 import ops

    if s["op"] == "layer_norm":
        out = TYPES[s["out"]]
        if s["pass"] == "forward":
            return {"y": ops.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, out_dtype=out)}
        x, w, b = (s[k].detach().requires_grad_() for k in ("x", "weight", "bias"))
        y = ops.layer_norm(x, w, b, eps=EPS, out_dtype=out)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["grad"])
        return {"y": y, "dx": dx, "dweight": dw, "dbias": db}
    if s["op"] == "linear":
        kind = None if s["activation"] == "none" else s["activation"]
        if s["grad"] is None:
            return {"y": ops.linear(s["x"], s["weight"], s["bias"], activation=kind, residual=s["residual"])}
        leaves = [s[k].detach().requires_grad_() for k in ("x", "weight", "bias") if s[k] is not None]
        y = ops.linear(leaves[0], leaves[1], leaves[2] if len(leaves) == 3 else None, activation=kind, residual=s["residual"])
        grads = torch.autograd.grad(y, leaves, s["grad"])
        return {"y": y, **dict(zip(("dx", "dweight", "dbias"), grads))}
    if s["op"] == "token_logprobs":
        if s["pass"] == "forward":
            r = ops.token_logprobs(s["logits"], s["tokens"], top=s["top"], ignore_index=IGNORED)
            out = {"logprobs": r.logprobs, "entropy": r.entropy}
            if s["top"]:
                out.update(top_tokens=r.top_tokens, top_logprobs=r.top_logprobs)
            return out
        x = s["logits"].detach().requires_grad_()
        r = ops.token_logprobs(x, s["tokens"], ignore_index=IGNORED)
        (d,) = torch.autograd.grad((r.logprobs, r.entropy), (x,), (s["grad"], s["grad_entropy"]))
        return {"logprobs": r.logprobs, "entropy": r.entropy, "dlogits": d}
    return {"update": ops.orthogonalize(s["update"], steps=NS_STEPS, coefficients=NS, eps=NS_EPS)}


def run(state):
    if own:
        return _own(state)
    return {"layer_norm": _layer_norm, "linear": _linear, "token_logprobs": _token_logprobs, "orthogonalize": _orthogonalize}[state["op"]](state)


def work(case):
    e = SIZE[case["type"]]
    train = case["pass"] == "train"
    if case["op"] == "layer_norm":
        n, o, d = case["rows"] * case["width"], SIZE[case["out"]], case["width"]
        # forward: x, scale and shift in, y out; gradients: x is there already, dy in, dx and two rows of sums out
        return {"bytes": n * (e + o) + 8 * d + (n * (o + e) + 8 * d if train else 0), "flops": n * (8 + (14 if train else 0))}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["inner"], case["width"]
        o = 4 if case["residual"] == "fp32" else e
        nbytes = e * (m * k + n * k) + o * m * n + (e * n if case["bias"] else 0) + (0 if case["residual"] == "none" else o * m * n)
        if train:
            nbytes += o * m * n + e * (m * k + n * k) + (e * n if case["bias"] else 0)
        return {"bytes": nbytes, "flops": 2 * m * k * n * (3 if train else 1)}
    if case["op"] == "token_logprobs":
        m, v = case["rows"], case["vocab"]
        return {"bytes": m * v * e * (2 if train else 1) + m * (16 + 12 * case["top"] + (8 if train else 0)), "flops": m * v * (6 + (8 if train else 0))}
    b, m, n = case["batch"], min(case["height"], case["width"]), max(case["height"], case["width"])
    # two of the three products of a step give a symmetric matrix, of which one half is enough
    return {"bytes": b * m * n * (e + 2), "flops": NS_STEPS * b * (2 * m * m * n + m * m * n + m * m * m)}


def exact(case, seed):
    """The operators' definitions in 64 bits, gradients by their formulas over whole rows."""
    s = prepare(case, seed)
    if case["op"] == "layer_norm":
        x, w, n = s["x"].double(), s["weight"].double(), case["width"]
        mean = x.sum(1) / n
        var = ((x - mean[:, None]) ** 2).sum(1) / n
        h = (x - mean[:, None]) / (var + EPS).sqrt()[:, None]
        out = {"y": torch.addcmul(s["bias"].double(), h, w)}
        if case["pass"] == "train":
            g = s["grad"].double()
            # dx = (I - 11'/n - hh'/n) (g w) / sigma
            gw = g * w
            along, flat = torch.einsum("ij,ij->i", gw, h) / n, gw.sum(1) / n
            out["dx"] = (gw - flat[:, None] - h * along[:, None]) / (var + EPS).sqrt()[:, None]
            out["dweight"], out["dbias"] = torch.einsum("ij,ij->j", g, h), torch.einsum("ij->j", g)
        return out
    if case["op"] == "linear":
        x, w = s["x"].double().requires_grad_(), s["weight"].double().requires_grad_()
        leaves = [x, w]
        y = torch.einsum("mk,nk->mn", x, w)
        if s["bias"] is not None:
            leaves.append(s["bias"].double().requires_grad_())
            y = y + leaves[2]
        if case["activation"] == "gelu_tanh":
            u = 2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)
            y = y * torch.sigmoid(u)  # (1 + tanh(u / 2)) / 2
        elif case["activation"] == "silu":
            y = y * torch.sigmoid(y)
        elif case["activation"] == "relu":
            y = torch.where(y > 0, y, torch.zeros_like(y))
        if s["residual"] is not None:
            y = y + s["residual"].double()
        out = {"y": y.detach()}
        if s["grad"] is not None:
            out.update(zip(("dx", "dweight", "dbias"), torch.autograd.grad(y, leaves, s["grad"].double())))
        return out
    if case["op"] == "token_logprobs":
        x = s["logits"].double()
        m = torch.arange(x.shape[0], device=x.device)
        lse = torch.logsumexp(x, 1)
        kept = s["tokens"] >= 0
        at = s["tokens"].clamp(min=0)
        p = torch.exp(x - lse[:, None])
        mean = torch.where(p > 0, p * x, 0.0).sum(1)
        out = {"logprobs": torch.where(kept, x[m, at] - lse, 0.0), "entropy": torch.where(kept, lse - mean, 0.0)}
        if case["top"]:
            value, i = torch.sort(s["logits"], dim=1, descending=True, stable=True)
            i, value = i[:, :case["top"]], value[:, :case["top"]].double()
            out["top_tokens"] = torch.where(kept[:, None], i, -1)
            out["top_logprobs"] = torch.where(kept[:, None], value - lse[:, None], 0.0)
        if case["pass"] == "train":
            a, b = s["grad"].double() * kept, s["grad_entropy"].double() * kept
            # d entropy / d x_j = p_j (mean - x_j)
            d = b[:, None] * torch.where(p > 0, p * (mean[:, None] - x), 0.0) - a[:, None] * p
            d[m, at] += a
            out["dlogits"] = d
        return out
    a, b, c = NS
    x = s["update"].double()
    x = x / (torch.linalg.matrix_norm(x)[:, None, None] + NS_EPS)
    right = x.shape[1] >= x.shape[2]  # the smaller of the two Gram matrices
    one = torch.eye(min(x.shape[1:]), device=x.device, dtype=x.dtype)
    for _ in range(NS_STEPS):
        q = x.mT @ x if right else x @ x.mT
        poly = a * one + q @ (b * one + c * q)
        x = x @ poly if right else poly @ x
    return {"update": x}
