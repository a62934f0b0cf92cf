"""More operators of a training step, as measurable cases: attention, the loss from hidden rows, the optimiser's step.

A case is a dict of plain values: ``op`` names the operator, ``pass`` what one call does (``forward``, or
``train``: forward and gradients), the other keys its sizes and types.

  attention             causal attention with a sliding window and first tokens that stay visible (sinks), several
                        query heads to a key and value head; gradients of queries, keys and values
  linear_cross_entropy  cross entropy of x W^T over a vocabulary; gradients of x and W
  adamw                 one AdamW step over many tensors, moments in 32 bits or in 8 bits with a scale a block

Where ``own`` is false the operators are computed from elementary torch operations in 32 bits.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
IGNORED = -100
BETAS, EPS, DECAY, LR = (0.9, 0.999), 1e-8, 0.01, 3e-4
BLOCK = 256  # values that share a scale


def listed():
    return [
        # one new token behind a context as long as the model's: nothing but latency
        {"name": "attention_one_token", "op": "attention", "pass": "forward", "batch": 1, "heads": 12, "kv_heads": 12, "queries": 1, "keys": 1024, "head": 64, "type": "bf16", "window": 0, "sinks": 0},
        # one new token of each of several long texts, of which a window and the first tokens are seen
        {"name": "attention_tokens_32k", "op": "attention", "pass": "forward", "batch": 16, "heads": 16, "kv_heads": 4, "queries": 1, "keys": 32768, "head": 128, "type": "bf16", "window": 8192, "sinks": 4},
        # one layer of the trainer's model at batch 8, sequence 1024
        {"name": "attention_train_8x1024", "op": "attention", "pass": "train", "batch": 8, "heads": 12, "kv_heads": 12, "queries": 1024, "keys": 1024, "head": 64, "type": "bf16", "window": 0, "sinks": 0},
        # sequences of a ragged length with a short window, heads that share keys, a head that fills no tile
        {"name": "attention_train_ragged", "op": "attention", "pass": "train", "batch": 3, "heads": 10, "kv_heads": 5, "queries": 1777, "keys": 1777, "head": 80, "type": "fp16", "window": 300, "sinks": 5},
        # a long text in one piece
        {"name": "attention_train_8192", "op": "attention", "pass": "train", "batch": 1, "heads": 16, "kv_heads": 4, "queries": 8192, "keys": 8192, "head": 128, "type": "bf16", "window": 4096, "sinks": 4},
        # the loss of one token, from the last hidden row of the model
        {"name": "loss_one_token", "op": "linear_cross_entropy", "pass": "forward", "rows": 1, "inner": 768, "vocab": 50257, "type": "bf16", "reduction": "none"},
        # the trainer's loss: all rows of a batch, with the gradients of the last hidden rows and the tied embedding
        {"name": "loss_train_8192", "op": "linear_cross_entropy", "pass": "train", "rows": 8192, "inner": 768, "vocab": 50257, "type": "bf16", "reduction": "mean"},
        # a wider model over packed sequences of a ragged total length, each row with a weight of its own
        {"name": "loss_train_ragged", "op": "linear_cross_entropy", "pass": "train", "rows": 4109, "inner": 1600, "vocab": 32003, "type": "fp16", "reduction": "none"},
        # one bias: nothing but latency
        {"name": "adamw_one_bias", "op": "adamw", "pass": "step", "shapes": "768", "copies": 1, "shift": 0, "type": "fp32", "grad": "fp32", "bits": 32, "step": 1},
        # all parameters of the trainer's model (embeddings, twelve blocks, last norm) with their gradients in buckets
        {"name": "adamw_gpt2_small", "op": "adamw", "pass": "step", "shapes": MODEL, "copies": 1, "shift": 0, "type": "fp32", "grad": "fp32", "bits": 32, "step": 1000},
        # the same with the moments in 8 bits
        {"name": "adamw_gpt2_small_8bit", "op": "adamw", "pass": "step", "shapes": MODEL, "copies": 1, "shift": 0, "type": "fp32", "grad": "fp32", "bits": 8, "step": 1000},
        # bf16 weights of odd sizes that begin anywhere in their buffer
        {"name": "adamw_ragged_bf16", "op": "adamw", "pass": "step", "shapes": "5003x1201,5003,77x31,1,1201x333,255,257", "copies": 7, "shift": 1, "type": "bf16", "grad": "bf16", "bits": 8, "step": 20},
    ]


def _model():
    d, layers, vocab, seq = 768, 12, 50257, 1024
    block = "%d,%d,%dx%d,%d,%dx%d,%d,%d,%d,%dx%d,%d,%dx%d,%d" % (d, d, 3 * d, d, 3 * d, d, d, d, d, d, 4 * d, d, 4 * d, d, 4 * d, d)
    return ",".join(["%dx%d,%dx%d" % (vocab, d, seq, d)] + [block] * layers + ["%d,%d" % (d, d)])


MODEL = _model()


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm; one in three is rounded to a multiple of 8."""
    v = min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return max(8, v // 8 * 8) if v >= 8 and rng.random() < 0.34 else v


def draw(rng):
    op = rng.choice(["attention", "attention", "linear_cross_entropy", "adamw"])
    if op == "attention":
        most = 12 * 8192 * 8192  # scores: those that the largest case sees
        kv, group = rng.choice([1, 2, 3, 4, 8, 12]), rng.choice([1, 1, 2, 4, 5])
        case = {"op": op, "pass": rng.choice(["forward", "train"]), "batch": _spread(rng, 1, 16), "heads": kv * group, "kv_heads": kv}
        keys = _spread(rng, 1, 8192)
        if rng.random() < 0.6:  # whole sequences
            case["queries"] = keys = min(keys, math.isqrt(most // case["heads"]))
        elif rng.random() < 0.7:  # new tokens
            case["queries"], keys = _spread(rng, 1, 16), _spread(rng, 1, 32768)
        else:  # a chunk
            case["queries"] = _spread(rng, 1, 1024)
        case |= {"keys": keys, "head": rng.choice([16, 32, 64, 64, 72, 80, 96, 128, 128]), "type": rng.choice(["bf16", "bf16", "fp16"]),
                 "window": rng.choice([0, 1, _spread(rng, 2, 8192), _spread(rng, 2, 8192)])}
        case["sinks"] = rng.choice([0, 1, 4, 130]) if case["window"] else 0
        case["batch"] = max(1, min(case["batch"], most // (case["heads"] * case["queries"] * keys), 16 * 4 * 32768 * 128 // (kv * keys * case["head"])))
    elif op == "linear_cross_entropy":
        case = {"op": op, "pass": rng.choice(["forward", "train"]), "rows": _spread(rng, 1, 16384), "inner": _spread(rng, 64, 4096), "vocab": _spread(rng, 257, 131072),
                "type": rng.choice(["bf16", "bf16", "fp16"]), "reduction": rng.choice(["none", "sum", "mean"])}
        case["rows"] = min(case["rows"], max(1, 8192 * 768 * 50257 // (case["inner"] * case["vocab"])), max(1, 8192 * 50257 // case["vocab"]))
    else:
        count, room, shapes = _spread(rng, 1, 60), 1 << 26, []
        for _ in range(count):
            n = min(_spread(rng, 1, 1 << 24), room)
            if n < 1:
                break
            room -= n
            h = _spread(rng, 1, n) if rng.random() < 0.5 else 1
            shapes.append("%dx%d" % (h, n // h) if h > 1 else str(n))
        kind = rng.choice(["fp32", "fp32", "bf16", "fp16"])
        case = {"op": op, "pass": "step", "shapes": ",".join(shapes), "copies": 1, "shift": rng.choice([0, 0, 1, 3]), "type": kind,
                "grad": rng.choice(["fp32", "bf16"]) if kind == "fp32" else kind, "bits": rng.choice([32, 8]), "step": _spread(rng, 1, 100000)}
    return case


def _random(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _shapes(case):
    return [tuple(int(n) for n in part.split("x")) for part in case["shapes"].split(",")] * case["copies"]


def _places(case):
    """Where each tensor begins in a buffer of parameters or gradients, and in one of moments (whole blocks); the buffers' lengths."""
    at, first, length, held = [], [], case["shift"], 0
    for shape in _shapes(case):
        n = math.prod(shape)
        at.append(length)
        first.append(held)
        length += n + case["shift"]
        held += -(-n // BLOCK) * BLOCK
    return at, first, length, held


def prepare(case, seed):
    g = _random(seed)
    t = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    s = dict(case)
    if case["op"] == "attention":
        b, d = case["batch"], case["head"]
        # as a projection leaves them: (batch, position, head, value); keys have an offset of their own, the first one draws attention
        k = normal(b, case["keys"], case["kv_heads"], d) + 0.5 * normal(1, 1, case["kv_heads"], d)
        k[:, 0] *= 2
        s["q"] = (1.5 * normal(b, case["queries"], case["heads"], d)).to(t).transpose(1, 2)
        s["k"], s["v"] = k.to(t).transpose(1, 2), normal(b, case["keys"], case["kv_heads"], d).to(t).transpose(1, 2)
        s["grad"] = normal(b, case["queries"], case["heads"], d).to(t).transpose(1, 2) if case["pass"] == "train" else None
    elif case["op"] == "linear_cross_entropy":
        m, k, n = case["rows"], case["inner"], case["vocab"]
        w = normal(n, k) * (2 / math.sqrt(k))
        targets = torch.randint(0, n, (m,), device="cuda", generator=g)
        sure = torch.rand(m, 1, device="cuda", generator=g) < 0.5  # rows whose token the model has learnt
        s["x"] = (normal(m, k) + torch.where(sure, 2.0, 0.0) * w[targets]).to(t)
        s["weight"] = w.to(t)
        padded = torch.rand(m, device="cuda", generator=g) < 0.03
        padded[0] = False
        s["targets"] = torch.where(padded, IGNORED, targets)
        # weights of the rows, or a loss scale as 16 bits need it
        s["grad"] = normal(m) if case["reduction"] == "none" else torch.tensor(4096.0 if case["type"] == "fp16" else 1.0, device="cuda")
    else:
        at, first, length, held = _places(case)
        s["param"] = (0.05 * normal(length)).to(t)
        s["gradient"] = (1e-3 * normal(length) * torch.exp(2 * normal(length))).to(TYPES[case["grad"]])
        if case["bits"] == 32:
            s["exp_avg"] = 3e-4 * normal(held)
            s["exp_avg_sq"] = (1e-3 * torch.exp(normal(held))).square()
            s["scales"] = None
        else:
            blocks = held // BLOCK
            code = torch.randint(0, 256, (held, 2), device="cuda", generator=g, dtype=torch.uint8)
            s["exp_avg"], s["exp_avg_sq"] = code[:, 0].contiguous(), code[:, 1].contiguous()
            s["scales"] = 1e-3 * torch.exp(normal(blocks, 2))
        shapes = _shapes(case)
        s["params"] = [s["param"][a:a + math.prod(n)].view(n) for a, n in zip(at, shapes)]
        s["grads"] = [s["gradient"][a:a + math.prod(n)].view(n) for a, n in zip(at, shapes)]
        s["exp_avgs"] = [s["exp_avg"][a:a + math.prod(n)].view(n) for a, n in zip(first, shapes)]
        s["exp_avg_sqs"] = [s["exp_avg_sq"][a:a + math.prod(n)].view(n) for a, n in zip(first, shapes)]
        s["block_scales"] = None if s["scales"] is None else [s["scales"][a // BLOCK:-(-(a + math.prod(n)) // BLOCK)] for a, n in zip(first, shapes)]
        s["seed"] = seed & 0xFFFF
    return s


def _seen(s, device):
    """Which keys each query sees: those up to its own position, within the window or among the first ones."""
    at = torch.arange(s["queries"], device=device)[:, None] + (s["keys"] - s["queries"])
    j = torch.arange(s["keys"], device=device)[None, :]
    seen = j <= at
    return seen & ((at - j < s["window"]) | (j < s["sinks"])) if s["window"] else seen


def _attention(s):
    t, (b, h, m, d), kv = s["q"].dtype, s["q"].shape, s["kv_heads"]
    q = s["q"].float().reshape(b, kv, h // kv, m, d)
    k, v = s["k"].float()[:, :, None], s["v"].float()[:, :, None]
    scale = 1 / math.sqrt(d)
    seen = _seen(s, q.device)
    x = (q @ k.mT).mul_(scale).masked_fill_(~seen, -math.inf)
    top = x.max(-1, keepdim=True).values
    p = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total))
    o = p @ v
    out = {"o": o.reshape(b, h, m, d).to(t)}
    if s["pass"] == "train":
        g = s["grad"].float().reshape(b, kv, h // kv, m, d)
        dv = (p.mT @ g).sum(2)
        ds = (g @ v.mT).sub_((g * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        out |= {"dq": (ds @ k).reshape(b, h, m, d).to(t), "dk": (ds.mT @ q).sum(2).to(t), "dv": dv.to(t)}
    return out


def _linear_cross_entropy(s):
    t = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    kept = s["targets"] != IGNORED
    at = torch.where(kept, s["targets"], 0)[:, None]
    z = x @ w.t()
    z = z.sub_(z.max(1, keepdim=True).values)
    total = torch.exp(z).sum(1, keepdim=True)
    loss = torch.where(kept, torch.log(total)[:, 0] - z.gather(1, at)[:, 0], 0.0)
    count = kept.sum()
    out = {"loss": loss if s["reduction"] == "none" else loss.sum() if s["reduction"] == "sum" else loss.sum() / count}
    if s["pass"] == "train":
        a = s["grad"] / count if s["reduction"] == "mean" else s["grad"]
        a = torch.where(kept, a, 0.0)[:, None]
        g = z.exp_().mul_(a / total)
        g.scatter_add_(1, at, -a)
        out |= {"dx": (g @ w).to(t), "dweight": (g.t() @ x).to(t)}
    return out


def _mixed(x):
    """A whole number below 2^32 with its bits spread (the last steps of MurmurHash3, 32 bits); of numbers or tensors."""
    x = ((x ^ (x >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
    x = ((x ^ (x >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
    return x ^ (x >> 16)


TOP_M, TOP_V = 0.9375, 0.96875  # what the largest code stands for before the scale
DOWN, UP = 2.0 ** -111, 2.0 ** 111  # the lowest exponent of a code and fp32's: codes are then the top bits of fp32 numbers
LEAST = 2.0 ** -100  # a block whose largest value is below this is held as zeros


def _blocks(x):
    """The values in rows of a block each, with zeros behind the last."""
    return torch.nn.functional.pad(x.reshape(-1), (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _held(code, scale, bits, top):
    """What codes stand for, without their sign: blocks of codes whose lowest bit is number `bits` of an fp32 number."""
    return ((code.int() << bits).view(torch.float32) * UP) * torch.tensor(1 / top, device=code.device) * scale[:, None]


def _coded(size, random, bits, top, most):
    """Codes of values that are not negative, rounded up or down at random in proportion to what is lost, and their blocks' scales."""
    largest = size.amax(1)
    scale = torch.where(largest < LEAST, 0.0, torch.where(largest.isfinite(), largest, math.nan))
    usable = scale >= LEAST
    y = size * torch.where(usable, 1 / torch.where(usable, scale, 1.0), 0.0)[:, None] * top * DOWN
    code = torch.clamp(((y.view(torch.int32).long() + random) >> bits), max=most)
    return torch.where(usable[:, None], code, 0), scale


def _adamw(s):
    b1, b2 = BETAS
    t = s["step"]
    root = 1 / math.sqrt(1 - b2 ** t)
    size = LR / (1 - b1 ** t)
    for i, (p, g, m, v) in enumerate(zip(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"])):
        f = g.float()
        if s["bits"] == 32:
            m0, v0 = m, v
        else:
            c, r, scale = _blocks(m), _blocks(v), s["block_scales"][i]
            m0 = _held(c & 127, scale[:, 0], 20, TOP_M)
            m0 = torch.where(c >= 128, -m0, m0).view(-1)[:f.numel()].view(f.shape)
            v0 = _held(r, scale[:, 1], 19, TOP_V).square().view(-1)[:f.numel()].view(f.shape)
        m1 = m0 * b1 + f * (1 - b1)
        v1 = v0 * b2 + f * f * (1 - b2)
        r1 = v1.sqrt()
        p.copy_(p.float() * (1 - LR * DECAY) - m1 / (r1 * root + EPS) * size)
        if s["bits"] == 32:
            m.copy_(m1)
            v.copy_(v1)
            continue
        key = _mixed((_mixed((s["seed"] + t * 0x9E3779B9) & 0xFFFFFFFF) + i) & 0xFFFFFFFF)
        number = torch.arange(m.numel(), device=p.device)
        h = _blocks(_mixed((number * 0x9E3779B1 + key) & 0xFFFFFFFF))
        code, scale[:, 0] = _coded(_blocks(m1.abs()), ((h & 0xFFFF) << 4) + 8, 20, TOP_M, 127)
        code = code + 128 * ((_blocks(m1) < 0) & (code > 0)).long()
        m.view(-1).copy_(code.view(-1)[:m.numel()])
        code, scale[:, 1] = _coded(_blocks(r1), ((h >> 16) << 3) + 4, 19, TOP_V, 255)
        code = torch.where((_blocks(r1) > 0) & (scale[:, 1:] > 0), code.clamp(min=1), code)  # a root above 0 stays above it
        v.view(-1).copy_(code.view(-1)[:v.numel()])
    s["step"] = t + 1
    if s["bits"] == 32:
        return {"param": s["param"], "exp_avg": s["exp_avg"], "exp_avg_sq": s["exp_avg_sq"]}
    c, r = _blocks(s["exp_avg"]), _blocks(s["exp_avg_sq"])
    m = _held(c & 127, s["scales"][:, 0], 20, TOP_M)
    return {"param": s["param"], "exp_avg": torch.where(c >= 128, -m, m).view(-1), "exp_avg_sq": _held(r, s["scales"][:, 1], 19, TOP_V).square().view(-1)}


def _own(s):
    from tirocinio_triennale_b200 import ops

    if s["op"] == "attention":
        window = s["window"] or None
        if s["pass"] == "forward":
            return {"o": ops.attention(s["q"], s["k"], s["v"], window=window, sinks=s["sinks"])}
        leaves = [s[n].detach().requires_grad_() for n in ("q", "k", "v")]
        o = ops.attention(*leaves, window=window, sinks=s["sinks"])
        dq, dk, dv = torch.autograd.grad(o, leaves, s["grad"])
        return {"o": o, "dq": dq, "dk": dk, "dv": dv}
    if s["op"] == "linear_cross_entropy":
        if s["pass"] == "forward":
            return {"loss": ops.linear_cross_entropy(s["x"], s["weight"], s["targets"], ignore_index=IGNORED, reduction=s["reduction"])}
        x, w = s["x"].detach().requires_grad_(), s["weight"].detach().requires_grad_()
        loss = ops.linear_cross_entropy(x, w, s["targets"], ignore_index=IGNORED, reduction=s["reduction"])
        dx, dw = torch.autograd.grad(loss, (x, w), s["grad"])
        return {"loss": loss, "dx": dx, "dweight": dw}
    ops.adamw_step(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], s["block_scales"], step=s["step"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, seed=s["seed"])
    s["step"] += 1
    if s["bits"] == 32:
        return {"param": s["param"], "exp_avg": s["exp_avg"], "exp_avg_sq": s["exp_avg_sq"]}
    m, v = ops.adamw_values(s["exp_avg"], s["exp_avg_sq"], s["scales"])
    return {"param": s["param"], "exp_avg": m, "exp_avg_sq": v}


def run(state):
    if own:
        return _own(state)
    return {"attention": _attention, "linear_cross_entropy": _linear_cross_entropy, "adamw": _adamw}[state["op"]](state)


def _pairs(case):
    """How many pairs of a query and a key that it sees one head has."""
    total, off = 0, case["keys"] - case["queries"]
    for i in range(case["queries"]):
        n = max(0, i + off + 1)  # up to its own position
        total += min(n, max(min(case["sinks"], n), 0) + min(case["window"], n)) if case["window"] else n
    return total


def work(case):
    e = SIZE[case["type"]]
    train = case["pass"] == "train"
    if case["op"] == "attention":
        off = case["keys"] - case["queries"]
        # keys that no query sees need not be read
        read = min(case["keys"], case["sinks"] + case["window"] + case["queries"] - 1 - min(0, off)) if case["window"] else case["keys"]
        q, kv = case["batch"] * case["heads"] * case["queries"] * case["head"], case["batch"] * case["kv_heads"] * read * case["head"]
        whole = case["batch"] * case["kv_heads"] * case["keys"] * case["head"]
        nbytes = e * (2 * q + 2 * kv) + (e * (2 * q + 2 * whole) if train else 0)
        return {"bytes": nbytes, "flops": case["batch"] * case["heads"] * _pairs(case) * case["head"] * (14 if train else 4)}
    if case["op"] == "linear_cross_entropy":
        m, k, n = case["rows"], case["inner"], case["vocab"]
        return {"bytes": e * (m * k + n * k) * (2 if train else 1) + 8 * m + (4 * m if case["reduction"] == "none" else 0), "flops": 2 * m * k * n * (3 if train else 1)}
    n = sum(math.prod(shape) for shape in _shapes(case))
    # parameter in and out, gradient in, moments in and out; of moments in 8 bits also the values that they stand for
    moments = 16 * n if case["bits"] == 32 else 4 * n + 8 * n + 32 * (n // BLOCK + 1)
    return {"bytes": n * (2 * e + SIZE[case["grad"]]) + moments, "flops": 16 * n}


def exact(case, seed):
    """The operators' definitions in 64 bits, gradients by autograd, a head at a time."""
    s = prepare(case, seed)
    if case["op"] == "attention":
        group = case["heads"] // case["kv_heads"]
        if case["batch"] * case["heads"] > 512:
            return None
        seen = _seen(s, s["q"].device)
        some = seen.any(1, keepdim=True)
        out = {n: torch.zeros(s[f].shape, dtype=torch.float64, device="cuda") for n, f in (("o", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v"))}
        for b in range(case["batch"]):
            for h in range(case["heads"]):
                q, k, v = (s[n][b, i].double().requires_grad_(case["pass"] == "train") for n, i in (("q", h), ("k", h // group), ("v", h // group)))
                x = torch.einsum("id,jd->ij", q, k) / case["head"] ** 0.5
                x = torch.where(some, torch.where(seen, x, -math.inf), 0.0)
                o = torch.einsum("ij,jd->id", torch.softmax(x, 1) * some, v)
                out["o"][b, h] = o.detach()
                if case["pass"] == "train":
                    dq, dk, dv = torch.autograd.grad(o, (q, k, v), s["grad"][b, h].double())
                    out["dq"][b, h] = dq
                    out["dk"][b, h // group] += dk
                    out["dv"][b, h // group] += dv
        return out if case["pass"] == "train" else {"o": out["o"]}
    if case["op"] == "linear_cross_entropy":
        train = case["pass"] == "train"
        x, w = s["x"].double().requires_grad_(train), s["weight"].double().requires_grad_(train)
        losses = torch.zeros(case["rows"], dtype=torch.float64, device="cuda")
        dx, dw = torch.zeros_like(x), torch.zeros_like(w)
        weight = s["grad"].double()
        if case["reduction"] == "mean":
            weight = weight / (s["targets"] >= 0).sum()
        weight = weight.expand(case["rows"])
        for i in range(0, case["rows"], 1024):
            rows = slice(i, i + 1024)
            loss = torch.nn.functional.cross_entropy(torch.einsum("mk,nk->mn", x[rows], w), s["targets"][rows], ignore_index=IGNORED, reduction="none")
            losses[rows] = loss.detach()
            if train:
                a, b = torch.autograd.grad(loss, (x, w), weight[rows])
                dx += a
                dw += b
        if case["reduction"] == "mean":
            losses = losses.sum() / (s["targets"] >= 0).sum()
        elif case["reduction"] == "sum":
            losses = losses.sum()
        return {"loss": losses, "dx": dx, "dweight": dw} if train else {"loss": losses}
    b1, b2 = BETAS
    t = case["step"]
    out = {n: s[n].double() for n in (("param", "exp_avg", "exp_avg_sq") if case["bits"] == 32 else ("param",))}
    at, first, _, _ = _places(case)
    if case["bits"] == 32:
        m0, v0 = s["exp_avg"].double(), s["exp_avg_sq"].double()
    else:
        # a code is a number with 4 bits of exponent, the lowest exponent without a leading one
        def number(code, fraction):
            e, f = code >> fraction, (code & ((1 << fraction) - 1)).double() / (1 << fraction)
            return torch.where(e > 0, 1 + f, f) * torch.exp2(e.clamp(min=1).double() - 16)

        c, r = s["exp_avg"].long(), s["exp_avg_sq"].long()
        scale = s["scales"].double().repeat_interleave(BLOCK, 0)
        m0 = torch.where(c >= 128, -1.0, 1.0) * number(c & 127, 3) / TOP_M * scale[:, 0]
        v0 = (number(r, 4) / TOP_V * scale[:, 1]) ** 2
    for a, f, shape in zip(at, first, _shapes(case)):
        n = math.prod(shape)
        g = s["gradient"][a:a + n].double()
        m = m0[f:f + n].lerp(g, 1 - b1)
        v = v0[f:f + n].lerp(g * g, 1 - b2)
        adam = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + EPS)
        p = out["param"][a:a + n]
        out["param"][a:a + n] = p - LR * DECAY * p - LR * adam
        if case["bits"] == 32:
            out["exp_avg"][f:f + n], out["exp_avg_sq"][f:f + n] = m, v
    return out if case["bits"] == 32 else {"param": out["param"], "exp_avg": None, "exp_avg_sq": None}
