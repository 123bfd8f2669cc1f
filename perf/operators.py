"""Measured cases of the fine-tuning operators: the residual join of a block with its norms, the
log-probability losses, and the clipped optimizer step.

``own`` chooses what ``run`` calls: the plain form in elementary torch operations, or this
package's operators."""
import math

import torch

own = False

LOW = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


# -- the cases ------------------------------------------------------------------------------------

def _residual(name, batch, seq, width, stream, update, out, params, kind="rms", post=False,
              gate="none", scale=1.0, next=True, train=True):
    return {"name": name, "op": "residual_norm", "batch": batch, "seq": seq, "width": width,
            "stream": stream, "update": update, "out": out, "params": params, "kind": kind,
            "post": post, "gate": gate, "scale": scale, "next": next, "train": train}


def _logits(name, op, batch, seq, vocab, ld, dtype, prompt=0, kl=0.0, packed=False, smoothing=0.0,
            average=False, train=True):
    return {"name": name, "op": op, "batch": batch, "seq": seq, "vocab": vocab, "ld": ld,
            "dtype": dtype, "prompt": prompt, "kl": kl, "packed": packed, "smoothing": smoothing,
            "average": average, "train": train}


def listed():
    return [
        # the join of attention and MLP in the GPT-2 benchmark: fp32 stream under bf16 autocast
        _residual("gpt2 join", 8, 1024, 768, "fp32", "bf16", "bf16", "fp32", kind="layer"),
        # Llama-1.3B with a norm on either side of the block and a learned gate on each channel
        _residual("llama-1.3b sandwich", 4, 2048, 2048, "bf16", "bf16", "bf16", "bf16", post=True,
                  gate="channel", scale=0.5),
        # Llama-3-8B width, every sequence with a gate of its own (conditioned blocks)
        _residual("llama3-8b gates", 2, 2048, 4096, "bf16", "bf16", "bf16", "bf16", post=True,
                  gate="sequence"),
        # one new token for each of eight sequences: latency counts
        _residual("one token each", 8, 1, 2048, "bf16", "bf16", "bf16", "bf16", post=True,
                  gate="channel", train=False),
        # an odd width, where rows begin at any address; the block's end, without a following norm
        _residual("odd width", 3, 1111, 1001, "fp32", "fp32", "fp32", "fp32", post=True,
                  gate="sequence", scale=0.7, next=False),
        # log-probabilities under the frozen reference model
        _logits("reference logprobs", "token_logprobs", 8, 1024, 50257, 50304, "bf16", train=False),
        # a policy step on GPT-2: sampled answers behind a prompt, a KL term to the reference
        _logits("policy gpt2", "policy_loss", 8, 1024, 50257, 50304, "bf16", prompt=128, kl=0.04),
        # a few short answers, full precision, rows that begin at any address
        _logits("policy small", "policy_loss", 3, 41, 32001, 32001, "fp32", prompt=9),
        # pairs of answers of unequal lengths packed one behind the other
        _logits("preference packed", "preference_loss", 8, 700, 32000, 32000, "bf16", prompt=60,
                packed=True),
        # a pair of long answers over Llama-3's vocabulary
        _logits("preference llama3", "preference_loss", 2, 2048, 128256, 128256, "bf16", prompt=512,
                smoothing=0.1),
        # the gradients of llama-125m as the list that a model's parameters hold
        {"name": "norm llama-125m", "op": "grad_norm", "layers": 12, "width": 768, "ffn": 2048,
         "vocab": 32000, "dtype": "fp32"},
        # the optimizer step of the GPT-2 benchmark with its gradients clipped
        {"name": "clipped step", "op": "clipped_adamw", "n": 124_475_904, "clip": 0.25},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["residual_norm", "residual_norm", "token_logprobs", "policy_loss",
                     "preference_loss", "grad_norm", "clipped_adamw"])
    if op == "residual_norm":
        width = _spread(rng, 64, 8192)
        if rng.random() < 0.7:
            width = max(64, width // 64 * 64)
        rows = _spread(rng, 1, min(16384, 16_000_000 // width))
        batch = rng.randint(1, min(rows, 9))
        stream, update, out, params = rng.choice([
            ("fp32", "bf16", "bf16", "fp32"), ("fp32", "fp32", "fp32", "fp32"),
            ("bf16", "bf16", "bf16", "bf16"), ("fp16", "fp16", "fp16", "fp16"),
            ("fp32", "fp16", "fp16", "fp32")])
        case = _residual("", batch, rows // batch, width, stream, update, out, params,
                         kind=rng.choice(["rms", "layer"]), post=rng.random() < 0.5,
                         gate=rng.choice(["none", "channel", "sequence"]),
                         scale=rng.choice([1.0, 0.5, 1.0 / math.sqrt(24)]),
                         next=rng.random() < 0.8, train=rng.random() < 0.8)
    elif op in ("token_logprobs", "policy_loss", "preference_loss"):
        vocab = _spread(rng, 256, 131072)
        ld = vocab if rng.random() < 0.5 else -(-vocab // 64) * 64
        rows = _spread(rng, 2, min(8192, 400_000_000 // ld))
        batch = rng.randint(1, max(1, min(4, rows // 2))) * 2
        seq = max(1, rows // batch)
        case = _logits("", op, batch, seq, vocab, ld, rng.choice(["bf16", "bf16", "fp32", "fp16"]),
                       prompt=rng.randint(0, seq // 3), kl=rng.choice([0.0, 0.02, 0.1]),
                       packed=rng.random() < 0.5, smoothing=rng.choice([0.0, 0.1]),
                       average=rng.random() < 0.3,
                       train=op != "token_logprobs" or rng.random() < 0.5)
        if case["dtype"] == "fp32":
            case["seq"] = max(1, seq // 2)
            case["prompt"] = min(case["prompt"], case["seq"] // 3)
    elif op == "grad_norm":
        case = {"name": "", "op": op, "layers": rng.randint(1, 16), "width": _spread(rng, 33, 900),
                "ffn": _spread(rng, 33, 2500), "vocab": _spread(rng, 256, 40000),
                "dtype": rng.choice(["fp32", "bf16", "fp16"])}
    else:
        case = {"name": "", "op": op, "n": _spread(rng, 1000, 100_000_000),
                "clip": rng.choice([0.1, 0.5, 1e6])}
    del case["name"]
    return case


# -- what the cases have to move and compute --------------------------------------------------------

def _lengths(case):
    """Tokens of each sequence.  Packed answers differ in length by a fixed rule."""
    if not case["packed"]:
        return [case["seq"]] * case["batch"]
    return [max(1, case["seq"] - (i * 37 + 11) % max(1, case["seq"] // 2)) for i in range(case["batch"])]


def _counted(case):
    return sum(max(0, length - case["prompt"]) for length in _lengths(case))


def _shapes(case):
    w, f, v = case["width"], case["ffn"], case["vocab"]
    block = [(w,), (w,), (w, w), (w, w), (w, w), (w, w), (f, w), (f, w), (w, f)]
    return [(v, w)] + block * case["layers"] + [(w,), (v, w)]


def work(case):
    op = case["op"]
    if op == "residual_norm":
        n = case["batch"] * case["seq"] * case["width"]
        s, u, o = BYTES[case["stream"]], BYTES[case["update"]], BYTES[case["out"]]
        low = n * (2 * s + u + (o if case["next"] else 0))
        if case["train"]:                      # both output gradients in, both input gradients out
            low += n * (2 * s + u + (o if case["next"] else 0))
        return {"bytes": low, "flops": n * (30 if case["train"] else 12)}
    if op in ("token_logprobs", "policy_loss", "preference_loss"):
        size, rows = BYTES[case["dtype"]], sum(_lengths(case))
        read = _counted(case) * case["vocab"] * size
        write = rows * case["ld"] * size if case["train"] else 0
        return {"bytes": read + write + 16 * rows,
                "flops": _counted(case) * case["vocab"] * (8 if case["train"] else 4)}
    if op == "grad_norm":
        n = sum(math.prod(s) for s in _shapes(case))
        return {"bytes": n * BYTES[case["dtype"]], "flops": 2 * n}
    return {"bytes": 28 * case["n"], "flops": 16 * case["n"]}


# -- inputs ---------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32, std=1.0, mean=0.0):
        return torch.empty(*shape, device="cuda", dtype=torch.float32).normal_(mean, std, generator=g).to(dtype)

    s = {"case": case}
    op = case["op"]
    if op == "residual_norm":
        b, t, d = case["batch"], case["seq"], case["width"]
        stream, params = LOW[case["stream"]], LOW[case["params"]]
        s["residual"] = normal(b, t, d, dtype=stream, std=1.5, mean=0.1)
        s["update"] = normal(b, t, d, dtype=LOW[case["update"]], std=0.6)
        layer = case["kind"] == "layer"
        s["weight"] = normal(d, dtype=params, std=0.2, mean=1.0) if case["next"] else None
        s["bias"] = normal(d, dtype=params, std=0.1) if case["next"] and layer else None
        s["post_weight"] = normal(d, dtype=params, std=0.2, mean=1.0) if case["post"] else None
        s["post_bias"] = normal(d, dtype=params, std=0.1) if case["post"] and layer else None
        s["gate"] = None
        if case["gate"] != "none":
            shape = (d,) if case["gate"] == "channel" else (b, 1, d)
            s["gate"] = normal(*shape, dtype=params, std=0.3, mean=0.8)
        if case["train"]:
            s["d_stream"] = normal(b, t, d, dtype=stream)
            s["d_normed"] = normal(b, t, d, dtype=LOW[case["out"]]) if case["next"] else None
            for name in ("residual", "update", "weight", "bias", "post_weight", "post_bias", "gate"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
    elif op in ("token_logprobs", "policy_loss", "preference_loss"):
        lengths, vocab, ld = _lengths(case), case["vocab"], case["ld"]
        rows = sum(lengths)
        logits = normal(rows, ld, dtype=LOW[case["dtype"]], std=2.0)
        targets = torch.randint(vocab, (rows,), device="cuda", generator=g)
        at = torch.arange(rows, device="cuda")
        logits[at, targets] += 6.0             # a model gives what was sampled a good share
        length = torch.tensor(lengths, device="cuda")
        offsets = torch.zeros(len(lengths) + 1, dtype=torch.int64, device="cuda")
        offsets[1:] = length.cumsum(0)
        which = torch.repeat_interleave(torch.arange(len(lengths), device="cuda"), length)
        targets = torch.where(at - offsets[which] < case["prompt"], torch.full_like(targets, -100), targets)
        s["which"], s["offsets"] = which, offsets
        logprobs, _ = _plain_logprobs(logits, targets, vocab)
        if op == "policy_loss":
            drift = normal(rows, std=0.15)
            ratio = drift.exp()                # no token on the clip's edge, where the gradient jumps
            edge = ((ratio - 1.2).abs() < 1e-3) | ((ratio - 0.8).abs() < 1e-3)
            s["old"] = logprobs - torch.where(edge, torch.zeros_like(drift), drift)
            s["reference"] = logprobs + normal(rows, std=0.2) if case["kl"] else None
            s["advantages"] = normal(len(lengths))[which].contiguous()
        elif op == "preference_loss":
            so_far = torch.cat([logprobs.new_zeros(1).double(), logprobs.double().cumsum(0)])
            sums = so_far[offsets[1:]] - so_far[offsets[:-1]]
            # the policy has drifted by a few hundredths for each token of an answer
            s["reference"] = (sums + normal(len(lengths)) * (2.0 + 0.02 * length)).float()
        else:
            s["d_logprobs"] = normal(rows)
        if not case["packed"]:
            shape = (case["batch"], case["seq"])
            logits, targets = logits.view(*shape, ld), targets.view(shape)
            for name in ("old", "reference", "advantages", "d_logprobs"):
                if s.get(name) is not None and op != "preference_loss":
                    s[name] = s[name].view(shape)
        s["logits"], s["targets"] = logits, targets
        if case["train"]:
            logits.requires_grad_(True)
    elif op == "grad_norm":
        s["grads"] = [normal(*shape, dtype=LOW[case["dtype"]], std=3e-3) for shape in _shapes(case)]
    else:
        n = case["n"]
        s["p"], s["g"] = normal(n, std=0.02), normal(n, std=2e-4)
        s["max_norm"] = case["clip"] * 2e-4 * math.sqrt(n)
    return s


ADAM = {"lr": 3e-4, "betas": (0.9, 0.95), "eps": 1e-8, "weight_decay": 0.1}
CLIP, BETA = 0.2, 0.1


# -- the operators --------------------------------------------------------------------------------

def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _own_residual_norm(s):
    from gpubridge_b200.ops.residual_norm import residual_norm
    c = s["case"]
    names = [n for n in ("residual", "update", "weight", "bias", "post_weight", "post_bias", "gate")
             if s[n] is not None]
    stream, normed = residual_norm(
        s["residual"], s["update"], s["weight"], s["bias"], post_weight=s["post_weight"],
        post_bias=s["post_bias"], gate=s["gate"], scale=c["scale"], kind=c["kind"],
        out_dtype=LOW[c["out"]])
    out = {"stream": stream.detach()}
    if normed is not None:
        out["normed"] = normed.detach()
    if c["train"]:
        outputs, grads = [stream], [s["d_stream"]]
        if normed is not None:
            outputs, grads = [stream, normed], [s["d_stream"], s["d_normed"]]
        for name, grad in zip(names, torch.autograd.grad(outputs, [s[n] for n in names], grads)):
            out["d_" + name] = grad
    return out


def _own_token_logprobs(s):
    from gpubridge_b200.ops.logprob import token_logprobs
    c = s["case"]
    logprobs = token_logprobs(s["logits"], s["targets"], c["vocab"])
    out = {"logprobs": logprobs.detach()}
    if c["train"]:
        out["d_logits"], = torch.autograd.grad(logprobs, s["logits"], s["d_logprobs"])
    return out


def _own_policy_loss(s):
    from gpubridge_b200.ops.logprob import policy_loss
    c = s["case"]
    r = policy_loss(s["logits"], s["targets"], s["old"], s["advantages"], vocab=c["vocab"],
                    ref_logprobs=s["reference"], clip=(CLIP, CLIP), kl_coef=c["kl"], unit_grad=True)
    d, = torch.autograd.grad(r.loss, s["logits"])
    return {"loss": r.loss.detach(), "logprobs": r.logprobs, "kl": r.kl, "clipped": r.clipped,
            "d_logits": d}


def _own_preference_loss(s):
    from gpubridge_b200.ops.logprob import preference_loss
    c = s["case"]
    r = preference_loss(s["logits"], s["targets"], s["reference"], vocab=c["vocab"], beta=BETA,
                        offsets=s["offsets"] if c["packed"] else None, average=c["average"],
                        label_smoothing=c["smoothing"])
    d, = torch.autograd.grad(r.loss, s["logits"])
    return {"loss": r.loss.detach(), "rewards": r.rewards, "logprobs": r.logprobs, "d_logits": d}


def _own_grad_norm(s):
    from gpubridge_b200.ops.grad_clip import grad_norm
    return {"norm": grad_norm(s["grads"])}


def _own_clipped_adamw(s):
    if "optimizer" not in s:                   # a program keeps its optimizer from step to step
        from gpubridge_b200.ops.optim import FlatAdamW
        s["optimizer"] = FlatAdamW(s["p"], s["g"], **ADAM)
    o = s["optimizer"]
    o.step(max_norm=s["max_norm"], zero_grad=False)
    return {"p": o.p, "m": o.m, "v": o.v, "norm": o.grad_norm}


def _norm(x, weight, bias, kind):
    """(output, normalised x, reciprocal deviation) over the last dimension, eps 1e-5."""
    centred = x - x.mean(-1, keepdim=True) if kind == "layer" else x
    rstd = (centred.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    hat = centred * rstd
    y = hat * weight
    return (y + bias if bias is not None else y), hat, rstd


def _norm_grad(dy, hat, rstd, weight, kind):
    d = dy * weight
    inner = d - hat * (d * hat).mean(-1, keepdim=True)
    return rstd * (inner - d.mean(-1, keepdim=True) if kind == "layer" else inner)


def _residual_norm(s, wide):
    """The formulas, in ``wide``.  The norm that follows is that of the stream as it is returned."""
    c = s["case"]
    kind, scale, d = c["kind"], c["scale"], c["width"]
    low, par = LOW[c["stream"]], LOW[c["params"]]

    def up(name):
        return None if s.get(name) is None else s[name].detach().to(wide)

    u, gate, w, pw = up("update"), up("gate"), up("weight"), up("post_weight")
    if pw is not None:
        v, uhat, urstd = _norm(u, pw, up("post_bias"), kind)
    else:
        v = u
    gv = v if gate is None else v * gate
    stream = (up("residual") + scale * gv).to(low)
    out = {"stream": stream}
    if w is not None:
        y, hat, rstd = _norm(stream.to(wide), w, up("bias"), kind)
        out["normed"] = y.to(LOW[c["out"]])
    if not c["train"]:
        return out
    dr = up("d_stream")
    if w is not None:
        dy = up("d_normed")
        dr = dr + _norm_grad(dy, hat, rstd, w, kind)
        out["d_weight"] = (dy * hat).reshape(-1, d).sum(0).to(par)
        if s["bias"] is not None:
            out["d_bias"] = dy.reshape(-1, d).sum(0).to(par)
    out["d_residual"] = dr.to(low)
    dv = dr * scale
    if gate is not None:
        dg = dv * v
        out["d_gate"] = (dg.sum(1, keepdim=True) if c["gate"] == "sequence" else dg.reshape(-1, d).sum(0)).to(par)
        dv = dv * gate
    if pw is not None:
        out["d_post_weight"] = (dv * uhat).reshape(-1, d).sum(0).to(par)
        if s["post_bias"] is not None:
            out["d_post_bias"] = dv.reshape(-1, d).sum(0).to(par)
        dv = _norm_grad(dv, uhat, urstd, pw, kind)
    out["d_update"] = dv.to(LOW[c["update"]])
    return out


def _plain_residual_norm(s):
    return _residual_norm(s, torch.float32)


def _plain_logprobs(logits, targets, vocab):
    """(log-probability of each row's target or 0, the softmax of each row) in 32 bits."""
    x = logits[:, :vocab].float()
    x = x - x.amax(-1, keepdim=True)
    e = x.exp()
    total = e.sum(-1, keepdim=True)
    counted = targets >= 0
    at = targets.clamp(min=0)[:, None]
    logprobs = x.gather(1, at) - total.log()
    return torch.where(counted, logprobs[:, 0], torch.zeros_like(logprobs[:, 0])), e / total


def _spread_grad(coef, p, targets, logits):
    """Gradient of the logits where ``coef`` is that of each row's log-probability."""
    d = p * -coef[:, None]
    at = targets.clamp(min=0)[:, None]
    d.scatter_add_(1, at, coef[:, None])
    full = torch.zeros(logits.shape, dtype=logits.dtype, device=logits.device)
    full.view(-1, logits.shape[-1])[:, :d.shape[1]] = d.to(logits.dtype)
    return full


def _flat(s):
    logits, targets = s["logits"].detach(), s["targets"].reshape(-1)
    return logits, logits.reshape(-1, logits.shape[-1]), targets


def _plain_token_logprobs(s):
    c = s["case"]
    logits, rows, targets = _flat(s)
    logprobs, p = _plain_logprobs(rows, targets, c["vocab"])
    out = {"logprobs": logprobs.view(s["targets"].shape)}
    if c["train"]:
        coef = torch.where(targets >= 0, s["d_logprobs"].reshape(-1), torch.zeros_like(logprobs))
        out["d_logits"] = _spread_grad(coef, p, targets, logits)
    return out


def _policy_terms(s, logprobs, targets):
    """(loss, kl, clipped share, gradient of each log-probability) in the type of ``logprobs``."""
    c, wide = s["case"], logprobs.dtype
    w = (targets >= 0).to(wide)
    w = w / w.sum()
    a = s["advantages"].reshape(-1).to(wide)
    ratio = (logprobs - s["old"].reshape(-1).to(wide)).exp()
    outside = ((a > 0) & (ratio > 1 + CLIP)) | ((a < 0) & (ratio < 1 - CLIP))
    surrogate = torch.minimum(ratio * a, ratio.clamp(1 - CLIP, 1 + CLIP) * a)
    d = torch.where(outside, torch.zeros_like(a), -a * ratio)
    loss, kl = -surrogate, torch.zeros_like(a)
    if s["reference"] is not None:
        gap = s["reference"].reshape(-1).to(wide) - logprobs
        kl = gap.expm1() - gap
        loss = loss + c["kl"] * kl
        d = d - c["kl"] * gap.expm1()
    return (w * loss).sum(), (w * kl).sum(), (w * outside).sum(), w * d


def _plain_policy_loss(s):
    logits, rows, targets = _flat(s)
    logprobs, p = _plain_logprobs(rows, targets, s["case"]["vocab"])
    loss, kl, clipped, coef = _policy_terms(s, logprobs, targets)
    return {"loss": loss, "logprobs": logprobs.view(s["targets"].shape), "kl": kl,
            "clipped": clipped, "d_logits": _spread_grad(coef, p, targets, logits)}


def _preference_terms(s, logprobs, targets):
    """(loss, rewards, log-probability and row gradients of each sequence), first half chosen."""
    c, which, wide = s["case"], s["which"], logprobs.dtype
    n = c["batch"]
    sums = torch.zeros(n, dtype=wide, device=logprobs.device).index_add_(0, which, logprobs)
    share = torch.ones_like(sums)
    if c["average"]:
        share = torch.zeros_like(sums).index_add_(0, which, (targets >= 0).to(wide)).clamp(min=1).reciprocal()
    sums = sums * share
    rewards = BETA * (sums - s["reference"].to(wide))
    margin, e = rewards[:n // 2] - rewards[n // 2:], c["smoothing"]
    softplus = margin.abs().neg().exp().log1p()
    loss = ((1 - e) * (softplus + (-margin).clamp(min=0)) + e * (softplus + margin.clamp(min=0))).mean()
    d = (torch.sigmoid(margin) - (1 - e)) * BETA / (n // 2)
    coef = (torch.cat([d, -d]) * share)[which]
    return loss, rewards, sums, torch.where(targets >= 0, coef, torch.zeros_like(coef))


def _plain_preference_loss(s):
    logits, rows, targets = _flat(s)
    logprobs, p = _plain_logprobs(rows, targets, s["case"]["vocab"])
    loss, rewards, sums, coef = _preference_terms(s, logprobs.double(), targets)
    return {"loss": loss.float(), "rewards": rewards.float(), "logprobs": sums.float(),
            "d_logits": _spread_grad(coef.float(), p, targets, logits)}


def _plain_grad_norm(s):
    return {"norm": torch.stack([g.double().square().sum() for g in s["grads"]]).sum().sqrt().float()}


def _adamw(s, p, g, m, v, step):
    b1, b2 = ADAM["betas"]
    norm = g.square().sum(dtype=torch.float64).sqrt()
    g = g * (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).to(g.dtype)
    p = p * (1 - ADAM["lr"] * ADAM["weight_decay"])
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    denominator = v.sqrt() / math.sqrt(1 - b2 ** step) + ADAM["eps"]
    return p - (ADAM["lr"] / (1 - b1 ** step)) * m / denominator, m, v, norm


def _plain_clipped_adamw(s):
    if "m" not in s:
        s["m"], s["v"], s["step"] = torch.zeros_like(s["p"]), torch.zeros_like(s["p"]), 0
    s["step"] += 1
    p, m, v, norm = _adamw(s, s["p"], s["g"], s["m"], s["v"], s["step"])
    s["p"].copy_(p), s["m"].copy_(m), s["v"].copy_(v)
    return {"p": s["p"], "m": s["m"], "v": s["v"], "norm": norm.float()}


_own = {"residual_norm": _own_residual_norm, "token_logprobs": _own_token_logprobs,
        "policy_loss": _own_policy_loss, "preference_loss": _own_preference_loss,
        "grad_norm": _own_grad_norm, "clipped_adamw": _own_clipped_adamw}
_plain = {"residual_norm": _plain_residual_norm, "token_logprobs": _plain_token_logprobs,
          "policy_loss": _plain_policy_loss, "preference_loss": _plain_preference_loss,
          "grad_norm": _plain_grad_norm, "clipped_adamw": _plain_clipped_adamw}


# -- 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    """The operators from their definitions in 64 bits, through autograd where there are gradients."""
    s = prepare(case, seed)
    op = case["op"]
    if op == "residual_norm":
        return _exact_residual_norm(s, case)
    if op == "grad_norm":
        return {"norm": math.sqrt(sum(float((g.double() ** 2).sum()) for g in s["grads"]))}
    if op == "clipped_adamw":
        g = s["g"].double()
        norm = (g ** 2).sum().sqrt()
        g = g * min(1.0, s["max_norm"] / (float(norm) + 1e-6))
        (b1, b2), p = ADAM["betas"], s["p"].double()
        m, v = (1 - b1) * g, (1 - b2) * g ** 2      # from zero, first step
        p = p - ADAM["lr"] * ADAM["weight_decay"] * p
        p = p - ADAM["lr"] * (m / (1 - b1)) / ((v / (1 - b2)).sqrt() + ADAM["eps"])
        return {"p": p, "m": m, "v": v, "norm": norm}
    logits, rows, targets = _flat(s)
    logprobs = torch.zeros(targets.shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros_like(logprobs)
    step = max(1, 100_000_000 // case["ld"])
    for lo in range(0, len(targets), step):
        x = rows[lo:lo + step, :case["vocab"]].double()
        t = targets[lo:lo + step]
        lse[lo:lo + step] = torch.logsumexp(x, -1)
        picked = x.gather(1, t.clamp(min=0)[:, None])[:, 0] - lse[lo:lo + step]
        logprobs[lo:lo + step] = torch.where(t >= 0, picked, 0.0)
    leaf = logprobs.clone().requires_grad_(True)
    counted = targets >= 0
    if op == "token_logprobs":
        out = {"logprobs": logprobs.view(s["targets"].shape)}
        if not case["train"]:
            return out
        (coef,) = torch.autograd.grad(leaf, leaf, s["d_logprobs"].reshape(-1).double())
    elif op == "policy_loss":
        a = s["advantages"].reshape(-1).double()
        ratio = torch.exp(leaf - s["old"].reshape(-1).double())
        each = -torch.min(ratio * a, torch.clamp(ratio, 1 - CLIP, 1 + CLIP) * a)
        kl = torch.zeros_like(each)
        if s["reference"] is not None:
            gap = s["reference"].reshape(-1).double() - leaf
            kl = torch.exp(gap) - gap - 1
        loss = (each + case["kl"] * kl)[counted].mean()
        cut = ((a > 0) & (ratio > 1 + CLIP)) | ((a < 0) & (ratio < 1 - CLIP))
        out = {"loss": loss.detach(), "logprobs": logprobs.view(s["targets"].shape),
               "kl": kl[counted].mean().detach(), "clipped": cut[counted].double().mean()}
        (coef,) = torch.autograd.grad(loss, leaf)
    else:
        n, offsets = case["batch"], s["offsets"].tolist()
        sums = []
        for i in range(n):
            inside = leaf[offsets[i]:offsets[i + 1]]
            tokens = int(counted[offsets[i]:offsets[i + 1]].sum())
            sums.append(inside.sum() / (max(1, tokens) if case["average"] else 1))
        sums = torch.stack(sums)
        rewards = BETA * (sums - s["reference"].double())
        margin, e = rewards[:n // 2] - rewards[n // 2:], case["smoothing"]
        log_sigmoid = torch.nn.functional.logsigmoid
        loss = (-(1 - e) * log_sigmoid(margin) - e * log_sigmoid(-margin)).mean()
        (coef,) = torch.autograd.grad(loss, leaf)
        out = {"loss": loss.detach(), "rewards": rewards.detach(), "logprobs": sums.detach()}
    coef = torch.where(counted, coef, 0.0)
    d = torch.zeros(rows.shape, dtype=torch.float64, device="cuda")
    for lo in range(0, len(targets), step):
        t, c = targets[lo:lo + step].clamp(min=0)[:, None], coef[lo:lo + step, None]
        p = torch.exp(rows[lo:lo + step, :case["vocab"]].double() - lse[lo:lo + step, None])
        d[lo:lo + step, :case["vocab"]] = -c * p
        d[lo:lo + step].scatter_add_(1, t, c)
    return {**out, "d_logits": d.view(logits.shape)}


def _exact_residual_norm(s, case):
    names = [n for n in ("residual", "update", "weight", "bias", "post_weight", "post_bias", "gate")
             if s[n] is not None]
    leaf = {n: s[n].detach().double().requires_grad_(case["train"]) for n in names}

    def norm(x, weight, bias):
        if case["kind"] == "layer":
            var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
            y = (x - mean) / torch.sqrt(var + 1e-5) * weight
        else:
            y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * weight
        return y if bias is None else y + bias

    u = leaf["update"]
    if case["post"]:
        u = norm(u, leaf["post_weight"], leaf.get("post_bias"))
    if case["gate"] != "none":
        u = u * leaf["gate"]
    whole = leaf["residual"] + case["scale"] * u
    # the norm that follows is that of the stream as it is returned: its values are rounded, its
    # gradient is that of the sum
    rounded = whole + (whole.detach().to(LOW[case["stream"]]).double() - whole.detach())
    out = {"stream": whole.detach()}
    outputs = [whole]
    if case["next"]:
        normed = norm(rounded, leaf["weight"], leaf.get("bias"))
        out["normed"] = normed.detach()
        outputs.append(normed)
    if case["train"]:
        grads = [s["d_stream"].double()] + ([s["d_normed"].double()] if case["next"] else [])
        for name, grad in zip(names, torch.autograd.grad(outputs, [leaf[n] for n in names], grads)):
            out["d_" + name] = grad
    return out
