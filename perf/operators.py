"""The training-step operators of this framework: what is measured, on which inputs, and what the results have to be.

Four operators surround the propagation / transition operators in a training step of a Jakal-Net model:

* ``layer_norm`` forward: the apply step of a layer, sum = x + scale * delta, y = norm(sum) * weight + bias;
* ``layer_norm`` backward: the gradients of x, delta, weight and bias, with the gradient that reaches the sum from later layers;
* ``cross_entropy`` over the query head's vocabulary: the loss alone, the loss with its gradient, the gradient from a kept log-sum;
* ``clip_grad_norm``: the norm over all gradients of a model, and their clipping.

``run`` takes either the plain torch form (``own`` false) or the framework's calls (``own`` true) on what ``prepare`` made.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_SIZES = {"float32": 4, "bfloat16": 2, "float16": 2}
IGNORED = -100
EPS = 1e-5


def listed():
    return [
        # one token of one sequence: the smallest apply step, all latency
        dict(name="norm-forward-token", op="norm_forward", rows=1, dim=512, dtype="bfloat16", params="float32", delta=True, scale=1.0),
        # the S layer of the query-block model: batch 32, prefix 1024, dim 512
        dict(name="norm-forward-prefix", op="norm_forward", rows=32 * 1024, dim=512, dtype="bfloat16", params="float32", delta=True, scale=0.5),
        # the single dense layer in f32: batch 2, 256 nodes, dim 128
        dict(name="norm-backward-small", op="norm_backward", rows=2 * 256, dim=128, dtype="float32", params="float32", delta=True, scale=1.0),
        # long context: batch 4, 32768 nodes, dim 512
        dict(name="norm-backward-long", op="norm_backward", rows=4 * 32768, dim=512, dtype="bfloat16", params="float32", delta=True, scale=1.0),
        # a wide model whose width is odd, parameters in the activations' type, no residual
        dict(name="norm-backward-odd", op="norm_backward", rows=3001, dim=5001, dtype="float16", params="float16", delta=False, scale=1.0),
        # a short fine-tuning batch over a small vocabulary, some positions padded
        dict(name="loss-grad-small", op="loss", part="both", rows=24, vocab=1000, dtype="float32", smoothing=0.0, ignored=0.25, masked=0),
        # the query head: batch 32, 128 query slots, vocabulary 16384
        dict(name="loss-grad-head", op="loss", part="both", rows=32 * 128, vocab=16384, dtype="bfloat16", smoothing=0.0, ignored=0.0, masked=0),
        # validation: no gradient, a large odd vocabulary with banned tokens at its end
        dict(name="loss-eval-odd", op="loss", part="loss", rows=4096, vocab=50001, dtype="bfloat16", smoothing=0.0, ignored=0.1, masked=33),
        # a backward pass through autograd, from the log-sums that the forward pass kept, with label smoothing
        dict(name="loss-backward-smooth", op="loss", part="backward", rows=2047, vocab=32000, dtype="float16", smoothing=0.1, ignored=0.1, masked=0),
        # a toy model late in training: few small gradients, under the limit, left as they are
        dict(name="clip-toy", op="clip", dim=32, vocab=64, blocks=1, rank=8, dtype="float16", out="float16", limit=3.0, pad=64),
        # the query-block model's size in f32, above the limit, clipped where they lie
        dict(name="clip-model", op="clip", dim=512, vocab=16384, blocks=6, rank=64, dtype="float32", out="float32", limit=0.3, pad=64),
        # a large model's bf16 gradients, one after the other in a bucket, clipped into the f32 gradients of its optimizer
        dict(name="clip-large", op="clip", dim=1024, vocab=32768, blocks=16, rank=64, dtype="bfloat16", out="float32", limit=0.3, pad=1),
    ]


def draw(rng):
    def size(low, high):
        n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
        return max(low, min(high, n | 1 if rng.random() < 0.4 else n))

    kind = rng.choice(["norm_forward", "norm_backward", "loss", "clip"])
    dtype = rng.choice(sorted(_TYPES))
    if kind.startswith("norm"):
        dim = size(32, 8192)
        rows = size(1, min(131072, 2 ** 26 // dim))
        delta = rng.random() < 0.6
        return dict(op=kind, rows=rows, dim=dim, dtype=dtype, params=rng.choice([dtype, "float32"]), delta=delta,
                    scale=rng.choice([1.0, 0.5]) if delta else 1.0)
    if kind == "loss":
        vocab = size(64, 131072)
        rows = size(1, min(16384, 2 ** 27 // vocab))
        masked = rng.choice([0, 0, min(vocab // 8, 57)])
        return dict(op="loss", part=rng.choice(["both", "both", "loss", "backward"]), rows=rows, vocab=vocab, dtype=dtype,
                    smoothing=0.0 if masked else rng.choice([0.0, 0.1]), ignored=rng.choice([0.0, 0.15, 0.5]), masked=masked)
    dim = size(16, 1024)
    return dict(op="clip", dim=dim, vocab=size(32, 32768), blocks=size(1, 16), rank=rng.choice([16, 32, 64]), dtype=dtype,
                out=rng.choice([dtype, dtype, "float32"]), limit=rng.choice([0.3, 3.0]), pad=rng.choice([1, 64]))


def _gradient_shapes(case):
    """The parameters of a model: embedding and head, and in each block a propagation (two projections, core weight,
    bias), a value projection, a feed-forward pair and three norms."""
    d, v, r = case["dim"], case["vocab"], case["rank"]
    block = [(r, d), (r, d), (r,), (1,), (d, d), (d,), (4 * d, d), (4 * d,), (d, 4 * d), (d,)] + [(d,), (d,)] * 3
    return [(v, d)] + block * case["blocks"] + [(d,), (d,), (v, d), (v,)]


def _views(flat, shapes, pad):
    at, got = 0, []
    for s in shapes:
        n = math.prod(s)
        got.append(flat[at:at + n].view(s))
        at += -(-n // pad) * pad
    return got


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dtype = _TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device=dev)

    if case["op"].startswith("norm"):
        n, d = case["rows"], case["dim"]
        params = _TYPES[case["params"]]
        # a residual stream: each channel has its own offset and spread, a few are far larger than the others
        spread = torch.exp(0.3 * normal(d)) * torch.where(uniform(d) < 0.01, 8.0, 1.0)
        x = (normal(n, d) * spread + 0.5 * normal(d)).to(dtype)
        s = dict(case=case, x=x, weight=(1.0 + 0.1 * normal(d)).to(params), bias=(0.1 * normal(d)).to(params),
                 delta=(0.3 * normal(n, d)).to(dtype) if case["delta"] else None)
        if case["op"] == "norm_backward":
            # x is the sum that the forward pass kept, with its statistics
            xf = x.float()
            mean = xf.mean(-1)
            s.update(delta=None, mean=mean, rstd=torch.rsqrt((xf - mean[:, None]).square().mean(-1) + EPS),
                     grad_y=(0.01 * normal(n, d)).to(dtype), grad_sum=(0.01 * normal(n, d)).to(dtype) if case["delta"] else None)
        return s
    if case["op"] == "loss":
        n, v = case["rows"], case["vocab"]
        targets = torch.randint(0, v - case["masked"], (n,), generator=g, device=dev)
        logits = (2.0 * normal(n, v)).to(dtype)
        # what a model has learned: most targets stand out, by more or less
        logits[torch.arange(n, device=dev), targets] += (6.0 * uniform(n)).to(dtype)
        if case["masked"]:
            logits[:, v - case["masked"]:] = -math.inf
        targets[uniform(n) < case["ignored"]] = IGNORED
        targets[0] = int(seed) % (v - case["masked"])
        # f16 gradients go with a loss scaler
        s = dict(case=case, logits=logits, targets=targets, grad_scale=32768.0 if dtype == torch.float16 else 1.0)
        if case["part"] == "backward":
            s.update(lse=torch.where(targets == IGNORED, 0.0, torch.logsumexp(logits.float(), -1)),
                     grad_loss=torch.full((), s["grad_scale"], device=dev))
        return s
    shapes = _gradient_shapes(case)
    pad = case["pad"]
    total = sum(-(-math.prod(q) // pad) * pad for q in shapes)
    flat = torch.zeros(total, device=dev, dtype=dtype)
    grads = _views(flat, shapes, pad)
    scales, square = random.Random(int(seed)), 0.0
    for q in grads:
        # f16 gradients come out of a loss scaler, so they are no smaller than bf16 ones
        scale = 0.1 * 4.0 ** -scales.random()
        q.copy_(normal(*q.shape).mul_(scale))
        square += q.numel() * scale * scale
    out = flat if case["out"] == case["dtype"] else torch.zeros(total, device=dev, dtype=_TYPES[case["out"]])
    return dict(case=case, grads=grads, flat=flat, out=out, max_norm=case["limit"] * math.sqrt(square),
                outs=None if out is flat else _views(out, shapes, pad))


_module = None


def _framework():
    global _module
    if _module is None:
        path = str(Path.cwd() / "jakal-net_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import jakal_net_b200
        _module = jakal_net_b200
    return _module


def run(s):
    case = s["case"]
    op = case["op"]
    if op == "clip":
        max_norm = s["max_norm"]
        # a limit that falls a little with each step, so that gradients clipped in place are above it again in the next pass
        s["max_norm"] = max_norm * (0.9999 if case["limit"] < 1.0 else 1.0)
        if own:
            norm = _framework().clip_grad_norm_(s["grads"], max_norm, out=s["outs"])
        else:
            norm = _plain_clip(s["grads"], max_norm, s["outs"])
        return {"norm": norm, "grads": s["out"]}
    if op == "norm_forward":
        f = _framework().layer_norm_forward_cuda if own else _plain_norm_forward
        y, total, mean, rstd = f(s["x"], s["weight"], s["bias"], EPS, s["delta"], case["scale"])
        return {"y": y, "sum": total if case["delta"] else None, "mean": mean, "rstd": rstd}
    if op == "norm_backward":
        f = _framework().layer_norm_backward_cuda if own else _plain_norm_backward
        grad_x, grad_delta, grad_weight, grad_bias = f(s["grad_y"], s["x"], s["mean"], s["rstd"], s["weight"], s["grad_sum"],
                                                       case["scale"])
        return {"x": grad_x, "delta": grad_delta if case["scale"] != 1.0 else None, "weight": grad_weight, "bias": grad_bias}
    if case["part"] == "both":
        f = _framework().cross_entropy_with_grad_cuda if own else _plain_loss_with_grad
        loss, grad = f(s["logits"], s["targets"], IGNORED, case["smoothing"], "mean", s["grad_scale"])
        return {"loss": loss, "grad": grad}
    if case["part"] == "loss":
        f = _framework().cross_entropy_forward_cuda if own else _plain_loss
        loss, lse = f(s["logits"], s["targets"], IGNORED, case["smoothing"])
        return {"loss": loss, "lse": lse}
    f = _framework().cross_entropy_backward_cuda if own else _plain_loss_backward
    return {"grad": f(s["grad_loss"], s["logits"], s["targets"], s["lse"], IGNORED, case["smoothing"])}


# ---- plain forms: 32 bits throughout, rounded once at the end

def _plain_norm_forward(x, weight, bias, eps, delta, scale):
    h = x.float()
    if delta is not None:
        h = h + scale * delta.float()
    mean = h.mean(-1, keepdim=True)
    centred = h - mean
    rstd = torch.rsqrt(centred.square().mean(-1, keepdim=True) + eps)
    y = centred * rstd * weight.float() + bias.float()
    return y.to(x.dtype), h.to(x.dtype), mean.squeeze(-1), rstd.squeeze(-1)


def _plain_norm_backward(grad_y, x, mean, rstd, weight, grad_sum, scale):
    dy = grad_y.float()
    hat = (x.float() - mean[:, None]) * rstd[:, None]
    dhat = dy * weight.float()
    dx = rstd[:, None] * (dhat - dhat.mean(-1, keepdim=True) - hat * (dhat * hat).mean(-1, keepdim=True))
    if grad_sum is not None:
        dx = dx + grad_sum.float()
    return dx.to(x.dtype), (scale * dx).to(x.dtype), (dy * hat).sum(0).to(weight.dtype), dy.sum(0).to(weight.dtype)


def _plain_lse(z):
    top = z.amax(-1, keepdim=True)
    return (z - top).exp().sum(-1, keepdim=True).log() + top


def _plain_losses(z, lse, targets, ignore_index, smoothing):
    valid = targets != ignore_index
    picked = z.gather(-1, torch.where(valid, targets, 0)[:, None]).squeeze(-1)
    losses = lse - picked
    if smoothing:
        losses = (1.0 - smoothing) * losses + smoothing * (lse - z.mean(-1))
    return torch.where(valid, losses, 0.0).sum() / valid.sum()


def _plain_loss(logits, targets, ignore_index, smoothing):
    z = logits.float()
    lse = _plain_lse(z).squeeze(-1)
    # a row that is ignored has no log-sum that anyone asks for: 0
    return _plain_losses(z, lse, targets, ignore_index, smoothing), torch.where(targets == ignore_index, 0.0, lse)


def _plain_grad(z, lse, targets, ignore_index, smoothing, scale):
    valid = targets != ignore_index
    grad = (z - lse[:, None]).exp() - smoothing / z.shape[-1]
    grad.scatter_add_(-1, torch.where(valid, targets, 0)[:, None], torch.full_like(lse, smoothing - 1.0)[:, None])
    return torch.where(valid[:, None], grad * (scale / valid.sum()), 0.0)


def _plain_loss_with_grad(logits, targets, ignore_index, smoothing, reduction, grad_scale):
    z = logits.float()
    lse = _plain_lse(z).squeeze(-1)
    loss = _plain_losses(z, lse, targets, ignore_index, smoothing)
    return loss, _plain_grad(z, lse, targets, ignore_index, smoothing, grad_scale).to(logits.dtype)


def _plain_loss_backward(grad_loss, logits, targets, lse, ignore_index, smoothing):
    return _plain_grad(logits.float(), lse, targets, ignore_index, smoothing, grad_loss).to(logits.dtype)


def _plain_clip(grads, max_norm, outs):
    total = torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()
    coef = (max_norm / (total + 1e-6)).clamp(max=1.0)
    [o.copy_(g.float() * coef) for g, o in zip(grads, grads if outs is None else outs)]
    return total


# ---- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        flat = s["flat"].double()
        norm = torch.linalg.vector_norm(flat)
        return {"norm": norm, "grads": flat.mul_(min(1.0, s["max_norm"] / (norm.item() + 1e-6)))}
    if case["op"] == "norm_forward":
        h = s["x"].double()
        if case["delta"]:
            h += s["delta"].double() * case["scale"]
        var, mean = torch.var_mean(h, -1, correction=0)
        rstd = (var + EPS) ** -0.5
        y = torch.addcmul(s["bias"].double(), (h - mean[:, None]).mul_(rstd[:, None]), s["weight"].double())
        return {"y": y, "sum": h if case["delta"] else None, "mean": mean, "rstd": rstd}
    if case["op"] == "norm_backward":
        n, d = case["rows"], case["dim"]
        dy, w, rstd = s["grad_y"].double(), s["weight"].double(), s["rstd"].double()[:, None]
        hat = (s["x"].double() - s["mean"].double()[:, None]) * rstd
        u = dy * w
        along = torch.einsum("nd,nd->n", u, hat)[:, None] / d
        dx = rstd * (u - (dy @ w)[:, None] / d - along * hat)
        if case["delta"]:
            dx += s["grad_sum"].double()
        return {"x": dx, "delta": dx * case["scale"] if case["scale"] != 1.0 else None,
                "weight": torch.einsum("nd,nd->d", dy, hat), "bias": dy.sum(0)}
    z, targets = s["logits"].double(), s["targets"]
    rows = (targets != IGNORED).nonzero().squeeze(-1)
    q, v, eps = targets[rows], case["vocab"], case["smoothing"]
    if case["part"] == "backward":
        lse = s["lse"].double()[rows]
    else:
        lse = torch.logsumexp(z[rows], -1)
    answer = {}
    if case["part"] != "backward":
        share = z[rows].sum(-1) * (eps / v) if eps else 0.0
        answer["loss"] = (lse - (1.0 - eps) * z[rows, q] - share).sum() / rows.numel()
    if case["part"] == "loss":
        answer["lse"] = torch.zeros(targets.numel(), dtype=torch.float64, device=z.device).index_copy_(0, rows, lse)
        return answer
    p = torch.exp(z[rows] - lse[:, None])
    if eps:
        p -= eps / v
    p[torch.arange(rows.numel(), device=z.device), q] -= 1.0 - eps
    p *= s["grad_scale"] / rows.numel()
    answer["grad"] = torch.zeros_like(z).index_copy_(0, rows, p)
    return answer


def work(case):
    size = _SIZES[case["dtype"]]
    if case["op"].startswith("norm"):
        n, d = case["rows"], case["dim"]
        params = 2 * d * _SIZES[case["params"]]
        if case["op"] == "norm_forward":  # x and delta in, sum and y out, both statistics
            return {"bytes": n * d * size * (4 if case["delta"] else 2) + params + 8 * n, "flops": n * d * (11 if case["delta"] else 9)}
        # grad_y, x and the sum's gradient in, the gradients of x and of delta out; the weight in, its and the bias's gradient out
        passes = 3 + (1 if case["delta"] else 0) + (1 if case["scale"] != 1.0 else 0)
        return {"bytes": n * d * size * passes + 3 * params // 2 + 8 * n, "flops": n * d * 16}
    if case["op"] == "loss":
        n, v = case["rows"], case["vocab"]
        valid = 1.0 - case["ignored"]  # rows that count: the others are not read, and their gradient is zero
        bytes_ = n * v * size * (valid + (0 if case["part"] == "loss" else 1)) + 16 * n
        return {"bytes": bytes_, "flops": n * v * valid * (5 if case["part"] == "loss" else 8)}
    n = sum(math.prod(q) for q in _gradient_shapes(case))
    # under the limit a gradient that stays where it is need not be written
    write = 0 if case["limit"] > 1.0 and case["out"] == case["dtype"] else _SIZES[case["out"]]
    return {"bytes": n * (size + write) + 4, "flops": 3 * n}
