"""The operators of a training step around its products: the loss, the experts' router, the gradients' norm.

Three operators are covered, each through `flash_train.torch`:

  loss   linear_cross_entropy: hidden states times a large vocabulary's weight, and the cross entropy of that, without the
         logits ever being kept; with the gradients of both operands (a step) or without (scoring)
  route  expert_routing: softmax over experts, the top k of each token, how many tokens each expert got, and the balance loss;
         with the gradient of the router's logits (a step) or without
  clip   grad_norm and clip_grads: the norm over a list of gradients, and the gradients scaled to at most a given norm

Sizes are those of the repository's benchmark configurations (4096 wide, 14336 in the MLP, up to 16384 rows), general ones, and
ragged ones around them. Run from the repository root on a built tree.
"""
import math
import sys
from pathlib import Path

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_IGNORED = -100


def _framework():
    path = str(Path(__file__).resolve().parents[1] / "flash-train_b200" / "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import flash_train.torch as ft

    return ft


def listed():
    return [
        # The head of an 8B-class model over a batch of 8192 tokens, loss and gradients: the ordinary step, and the largest.
        {"name": "loss_step_bf16_8192x4096x131072", "op": "loss", "step": True, "type": "bf16", "tokens": 8192, "depth": 4096, "vocabulary": 131072},
        # A smaller model trained in FP32, the type of the framework's products.
        {"name": "loss_step_fp32_2048x2048x32000", "op": "loss", "step": True, "type": "fp32", "tokens": 2048, "depth": 2048, "vocabulary": 32000},
        # Packed sequences that end anywhere, a vocabulary that no tile divides, FP16 with a scaled loss.
        {"name": "loss_step_fp16_1999x2048x50257", "op": "loss", "step": True, "type": "fp16", "tokens": 1999, "depth": 2048, "vocabulary": 50257},
        # A test-sized model: launches and latency.
        {"name": "loss_step_fp32_129x512x8191", "op": "loss", "step": True, "type": "fp32", "tokens": 129, "depth": 512, "vocabulary": 8191},
        # Scoring a short prompt, a loss for every token and no gradients: the weight is streamed once.
        {"name": "loss_score_bf16_257x4096x131072", "op": "loss", "step": False, "type": "bf16", "tokens": 257, "depth": 4096, "vocabulary": 131072},
        # One token at a time through a small layer of experts.
        {"name": "route_one_fp32_1x8_top2", "op": "route", "step": False, "type": "fp32", "tokens": 1, "experts": 8, "top_k": 2},
        # A training batch and a middle number of experts.
        {"name": "route_step_fp32_16384x64_top8", "op": "route", "step": True, "type": "fp32", "tokens": 16384, "experts": 64, "top_k": 8},
        # A large batch over many experts, logits from a 16-bit product (equal logits are common), some of the batch padding.
        {"name": "route_step_bf16_65535x256_top8", "op": "route", "step": True, "type": "bf16", "tokens": 65535, "experts": 256, "top_k": 8, "masked": True},
        # The gradients of a tiny model.
        {"name": "clip_fp32_tiny", "op": "clip", "clip": True, "layers": 2, "width": 64, "inner": 160, "type": "fp32", "out": "fp32"},
        # The gradients of four layers of an 8B-class model, handed to an optimizer that keeps FP32.
        {"name": "clip_bf16_4x4096x14336", "op": "clip", "clip": True, "layers": 4, "width": 4096, "inner": 14336, "type": "bf16", "out": "fp32"},
        # Very many layers of odd widths: 1024 tensors whose ends, and beginnings in the optimizer's buffer, fall anywhere.
        {"name": "clip_fp32_128x255x511", "op": "clip", "clip": True, "layers": 128, "width": 255, "inner": 511, "type": "fp32", "out": "fp32"},
        # The norm alone, as a training loop logs it.
        {"name": "norm_fp32_2x4096x14336", "op": "clip", "clip": False, "layers": 2, "width": 4096, "inner": 14336, "type": "fp32", "out": None},
    ]


def _spread(rng, low, high, odd=0.4):
    """A size between low and high, even over the logarithm; a multiple of 64 / 8 / 1 by chance."""
    size = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() > odd:
        unit = 64 if size >= 512 else 8
        size = max(unit, size // unit * unit)
    return min(max(size, low), high)


def draw(rng):
    kind = rng.choice(["loss", "loss", "loss", "route", "route", "clip", "clip"])
    kinds = ["fp32", "bf16", "fp16"]
    if kind == "loss":
        tokens, depth = _spread(rng, 1, 8192), _spread(rng, 64, 4096)
        return {"op": "loss", "step": rng.random() < 0.7, "type": rng.choice(kinds), "tokens": tokens, "depth": depth,
                "vocabulary": _spread(rng, 128, 131072)}
    if kind == "route":
        experts = _spread(rng, 4, 512)
        return {"op": "route", "step": rng.random() < 0.7, "type": rng.choice(kinds), "tokens": _spread(rng, 1, 65536), "experts": experts,
                "top_k": rng.randint(1, min(experts, 8)), "masked": rng.random() < 0.3}
    clip, kind = rng.random() < 0.7, rng.choice(kinds)
    width = _spread(rng, 33, 4096)
    return {"op": "clip", "clip": clip, "layers": max(1, min(_spread(rng, 1, 128), int(6e8 / (13.5 * width * width)))), "width": width,
            "inner": int(3.5 * width), "type": kind, "out": rng.choice([kind, "fp32"]) if clip else None}


# ---------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _loss_inputs(case, seed):
    """Hidden states of unit variance, a weight that gives logits of deviation two, targets of which one in sixteen is padding."""
    generator, kind = _generator(seed), _TYPES[case["type"]]
    tokens, depth, vocabulary = case["tokens"], case["depth"], case["vocabulary"]
    hidden = torch.randn(tokens, depth, device="cuda", generator=generator).to(kind)
    weight = torch.empty(vocabulary, depth, device="cuda", dtype=kind)
    for at in range(0, vocabulary, 16384):
        rows = min(16384, vocabulary - at)
        weight[at:at + rows] = torch.randn(rows, depth, device="cuda", generator=generator).mul_(2 * depth ** -0.5).to(kind)
    target = torch.randint(0, vocabulary, (tokens,), device="cuda", generator=generator)
    padding = torch.rand(tokens, device="cuda", generator=generator) < 1 / 16
    target = torch.where(padding, torch.full_like(target, _IGNORED), target)
    # FP16 gradients want a scaled loss.
    return hidden, weight, target, torch.tensor(65536.0 if case["type"] == "fp16" else 1.0, device="cuda")


def _route_inputs(case, seed):
    """Logits of deviation one with some experts preferred, upstream gradients of the size that a mean over the tokens has."""
    generator, kind = _generator(seed), _TYPES[case["type"]]
    tokens, experts, k = case["tokens"], case["experts"], case["top_k"]
    logits = torch.randn(tokens, experts, device="cuda", generator=generator)
    logits = (logits + 0.5 * torch.randn(experts, device="cuda", generator=generator)).to(kind)
    mask = torch.rand(tokens, device="cuda", generator=generator) >= 0.1 if case.get("masked") else None
    scale = 65536.0 if case["type"] == "fp16" else 1.0
    grad_weights = torch.randn(tokens, k, device="cuda", generator=generator).mul_(0.01 * scale / tokens)
    return logits, mask, grad_weights, torch.tensor(0.01 * scale, device="cuda")


def _clip_inputs(case, seed):
    """Per layer two norm weights, four projections of the attention, and the three of an MLP."""
    generator, kind = _generator(seed), _TYPES[case["type"]]
    width, inner = case["width"], case["inner"]
    shapes = [(width,), (width,)] + [(width, width)] * 3 + [(inner, width)] * 2 + [(width, inner)]
    gradients = []
    for _ in range(case["layers"]):
        gradients += [torch.randn(shape, device="cuda", generator=generator).mul_(0.02).to(kind) for shape in shapes]
    return gradients


def prepare(case, seed):
    state = dict(case)
    if case["op"] == "loss":
        hidden, weight, target, grad = _loss_inputs(case, seed)
        state.update(hidden=hidden.requires_grad_(case["step"]), weight=weight.requires_grad_(case["step"]), target=target, grad=grad)
    elif case["op"] == "route":
        logits, mask, grad_weights, grad_loss = _route_inputs(case, seed)
        state.update(logits=logits.requires_grad_(case["step"]), mask=mask, grad_weights=grad_weights, grad_loss=grad_loss)
    else:
        state["gradients"] = _clip_inputs(case, seed)
        if case["clip"]:
            # An optimizer's gradients lie in one buffer, each tensor right behind the one before.
            state["flat"] = torch.empty(_elements(case), device="cuda", dtype=_TYPES[case["out"]])
            pieces = state["flat"].split([g.numel() for g in state["gradients"]])
            state["buffers"] = [piece.view(g.shape) for piece, g in zip(pieces, state["gradients"])]
    return state


# ---------------------------------------------------------------- the operators in plain form

def _plain_loss(state):
    hidden, weight, target = state["hidden"].detach().float(), state["weight"].detach().float(), state["target"]
    tokens, vocabulary = hidden.shape[0], weight.shape[0]
    valid = target != _IGNORED
    index = torch.where(valid, target, torch.zeros_like(target))
    losses = torch.empty(tokens, device="cuda")
    count = valid.sum().clamp(min=1)
    if state["step"]:
        hidden_grad, weight_grad = torch.empty_like(hidden), torch.zeros_like(weight)
        each = torch.where(valid, state["grad"] / count, torch.zeros_like(losses))
    rows = max(1, min(tokens, (1 << 28) // vocabulary))
    for at in range(0, tokens, rows):
        part = slice(at, min(at + rows, tokens))
        logits = hidden[part] @ weight.t()
        largest = logits.amax(1, keepdim=True)
        lse = largest + (logits - largest).exp_().sum(1, keepdim=True).log_()
        picked = logits.gather(1, index[part, None])
        losses[part] = torch.where(valid[part], (lse - picked)[:, 0], torch.zeros_like(losses[part]))
        if state["step"]:
            slope = (logits - lse).exp_()
            slope.scatter_add_(1, index[part, None], torch.full_like(picked, -1.0))
            slope *= each[part, None]
            hidden_grad[part] = slope @ weight
            weight_grad += slope.t() @ hidden[part]
    if not state["step"]:
        return {"loss": losses}
    kind = state["hidden"].dtype
    return {"loss": losses.double().sum().div(count).float(), "hidden_grad": hidden_grad.to(kind), "weight_grad": weight_grad.to(kind)}


def _plain_route(state):
    given = state["logits"].detach()
    logits, k = given.float(), state["top_k"]
    tokens, experts = logits.shape
    mask = state["mask"] if state["mask"] is not None else torch.ones(tokens, dtype=torch.bool, device="cuda")
    live = mask[:, None].float()
    p = (logits - logits.amax(1, keepdim=True)).exp()
    p = p / p.sum(1, keepdim=True)
    chosen = logits.sort(dim=1, descending=True, stable=True).indices[:, :k]  # equal ones: the lowest index first
    picked = p.gather(1, chosen)
    total = picked.sum(1, keepdim=True)
    weights = picked / total * live
    hits = torch.zeros(tokens, experts, device="cuda").scatter_(1, chosen, 1.0) * live
    counts = hits.sum(0, dtype=torch.float64)
    count = mask.sum().clamp(min=1).double()
    shares = counts / (count * k)
    loss = (experts * (shares * (p * live).sum(0, dtype=torch.float64) / count).sum()).float()
    out = {"weights": weights, "experts": torch.where(mask[:, None], chosen, torch.full_like(chosen, -1)).int(), "counts": counts.int(), "loss": loss}
    if state["step"]:
        # Through the weights (a softmax over the chosen), and through the mean of p.
        grad = state["grad_weights"]
        inner = weights * (grad - (grad * weights).sum(1, keepdim=True))
        slope = state["grad_loss"] * experts / count.float() * shares.float()
        outer = p * (slope - (p * slope).sum(1, keepdim=True)) * live
        out["logits_grad"] = outer.scatter_add(1, chosen, inner).to(given.dtype)
    return out


def _plain_clip(state):
    gradients = state["gradients"]
    norm = torch.stack([g.float().square().sum(dtype=torch.float64) for g in gradients]).sum().sqrt()
    if not state["clip"]:
        return {"norm": norm.float()}
    factor = (1.0 / (norm + 1e-6)).clamp(max=1.0).float()
    for gradient, buffer in zip(gradients, state["buffers"]):
        buffer.copy_(gradient.float() * factor)
    return {"norm": norm.float(), "clipped": state["flat"]}


# ---------------------------------------------------------------- one pass

def run(state):
    if not own:
        return {"loss": _plain_loss, "route": _plain_route, "clip": _plain_clip}[state["op"]](state)
    ft = _framework()
    if state["op"] == "loss":
        if not state["step"]:
            return {"loss": ft.linear_cross_entropy(state["hidden"], state["weight"], state["target"], reduction="none")}
        loss = ft.linear_cross_entropy(state["hidden"], state["weight"], state["target"])
        hidden_grad, weight_grad = torch.autograd.grad(loss, (state["hidden"], state["weight"]), state["grad"])
        return {"loss": loss.detach(), "hidden_grad": hidden_grad, "weight_grad": weight_grad}
    if state["op"] == "route":
        routing = ft.expert_routing(state["logits"], state["top_k"], mask=state["mask"])
        out = {"weights": routing.weights.detach(), "experts": routing.experts, "counts": routing.counts, "loss": routing.balance_loss.detach()}
        if state["step"]:
            out["logits_grad"], = torch.autograd.grad((routing.weights, routing.balance_loss), state["logits"],
                                                      (state["grad_weights"], state["grad_loss"]))
        return out
    if not state["clip"]:
        return {"norm": ft.grad_norm(state["gradients"])}
    return {"norm": ft.clip_grads(state["gradients"], 1.0, out=state["buffers"]), "clipped": state["flat"]}


def _elements(case):
    return case["layers"] * (2 * case["width"] + 3 * case["width"] ** 2 + 3 * case["width"] * case["inner"])


def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}
    if case["op"] == "loss":
        tokens, depth, vocabulary = case["tokens"], case["depth"], case["vocabulary"]
        operands = size[case["type"]] * depth * (tokens + vocabulary)
        if not case["step"]:
            return {"bytes": float(operands + 12 * tokens), "flops": 2.0 * tokens * depth * vocabulary}
        return {"bytes": float(2 * operands + 8 * tokens), "flops": 6.0 * tokens * depth * vocabulary}
    if case["op"] == "route":
        tokens, experts, k = case["tokens"], case["experts"], case["top_k"]
        one = size[case["type"]] * tokens * experts
        forward = one + 8 * tokens * k + 4 * experts + (tokens if case.get("masked") else 0)
        # Softmax: an exponential, a sum and a division for each logit, and about as much for the gradient.
        return {"bytes": float(forward + (one + 4 * tokens * k if case["step"] else 0)), "flops": (8.0 if case["step"] else 4.0) * tokens * experts}
    elements = _elements(case)
    return {"bytes": float(elements * (size[case["type"]] + (size[case["out"]] if case["clip"] else 0))), "flops": (3.0 if case["clip"] else 2.0) * elements}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_loss(case, seed):
    hidden, weight, target, grad = _loss_inputs(case, seed)
    tokens, vocabulary = case["tokens"], case["vocabulary"]
    weight = weight.double()
    valid = (target >= 0).nonzero()[:, 0]
    losses = torch.zeros(tokens, dtype=torch.float64, device="cuda")
    hidden_grad = torch.zeros(tokens, case["depth"], dtype=torch.float64, device="cuda")
    weight_grad = torch.zeros_like(weight) if case["step"] else None
    for rows in valid.split(max(1, (1 << 27) // vocabulary)):
        h, y = hidden[rows].double(), target[rows]
        log_p = torch.log_softmax(h @ weight.T, dim=1)
        at = torch.arange(len(rows), device="cuda")
        losses[rows] = -log_p[at, y]
        if case["step"]:
            slope = log_p.exp()
            slope[at, y] -= 1.0
            slope *= grad.double() / max(1, len(valid))
            hidden_grad[rows] = slope @ weight
            weight_grad += slope.T @ h
    if not case["step"]:
        return {"loss": losses}
    return {"loss": losses.sum() / max(1, len(valid)), "hidden_grad": hidden_grad, "weight_grad": weight_grad}


def _exact_route(case, seed):
    logits, mask, grad_weights, grad_loss = _route_inputs(case, seed)
    tokens, experts, k = case["tokens"], case["experts"], case["top_k"]
    wide = logits.double()
    p = torch.softmax(wide, dim=1)
    # k rounds of the largest left, the lowest index among equals.
    left, chosen, index = wide.clone(), [], torch.arange(experts, device="cuda")
    for _ in range(k):
        first = torch.where(left == left.max(1, keepdim=True).values, index, experts).min(1).indices
        chosen.append(first)
        left[torch.arange(tokens, device="cuda"), first] = -math.inf
    chosen = torch.stack(chosen, 1)
    on = mask if mask is not None else torch.ones(tokens, dtype=torch.bool, device="cuda")
    count = max(1, int(on.sum()))
    counts = torch.bincount(chosen[on].flatten(), minlength=experts)
    shares = counts.double() / (count * k)
    weights = torch.where(on[:, None], torch.softmax(wide.gather(1, chosen), dim=1), 0.0)
    out = {"weights": weights, "experts": torch.where(on[:, None], chosen, -1).int(), "counts": counts.int(),
           "loss": experts * (shares * p[on].sum(0) / count).sum()}
    if case["step"]:
        slope = grad_loss.double() * experts / count * shares
        logits_grad = torch.where(on[:, None], p * (slope - (p @ slope)[:, None]), 0.0)
        upstream = grad_weights.double()
        logits_grad.scatter_add_(1, chosen, weights * (upstream - (weights * upstream).sum(1, keepdim=True)))
        out["logits_grad"] = logits_grad
    return out


def exact(case, seed):
    if case["op"] == "loss":
        return _exact_loss(case, seed)
    if case["op"] == "route":
        return _exact_route(case, seed)
    gradients = _clip_inputs(case, seed)
    norm = math.sqrt(math.fsum(float((g.double() ** 2).sum()) for g in gradients))
    total = torch.tensor(norm, dtype=torch.float64, device="cuda")
    if not case["clip"]:
        return {"norm": total}
    return {"norm": total, "clipped": torch.cat([g.flatten() for g in gradients]).double() * min(1.0, 1.0 / (norm + 1e-6))}
