"""Performance cases of the operators between a network's categorical head and a circuit: what a program that serves, scores
and trains such a head, or feeds its outputs to a circuit as soft evidence, has them do.

Every case is one pass of one `kind`:

  logprobs       log-probabilities of given categories, entropy and best alternatives of logits [rows, cats]
  logprobs_grad  the same and the gradient of the logits, as a training step has it
  evidence       logits [rows, vars, cats] as normalised log-weights, the row index fastest: a circuit's soft evidence
  evidence_grad  the same and the gradient of the logits
  head           logits of few feature vectors by a head whose weights are held in 4 bits with group scales

`own = False` computes them with elementary torch operations in 32 bits, `own = True` through `lvd_pg_b200.api`.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = torch.device("cuda", 0)
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # Serving: the logits of one new position over a large vocabulary, with the twenty best alternatives.  Latency counts.
        dict(name="logprobs_one_position", kind="logprobs", rows=1, cats=131072, dtype="f32", top=20, temperature=1.0),
        # Scoring: every position of a long text, a tenth of the vocabulary ruled out.
        dict(name="logprobs_text", kind="logprobs", rows=2048, cats=131072, dtype="bf16", top=8, temperature=1.0),
        # Scoring images: one distribution of 256 levels for each of 784 pixels of 512 images.
        dict(name="logprobs_pixels", kind="logprobs", rows=512 * 784, cats=256, dtype="f16", top=1, temperature=1.0),
        # Training a vocabulary head: rows that start at every alignment, some positions without a given token.
        dict(name="grad_tokens", kind="logprobs_grad", rows=1021, cats=50021, dtype="bf16", top=4, temperature=0.8),
        # Training a pixel head with few levels, an entropy term in the loss.
        dict(name="grad_pixels", kind="logprobs_grad", rows=300 * 784, cats=200, dtype="f32", top=0, temperature=1.0),
        # A batch of image teachers' outputs as evidence for one EM step.
        dict(name="evidence_images", kind="evidence", rows=512, vars=784, cats=256, dtype="bf16", missing=0.0, temperature=1.0),
        # Codes of one patch position: a ragged batch, a codebook of 500, some codes unknown.
        dict(name="evidence_codes", kind="evidence", rows=37, vars=192, cats=500, dtype="f32", missing=0.15, temperature=0.7),
        # Training the teacher of patch circuits (192 pixels) through its evidence.
        dict(name="evidence_grad_patches", kind="evidence_grad", rows=500, vars=192, cats=256, dtype="f16", missing=0.05, temperature=1.3),
        # Binary variables: the shortest distributions.
        dict(name="evidence_grad_binary", kind="evidence_grad", rows=1000, vars=784, cats=2, dtype="f32", missing=0.1, temperature=1.0),
        # Serving: one feature vector against a large vocabulary head.
        dict(name="head_one_position", kind="head", rows=1, cats=131072, features=4096, dtype="bf16", group=64, bias=False),
        # Serving: sixteen positions at once, half-precision features and logits.
        dict(name="head_sixteen", kind="head", rows=16, cats=32000, features=2048, dtype="f16", group=128, bias=False),
        # A small head over a codebook, odd sizes everywhere, full-precision features.
        dict(name="head_codebook", kind="head", rows=3, cats=1000, features=777, dtype="f32", group=32, bias=True),
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["logprobs", "logprobs_grad", "evidence", "evidence_grad", "head"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind == "head":
        cats, features = _between(rng, 8, 131072), _between(rng, 32, 8192)
        features = min(features, max(32, 2 ** 29 // cats))
        return dict(kind=kind, rows=_between(rng, 1, 16), cats=cats, features=features, dtype=dtype, group=rng.choice([32, 64, 128]),
                    bias=rng.random() < 0.5)
    temperature = rng.choice([1.0, 0.7, 1.3])
    if kind.startswith("evidence"):
        cats, variables = _between(rng, 2, 2048), _between(rng, 1, 784)
        most = 2 ** 26 // (cats * variables)
        return dict(kind=kind, rows=_between(rng, 1, max(2, min(1000, most))), vars=variables, cats=cats, dtype=dtype,
                    missing=rng.choice([0.0, 0.1]), temperature=temperature)
    if rng.random() < 0.5:   # few categories, many rows
        cats = _between(rng, 2, 1024)
        rows = _between(rng, 1, 2 ** 26 // cats // (2 if kind == "logprobs_grad" else 1))
    else:
        cats = _between(rng, 1025, 131072)
        rows = _between(rng, 1, min(2048, 2 ** 27 // cats // (2 if kind == "logprobs_grad" else 1)))
    return dict(kind=kind, rows=rows, cats=cats, dtype=dtype, top=rng.randint(0, min(20, cats)), temperature=temperature)


# ---- inputs -----------------------------------------------------------------------------------------

def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE)


def _logits(gen, rows, cats, dtype):
    """Some categories are likelier everywhere, the rest is the position's own; the common offset is what training leaves open."""
    x = torch.empty(rows, cats, dtype=TYPES[dtype], device=DEVICE)
    common = 2.0 * _randn(gen, cats)
    step = max(1, 2 ** 25 // cats)
    for at in range(0, rows, step):   # a few 32-bit rows at a time
        part = x[at:at + step]
        part.copy_(common + 1.7 * _randn(gen, part.shape[0], cats) + _randn(gen, part.shape[0], 1))
    return x


def _logprob_inputs(case, gen):
    rows, cats = case["rows"], case["cats"]
    x = _logits(gen, rows, cats, case["dtype"])
    ruled_out = None
    if case["dtype"] == "bf16" and cats >= 64:
        ruled_out = torch.rand(cats, generator=gen, device=DEVICE) < 0.1
        ruled_out[0] = False
        x.masked_fill_(ruled_out, -math.inf)
    tokens = torch.randint(0, cats, (rows,), generator=gen, device=DEVICE)
    if ruled_out is not None:
        tokens = torch.where(ruled_out[tokens], 0, tokens)
    state = {"x": x, "tokens": tokens}
    if case["kind"] == "logprobs_grad":
        state["tokens"] = torch.where(torch.rand(rows, generator=gen, device=DEVICE) < 0.02, -1, tokens)
        state["g_logp"], state["g_entropy"] = _randn(gen, rows), 0.3 * _randn(gen, rows)
        state["g_top"] = _randn(gen, rows, case["top"]) if case["top"] else None
    return state


def _evidence_inputs(case, gen):
    rows, variables, cats = case["rows"], case["vars"], case["cats"]
    x = _logits(gen, rows * variables, cats, case["dtype"]).view(rows, variables, cats)
    miss = torch.rand(rows, variables, generator=gen, device=DEVICE) < case["missing"] if case["missing"] else None
    state = {"x": x, "miss": miss}
    if case["kind"] == "evidence_grad":
        state["g"] = _randn(gen, cats, variables, rows).permute(2, 1, 0)   # laid out as the evidence is
    return state


def _head_inputs(case, gen):
    cats, features, group = case["cats"], case["features"], case["group"]
    codes = (2.4 * _randn(gen, cats, features + features % 2)).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
    packed = codes[:, 0::2] | (codes[:, 1::2] << 4)   # two codes a byte, the even column in the low half
    groups = -(-features // group)
    scales = (0.5 + torch.rand(cats, groups, generator=gen, device=DEVICE)) / (2.4 * features ** 0.5)
    scales = scales.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float16)
    bias = _randn(gen, cats) if case["bias"] else None
    x = _randn(gen, case["rows"], features).to(TYPES[case["dtype"]])
    return {"x": x, "packed": packed, "scales": scales, "bias": bias}


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    make = _head_inputs if case["kind"] == "head" else _evidence_inputs if case["kind"].startswith("evidence") else _logprob_inputs
    state = {"case": case, **make(case, gen)}
    if own:
        if case["kind"] == "head":   # the weights in the kernel's order, once
            from lvd_pg_b200 import api
            state["head"] = api.QuantHead.from_codes(state["packed"], state["scales"], case["features"], case["group"], bias=state["bias"])
        elif case["kind"].endswith("grad"):
            state["x"].requires_grad_()
    return state


# ---- one pass ---------------------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "head":
        return _plain_head(state)
    return _plain_evidence(state) if kind.startswith("evidence") else _plain_logprobs(state)


def _run_own(state):
    from lvd_pg_b200 import api
    case = state["case"]
    kind = case["kind"]
    if kind == "head":
        return state["head"].logits(state["x"])
    x = state["x"]
    if kind.startswith("evidence"):
        out = api.soft_evidence(x, state["miss"], case["temperature"])
        return [out] if kind == "evidence" else [out, torch.autograd.grad(out, x, state["g"])[0]]
    out = api.token_logprobs(x, state["tokens"], case["top"], case["temperature"])
    answer = [out.logp, out.entropy] + ([out.top_ids, out.top_logp] if case["top"] else [])
    if kind == "logprobs_grad":
        outputs, weights = [out.logp, out.entropy], [state["g_logp"], state["g_entropy"]]
        if case["top"]:
            outputs, weights = outputs + [out.top_logp], weights + [state["g_top"]]
        answer = answer + [torch.autograd.grad(outputs, x, weights)[0]]
    return answer


def _log_softmax(x, temperature):
    """In 32 bits, over the last axis; a distribution without any possible category stays at -inf."""
    x = x.float()
    top = x.amax(-1, keepdim=True)
    d = (x - torch.where(top == -math.inf, 0.0, top)) / temperature
    total = d.exp().sum(-1, keepdim=True)
    return d - torch.where(total == 0, 1.0, total).log()


def _plain_logprobs(state):
    case, x, tokens = state["case"], state["x"], state["tokens"]
    logp = _log_softmax(x, case["temperature"])
    p = logp.exp()
    entropy = -(p * torch.where(p > 0, logp, 0.0)).sum(-1)
    given = tokens >= 0
    at = torch.where(given, tokens, 0)[:, None]
    answer = [torch.where(given, logp.gather(1, at)[:, 0], 0.0), entropy]
    if case["top"]:
        ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top"]]   # ties to the lowest index
        answer += [ids, logp.gather(1, ids)]
    if case["kind"] == "logprobs_grad":
        g = torch.where(given, state["g_logp"], 0.0)
        total = g + (state["g_top"].sum(-1) if case["top"] else 0.0)
        grad = -p * (total[:, None] + state["g_entropy"][:, None] * (torch.where(p > 0, logp, 0.0) + entropy[:, None]))
        grad.scatter_add_(1, at, g[:, None])
        if case["top"]:
            grad.scatter_add_(1, ids, state["g_top"])
        answer.append((grad / case["temperature"]).to(x.dtype))
    return answer


def _plain_evidence(state):
    case, x, miss = state["case"], state["x"], state["miss"]
    logp = _log_softmax(x, case["temperature"])
    out = logp if miss is None else torch.where(miss[:, :, None], 0.0, logp)
    out = out.permute(2, 1, 0).contiguous().permute(2, 1, 0)   # the row index fastest
    if case["kind"] == "evidence":
        return [out]
    g = state["g"] if miss is None else torch.where(miss[:, :, None], 0.0, state["g"])
    grad = (g - logp.exp() * g.sum(-1, keepdim=True)) / case["temperature"]
    return [out, grad.to(x.dtype).contiguous()]


def _plain_head(state):
    case, packed, scales = state["case"], state["packed"], state["scales"]
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(1)[:, :case["features"]].float() - 8.0
    weight = codes * scales.float().repeat_interleave(case["group"], 1)[:, :case["features"]]
    y = state["x"].float() @ weight.t()
    if state["bias"] is not None:
        y = y + state["bias"]
    return y.to(state["x"].dtype)


# ---- the same from the definition, in 64 bits ---------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "head":
        return _exact_head(case, state)
    return _exact_evidence(case, state) if case["kind"].startswith("evidence") else _exact_logprobs(case, state)


def _exact_logprobs(case, state):
    parts, step = [], max(1, 2 ** 26 // case["cats"])
    for at in range(0, case["rows"], step):
        rows = slice(at, at + step)
        x = state["x"][rows].detach().double().requires_grad_(case["kind"] == "logprobs_grad")
        scaled = x / case["temperature"]
        lse = torch.logsumexp(scaled, -1)
        logp = scaled - lse[:, None]
        possible = torch.isfinite(logp)
        finite = logp.masked_fill(~possible, 0.0)
        entropy = -(finite.exp() * finite).masked_fill(~possible, 0.0).sum(-1)
        tokens = state["tokens"][rows]
        chosen = logp.gather(1, tokens.clamp(min=0)[:, None])[:, 0].masked_fill(tokens < 0, 0.0)
        part = [chosen, entropy]
        if case["top"]:
            raw = x.detach()
            places = torch.arange(raw.shape[1], device=DEVICE)
            order = []
            left = raw.clone()
            for _ in range(case["top"]):   # the best that is left, and of equals the first
                best = left.amax(-1, keepdim=True)
                first = torch.where((left == best) & (left > -math.inf), places, raw.shape[1]).amin(-1)
                first = first.clamp(max=raw.shape[1] - 1)
                order.append(first)
                left.scatter_(1, first[:, None], -math.inf)
            ids = torch.stack(order, -1)
            part += [ids, logp.gather(1, ids)]
        if case["kind"] == "logprobs_grad":
            loss = (chosen * state["g_logp"][rows]).sum() + (entropy * state["g_entropy"][rows]).sum()
            if case["top"]:
                loss = loss + (part[3] * state["g_top"][rows]).sum()
            part.append(torch.autograd.grad(loss, x)[0])
        parts.append([t.detach() for t in part])
    return [torch.cat(column) for column in zip(*parts)]


def _exact_evidence(case, state):
    x = state["x"].detach().double().requires_grad_(case["kind"] == "evidence_grad")
    scaled = x / case["temperature"]
    out = scaled - torch.logsumexp(scaled, -1, keepdim=True)
    if state["miss"] is not None:
        out = out.masked_fill(state["miss"][:, :, None], 0.0)
    if case["kind"] == "evidence":
        return [out]
    return [out.detach(), torch.autograd.grad(out, x, state["g"].double())[0]]


def _exact_head(case, state):
    features, group = case["features"], case["group"]
    x, parts = state["x"].double(), []
    for at in range(0, case["cats"], 16384):
        packed, scales = state["packed"][at:at + 16384].long(), state["scales"][at:at + 16384].double()
        weight = torch.empty(packed.shape[0], 2 * packed.shape[1], dtype=torch.float64, device=DEVICE)
        weight[:, 0::2], weight[:, 1::2] = (packed % 16 - 8).double(), (packed // 16 - 8).double()
        weight = weight[:, :features] * scales[:, torch.arange(features, device=DEVICE) // group]
        parts.append(x @ weight.t())
    y = torch.cat(parts, 1)
    return y if state["bias"] is None else y + state["bias"].double()


# ---- what a pass cannot do without --------------------------------------------------------------------

def work(case):
    kind, rows, cats = case["kind"], case["rows"], case["cats"]
    size = 4 if case["dtype"] == "f32" else 2
    if kind == "head":
        features = case["features"]
        groups = -(-features // case["group"])
        weights = cats * (-(-features // 2) + 2 * groups) + (4 * cats if case["bias"] else 0)
        return {"bytes": weights + size * rows * (features + cats), "flops": 2 * rows * cats * features}
    if kind.startswith("evidence"):
        elements = rows * case["vars"] * cats
        masks = rows * case["vars"] if case["missing"] else 0
        backward = (4 + size) * elements if kind == "evidence_grad" else 0   # the evidence's gradient in, the logits' out
        return {"bytes": (size + 4) * elements + masks + backward, "flops": (10 if backward else 6) * elements}
    elements = rows * cats
    small = rows * (8 + 4 + 4 + 12 * case["top"])
    if kind == "logprobs_grad":
        return {"bytes": 2 * size * elements + small + rows * (8 + 4 * case["top"]), "flops": 16 * elements}
    return {"bytes": size * elements + small, "flops": 8 * elements}
