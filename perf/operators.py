"""The exact side of a decode step, as cases that can be timed: the router, the routed experts as a
whole, and the scores of the logits that come out.

Four operators, each in a plain form of elementary torch operations and, where `own` is true, as the
library's calls:

* "route": `route_tokens`, a router's softmax over the experts, its top k and their weights;
* "experts": `RoutedExperts`, all channels of the routed experts, for one token to a thousand;
* "logprobs": `token_logprobs`, log probabilities of given tokens with entropy and top alternatives;
* "compare": `compare_logits`, the divergence of two models' next-token distributions and whether
  their top tokens agree.

Weights, hidden rows and routing follow the synthetic layers of the benchmark.  Logits are Gaussian
with, in every second row, one token that stands out, which is how a language model's look.
"""

from __future__ import annotations

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def _route(name: str, **more: object) -> dict:
    return {"name": name, "op": "route", "tokens": 1, "experts": 128, "top_k": 8, "type": "bf16",
            "renormalize": True, "ids64": False, "weights16": False, **more}


def _experts(name: str, **more: object) -> dict:
    return {"name": name, "op": "experts", "tokens": 1, "hidden": 2048, "width": 768,
            "experts": 128, "top_k": 8, "activation": "silu", "inputs": "outliers",
            "skewed": False, "padding": 0, "ids64": False, "weights16": False, **more}


def _logprobs(name: str, **more: object) -> dict:
    return {"name": name, "op": "logprobs", "tokens": 1, "vocab": 151936, "type": "bf16",
            "top": 20, "extra": 0, "banned": False, **more}


def _compare(name: str, **more: object) -> dict:
    return {"name": name, "op": "compare", "tokens": 32, "vocab": 151936, "type": "bf16",
            "extra": 0, "noise": 0.05, **more}


def listed() -> list[dict]:
    return [
        # One user's chat: the router of a layer, then the layer itself.
        _route("route one token"),
        _experts("experts one token"),
        # A long prompt's rows through a router of many experts, in a fused engine's types.
        _route("route 1000 tokens", tokens=1000, experts=256, type="f32", renormalize=False,
               ids64=True, weights16=True),
        # A ragged batch of a GELU model with an odd width, padded as captured batches are.
        _experts("experts gelu 19 tokens", tokens=19, hidden=1152, width=704, experts=64, top_k=6,
                 activation="gelu_tanh", inputs="normal", padding=2, ids64=True, weights16=True),
        # The benchmark's batch on the benchmark's layer.
        _experts("experts 64 tokens", tokens=64),
        # A busy server with many small experts, heavy-tailed inputs and a skewed router.
        _experts("experts 256 tokens skewed", tokens=256, width=512, experts=256,
                 inputs="student_t", skewed=True, padding=13),
        # A piece of a prompt: rows outside the sparse policy.
        _experts("experts 1000 tokens", tokens=1000, width=1024, experts=64, inputs="normal"),
        # One sampled token with twenty alternatives.
        _logprobs("logprobs one token"),
        # A batch in FP32 after logits processors, an odd vocabulary, some tokens banned.
        _logprobs("logprobs 32 rows odd vocabulary", tokens=32, vocab=50257, type="f32", top=5,
                  banned=True),
        # Scoring a prompt: log probabilities and entropy of every position.
        _logprobs("logprobs 512 rows", tokens=512, top=0),
        # The decode study's batch: stock against sparse.
        _compare("compare 32 rows"),
        # Two far models over a padded vocabulary, in FP16.
        _compare("compare 300 rows far", tokens=300, vocab=32003, type="f16", extra=61, noise=1.0),
    ]


def _log_int(rng, low: int, high: int, step: int = 1) -> int:
    value = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, round(value / step) * step))


def draw(rng) -> dict:
    op = rng.choice(("route", "experts", "experts", "experts", "logprobs", "logprobs", "compare"))
    if op == "route":
        experts = _log_int(rng, 8, 512)
        case = _route("", tokens=_log_int(rng, 1, 1000), experts=min(experts, 256),
                      top_k=min(rng.choice((1, 2, 4, 6, 8, 8, 10)), experts),
                      type=rng.choice(("bf16", "f16", "f32")), renormalize=rng.random() < 0.7,
                      ids64=rng.random() < 0.5, weights16=rng.random() < 0.3)
    elif op == "experts":
        tokens = _log_int(rng, 1, 1000)
        hidden, width = _log_int(rng, 512, 4096, 128), _log_int(rng, 256, 1024, 16)
        experts = min(_log_int(rng, 16, 256), (1 << 28) // (hidden * width))  # 1.6 GB, as listed
        case = _experts("", tokens=tokens, hidden=hidden, width=width, experts=experts,
                        top_k=rng.choice((1, 2, 4, 6, 8, 8)),
                        activation=rng.choice(("silu", "silu", "gelu_tanh")),
                        inputs=rng.choice(("normal", "outliers", "student_t")),
                        skewed=rng.random() < 0.4, ids64=rng.random() < 0.5,
                        weights16=rng.random() < 0.3)
    else:
        make = _logprobs if op == "logprobs" else _compare
        case = make("", tokens=_log_int(rng, 1, 512), vocab=_log_int(rng, 1000, 262144),
                    type=rng.choice(("bf16", "bf16", "f16", "f32")),
                    extra=rng.choice((0, 0, 1, 64)))
        if op == "logprobs":
            case.update(top=rng.choice((0, 1, 5, 20, 32)), banned=rng.random() < 0.3)
        else:
            case.update(noise=rng.choice((0.02, 0.1, 1.0)))
    del case["name"]
    # Keep a drawn case below the largest listed one of its kind, whatever was drawn together.
    kin = [work(c) for c in listed() if c["op"] == op]
    most = {key: max(w[key] for w in kin) for key in ("bytes", "flops")}
    while case["tokens"] > 1 and any(work(case)[key] > most[key] for key in most):
        case["tokens"] = case["tokens"] * 3 // 4
    if op == "experts":
        case["padding"] = rng.randrange(0, 1 + case["tokens"] // 8)
    return case


# -- what a user's program has in hand -----------------------------------------------------
def _hidden_rows(case: dict, generator: torch.Generator) -> torch.Tensor:
    shape = (case["tokens"], case["hidden"])
    x = torch.randn(shape, device="cuda", generator=generator)
    if case["inputs"] == "student_t":  # three degrees of freedom, unit variance
        chi = torch.randn((*shape, 3), device="cuda", generator=generator).square().sum(-1)
        x = x / (chi / 3).sqrt() / math.sqrt(3.0)
    elif case["inputs"] == "outliers":  # one channel in a hundred is twenty times as large
        dims = torch.randperm(shape[1], device="cuda", generator=generator)
        x[:, dims[: math.ceil(0.01 * shape[1])]] *= 20.0
    return x.bfloat16()


def _prepare_experts(case: dict, generator: torch.Generator) -> dict:
    e, h, i, k = (case[x] for x in ("experts", "hidden", "width", "top_k"))
    gate_up = torch.empty((e, 2 * i, h), device="cuda", dtype=torch.bfloat16)
    gate_up.normal_(0.0, 0.02, generator=generator)
    down = torch.empty((e, i, h), device="cuda", dtype=torch.bfloat16)
    down.normal_(0.0, 0.02, generator=generator)
    down = down.transpose(1, 2)  # channel-major, as the sparse reader takes it
    hidden = _hidden_rows(case, generator)
    router = torch.randn((e, h), device="cuda", generator=generator)
    logits = hidden.float() @ (0.02 * router).T
    if case["skewed"]:
        logits = logits + torch.randn(e, device="cuda", generator=generator)
    weights, ids = torch.softmax(logits, dim=-1).topk(k, dim=-1)
    weights = weights / weights.sum(-1, keepdim=True)
    padding = None
    if case["padding"]:  # a captured batch is padded at its end
        padding = torch.arange(case["tokens"], device="cuda") >= case["tokens"] - case["padding"]
    state = {
        "gate_up": gate_up, "down": down, "hidden": hidden, "padding": padding,
        "ids": (ids if case["ids64"] else ids.int()).contiguous(),
        "weights": (weights.bfloat16() if case["weights16"] else weights).contiguous(),
    }
    if own:
        import cfm_b200  # noqa: F401  (registers the package alias)
        from cfm_b200.runtime.routed import RoutedExperts

        state["layer"] = RoutedExperts(gate_up, down, k, case["tokens"],
                                       activation=case["activation"])
    return state


def _logits(case: dict, generator: torch.Generator) -> torch.Tensor:
    """Rows of logits, some of a wider buffer: what an engine's padded vocabulary gives."""
    t, v = case["tokens"], case["vocab"]
    rows = 2.5 * torch.randn((t, v + case["extra"]), device="cuda", generator=generator)
    favourite = torch.randint(0, v, (t, 1), device="cuda", generator=generator)
    lift = 8.0 + 10.0 * torch.rand((t, 1), device="cuda", generator=generator)
    lift[::2] = 0.0
    return rows.scatter_add_(1, favourite, lift)


def prepare(case: dict, seed: int) -> dict:
    generator = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] == "experts":
        state.update(_prepare_experts(case, generator))
    elif case["op"] == "route":
        logits = 1.5 * torch.randn((case["tokens"], case["experts"]), device="cuda",
                                   generator=generator)
        state["logits"] = logits.to(_TYPES[case["type"]])
    else:
        t, v = case["tokens"], case["vocab"]
        rows = _logits(case, generator)
        if case["op"] == "compare":
            other = rows + case["noise"] * torch.randn(rows.shape, device="cuda",
                                                       generator=generator)
            state["other"] = other.to(_TYPES[case["type"]])[:, :v]
        elif case["banned"]:  # a twentieth of the vocabulary
            rows.masked_fill_(torch.rand(rows.shape, device="cuda", generator=generator) < 0.05,
                              -math.inf)
        if case["op"] == "logprobs":  # tokens sampled from the rows
            noise = torch.empty(rows.shape, device="cuda").exponential_(generator=generator)
            state["tokens"] = (rows - noise.log_())[:, :v].argmax(dim=-1)
        state["logits"] = rows.to(_TYPES[case["type"]])[:, :v]
    return state


# -- plain forms ---------------------------------------------------------------------------
def _largest(x: torch.Tensor, count: int) -> torch.Tensor:
    """Indices of the `count` largest values of every row, in order, ties to the lowest index."""
    return torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :count]


def _plain_route(state: dict):
    case = state["case"]
    x = state["logits"].float()
    ids = _largest(x, case["top_k"])
    e = torch.exp(x - x.amax(dim=-1, keepdim=True))
    kept = e.gather(1, ids)
    weights = kept / (kept if case["renormalize"] else e).sum(dim=-1, keepdim=True)
    return {"weights": weights.bfloat16() if case["weights16"] else weights,
            "ids": ids if case["ids64"] else ids.int()}


def _phi(gate: torch.Tensor, activation: str) -> torch.Tensor:
    if activation == "silu":
        return gate / (1.0 + torch.exp(-gate))
    return 0.5 * gate * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (gate + 0.044715 * gate**3)))


def _plain_experts(state: dict):
    case = state["case"]
    t, h, i, e, k = (case[x] for x in ("tokens", "hidden", "width", "experts", "top_k"))
    x = state["hidden"].float()
    ids, weights = state["ids"].long(), state["weights"].float()
    if state["padding"] is not None:
        weights = torch.where(state["padding"][:, None], 0.0, weights)
    gate_up, down = state["gate_up"], state["down"].transpose(1, 2)  # [E, I, H] in memory
    if 4 * t * k < e:  # each pair's expert apart
        rows = torch.matmul(gate_up[ids].float(), x[:, None, :, None])[..., 0]  # [T, K, 2 I]
        a = _phi(rows[..., :i], case["activation"]) * rows[..., i:] * weights[..., None]
        out = torch.matmul(a.reshape(t, 1, k * i), down[ids].float().reshape(t, k * i, h))[:, 0]
    else:  # all experts for all rows, weighted by zero where a row does not go
        mix = torch.zeros((t, e), device="cuda").scatter_add_(1, ids, weights)
        rows = torch.matmul(x, gate_up.reshape(-1, h).float().T).view(t, e, 2 * i)
        a = _phi(rows[..., :i], case["activation"]) * rows[..., i:] * mix[..., None]
        out = torch.matmul(a.reshape(t, e * i), down.reshape(-1, h).float())
    return out.bfloat16()


def _plain_logprobs(state: dict):
    x = state["logits"].float()
    shifted = x - x.amax(dim=-1, keepdim=True)
    e = torch.exp(shifted)
    z = e.sum(dim=-1, dtype=torch.float64)  # a long sum, next to one where a token stands out
    log_z = torch.log(z)
    entropy = log_z - torch.where(e > 0, e * shifted, 0.0).sum(dim=-1, dtype=torch.float64) / z
    given = shifted.gather(1, state["tokens"][:, None])[:, 0] - log_z
    out = {"logprobs": given.float(), "entropy": entropy.float()}
    if state["case"]["top"]:
        ids = _largest(x, state["case"]["top"])
        out["top_ids"] = ids.int()
        out["top_logprobs"] = (shifted.gather(1, ids) - log_z[:, None]).float()
    return out


def _plain_compare(state: dict):
    # In 64 bits: the divergence of near distributions is a small difference of long sums.
    a, b = state["logits"].double(), state["other"].double()
    log_p = a - a.amax(dim=-1, keepdim=True)
    log_p = log_p - log_p.exp().sum(dim=-1, keepdim=True).log()
    log_q = b - b.amax(dim=-1, keepdim=True)
    log_q = log_q - log_q.exp().sum(dim=-1, keepdim=True).log()
    p = log_p.exp()
    divergence = torch.where(p > 0, p * (log_p - log_q), 0.0).sum(dim=-1)
    return {"divergence": divergence.float(),
            "agreement": _largest(a, 1)[:, 0] == _largest(b, 1)[:, 0]}


def _library(state: dict):
    """The calls that a user makes."""
    from cfm_b200.runtime.fidelity import compare_logits, token_logprobs
    from cfm_b200.runtime.routing import route_tokens

    case = state["case"]
    if case["op"] == "route":
        weights, ids = route_tokens(
            state["logits"], case["top_k"], renormalize=case["renormalize"],
            weights_dtype=torch.bfloat16 if case["weights16"] else torch.float32,
            ids_dtype=torch.int64 if case["ids64"] else torch.int32)
        return {"weights": weights, "ids": ids}
    if case["op"] == "experts":
        return state["layer"](state["hidden"], state["ids"], state["weights"], state["padding"])
    if case["op"] == "logprobs":
        scores = token_logprobs(state["logits"], state["tokens"], top=case["top"])
        out = {"logprobs": scores.logprobs, "entropy": scores.entropy}
        if case["top"]:
            out.update(top_ids=scores.top_ids, top_logprobs=scores.top_logprobs)
        return out
    divergence, agreement = compare_logits(state["logits"], state["other"])
    return {"divergence": divergence, "agreement": agreement}


def run(state: dict):
    if own:
        return _library(state)
    op = state["case"]["op"]
    if op == "route":
        return _plain_route(state)
    if op == "experts":
        return _plain_experts(state)
    return _plain_logprobs(state) if op == "logprobs" else _plain_compare(state)


# -- from the definitions, in 64 bits ------------------------------------------------------
def _first_maxima(x: torch.Tensor, count: int) -> torch.Tensor:
    """The `count` largest of every row one after another, each the first among its equals."""
    left = torch.ones_like(x, dtype=torch.bool)
    places = torch.arange(x.shape[1], device=x.device).expand_as(x)
    found = []
    for _ in range(count):
        top = torch.where(left, x, -math.inf).amax(dim=-1, keepdim=True)
        first = torch.where(left & (x == top), places, x.shape[1]).amin(dim=-1, keepdim=True)
        left.scatter_(1, first, False)
        found.append(first)
    return torch.cat(found, dim=1)


def _exact_experts(case: dict, state: dict) -> torch.Tensor:
    i = case["width"]
    x = state["hidden"].double()
    out = torch.zeros_like(x)
    live = torch.ones(case["tokens"], dtype=torch.bool, device="cuda")
    if state["padding"] is not None:
        live = ~state["padding"]
    for expert in range(case["experts"]):
        tokens, slots = ((state["ids"] == expert) & live[:, None]).nonzero(as_tuple=True)
        if tokens.numel() == 0:
            continue
        rows = x[tokens] @ state["gate_up"][expert].double().T
        gate, up = rows[:, :i], rows[:, i:]
        if case["activation"] == "silu":
            gate = gate * torch.sigmoid(gate)
        else:
            inner = math.sqrt(2.0 / math.pi) * gate * (1.0 + 0.044715 * gate * gate)
            gate = gate * torch.sigmoid(2.0 * inner)  # (1 + tanh z) / 2 = sigmoid(2 z)
        rows = (gate * up) @ state["down"][expert].double().T
        out.index_add_(0, tokens, rows * state["weights"][tokens, slots].double()[:, None])
    return out


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["op"] == "experts":
        return _exact_experts(case, state)
    x = state["logits"].double()
    total = torch.logsumexp(x, dim=-1, keepdim=True)
    if case["op"] == "route":
        ids = _first_maxima(x, case["top_k"])
        weights = (x - total).gather(1, ids).exp()
        if case["renormalize"]:
            weights = weights / weights.sum(dim=-1, keepdim=True)
        return {"weights": weights, "ids": ids}
    if case["op"] == "logprobs":
        log_p = x - total
        out = {"logprobs": log_p.gather(1, state["tokens"][:, None])[:, 0],
               "entropy": -torch.where(log_p > -math.inf, log_p.exp() * log_p, 0.0).sum(dim=-1)}
        if case["top"]:
            out["top_ids"] = _first_maxima(x, case["top"])
            out["top_logprobs"] = log_p.gather(1, out["top_ids"])
        return out
    y = state["other"].double()
    log_p, log_q = x - total, y - torch.logsumexp(y, dim=-1, keepdim=True)
    # Each term with p - q added, which cancel over a row, so that none is negative.
    terms = log_p.exp() * (log_p - log_q + torch.expm1(log_q - log_p))
    return {"divergence": terms.sum(dim=-1),
            "agreement": _first_maxima(x, 1)[:, 0] == _first_maxima(y, 1)[:, 0]}


# -- what a pass cannot do without ---------------------------------------------------------
def work(case: dict) -> dict:
    t = case["tokens"]
    if case["op"] == "route":
        moved = t * case["experts"] * _BYTES[case["type"]] + t * case["top_k"] * (
            (8 if case["ids64"] else 4) + (2 if case["weights16"] else 4))
        return {"bytes": moved, "flops": 4 * t * case["experts"]}
    if case["op"] == "experts":
        h, i, e, k = (case[x] for x in ("hidden", "width", "experts", "top_k"))
        live = t - case["padding"]
        routed = e * (1 - (1 - min(k, e) / e) ** live)  # experts that some live row goes to
        moved = routed * 6 * i * h + t * (4 * h + k * ((8 if case["ids64"] else 4)
                                                       + (2 if case["weights16"] else 4)))
        return {"bytes": moved, "flops": 6 * live * k * i * h}
    entries = t * case["vocab"]
    if case["op"] == "logprobs":  # difference, exponential, two sums and a product
        return {"bytes": entries * _BYTES[case["type"]] + t * (16 + 8 * case["top"]),
                "flops": 5 * entries}
    return {"bytes": 2 * entries * _BYTES[case["type"]] + 5 * t, "flops": 10 * entries}
