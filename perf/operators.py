"""Operators around the mixers: the residual stream with its norms, and what is asked of the head's logits.

    add_rmsnorm               closes a block (norm behind it, gate, residual scale, sum) and opens the next one (norm, cast or
                              quantisation)
    token_logprobs            log probabilities of given tokens, entropy and the best alternatives, of logits
    scaled_mm_token_logprobs  the same of the head's int8 product, whose logits are never written

A case is one call.  Widths are those of the model configurations that the benchmark and the tests use, and generic ones; rows
are tokens: one for each sequence of a decoding batch, or all of a batch of prompts.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZES = {"fp16": 2, "bf16": 2, "fp32": 4, "int8": 1, "int8 rows": 1}
EPS = 1e-5
OUT_SCALE = 1.0 / 32                        # the static scale that a calibration would leave with the next projection


def _norm(name, rows, dim, x, residual, out, post=False, gate="none", act="none", scale="one", keep=True):
    case = {"op": "add_rmsnorm", "rows": rows, "dim": dim, "x": x, "residual": residual, "out": out, "post": post, "gate": gate, "act": act,
            "scale": scale, "keep": keep}
    return {"name": name, **case} if name else case


def _logits(name, rows, vocab, pad, x, top, masked=False):
    case = {"op": "token_logprobs", "rows": rows, "vocab": vocab, "pad": pad, "x": x, "top": top, "masked": masked}
    return {"name": name, **case} if name else case


def _head(name, rows, vocab, dim, row_scales, channel_scales, top):
    case = {"op": "scaled_mm_token_logprobs", "rows": rows, "vocab": vocab, "dim": dim, "row_scales": row_scales, "channel_scales": channel_scales, "top": top}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one user decoding with the smallest model: the residual sum and the norm in front of in_proj, int8 out; latency
        _norm("norm 1 x 768 to int8", 1, 768, "fp16", "fp32", "int8"),
        # a serving batch decoding, scale per token for the next product
        _norm("norm 64 x 2560 to int8 rows", 64, 2560, "fp16", "fp32", "int8 rows"),
        # the benchmark's prompts between two blocks of a float model: the plain sum and norm
        _norm("norm 16384 x 2560 to fp16", 16384, 2560, "fp16", "fp32", "fp16"),
        # a block with a norm behind it too, a gate per token and a residual scale per channel; ragged number of prompt tokens, odd width
        _norm("norms and gate 6131 x 4099 to bf16", 6131, 4099, "bf16", "bf16", "bf16", post=True, gate="rows", act="silu", scale="channels"),
        # one user decoding: the chosen token's log probability and some alternatives
        _logits("logprobs 1 x 50280 top 5", 1, 50280, 8, "fp16", 5),
        # a serving batch whose grammar masks a part of the vocabulary, as many alternatives as an API hands out
        _logits("logprobs 64 x 50280 top 20, masked", 64, 50280, 8, "fp16", 20, masked=True),
        # scoring the tokens of prompts, perplexity
        _logits("logprobs 4096 x 50280", 4096, 50280, 8, "bf16", 0),
        # a ragged number of tokens of a large vocabulary, fp32 logits, a few alternatives
        _logits("logprobs 509 x 256000 top 3", 509, 256000, 0, "fp32", 3),
        # one user decoding with the smallest model: the head's weights are the work
        _head("head 1 x 50280 x 768", 1, 50280, 768, True, True, 1),
        # a serving batch
        _head("head 64 x 50280 x 2560", 64, 50280, 2560, True, True, 1),
        # a prompt of odd length, one scale for all tokens
        _head("head 1021 x 50277 x 1536", 1021, 50277, 1536, False, False, 0),
        # the benchmark's prompts, scored
        _head("head 16384 x 50280 x 2560", 16384, 50280, 2560, True, True, 0),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(("norm", "logits", "head"))
    if kind == "norm":
        rows, x = _log_uniform(rng, 1, 16384), rng.choice(tuple(DTYPES))
        dim = rng.choice((768, 1024, 1536, 2048, 2560, 4096)) if rng.random() < 0.5 else _log_uniform(rng, 64, 8192)
        rows = min(rows, (1 << 26) // dim)
        gate = rng.choice(("none", "none", "rows", "channels"))
        return _norm(None, rows, dim, x, rng.choice(("none", x, "fp32")), rng.choice((x, "int8", "int8 rows")), rng.random() < 0.4, gate,
                     "none" if gate == "none" else rng.choice(("none", "sigmoid", "silu")), rng.choice(("one", "number", "channels")), rng.random() < 0.8)
    if kind == "logits":
        vocab = rng.choice((50280, 256000)) if rng.random() < 0.4 else _log_uniform(rng, 1000, 256000)
        rows = _log_uniform(rng, 1, max(1, (1 << 27) // vocab))
        return _logits(None, rows, vocab, rng.choice((0, 3, 8)), rng.choice(tuple(DTYPES)), rng.choice((0, 0, 1, 5, 20, 64)), rng.random() < 0.3)
    vocab = rng.choice((50280, 50277)) if rng.random() < 0.5 else _log_uniform(rng, 1000, 256000)
    dim = rng.choice((768, 1024, 1536, 2048, 2560, 4096)) if rng.random() < 0.6 else 16 * _log_uniform(rng, 8, 256)
    rows = _log_uniform(rng, 1, max(1, min(16384, (1 << 28) // vocab)))
    return _head(None, rows, vocab, dim, rng.random() < 0.5, rng.random() < 0.5, rng.choice((0, 1)))


# ---------------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device=dev)  # noqa: E731
    rows = case["rows"]
    if case["op"] == "add_rmsnorm":
        dim, x = case["dim"], DTYPES[case["x"]]
        loud = 1 + 9 * (torch.rand(dim, generator=g, device=dev) < 0.01)              # channels that stand out, as the stream has them
        return {"case": case,
                "x": (normal(rows, dim) * loud).to(x),
                "weight": (1 + 0.2 * normal(dim)).to(x),
                "post_weight": (1 + 0.2 * normal(dim)).to(x) if case["post"] else None,
                "residual": None if case["residual"] == "none" else (3 * normal(rows, dim) * loud).to(DTYPES[case["residual"]]),
                "gate": None if case["gate"] == "none" else (normal(rows, dim) if case["gate"] == "rows" else normal(dim)).to(x),
                "scale": {"one": 1.0, "number": 0.22}.get(case["scale"]) or (0.2 + 0.02 * normal(dim)).to(x),
                "static": torch.tensor(OUT_SCALE, dtype=torch.float16, device=dev)}
    vocab = case["vocab"]
    tokens = torch.randint(0, vocab, (rows,), generator=g, device=dev)
    tokens[torch.rand(rows, generator=g, device=dev) < 0.1] = -1                      # behind the end of a padded sequence
    if case["op"] == "token_logprobs":
        # (a few tokens far above the rest, frequent ones above rare ones)
        logits = torch.empty(rows, vocab + case["pad"], dtype=DTYPES[case["x"]], device=dev)
        rare = torch.arange(vocab, device=dev, dtype=torch.float32).add_(10).log_()[torch.randperm(vocab, generator=g, device=dev)]
        for r in range(0, rows, 1024):
            part = normal(min(1024, rows - r), vocab).mul_(2).sub_(rare)
            part += 6 * (torch.rand(part.shape, generator=g, device=dev) < 0.0001)
            if case["masked"]:
                part.masked_fill_(torch.rand(part.shape, generator=g, device=dev) < 0.4, float("-inf"))
            logits[r:r + 1024, :vocab] = part
        logits[:, vocab:] = 0
        return {"case": case, "logits": logits[:, :vocab], "tokens": tokens}
    dim, padded = case["dim"], (vocab + 15) // 16 * 16
    hidden = normal(rows, dim) * (1 + 4 * (torch.rand(dim, generator=g, device=dev) < 0.01))
    most = hidden.abs().amax(1, keepdim=True) if case["row_scales"] else hidden.abs().amax().view(1, 1)
    w = normal(padded, dim) * (1 + 0.3 * normal(padded, 1)).abs()
    w[vocab:] = 0
    w_most = w.abs().amax(1, keepdim=True).clamp(min=1e-5) if case["channel_scales"] else w.abs().amax().view(1, 1)
    return {"case": case, "tokens": tokens,
            "a": (hidden / most * 127).round().to(torch.int8),
            "b": (w / w_most * 127).round().to(torch.int8).t(),
            "a_scales": most / 127, "b_scales": w_most.t().contiguous() / 127 * (2.5 / math.sqrt(dim))}


# ---------------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    return RUNS[state["case"]["op"]](state)


def _rms(v):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)


def _add_rmsnorm(state):
    case = state["case"]
    quantized = case["out"].startswith("int8")
    if own:
        from quamba_amd import ops
        y, total, scales = ops.add_rmsnorm(
            state["x"], state["weight"], EPS, residual=state["residual"], post_weight=state["post_weight"], gate=state["gate"],
            gate_act=case["act"], residual_scale=state["scale"], prenorm=case["keep"],
            out_dtype=torch.int8 if quantized else DTYPES[case["out"]], out_scale=OUT_SCALE if case["out"] == "int8" else None)
    else:
        u = state["x"].float()
        if state["post_weight"] is not None:
            u = _rms(u) * state["post_weight"].float()
        if state["gate"] is not None:
            gate = state["gate"].float()
            u = u * (gate if case["act"] == "none" else torch.sigmoid(gate) if case["act"] == "sigmoid" else gate * torch.sigmoid(gate))
        total = u * state["scale"]
        if state["residual"] is not None:
            total = state["residual"].float() + total
        y, scales = _rms(total) * state["weight"].float(), None
        if case["out"] == "int8 rows":
            scales = y.abs().amax(-1).clamp(min=1e-5) / 127
            y = (y / scales[:, None]).round().clamp(-128, 127)
        elif case["out"] == "int8":
            y = (y / OUT_SCALE).round().clamp(-128, 127)
        else:
            y = y.to(DTYPES[case["out"]])
        total = total.to(state["x"].dtype if state["residual"] is None else state["residual"].dtype) if case["keep"] else None
    if quantized:
        # (the values that the codes stand for)
        y = (y * (state["static"] if scales is None else scales[:, None].half())).half()
    return {k: v for k, v in (("y", y), ("residual", total), ("scales", scales)) if v is not None}


def _of_logits(logits, tokens, top):
    """Log probabilities of `tokens` (0 for a negative one), entropies, the `top` best and their indices, of fp32 logits."""
    most = logits.amax(-1, keepdim=True)
    above = logits - most
    e = torch.exp(above)
    total = e.sum(-1, keepdim=True)
    entropy = torch.log(total) - (e * above.clamp(min=-200)).sum(-1, keepdim=True) / total
    best, at = _best(logits, top)
    norm = most + torch.log(total)
    logprobs = logits.gather(1, tokens.clamp(min=0)[:, None]) - norm
    return {"logprobs": torch.where(tokens < 0, 0.0, logprobs[:, 0]), "entropy": entropy[:, 0], "top_logprobs": best - norm, "top_tokens": at}


def _best(logits, top):
    # (of equal ones the lowest index first)
    if top == 1:
        best = logits.amax(-1, keepdim=True)
        return best, (logits == best).to(torch.uint8).argmax(-1, keepdim=True)
    best, at = torch.sort(logits, dim=-1, descending=True, stable=True) if top else (logits, torch.zeros_like(logits[:, :0], dtype=torch.int64))
    return best[:, :top], at[:, :top]


def _token_logprobs(state):
    if own:
        from quamba_amd import ops
        return ops.token_logprobs(state["logits"], state["tokens"], top=state["case"]["top"])._asdict()
    return _of_logits(state["logits"].float(), state["tokens"], state["case"]["top"])


def _scaled_mm_token_logprobs(state):
    case = state["case"]
    if own:
        from quamba_amd import ops
        return ops.scaled_mm_token_logprobs(state["a"], state["b"], state["a_scales"], state["b_scales"], state["tokens"], top=case["top"],
                                            vocab=case["vocab"])._asdict()
    # (whole numbers below 2^24, however the sum is ordered: the products of a row and a column that are not alike stay far below it)
    acc = state["a"].float() @ state["b"][:, :case["vocab"]].float()
    return _of_logits(state["a_scales"] * (state["b_scales"][:, :case["vocab"]] * acc), state["tokens"], case["top"])


RUNS = {"add_rmsnorm": _add_rmsnorm, "token_logprobs": _token_logprobs, "scaled_mm_token_logprobs": _scaled_mm_token_logprobs}


# ---------------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    rows = case["rows"]
    if case["op"] == "add_rmsnorm":
        n, x = rows * case["dim"], SIZES[case["x"]]
        residual = 0 if case["residual"] == "none" else SIZES[case["residual"]]
        kept = (residual or x) if case["keep"] else 0
        vectors = x * (1 + case["post"] + (case["gate"] == "channels") + (case["scale"] == "channels"))
        moved = n * (x + residual + kept + (x if case["gate"] == "rows" else 0) + SIZES[case["out"]])
        return {"bytes": moved + case["dim"] * vectors + (4 * rows if case["out"] == "int8 rows" else 0),
                "flops": n * (6 + 4 * case["post"] + 4 * (case["act"] != "none"))}
    answers = rows * (8 + 4 + 4 + 12 * case["top"])
    if case["op"] == "token_logprobs":
        return {"bytes": rows * case["vocab"] * SIZES[case["x"]] + answers, "flops": 6 * rows * case["vocab"]}
    scales = 4 * (rows if case["row_scales"] else 1) + 4 * (case["vocab"] if case["channel_scales"] else 1)
    return {"bytes": (rows + case["vocab"]) * case["dim"] + scales + answers, "flops": 2 * rows * case["vocab"] * case["dim"]}


# ---------------------------------------------------------------------------------------------------------------------
# The definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "add_rmsnorm":
        wide = {k: v.double() for k, v in state.items() if isinstance(v, torch.Tensor)}
        block = wide["x"]
        if "post_weight" in wide:
            block = block * wide["post_weight"] * (block.square().sum(-1, keepdim=True) / case["dim"] + EPS).pow(-0.5)
        if "gate" in wide:
            block = block * (1 if case["act"] == "sigmoid" else wide["gate"])
            block = block if case["act"] == "none" else block / (1 + torch.exp(-wide["gate"]))
        stream = block * wide.get("scale", state["scale"]) + wide.get("residual", 0.0)
        y = stream * wide["weight"] * (stream.square().sum(-1, keepdim=True) / case["dim"] + EPS).pow(-0.5)
        found = {}
        if case["out"] == "int8 rows":
            found["scales"] = y.abs().max(-1).values.clamp(min=1e-5) / 127
            y = (y / found["scales"][:, None]).round() * found["scales"][:, None]
        elif case["out"] == "int8":
            y = (y / OUT_SCALE).round().clamp(-128, 127) * OUT_SCALE
        if case["keep"]:
            found["residual"] = stream
        return {k: {"y": y, **found}[k] for k in ("y", "residual", "scales") if k in {"y": y, **found}}
    parts, n = [], max(1, (1 << 27) // case["vocab"])
    for r in range(0, case["rows"], n):
        if case["op"] == "token_logprobs":
            logits = state["logits"][r:r + n].double()
        else:
            codes = state["b"][:, :case["vocab"]].float()
            logits = (state["a"][r:r + n].float() @ codes).double()                   # (whole numbers, exact)
            logits *= state["a_scales"][r:r + n].double() if case["row_scales"] else state["a_scales"].double()
            logits *= state["b_scales"][:, :case["vocab"]].double() if case["channel_scales"] else state["b_scales"].double()
        logp = logits - torch.logsumexp(logits, -1, keepdim=True)
        t = state["tokens"][r:r + n]
        given = logp[torch.arange(len(t), device=t.device), t.clamp(min=0)]
        best = torch.topk(logp, case["top"], -1).values
        logp *= logp.exp()
        parts.append((given.masked_fill(t < 0, 0.0), -logp.nan_to_num_(nan=0.0).sum(-1), best))
    given, entropy, best = (torch.cat(p) for p in zip(*parts))
    # (which of two nearly equal values is the larger one is the arithmetic's own: no indices)
    return {"logprobs": given, "entropy": entropy, "top_logprobs": best, "top_tokens": None}
