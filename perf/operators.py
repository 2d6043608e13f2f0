"""The operators of a decode step after its attention, as cases to measure.

Three operators that a serving step runs on a few rows at a time:

* ``w4_linear``: products with 4-bit weights and group scales,
* ``moe_decode``: a whole mixture-of-experts layer (router, experts, shared
  expert) for a few tokens, with bf16, block-FP8 or 4-bit experts,
* ``apply_logit_penalties``: penalties for repeated tokens, biases and grammar
  masks on the logits, in place.

``run`` computes them in their plain form from elementary torch operations in
32 bits, or, where ``own`` is set, through the package's entry points.
``exact`` restates the definitions in 64 bits.
"""

import math
import os
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FP8_BLOCK = 128

_ops = None


def _entry_points():
    global _ops
    if _ops is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "vllm-ernie_b200"))
        from vllm_ernie_b200 import ops

        _ops = ops
    return _ops


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # one token through the query up-projection (rank 1024 to 64 heads of
        # 128): the smallest call, where latency counts
        _linear("w4_query_up_1", tokens=1, k=1024, n=8192, group=64, zeros=False, dtype="bf16"),
        # one request's three draft tokens through the gated output projection,
        # asymmetric checkpoint with the finest groups
        _linear("w4_output_3", tokens=3, k=8192, n=4096, group=32, zeros=True, dtype="fp16"),
        # a small batch through the output gate
        _linear("w4_gate_16", tokens=16, k=4096, n=8192, group=128, zeros=False, dtype="bf16"),
        # the vocabulary projection of a step with 8 rows: the largest product,
        # an odd vocabulary
        _linear("w4_vocabulary_8", tokens=8, k=4096, n=129281, group=128, zeros=True, dtype="bf16"),
        # a small layer with 4-bit experts, two tokens: latency
        _moe("moe_small_2", tokens=2, pad=0, experts=32, top_k=4, hidden=1024, inner=512, shared=0, weights="w4",
             group=64, score="sigmoid", bias=True, renormalize=True, scale=1.0, router="fp32"),
        # one token, bf16 experts
        _moe("moe_bf16_1", tokens=1, pad=0, experts=64, top_k=6, hidden=4096, inner=1024, shared=0, weights="bf16",
             group=0, score="softmax", bias=False, renormalize=True, scale=1.0, router="bf16"),
        # odd sizes everywhere, weights of the selected experts not renormalised
        _moe("moe_odd_13", tokens=13, pad=2, experts=60, top_k=5, hidden=2080, inner=736, shared=1472, weights="bf16",
             group=0, score="softmax", bias=False, renormalize=False, scale=1.0, router="bf16"),
        # eight tokens, block-FP8 experts and a shared expert
        _moe("moe_fp8_8", tokens=8, pad=0, experts=128, top_k=8, hidden=4096, inner=1024, shared=1024, weights="fp8",
             group=0, score="sigmoid", bias=True, renormalize=True, scale=2.5, router="fp32"),
        # the largest: 64 rows of a padded graph batch, nearly every expert
        # read, 4-bit experts
        _moe("moe_w4_64", tokens=64, pad=5, experts=128, top_k=8, hidden=4096, inner=1024, shared=1024, weights="w4",
             group=128, score="sigmoid", bias=True, renormalize=True, scale=2.5, router="fp32"),
        # one request without bias or mask, short history
        _logits("logits_1", rows=1, vocab=32000, history=300, bias=0, mask=False, dtype="fp32"),
        # a batch of 64 requests under a grammar, with biases, histories of up
        # to 8192 tokens
        _logits("logits_grammar_64", rows=64, vocab=129280, history=8192, bias=32, mask=True, dtype="fp32"),
        # 192 rows with long histories, an odd vocabulary, bf16 logits
        _logits("logits_long_192", rows=192, vocab=151937, history=32768, bias=0, mask=False, dtype="bf16"),
    ]


def _linear(name, **c):
    return {"name": name, "op": "w4_linear", **c}


def _moe(name, **c):
    return {"name": name, "op": "moe", **c}


def _logits(name, **c):
    return {"name": name, "op": "logits", **c}


def _spread(rng, low, high, step=1):
    """A multiple of ``step``, spread over the logarithm of [low, high]."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high))) / step)) * step
    return min(max(v, (low + step - 1) // step * step), high // step * step)


def draw(rng):
    op = rng.choice(("w4_linear", "moe", "moe", "logits"))
    if op == "w4_linear":
        group = rng.choice((32, 64, 128))
        k = _spread(rng, 512, 8192, group)
        n = _spread(rng, 65, min(129281, 129281 * 4096 // k))
        return {"op": op, "tokens": _spread(rng, 1, 32), "k": k + group if k == 3072 else k, "n": n + 1 if n == 3072 else n,
                "group": group, "zeros": rng.random() < 0.5, "dtype": rng.choice(("bf16", "fp16"))}
    if op == "moe":
        weights = rng.choice(("bf16", "fp8", "w4"))
        group = rng.choice((32, 64, 128)) if weights == "w4" else 0
        step = max(32, group)
        hidden = _spread(rng, 512, 4096, step)
        inner = _spread(rng, 128, 1024, step)
        experts = _spread(rng, 8, 128)
        tokens = _spread(rng, 1, 64)
        if weights != "w4":  # as many bytes as the largest listed layer reads
            experts = min(experts, int(128 * 4096 * 1024 * 0.5 / (hidden * inner * (2 if weights == "bf16" else 1))))
        return {"op": op, "tokens": tokens, "pad": rng.randrange(0, (tokens + 7) // 8 + 1) if tokens > 1 else 0,
                "experts": experts, "top_k": rng.randint(1, 8), "hidden": hidden + step if hidden == 3072 else hidden,
                "inner": inner, "shared": inner * rng.choice((0, 0, 1)), "weights": weights, "group": group,
                "score": rng.choice(("softmax", "sigmoid")), "bias": rng.random() < 0.5,
                "renormalize": rng.random() < 0.5, "scale": rng.choice((1.0, 2.5)), "router": rng.choice(("bf16", "fp32"))}
    vocab, history = _spread(rng, 1000, 151937), _spread(rng, 16, 32768)
    return {"op": op, "rows": _spread(rng, 1, 192), "vocab": vocab + 1 if vocab == 3072 else vocab,
            "history": history + 1 if history == 3072 else history, "bias": rng.choice((0, 0, _spread(rng, 1, 300))),
            "mask": rng.random() < 0.5, "dtype": rng.choice(("fp32", "bf16", "fp16"))}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _codes(shape, gen):
    return torch.randint(0, 256, shape, generator=gen, device=DEV, dtype=torch.uint8)


def _scales(rows, k, group, dtype, gen):
    """Group scales that give a weight about 1 / sqrt(k) in size."""
    s = torch.rand((*rows, k // group), generator=gen, device=DEV)
    return ((0.5 + s) / (4.6 * math.sqrt(k))).to(dtype)


def _weights(c, rows, k, gen):
    """One weight tensor [*rows, k] of the case's format: (data, scales)."""
    if c["weights"] == "w4":
        return _codes((*rows, k // 2), gen), _scales(rows, k, c["group"], torch.bfloat16, gen)
    w = torch.randn((*rows, k), generator=gen, device=DEV, dtype=torch.bfloat16)
    if c["weights"] == "bf16":
        return w.mul_(1 / math.sqrt(k)), None
    blocks = (*rows[:-1], -(-rows[-1] // FP8_BLOCK), -(-k // FP8_BLOCK))
    s = torch.exp2(torch.randint(-2, 1, blocks, generator=gen, device=DEV).float()) / (60 * math.sqrt(k))
    return w.mul_(60).clamp_(-448, 448).to(torch.float8_e4m3fn), s


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if c["op"] == "w4_linear":
        dtype = TYPES[c["dtype"]]
        s = {"x": torch.randn((c["tokens"], c["k"]), generator=gen, device=DEV).to(dtype),
             "q": _codes((c["n"], c["k"] // 2), gen), "s": _scales((c["n"],), c["k"], c["group"], dtype, gen), "z": None}
        if c["zeros"]:
            s["z"] = torch.randint(5, 12, (c["n"], c["k"] // c["group"]), generator=gen, device=DEV, dtype=torch.uint8)
    elif c["op"] == "moe":
        h, i, e, t = c["hidden"], c["inner"], c["experts"], c["tokens"]
        s = {"x": torch.randn((t, h), generator=gen, device=DEV).to(torch.bfloat16),
             "router": (torch.randn((e, h), generator=gen, device=DEV) * (1.5 / math.sqrt(h))).to(TYPES[c["router"]]),
             "bias": torch.randn(e, generator=gen, device=DEV) * 0.1 if c["bias"] else None, "mask": None,
             "w13": _weights(c, (e, 2 * i), h, gen), "w2": _weights(c, (e, h), i, gen), "shared": None}
        if c["shared"]:
            s["shared"] = (_weights(c, (2 * c["shared"],), h, gen), _weights(c, (h,), c["shared"], gen))
        if c["pad"]:
            s["mask"] = torch.arange(t, device=DEV) < t - c["pad"]
    else:
        r, v, n = c["rows"], c["vocab"], c["history"]
        uniform = lambda low, high: low + (high - low) * torch.rand(r, generator=gen, device=DEV)  # noqa: E731
        # texts repeat few words often: token ids crowd at the low end
        ids = (torch.rand((r, n), generator=gen, device=DEV) ** 3 * v).to(torch.int32).clamp_(max=v - 1)
        lens = (uniform(0.25, 1.0) * n).to(torch.int32)
        s = {"logits": (torch.randn((r, v), generator=gen, device=DEV) * 3).to(TYPES[c["dtype"]]), "ids": ids,
             "prompt_lens": (lens * uniform(0.0, 1.0)).to(torch.int32), "seq_lens": lens, "repetition": uniform(0.9, 1.4),
             "frequency": uniform(-0.2, 0.5), "presence": uniform(-0.2, 0.5), "bias_ids": None, "bias_values": None, "allowed": None}
        if c["bias"]:
            first = torch.randint(0, v, (r, 1), generator=gen, device=DEV)
            step = max(1, v // (c["bias"] + 1))
            at = (first + step * torch.arange(c["bias"], device=DEV)) % v  # no id twice in a row
            used = torch.arange(c["bias"], device=DEV) < (uniform(0.3, 1.0) * c["bias"]).ceil().unsqueeze(1)
            s["bias_ids"] = torch.where(used, at, -1).to(torch.int32)
            s["bias_values"] = torch.randn((r, c["bias"]), generator=gen, device=DEV) * 2
        if c["mask"]:
            words = torch.randint(-2 ** 31, 2 ** 31, (r, -(-v // 32)), generator=gen, device=DEV)
            # a grammar allows few tokens in most places and nearly all in others
            dense = torch.rand((r, 1), generator=gen, device=DEV) < 0.3
            other = torch.randint(-2 ** 31, 2 ** 31, words.shape, generator=gen, device=DEV)
            third = torch.randint(-2 ** 31, 2 ** 31, words.shape, generator=gen, device=DEV)
            s["allowed"] = torch.where(dense, words | other | third, words & other & third).to(torch.int32)
    return {"case": c, **s}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(state):
    return {"w4_linear": _run_linear, "moe": _run_moe, "logits": _run_logits}[state["case"]["op"]](state)


def _unpack4(q, s, z):
    """[..., K / 2] codes (low nibble first) times group scales, in 32 bits."""
    codes = torch.stack((q & 15, q >> 4), -1).flatten(-2).float()
    groups = codes.unflatten(-1, (s.shape[-1], -1))
    return ((groups - (8.0 if z is None else z.float().unsqueeze(-1))) * s.float().unsqueeze(-1)).flatten(-2)


def _run_linear(s):
    if own:
        return _entry_points().w4_linear(s["x"], s["q"], s["s"], zeros=s["z"])
    return (s["x"].float() @ _unpack4(s["q"], s["s"], s["z"]).T).to(s["x"].dtype)


def _dense(w):
    data, s = w
    if data.dtype == torch.uint8:
        return _unpack4(data, s, None)
    if s is None:
        return data.float()
    full = s.repeat_interleave(FP8_BLOCK, -2).repeat_interleave(FP8_BLOCK, -1)
    return data.float() * full[..., : data.shape[-2], : data.shape[-1]]


def _gated(x, w13):
    """silu(x W1^T) * (x W3^T) for w13 = [W1; W3], all 32 bits."""
    gate, up = (x @ w13.transpose(-1, -2)).chunk(2, -1)
    return gate / (1 + torch.exp(-gate)) * up


def _run_moe(s):
    c = s["case"]
    if own:
        ops = _entry_points()
        shared = None
        if s["shared"] is not None:
            (a, sa), (b, sb) = s["shared"]
            shared = ops.MoEWeights(a, b, sa, sb)
        experts = ops.MoEWeights(s["w13"][0], s["w2"][0], s["w13"][1], s["w2"][1])
        return ops.moe_decode(s["x"], s["router"], experts, c["top_k"], score=c["score"], router_bias=s["bias"],
                              renormalize=c["renormalize"], routed_scale=c["scale"], shared=shared, token_mask=s["mask"])
    x = s["x"].float()
    if s["mask"] is not None:
        x = torch.where(s["mask"].unsqueeze(1), x, 0.0)
    logits = x @ s["router"].float().T
    if c["score"] == "softmax":
        score = torch.exp(logits - logits.amax(1, keepdim=True))
        score = score / score.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-logits))
    by = score if s["bias"] is None else score + s["bias"]
    ids = torch.sort(by, dim=1, descending=True, stable=True).indices[:, : c["top_k"]]
    weight = torch.gather(score, 1, ids)
    if c["renormalize"]:
        weight = weight / weight.sum(1, keepdim=True)
    weight = weight * c["scale"]
    if ids.numel() <= c["experts"]:  # few pairs: read the chosen experts only
        pairs = ids.flatten()
        pick = lambda w: _dense(tuple(None if v is None else v[pairs] for v in w))  # noqa: E731
        rows = x.repeat_interleave(c["top_k"], 0).unsqueeze(1)
        y = _gated(rows, pick(s["w13"])) * weight.reshape(-1, 1, 1)
        y = (y @ pick(s["w2"]).transpose(1, 2)).unflatten(0, ids.shape).sum((1, 2))
    else:
        dense = torch.zeros_like(logits).scatter_(1, ids, weight)
        y = _gated(x.unsqueeze(0), _dense(s["w13"])) * dense.T.unsqueeze(-1)
        y = (y @ _dense(s["w2"]).transpose(1, 2)).sum(0)
    if s["shared"] is not None:
        y = y + _gated(x, _dense(s["shared"][0])) @ _dense(s["shared"][1]).T
    if s["mask"] is not None:
        y = torch.where(s["mask"].unsqueeze(1), y, 0.0)
    return y.to(s["x"].dtype)


def _run_logits(s):
    if own:
        return _entry_points().apply_logit_penalties(
            s["logits"], s["ids"], s["prompt_lens"], s["seq_lens"], repetition=s["repetition"], frequency=s["frequency"],
            presence=s["presence"], bias_ids=s["bias_ids"], bias_values=s["bias_values"], allowed_bitmask=s["allowed"])
    x, ids = s["logits"].float(), s["ids"].long()
    at = torch.arange(ids.shape[1], device=x.device)
    prompt = at < s["prompt_lens"].unsqueeze(1)
    answer = (at < s["seq_lens"].unsqueeze(1)) & ~prompt
    count = torch.zeros_like(x).scatter_add_(1, ids, answer.float())
    seen = torch.zeros_like(x).scatter_add_(1, ids, prompt.float()) + count > 0
    if s["bias_ids"] is not None:
        used = s["bias_ids"] >= 0
        x.scatter_add_(1, s["bias_ids"].clamp(min=0).long(), torch.where(used, s["bias_values"], 0.0))
    r = s["repetition"].unsqueeze(1)
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"].unsqueeze(1) * count - s["presence"].unsqueeze(1) * (count > 0).float()
    if s["allowed"] is not None:
        v = torch.arange(x.shape[1], device=x.device)
        x = torch.where((s["allowed"][:, v // 32] >> (v % 32)) & 1 > 0, x, -math.inf)
    return s["logits"].copy_(x)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def _weight_bytes(c, rows, k):
    if c["weights"] == "w4":
        return rows * k / 2 + rows * k / c["group"] * 2
    return rows * k * (2 if c["weights"] == "bf16" else 1)


def work(case):
    c = case
    if c["op"] == "w4_linear":
        t, k, n = c["tokens"], c["k"], c["n"]
        groups = n * k // c["group"]
        return {"bytes": n * k // 2 + groups * (3 if c["zeros"] else 2) + 2 * t * (k + n), "flops": 2 * t * k * n}
    if c["op"] == "moe":
        t, h, i, e = c["tokens"] - c["pad"], c["hidden"], c["inner"], c["experts"]
        # experts that at least one token chooses, if all are as likely
        read = e * (1 - (1 - min(c["top_k"], e) / e) ** t)
        size = _weight_bytes(c, 2 * i, h) + _weight_bytes(c, h, i)
        shared = _weight_bytes(c, 2 * c["shared"], h) + _weight_bytes(c, h, c["shared"]) if c["shared"] else 0
        return {"bytes": read * size + shared + e * h * (4 if c["router"] == "fp32" else 2) + 4 * c["tokens"] * h,
                "flops": 2 * t * h * (e + 3 * i * min(c["top_k"], e) + 3 * c["shared"])}
    # in place: the history, the mask, the biases, and of the logits those
    # that change: one distinct token for about two in the history, and every
    # masked one (about a third of the rows mask 1 in 8, the others 7 in 8)
    size = 4 if c["dtype"] == "fp32" else 2
    tokens = 0.625 * c["history"]
    touched = min(0.5 * tokens + c["bias"], c["vocab"])
    each = 4 * tokens + 2 * size * touched + 8 * c["bias"]
    if c["mask"]:
        each += c["vocab"] / 8 + size * 0.65 * c["vocab"]
    return {"bytes": c["rows"] * each, "flops": c["rows"] * 6 * touched}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def _exact_weight(w, group_zero=None):
    data, s = w
    if data.dtype == torch.uint8:
        n, half = data.shape
        k = 2 * half
        v = torch.empty((n, k), dtype=torch.float64, device=DEV)
        v[:, 0::2], v[:, 1::2] = (data % 16).double(), torch.div(data, 16, rounding_mode="floor").double()
        group = torch.arange(k, device=DEV) // (k // s.shape[1])
        zero = 8.0 if group_zero is None else group_zero.double()[:, group]
        return (v - zero) * s.double()[:, group]
    if s is None:
        return data.double()
    row, col = (torch.arange(m, device=DEV) // FP8_BLOCK for m in data.shape)
    return data.double() * s.double()[row][:, col]


def exact(case, seed):
    s = prepare(case, seed)
    return {"w4_linear": _exact_linear, "moe": _exact_moe, "logits": _exact_logits}[case["op"]](case, s)


def _exact_linear(c, s):
    x, step = s["x"].double(), 16384
    parts = [x @ _exact_weight((s["q"][a:a + step], s["s"][a:a + step]), None if s["z"] is None else s["z"][a:a + step]).T
             for a in range(0, c["n"], step)]
    return torch.cat(parts, 1)


def _exact_expert(x, w13, w2):
    both = x @ _exact_weight(w13).T
    half = both.shape[1] // 2
    return (both[:, :half] * torch.sigmoid(both[:, :half]) * both[:, half:]) @ _exact_weight(w2).T


def _exact_moe(c, s):
    x = s["x"].double()
    logits = x @ s["router"].double().T
    score = torch.softmax(logits, 1) if c["score"] == "softmax" else torch.sigmoid(logits)
    by = (score if s["bias"] is None else score + s["bias"].double()).cpu().tolist()
    y = torch.zeros_like(x)
    chosen = [sorted(range(c["experts"]), key=lambda e, row=row: (-row[e], e))[: c["top_k"]] for row in by[: c["tokens"] - c["pad"]]]
    for e in range(c["experts"]):
        rows = [t for t, ids in enumerate(chosen) if e in ids]
        if not rows:
            continue
        weight = torch.stack([score[t, e] / (sum(score[t, j] for j in chosen[t]) if c["renormalize"] else 1.0) for t in rows])
        part = _exact_expert(x[rows], *(tuple(None if v is None else v[e] for v in s[w]) for w in ("w13", "w2")))
        y[rows] += part * (weight * c["scale"]).unsqueeze(1)
    if s["shared"] is not None:
        y += _exact_expert(x, *s["shared"])
    y[c["tokens"] - c["pad"]:] = 0
    return y


def _exact_logits(c, s):
    x = s["logits"].double()
    for r in range(c["rows"]):
        p, n = int(s["prompt_lens"][r]), int(s["seq_lens"][r])
        ids = s["ids"][r].long()
        if s["bias_ids"] is not None:
            used = s["bias_ids"][r] >= 0
            x[r, s["bias_ids"][r][used].long()] += s["bias_values"][r][used].double()
        count = torch.bincount(ids[p:n], minlength=c["vocab"]).double()
        seen = torch.unique(ids[:n])
        by = s["repetition"][r].double()
        v = x[r, seen]
        x[r, seen] = torch.where(v > 0, v / by, v * by)
        x[r] -= s["frequency"][r].double() * count
        x[r] -= s["presence"][r].double() * (count > 0)
        if s["allowed"] is not None:
            bits = torch.arange(32, device=DEV)
            ok = (((s["allowed"][r].unsqueeze(1) >> bits) & 1) == 1).reshape(-1)[: c["vocab"]]
            x[r][~ok] = -math.inf
    return x
