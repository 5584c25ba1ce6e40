"""What is timed of the operators that serve a network of dense layers token by token.

Three operators, as one step of such a network runs them:

  norm    root-mean-square norm of a layer's input, with the residual's addition,
          stored in the input's type or in 8 bits (e4m3) with scales for each row
          or for each group of columns;
  w4      the dense layer act(X @ W + b) of few rows, W in 4 bits with a scale
          (and optionally a zero) for each group of K and each column;
  tokens  log probabilities of given tokens, the entropy, and the most probable
          tokens, over the rows of logits that the last layer gives.

`own` chooses between the plain form, in elementary torch operations, and the
calls of this repository's package.
"""
import math
import sys

import torch

own = False

F = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1}
E4M3_MAX = 448.0
EPS = 1e-6


def _package():
    if "ml-edsl_b200" not in sys.path:
        sys.path.insert(0, "ml-edsl_b200")
    from mlir_edsl import serving
    return serving


def listed():
    return [
        # one token of one sequence: the smallest call there is
        {"name": "norm_token", "op": "norm", "M": 1, "N": 4096, "type": "bf16", "residual": True,
         "quant": True, "group": 0},
        # odd rows in 32 bits, nothing fused around the norm
        {"name": "norm_ragged", "op": "norm", "M": 1000, "N": 1001, "type": "f32",
         "residual": False, "quant": False, "group": 0},
        # a batch of 512 rows that goes on into an 8-bit product with group scales
        {"name": "norm_batch", "op": "norm", "M": 512, "N": 4096, "type": "f16", "residual": True,
         "quant": True, "group": 128},
        # a long prompt: the largest, bound by memory
        {"name": "norm_prompt", "op": "norm", "M": 65536, "N": 4096, "type": "bf16",
         "residual": True, "quant": False, "group": 0},
        # one token through a square layer
        {"name": "w4_token", "op": "w4", "M": 1, "K": 4096, "N": 4096, "type": "bf16",
         "group": 128, "zeros": False, "bias": False, "act": 0, "out": "bf16"},
        # one token through the first layer of the 4096 -> 11008 -> 4096 network, in 32 bits
        {"name": "w4_up", "op": "w4", "M": 1, "K": 4096, "N": 11008, "type": "f32", "group": 128,
         "zeros": False, "bias": True, "act": 1, "out": "f32"},
        # sixteen tokens through its second layer, from 8-bit rows, weights with zeros
        {"name": "w4_down", "op": "w4", "M": 16, "K": 11008, "N": 4096, "type": "e4m3",
         "group": 64, "zeros": True, "bias": False, "act": 0, "out": "bf16"},
        # odd in every size, small groups
        {"name": "w4_ragged", "op": "w4", "M": 7, "K": 1001, "N": 999, "type": "f32", "group": 32,
         "zeros": True, "bias": True, "act": 0, "out": "f32"},
        # the largest batch that is still served from 4-bit weights
        {"name": "w4_batch", "op": "w4", "M": 64, "K": 8192, "N": 8192, "type": "f16",
         "group": 128, "zeros": False, "bias": True, "act": 1, "out": "f16"},
        # one token's choice among a large vocabulary
        {"name": "tokens_one", "op": "tokens", "T": 1, "V": 131072, "type": "bf16", "top": 20,
         "masked": 0.0},
        # a batch of steps over an odd vocabulary, a part of it not allowed
        {"name": "tokens_batch", "op": "tokens", "T": 512, "V": 32001, "type": "bf16", "top": 5,
         "masked": 0.25},
        # scores of a whole prompt in 32 bits: the largest
        {"name": "tokens_prompt", "op": "tokens", "T": 4096, "V": 65536, "type": "f32", "top": 0,
         "masked": 0.0},
    ]


def _spread(rng, low, high):
    """A whole number whose logarithm is spread evenly over [low, high]."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _size(rng, low, high):
    """As _spread; half of the sizes are multiples of 64."""
    n = _spread(rng, low, high)
    return max(low, n // 64 * 64) if rng.random() < 0.5 and n >= 64 else n


def draw(rng):
    op = rng.choice(["norm", "w4", "tokens"])
    if op == "norm":
        n = _size(rng, 64, 16384)
        quant = rng.random() < 0.6
        return {"op": op, "M": _spread(rng, 1, min(65536, 65536 * 2048 // n)), "N": n,
                "type": rng.choice(["f32", "bf16", "f16"]), "residual": rng.random() < 0.6,
                "quant": quant, "group": rng.choice([0, 32, 64, 128]) if quant else 0}
    if op == "w4":
        kind = rng.choice(["f32", "bf16", "f16", "e4m3"])
        k = _size(rng, 256, 16384)
        return {"op": op, "M": _spread(rng, 1, 64), "K": k,
                "N": _size(rng, 256, min(16384, 8192 * 8192 // k)), "type": kind,
                "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5,
                "bias": rng.random() < 0.5, "act": rng.choice([0, 1]),
                "out": rng.choice(["bf16", "f16"]) if kind == "e4m3" else kind}
    v = _size(rng, 1000, 200000)
    return {"op": op, "T": _spread(rng, 1, min(4096, 4096 * 32768 // v)), "V": v,
            "type": rng.choice(["f32", "bf16", "f16"]), "top": rng.choice([0, 1, 5, 20]),
            "masked": rng.choice([0.0, 0.0, 0.25])}


def _random(case, seed):
    """The inputs of a case, on the GPU, from its seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def whole(high, *shape, kind=torch.uint8):
        return torch.randint(0, high, shape, device="cuda", generator=g, dtype=kind)

    kind = F[case["type"]]
    if case["op"] == "norm":
        m, n = case["M"], case["N"]
        return {"x": normal(m, n).mul_(2.0).to(kind), "weight": normal(n).mul_(0.1).add_(1.0).to(kind),
                "residual": normal(m, n).mul_(3.0).to(kind) if case["residual"] else None}
    if case["op"] == "w4":
        m, k, n, group = case["M"], case["K"], case["N"], case["group"]
        parts = -(-k // group)
        held = torch.float32 if case["type"] == "f32" else F[case["out"]]
        s = {"codes": whole(16, k, n), "zeros": whole(16, parts, n) if case["zeros"] else None,
             "scales": normal(parts, n).mul_(0.2).exp_().mul_(0.3 / math.sqrt(k)).to(held),
             "bias": normal(n).to(held) if case["bias"] else None, "x_scales": None}
        x = normal(m, k)
        if case["type"] == "e4m3":
            s["x_scales"] = x.abs().amax(1, keepdim=True) / E4M3_MAX
            x = x / s["x_scales"]
        s["x"] = x.to(kind)
        return s
    t, v = case["T"], case["V"]
    logits = normal(t, v).mul_(2.5).to(kind)
    if case["masked"]:  # a vocabulary of which a part is not allowed, the same in every row
        shut = torch.rand(v, device="cuda", generator=g) < case["masked"]
        shut[:32] = False
        logits.masked_fill_(shut, -math.inf)
    tokens = whole(v, t, kind=torch.int32)
    if case["masked"]:
        tokens[1::8] = -1  # rows of a padded batch have no token
    return {"logits": logits, "tokens": tokens}


def prepare(case, seed):
    state = dict(case, **_random(case, seed))
    if own and case["op"] == "w4":  # a user's program keeps the packed weights
        state["packed"] = _package().pack_w4(state["codes"], state["scales"], state["zeros"],
                                             group=case["group"])
    if own:
        state["serving"] = _package()
    return state


def _groups(a, group, dim):
    """[..., n, ...] -> [..., parts, group, ...] along `dim`, filled up with zeros."""
    n = a.shape[dim]
    parts = -(-n // group)
    if parts * group != n:
        more = list(a.shape)
        more[dim] = parts * group - n
        a = torch.cat([a, a.new_zeros(more)], dim)
    return a.unflatten(dim, (parts, group))


def _norm(s):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * s["weight"].float()
    kind = s["x"].dtype
    if s["quant"]:
        n = y.shape[1]
        parts = _groups(y, s["group"] or n, 1)
        most = parts.abs().amax(2, keepdim=True)
        scales = torch.where(most > 0, most / E4M3_MAX, torch.ones_like(most))
        codes = (parts / scales).clamp(-E4M3_MAX, E4M3_MAX).flatten(1)[:, :n]
        out = [codes.to(torch.float8_e4m3fn), scales[:, :, 0]]
    else:
        out = [y.to(kind)]
    return out + [h.to(kind)] if s["residual"] is not None else out


def _w4(s):
    k = s["codes"].shape[0]
    codes = _groups(s["codes"].float(), s["group"], 0)
    zeros = s["zeros"].float()[:, None, :] if s["zeros"] is not None else 8.0
    w = ((codes - zeros) * s["scales"].float()[:, None, :]).flatten(0, 1)[:k]
    y = s["x"].float() @ w
    if s["x_scales"] is not None:
        y = y * s["x_scales"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return (torch.clamp(y, min=0) if s["act"] == 1 else y).to(F[s["out"]])


def _ordered(x):
    """Whole numbers in the order of the values of x, -0 as 0."""
    bits = (x + 0.0).view(torch.int32)
    return torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()


def _tokens(s):
    x = s["logits"].float()
    t = x - x.amax(1, keepdim=True)
    e = torch.exp(t)
    total = e.sum(1)
    log_total = torch.log(total)
    entropy = log_total - torch.where(e > 0, t * e, 0.0).sum(1) / total
    given = s["tokens"].long()
    at = torch.gather(t, 1, given.clamp(min=0)[:, None])[:, 0] - log_total
    out = [torch.where(given < 0, 0.0, at), entropy]
    if s["top"]:
        v = x.shape[1]
        # one whole number for each token: its logit's order, then the lowest index first
        keys = (_ordered(x) << 32) + (v - 1 - torch.arange(v, device=x.device))
        first = v - 1 - (torch.topk(keys, s["top"], dim=1).values & 0xFFFFFFFF)
        out += [torch.gather(t, 1, first) - log_total[:, None], first.int()]
    return out


def run(state):
    if own:
        serving = state["serving"]
        if state["op"] == "norm":
            out = serving.rms_norm(state["x"], state["weight"], residual=state["residual"], eps=EPS,
                                   quant="e4m3" if state["quant"] else None, group=state["group"])
            return list(out) if isinstance(out, tuple) else [out]
        if state["op"] == "w4":
            return serving.dense_w4(state["x"], state["packed"], state["bias"], act=state["act"],
                                    x_scales=state["x_scales"], out_dtype=F[state["out"]])
        return [v for v in serving.token_logprobs(state["logits"], state["tokens"],
                                                  top=state["top"]) if v is not None]
    return {"norm": _norm, "w4": _w4, "tokens": _tokens}[state["op"]](state)


def work(case):
    b = SIZE[case["type"]]
    if case["op"] == "norm":
        m, n = case["M"], case["N"]
        moved = m * n * b * (3 if case["residual"] else 1) + n * b
        if case["quant"]:
            moved += m * n + 4 * m * (-(-n // case["group"]) if case["group"] else 1)
        else:
            moved += m * n * b
        return {"bytes": moved, "flops": 5 * m * n}
    if case["op"] == "w4":
        m, k, n = case["M"], case["K"], case["N"]
        held = 4 if case["type"] == "f32" else SIZE[case["out"]]
        parts = -(-k // case["group"])
        moved = k * n / 2 + parts * n * (held + (0.5 if case["zeros"] else 0))
        moved += m * k * b + m * n * SIZE[case["out"]] + (n * held if case["bias"] else 0)
        return {"bytes": moved, "flops": 2 * m * k * n}
    t, v = case["T"], case["V"]
    return {"bytes": t * v * b + t * (12 + 8 * case["top"]), "flops": 6 * t * v}


def exact(case, seed):
    """The definitions, in 64 bits. Codes of 8 bits are given before their rounding."""
    s = _random(case, seed)
    if case["op"] == "norm":
        h = s["x"].double()
        if case["residual"]:
            h += s["residual"].double()
        rms = torch.sqrt(h.square().sum(1) / case["N"] + EPS)
        y = h / rms[:, None] * s["weight"].double()
        out = []
        if case["quant"]:
            step = case["group"] or case["N"]
            cut = [y[:, i:i + step] for i in range(0, case["N"], step)]
            scale = [c.abs().max(1, keepdim=True).values / 448 for c in cut]
            out += [torch.cat([c / a for c, a in zip(cut, scale)], 1), torch.cat(scale, 1)]
        else:
            out.append(y)
        return out + [h] if case["residual"] else out
    if case["op"] == "w4":
        k = case["K"]
        of = torch.arange(k, device="cuda") // case["group"]
        w = s["codes"].double()
        w -= s["zeros"].double()[of] if case["zeros"] else 8
        w *= s["scales"].double()[of]
        y = torch.einsum("mk,kn->mn", s["x"].double(), w)
        if s["x_scales"] is not None:
            y *= s["x_scales"].double()
        if case["bias"]:
            y += s["bias"].double()
        return y.relu() if case["act"] else y
    x = s["logits"].double()
    lse = torch.logsumexp(x, 1, keepdim=True)
    p = torch.exp(x - lse)
    entropy = -torch.special.xlogy(p, p).sum(1)
    given = s["tokens"].long()
    logs = torch.where(given < 0, torch.zeros_like(entropy),
                       x.gather(1, given.clamp(min=0)[:, None])[:, 0] - lse[:, 0])
    out = [logs, entropy]
    if case["top"]:
        out += [x.topk(case["top"], 1).values - lse, None]
    return out
