"""Performance cases of what a net that reads tokens computes behind its input: gated layers, the log probabilities of its
answers, and products with 4-bit weights.

A gated layer is a hidden layer of two projections; training needs its gradient.  A policy gradient needs the log
probabilities of the actions or tokens that were taken, with the entropy and the likeliest alternatives, and their gradient.
A net that answers for few states reads every weight once: in 4 bits, with a scale per group.  ``listed`` names sizes of
real use, ``draw`` takes others from the same ranges.

``run`` computes an operator in its plain form, elementary torch operations in 32 bits, or, where ``own`` is true,
through this package.  ``exact`` computes the same from the definition in 64 bits.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ITEM = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # The head of one decision: 256 states, ten actions, some of them legal, f32 logits.  A latency-bound call.
        {"name": "log_probs_256_states", "kind": "log_probs", "rows": 256, "cols": 10, "type": "f32", "mask": True, "top": 2, "index": "i32", "scale": 1.0},
        # A batch of 4096 positions over a large vocabulary whose rows start anywhere, with eight alternatives.
        {"name": "log_probs_4096x50001", "kind": "log_probs", "rows": 4096, "cols": 50001, "type": "bf16", "mask": False, "top": 8, "index": "i64", "scale": 1.0},
        # Answers for eight sequences at a temperature: few long rows, many alternatives.
        {"name": "log_probs_8x131072", "kind": "log_probs", "rows": 8, "cols": 131072, "type": "f16", "mask": False, "top": 32, "index": "i32", "scale": 1.25},
        # A policy gradient over the benchmark's batch of 65536 states.
        {"name": "log_probs_grad_65536_states", "kind": "log_probs_grad", "rows": 65536, "cols": 10, "type": "f32", "mask": True, "index": "i32", "scale": 1.0},
        # The gradient of the large vocabulary.
        {"name": "log_probs_grad_4096x50001", "kind": "log_probs_grad", "rows": 4096, "cols": 50001, "type": "bf16", "mask": False, "index": "i64", "scale": 1.0},
        # A gated layer for a single state.
        {"name": "gated_1", "kind": "gated", "m": 1, "f": 4096, "k": 1024, "type": "bf16", "act": "silu", "saved": False},
        # Sizes that fit no tile (those of the ragged products), for training.
        {"name": "gated_ragged", "kind": "gated", "m": 4001, "f": 3000, "k": 1000, "type": "f16", "act": "gelu", "saved": True},
        # A training batch behind a 1024-wide layer.
        {"name": "gated_16384", "kind": "gated", "m": 16384, "f": 4096, "k": 1024, "type": "bf16", "act": "silu", "saved": True},
        # The gradients of both.
        {"name": "gated_grad_ragged", "kind": "gated_grad", "m": 4001, "f": 3000, "k": 1000, "type": "f16", "act": "gelu"},
        {"name": "gated_grad_8192", "kind": "gated_grad", "m": 8192, "f": 4096, "k": 1024, "type": "bf16", "act": "silu"},
        # A dense layer for a single state with weights in 4 bits.
        {"name": "int4_1", "kind": "int4", "m": 1, "n": 4096, "k": 4096, "group": 128, "type": "bf16"},
        # Sixteen states at once, a larger layer and smaller groups.
        {"name": "int4_16", "kind": "int4", "m": 16, "n": 8192, "k": 8192, "group": 64, "type": "f16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["log_probs", "log_probs", "log_probs_grad", "gated", "gated", "gated_grad", "int4", "int4"])
    if kind.startswith("log_probs"):
        # Actions of a policy, or a vocabulary.
        cols = rng.choice([_log(rng, 2, 256), _log(rng, 256, 150000)])
        case = {"kind": kind, "rows": _log(rng, 1, min(1 << 18, (200 << 20) // cols)), "cols": cols, "type": rng.choice(["f32", "bf16", "f16"]),
                "mask": cols <= 1024 and rng.random() < 0.5, "index": rng.choice(["i32", "i64"]), "scale": rng.choice([1.0, 0.8, 1.25])}
        if case["type"] == "f32":
            case["rows"] = (case["rows"] + 1) // 2
        if kind == "log_probs":
            case["top"] = min(2 if case["mask"] else cols, rng.choice([0, 1, _log(rng, 1, 32)]))
        return case
    if kind == "int4":
        n, k = _log(rng, 64, 16384), 8 * _log(rng, 8, 2048)
        return {"kind": kind, "m": rng.choice([1, _log(rng, 1, 64)]), "n": n, "k": k, "group": rng.choice([32, 64, 128]), "type": rng.choice(["bf16", "f16"])}
    f, k = 8 * _log(rng, 8, 1024), 8 * _log(rng, 8, 512)
    most = 16384 * 4096 * 1024 if kind == "gated" else 8192 * 4096 * 1024
    case = {"kind": kind, "m": _log(rng, 1, min(16384, most // (f * k))), "f": f, "k": k, "type": rng.choice(["bf16", "f16"]),
            "act": rng.choice(["silu", "gelu", "relu"])}
    return {**case, "saved": rng.random() < 0.5} if kind == "gated" else case


# -- inputs ----------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _prepare_rows(case, g, s):
    rows, cols = case["rows"], case["cols"]
    s["logits"] = _normal(g, (rows, cols), TYPES[case["type"]], std=2.0)
    s["mask"] = None
    if case["mask"]:
        # At least two legal actions in every row, the others legal with one chance in two.
        order = torch.rand((rows, cols), generator=g, device="cuda")
        keep = (order <= torch.topk(order, 2, 1, largest=False).values[:, 1:]) | (torch.rand((rows, cols), generator=g, device="cuda") < 0.5)
        s["mask"] = keep.to(torch.uint8)
    # The tokens that were taken: drawn from the distribution.
    x = s["logits"].float() * case["scale"]
    if case["mask"]:
        x = torch.where(s["mask"] != 0, x, -math.inf)
    x -= torch.log(-torch.log(torch.rand((rows, cols), generator=g, device="cuda").clamp_(1e-20, 1.0 - 1e-7)))
    s["tokens"] = x.argmax(1).to(torch.int64 if case["index"] == "i64" else torch.int32)
    s["entropy"] = torch.empty(rows, dtype=torch.float32, device="cuda")
    s["stats"] = torch.empty((rows, 2), dtype=torch.float32, device="cuda")


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    s = {"case": case}
    if kind == "log_probs":
        _prepare_rows(case, g, s)
        s["out"] = torch.empty(case["rows"], dtype=torch.float32, device="cuda")
        if case["top"]:
            s["top"] = torch.empty((case["rows"], case["top"]), dtype=torch.float32, device="cuda")
            s["top_tokens"] = torch.empty((case["rows"], case["top"]), dtype=torch.int32, device="cuda")
    elif kind == "log_probs_grad":
        _prepare_rows(case, g, s)
        # What the forward pass left, and the gradients of a loss: advantages and the weight of the entropy.
        d, top, e, total = _scaled(s)
        s["stats"].copy_(torch.stack([top[:, 0], torch.log(total[:, 0])], 1))
        s["entropy"].copy_(torch.log(total[:, 0]) - (e * d.clamp_min(-1e30)).sum(1) / total[:, 0])
        s["dout"] = _normal(g, (case["rows"],), std=1.0 / case["rows"])
        s["dentropy"] = _normal(g, (case["rows"],), std=0.1 / case["rows"])
        s["dlogits"] = torch.empty_like(s["logits"])
    elif kind in ("gated", "gated_grad"):
        m, f, k, dtype = case["m"], case["f"], case["k"], TYPES[case["type"]]
        s["x"], s["w"] = _normal(g, (m, k), dtype), _normal(g, (2 * f, k), dtype, std=k ** -0.5)
        if kind == "gated":
            s["out"] = torch.empty((m, f), dtype=dtype, device="cuda")
            s["saved"] = torch.empty((m, 2 * f), dtype=dtype, device="cuda") if case["saved"] else None
        else:
            s["saved"] = (s["x"].float() @ s["w"].float().t()).to(dtype)
            s["dout"] = _normal(g, (m, f), dtype)
            s["dx"], s["dw"] = torch.empty_like(s["x"]), torch.empty_like(s["w"])
    else:
        m, n, k, group, dtype = case["m"], case["n"], case["k"], case["group"], TYPES[case["type"]]
        s["a"] = _normal(g, (m, k), dtype)
        s["bias"] = _normal(g, (n,), std=0.1)
        # Weights as they are kept: codes 0 .. 15 of (w / scale + 8), two in a byte, and a scale per group and row.
        blocks = torch.nn.functional.pad(_normal(g, (n, k), std=k ** -0.5), (0, -k % group)).view(n, -1, group)
        s["scales"] = (blocks.abs().amax(2) / 7.0).to(dtype).t().contiguous()
        codes = torch.round(blocks / s["scales"].t().float()[:, :, None]).clamp_(-8, 7) + 8
        codes = codes.view(n, -1)[:, :k].to(torch.uint8)
        s["codes"] = (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous()
        s["out"] = torch.empty((m, n), dtype=dtype, device="cuda")
    return s


# -- one pass --------------------------------------------------------------------------------------------
_package = []


def _sb():
    if not _package:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "spiral-s-ml-library_b200")
        if at not in sys.path:
            sys.path.insert(0, at)
        import spiral_b200
        _package.append(spiral_b200)
    return _package[0]


def run(s):
    return (_own if own else _plain)[s["case"]["kind"]](s)


def _own_log_probs(s):
    _sb().primitives.log_probs(s["logits"], s["tokens"], s["out"], entropy=s["entropy"], stats=s["stats"], top=s.get("top"),
                               top_tokens=s.get("top_tokens"), mask=s["mask"], scale=s["case"]["scale"])
    return {k: s[k] for k in ("out", "entropy", "stats") + (("top", "top_tokens") if s["case"]["top"] else ())}


def _own_log_probs_grad(s):
    return _sb().primitives.log_probs_grad(s["logits"], s["tokens"], s["stats"], s["dlogits"], dout=s["dout"], dentropy=s["dentropy"],
                                           entropy=s["entropy"], mask=s["mask"], scale=s["case"]["scale"])


def _own_gated(s):
    _sb().gated(s["x"], s["w"], s["out"], activation=s["case"]["act"], saved=s["saved"])
    return (s["out"], s["saved"]) if s["case"]["saved"] else s["out"]


def _own_gated_grad(s):
    _sb().gated_grad(s["dout"], s["x"], s["w"], s["saved"], dx=s["dx"], dw=s["dw"], activation=s["case"]["act"])
    return s["dx"], s["dw"]


def _own_int4(s):
    return _sb().matmul_int4(s["a"], s["codes"], s["scales"], s["out"], group=s["case"]["group"], epilogue=("bias", "relu"), bias=s["bias"])


_own = {"log_probs": _own_log_probs, "log_probs_grad": _own_log_probs_grad, "gated": _own_gated, "gated_grad": _own_gated_grad, "int4": _own_int4}


def _scaled(s):
    """Scaled distances from the row's largest logit, that logit, exp of the distances and their sum."""
    x = s["logits"].float()
    if s["mask"] is not None:
        x = torch.where(s["mask"] != 0, x, -math.inf)
    top = x.amax(1, keepdim=True)
    d = (x - top) * s["case"]["scale"]
    e = torch.exp(d)
    return d, top, e, e.sum(1, keepdim=True)


def _plain_log_probs(s):
    d, top, e, total = _scaled(s)
    log_total = torch.log(total)
    at = s["tokens"].long()[:, None]
    entropy = log_total[:, 0] - (e * d.clamp_min(-1e30)).sum(1) / total[:, 0]
    out = {"out": (d.gather(1, at) - log_total)[:, 0], "entropy": entropy, "stats": torch.cat([top, log_total], 1)}
    if s["case"]["top"]:
        # Equal logits in the order of their places.
        order = torch.sort(d, dim=1, descending=True, stable=True)
        out["top"] = order.values[:, :s["case"]["top"]] - log_total
        out["top_tokens"] = order.indices[:, :s["case"]["top"]].int()
    return out


def _plain_log_probs_grad(s):
    x = s["logits"].float()
    if s["mask"] is not None:
        x = torch.where(s["mask"] != 0, x, -math.inf)
    lp = (x - s["stats"][:, :1]) * s["case"]["scale"] - s["stats"][:, 1:]
    p = torch.exp(lp)
    dx = -p * (s["dout"][:, None] + s["dentropy"][:, None] * (lp.clamp_min(-1e30) + s["entropy"][:, None]))
    dx.scatter_add_(1, s["tokens"].long()[:, None], s["dout"][:, None])
    return (dx * s["case"]["scale"]).to(s["logits"].dtype)


def _act(kind, g):
    """The activation and its derivative."""
    if kind == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if kind == "silu":
        t = 1.0 / (1.0 + torch.exp(-g))
        return g * t, t * (1.0 + g * (1.0 - t))
    c = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * c, c + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_gated(s):
    f, dtype = s["case"]["f"], s["x"].dtype
    y = s["x"].float() @ s["w"].float().t()
    h = (_act(s["case"]["act"], y[:, :f])[0] * y[:, f:]).to(dtype)
    return (h, y.to(dtype)) if s["case"]["saved"] else h


def _plain_gated_grad(s):
    f, dtype = s["case"]["f"], s["x"].dtype
    d, y = s["dout"].float(), s["saved"].float()
    a, da = _act(s["case"]["act"], y[:, :f])
    dy = torch.cat([d * y[:, f:] * da, d * a], 1)
    return (dy @ s["w"].float()).to(dtype), (dy.t() @ s["x"].float()).to(dtype)


def _plain_int4(s):
    codes = torch.stack([s["codes"] & 15, s["codes"] >> 4], 2).view(s["case"]["n"], -1).float() - 8.0
    scales = s["scales"].t().float().repeat_interleave(s["case"]["group"], 1)[:, :s["case"]["k"]]
    return torch.clamp_min(s["a"].float() @ (codes * scales).t() + s["bias"], 0.0).to(s["out"].dtype)


_plain = {"log_probs": _plain_log_probs, "log_probs_grad": _plain_log_probs_grad, "gated": _plain_gated, "gated_grad": _plain_gated_grad,
          "int4": _plain_int4}


# -- what a pass cannot do without -----------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind in ("log_probs", "log_probs_grad"):
        rows, size = case["rows"], case["rows"] * case["cols"]
        each = ITEM[case["type"]] * (1 if kind == "log_probs" else 2) + (1 if case["mask"] else 0)
        row = (8 if case["index"] == "i64" else 4) + (16 + 8 * case["top"] if kind == "log_probs" else 20)
        return {"bytes": size * each + rows * row, "flops": 6 * size}
    if kind in ("gated", "gated_grad"):
        m, f, k = case["m"], case["f"], case["k"]
        if kind == "gated":
            return {"bytes": 2 * (m * k + 2 * f * k + m * f * (3 if case["saved"] else 1)), "flops": 4 * m * f * k}
        return {"bytes": 2 * (2 * m * k + 4 * f * k + 3 * m * f), "flops": 8 * m * f * k}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": n * k / 2 + 2 * n * -(-k // case["group"]) + 2 * m * (k + n) + 4 * n, "flops": 2 * m * n * k}


# -- the same from the definition in 64 bits -------------------------------------------------------------
def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "log_probs":
        return _exact_log_probs(s)
    if kind == "log_probs_grad":
        scale, stats = case["scale"], s["stats"].double()
        # Through the logarithms of the probabilities that the saved statistics give.
        lp = torch.sub(s["logits"].double() * scale, (stats[:, 0] * scale + stats[:, 1])[:, None])
        p = lp.exp()
        if case["mask"]:
            p = p * s["mask"]
        taken = torch.zeros_like(p)
        taken[torch.arange(case["rows"], device="cuda"), s["tokens"].long()] = 1.0
        return scale * (s["dout"].double()[:, None] * (taken - p) - (s["dentropy"].double()[:, None] * p) * (lp + s["entropy"].double()[:, None]))
    if kind in ("gated", "gated_grad"):
        if work(case)["flops"] > 4e11:
            return None
        return _exact_gated(s) if kind == "gated" else _exact_gated_grad(s)
    k = case["k"]
    column = torch.arange(k, device="cuda")
    codes = (s["codes"].long()[:, column // 2] >> (4 * (column % 2))) & 15
    w = (codes - 8).double() * s["scales"].double()[column // case["group"]].t()
    return torch.relu(torch.einsum("mk,nk->mn", s["a"].double(), w) + s["bias"].double())


def _exact_log_probs(s):
    case = s["case"]
    x = s["logits"].double()
    if case["mask"]:
        x = x.masked_fill(s["mask"] == 0, -math.inf)
    z = x * case["scale"]
    lse = torch.logsumexp(z, 1)
    rows = torch.arange(case["rows"], device="cuda")
    lp = z - lse[:, None]
    p = lp.exp()
    out = {"out": lp[rows, s["tokens"].long()], "entropy": -torch.where(p > 0, p * lp, 0.0).sum(1)}
    largest = x.amax(1)
    out["stats"] = torch.stack([largest, lse - largest * case["scale"]], 1)
    if case["top"]:
        # The largest that is left, at the lowest place that holds it, again and again.
        places = torch.arange(case["cols"], device="cuda", dtype=torch.int32)
        tokens = []
        for _ in range(case["top"]):
            at = torch.where(x == x.amax(1, keepdim=True), places, case["cols"]).amin(1)
            tokens.append(at)
            x[rows, at.long()] = -math.inf
        out["top_tokens"] = torch.stack(tokens, 1)
        out["top"] = torch.stack([lp[rows, t.long()] for t in tokens], 1)
    return {k: out[k] for k in ("out", "entropy", "stats") + (("top", "top_tokens") if case["top"] else ())}


def _exact_act(kind, g):
    return {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.nn.functional.relu}[kind](g)


def _exact_gated(s):
    gate, up = s["w"].double().chunk(2)
    x = s["x"].double()
    g, u = torch.einsum("mk,fk->mf", x, gate), torch.einsum("mk,fk->mf", x, up)
    h = _exact_act(s["case"]["act"], g) * u
    return (h, torch.cat([g, u], 1)) if s["case"]["saved"] else h


def _exact_gated_grad(s):
    # The derivative of the product through what was saved, by automatic differentiation, then the projections'.
    y = s["saved"].double().requires_grad_()
    g, u = y.chunk(2, 1)
    (_exact_act(s["case"]["act"], g) * u).backward(s["dout"].double())
    return torch.einsum("mf,fk->mk", y.grad, s["w"].double()), torch.einsum("mf,mk->fk", y.grad, s["x"].double())
