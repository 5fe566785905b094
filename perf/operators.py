"""Performance cases of the operators around the dense layers of a net that reads tokens.

A policy net whose states are sequences of small integers (cards, actions, history) trains and answers with four
operators beside its dense layers: the embedding lookup and its gradient, layer normalisation and its gradient, one
AdamW step over all parameter tensors (states in 32 bits or in 8), and products in 8-bit floating point with a scale
per block of 128.  ``listed`` names sizes of real use, ``draw`` takes others from the same ranges.

``run`` computes an operator in its plain form, elementary torch operations in 32 bits, or, where ``own`` is true,
through this package.  ``exact`` computes the same from the definition in 64 bits.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ITEM = {"f32": 4, "bf16": 2, "f16": 2}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
SCALE_FLOOR = 2.0 ** -100                    # the largest magnitude that a block is taken to have at least
STATE_BLOCK = 256                            # elements of an optimizer state that share a scale
# Odd multipliers of the dither's hash: the golden ratio's and the leading 32 bits behind the point of roots.
ROOT5, ROOT2, ROOT3, ROOT7, R_SALT = 0x9E3779B1, 0x6A09E667, 0xBB67AE85, 0xA54FF53B, 0x3C6EF373
EMBED_SCALE = 0.0625
EPS = 1e-5
LR, BETA1, BETA2, ADAM_EPS, DECAY, STEP = 1e-3, 0.9, 0.999, 1e-8, 0.01, 7


def listed():
    return [
        # Sixteen tokens for each of 256 game states: the lookup of one decision, a latency-bound call.
        {"name": "embed_256_states", "kind": "embed", "n": 4096, "vocab": 256, "dim": 64, "table": "f32", "out": "bf16", "index": "i32"},
        # Training on a benchmark batch of 65536 states, eight cards each: few distinct tokens, long runs of each.
        {"name": "embed_grad_cards", "kind": "embed_grad", "n": 524288, "vocab": 53, "dim": 64, "out": "bf16", "index": "i32"},
        # A large vocabulary with common and rare tokens; sizes that fit no tile, 64-bit indices.
        {"name": "embed_grad_50001", "kind": "embed_grad", "n": 65537, "vocab": 50001, "dim": 1000, "out": "f32", "index": "i64"},
        # The normalisation in front of a small net, for the states of one decision.
        {"name": "norm_256x64", "kind": "norm", "rows": 256, "cols": 64, "type": "f16"},
        # Odd sizes of the ragged GEMM tests, 32-bit storage.
        {"name": "norm_grad_4001x1001", "kind": "norm_grad", "rows": 4001, "cols": 1001, "type": "f32"},
        # Behind a 1024-wide layer at the benchmark's batch of 65536 states.
        {"name": "norm_grad_65536x1024", "kind": "norm_grad", "rows": 65536, "cols": 1024, "type": "bf16"},
        # The optimizer step of the 512-1024x4-10 net: five weight matrices and five biases, bf16 compute copies.
        {"name": "adamw_policy_net", "kind": "adamw", "net": "holdem", "tensors": 10, "total": 3689482, "state": "f32", "grad": "f32", "copy": "bf16"},
        # Many tensors of mixed sizes with states in 8 bits and 16-bit gradients.
        {"name": "adamw_8bit_200_tensors", "kind": "adamw", "net": "", "tensors": 200, "total": 40000000, "state": "e4m3", "grad": "bf16", "copy": ""},
        # A large model on one GPU.
        {"name": "adamw_100m", "kind": "adamw", "net": "", "tensors": 64, "total": 100000000, "state": "f32", "grad": "f32", "copy": "bf16"},
        # A dense layer for sixteen states at once: quantise the activations, then a product that reads all weights.
        {"name": "fp8_layer_16", "kind": "fp8_layer", "m": 16, "n": 4096, "k": 4096, "type": "bf16"},
        # Operands already in 8 bits, sizes that fit no tile (the benchmark's ragged product).
        {"name": "fp8_product_ragged", "kind": "fp8_product", "m": 4000, "n": 3000, "k": 1008, "out": "f16"},
        # The same layer at a batch that fills the GPU many times.
        {"name": "fp8_layer_16384", "kind": "fp8_layer", "m": 16384, "n": 4096, "k": 4096, "type": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["embed", "embed_grad", "embed_grad", "norm", "norm_grad", "adamw", "adamw", "fp8_quantize", "fp8_layer", "fp8_product"])
    if kind in ("embed", "embed_grad"):
        dim, vocab = _log(rng, 8, 2048), _log(rng, 2, 65536)
        case = {"kind": kind, "n": _log(rng, 1, min(1 << 20, (1 << 26) // dim)), "vocab": vocab, "dim": dim,
                "out": rng.choice(["f32", "bf16", "f16"]), "index": rng.choice(["i32", "i64"])}
        return {**case, "table": rng.choice(["f32", "bf16", "f16"])} if kind == "embed" else case
    if kind in ("norm", "norm_grad"):
        cols = _log(rng, 8, 16384)
        return {"kind": kind, "rows": _log(rng, 1, min(1 << 18, (1 << 26) // cols)), "cols": cols, "type": rng.choice(["f32", "bf16", "f16"])}
    if kind == "adamw":
        tensors = _log(rng, 1, 300)
        return {"kind": kind, "net": "", "tensors": tensors, "total": _log(rng, 1000 * tensors, 64000000), "state": rng.choice(["f32", "e4m3"]),
                "grad": rng.choice(["f32", "bf16", "f16"]), "copy": rng.choice(["", "bf16", "f16"])}
    if kind == "fp8_quantize":
        cols = 16 * _log(rng, 1, 512)
        return {"kind": kind, "rows": _log(rng, 1, min(1 << 18, (1 << 26) // cols)), "cols": cols, "type": rng.choice(["f32", "bf16", "f16"]),
                "block_rows": rng.choice([1, 128])}
    n, k = _log(rng, 16, 8192), 16 * _log(rng, 1, 512)
    m = _log(rng, 1, min(1 << 15, (1 << 38) // (n * k)))
    if kind == "fp8_layer":
        return {"kind": kind, "m": m, "n": n, "k": k, "type": rng.choice(["bf16", "f16"])}
    return {"kind": kind, "m": m, "n": n, "k": k, "out": rng.choice(["f32", "bf16", "f16"])}


# -- inputs ----------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _tokens(g, case):
    """Common tokens first: an id's share falls with the id; one position in ten is padding (no token)."""
    u = torch.rand(case["n"], generator=g, device="cuda", dtype=torch.float64)
    ids = ((case["vocab"] + 1.0) ** u - 1.0).long().clamp_(0, case["vocab"] - 1)
    ids = torch.where(torch.rand(case["n"], generator=g, device="cuda") < 0.1, torch.full_like(ids, -1), ids)
    return ids.to(torch.int64 if case["index"] == "i64" else torch.int32)


def _tensor_sizes(case):
    if case["net"] == "holdem":
        widths = [512, 1024, 1024, 1024, 1024, 10]
        return [s for a, b in zip(widths, widths[1:]) for s in (a * b, b)]
    # Sizes over a range of a thousand, the same for every seed.
    r = np.random.RandomState(case["tensors"])
    share = np.exp(r.uniform(0.0, math.log(1000.0), case["tensors"]))
    return [max(1, int(s)) for s in share / share.sum() * case["total"]]


def _blocks_of(x, rows):
    """Rows and columns of a matrix as whole blocks of rows x 128, filled with zeros."""
    r, c = x.shape
    x = torch.nn.functional.pad(x, (0, -c % 128, 0, -r % rows))
    return x.view(x.shape[0] // rows, rows, x.shape[1] // 128, 128)


def _quantized(x, rows):
    """E4M3 codes of a matrix and the scale of each block of `rows` x 128 of it."""
    blocks = _blocks_of(x.float(), rows)
    largest = blocks.abs().amax((1, 3), keepdim=True).clamp_min(SCALE_FLOOR)
    top = torch.full_like(largest, E4M3_MAX)
    codes = (blocks * (top / largest)).to(E4M3).view(blocks.shape[0] * rows, -1)
    return codes[:x.shape[0], :x.shape[1]].contiguous(), (largest / top)[:, 0, :, 0]


def _dequantized(codes, scales, rows):
    blocks = _blocks_of(codes.float(), rows) * scales[:, None, :, None]
    return blocks.view(blocks.shape[0] * rows, -1)[:codes.shape[0], :codes.shape[1]]


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    s = {"case": case}
    if kind == "embed":
        s["tokens"] = _tokens(g, case)
        s["table"] = _normal(g, (case["vocab"], case["dim"]), TYPES[case["table"]])
        s["out"] = torch.empty((case["n"], case["dim"]), dtype=TYPES[case["out"]], device="cuda")
    elif kind == "embed_grad":
        s["tokens"] = _tokens(g, case)
        s["dout"] = _normal(g, (case["n"], case["dim"]), TYPES[case["out"]])
        s["dtable"] = torch.empty((case["vocab"], case["dim"]), dtype=torch.float32, device="cuda")
    elif kind in ("norm", "norm_grad"):
        rows, cols, dtype = case["rows"], case["cols"], TYPES[case["type"]]
        # Activations with an offset of their own in every row.
        s["x"] = (_normal(g, (rows, cols)) + _normal(g, (rows, 1))).to(dtype)
        s["weight"] = 1.0 + _normal(g, (cols,), std=0.1)
        s["mean"], s["rstd"] = (torch.empty(rows, dtype=torch.float32, device="cuda") for _ in range(2))
        if kind == "norm":
            s["bias"] = _normal(g, (cols,), std=0.1)
            s["out"] = torch.empty_like(s["x"])
        else:
            x = s["x"].float()
            s["mean"].copy_(x.mean(1))
            s["rstd"].copy_(1.0 / torch.sqrt((x - s["mean"][:, None]).square().mean(1) + EPS))
            s["dy"] = _normal(g, (rows, cols), dtype)
            s["dx"] = torch.empty_like(s["x"])
            s["dweight"], s["dbias"] = (torch.empty(cols, dtype=torch.float32, device="cuda") for _ in range(2))
    elif kind == "adamw":
        sizes = _tensor_sizes(case)
        # One arena, as parameters are kept: tensors begin at whole blocks of the states.
        begin = np.concatenate([[0], np.cumsum([-(-n // STATE_BLOCK) * STATE_BLOCK for n in sizes])]).tolist()
        real = torch.zeros(begin[-1], dtype=torch.bool, device="cuda")
        for b, n in zip(begin, sizes):
            real[b:b + n] = True
        s["sizes"], s["begin"], s["seed"] = sizes, begin, int(seed) & 0x7fffffff
        s["params"] = _normal(g, begin[-1], std=0.05) * real
        s["grads"] = (_normal(g, begin[-1], std=0.01) * real).to(TYPES[case["grad"]])
        m, r = _normal(g, begin[-1], std=0.003) * real, (_normal(g, begin[-1], std=0.01).abs() + 1e-4) * real
        if case["state"] == "f32":
            s["m"], s["v"] = m, r * r
        else:
            s["m"], s["m_scale"] = _state_codes(m)
            s["r"], s["r_scale"] = _state_codes(r)
        if case["copy"]:
            s["copy"] = s["params"].to(TYPES[case["copy"]])
    elif kind == "fp8_quantize":
        rows, cols = case["rows"], case["cols"]
        # Some columns carry much larger values than the rest, as activations do.
        s["x"] = (_normal(g, (rows, cols)) * torch.exp(_normal(g, (1, cols)))).to(TYPES[case["type"]])
        up = -(-rows // case["block_rows"])
        s["codes"] = torch.empty((rows, cols), dtype=E4M3, device="cuda")
        s["scales"] = torch.empty((-(-cols // 128), up) if case["block_rows"] == 1 else (up, -(-cols // 128)), dtype=torch.float32, device="cuda")
    else:
        m, n, k = case["m"], case["n"], case["k"]
        x = _normal(g, (m, k)) * torch.exp(_normal(g, (1, k), std=0.5))
        s["w"], s["w_scale"] = _quantized(_normal(g, (n, k), std=k ** -0.5), 128)
        s["a"] = torch.empty((m, k), dtype=E4M3, device="cuda")
        s["a_scale"] = torch.empty((-(-k // 128), m), dtype=torch.float32, device="cuda")
        if kind == "fp8_layer":
            s["x"] = x.to(TYPES[case["type"]])
            s["bias"] = _normal(g, (n,), std=0.1)
        else:
            codes, scales = _quantized(x, 1)
            s["a"].copy_(codes)
            s["a_scale"].copy_(scales.t())
        s["out"] = torch.empty((m, n), dtype=TYPES[case["type"] if kind == "fp8_layer" else case["out"]], device="cuda")
    return s


def _state_codes(x):
    """An optimizer state in 8 bits, rounded to nearest: what the program has from its earlier steps."""
    b = x.view(-1, STATE_BLOCK)
    largest = b.abs().amax(1, keepdim=True).clamp_min(SCALE_FLOOR)
    top = torch.full_like(largest, E4M3_MAX)
    return (b * (top / largest)).to(E4M3).view(-1), (largest / top).view(-1)


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


def _own_embed(s):
    return _sb().primitives.embedding(s["tokens"], s["table"], s["out"], scale=EMBED_SCALE)


def _own_embed_grad(s):
    return _sb().primitives.embedding_grad(s["tokens"], s["dout"], s["dtable"], scale=EMBED_SCALE)


def _own_norm(s):
    _sb().primitives.layer_norm(s["x"], s["out"], s["weight"], s["bias"], eps=EPS, mean=s["mean"], rstd=s["rstd"])
    return s["out"], s["mean"], s["rstd"]


def _own_norm_grad(s):
    _sb().primitives.layer_norm_grad(s["dy"], s["x"], s["mean"], s["rstd"], s["dx"], s["weight"], s["dweight"], s["dbias"])
    return s["dx"], s["dweight"], s["dbias"]


def _adamw_outputs(s):
    names = ("params", "m", "v") if s["case"]["state"] == "f32" else ("params", "m", "m_scale", "r", "r_scale")
    return {k: s[k] for k in names + (("copy",) if s["case"]["copy"] else ())}


def _own_adamw(s):
    opt = s.get("optimizer")
    if opt is None:                          # kept for the life of the program, as the tensors are
        def parts(x):
            return [x[b:b + n] for b, n in zip(s["begin"], s["sizes"])]

        def scales(x):
            return [x[b // STATE_BLOCK:-(-(b + n) // STATE_BLOCK)] for b, n in zip(s["begin"], s["sizes"])]
        more = {}
        if s["case"]["state"] == "e4m3":
            more = {"exp_avg_scale": scales(s["m_scale"]), "exp_avg_sq_scale": scales(s["r_scale"])}
        opt = s["optimizer"] = _sb().AdamW(parts(s["params"]), parts(s["grads"]), exp_avg=parts(s["m"]),
                                           exp_avg_sq=parts(s["v" if s["case"]["state"] == "f32" else "r"]),
                                           copies=parts(s["copy"]) if s["case"]["copy"] else None, state=s["case"]["state"], **more)
    opt.step(LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=DECAY, step=STEP, seed=s["seed"])
    return _adamw_outputs(s)


def _own_fp8_quantize(s):
    _sb().quantize_fp8(s["x"], s["codes"], s["scales"], block_rows=s["case"]["block_rows"])
    return s["codes"], s["scales"]


def _own_fp8_layer(s):
    sb = _sb()
    sb.quantize_fp8(s["x"], s["a"], s["a_scale"])
    return sb.matmul_fp8(s["a"], s["a_scale"], s["w"], s["w_scale"], s["out"], epilogue=("bias", "relu"), bias=s["bias"])


def _own_fp8_product(s):
    return _sb().matmul_fp8(s["a"], s["a_scale"], s["w"], s["w_scale"], s["out"])


_own = {"embed": _own_embed, "embed_grad": _own_embed_grad, "norm": _own_norm, "norm_grad": _own_norm_grad, "adamw": _own_adamw,
        "fp8_quantize": _own_fp8_quantize, "fp8_layer": _own_fp8_layer, "fp8_product": _own_fp8_product}


def _valid(s, vocab):
    return (s["tokens"] >= 0) & (s["tokens"] < vocab)


def _plain_embed(s):
    ok = _valid(s, s["table"].shape[0])
    rows = s["table"][torch.where(ok, s["tokens"], 0)].float() * EMBED_SCALE
    return torch.where(ok[:, None], rows, 0.0).to(s["out"].dtype)


def _plain_embed_grad(s):
    vocab = s["dtable"].shape[0]
    rows = torch.where(_valid(s, vocab), s["tokens"], vocab)
    sums = torch.zeros((vocab + 1, s["dout"].shape[1]), dtype=torch.float32, device="cuda")
    return sums.index_add_(0, rows, s["dout"].float())[:vocab] * EMBED_SCALE


def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    return (d * rstd * s["weight"] + s["bias"]).to(s["x"].dtype), mean[:, 0], rstd[:, 0]


def _plain_norm_grad(s):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xhat = (s["x"].float() - s["mean"][:, None]) * rstd
    g = dy * s["weight"]
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return dx.to(s["x"].dtype), (dy * xhat).sum(0), dy.sum(0)


def _noise(s, salt):
    """20 bits for each element of each tensor, from its index and the step's seed: the dither of a rounding to 8 bits."""
    if "index" not in s:
        at = torch.arange(s["begin"][-1], device="cuda")
        s["index"] = at - torch.tensor(s["begin"][:-1], device="cuda").repeat_interleave(torch.diff(torch.tensor(s["begin"], device="cuda")), output_size=at.numel())
    u = (s["index"] * ROOT5 + s["seed"] * ROOT2 + salt) & 0xffffffff
    u = ((u ^ (u >> 16)) * ROOT3) & 0xffffffff
    u = ((u ^ (u >> 15)) * ROOT7) & 0xffffffff
    return (u >> 12).int()


def _dithered(x, noise):
    """E4M3 codes of a state and its blocks' scales: magnitudes rounded up with the probability of the part cut off."""
    b = x.view(-1, STATE_BLOCK)
    largest = b.abs().amax(1, keepdim=True).clamp_min(SCALE_FLOOR)
    top = torch.full_like(largest, E4M3_MAX)
    y = (b * (top / largest)).view(-1)
    # A magnitude times 2^-120 has the code's bits from bit 20 on.
    code = (((y.abs() * 2.0 ** -120).view(torch.int32) + noise) >> 20).clamp_max(126)
    code = torch.where(y.view(torch.int32) < 0, code | 128, code)
    return code.to(torch.uint8).view(E4M3), (largest / top).view(-1)


def _spread(codes, scales):
    return (codes.float().view(-1, STATE_BLOCK) * scales[:, None]).view(-1)


def _plain_adamw(s):
    wide = s["case"]["state"] == "f32"
    g = s["grads"].float()
    m = s["m"] if wide else _spread(s["m"], s["m_scale"])
    r = None if wide else _spread(s["r"], s["r_scale"])
    v = s["v"] if wide else r * r
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + g * (1.0 - BETA2) * g
    r = torch.sqrt(v)
    p = s["params"] * (1.0 - LR * DECAY)
    p = p - m / (r * (1.0 / math.sqrt(1.0 - BETA2 ** STEP)) + ADAM_EPS) * (LR / (1.0 - BETA1 ** STEP))
    s["params"].copy_(p)
    if wide:
        s["m"].copy_(m)
        s["v"].copy_(v)
    else:
        codes, scales = _dithered(m, _noise(s, 0))
        s["m"].copy_(codes)
        s["m_scale"].copy_(scales)
        codes, scales = _dithered(r, _noise(s, R_SALT))
        # No positive magnitude becomes zero: the next step divides by it.
        codes = torch.where((r > 0) & (codes.view(torch.uint8) == 0), 1, codes.view(torch.uint8)).view(E4M3)
        s["r"].copy_(codes)
        s["r_scale"].copy_(scales)
    if s["case"]["copy"]:
        s["copy"].copy_(p)
    return _adamw_outputs(s)


def _plain_fp8_quantize(s):
    codes, scales = _quantized(s["x"], s["case"]["block_rows"])
    return codes, scales.t() if s["case"]["block_rows"] == 1 else scales


def _plain_product(s, codes, scales):
    return _dequantized(codes, scales, 1) @ _dequantized(s["w"], s["w_scale"], 128).t()


def _plain_fp8_layer(s):
    return torch.clamp_min(_plain_product(s, *_quantized(s["x"], 1)) + s["bias"], 0.0).to(s["out"].dtype)


def _plain_fp8_product(s):
    return _plain_product(s, s["a"], s["a_scale"].t()).to(s["out"].dtype)


_plain = {"embed": _plain_embed, "embed_grad": _plain_embed_grad, "norm": _plain_norm, "norm_grad": _plain_norm_grad, "adamw": _plain_adamw,
          "fp8_quantize": _plain_fp8_quantize, "fp8_layer": _plain_fp8_layer, "fp8_product": _plain_fp8_product}


# -- what a pass cannot do without -----------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "embed":
        # Every distinct token's row is read once at least.
        table = min(case["n"], case["vocab"]) * case["dim"] * ITEM[case["table"]]
        return {"bytes": case["n"] * (case["dim"] * ITEM[case["out"]] + (8 if case["index"] == "i64" else 4)) + table, "flops": case["n"] * case["dim"]}
    if kind == "embed_grad":
        rows = case["n"] * (case["dim"] * ITEM[case["out"]] + (8 if case["index"] == "i64" else 4))
        return {"bytes": rows + case["vocab"] * case["dim"] * 4, "flops": case["n"] * case["dim"]}
    if kind == "norm":
        return {"bytes": 2 * case["rows"] * case["cols"] * ITEM[case["type"]] + 8 * (case["rows"] + case["cols"]), "flops": 7 * case["rows"] * case["cols"]}
    if kind == "norm_grad":
        return {"bytes": 3 * case["rows"] * case["cols"] * ITEM[case["type"]] + 8 * case["rows"] + 12 * case["cols"], "flops": 13 * case["rows"] * case["cols"]}
    if kind == "adamw":
        each = 8 + ITEM[case["grad"]] + (16 if case["state"] == "f32" else 4 + 16 / STATE_BLOCK) + (2 if case["copy"] else 0)
        return {"bytes": case["total"] * each, "flops": 16 * case["total"]}
    if kind == "fp8_quantize":
        return {"bytes": case["rows"] * case["cols"] * (ITEM[case["type"]] + 1 + 4 / (128 * case["block_rows"])), "flops": 2 * case["rows"] * case["cols"]}
    m, n, k = case["m"], case["n"], case["k"]
    a = m * k * ITEM[case["type"]] if kind == "fp8_layer" else m * k * (1 + 4 / 128)
    return {"bytes": a + n * k + m * n * ITEM[case["type"] if kind == "fp8_layer" else case["out"]], "flops": 2 * m * n * k}


# -- the same from the definition in 64 bits -------------------------------------------------------------
def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "embed":
        table = torch.cat([s["table"].double(), torch.zeros_like(s["table"][:1], dtype=torch.float64)])
        t = s["tokens"].long()
        return table[torch.where((t < 0) | (t >= case["vocab"]), case["vocab"], t)] * EMBED_SCALE
    if kind == "embed_grad":
        keep = s["tokens"] >= 0
        total = torch.zeros((case["vocab"], case["dim"]), dtype=torch.float64, device="cuda")
        total.index_put_((s["tokens"][keep].long(),), s["dout"][keep].double(), accumulate=True)
        return total * EMBED_SCALE
    if kind == "norm":
        x = s["x"].double()
        var, mean = torch.var_mean(x, 1, correction=0)
        rstd = (var + EPS).rsqrt()
        return torch.addcmul(s["bias"].double(), (x - mean[:, None]) * rstd[:, None], s["weight"].double()), mean, rstd
    if kind == "norm_grad":
        x, w = s["x"].double(), s["weight"].double().requires_grad_()
        b = torch.zeros_like(w).requires_grad_()
        # The derivative through the statistics that the forward pass left.
        mean, rstd = s["mean"].double()[:, None], s["rstd"].double()[:, None]
        xhat, dy = (x - mean) * rstd, s["dy"].double()
        (xhat * w + b).backward(dy)
        t = dy * w.detach()
        cols = case["cols"]
        return (t * cols - t.sum(1, keepdim=True) - xhat * torch.einsum("rc,rc->r", t, xhat)[:, None]) * rstd / cols, w.grad, b.grad
    if kind == "adamw":
        return _exact_adamw(s)
    if kind == "fp8_quantize":
        codes, scales = _exact_codes(s["x"], case["block_rows"])
        return codes, scales.t() if case["block_rows"] == 1 else scales
    if kind == "fp8_layer":
        codes, scales = _exact_codes(s["x"], 1)
    else:
        codes, scales = s["a"].double(), s["a_scale"].double().t()
    k = case["k"]
    block = torch.arange(k, device="cuda") // 128
    w = s["w"].double() * s["w_scale"].double()[torch.arange(case["n"], device="cuda") // 128][:, block]
    y = torch.einsum("mk,nk->mn", codes * scales[:, block], w)
    return torch.relu(y + s["bias"].double()) if kind == "fp8_layer" else y


def _round_e4m3(y):
    """Nearest values of the format: 3 bits behind the leading one, steps of 2^-9 below 2^-6; ties to even."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3.0)
    return (torch.round(y / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_codes(x, rows):
    r, c = x.shape
    x = x.double()
    up, across = -(-r // rows), -(-c // 128)
    which = (torch.arange(r, device="cuda") // rows)[:, None] * across + (torch.arange(c, device="cuda") // 128)[None, :]
    largest = torch.zeros(up * across, dtype=torch.float64, device="cuda")
    largest.scatter_reduce_(0, which.reshape(-1), x.abs().reshape(-1), "amax")
    scales = largest.clamp_min(SCALE_FLOOR) / E4M3_MAX
    return _round_e4m3(x / scales[which]), scales.view(up, across)


def _exact_noise(s, salt):
    parts = []
    for begin, end in zip(s["begin"], s["begin"][1:]):
        with np.errstate(over="ignore"):
            u = np.arange(end - begin, dtype=np.uint32) * np.uint32(ROOT5) + np.uint32((s["seed"] * ROOT2 + salt) % 2 ** 32)
            u = (u ^ (u >> np.uint32(16))) * np.uint32(ROOT3)
            u = (u ^ (u >> np.uint32(15))) * np.uint32(ROOT7)
        parts.append(u >> np.uint32(12))
    return torch.from_numpy(np.concatenate(parts).astype(np.int64)).cuda()


def _exact_adamw(s):
    case = s["case"]
    g, p = s["grads"].double(), s["params"].double()

    def held(name):
        return s[name].double() * s[name + "_scale"].double().repeat_interleave(STATE_BLOCK)
    m = s["m"].double() if case["state"] == "f32" else held("m")
    v = s["v"].double() if case["state"] == "f32" else held("r") ** 2
    m = torch.lerp(g, m, BETA1)
    v = torch.lerp(g * g, v, BETA2)
    unbiased = (v / (1.0 - BETA2 ** STEP)).sqrt() + ADAM_EPS
    p = p - LR * DECAY * p - LR * (m / (1.0 - BETA1 ** STEP)) / unbiased
    out = {"params": p}
    if case["state"] == "f32":
        out.update(m=m, v=v)
    else:
        for name, x, salt in (("m", m, 0), ("r", v.sqrt(), R_SALT)):
            scale = x.abs().view(-1, STATE_BLOCK).amax(1).clamp_min(SCALE_FLOOR) / E4M3_MAX
            y = x / scale.repeat_interleave(STATE_BLOCK)
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3.0)
            up = torch.floor(y.abs() / step + _exact_noise(s, salt).double() / 2.0 ** 20) * step
            up = up.clamp_max(E4M3_MAX)
            if name == "r":
                up = torch.where(x > 0, up.clamp_min(2.0 ** -9), up)
            out[name], out[name + "_scale"] = up * y.sign(), scale
    if case["copy"]:
        out["copy"] = p
    return out
