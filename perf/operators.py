"""The operators of a deep gated residual trunk: cases, plain forms and exact values.

Three operators that are used together: the gated feed-forward block, the RMS norms before and
after a block fused with its gate and residual scale, and the AdamW step over many tensors that
trains a stack of such blocks. ``run`` computes them in plain torch operations in 32 bits, or,
where ``own`` is true, by the calls a user makes of the framework.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
BLOCK = 256  # values that share one scale of an 8-bit optimizer state
ADAM = {"lr": 1e-3, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8, "weight_decay": 0.01}
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def _framework():
    """The framework's package (imported only where its kernels are run)."""
    package = str(Path(__file__).resolve().parents[1] / "expanded-gpu-optimization_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import fused_hoad

    return fused_hoad


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------


def _ffn(name, tokens, width, hidden, dtype, activation, bias, train):
    return {"name": name, "op": "ffn", "tokens": tokens, "width": width, "hidden": hidden,
            "dtype": dtype, "activation": activation, "bias": bias, "train": train}


def _norm(name, rows, width, dtype, residual_dtype, gate, post, train):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "dtype": dtype,
            "residual_dtype": residual_dtype, "gate": gate, "post": post, "train": train}


def _adam(name, width, hidden, blocks, dtype, bits):
    return {"name": name, "op": "adam", "width": width, "hidden": hidden, "blocks": blocks,
            "dtype": dtype, "bits": bits}


def listed():
    return [
        # one token (or one point) through a block when answering: latency and the weights' bytes
        _ffn("ffn one token", 1, 1024, 4096, "bfloat16", "silu", False, False),
        # a small batch of tokens in flight when serving: still bound by the weights' bytes
        _ffn("ffn batch of 48", 48, 2048, 5632, "bfloat16", "silu", False, False),
        # a long prompt, or a large evaluation batch: three large products
        _ffn("ffn 8192 evaluation", 8192, 4096, 11008, "bfloat16", "silu", False, False),
        # a training step's block at an ordinary model size
        _ffn("ffn 16384 training", 16384, 2048, 5632, "bfloat16", "silu", False, True),
        # the framework's own width, type, activation and point count, in training
        _ffn("ffn 64 wide points", 65536, 64, 256, "float32", "tanh", True, True),
        # odd sizes in float32: rows that no wide load or tile divides
        _ffn("ffn odd sizes", 1000, 201, 533, "float32", "silu", True, True),
        # between two blocks for one token
        _norm("norm one token", 1, 2048, "bfloat16", "bfloat16", "channel", True, False),
        # the framework's own width and point count, in training
        _norm("norm 64 wide points", 65536, 64, "float32", "float32", "channel", True, True),
        # a training batch of 16 samples, each with a gate of its own, residual kept in 32 bits
        _norm("norm 16384 training", 16384, 2048, "bfloat16", "float32", "sample", True, True),
        # the framework's MLP sizes: many small tensors, launch latency
        _adam("adamw small trunk", 64, 170, 4, "float32", 32),
        # a mid-sized model, 32-bit states
        _adam("adamw 32-bit states", 1024, 2816, 12, "float32", 32),
        # a larger model trained in bfloat16 with 8-bit states
        _adam("adamw 8-bit states", 2048, 5633, 6, "bfloat16", 8),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread evenly over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["ffn", "ffn", "norm", "adam"])
    dtype = rng.choice(["float32", "bfloat16"])
    train = rng.random() < 0.5
    if op == "ffn":
        while True:
            tokens = _spread(rng, 1, 65536)
            width = _spread(rng, 32, 4096)
            hidden = _spread(rng, 32, 11008)
            if rng.random() < 0.6:  # most models' sizes are round, some are not
                width, hidden = max(64, width // 64 * 64), max(64, hidden // 64 * 64)
            if width != 3072 and hidden != 3072 and tokens * width * hidden <= 1.8e11:
                break
        return {"op": "ffn", "tokens": tokens, "width": width, "hidden": hidden, "dtype": dtype,
                "activation": rng.choice(["silu", "tanh"]), "bias": rng.random() < 0.5,
                "train": train}
    if op == "norm":
        while True:
            rows = _spread(rng, 1, 65536)
            width = _spread(rng, 32, 8192)
            if rng.random() < 0.6:
                width = max(32, width // 32 * 32)
            if width != 3072 and rows * width <= 2 ** 25:
                break
        return {"op": "norm", "rows": rows, "width": width, "dtype": dtype,
                "residual_dtype": rng.choice(["float32", dtype]),
                "gate": rng.choice(["none", "channel", "sample", "full"]),
                "post": rng.random() < 0.7, "train": train}
    while True:
        width, blocks = _spread(rng, 32, 2048), _spread(rng, 1, 24)
        hidden = _spread(rng, 32, 5633)
        if width != 3072 and hidden != 3072 and blocks * width * hidden <= 34e6:
            break
    return {"op": "adam", "width": width, "hidden": hidden, "blocks": blocks, "dtype": dtype,
            "bits": rng.choice([8, 32])}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------


def _samples(rows):
    """Samples a batch of rows is made of: 16 where they divide it, else one gate row a row."""
    return 16 if rows % 16 == 0 else rows


def prepare(case, seed):
    generator = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=generator, device=DEVICE) * std).to(dtype)

    dtype = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "ffn":
        t, d, h = case["tokens"], case["width"], case["hidden"]
        state["x"] = normal(t, d, dtype=dtype)
        state["w_gate"] = normal(h, d, std=d ** -0.5, dtype=dtype)
        state["w_up"] = normal(h, d, std=d ** -0.5, dtype=dtype)
        state["w_down"] = normal(d, h, std=h ** -0.5, dtype=dtype)
        if case["bias"]:
            state["b_gate"] = normal(h, std=0.1, dtype=dtype)
            state["b_up"] = normal(h, std=0.1, dtype=dtype)
            state["b_down"] = normal(d, std=0.1, dtype=dtype)
        if case["train"]:
            state["grad"] = normal(t, d, dtype=dtype)
    elif case["op"] == "norm":
        n, c = case["rows"], case["width"]
        residual_dtype = DTYPES[case["residual_dtype"]]
        state["residual"] = normal(n, c, dtype=residual_dtype)
        state["branch"] = normal(n, c, std=0.7, dtype=dtype)
        state["pre_weight"] = (1.0 + normal(c, std=0.1)).to(dtype)
        state["residual_scale"] = 0.9 + normal(1, std=0.05)
        if case["post"]:
            state["post_weight"] = (1.0 + normal(c, std=0.1)).to(dtype)
        if case["gate"] == "channel":
            state["gate"] = (0.5 + normal(c, std=0.2)).to(dtype)
        elif case["gate"] == "sample":
            state["gate"] = (0.5 + normal(_samples(n), c, std=0.2)).to(dtype)
        elif case["gate"] == "full":
            state["gate"] = (0.5 + normal(n, c, std=0.2)).to(dtype)
        if case["train"]:
            # a loss pulls on the stream's own size too, so the scale has a gradient
            pull = 0.2 * state["residual"].float() + normal(n, c)
            state["grad_residual"] = pull.to(residual_dtype)
            state["grad_normed"] = normal(n, c, dtype=dtype)
    else:
        shapes = _adam_shapes(case)
        sizes = [math.prod(shape) for shape in shapes]
        total = sum(_padded(n) for n in sizes)
        flat = {"params": normal(total, std=0.05, dtype=dtype),
                "exp_avgs": normal(total, std=0.003),
                "exp_avg_sqs": normal(total, std=0.01).square()}
        if case["bits"] == 8:  # every tensor starts a block, so the flat buffer's blocks are theirs
            flat["exp_avgs"], flat["exp_avg_scales"] = _encode(flat["exp_avgs"])
            flat["exp_avg_sqs"], flat["exp_avg_sq_scales"] = _encode_square(flat["exp_avg_sqs"])
        state["flat"] = flat
        for name, buffer in flat.items():
            if name.endswith("scales"):
                state[name] = _pieces(buffer, [(-(-n // BLOCK),) for n in sizes], 1)
            else:
                state[name] = _pieces(buffer, shapes, BLOCK)
        state["grads"] = _pieces(normal(total, std=0.01, dtype=dtype), shapes, BLOCK)
        state["step"] = torch.full((1,), 10, dtype=torch.int64, device=DEVICE)
    return state


def _padded(count, unit=BLOCK):
    return -(-count // unit) * unit


def _pieces(buffer, shapes, unit):
    """The tensors of a flat buffer, each on a multiple of `unit` values."""
    sizes = [math.prod(shape) for shape in shapes]
    parts = torch.split(buffer, [_padded(n, unit) for n in sizes])
    return [part[:n].view(shape) for part, n, shape in zip(parts, sizes, shapes)]


def _adam_shapes(case):
    """The tensors of a stack of gated blocks with their norms, and its two outer layers."""
    d, h = case["width"], case["hidden"]
    block = [(h, d), (h, d), (d, h), (h,), (h,), (d,), (d,), (d,), (d,)]
    return [(d, 2), (d,)] + block * case["blocks"] + [(1, d), (1,)]


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return {"ffn": _own_ffn, "norm": _own_norm, "adam": _own_adam}[op](state)
    return {"ffn": _plain_ffn, "norm": _plain_norm, "adam": _plain_adam}[op](state)


def _own_ffn(s):
    fused_hoad, case = _framework(), s["case"]
    names = [n for n in ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down") if n in s]
    if not case["train"]:
        with torch.no_grad():
            return {"y": fused_hoad.gated_feed_forward(
                **{n: s[n] for n in names}, activation=case["activation"])}
    leaves = {n: s[n].detach().requires_grad_() for n in names}
    y = fused_hoad.gated_feed_forward(**leaves, activation=case["activation"])
    grads = torch.autograd.grad(y, list(leaves.values()), s["grad"])
    return {"y": y.detach(), **{"d_" + n: g for n, g in zip(names, grads)}}


def _gate_argument(s):
    """The gate as the call takes it: [C], [samples, 1, C] (broadcast over a sample's rows) or
    full; and how the rows are shaped to go with it."""
    case = s["case"]
    if case["gate"] == "sample":
        groups = s["gate"].shape[0]
        return s["gate"].unsqueeze(1), (groups, case["rows"] // groups, case["width"])
    return s.get("gate"), (case["rows"], case["width"])


def _own_norm(s):
    fused_hoad, case = _framework(), s["case"]
    gate, shape = _gate_argument(s)
    tensors = {"residual": s["residual"].view(shape), "branch": s["branch"].view(shape),
               "pre_weight": s["pre_weight"], "post_weight": s.get("post_weight"), "gate": gate,
               "residual_scale": s["residual_scale"]}
    tensors = {n: t for n, t in tensors.items() if t is not None}
    if not case["train"]:
        with torch.no_grad():
            residual, normed = fused_hoad.residual_norm(**tensors, eps=EPS)
            return {"residual": residual, "normed": normed}
    leaves = {n: t.detach().requires_grad_() for n, t in tensors.items()}
    residual, normed = fused_hoad.residual_norm(**leaves, eps=EPS)
    grads = torch.autograd.grad(
        (residual, normed), list(leaves.values()),
        (s["grad_residual"].view(shape), s["grad_normed"].view(shape)))
    return {"residual": residual.detach(), "normed": normed.detach(),
            **{"d_" + n: g for n, g in zip(leaves, grads)}}


def _own_adam(s):
    fused_hoad, a = _framework(), ADAM
    fused_hoad.adamw_step(
        s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], s["step"], lr=a["lr"],
        betas=(a["beta1"], a["beta2"]), eps=a["eps"], weight_decay=a["weight_decay"],
        exp_avg_scales=s.get("exp_avg_scales"), exp_avg_sq_scales=s.get("exp_avg_sq_scales"))
    return _adam_outputs(s)


# ---- plain forms: elementary torch operations in 32 bits, rounded once at the end ----


def _activation(g, name):
    """The activation and its derivative."""
    if name == "tanh":
        a = torch.tanh(g)
        return a, 1.0 - a * a
    sigma = 1.0 / (1.0 + torch.exp(-g))
    return g * sigma, sigma * (1.0 + g * (1.0 - sigma))


def _ffn_math(s, cast):
    """The block and its gradients by the formulas, in the type `cast` gives."""
    case, out = s["case"], {}
    x, wg, wu, wd = (cast(s[n]) for n in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.T, x @ wu.T
    if case["bias"]:
        g, u = g + cast(s["b_gate"]), u + cast(s["b_up"])
    a, slope = _activation(g, case["activation"])
    h = a * u
    y = h @ wd.T
    out["y"] = y + cast(s["b_down"]) if case["bias"] else y
    if case["train"]:
        dy = cast(s["grad"])
        dh = dy @ wd
        du, dg = dh * a, dh * u * slope
        out["d_x"] = dg @ wg + du @ wu
        out["d_w_gate"], out["d_w_up"], out["d_w_down"] = dg.T @ x, du.T @ x, dy.T @ h
        if case["bias"]:
            out["d_b_gate"], out["d_b_up"], out["d_b_down"] = dg.sum(0), du.sum(0), dy.sum(0)
    return out


def _plain_ffn(s):
    dtype = s["x"].dtype
    return {n: t.to(dtype) for n, t in _ffn_math(s, lambda t: t.float()).items()}


def _norm_math(s, cast):
    """The norms, gate and residual scale and their gradients, in the type `cast` gives."""
    case = s["case"]
    gate, shape = _gate_argument(s)
    r, b = cast(s["residual"]).view(shape), cast(s["branch"]).view(shape)
    alpha, w_pre = cast(s["residual_scale"]), cast(s["pre_weight"])
    w_post = cast(s["post_weight"]) if case["post"] else None
    z = b
    if case["post"]:
        inv_b = 1.0 / torch.sqrt((b * b).mean(-1, keepdim=True) + EPS)
        b_hat = b * inv_b
        z = b_hat * w_post
    gamma = cast(gate) if gate is not None else None
    total = alpha * r + (z if gamma is None else gamma * z)
    inv_t = 1.0 / torch.sqrt((total * total).mean(-1, keepdim=True) + EPS)
    t_hat = total * inv_t
    out = {"residual": total, "normed": t_hat * w_pre}
    if case["train"]:
        d_total, d_n = cast(s["grad_residual"]).view(shape), cast(s["grad_normed"]).view(shape)
        q = d_n * w_pre
        d_total = d_total + inv_t * (q - t_hat * (q * t_hat).mean(-1, keepdim=True))
        rows = tuple(range(len(shape) - 1))
        out["d_residual"] = alpha * d_total
        out["d_residual_scale"] = (d_total * r).sum().reshape(1)
        out["d_pre_weight"] = (d_n * t_hat).sum(rows)
        d_z = d_total
        if gamma is not None:
            d_gate = d_total * z
            out["d_gate"] = {"channel": lambda: d_gate.sum(rows), "full": lambda: d_gate,
                             "sample": lambda: d_gate.sum(1, keepdim=True)}[case["gate"]]()
            d_z = d_total * gamma
        if case["post"]:
            out["d_post_weight"] = (d_z * b_hat).sum(rows)
            p = d_z * w_post
            d_z = inv_b * (p - b_hat * (p * b_hat).mean(-1, keepdim=True))
        out["d_branch"] = d_z
    return out


def _norm_types(s):
    """Each output has the type of the input it belongs to."""
    types = {"residual": s["residual"].dtype, "normed": s["branch"].dtype}
    for n in ("residual", "branch", "pre_weight", "post_weight", "gate", "residual_scale"):
        if n in s:
            types["d_" + n] = s[n].dtype
    return types


def _plain_norm(s):
    types = _norm_types(s)
    return {n: t.to(types[n]) for n, t in _norm_math(s, lambda t: t.float()).items()}


def _blocks(values):
    """Flat values as rows of one block each, the last one filled up with zeros."""
    flat = values.reshape(-1)
    return torch.nn.functional.pad(flat, (0, -flat.numel() % BLOCK)).view(-1, BLOCK)


def _encode(values):
    """(e4m3 codes, one scale a block): the block's largest magnitude becomes 448."""
    rows = _blocks(values)
    scale = (rows.abs().amax(1) * (1.0 / 448.0)).clamp(min=2.0 ** -126)
    codes = (rows / scale[:, None]).float().to(torch.float8_e4m3fn)
    return codes.reshape(-1)[: values.numel()].view(values.shape), scale.float()


def _encode_square(values):
    """The square root of a second moment, coded the same way; what is not zero stays not zero."""
    rows = torch.sqrt(_blocks(values))
    scale = (rows.amax(1) * (1.0 / 448.0)).clamp(min=2.0 ** -126)
    units = rows / scale[:, None]
    units = torch.where(rows > 0, units.clamp(min=2.0 ** -9), units)
    codes = units.float().to(torch.float8_e4m3fn)
    return codes.reshape(-1)[: values.numel()].view(values.shape), scale.float()


def _decode(codes, scale, like):
    rows = _blocks(codes.to(like)) * scale.to(like)[:, None]
    return rows.reshape(-1)[: codes.numel()].view(codes.shape)


def _adam_math(s, like):
    """New parameters and moments, in the type `like`."""
    a, t = ADAM, int(s["step"]) + 1
    step_size = a["lr"] / (1.0 - a["beta1"] ** t)
    root = math.sqrt(1.0 - a["beta2"] ** t)
    if s["case"]["bits"] == 32:
        ms = [m.to(like) for m in s["exp_avgs"]]
        vs = [v.to(like) for v in s["exp_avg_sqs"]]
    else:
        ms = [_decode(c, q, like) for c, q in zip(s["exp_avgs"], s["exp_avg_scales"])]
        vs = [_decode(c, q, like) for c, q in zip(s["exp_avg_sqs"], s["exp_avg_sq_scales"])]
        vs = [v * v for v in vs]
    gs = [g.to(like) for g in s["grads"]]
    ms = [m * a["beta1"] + g * (1.0 - a["beta1"]) for m, g in zip(ms, gs)]
    vs = [v * a["beta2"] + (g * g) * (1.0 - a["beta2"]) for v, g in zip(vs, gs)]
    ps = [p.to(like) * (1.0 - a["lr"] * a["weight_decay"])
          - step_size * (m / (torch.sqrt(v) / root + a["eps"]))
          for p, m, v in zip(s["params"], ms, vs)]
    return ps, ms, vs


def _plain_adam(s):
    ps, ms, vs = _adam_math(s, torch.float32)
    _ = [p.copy_(q) for p, q in zip(s["params"], ps)]
    if s["case"]["bits"] == 32:
        _ = [a.copy_(b) for a, b in zip(s["exp_avgs"] + s["exp_avg_sqs"], ms + vs)]
    else:
        coded = [_encode(m) for m in ms]
        _ = [a.copy_(c) for a, (c, _) in zip(s["exp_avgs"], coded)]
        _ = [a.copy_(q) for a, (_, q) in zip(s["exp_avg_scales"], coded)]
        coded = [_encode_square(v) for v in vs]
        _ = [a.copy_(c) for a, (c, _) in zip(s["exp_avg_sqs"], coded)]
        _ = [a.copy_(q) for a, (_, q) in zip(s["exp_avg_sq_scales"], coded)]
    s["step"] += 1
    return _adam_outputs(s)


def _adam_outputs(s):
    """The buffers that the parameters, moments and scales are pieces of, whole."""
    return {**s["flat"], "step": s["step"]}


# ---------------------------------------------------------------------------------------------
# the floor and the exact values
# ---------------------------------------------------------------------------------------------


def work(case):
    """Bytes of the inputs and outputs, each once, and the operations of the products."""
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "ffn":
        t, d, h = case["tokens"], case["width"], case["hidden"]
        weights = 3 * d * h + (2 * h + d if case["bias"] else 0)
        passes = 3 if case["train"] else 1
        moved = 2 * t * d + weights + (2 * t * d + weights if case["train"] else 0)
        return {"bytes": moved * size, "flops": passes * 6 * t * d * h}
    if case["op"] == "norm":
        n, c = case["rows"], case["width"]
        wide = 4 if case["residual_dtype"] == "float32" else 2
        gate = {"none": 0, "channel": c, "full": n * c, "sample": _samples(n) * c}[case["gate"]]
        small = (c + gate + (c if case["post"] else 0)) * size + 4
        moved = 2 * n * c * (wide + size) + small
        if case["train"]:
            moved += 2 * n * c * (wide + size) + small
        return {"bytes": moved, "flops": n * c * (30 if case["train"] else 10)}
    count = sum(math.prod(s) for s in _adam_shapes(case))
    states = 16 * count if case["bits"] == 32 else 4 * count + 16 * -(-count // BLOCK)
    return {"bytes": 3 * size * count + states, "flops": 15 * count}


def _exact_activation(g, name):
    if name == "tanh":
        return torch.tanh(g), torch.cosh(g).pow(-2)
    s = torch.special.expit(g)
    return g * s, s + g * s * torch.special.expit(-g)


def exact(case, seed):
    s = prepare(case, seed)
    f64 = {n: t.double() for n, t in s.items() if torch.is_tensor(t) and t.is_floating_point()}
    if case["op"] == "ffn":
        # fp64 products run at a few per cent of the lower types' rate
        zero = torch.zeros((), dtype=torch.float64, device=DEVICE)
        gate = torch.addmm(f64.get("b_gate", zero), f64["x"], f64["w_gate"].t())
        up = torch.addmm(f64.get("b_up", zero), f64["x"], f64["w_up"].t())
        act, slope = _exact_activation(gate, case["activation"])
        out = {"y": torch.addmm(f64.get("b_down", zero), act * up, f64["w_down"].t())}
        if case["train"]:
            d_hidden = torch.mm(f64["grad"], f64["w_down"])
            d_up = d_hidden * act
            d_gate = d_hidden * up * slope
            out["d_w_down"] = torch.mm(f64["grad"].t(), act * up)
            del gate, up, act, slope, d_hidden
            out["d_w_gate"] = torch.mm(d_gate.t(), f64["x"])
            out["d_w_up"] = torch.mm(d_up.t(), f64["x"])
            out["d_x"] = torch.mm(d_gate, f64["w_gate"]).addmm_(d_up, f64["w_up"])
            if case["bias"]:
                ones = torch.ones(1, case["tokens"], dtype=torch.float64, device=DEVICE)
                out["d_b_gate"] = torch.mm(ones, d_gate)[0]
                out["d_b_up"] = torch.mm(ones, d_up)[0]
                out["d_b_down"] = torch.mm(ones, f64["grad"])[0]
        return out
    if case["op"] == "norm":
        return _exact_norm(case, s, f64)
    return _exact_adam(case, s)


def _exact_norm(case, s, f64):
    """By differentiating the definition itself, written with norms of vectors."""
    gate, shape = _gate_argument(s)
    leaves = {n: f64[n].clone().requires_grad_() for n in
              ("residual", "branch", "pre_weight", "post_weight", "residual_scale") if n in f64}
    if gate is not None:
        leaves["gate"] = gate.double().requires_grad_()

    def unit(v):
        return v / (torch.linalg.vector_norm(v, dim=-1, keepdim=True).square() / v.shape[-1]
                    + EPS).sqrt()

    inner = leaves["branch"].view(shape)
    if case["post"]:
        inner = unit(inner) * leaves["post_weight"]
    if gate is not None:
        inner = inner * leaves["gate"]
    total = leaves["residual"].view(shape) * leaves["residual_scale"] + inner
    normed = unit(total) * leaves["pre_weight"]
    out = {"residual": total.detach(), "normed": normed.detach()}
    if case["train"]:
        grads = torch.autograd.grad(
            (total, normed), list(leaves.values()),
            (f64["grad_residual"].view(shape), f64["grad_normed"].view(shape)))
        out.update({"d_" + n: g.view(shape) if n in ("residual", "branch") else g
                    for n, g in zip(leaves, grads)})
    return out


def _exact_adam(case, s):
    """The definition over the flat buffers, as if they were one tensor: every tensor starts a
    block of its own, and what lies between two tensors stays as it was."""
    a, t, flat = ADAM, int(s["step"]) + 1, s["flat"]
    shapes = _adam_shapes(case)
    inside = torch.zeros(flat["params"].numel(), dtype=torch.bool, device=DEVICE)
    gradient = torch.zeros(flat["params"].numel(), dtype=torch.float64, device=DEVICE)
    for place, values, g in zip(_pieces(inside, shapes, BLOCK), _pieces(gradient, shapes, BLOCK),
                                s["grads"]):
        place.fill_(True)
        values.copy_(g)
    m, v = flat["exp_avgs"].double(), flat["exp_avg_sqs"].double()
    if case["bits"] == 8:
        m = m * flat["exp_avg_scales"].double().repeat_interleave(BLOCK)
        v = (v * flat["exp_avg_sq_scales"].double().repeat_interleave(BLOCK)).pow(2)
    m = torch.lerp(m, gradient, 1.0 - a["beta1"])
    v = torch.lerp(v, gradient.pow(2), 1.0 - a["beta2"])
    m_fair, v_fair = m / (1.0 - a["beta1"] ** t), v / (1.0 - a["beta2"] ** t)
    p = flat["params"].double()
    p = p - a["lr"] * (a["weight_decay"] * p + m_fair / (v_fair.sqrt() + a["eps"]))
    new = {"params": p, "exp_avgs": m, "exp_avg_sqs": v}
    out = {"step": s["step"] + 1}
    if case["bits"] == 8:
        blank = torch.zeros((), dtype=torch.float64, device=DEVICE)
        for name, scales, power in (("exp_avgs", "exp_avg_scales", 1.0),
                                    ("exp_avg_sqs", "exp_avg_sq_scales", 0.5)):
            held = torch.where(inside, new[name], blank)  # a scale is that of its tensor's values
            held = (held if power == 1.0 else held.pow(power)).view(-1, BLOCK)
            out[scales] = held.abs().amax(1) / 448.0
            units = held / out[scales].clamp(min=2.0 ** -126)[:, None]
            low = 0.0 if power == 1.0 else 2.0 ** -9
            units = torch.where(units != 0, units.sign() * units.abs().clamp(min=low), units)
            new[name] = units.reshape(-1).float().to(torch.float8_e4m3fn).double()
    for name, values in new.items():
        out[name] = torch.where(inside, values, flat[name].double())
    return out
