"""The operators of a Swin block's training step, measured: each case is one pass through one
operator, from inputs a training program holds on the GPU to its outputs and gradients.

* ``bias``: the learned relative-position bias by buckets (``table[index]`` per head) and the
  gradient of its table;
* ``attention``: window attention from the packed qkv with that bias and the shifted-window
  mask, forward and backward (gradients of qkv and of the bias table);
* ``norm``: a branch's optional post-norm, gate and per-sample residual scale, the residual add
  and the next norm, forward (``"pass": "forward"``) or backward;
* ``gelu``: GELU whose input is kept in 8 bits, forward and backward (the output, the input's
  gradient and the output recomputed for the next Linear's weight gradient).

``run`` computes them with elementary torch operations in 32 bits where ``own`` is false, and
through ``crumpet_b200`` where it is true.  ``exact`` gives the same outputs in 64 bits, with
gradients from autograd instead of the formulas the plain forms use.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5
GROUP = 32  # neighbouring channels that share one 8-bit scale


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # the bias of a 7x7x7 window for the 24 heads of the deepest stage
        {"name": "bias 7x7x7 h24 f32", "op": "bias", "window": "7,7,7", "rows": 343, "cols": 343,
         "buckets": 2197, "heads": 24, "dtype": "f32"},
        # a generic long sequence with 32 logarithmic distance buckets
        {"name": "bias 1024x1024 log h16 bf16", "op": "bias", "window": "", "rows": 1024,
         "cols": 1024, "buckets": 32, "heads": 16, "dtype": "bf16"},
        # the deepest stage of a 96^3 volume: one window of 6^3 tokens per sample, two samples
        {"name": "attn 6x6x6 h24 b2 bf16", "op": "attention", "window": "6,6,6", "grid": "1,1,1",
         "shift": "0,0,0", "batch": 2, "heads": 24, "head_dim": 16, "dtype": "bf16",
         "table": "f32"},
        # the first stage of a 96^3 volume (48^3 tokens, padded to 49^3), a shifted block
        {"name": "attn 7x7x7 h3 b343 f16", "op": "attention", "window": "7,7,7", "grid": "7,7,7",
         "shift": "3,3,3", "batch": 1, "heads": 3, "head_dim": 16, "dtype": "f16", "table": "f32"},
        # the same for a batch of four volumes
        {"name": "attn 7x7x7 h3 b1372 bf16", "op": "attention", "window": "7,7,7",
         "grid": "7,7,7", "shift": "3,3,3", "batch": 4, "heads": 3, "head_dim": 16,
         "dtype": "bf16", "table": "f32"},
        # small windows of wide heads, the whole model in 16 bits
        {"name": "attn 4x4x4 h8 d32 b512 bf16", "op": "attention", "window": "4,4,4",
         "grid": "8,8,8", "shift": "2,2,2", "batch": 1, "heads": 8, "head_dim": 32,
         "dtype": "bf16", "table": "bf16"},
        # training without autocast, an odd window
        {"name": "attn 5x5x5 h3 b64 f32", "op": "attention", "window": "5,5,5", "grid": "4,4,4",
         "shift": "2,2,2", "batch": 1, "heads": 3, "head_dim": 16, "dtype": "f32", "table": "f32"},
        # the first stage's tokens: drop path, residual add and norm2
        {"name": "norm fwd 110592x48 bf16", "op": "norm", "pass": "forward", "samples": 1,
         "tokens": 110592, "channels": 48, "post": False, "gate": False, "scale": True,
         "pre": True, "dtype": "bf16", "stream": "bf16"},
        # four volumes under autocast (fp32 residual stream), post-norm and layer scale too
        {"name": "norm bwd 442368x48 f16 f32", "op": "norm", "pass": "backward", "samples": 4,
         "tokens": 110592, "channels": 48, "post": True, "gate": True, "scale": True,
         "pre": True, "dtype": "f16", "stream": "f32"},
        # the deepest stage: few rows, where latency counts
        {"name": "norm bwd 432x384 f32", "op": "norm", "pass": "backward", "samples": 2,
         "tokens": 216, "channels": 384, "post": False, "gate": True, "scale": True, "pre": True,
         "dtype": "f32", "stream": "f32"},
        # the MLP's hidden layer for four volumes of the first stage
        {"name": "gelu 442368x192 bf16", "op": "gelu", "tokens": 442368, "channels": 192,
         "dtype": "bf16"},
        # a ragged width in fp32
        {"name": "gelu 1029x250 f32", "op": "gelu", "tokens": 1029, "channels": 250,
         "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["bias", "attention", "attention", "norm", "norm", "gelu"])
    if op == "bias":
        heads = rng.randint(1, 24)
        if rng.random() < 0.5:
            win = [rng.randint(1, 8) for _ in range(3)]
            n = win[0] * win[1] * win[2]
            return {"op": op, "window": ",".join(map(str, win)), "rows": n, "cols": n,
                    "buckets": (2 * win[0] - 1) * (2 * win[1] - 1) * (2 * win[2] - 1),
                    "heads": heads, "dtype": rng.choice(list(DTYPES))}
        return {"op": op, "window": "", "rows": _log(rng, 1, 1500), "cols": _log(rng, 1, 1500),
                "buckets": rng.randint(2, 64), "heads": heads, "dtype": rng.choice(list(DTYPES))}
    if op == "attention":
        win = [rng.randint(2, 7) for _ in range(3)]
        n = win[0] * win[1] * win[2]
        heads = _log(rng, 1, 24)
        grid = [rng.randint(1, 7) for _ in range(3)]
        windows = grid[0] * grid[1] * grid[2]
        dtype = rng.choice(["f16", "bf16", "bf16", "f32"])
        head_dim = rng.choice([16, 16, 32])
        # at most a quarter of the largest listed case's scores (a sixteenth in fp32)
        most = 1372 * 3 * 343 * 343 // (16 if dtype == "f32" else 4) * 16 // head_dim
        while windows * heads * n * n > most:
            if heads > 3:
                heads = max(1, heads // 2)
            else:
                grid[grid.index(max(grid))] = max(1, max(grid) // 2)
            windows = grid[0] * grid[1] * grid[2]
        batch = _log(rng, 1, max(1, min(64, most // (windows * heads * n * n))))
        shifted = rng.random() < 0.6
        shift = [w // 2 if shifted and g > 1 else 0 for w, g in zip(win, grid)]
        return {"op": op, "window": ",".join(map(str, win)), "grid": ",".join(map(str, grid)),
                "shift": ",".join(map(str, shift)), "batch": batch, "heads": heads,
                "head_dim": head_dim, "dtype": dtype, "table": rng.choice(["f32", dtype])}
    if op == "norm":
        channels = _log(rng, 8, 1024)
        samples = rng.randint(1, 5)
        tokens = _log(rng, 1, max(1, 442368 * 48 // channels // samples // 2))
        dtype = rng.choice(list(DTYPES))
        post, gate, scale, pre = (rng.random() < p for p in (0.4, 0.5, 0.7, 0.8))
        return {"op": op, "pass": rng.choice(["forward", "backward"]), "samples": samples,
                "tokens": tokens, "channels": channels, "post": post, "gate": gate,
                "scale": scale, "pre": pre, "dtype": dtype,
                "stream": rng.choice(["f32", dtype])}
    channels = _log(rng, 1, 4096)
    dtype = rng.choice(list(DTYPES))
    return {"op": op, "tokens": _log(rng, 1, max(1, 442368 * 192 // channels // 2)),
            "channels": channels, "dtype": dtype}


# ------------------------------------------------------------------------------ inputs
def _triple(text):
    return [int(v) for v in text.split(",")]


def _window_index(win, device):
    """Bucket of every (query, key) pair of a 3D window: its relative coordinate."""
    at = torch.stack(torch.meshgrid(*(torch.arange(w, device=device) for w in win),
                                    indexing="ij")).flatten(1)
    rel = at[:, :, None] - at[:, None, :]
    rel = rel + (torch.tensor(win, device=device) - 1)[:, None, None]
    return (rel[0] * (2 * win[1] - 1) + rel[1]) * (2 * win[2] - 1) + rel[2]


def _log_index(rows, cols, buckets, device):
    """Buckets of the distance |i - j|: exact while short, logarithmic beyond."""
    dist = (torch.arange(rows, device=device)[:, None] - torch.arange(cols, device=device)).abs()
    short = buckets // 2
    far = short + (torch.log(dist.double().clamp(min=1) / max(1, short))
                   / math.log(max(rows, cols, 2 * short + 2) / max(1, short))
                   * (buckets - short)).floor().long().clamp(min=0)
    return torch.where(dist < short, dist, far).clamp(max=buckets - 1)


def _codes(win, grid, shift, device):
    """Region number of every token of every window of the rolled grid, [windows, tokens]."""
    parts = []
    for w, g, s in zip(win, grid, shift):
        at = torch.arange(w * g, device=device)
        region = (at >= w * g - w).long() + (at >= w * g - s).long() if s else torch.zeros_like(at)
        parts.append(region.view(g, w))
    d, h, w = parts
    code = (d[:, None, None, :, None, None] * 9 + h[None, :, None, None, :, None] * 3
            + w[None, None, :, None, None, :])
    return code.reshape(grid[0] * grid[1] * grid[2], win[0] * win[1] * win[2])


def _make(case, seed):
    """The inputs alone, the same for every form of the operator."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=dtype):
        x = torch.randn(shape, generator=gen, device=dev)
        return (x * std + mean).to(dtype)

    if case["op"] == "bias":
        if case["window"]:
            index = _window_index(_triple(case["window"]), dev)
        else:
            index = _log_index(case["rows"], case["cols"], case["buckets"], dev)
        return {"index": index, "table": normal(case["buckets"], case["heads"], std=0.5),
                "grad": normal(case["heads"], case["rows"], case["cols"], std=1e-2)}
    if case["op"] == "attention":
        win, grid, shift = (_triple(case[k]) for k in ("window", "grid", "shift"))
        n, h, d = win[0] * win[1] * win[2], case["heads"], case["head_dim"]
        b = case["batch"] * grid[0] * grid[1] * grid[2]
        t = (2 * win[0] - 1) * (2 * win[1] - 1) * (2 * win[2] - 1)
        return {"qkv": normal(b, n, 3, h, d), "table": normal(t, h, std=0.5,
                                                              dtype=DTYPES[case["table"]]),
                "grad": normal(b, n, h * d), "index": _window_index(win, dev),
                "codes": _codes(win, grid, shift, dev) if any(shift) else None}
    if case["op"] == "norm":
        s, m, c = case["samples"], case["tokens"], case["channels"]
        stream = DTYPES[case["stream"]]
        keep = 0.8  # drop path at rate 0.2: a sample's branch is dropped or scaled up
        drop = (torch.rand(s, generator=gen, device=dev) < keep).float() / keep
        drop[0] = 1 / keep
        state = {
            "branch": normal(s * m, c),
            "gate": normal(c, std=0.2, mean=0.5, dtype=torch.float32) if case["gate"] else None,
            "scale": drop if case["scale"] else None,
            "post": tuple(normal(c, std=0.1, mean=v, dtype=torch.float32) for v in (1.0, 0.0))
            if case["post"] else None,
            "pre": tuple(normal(c, std=0.1, mean=v, dtype=torch.float32) for v in (1.0, 0.0))
            if case["pre"] else None,
        }
        if case["pass"] == "forward":
            state["residual"] = normal(s * m, c, dtype=stream)
        else:
            state["out"] = normal(s * m, c, std=1.5, mean=0.1, dtype=stream)
            state["grad_out"] = normal(s * m, c, dtype=stream)
            state["grad_normed"] = normal(s * m, c) if case["pre"] else None
        return state
    return {"x": normal(case["tokens"], case["channels"], std=1.2),
            "grad": normal(case["tokens"], case["channels"])}


def prepare(case, seed):
    state = dict(_make(case, seed), case=case)
    if own and "index" in state:
        import crumpet_b200 as crumpet

        # the plan of a module's fixed index, made once when the module is built
        state["buckets"] = crumpet.relative_position_buckets(state["index"],
                                                             state["table"].shape[0])
    return state


# ------------------------------------------------------------------------- plain forms
def _plain_bias(s):
    table, index, grad = s["table"], s["index"], s["grad"]
    bias = table[index].permute(2, 0, 1).contiguous()
    h = table.shape[1]
    flat = grad.float().permute(1, 2, 0).reshape(-1, h)
    grad_table = torch.zeros(table.shape, device=table.device).index_add_(0, index.reshape(-1), flat)
    return {"bias": bias, "grad_table": grad_table.to(table.dtype)}


def _plain_attention(s):
    qkv, table, index = s["qkv"], s["table"], s["index"]
    b, n, _, h, d = qkv.shape
    scale = d ** -0.5
    q, k, v = qkv.float().permute(2, 0, 3, 1, 4).unbind(0)
    score = q @ k.transpose(-2, -1) * scale + table.float()[index].permute(2, 0, 1)
    if s["codes"] is not None:
        apart = (s["codes"][:, :, None] != s["codes"][:, None, :]).float() * -100.0
        score = (score.view(-1, apart.shape[0], h, n, n) + apart[:, None]).view(b, h, n, n)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = (p @ v).transpose(1, 2).reshape(b, n, h * d)
    g = s["grad"].float().view(b, n, h, d).transpose(1, 2)
    dp = g @ v.transpose(-2, -1)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    grads = torch.stack((ds @ k * scale, ds.transpose(-2, -1) @ q * scale,
                         p.transpose(-2, -1) @ g))
    grad_bias = ds.sum(0).permute(1, 2, 0).reshape(n * n, h)
    grad_table = torch.zeros(table.shape, device=qkv.device).index_add_(0, index.reshape(-1),
                                                                        grad_bias)
    return {"out": out.to(qkv.dtype), "grad_qkv": grads.permute(1, 3, 0, 2, 4).to(qkv.dtype),
            "grad_table": grad_table.to(table.dtype)}


def _centred(x):
    x = x - x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * rstd, rstd


def _row_scale(scale, rows):
    return scale.repeat_interleave(rows // scale.numel())[:, None]


def _plain_norm_forward(s):
    branch, residual = s["branch"].float(), s["residual"]
    if s["post"] is not None:
        branch = _centred(branch)[0] * s["post"][0] + s["post"][1]
    if s["gate"] is not None:
        branch = branch * s["gate"]
    if s["scale"] is not None:
        branch = branch * _row_scale(s["scale"], branch.shape[0])
    out = (residual.float() + branch).to(residual.dtype)
    result = {"out": out}
    if s["pre"] is not None:  # the next norm reads the stream as it is stored
        normed = _centred(out.float())[0] * s["pre"][0] + s["pre"][1]
        result["normed"] = normed.to(s["branch"].dtype)
    return result


def _norm_gradient(x_hat, rstd, weight, grad):
    g = grad * weight
    g = (g - g.mean(-1, keepdim=True) - x_hat * (g * x_hat).mean(-1, keepdim=True)) * rstd
    return g, (grad * x_hat).sum(0), grad.sum(0)


def _plain_norm_backward(s):
    branch, result = s["branch"].float(), {}
    grad = s["grad_out"].float()
    if s["pre"] is not None:
        x_hat, rstd = _centred(s["out"].float())
        g, result["pre_weight"], result["pre_bias"] = _norm_gradient(
            x_hat, rstd, s["pre"][0], s["grad_normed"].float())
        grad = grad + g
    result["residual"] = grad.to(s["out"].dtype)
    if s["scale"] is not None:
        grad = grad * _row_scale(s["scale"], branch.shape[0])
    if s["post"] is not None:
        x_hat, rstd = _centred(branch)
        normed = x_hat * s["post"][0] + s["post"][1]
    else:
        normed = branch
    if s["gate"] is not None:
        result["gate"] = (grad * normed).sum(0)
        grad = grad * s["gate"]
    if s["post"] is not None:
        grad, result["post_weight"], result["post_bias"] = _norm_gradient(
            x_hat, rstd, s["post"][0], grad)
    result["branch"] = grad.to(s["branch"].dtype)
    return result


def _eight_bits(x):
    """What 8 bits keep of x: per 32 neighbouring channels of a row, whole multiples (at most
    127 of them) of the least power of two that reaches the largest magnitude."""
    rows, c = x.shape
    pad = -c % GROUP
    g = torch.cat((x, x.new_zeros(rows, pad)), 1).view(rows, -1, GROUP)
    mantissa, exponent = torch.frexp(g.abs().amax(-1, keepdim=True))
    exponent = exponent - 7 + (mantissa > 127 / 128).to(exponent.dtype)
    exponent = exponent.clamp(min=-126)
    step = ((exponent + 127) << 23).view(torch.float32)  # 2^exponent by its bits
    return (torch.round(g / step) * step).view(rows, -1)[:, :c]


def _plain_gelu(s):
    x, grad = s["x"].float(), s["grad"].float()
    kept = _eight_bits(x)
    cdf = 0.5 * (1 + torch.erf(kept * math.sqrt(0.5)))
    pdf = torch.exp(-0.5 * kept * kept) / math.sqrt(2 * math.pi)
    y = x * 0.5 * (1 + torch.erf(x * math.sqrt(0.5)))
    dtype = s["x"].dtype
    return {"y": y.to(dtype), "grad_x": (grad * (cdf + kept * pdf)).to(dtype),
            "again": (kept * cdf).to(dtype)}


# --------------------------------------------------------------------- the framework's
def _own_attention(s):
    import crumpet_b200 as crumpet

    c = s["case"]
    place = dict(num_windows=_triple(c["grid"]), window_size=_triple(c["window"]),
                 shift_size=_triple(c["shift"]))
    out = crumpet.swin_window_attention_train(s["qkv"], s["table"], s["buckets"], **place)
    grad_qkv, grad_table = crumpet.swin_window_attention_backward(s["grad"], s["qkv"], s["table"],
                                                                  s["buckets"], **place)
    return {"out": out, "grad_qkv": grad_qkv, "grad_table": grad_table}


def _own_norm(s):
    import crumpet_b200 as crumpet

    how = dict(gate=s["gate"], row_scale=s["scale"], post_norm=s["post"], pre_norm=s["pre"],
               eps=EPS)
    if s["case"]["pass"] == "forward":
        out, normed = crumpet.norm_gate_residual(s["branch"], s["residual"], **how)
        return {"out": out, "normed": normed}
    grads = crumpet.norm_gate_residual_backward(s["grad_out"], s["grad_normed"], s["out"],
                                                s["branch"], **how)
    return grads._asdict()


def _own(s):
    import crumpet_b200 as crumpet

    op = s["case"]["op"]
    if op == "bias":
        return {"bias": crumpet.relative_position_bias(s["table"], s["buckets"]),
                "grad_table": crumpet.relative_position_bias_backward(s["grad"], s["buckets"])}
    if op == "attention":
        return _own_attention(s)
    if op == "norm":
        return _own_norm(s)
    y, kept = crumpet.gelu_checkpoint(s["x"])
    grad_x, again = crumpet.gelu_checkpoint_backward(s["grad"], kept)
    return {"y": y, "grad_x": grad_x, "again": again}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "norm":
        return (_plain_norm_forward if state["case"]["pass"] == "forward"
                else _plain_norm_backward)(state)
    return {"bias": _plain_bias, "attention": _plain_attention, "gelu": _plain_gelu}[op](state)


# -------------------------------------------------------------------------------- work
def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    e = size[case["dtype"]]
    if case["op"] == "bias":
        pairs, h = case["rows"] * case["cols"], case["heads"]
        # the bucket numbers, the bias written and its gradient read, the table and its gradient
        return {"bytes": 8 * pairs + 2 * pairs * h * e + 2 * case["buckets"] * h * e,
                "flops": pairs * h}
    if case["op"] == "attention":
        win, grid = _triple(case["window"]), _triple(case["grid"])
        n, h, d = win[0] * win[1] * win[2], case["heads"], case["head_dim"]
        b = case["batch"] * grid[0] * grid[1] * grid[2]
        t = (2 * win[0] - 1) * (2 * win[1] - 1) * (2 * win[2] - 1)
        # qkv and its gradient, the output and its gradient; two products forward, five back
        return {"bytes": 8 * b * n * h * d * e + 8 * n * n + 2 * t * h * size[case["table"]],
                "flops": 14 * b * h * n * n * d}
    if case["op"] == "norm":
        x = case["samples"] * case["tokens"] * case["channels"]
        r = size[case["stream"]]
        if case["pass"] == "forward":
            return {"bytes": x * (e + 2 * r + (e if case["pre"] else 0)), "flops": 12 * x}
        reads_branch = case["post"] or case["gate"]
        return {"bytes": x * ((e if reads_branch else 0) + 2 * r + e
                              + (e + r if case["pre"] else 0)), "flops": 25 * x}
    x = case["tokens"] * case["channels"]
    # x read, y, the 8 bits and their scales written; those read back, a gradient in, two out
    return {"bytes": x * (2 * e + 2 + 3 * e) + 2 * case["tokens"] * -(-case["channels"] // GROUP),
            "flops": 60 * x}


# ------------------------------------------------------------------------------- exact
def exact(case, seed):
    s = _make(case, seed)
    wide = lambda t: t.double().requires_grad_(True)  # noqa: E731
    with torch.enable_grad():
        if case["op"] == "bias":
            table = wide(s["table"])
            bias = torch.stack([table[:, h].take(s["index"]) for h in range(case["heads"])])
            (grad,) = torch.autograd.grad(bias, table, s["grad"].double())
            return {"bias": bias.detach(), "grad_table": grad}
        if case["op"] == "attention":
            return _exact_attention(s, wide)
        if case["op"] == "norm":
            return _exact_norm(case, s, wide)
        return _exact_gelu(s, wide)


def _exact_attention(s, wide):
    b, n, _, h, d = s["qkv"].shape
    table = wide(s["table"])
    per = 1 if s["codes"] is None else s["codes"].shape[0]
    step = max(1, (1 << 27) // (h * n * n))  # windows at a time
    outs, grads, grad_table = [], [], torch.zeros_like(table)
    for at in range(0, b, step):
        qkv = wide(s["qkv"][at:at + step])
        logits = torch.einsum("bihd,bjhd->bhij", qkv[:, :, 0], qkv[:, :, 1]) / math.sqrt(d)
        logits = logits + torch.movedim(table[s["index"]], 2, 0)
        if s["codes"] is not None:
            code = s["codes"][torch.arange(at, min(b, at + step), device=logits.device) % per]
            logits = torch.where((code[:, :, None] == code[:, None, :])[:, None], logits,
                                 logits - 100)
        out = torch.einsum("bhij,bjhd->bihd", torch.softmax(logits, -1), qkv[:, :, 2])
        out = out.reshape(out.shape[0], n, h * d)
        g_qkv, g_table = torch.autograd.grad(out, (qkv, table), s["grad"][at:at + step].double())
        outs.append(out.detach())
        grads.append(g_qkv)
        grad_table = grad_table + g_table
    return {"out": torch.cat(outs), "grad_qkv": torch.cat(grads), "grad_table": grad_table}


def _exact_norm(case, s, wide):
    norm = lambda x, p: torch.nn.functional.layer_norm(x, x.shape[-1:], *p, EPS)  # noqa: E731
    branch = wide(s["branch"])
    rows, c = branch.shape
    post = None if s["post"] is None else tuple(wide(t) for t in s["post"])
    pre = None if s["pre"] is None else tuple(wide(t) for t in s["pre"])
    gate = None if s["gate"] is None else wide(s["gate"])
    added = branch if post is None else norm(branch, post)
    if gate is not None:
        added = added * gate
    if s["scale"] is not None:
        added = (added.view(s["scale"].numel(), -1, c) * s["scale"].double()[:, None, None]
                 ).view(rows, c)
    if case["pass"] == "forward":
        out = s["residual"].double() + added
        kept = out.detach().to(s["residual"].dtype).double()
        return {"out": out.detach(),
                **({} if pre is None else {"normed": norm(kept, pre).detach()})}
    # out = residual + added, with the residual that gives the stored out
    residual = (s["out"].double() - added).detach().requires_grad_(True)
    out = residual + added
    ends, seeds = [out], [s["grad_out"].double()]
    names, leaves = ["residual", "branch"], [residual, branch]
    if pre is not None:
        ends.append(norm(out, pre))
        seeds.append(s["grad_normed"].double())
        names += ["pre_weight", "pre_bias"]
        leaves += list(pre)
    if gate is not None:
        names.append("gate")
        leaves.append(gate)
    if post is not None:
        names += ["post_weight", "post_bias"]
        leaves += list(post)
    return dict(zip(names, torch.autograd.grad(ends, leaves, seeds)))


def _exact_gelu(s, wide):
    gelu = torch.nn.functional.gelu
    x = s["x"].double()
    rows, c = x.shape
    kept = torch.nn.functional.pad(x, (0, -c % GROUP)).view(rows, -1, GROUP)
    top = kept.abs().amax(-1, keepdim=True)
    step = torch.where(top > 0, 2.0 ** torch.ceil(torch.log2(top / 127)).clamp(min=-126), 1.0)
    kept = wide((torch.round(kept / step) * step).view(rows, -1)[:, :c])
    again = gelu(kept)
    (grad,) = torch.autograd.grad(again, kept, s["grad"].double())
    return {"y": gelu(x), "grad_x": grad, "again": again.detach()}
