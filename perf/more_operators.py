"""The operators of a training step's end, as they are measured: softmax cross
entropy straight from hidden rows and the (tied) vocabulary matrix, without
keeping the logits, its gradients for both, and one AdamW step over a whole
model's tensors, with moments in 32 or in 8 bits and the gradients' norm
clipped.

``run`` computes them in plain torch operations, or, with ``own`` set, by the
calls of the framework's C ABI on device buffers.  Token ids are int32 tensors
whose bits are the ABI's u32 (-1 is 0xFFFFFFFF: no token).
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "none": 0}
BLOCK = 256  # elements that share a scale of the 8-bit moments
E4M3_MAX = 448.0
B1, B2, EPS, LR, WD, T = 0.9, 0.95, 1e-8, 3e-4, 0.1, 100


def listed():
    return [
        # The surprisal of one stream's next token at the headline model's size.  Latency.
        {"name": "ce_one_row", "op": "ce", "dtype": "f32", "rows": 1, "width": 1024, "vocab": 32768, "pad": 0,
         "ignored": 0.0},
        # A held-out loss of the smallest model.
        {"name": "ce_small", "op": "ce", "dtype": "f32", "rows": 256, "width": 192, "vocab": 1024, "pad": 0,
         "ignored": 0.0},
        # A held-out loss under a large vocabulary.
        {"name": "ce_long_vocab", "op": "ce", "dtype": "bf16", "rows": 4096, "width": 2048, "vocab": 131072, "pad": 0,
         "ignored": 0.0},
        # A padded batch, odd sizes, rows that start at odd addresses.
        {"name": "ce_odd_padded", "op": "ce", "dtype": "f16", "rows": 1021, "width": 767, "vocab": 50021, "pad": 1,
         "ignored": 0.125},
        # A training batch of the headline model.
        {"name": "ce_grad", "op": "ce_grad", "dtype": "bf16", "rows": 8192, "width": 1024, "vocab": 32768, "pad": 0,
         "ignored": 0.0},
        # A padded training batch of the long-prompt model, in its own type.
        {"name": "ce_grad_f32", "op": "ce_grad", "dtype": "f32", "rows": 4096, "width": 768, "vocab": 16384, "pad": 0,
         "ignored": 0.125},
        # Odd sizes.
        {"name": "ce_grad_odd", "op": "ce_grad", "dtype": "f16", "rows": 1531, "width": 1000, "vocab": 32003, "pad": 3,
         "ignored": 0.0},
        # The largest: a training batch under a large vocabulary.
        {"name": "ce_grad_long_vocab", "op": "ce_grad", "dtype": "bf16", "rows": 8192, "width": 2048, "vocab": 131072,
         "pad": 0, "ignored": 0.0},
        # The step of the smallest model: few bytes, many tensors.  Latency.
        {"name": "adamw_small", "op": "adamw", "bits": 32, "layers": 3, "width": 192, "vocab": 1024, "grad": "f32",
         "copy": "none", "clip": 0.0},
        # The step of the headline model, everything in 32 bits, clipped.
        {"name": "adamw_32", "op": "adamw", "bits": 32, "layers": 24, "width": 1024, "vocab": 32768, "grad": "f32",
         "copy": "none", "clip": 1.0},
        # The same with moments in 8 bits, 16-bit gradients and a 16-bit copy of the weights for the next pass.
        {"name": "adamw_8", "op": "adamw", "bits": 8, "layers": 24, "width": 1024, "vocab": 32768, "grad": "bf16",
         "copy": "bf16", "clip": 1.0},
        # Tensors of odd sizes whose last blocks are short.
        {"name": "adamw_8_odd", "op": "adamw", "bits": 8, "layers": 11, "width": 333, "vocab": 10007, "grad": "f32",
         "copy": "f16", "clip": 0.0},
    ]


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]; even and odd ones, powers of two now and then."""
    n = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    if rng.random() < 0.25:
        n = 2 ** round(math.log2(n))
    return max(lo, min(hi, int(n)))


def draw(rng):
    op = rng.choice(["ce", "ce", "ce_grad", "ce_grad", "adamw"])
    if op == "adamw":
        return {"op": op, "bits": rng.choice([32, 8]), "layers": _spread(rng, 1, 24), "width": _spread(rng, 32, 1024),
                "vocab": _spread(rng, 1000, 32768), "grad": rng.choice(["f32", "f16", "bf16"]),
                "copy": rng.choice(["none", "f16", "bf16"]), "clip": rng.choice([0.0, 1.0, 0.25])}
    dtype = rng.choice(["f32", "f16", "bf16"])
    width, vocab = _spread(rng, 32, 4096), _spread(rng, 1000, 131072)
    most = 2048 * 131072 * (4096 if op == "ce" else 8192) // (1 if dtype != "f32" else 4)
    rows = _spread(rng, 1 if op == "ce" else 64, max(64, min(16384, most // (width * vocab), (1 << 30) // vocab)))
    return {"op": op, "dtype": dtype, "rows": rows, "width": width, "vocab": vocab, "pad": rng.choice([0, 0, 0, 1, 8]),
            "ignored": rng.choice([0.0, 0.0, 0.125, 0.4])}


def _n_ignored(case):
    return int(case["rows"] * case["ignored"])


def _sizes(case):
    """(elements, whether weight decay applies) of each tensor of a model of this framework."""
    d, v = case["width"], case["vocab"]
    layer = [(d, False), (3 * d * d, True), (3 * d, False), (4 * d, True), (d, False), (d * d, True), (d, False),
             (d, False), (6 * d * d, True), (6 * d, False), (3 * d * d, True), (d, False)]
    return [(v * d, True)] + layer * case["layers"] + [(d, False)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def empty(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    s = {"case": case}
    if case["op"] == "adamw":
        # Every tensor starts at a block of its own in one allocation for each array.
        sizes = _sizes(case)
        blocks = [-(-n // BLOCK) for n, _ in sizes]
        s["sizes"], s["blocks"] = sizes, torch.tensor(blocks, device="cuda")
        s["decay"] = torch.tensor([float(w) for _, w in sizes], device="cuda")
        nb = sum(blocks)
        used = torch.tensor([n for n, _ in sizes], device="cuda")
        start = torch.cumsum(s["blocks"], 0) - s["blocks"]
        tensor = torch.repeat_interleave(torch.arange(len(sizes), device="cuda"), s["blocks"], output_size=nb)
        left = used[tensor] - (torch.arange(nb, device="cuda") - start[tensor]) * BLOCK
        room = torch.arange(BLOCK, device="cuda") < left[:, None]
        s["val"] = 0.02 * randn(nb, BLOCK) * room
        # Gradients whose sizes differ from row to row by orders of magnitude.
        grad = randn(nb, BLOCK) * torch.exp(1.5 * randn(nb, 1) - 9.0) * room
        m = 0.3 * grad + 0.3 * randn(nb, BLOCK) * grad.abs()
        v = grad.square() * torch.exp(randn(nb, BLOCK))
        s["grad"] = grad.to(DTYPES[case["grad"]])
        del grad, room, left
        if case["bits"] == 32:
            s["m"], s["v"] = m, v
        else:
            u = torch.sqrt(v)
            s["m_scale"], s["v_scale"] = m.abs().amax(1) / E4M3_MAX, u.amax(1) / E4M3_MAX
            s["m"] = (m / s["m_scale"].clamp(min=1e-30)[:, None]).to(torch.float8_e4m3fn)
            s["v"] = (u / s["v_scale"].clamp(min=1e-30)[:, None]).to(torch.float8_e4m3fn)
        s["copy"] = empty(nb, BLOCK, dtype=DTYPES[case["copy"]]).zero_() if case["copy"] != "none" else None
        s["norm"] = empty(1) if case["clip"] else None
        return s

    rows, d, V, dt = case["rows"], case["width"], case["vocab"], DTYPES[case["dtype"]]
    # Logits of a spread of about 2, a trained model's: sure of most tokens.
    w = empty(V, d + case["pad"], dtype=dt)
    w.copy_(randn(V, d + case["pad"]) * (2.0 / math.sqrt(d)))
    s["w"] = w[:, :d]
    ids = torch.randint(0, V, (rows,), generator=g, device="cuda")
    sure = torch.rand(rows, 1, generator=g, device="cuda") < 0.6
    along = s["w"][ids].float()
    along = along / along.norm(dim=1, keepdim=True)
    x = randn(rows, d + case["pad"])
    x[:, :d] += torch.where(sure, 6.0, 1.5) * along
    s["x"] = x.to(dt)[:, :d]
    s["targets"] = ids.to(torch.int32)
    s["targets"][torch.randperm(rows, generator=g, device="cuda")[:_n_ignored(case)]] = -1
    s["loss"], s["stats"] = empty(rows), empty(rows, 2)
    if case["op"] == "ce_grad":
        # What the forward call leaves.
        stats, _ = _exact_rows(s)
        s["stats"].copy_(stats)
        s["weight"] = torch.rand(rows, generator=g, device="cuda") + 0.5
        s["dx"], s["dw"] = empty(rows, d, dtype=dt), empty(V, d, dtype=dt)
    return s


# ---------------------------------------------------------------- plain forms
def _plain_ce(s):
    z = s["x"].float() @ s["w"].float().T
    m = z.amax(-1, keepdim=True)
    z -= m
    given = s["targets"].long()
    gone = given < 0
    at = z.gather(1, given.clamp(min=0)[:, None])
    log_s = torch.log(torch.exp(z).sum(-1, keepdim=True))
    return {"loss": (log_s - at)[:, 0].masked_fill(gone, 0.0),
            "stats": torch.cat([m, log_s], 1).masked_fill(gone[:, None], 0.0)}


def _plain_ce_grad(s):
    x, w = s["x"].float(), s["w"].float()
    given = s["targets"].long()
    p = torch.exp((x @ w.T - s["stats"][:, :1]) - s["stats"][:, 1:])
    p.scatter_add_(1, given.clamp(min=0)[:, None], torch.full_like(s["stats"][:, :1], -1.0))
    p *= (s["weight"] / x.shape[0]).masked_fill(given < 0, 0.0)[:, None]
    return {"dx": (p @ w).to(s["x"].dtype), "dw": (p.T @ x).to(s["w"].dtype)}


def _f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


def _bias(b):
    """1 / (1 - b^t), rounded to 32 bits at each step."""
    one = torch.tensor(1.0)
    return float(one / (one - torch.tensor(b) ** T))


def _plain_adamw(s):
    c = s["case"]
    g = s["grad"].float()
    if c["clip"]:
        s["norm"].copy_(torch.sqrt(torch.sum(g.double().square())))
        g = g * torch.where(s["norm"] > c["clip"], c["clip"] / s["norm"], 1.0)
    small = c["bits"] == 8
    m = s["m"].float() * s["m_scale"][:, None] if small else s["m"]
    v = (s["v"].float() * s["v_scale"][:, None]).square() if small else s["v"]
    m = m * B1 + g * (1.0 - _f32(B1))
    v = v * B2 + (g * (1.0 - _f32(B2))) * g
    val = s["val"]
    step = (m * _bias(B1)) / (torch.sqrt(v * _bias(B2)) + EPS)
    decay = torch.repeat_interleave(s["decay"], s["blocks"], output_size=val.shape[0])[:, None]
    step += decay * (val * WD)
    val -= step * LR
    if small:
        u = torch.sqrt(v)
        for name, x in (("m", m), ("v", u)):
            top = x.abs().amax(1)
            y = x * torch.where(top > 0, E4M3_MAX / top, 0.0)[:, None]
            # A second moment that is not zero stays above zero.
            y = torch.where((x > 0) & (y < 2.0 ** -9), 2.0 ** -9, y) if name == "v" else y
            s[name].copy_(y.to(torch.float8_e4m3fn))
            s[name + "_scale"].copy_(top / E4M3_MAX)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    if s["copy"] is not None:
        s["copy"].copy_(val)
    return _adamw_out(s)


def _adamw_out(s):
    return {k: s[k] for k in ("val", "m", "v", "m_scale", "v_scale", "copy", "norm") if s.get(k) is not None}


# ---------------------------------------------------------------- the framework's calls
def _workspace(nb, s, backward):
    """The workspace that a program keeps for its calls of these sizes."""
    if "workspace" not in s:
        c = s["case"]
        n = nb.train.linear_ce_workspace(CODES[c["dtype"]], c["rows"], c["width"], c["vocab"], s["w"].data_ptr(),
                                         s["w"].stride(0), backward)
        s["workspace"] = torch.empty(n, dtype=torch.uint8, device="cuda")
    return s["workspace"]


def _own_ce(nb, s, stream):
    c, x, w = s["case"], s["x"], s["w"]
    room = _workspace(nb, s, False)
    nb._check(nb.lib().nk_linear_ce_device(
        x.data_ptr(), CODES[c["dtype"]], c["rows"], c["width"], x.stride(0), w.data_ptr(), c["vocab"], w.stride(0),
        s["targets"].data_ptr(), s["loss"].data_ptr(), s["stats"].data_ptr(), room.data_ptr(), room.numel(), stream))
    return {"loss": s["loss"], "stats": s["stats"]}


def _own_ce_grad(nb, s, stream):
    c, x, w, dx, dw = s["case"], s["x"], s["w"], s["dx"], s["dw"]
    room = _workspace(nb, s, True)
    code = CODES[c["dtype"]]
    nb._check(nb.lib().nk_linear_ce_backward_device(
        x.data_ptr(), code, c["rows"], c["width"], x.stride(0), w.data_ptr(), c["vocab"], w.stride(0),
        s["targets"].data_ptr(), s["stats"].data_ptr(), s["weight"].data_ptr(), 1.0 / c["rows"], dx.data_ptr(),
        dx.stride(0), dw.data_ptr(), code, dw.stride(0), 0, room.data_ptr(), room.numel(), stream))
    return {"dx": dx, "dw": dw}


def _own_adamw(nb, s, stream):
    c = s["case"]
    if "plan" not in s:
        # The tensors that a program registers once, before its first step.
        small, copy, at, tensors = c["bits"] == 8, s["copy"], 0, []
        for n, decay in s["sizes"]:
            tensors.append(nb.train.AdamwTensor(
                val=s["val"][at].data_ptr(), grad=s["grad"][at].data_ptr(), m=s["m"][at].data_ptr(),
                v=s["v"][at].data_ptr(), m_scale=s["m_scale"][at:].data_ptr() if small else None,
                v_scale=s["v_scale"][at:].data_ptr() if small else None,
                copy=None if copy is None else copy[at].data_ptr(), n=n, grad_dtype=CODES[c["grad"]],
                copy_dtype=0 if copy is None else CODES[c["copy"]], state_bits=c["bits"], decay=int(decay)))
            at += -(-n // BLOCK)
        s["plan"] = nb.train.AdamwMany(tensors)
    s["plan"].step(lr=LR, t=T, b1=B1, b2=B2, eps=EPS, wd=WD, max_norm=c["clip"],
                   norm=None if s["norm"] is None else s["norm"].data_ptr(), stream=stream)
    return _adamw_out(s)


PLAIN = {"ce": _plain_ce, "ce_grad": _plain_ce_grad, "adamw": _plain_adamw}
OWN = {"ce": _own_ce, "ce_grad": _own_ce_grad, "adamw": _own_adamw}


def run(state):
    op = state["case"]["op"]
    if own:
        import noetic_b200 as nb

        return OWN[op](nb, state, torch.cuda.current_stream().cuda_stream)
    return PLAIN[op](state)


def work(case):
    if case["op"] == "adamw":
        n = sum(n for n, _ in _sizes(case))
        blocks = sum(-(-n // BLOCK) for n, _ in _sizes(case))
        small = case["bits"] == 8
        return {"bytes": n * (8 + SIZE[case["grad"]] + SIZE[case["copy"]] + (4 if small else 16)) + 16 * blocks * small,
                "flops": (18 + 12 * small) * n}
    rows, d, V, b = case["rows"], case["width"], case["vocab"], SIZE[case["dtype"]]
    live = rows - _n_ignored(case)
    if case["op"] == "ce":
        return {"bytes": (live + V) * d * b + 16 * rows, "flops": live * V * (2 * d + 4)}
    return {"bytes": (live + V) * d * b + (rows + V) * d * b + 16 * rows, "flops": live * V * (6 * d + 5)}


# ---------------------------------------------------------------- in 64 bits, from the definitions
def _row_blocks(s):
    rows, step = s["x"].shape[0], max(1, 250_000_000 // s["w"].shape[0])
    return [slice(r, min(rows, r + step)) for r in range(0, rows, step)]


def _exact_rows(s):
    """(maximum, log of the sum relative to it) and the loss of each row, in 64 bits."""
    w, stats, loss = s["w"].double(), [], []
    for b in _row_blocks(s):
        z = torch.einsum("rd,vd->rv", s["x"][b].double(), w)
        t = s["targets"][b].long()
        lse, m = torch.logsumexp(z, -1), z.max(-1).values
        live = t >= 0
        loss.append(torch.where(live, lse - torch.gather(z, 1, torch.where(live, t, 0)[:, None])[:, 0], 0.0))
        stats.append(torch.stack([m, lse - m], 1) * live[:, None])
    return torch.cat(stats), torch.cat(loss)


def _grid(y):
    """The nearest values of 4 exponent and 3 fraction bits (ties to even), |y| <= 448, steps of 2^-9 near zero."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "ce":
        stats, loss = _exact_rows(s)
        return {"loss": loss, "stats": stats}
    if case["op"] == "ce_grad":
        # From the statistics that the call is given, which are 32-bit inputs.
        w, dx, dw = s["w"].double(), [], 0.0
        for b in _row_blocks(s):
            x, st, t = s["x"][b].double(), s["stats"][b].double(), s["targets"][b].long()
            live = t >= 0
            dz = torch.exp(torch.einsum("rd,vd->rv", x, w) - st.sum(1, keepdim=True))
            dz[torch.arange(len(t), device="cuda"), torch.where(live, t, 0)] -= 1.0
            dz *= torch.where(live, s["weight"][b].double() / case["rows"], 0.0)[:, None]
            dx.append(torch.einsum("rv,vd->rd", dz, w))
            dw = dw + torch.einsum("rv,rd->vd", dz, x)
        return {"dx": torch.cat(dx), "dw": dw}
    small, out = case["bits"] == 8, {}
    g, scale = s["grad"].double(), 1.0
    if case["clip"]:
        out["norm"] = torch.linalg.vector_norm(g).reshape(1)
        scale = min(1.0, case["clip"] / float(out["norm"]))
    b1, b2, lr, wd = _f32(B1), _f32(B2), _f32(LR), _f32(WD)
    m, v = s["m"].double(), s["v"].double()
    if small:
        m, v = m * s["m_scale"].double()[:, None], (v * s["v_scale"].double()[:, None]) ** 2
    m = b1 * m + (1 - b1) * scale * g
    v = b2 * v + (1 - b2) * (scale * g) ** 2
    del g
    val = s["val"].double()
    decay = torch.cat([torch.full((-(-n // BLOCK),), float(w)) for n, w in s["sizes"]]).cuda().double()[:, None]
    out["val"] = val - lr * (m / (1 - b1 ** T) / (torch.sqrt(v / (1 - b2 ** T)) + _f32(EPS)) + wd * decay * val)
    if small:
        for name, x in (("m", m), ("v", torch.sqrt(v))):
            top = x.abs().amax(1)
            y = _grid(torch.nan_to_num(x * E4M3_MAX / top[:, None]))
            out[name] = torch.where((x > 0) & (y == 0), 2.0 ** -9, y) if name == "v" else y
            out[name + "_scale"] = top / E4M3_MAX
    else:
        out["m"], out["v"] = m, v
    if s["copy"] is not None:
        out["copy"] = out["val"]
    return out
