"""The operators at the model's end, as they are measured: log probabilities of
given tokens (with entropy and top alternatives) and their gradient, the
distillation loss with its gradient, and layer norm with its backward pass.

``run`` computes them in plain torch operations, or, with ``own`` set, by the
calls of the framework's C ABI on device buffers.  Token ids are int32 tensors
whose bits are the ABI's u32 (-1 is 0xFFFFFFFF: no token).
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5


def listed():
    return [
        # One decode step of one stream: the token just drawn, with 20 alternatives to show.  Latency.
        {"name": "logprobs_one_row", "op": "logprobs", "dtype": "f32", "rows": 1, "vocab": 32768, "pad": 0, "top": 20,
         "temperature": 1.0, "ignored": 0.0, "masked": 0.0},
        # Scoring a batch of prompts under a large vocabulary, alternatives kept for a student.
        {"name": "logprobs_long_rows", "op": "logprobs", "dtype": "bf16", "rows": 4096, "vocab": 131072, "pad": 0,
         "top": 20, "temperature": 1.0, "ignored": 0.0, "masked": 0.0},
        # A padded batch with an odd vocabulary, part of which a grammar rules out, at a sampling temperature.
        {"name": "logprobs_odd_padded", "op": "logprobs", "dtype": "f16", "rows": 1021, "vocab": 50021, "pad": 0,
         "top": 8, "temperature": 0.8, "ignored": 0.125, "masked": 0.25},
        # Policy gradient with an entropy bonus at the headline model's vocabulary.
        {"name": "logprobs_grad", "op": "logprobs_grad", "dtype": "f32", "rows": 4096, "vocab": 32768, "pad": 0,
         "top": 0, "temperature": 1.0, "ignored": 0.125, "masked": 0.0},
        # The same in half the bytes, rows that start at odd addresses.
        {"name": "logprobs_grad_odd", "op": "logprobs_grad", "dtype": "bf16", "rows": 2048, "vocab": 65537, "pad": 0,
         "top": 0, "temperature": 1.0, "ignored": 0.0, "masked": 0.0},
        # A held-out distillation loss of the smallest model, no gradient.
        {"name": "distill_loss_small", "op": "distill", "dtype": "f32", "rows": 256, "vocab": 1024, "pad": 0,
         "teacher": 8, "temperature": 1.0, "ignored": 0.0, "grad": False},
        # A student's training step on the long-prompt model's vocabulary, padded.
        {"name": "distill_grad", "op": "distill", "dtype": "f32", "rows": 4096, "vocab": 16384, "pad": 0,
         "teacher": 32, "temperature": 2.0, "ignored": 0.125, "grad": True},
        # The largest: a student's training step under a large vocabulary.
        {"name": "distill_grad_long_rows", "op": "distill", "dtype": "bf16", "rows": 8192, "vocab": 131072, "pad": 0,
         "teacher": 64, "temperature": 1.0, "ignored": 0.0, "grad": True},
        # One norm of a 64-stream decode step at the headline width.  Latency.
        {"name": "norm_step", "op": "norm", "dtype": "f32", "rows": 64, "width": 1024, "pad": 0, "rms": True},
        # A prompt chunk's norm at a generic large width.
        {"name": "norm_wide", "op": "norm", "dtype": "bf16", "rows": 16384, "width": 4096, "pad": 0, "rms": False},
        # A training batch's norm gradient at the headline width.
        {"name": "norm_grad", "op": "norm_grad", "dtype": "bf16", "rows": 65536, "width": 1024, "pad": 0, "rms": False},
        # Rows that no wide load fits.
        {"name": "norm_grad_odd", "op": "norm_grad", "dtype": "f32", "rows": 4099, "width": 767, "pad": 0,
         "rms": False},
    ]


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]; even and odd ones, powers of two now and then."""
    n = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    if rng.random() < 0.25:
        n = 2 ** round(math.log2(n))
    return max(lo, min(hi, int(n)))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "logprobs_grad", "distill", "distill", "norm", "norm_grad"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op.startswith("norm"):
        width = _spread(rng, 16, 16384)
        rows = _spread(rng, 1, max(1, min(65536, 200_000_000 // (width * SIZE[dtype]))))
        return {"op": op, "dtype": dtype, "rows": rows, "width": width, "pad": rng.choice([0, 0, 1, 8, 24]),
                "rms": rng.random() < 0.5}
    vocab = _spread(rng, 1000, 200_000)
    rows = _spread(rng, 1, max(1, min(16384, 1_000_000_000 // (vocab * SIZE[dtype]))))
    case = {"op": op, "dtype": dtype, "rows": rows, "vocab": vocab, "pad": rng.choice([0, 0, 1, 8, 24]),
            "temperature": rng.choice([1.0, 1.0, 0.7, 2.0, round(rng.uniform(0.5, 4.0), 3)]),
            "ignored": rng.choice([0.0, 0.0, 0.125, 0.4])}
    if op == "distill":
        case.update(teacher=_spread(rng, 1, 128), grad=rng.random() < 0.75)
    else:
        case.update(top=_spread(rng, 1, 128) if op == "logprobs" and rng.random() < 0.8 else 0,
                    masked=rng.choice([0.0, 0.0, 0.25, 0.9]))
    return case


def _n_ignored(case):
    return int(case["rows"] * case["ignored"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, dt = case["rows"], DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def empty(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    s = {"case": case}
    if case["op"].startswith("norm"):
        d, stride = case["width"], case["width"] + case["pad"]
        # Residual-stream rows: every row its own scale and offset.
        x = randn(rows, stride) * torch.exp(0.5 * randn(rows, 1)) + 0.3 * randn(rows, 1)
        s["x"] = x.to(dt)[:, :d]
        s["gain"] = 1.0 + 0.2 * randn(d)
        s["bias"] = None if case["rms"] else 0.1 * randn(d)
        s["y"] = empty(rows, d, dtype=dt)
        s["mean"] = None if case["rms"] else empty(rows)
        s["rstd"] = empty(rows)
        if case["op"] == "norm_grad":
            s["dy"] = (randn(rows, stride) * 0.01).to(dt)[:, :d]
            s["dx"] = empty(rows, d, dtype=dt)
            s["dgain"] = empty(d)
            s["dbias"] = None if case["rms"] else empty(d)
            # Room for 2 * 1024 partial rows, what the call asks for at most.
            s["workspace"] = empty(2048 * d)
            xf = s["x"].double()
            mean = xf.mean(-1) if not case["rms"] else torch.zeros(rows, device="cuda", dtype=torch.float64)
            s["rstd"].copy_(torch.rsqrt((xf - mean[:, None]).square().mean(-1) + EPS))
            if s["mean"] is not None:
                s["mean"].copy_(mean)
        return s

    V, stride = case["vocab"], case["vocab"] + case["pad"]
    z = empty(rows, stride, dtype=dt)
    ids = torch.randint(0, V, (rows,), generator=g, device="cuda")
    sure = torch.rand(rows, generator=g, device="cuda") < 0.6
    step = max(1, 100_000_000 // stride)
    for r in range(0, rows, step):
        z[r:r + step] = 2.0 * randn(min(step, rows - r), stride) - 3.0
    # A trained model is sure of most tokens.
    z[torch.arange(rows, device="cuda"), ids] += torch.where(sure, 14.0, 3.0).to(dt)
    skip = torch.randperm(rows, generator=g, device="cuda")[:_n_ignored(case)]
    s["logits"] = z[:, :V]
    if case["op"] == "distill":
        K = case["teacher"]
        # The teacher's K largest, in its order: distinct ids, the given token nearly always among them.
        start = torch.randint(0, V, (rows, 1), generator=g, device="cuda")
        t_ids = (start + (V // K) * torch.arange(K, device="cuda")) % V
        first = ids[:, None] == t_ids
        t_ids[:, 0] = torch.where(first.any(-1), t_ids[:, 0], ids)
        s["t_ids"] = t_ids.to(torch.int32)
        s["t_ids"][skip] = -1
        s["t_logits"] = torch.sort(2.0 * randn(rows, K) + 5.0, dim=-1, descending=True).values.to(dt).contiguous()
        s["weight"] = torch.rand(rows, generator=g, device="cuda") + 0.5
        s["loss"] = empty(rows)
        s["dlogits"] = empty(rows, V, dtype=dt) if case["grad"] else None
        return s

    if case["masked"]:
        # Columns that a grammar forbids, and the vocabulary's unused tail.
        dead = torch.rand(V, generator=g, device="cuda") < case["masked"]
        s["logits"].masked_fill_(dead, float("-inf"))
        kept = (1.0 + randn(rows)).to(dt)
        s["logits"].scatter_(1, ids[:, None], kept[:, None])
    s["targets"] = ids.to(torch.int32)
    s["targets"][skip] = -1
    s["logprob"], s["entropy"], s["stats"] = empty(rows), empty(rows), empty(rows, 2)
    if case["op"] == "logprobs":
        s["top_ids"] = empty(rows, case["top"], dtype=torch.int32) if case["top"] else None
        s["top_logprobs"] = empty(rows, case["top"]) if case["top"] else None
    else:
        # What the forward call leaves.
        st, ent = _exact_stats(s["logits"], case["temperature"])
        gone = s["targets"] < 0
        s["stats"].copy_(st.masked_fill(gone[:, None], 0.0))
        s["entropy"].copy_(ent.masked_fill(gone, 0.0))
        s["g_logprob"] = randn(rows) / rows
        s["g_entropy"] = 0.01 * torch.rand(rows, generator=g, device="cuda") / rows
        s["dlogits"] = empty(rows, V, dtype=dt)
    return s


# ---------------------------------------------------------------- plain forms
def _plain_logprobs(s):
    c = s["case"]
    z = s["logits"].float()
    m = z.amax(-1, keepdim=True)
    d = (z - m) / c["temperature"]
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    log_s = torch.log(total)
    entropy = log_s[:, 0] - torch.where(e > 0, e * d, 0.0).sum(-1) / total[:, 0]
    given = s["targets"].long()
    gone = given < 0
    logprob = (d.gather(1, given.clamp(min=0)[:, None]) - log_s)[:, 0]
    out = {"logprob": logprob.masked_fill(gone, 0.0), "entropy": entropy.masked_fill(gone, 0.0),
           "stats": torch.cat([m, log_s], 1).masked_fill(gone[:, None], 0.0)}
    if c["top"]:
        # Value first, then the lower index: one whole-number key for both.
        bits = (z + 0.0).view(torch.int32).long()
        bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        key = (bits << 32) + (0xFFFFFFFF - torch.arange(z.shape[1], device=z.device))
        key = torch.topk(key, min(c["top"], z.shape[1]), dim=-1).values
        ids = 0xFFFFFFFF - (key & 0xFFFFFFFF)
        top = d.gather(1, ids) - log_s
        none = torch.isinf(top) | gone[:, None]
        out["top_ids"] = ids.masked_fill(none, -1).to(torch.int32)
        out["top_logprobs"] = top.masked_fill(none, float("-inf"))
    return out


def _plain_logprobs_grad(s):
    T = s["case"]["temperature"]
    z = s["logits"].float()
    y = (z - s["stats"][:, :1]) / T - s["stats"][:, 1:]
    p = torch.exp(y)
    gl, ge = s["g_logprob"][:, None], s["g_entropy"][:, None]
    dz = -p * gl - torch.where(p > 0, p * (y + s["entropy"][:, None]), 0.0) * ge
    given = s["targets"].long()[:, None]
    dz.scatter_add_(1, given.clamp(min=0), gl)
    return {"dlogits": (dz / T).masked_fill(given < 0, 0.0).to(s["logits"].dtype)}


def _plain_distill(s):
    c = s["case"]
    T = c["temperature"]
    z = s["logits"].float()
    ids = s["t_ids"].long()
    none = ids < 0
    gone = none.all(-1)
    t = (s["t_logits"].float() / T).masked_fill(none, float("-inf")).masked_fill(gone[:, None], 0.0)
    t = t - t.amax(-1, keepdim=True)
    logq = t - torch.log(torch.exp(t).sum(-1, keepdim=True))
    q = torch.exp(logq)
    y = (z - z.amax(-1, keepdim=True)) / T
    y = y - torch.log(torch.exp(y).sum(-1, keepdim=True))
    kl = torch.where(q > 0, q * (logq - y.gather(1, ids.clamp(min=0))), 0.0).sum(-1)
    out = {"loss": (T * T * kl).masked_fill(gone, 0.0)}
    if c["grad"]:
        dz = torch.exp(y)
        dz.scatter_add_(1, ids.clamp(min=0), -q.masked_fill(none, 0.0))
        dz *= (T * s["weight"] / z.shape[0]).masked_fill(gone, 0.0)[:, None]
        out["dlogits"] = dz.to(s["logits"].dtype)
    return out


def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(-1, keepdim=True) if s["mean"] is not None else torch.zeros_like(x[:, :1])
    rstd = torch.rsqrt((x - mean).square().mean(-1, keepdim=True) + EPS)
    y = (x - mean) * rstd * s["gain"]
    out = {"rstd": rstd[:, 0]}
    if s["mean"] is not None:
        y = y + s["bias"]
        out["mean"] = mean[:, 0]
    out["y"] = y.to(s["x"].dtype)
    return out


def _plain_norm_grad(s):
    dy = s["dy"].float()
    rstd = s["rstd"][:, None]
    xh = (s["x"].float() - (s["mean"][:, None] if s["mean"] is not None else 0.0)) * rstd
    c = dy * s["gain"]
    dx = c - xh * (c * xh).mean(-1, keepdim=True)
    out = {"dgain": (dy * xh).sum(0)}
    if s["mean"] is not None:
        dx = dx - c.mean(-1, keepdim=True)
        out["dbias"] = dy.sum(0)
    out["dx"] = (dx * rstd).to(s["x"].dtype)
    return out


# ---------------------------------------------------------------- the framework's calls
def _ptr(t):
    return None if t is None else t.data_ptr()


def _own_logprobs(nb, s, stream):
    c, z = s["case"], s["logits"]
    nb._check(nb.lib().nk_token_logprobs_device(
        z.data_ptr(), CODES[c["dtype"]], c["rows"], c["vocab"], z.stride(0), s["targets"].data_ptr(),
        c["temperature"], c["top"], s["logprob"].data_ptr(), s["entropy"].data_ptr(), s["stats"].data_ptr(),
        _ptr(s["top_ids"]), _ptr(s["top_logprobs"]), stream))
    out = {"logprob": s["logprob"], "entropy": s["entropy"], "stats": s["stats"]}
    if c["top"]:
        out.update(top_ids=s["top_ids"], top_logprobs=s["top_logprobs"])
    return out


def _own_logprobs_grad(nb, s, stream):
    c, z = s["case"], s["logits"]
    nb._check(nb.lib().nk_token_logprobs_backward_device(
        z.data_ptr(), CODES[c["dtype"]], c["rows"], c["vocab"], z.stride(0), s["targets"].data_ptr(),
        c["temperature"], s["stats"].data_ptr(), s["entropy"].data_ptr(), s["g_logprob"].data_ptr(),
        s["g_entropy"].data_ptr(), s["dlogits"].data_ptr(), s["dlogits"].stride(0), stream))
    return {"dlogits": s["dlogits"]}


def _own_distill(nb, s, stream):
    c, z, dz = s["case"], s["logits"], s["dlogits"]
    code = CODES[c["dtype"]]
    nb._check(nb.lib().nk_distill_device(
        z.data_ptr(), code, c["rows"], c["vocab"], z.stride(0), s["t_ids"].data_ptr(), s["t_logits"].data_ptr(), code,
        c["teacher"], c["temperature"], s["loss"].data_ptr(), s["weight"].data_ptr(), 1.0 / c["rows"], _ptr(dz),
        0 if dz is None else dz.stride(0), stream))
    return {"loss": s["loss"]} if dz is None else {"loss": s["loss"], "dlogits": dz}


def _own_norm(nb, s, stream):
    c, x, y = s["case"], s["x"], s["y"]
    nb._check(nb.lib().nk_layer_norm_device(
        x.data_ptr(), CODES[c["dtype"]], c["rows"], c["width"], x.stride(0), s["gain"].data_ptr(), _ptr(s["bias"]),
        EPS, int(c["rms"]), y.data_ptr(), y.stride(0), _ptr(s["mean"]), s["rstd"].data_ptr(), stream))
    out = {"rstd": s["rstd"], "y": y}
    if not c["rms"]:
        out["mean"] = s["mean"]
    return out


def _own_norm_grad(nb, s, stream):
    c, x, dy, dx = s["case"], s["x"], s["dy"], s["dx"]
    nb._check(nb.lib().nk_layer_norm_backward_device(
        x.data_ptr(), CODES[c["dtype"]], c["rows"], c["width"], x.stride(0), s["gain"].data_ptr(), _ptr(s["mean"]),
        s["rstd"].data_ptr(), int(c["rms"]), dy.data_ptr(), dy.stride(0), dx.data_ptr(), dx.stride(0),
        s["dgain"].data_ptr(), _ptr(s["dbias"]), 0, s["workspace"].data_ptr(), 4 * s["workspace"].numel(), stream))
    out = {"dgain": s["dgain"], "dx": dx}
    if not c["rms"]:
        out["dbias"] = s["dbias"]
    return out


PLAIN = {"logprobs": _plain_logprobs, "logprobs_grad": _plain_logprobs_grad, "distill": _plain_distill,
         "norm": _plain_norm, "norm_grad": _plain_norm_grad}
OWN = {"logprobs": _own_logprobs, "logprobs_grad": _own_logprobs_grad, "distill": _own_distill, "norm": _own_norm,
       "norm_grad": _own_norm_grad}


def run(state):
    op = state["case"]["op"]
    if own:
        import noetic_b200 as nb

        return OWN[op](nb, state, torch.cuda.current_stream().cuda_stream)
    return PLAIN[op](state)


def work(case):
    rows, b = case["rows"], SIZE[case["dtype"]]
    if case["op"] == "norm":
        n = rows * case["width"]
        return {"bytes": 2 * n * b + 8 * case["width"] + 8 * rows, "flops": 7 * n}
    if case["op"] == "norm_grad":
        n = rows * case["width"]
        return {"bytes": 3 * n * b + 12 * case["width"] + 8 * rows, "flops": 14 * n}
    live, n = rows - _n_ignored(case), (rows - _n_ignored(case)) * case["vocab"]
    if case["op"] == "logprobs":
        return {"bytes": n * b + 20 * rows + 8 * rows * case["top"], "flops": 7 * n}
    if case["op"] == "logprobs_grad":
        return {"bytes": n * b + rows * case["vocab"] * b + 24 * rows, "flops": 8 * n}
    grad = case["grad"]
    return {"bytes": n * b + (rows * case["vocab"] * b if grad else 0) + rows * case["teacher"] * (4 + b) + 8 * rows,
            "flops": (9 if grad else 5) * n + 6 * live * case["teacher"]}


# ---------------------------------------------------------------- in 64 bits, from the definitions
def _blocks(rows, width):
    step = max(1, 50_000_000 // width)
    return [slice(r, min(rows, r + step)) for r in range(0, rows, step)]


def _exact_stats(logits, T):
    """(maximum, log of the sum relative to it) and the entropy of each row, in 64 bits."""
    stats, ent = [], []
    for b in _blocks(*logits.shape):
        z = logits[b].double()
        m = z.max(-1).values
        y = z / T - torch.logsumexp(z / T, -1, keepdim=True)
        stats.append(torch.stack([m, torch.logsumexp(z / T, -1) - m / T], 1))
        ent.append(torch.special.entr(torch.exp(y)).sum(-1))
    return torch.cat(stats), torch.cat(ent)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x = s["x"].double()
        out = {}
        if case["rms"]:
            var = (x * x).sum(-1) / x.shape[1]
        else:
            var, out["mean"] = torch.var_mean(x, -1, correction=0)
            x = x - out["mean"][:, None]
        out["rstd"] = 1.0 / torch.sqrt(var + EPS)
        y = x * out["rstd"][:, None] * s["gain"].double()
        out["y"] = y if case["rms"] else y + s["bias"].double()
        return out
    if case["op"] == "norm_grad":
        # From the statistics that the call is given, which are 32-bit inputs.
        x, dy, r = s["x"].double(), s["dy"].double(), s["rstd"].double()[:, None]
        n = x.shape[1]
        if not case["rms"]:
            x = x - s["mean"].double()[:, None]
        c = dy * s["gain"].double()
        along = (c * x).sum(-1, keepdim=True) * r * r * r / n
        out = {"dgain": torch.einsum("rd,rd,r->d", dy, x, r[:, 0]), "dx": c * r - x * along}
        if not case["rms"]:
            out["dx"] -= c.sum(-1, keepdim=True) * r / n
            out["dbias"] = torch.einsum("rd->d", dy)
        return out

    T, blocks = case["temperature"], _blocks(case["rows"], case["vocab"])
    if case["op"] == "distill":
        loss, grads = [], []
        for b in blocks:
            z, ids, t = s["logits"][b].double() / T, s["t_ids"][b].long(), s["t_logits"][b].double() / T
            live = ids >= 0
            logq = torch.where(live, t - torch.logsumexp(torch.where(live, t, -torch.inf), -1, keepdim=True), 0.0)
            q = torch.where(live, torch.exp(logq), 0.0)
            lse = torch.logsumexp(z, -1, keepdim=True)
            at = torch.gather(z, 1, torch.where(live, ids, 0)) - lse
            loss.append(T * T * (q * (logq - at)).sum(-1))
            if case["grad"]:
                p = torch.exp(z - lse) * live.any(-1, keepdim=True)
                p -= torch.zeros_like(p).scatter_add_(1, torch.where(live, ids, 0), q)
                grads.append(p * (T / case["rows"]) * s["weight"][b].double()[:, None])
        out = {"loss": torch.cat(loss)}
        if grads:
            out["dlogits"] = torch.cat(grads)
        return out

    given = s["targets"].long()
    if case["op"] == "logprobs_grad":
        # From the maximum, log-sum and entropy that the call is given, which are 32-bit inputs.
        out = []
        for b in blocks:
            z, st, t = s["logits"][b].double(), s["stats"][b].double(), given[b]
            logp = (z - st[:, :1]) / T - st[:, 1:]
            p = torch.exp(logp)
            hot = torch.zeros_like(p).scatter_(1, t.clamp(min=0)[:, None], 1.0)
            of_h = -(torch.xlogy(p, p) + p * s["entropy"][b].double()[:, None])
            dz = (hot - p) * s["g_logprob"][b].double()[:, None] + of_h * s["g_entropy"][b].double()[:, None]
            out.append(dz * (t >= 0)[:, None] / T)
        return {"dlogits": torch.cat(out)}

    stats, ent = _exact_stats(s["logits"], T)
    gone = given < 0
    out = {"stats": stats, "entropy": ent}
    z_t = s["logits"].gather(1, given.clamp(min=0)[:, None])[:, 0].double()
    out["logprob"] = (z_t - stats[:, 0]) / T - stats[:, 1]
    if case["top"]:
        ids, top = [], []
        for b in blocks:
            v, i = torch.sort(s["logits"][b].double(), dim=-1, descending=True, stable=True)
            v, i = v[:, :case["top"]], i[:, :case["top"]]
            none = (v == -torch.inf) | gone[b][:, None]
            top.append(torch.where(none, -torch.inf, (v - stats[b, :1]) / T - stats[b, 1:]))
            ids.append(torch.where(none, -1, i).to(torch.int32))
        out["top_logprobs"], out["top_ids"] = torch.cat(top), torch.cat(ids)
    for name in ("stats", "entropy", "logprob"):
        out[name][gone] = 0.0
    return out
