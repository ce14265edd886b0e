"""The operators at the model's end (include/noetic/head.h) on the GPU against
their definitions in 64 bits: log probabilities with entropy and alternatives,
distillation, layer norm and RMSNorm, and their gradients.

Tolerances count roundings.  U = 2^-24 is half a step of f32.
 - y = (z - m) / T costs a rounding of the difference, one of the product with
   log2(e) / T, one of that constant and one more in a later difference, 4 |y| U in
   all; 2^y by the special-function unit 2^-22 = 4 U; a sum of N terms in which every
   term passes through at most N / 256 + 40 additions that many U.  So a row's
   sum s is off by at most REL = (4 Y + N / 256 + 48) U of itself, Y the largest |y|
   of a term that is not below 2^-24 / N of the sum (smaller ones add nothing).
 - a result of a narrower type is off by half a step more: eps / 2 of it, or
   half of the smallest subnormal.
"""

import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0**-24
NONE = -1  # 0xFFFFFFFF as int32
INF, NAN = float("inf"), float("nan")
CODE = {"f32": 0, "f16": 1, "bf16": 2}


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


def _dt(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _st(torch):
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _matrix(torch, rows, width, dtype, pad=0, shift=0, scale=3.0, seed=0, offset=0.0):
    """A [rows, width] view whose rows start `shift` elements into an array of
    row stride width + pad, and that whole array (NaN around the rows)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    whole = torch.full((shift + rows * (width + pad) + 8,), NAN, device="cuda", dtype=_dt(torch, dtype))
    v = whole[shift:shift + rows * (width + pad)].view(rows, width + pad)[:, :width]
    v.copy_(torch.randn(rows, width, generator=g, device="cuda") * scale + offset)
    return v, whole


def _out_tol(torch, dtype, ref):
    """Half a step of the output type."""
    if dtype == "f32":
        return U * ref.abs()
    f = torch.finfo(_dt(torch, dtype))
    return (f.eps / 2) * ref.abs() + f.smallest_normal * f.eps / 2


def _sum_rel(n, y):
    return (4 * y + n / 256 + 48) * U


def _span(n):
    """Y: terms of a sum below 2^-24 / N of it do not matter."""
    return np.log(2.0**24 * n)


# ---------------------------------------------------------------- log probabilities
def _logprobs(nb, torch, z, targets, T, top, dtype):
    rows, V = z.shape
    f = dict(device="cuda", dtype=torch.float32)
    out = {"logprob": torch.full((rows,), NAN, **f) if targets is not None else None,
           "entropy": torch.full((rows,), NAN, **f), "stats": torch.full((rows, 2), NAN, **f)}
    ids = torch.full((rows, top), 77, device="cuda", dtype=torch.int32) if top else None
    lps = torch.full((rows, top), NAN, **f) if top else None
    nb._check(nb.lib().nk_token_logprobs_device(
        _p(z), CODE[dtype], rows, V, z.stride(0), _p(targets), T, top, _p(out["logprob"]), _p(out["entropy"]),
        _p(out["stats"]), _p(ids), _p(lps), _st(torch)))
    torch.cuda.synchronize()
    out.update(top_ids=ids, top_logprobs=lps)
    return out


def _ref_rows(torch, z, T):
    """(maximum, log-sum, log p, entropy) of finite or masked rows in 64 bits."""
    z = z.double()
    m = z.amax(-1, keepdim=True)
    y = (z - torch.where(torch.isinf(m), 0.0, m)) / T
    log_s = torch.logsumexp(y, -1, keepdim=True)
    logp = y - log_s
    return m[:, 0], log_s[:, 0], logp, torch.special.entr(torch.exp(logp)).sum(-1)


def _ref_top(torch, z, top):
    """Ids by value, then by index."""
    v, i = torch.sort(z.double(), dim=-1, descending=True, stable=True)
    k = min(top, z.shape[1])
    ids = torch.full((z.shape[0], top), NONE, device="cuda", dtype=torch.int32)
    ids[:, :k] = torch.where(v[:, :k] == -INF, NONE, i[:, :k]).to(torch.int32)
    return ids


def _check_logprobs(torch, out, z, targets, T, top):
    V = z.shape[1]
    m, log_s, logp, ent = _ref_rows(torch, z, T)
    live = torch.ones_like(m, dtype=torch.bool) if targets is None else (targets >= 0) & (targets < V)
    assert torch.equal(out["stats"][live, 0].double(), m[live])
    rel = _sum_rel(V, _span(V))
    # log s: s's relative error, and the rounding of the logarithm (2 ulp) itself.
    assert ((out["stats"][live, 1] - log_s[live]).abs() <= rel + 4 * U * log_s[live].abs()).all()
    # H = log s + (sum e |y|) / s: both sums, the second of at most log V times s.
    assert ((out["entropy"][live] - ent[live]).abs() <= (rel + 8 * U) * (2 + 2 * np.log(V))).all()
    if targets is not None:
        lp = logp.gather(1, targets.long().clamp(0, V - 1)[:, None])[:, 0][live]
        got = out["logprob"][live].double()
        fin = torch.isfinite(lp)
        assert torch.equal(got[~fin], lp[~fin])
        tol = rel + 4 * U * (log_s[live].abs() + (lp - log_s[live]).abs() + lp.abs())
        assert ((got - lp).abs() <= tol)[fin].all()
        for k in ("logprob", "entropy"):
            assert (out[k][~live] == 0).all()
        assert (out["stats"][~live] == 0).all()
    if top:
        ids = _ref_top(torch, z, top)
        ids[~live] = NONE
        assert torch.equal(out["top_ids"], ids)
        none = ids == NONE
        assert (out["top_logprobs"][none] == -INF).all()
        lp = logp.gather(1, ids.long().clamp(min=0))
        tol = rel + 4 * U * (log_s[:, None].abs() + 2 * lp.abs())
        # (low - m) / T of the type's lowest value is beyond f32's range where T < 1: it rounds to -infinity.
        far = ~none & (lp < torch.finfo(torch.float32).min)
        assert (out["top_logprobs"][far] == -INF).all()
        assert ((out["top_logprobs"].double() - lp).abs() <= tol)[~none & ~far].all()


SHAPES = [(1, 1, 0, 0), (3, 2, 0, 1), (2, 19, 5, 0), (5, 255, 0, 1), (4, 256, 0, 0), (4, 257, 8, 3), (7, 1000, 0, 0),
          (3, 1023, 1, 2), (2, 4097, 7, 0), (3, 32768, 0, 0), (2, 50021, 0, 1), (1, 131072, 0, 0), (700, 1024, 0, 0),
          (160, 8191, 1, 0), (2, 300001, 0, 0)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,V,pad,shift", SHAPES + [(600, 3, 0, 0), (700, 1, 2, 1), (900, 9, 1, 0)])
def test_logprobs_over_sizes(gpu, torch, dtype, rows, V, pad, shift):
    z, whole = _matrix(torch, rows, V, dtype, pad, shift, seed=V + rows)
    before = whole.clone()
    targets = torch.randint(0, V, (rows,), device="cuda", dtype=torch.int32)
    if rows > 2:
        targets[rows // 2] = NONE
    for T, top in [(1.0, 0), (1.0, 5), (0.7, 20), (2.5, 128), (1.0, 1)]:
        out = _logprobs(gpu, torch, z, targets, T, top, dtype)
        _check_logprobs(torch, out, z, targets, T, top)
    _check_logprobs(torch, _logprobs(gpu, torch, z, None, 1.0, 7, dtype), z, None, 1.0, 7)
    assert torch.equal(torch.nan_to_num(whole.float(), 123.0), torch.nan_to_num(before.float(), 123.0))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [40, 2048, 40001, 131072, 700000])
def test_logprobs_alternatives_in_awkward_orders(gpu, torch, dtype, V):
    # Sorted rows, constant rows, few values, the largest side by side, zeros
    # of both signs: ties go to the lower id.
    lin = torch.linspace(-8, 8, V, device="cuda")
    few = torch.randint(0, 3, (V,), device="cuda").float()
    block = torch.zeros(V, device="cuda")
    block[V // 2:V // 2 + 300] = 5.0 + lin[V // 2:V // 2 + 300]
    zeros = torch.where(torch.arange(V, device="cuda") % 2 == 0, -0.0, 0.0)
    last = torch.full((V,), -INF, device="cuda")
    last[-1] = 2.0
    stripe = lin.clone()
    stripe[::256] += 10.0
    z = torch.stack([lin, lin.flip(0), torch.full_like(lin, 1.5), few, block, zeros, last, stripe]).to(_dt(torch, dtype))
    for top in (1, 20, 128):
        out = _logprobs(gpu, torch, z, None, 1.0, top, dtype)
        _check_logprobs(torch, out, z, None, 1.0, top)


def test_logprobs_masks_and_special_values(gpu, torch):
    V, low = 1000, torch.finfo(torch.float32).min
    z, _ = _matrix(torch, 9, V, "f32", seed=5)
    z = z.clone()
    z[0] = -INF                      # nothing left
    z[1] = low                       # all at the lowest value: uniform
    z[2, 10:] = low                  # masked by the lowest value
    z[3, 10:] = -INF                 # masked by -infinity
    z[4, 3] = NAN
    z[5, 7] = INF
    z[6] += 1e4                      # a common offset costs no accuracy beyond the inputs' own
    z[7] = -INF
    z[7, 999] = low                  # one value, the lowest
    z[8, 5] = NAN                    # in a row that is not read
    targets = torch.tensor([3, 3, 3, 3, 3, 3, 3, 999, NONE], device="cuda", dtype=torch.int32)
    for T in (1.0, 0.25):
        out = _logprobs(gpu, torch, z, targets, T, 12, "f32")
        lp, ent, st, ids = out["logprob"], out["entropy"], out["stats"], out["top_ids"]
        assert lp[0] == -INF and ent[0] == 0 and (st[0] == -INF).all() and (ids[0] == NONE).all()
        assert (out["top_logprobs"][0] == -INF).all()
        assert torch.isnan(lp[4]) and torch.isnan(ent[4]) and torch.isnan(lp[5]) and torch.isnan(ent[5])
        assert NONE not in ids[4].tolist() and 3 not in ids[4].tolist() and ids[5, 0] == 7
        assert lp[8] == 0 and ent[8] == 0 and (ids[8] == NONE).all()
        assert (ids[3, 10:] == NONE).all() and (ids[3, :10] != NONE).all()
        assert ids[7, 0] == 999 and lp[7] == 0 and ent[7] == 0
        keep = torch.tensor([1, 2, 3, 6, 7], device="cuda")
        _check_logprobs(torch, {k: v[keep] for k, v in out.items()}, z[keep], targets[keep], T, 12)
    # A masked target has log probability -infinity.
    assert _logprobs(gpu, torch, z[3:4], torch.tensor([500], device="cuda", dtype=torch.int32), 1.0, 0, "f32")["logprob"][0] == -INF
    # An id beyond the vocabulary is no token.
    out = _logprobs(gpu, torch, z[6:7], torch.tensor([1000], device="cuda", dtype=torch.int32), 1.0, 3, "f32")
    assert out["logprob"][0] == 0 and (out["top_ids"] == NONE).all()


def _grad(nb, torch, z, targets, T, stats, ent, gl, ge, dtype, dz=None):
    rows, V = z.shape
    dz = torch.full((rows, V), 7.0, device="cuda", dtype=z.dtype) if dz is None else dz
    nb._check(nb.lib().nk_token_logprobs_backward_device(
        _p(z), CODE[dtype], rows, V, z.stride(0), _p(targets), T, _p(stats), _p(ent), _p(gl), _p(ge), _p(dz),
        dz.stride(0), _st(torch)))
    torch.cuda.synchronize()
    return dz


def _ref_grad(torch, z, targets, T, stats, ent, gl, ge):
    """(dz, bound without the output's rounding) from the given statistics."""
    st = stats.double()
    y = (z.double() - st[:, :1]) / T - st[:, 1:]
    p = torch.exp(y)
    zero = torch.zeros(z.shape[0], 1, device="cuda", dtype=torch.float64)
    gl = zero if gl is None else gl.double()[:, None]
    ge_, h = (zero, zero) if ge is None else (ge.double()[:, None], ent.double()[:, None])
    yp = torch.where(p > 0, y, 0.0)
    dz = -p * gl - ge_ * p * (yp + h)
    size = p * (gl.abs() + ge_.abs() * (yp.abs() + h))
    if targets is not None:
        live = (targets >= 0) & (targets < z.shape[1])
        hot = torch.zeros_like(p).scatter_(1, targets.long().clamp(0, z.shape[1] - 1)[:, None], 1.0)
        dz = (dz + hot * gl) * live[:, None]
        size = size + hot * gl.abs()
    # p: 4 roundings of the sizes of (z - m) / T and log s, which are at most |y| + 2 |log s|, and 2^y.
    rel = (4 * (yp.abs() + 2 * st[:, 1:].abs()) + 16) * U
    return dz / T, rel * size / T + 2.0**-126


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,V,pad,shift", SHAPES)
def test_logprobs_gradient_over_sizes(gpu, torch, dtype, rows, V, pad, shift):
    z, _ = _matrix(torch, rows, V, dtype, pad, shift, seed=3 * V + rows)
    z[:, V // 3:V // 2] = -INF
    targets = torch.randint(0, max(1, V // 3), (rows,), device="cuda", dtype=torch.int32)
    if rows > 2:
        targets[1] = NONE
    gl, ge = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
    for T, a, b in [(1.0, gl, None), (0.7, gl, ge), (2.0, None, ge)]:
        fw = _logprobs(gpu, torch, z, targets, T, 0, dtype)
        got = _grad(gpu, torch, z, targets, T, fw["stats"], fw["entropy"], a, b, dtype)
        ref, tol = _ref_grad(torch, z, targets, T, fw["stats"], fw["entropy"], a, b)
        assert ((got.double() - ref).abs() <= tol + _out_tol(torch, dtype, ref)).all()
    # Into rows of another alignment, what lies between them untouched; then in place.
    out, whole = _matrix(torch, rows, V, dtype, pad + 3, shift + 1)
    got2 = _grad(gpu, torch, z, targets, T, fw["stats"], fw["entropy"], a, b, dtype, out)
    assert torch.equal(got2, got)
    gaps = torch.ones(whole.numel(), dtype=torch.bool, device="cuda")
    gaps[shift + 1:shift + 1 + rows * (V + pad + 3)].view(rows, -1)[:, :V] = False
    assert torch.isnan(whole[gaps]).all()
    assert torch.equal(_grad(gpu, torch, z, targets, T, fw["stats"], fw["entropy"], a, b, dtype, z), got)


def test_logprobs_gradient_of_special_rows(gpu, torch):
    z = torch.randn(5, 300, device="cuda")
    z[0] = -INF
    z[1, 4] = NAN
    z[2, 9] = -INF
    z[3] = torch.finfo(torch.float32).min
    targets = torch.tensor([3, 3, 9, 3, NONE], device="cuda", dtype=torch.int32)
    z[4] = NAN
    one = torch.ones(5, device="cuda")
    fw = _logprobs(gpu, torch, z, targets, 1.0, 0, "f32")
    g = _grad(gpu, torch, z, targets, 1.0, fw["stats"], fw["entropy"], one, one, "f32")
    assert (g[0] == 0).all() and torch.isnan(g[1]).all() and (g[4] == 0).all()
    # The target's own logit is masked: 1 - 0 there, as the formula has it.
    assert g[2, 9] == 1.0 and torch.isfinite(g[2]).all()
    assert torch.allclose(g[3, :3], torch.full((3,), -1 / 300, device="cuda"), atol=1e-7) and abs(g[3, 3] - 299 / 300) < 1e-6


def test_logprobs_gradient_against_differences(gpu, torch):
    z, _ = _matrix(torch, 4, 23, "f32", seed=11)
    t = torch.tensor([0, 5, 22, 7], device="cuda", dtype=torch.int32)
    gl, ge = torch.randn(4, device="cuda"), torch.randn(4, device="cuda")
    T, h = 1.3, 1e-5
    fw = _logprobs(gpu, torch, z, t, T, 0, "f32")
    got = _grad(gpu, torch, z, t, T, fw["stats"], fw["entropy"], gl, ge, "f32").double()

    def f(zz):
        _, _, logp, ent = _ref_rows(torch, zz, T)
        return (gl * logp.gather(1, t.long()[:, None])[:, 0] + ge * ent).sum(-1)

    for r in range(4):
        for j in range(23):
            d = torch.zeros(4, 23, device="cuda", dtype=torch.float64)
            d[r, j] = h
            num = (f(z.double() + d) - f(z.double() - d)) / (2 * h)
            # h^2 times a third derivative of a few units, and 1e-16 / h; the gradient's own f32.
            assert abs(num - got[r, j]) < 1e-5 * (1 + got[r].abs().max())


# ---------------------------------------------------------------- distillation
def _distill(nb, torch, z, ids, t, T, w, scale, dtype, t_dtype, grad=True, loss=True, dz=None):
    rows, V = z.shape
    ls = torch.full((rows,), NAN, device="cuda") if loss else None
    if grad and dz is None:
        dz = torch.full((rows, V), 7.0, device="cuda", dtype=z.dtype)
    nb._check(nb.lib().nk_distill_device(
        _p(z), CODE[dtype], rows, V, z.stride(0), _p(ids), _p(t), CODE[t_dtype], ids.shape[1], T, _p(ls), _p(w), scale,
        _p(dz), 0 if dz is None else dz.stride(0), _st(torch)))
    torch.cuda.synchronize()
    return ls, dz


def _ref_distill(torch, z, ids, t, T, w, scale):
    """(loss, its bound, dlogits, their bound) in 64 bits."""
    V, K = z.shape[1], ids.shape[1]
    live = (ids >= 0) & (ids < V) & (t.double() != -INF)
    some = live.any(-1)
    tt = torch.where(live, t.double() / T, -INF)
    logq = torch.where(live, tt - torch.logsumexp(torch.where(some[:, None], tt, 0.0), -1, keepdim=True), 0.0)
    q = torch.where(live, torch.exp(logq), 0.0)
    m, log_s, logp, _ = _ref_rows(torch, z, T)
    at = logp.gather(1, torch.where(live, ids, 0).long())
    loss = T * T * torch.where(q > 0, q * (logq - at), 0.0).sum(-1)
    rel = _sum_rel(V, _span(V))
    # Each term's q (a sum of K, an exponential of |log q|), its two logarithms, and the sum over K.
    terms = torch.where(q > 0, q * (1 + logq.abs() + at.abs() + log_s[:, None].abs()), 0.0)
    loss_tol = T * T * (terms * (rel + (4 * logq.abs() + 4 * log_s[:, None].abs() + K + 64) * U)).sum(-1)
    share = torch.zeros_like(logp).scatter_add_(1, torch.where(live, ids, 0).long(), q)
    p = torch.exp(logp) * some[:, None]
    weight = scale * T * (1.0 if w is None else w.double()[:, None])
    dz = weight * (p - share)
    yp = torch.where(p > 0, logp, 0.0).abs()
    tol = abs(scale) * T * (1.0 if w is None else w.double().abs()[:, None]) * (
        p * (rel + (4 * yp + 8 * log_s[:, None].abs() + 16) * U) + share * (_span(K) * 4 + K + 64) * U)
    return loss, loss_tol, dz, tol + 2.0**-126


@pytest.mark.parametrize("dtype,t_dtype", [("f32", "f32"), ("f16", "f32"), ("bf16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("rows,V,pad,shift", SHAPES + [(600, 3, 0, 0), (700, 1, 2, 1), (513, 7, 0, 0), (900, 9, 1, 0),
                                                       (512, 8, 0, 0), (3, 4, 0, 1)])
def test_distill_over_sizes(gpu, torch, dtype, t_dtype, rows, V, pad, shift):
    z, _ = _matrix(torch, rows, V, dtype, pad, shift, seed=7 * V + rows)
    for K, T, weighted in [(1, 1.0, False), (8, 2.0, True), (min(V, 33), 0.8, True), (256, 1.0, True)]:
        # Ids may repeat; some are no entries.
        ids = torch.randint(0, V, (rows, K), device="cuda", dtype=torch.int32)
        if K > 8:
            ids[:, 3] = NONE
            ids[:, 5] = V  # beyond the vocabulary
            ids[:, 4] = ids[:, 6]
        if rows > 2:
            ids[2] = NONE
        t = (3 * torch.randn(rows, K, device="cuda")).to(_dt(torch, t_dtype))
        if K > 8:
            t[:, 7] = -INF
        w = torch.randn(rows, device="cuda") if weighted else None
        if weighted and rows > 1:
            w[1] = 0.0
        loss, dz = _distill(gpu, torch, z, ids, t, T, w, 0.5, dtype, t_dtype)
        ref, tol, rdz, ztol = _ref_distill(torch, z, ids, t, T, w, 0.5)
        assert ((loss.double() - ref).abs() <= tol).all()
        assert ((dz.double() - rdz).abs() <= ztol + _out_tol(torch, dtype, rdz)).all()
        if weighted and rows > 1:
            assert (dz[1] == 0).all()
        if rows > 2:
            assert loss[2] == 0 and (dz[2] == 0).all()
        # The loss alone, the gradient alone, and other layouts give the same bits.
        assert torch.equal(_distill(gpu, torch, z, ids, t, T, w, 0.5, dtype, t_dtype, grad=False)[0], loss)
        assert torch.equal(_distill(gpu, torch, z, ids, t, T, w, 0.5, dtype, t_dtype, loss=False)[1], dz)
    out, whole = _matrix(torch, rows, V, dtype, pad + 5, shift + 1)
    assert torch.equal(_distill(gpu, torch, z, ids, t, T, w, 0.5, dtype, t_dtype, dz=out)[1], dz)
    gaps = torch.ones(whole.numel(), dtype=torch.bool, device="cuda")
    gaps[shift + 1:shift + 1 + rows * (V + pad + 5)].view(rows, -1)[:, :V] = False
    assert torch.isnan(whole[gaps]).all()
    ls, same = _distill(gpu, torch, z, ids, t, T, w, 0.5, dtype, t_dtype, dz=z)
    assert torch.equal(same, dz) and torch.equal(ls, loss)


@pytest.mark.parametrize("rows,V,dtype,K", [(3700, 4200, "f32", 20), (7500, 4997, "f32", 70), (1900, 17600, "f32", 5),
                                            (3600, 8800, "bf16", 33), (1000, 70001, "bf16", 64)])
def test_distill_of_many_rows(gpu, torch, rows, V, dtype, K):
    # More rows than the GPU works on at once, among them rows without entries, side by
    # side, at the ends and scattered, and rows of weight 0.
    z, _ = _matrix(torch, rows, V, dtype, seed=rows)
    ids = torch.randint(0, V, (rows, K), device="cuda", dtype=torch.int32)
    for gone in (slice(0, 1), slice(5, 12), slice(rows - 3, rows), torch.randperm(rows, device="cuda")[:rows // 6]):
        ids[gone] = NONE
    t = torch.randn(rows, K, device="cuda")
    w = torch.rand(rows, device="cuda") + 0.5
    w[20:30] = 0.0
    w[torch.randperm(rows, device="cuda")[:rows // 10]] = 0.0
    loss, dz = _distill(gpu, torch, z, ids, t, 1.5, w, 0.5, dtype, "f32")
    alone = _distill(gpu, torch, z, ids, t, 1.5, w, 0.5, dtype, "f32", grad=False)[0]
    for r in range(0, rows, 500):
        b = slice(r, r + 500)
        ref, tol, rdz, ztol = _ref_distill(torch, z[b], ids[b], t[b], 1.5, w[b], 0.5)
        for got in (loss, alone):
            assert ((got[b].double() - ref).abs() <= tol).all()
        assert ((dz[b].double() - rdz).abs() <= ztol + _out_tol(torch, dtype, rdz)).all()
    assert (dz[w == 0] == 0).all()
    _, same = _distill(gpu, torch, z, ids, t, 1.5, w, 0.5, dtype, "f32", dz=z)
    assert torch.equal(same, dz)


@pytest.mark.parametrize("rows,V,dtype,top", [(5000, 300, "f32", 5), (3000, 4100, "bf16", 20), (1100, 9001, "f16", 40),
                                              (1500, 20000, "f32", 70), (700, 40000, "bf16", 3)])
def test_logprobs_of_many_rows(gpu, torch, rows, V, dtype, top):
    z, _ = _matrix(torch, rows, V, dtype, seed=rows)
    t = torch.randint(0, V, (rows,), device="cuda", dtype=torch.int32)
    t[torch.randperm(rows, device="cuda")[:rows // 5]] = NONE
    out = _logprobs(gpu, torch, z, t, 0.9, top, dtype)
    for r in range(0, rows, 500):
        b = slice(r, r + 500)
        _check_logprobs(torch, {k: v[b] for k, v in out.items()}, z[b], t[b], 0.9, top)


def test_logprobs_of_sure_tokens_keep_their_digits(gpu, torch):
    # log p = -log(1 + rest) of a rest down to 1e-5: with few rows the rest is summed by
    # itself, so the result is good to a relative 1e-5 at 16384 terms (each exponential 4 U
    # and 4 |y| U, the sum below 112 U, the logarithm's rounding), not to 2^-24 absolutely.
    for V, gap in [(16384, 12.0), (16384, 20.0), (300, 9.0), (40001, 16.0)]:
        z = torch.randn(3, V, device="cuda")
        z[:, 7] = z.amax() + gap
        t = torch.full((3,), 7, device="cuda", dtype=torch.int32)
        out = _logprobs(gpu, torch, z, t, 1.0, 2, "f32")
        zd = z.double()
        rest = torch.exp(zd - zd[:, 7:8])
        rest[:, 7] = 0
        want = -torch.log1p(rest.sum(-1))
        assert ((out["logprob"].double() - want).abs() <= 1e-5 * want.abs()).all()


def test_distill_special_rows(gpu, torch):
    z = torch.randn(6, 500, device="cuda")
    z[0] = NAN                       # a row without entries is not read
    z[1, 40:] = -INF                 # a masked student
    z[2, 7] = NAN
    z[4] = NAN                       # weight 0: no gradient
    ids = torch.arange(4, device="cuda", dtype=torch.int32).repeat(6, 1)
    ids[0] = NONE
    t = torch.randn(6, 4, device="cuda")
    t[3] = -INF                      # no entries either
    ids[5, 0] = 450
    z[5, 450] = -INF                 # the teacher wants what the student cannot say
    w = torch.tensor([1.0, 1, 1, 1, 0, 1], device="cuda")
    loss, dz = _distill(gpu, torch, z, ids, t, 1.0, w, 1.0, "f32", "f32")
    assert loss[0] == 0 and (dz[0] == 0).all() and loss[3] == 0 and (dz[3] == 0).all()
    assert torch.isfinite(loss[1]) and (dz[1, 40:] == 0).all()
    assert torch.isnan(loss[2]) and torch.isnan(dz[2]).all()
    assert torch.isnan(loss[4]) and (dz[4] == 0).all()
    assert loss[5] == INF and torch.isfinite(dz[5]).all()
    # A student that can say nothing: infinity, and no direction to go.
    z[1] = -INF
    loss, dz = _distill(gpu, torch, z[1:2], ids[1:2], t[1:2], 1.0, None, 1.0, "f32", "f32")
    assert loss[0] == INF and (dz == 0).all()
    # A teacher without any places.
    none = torch.empty(6, 0, device="cuda", dtype=torch.int32)
    loss, dz = _distill(gpu, torch, z, none, none.float(), 1.0, w, 1.0, "f32", "f32")
    assert (loss == 0).all() and (dz == 0).all()


def test_distill_gradient_against_differences(gpu, torch):
    z, _ = _matrix(torch, 3, 17, "f32", seed=2)
    ids = torch.tensor([[1, 2, 1], [16, 0, 3], [4, NONE, 5]], device="cuda", dtype=torch.int32)
    t = torch.randn(3, 3, device="cuda")
    w, T, h = torch.tensor([0.5, 2.0, -1.0], device="cuda"), 1.7, 1e-5
    _, dz = _distill(gpu, torch, z, ids, t, T, w, 0.25, "f32", "f32")
    for r in range(3):
        for j in range(17):
            d = torch.zeros(3, 17, device="cuda", dtype=torch.float64)
            d[r, j] = h
            up, down = (_ref_distill(torch, z.double() + e, ids, t, T, w, 0.25)[0] for e in (d, -d))
            num = 0.25 * (w * (up - down)).sum() / (2 * h)
            assert abs(num - dz[r, j]) < 1e-5


# ---------------------------------------------------------------- norms
NORM_SHAPES = [(1, 1, 0, 0), (3, 2, 0, 1), (5, 19, 3, 0), (64, 192, 0, 0), (33, 255, 0, 1), (16, 512, 8, 0),
               (9, 767, 1, 0), (300, 768, 0, 0), (70, 1024, 0, 0), (5, 1025, 0, 1), (40, 2048, 0, 0), (7, 4099, 0, 2),
               (12, 8192, 0, 0), (3, 8193, 0, 0), (6, 16384, 8, 0), (2, 40000, 0, 0), (1200, 96, 0, 0), (2500, 40, 0, 0),
               (310, 10240, 0, 0), (301, 12289, 0, 1), (9, 16383, 1, 1), (160, 20001, 0, 0), (75, 33000, 8, 4), (41, 65520, 0, 0),
               (39, 65497, 0, 2), (3, 65535, 0, 0), (2, 131075, 0, 0)]


def _norm(nb, torch, x, gain, bias, eps, rms, dtype, y=None):
    rows, d = x.shape
    y = torch.full((rows, d), 7.0, device="cuda", dtype=x.dtype) if y is None else y
    mean = None if rms else torch.full((rows,), NAN, device="cuda")
    rstd = torch.full((rows,), NAN, device="cuda")
    nb._check(nb.lib().nk_layer_norm_device(_p(x), CODE[dtype], rows, d, x.stride(0), _p(gain), _p(bias), eps, int(rms),
                                            _p(y), y.stride(0), _p(mean), _p(rstd), _st(torch)))
    torch.cuda.synchronize()
    return y, mean, rstd


def _norm_grad(nb, torch, x, dy, gain, mean, rstd, dtype, dx=True, dgain=True, dbias=True, accumulate=0, before=None):
    rows, d = x.shape
    rms = mean is None
    if dx is True:
        dx = torch.full((rows, d), 7.0, device="cuda", dtype=x.dtype)
    dg = (torch.full((d,), NAN, device="cuda") if before is None else before.clone()) if dgain else None
    db = (torch.full((d,), NAN, device="cuda") if before is None else before.clone()) if dbias and not rms else None
    n = C.c_uint64()
    nb._check(nb.lib().nk_layer_norm_backward_workspace(rows, d, C.byref(n)))
    ws = torch.full((max(n.value // 4, 4),), NAN, device="cuda")
    nb._check(nb.lib().nk_layer_norm_backward_device(
        _p(x), CODE[dtype], rows, d, x.stride(0), _p(gain), _p(mean), _p(rstd), int(rms), _p(dy), dy.stride(0), _p(dx),
        0 if dx is None else dx.stride(0), _p(dg), _p(db), accumulate, _p(ws), n.value, _st(torch)))
    torch.cuda.synchronize()
    return dx, dg, db


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,d,pad,shift", NORM_SHAPES)
def test_norm_over_sizes(gpu, torch, rms, dtype, rows, d, pad, shift):
    x, whole = _matrix(torch, rows, d, dtype, pad, shift, scale=1.5, seed=d, offset=0.7)
    gain = 1 + 0.3 * torch.randn(d, device="cuda")
    bias = None if rms else torch.randn(d, device="cuda")
    eps = 1e-5
    y, mean, rstd = _norm(gpu, torch, x, gain, bias, eps, rms, dtype)
    xd = x.double()
    mu = torch.zeros(rows, 1, device="cuda", dtype=torch.float64) if rms else xd.mean(-1, keepdim=True)
    var = (xd - mu).square().mean(-1, keepdim=True)
    r = torch.rsqrt(var + eps)
    n_add = (d / 256 + 48) * U
    # The mean: a sum of d terms, then a division.
    mean_tol = 0.0 if rms else (n_add + 2 * U) * xd.abs().mean(-1, keepdim=True)
    # The variance: the mean's error counts squared, each square 4 roundings; rstd half of it and 3 more.
    r_rel = 0.5 * (n_add + 8 * U + (mean_tol**2 + 2 * U * (xd.abs().amax(-1, keepdim=True)) ** 2) / (var + eps)) + 4 * U
    if not rms:
        assert ((mean[:, None] - mu).abs() <= mean_tol).all()
    assert ((rstd[:, None] - r).abs() <= r_rel * r).all()
    hh = (xd - mu) * r
    ref = hh * gain + (0.0 if rms else bias)
    tol = gain.abs() * (hh.abs() * (r_rel + 4 * U) + r * (mean_tol + U * xd.abs())) + U * ref.abs() * 2
    assert ((y.double() - ref).abs() <= tol + _out_tol(torch, dtype, ref)).all()
    # Without gain and bias; in place; into another layout.
    plain, _, _ = _norm(gpu, torch, x, None, None, eps, rms, dtype)
    tol1 = hh.abs() * (r_rel + 4 * U) + r * (mean_tol + U * xd.abs())
    assert ((plain.double() - hh).abs() <= tol1 + _out_tol(torch, dtype, hh)).all()
    out, around = _matrix(torch, rows, d, dtype, pad + 3, shift + 1)
    # (Rows of another alignment are summed in another order: the same bound, not the same bits.)
    other = _norm(gpu, torch, x, gain, bias, eps, rms, dtype, out)[0]
    assert ((other.double() - ref).abs() <= tol + _out_tol(torch, dtype, ref)).all()
    gaps = torch.ones(around.numel(), dtype=torch.bool, device="cuda")
    gaps[shift + 1:shift + 1 + rows * (d + pad + 3)].view(rows, -1)[:, :d] = False
    assert torch.isnan(around[gaps]).all()
    assert torch.equal(_norm(gpu, torch, x, gain, bias, eps, rms, dtype, x)[0], y)


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,d,pad,shift", NORM_SHAPES)
def test_norm_gradient_over_sizes(gpu, torch, rms, dtype, rows, d, pad, shift):
    x, _ = _matrix(torch, rows, d, dtype, pad, shift, scale=1.5, seed=d, offset=0.7)
    dy, _ = _matrix(torch, rows, d, dtype, pad + 1, shift, scale=0.5, seed=d + 1, offset=0.1)
    gain = 1 + 0.3 * torch.randn(d, device="cuda")
    _, mean, rstd = _norm(gpu, torch, x, gain, None, 1e-5, rms, dtype)
    dx, dg, db = _norm_grad(gpu, torch, x, dy, gain, mean, rstd, dtype)
    xd, g, r = x.double(), dy.double(), rstd.double()[:, None]
    mu = 0.0 if rms else mean.double()[:, None]
    hh = (xd - mu) * r
    h_tol = hh.abs() * 2 * U + r * U * (xd - mu).abs()
    c = g * gain
    n_add = (d / 256 + 48) * U
    mc = 0.0 if rms else c.mean(-1, keepdim=True)
    mch = (c * hh).mean(-1, keepdim=True)
    ref = r * (c - mc - hh * mch)
    a_c, a_ch = c.abs().mean(-1, keepdim=True), (c * hh).abs().mean(-1, keepdim=True)
    tol = r * (4 * U * c.abs() + (n_add + 4 * U) * (0.0 if rms else a_c)
               + hh.abs() * (n_add + 8 * U) * a_ch + 4 * U * hh.abs() * mch.abs() + h_tol * mch.abs()) + 3 * U * ref.abs()
    assert ((dx.double() - ref).abs() <= tol + _out_tol(torch, dtype, ref)).all()
    # Sums over rows: each term through at most rows / 512 + 512 additions.
    adds = (rows / 512 + 512) * U
    assert ((dg - (g * hh).sum(0)).abs() <= (adds + 4 * U) * (g * hh).abs().sum(0) + (g.abs() * h_tol).sum(0)).all()
    if not rms:
        assert ((db - g.sum(0)).abs() <= adds * g.abs().sum(0)).all()
    # Adding to what is there; any subset of the outputs; dx on dy: the same values.
    before = torch.randn(d, device="cuda")
    _, dg2, db2 = _norm_grad(gpu, torch, x, dy, gain, mean, rstd, dtype, dx=None, accumulate=1, before=before)
    assert torch.equal(dg2, before + dg) and (rms or torch.equal(db2, before + db))
    only, _, _ = _norm_grad(gpu, torch, x, dy, gain, mean, rstd, dtype, dgain=False, dbias=False)
    assert torch.equal(only, dx)
    if not rms:
        _, none, db3 = _norm_grad(gpu, torch, x, dy, gain, mean, rstd, dtype, dx=None, dgain=False)
        assert none is None and torch.equal(db3, db)
    on_dy, dg4, _ = _norm_grad(gpu, torch, x, dy, gain, mean, rstd, dtype, dx=dy)
    assert torch.equal(on_dy, dx) and torch.equal(dg4, dg)


def test_norm_of_constant_and_special_rows(gpu, torch):
    x = torch.randn(5, 200, device="cuda")
    x[0] = 3.0
    x[1] = 0.0
    x[2, 5] = NAN
    x[3] = 1e19                      # squares beyond f32: RMSNorm gives 0 times it, layer norm's variance is 0
    y, mean, rstd = _norm(gpu, torch, x, None, None, 1e-5, False, "f32")
    assert (y[0] == 0).all() and (y[1] == 0).all() and torch.isnan(y[2]).all() and torch.isfinite(y[3]).all()
    assert mean[0] == 3.0 and torch.isfinite(y[4]).all()
    y, _, rstd = _norm(gpu, torch, x, None, None, 1e-5, True, "f32")
    assert (y[1] == 0).all() and torch.isfinite(rstd[1]) and torch.isnan(y[2]).all()


def test_norm_gradient_against_differences(gpu, torch):
    for rms in (False, True):
        x = torch.randn(3, 11, device="cuda")
        dy = torch.randn(3, 11, device="cuda")
        gain = torch.randn(11, device="cuda")
        _, mean, rstd = _norm(gpu, torch, x, gain, None, 1e-5, rms, "f32")
        dx, dg, db = _norm_grad(gpu, torch, x, dy, gain, mean, rstd, "f32")

        def f(xx, gg):
            mu = 0.0 if rms else xx.mean(-1, keepdim=True)
            return (dy * ((xx - mu) * torch.rsqrt((xx - mu).square().mean(-1, keepdim=True) + 1e-5) * gg)).sum()

        h = 1e-5
        for r in range(3):
            for j in range(11):
                e = torch.zeros(3, 11, device="cuda", dtype=torch.float64)
                e[r, j] = h
                num = (f(x.double() + e, gain.double()) - f(x.double() - e, gain.double())) / (2 * h)
                assert abs(num - dx[r, j]) < 2e-5 * (1 + abs(num))
        for j in range(11):
            e = torch.zeros(11, device="cuda", dtype=torch.float64)
            e[j] = h
            num = (f(x.double(), gain.double() + e) - f(x.double(), gain.double() - e)) / (2 * h)
            assert abs(num - dg[j]) < 2e-5 * (1 + abs(num))


def test_norm_gradient_without_rows(gpu, torch):
    x = torch.empty(0, 12, device="cuda")
    before = torch.randn(12, device="cuda")
    n = C.c_uint64()
    gpu._check(gpu.lib().nk_layer_norm_backward_workspace(0, 12, C.byref(n)))
    ws = torch.empty(n.value // 4, device="cuda")
    for acc in (1, 0):
        dg, db = before.clone(), before.clone()
        gpu._check(gpu.lib().nk_layer_norm_backward_device(None, 0, 0, 12, 12, None, None, None, 0, None, 12, None, 12,
                                                           _p(dg), _p(db), acc, _p(ws), n.value, _st(torch)))
        torch.cuda.synchronize()
        assert torch.equal(dg, before if acc else torch.zeros_like(before)) and torch.equal(db, dg)
    del x


# ---------------------------------------------------------------- how they are called
def test_many_short_rows_and_far_rows(gpu, torch):
    # More rows than a grid's small dimensions hold.
    z, _ = _matrix(torch, 140001, 5, "bf16", seed=1)
    t = torch.randint(0, 5, (140001,), device="cuda", dtype=torch.int32)
    _check_logprobs(torch, _logprobs(gpu, torch, z, t, 1.0, 3, "bf16"), z, t, 1.0, 3)
    y, mean, rstd = _norm(gpu, torch, z, None, None, 1e-5, False, "bf16")
    assert torch.isfinite(rstd).all()
    # Elements beyond 2^31, in rows that count.
    rows, V = 20000, 120000
    z = torch.empty(rows, V, device="cuda", dtype=torch.bfloat16)
    t = torch.full((rows,), NONE, device="cuda", dtype=torch.int32)
    at = torch.tensor([0, 17000, 18500, rows - 1], device="cuda")
    z[at] = (3 * torch.randn(4, V, device="cuda")).bfloat16()
    t[at] = torch.tensor([5, 119999, 0, 60000], device="cuda", dtype=torch.int32)
    out = _logprobs(gpu, torch, z, t, 1.0, 4, "bf16")
    _check_logprobs(torch, {k: v[at] for k, v in out.items()}, z[at], t[at], 1.0, 4)
    gl = torch.ones(rows, device="cuda")
    zs = z[at].clone()
    _grad(gpu, torch, z, t, 1.0, out["stats"], out["entropy"], gl, None, "bf16", z)
    ref, tol = _ref_grad(torch, zs, t[at], 1.0, out["stats"][at], None, gl[at], None)
    assert ((z[at].double() - ref).abs() <= tol + _out_tol(torch, "bf16", ref)).all()
    assert (z[1:100] == 0).all()


def _all_at_once(gpu, torch, s):
    """Every device call on the state's own buffers, on the current stream."""
    L, st = gpu.lib(), _st(torch)
    R, V, K, d = 6, 5000, 9, 600
    gpu._check(L.nk_token_logprobs_device(_p(s["z"]), 0, R, V, V, _p(s["t"]), 1.0, 8, _p(s["lp"]), _p(s["ent"]),
                                          _p(s["st"]), _p(s["ti"]), _p(s["tl"]), st))
    gpu._check(L.nk_token_logprobs_backward_device(_p(s["z"]), 0, R, V, V, _p(s["t"]), 1.0, _p(s["st"]), _p(s["ent"]),
                                                   _p(s["g"]), _p(s["g"]), _p(s["dz"]), V, st))
    gpu._check(L.nk_distill_device(_p(s["z"]), 0, R, V, V, _p(s["ids"]), _p(s["tz"]), 0, K, 1.0, _p(s["loss"]), None, 1.0,
                                   _p(s["dz2"]), V, st))
    gpu._check(L.nk_layer_norm_device(_p(s["x"]), 0, R, d, d, _p(s["gain"]), None, 1e-5, 0, _p(s["y"]), d, _p(s["mean"]),
                                      _p(s["rstd"]), st))
    gpu._check(L.nk_layer_norm_backward_device(_p(s["x"]), 0, R, d, d, _p(s["gain"]), _p(s["mean"]), _p(s["rstd"]), 0,
                                               _p(s["dy"]), d, _p(s["dx"]), d, _p(s["dg"]), _p(s["db"]), 0, _p(s["ws"]),
                                               4 * s["ws"].numel(), st))


def _state(torch, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    R, V, K, d = 6, 5000, 9, 600
    rn = lambda *n: torch.randn(*n, generator=g, device="cuda")  # noqa: E731
    em = lambda *n, t=torch.float32: torch.zeros(*n, device="cuda", dtype=t)  # noqa: E731
    return {"z": 3 * rn(R, V), "t": torch.randint(0, V, (R,), generator=g, device="cuda", dtype=torch.int32), "g": rn(R),
            "ids": torch.randint(0, V, (R, K), generator=g, device="cuda", dtype=torch.int32), "tz": rn(R, K),
            "x": rn(R, d), "dy": rn(R, d), "gain": rn(d), "lp": em(R), "ent": em(R), "st": em(R, 2),
            "ti": em(R, 8, t=torch.int32), "tl": em(R, 8), "dz": em(R, V), "loss": em(R), "dz2": em(R, V),
            "y": em(R, d), "mean": em(R), "rstd": em(R), "dx": em(R, d), "dg": em(d), "db": em(d),
            "ws": em(2048 * d)}


OUTS = ("lp", "ent", "st", "ti", "tl", "dz", "loss", "dz2", "y", "mean", "rstd", "dx", "dg", "db")


def test_other_streams_and_captured_graphs(gpu, torch):
    states = [_state(torch, s) for s in (1, 2)]
    want = []
    for s in states:
        _all_at_once(gpu, torch, s)
        torch.cuda.synchronize()
        want.append({k: s[k].clone() for k in OUTS})
    # Two streams at once, several times.
    streams = [torch.cuda.Stream() for _ in states]
    for s in states:
        for k in OUTS:
            s[k].zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for s, st in zip(states, streams):
            with torch.cuda.stream(st):
                _all_at_once(gpu, torch, s)
    torch.cuda.synchronize()
    for s, w in zip(states, want):
        assert all(torch.equal(s[k], w[k]) for k in OUTS)
    # Two graphs, replayed side by side and on new inputs.
    graphs = []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            _all_at_once(gpu, torch, s)
        graphs.append(g)
    for s in states:
        for k in OUTS:
            s[k].zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for s, w in zip(states, want):
        assert all(torch.equal(s[k], w[k]) for k in OUTS)
    for k in ("z", "t", "g", "ids", "tz", "x", "dy", "gain"):
        states[0][k].copy_(states[1][k])
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(states[0][k], want[1][k]) for k in OUTS)
    del graphs


def test_host_memory_is_refused(gpu, torch):
    a = np.zeros(64, np.float32)
    p = a.ctypes.data_as(C.c_void_p)
    d = torch.zeros(64, device="cuda")
    L = gpu.lib()
    assert L.nk_token_logprobs_device(p, 0, 2, 8, 8, None, 1.0, 0, None, _p(d), None, None, None, None) == gpu.NK_ERR_INVALID
    assert L.nk_layer_norm_device(p, 0, 2, 8, 8, None, None, 1e-5, 1, _p(d), 8, None, None, None) == gpu.NK_ERR_INVALID
    # Any array, not the first alone.
    e = torch.zeros(64, device="cuda")
    assert L.nk_token_logprobs_device(_p(d), 0, 2, 8, 8, p, 1.0, 0, _p(e), None, None, None, None, None) == gpu.NK_ERR_INVALID
    assert L.nk_token_logprobs_device(_p(d), 0, 2, 8, 8, None, 1.0, 0, None, p, None, None, None, None) == gpu.NK_ERR_INVALID
    assert L.nk_distill_device(_p(d), 0, 2, 8, 8, p, _p(e), 0, 1, 1.0, _p(e[32:]), None, 1.0, None, 8, None) == gpu.NK_ERR_INVALID
    assert L.nk_layer_norm_device(_p(d), 0, 2, 8, 8, p, None, 1e-5, 1, _p(e), 8, None, None, None) == gpu.NK_ERR_INVALID
    assert L.nk_layer_norm_backward_device(_p(d), 0, 2, 8, 8, None, None, p, 1, _p(d), 8, _p(e), 8, None, None, 0, None, 0,
                                           None) == gpu.NK_ERR_INVALID
    torch.cuda.synchronize()


def test_host_forms_match_the_device_forms(gpu, torch):
    rng = np.random.default_rng(4)
    for dtype in ("f32", "f16", "bf16"):
        zt, _ = _matrix(torch, 7, 333, dtype, seed=8)
        z = zt.contiguous()
        h = z.view(torch.uint16).cpu().numpy() if dtype == "bf16" else z.cpu().numpy()
        t = rng.integers(0, 333, 7).astype(np.uint32)
        t[3] = gpu.NO_TOKEN
        td = torch.from_numpy(t.view(np.int32)).cuda()
        dev = _logprobs(gpu, torch, z, td, 0.9, 6, dtype)
        out = gpu.token_logprobs(h, t, temperature=0.9, top=6)
        for k in ("logprob", "entropy", "stats", "top_logprobs"):
            assert np.array_equal(out[k], dev[k].cpu().numpy()), k
        assert np.array_equal(out["top_ids"].view(np.int32), dev["top_ids"].cpu().numpy())
        gl, ge = rng.standard_normal((2, 7)).astype(np.float32)
        dz = gpu.token_logprobs_backward(h, t, out["stats"], out["entropy"], gl, ge, temperature=0.9)
        want = _grad(gpu, torch, z, td, 0.9, dev["stats"], dev["entropy"], torch.from_numpy(gl).cuda(),
                     torch.from_numpy(ge).cuda(), dtype)
        view = (lambda a: a.view(torch.uint16) if dtype == "bf16" else a)
        assert np.array_equal(dz, view(want).cpu().numpy())
        ids = rng.integers(0, 333, (7, 5)).astype(np.uint32)
        tz = rng.standard_normal((7, 5)).astype(np.float32)
        loss, dz = gpu.distill(h, ids, tz, temperature=2.0, row_weight=gl, grad_scale=0.1)
        wl, wz = _distill(gpu, torch, z, torch.from_numpy(ids.view(np.int32)).cuda(), torch.from_numpy(tz).cuda(), 2.0,
                          torch.from_numpy(gl).cuda(), 0.1, dtype, "f32")
        assert np.array_equal(loss, wl.cpu().numpy()) and np.array_equal(dz, view(wz).cpu().numpy())
        gain = rng.standard_normal(333).astype(np.float32)
        nm = gpu.layer_norm(h, gain, gain, 1e-5)
        wy, wm, wr = _norm(gpu, torch, z, torch.from_numpy(gain).cuda(), torch.from_numpy(gain).cuda(), 1e-5, False, dtype)
        assert np.array_equal(nm["y"], view(wy).cpu().numpy()) and np.array_equal(nm["rstd"], wr.cpu().numpy())
        dx, dg, db = gpu.layer_norm_backward(h, h, gain, nm["mean"], nm["rstd"])
        wx, wg, wb = _norm_grad(gpu, torch, z, z, torch.from_numpy(gain).cuda(), wm, wr, dtype)
        assert np.array_equal(dx, view(wx).cpu().numpy()) and np.array_equal(dg, wg.cpu().numpy())
        assert np.array_equal(db, wb.cpu().numpy())
