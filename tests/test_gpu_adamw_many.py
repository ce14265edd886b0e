"""AdamW over many tensors (include/noetic/train.h) on the GPU.  32-bit moments:
bit for bit against nk_adamw_step and a restatement in torch, whose f32 operations
are rounded one by one as the kernel's are.  8-bit moments: against the definition in
64 bits.  With U = 2^-24, m' has the roundings of two products' factors, of two
products and of a sum: 5 U of |b1 m| + |(1 - b1) g|; v' 7 U; its root half of that and
2^-23 of its own; the update 2^-22 (the reciprocal), m''s and the root's: 16 U at most;
val one more.  A moment is stored within half a step of the grid of e4m3 (16 values a
power of two, 2^-9 apart below 2^-6, of 448 for the block's largest), whose place has the
moment's error, the largest's, and 4 U of the scale: 16 U of the value."""

import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0**-24
CODE = {"f32": 0, "f16": 1, "bf16": 2}
SIZES = [1, 2, 255, 256, 257, 1000, 4096, 70001, 3, 513, 1 << 18]
HYPER = dict(lr=3e-3, t=7, b1=0.9, b2=0.95, eps=1e-8, wd=0.1)


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


def _dt(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


class Tensors:
    """Parameter tensors at places `shift` elements into their arrays."""

    def __init__(self, torch, sizes, grad="f32", bits=32, copy=None, shift=0, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.torch, self.bits, self.grad, self.copy = torch, bits, grad, copy
        self.t = []

        def array(n, dtype, v=None):
            whole = torch.zeros(n + shift + 8, device="cuda", dtype=dtype)
            a = whole[shift:shift + n]
            if v is not None:
                a.copy_(v)
            return a

        for i, n in enumerate(sizes):
            nb = -(-n // 256)
            size = torch.exp(2 * torch.randn(nb, generator=g, device="cuda") - 6).repeat_interleave(256)[:n]
            gr = torch.randn(n, generator=g, device="cuda") * size
            t = {"val": array(n, torch.float32, torch.randn(n, generator=g, device="cuda")),
                 "grad": array(n, _dt(torch, grad), gr), "decay": i % 2, "n": n}
            if bits == 32:
                t["m"] = array(n, torch.float32, gr * 0.3)
                t["v"] = array(n, torch.float32, gr.square() * torch.rand(n, generator=g, device="cuda"))
            else:
                t["m"] = array(n, torch.uint8, torch.randint(0, 127, (n,), generator=g, device="cuda") +
                               128 * torch.randint(0, 2, (n,), generator=g, device="cuda"))
                t["v"] = array(n, torch.uint8, torch.randint(0, 127, (n,), generator=g, device="cuda"))
                t["m_scale"] = array(nb, torch.float32, torch.rand(nb, generator=g, device="cuda") * 1e-4)
                t["v_scale"] = array(nb, torch.float32, torch.rand(nb, generator=g, device="cuda") * 1e-4)
            if copy:
                t["copy"] = array(n, _dt(torch, copy))
            self.t.append(t)

    def plan(self, nb):
        def at(t, k):
            return t[k].data_ptr() if k in t and t["n"] else None

        return nb.train.AdamwMany([nb.train.AdamwTensor(
            val=at(t, "val"), grad=at(t, "grad"), m=at(t, "m"), v=at(t, "v"), n=t["n"], m_scale=at(t, "m_scale"),
            v_scale=at(t, "v_scale"), copy=at(t, "copy"), grad_dtype=CODE[self.grad],
            copy_dtype=CODE[self.copy or "bf16"], state_bits=self.bits, decay=t["decay"]) for t in self.t])

    def clone(self):
        return [{k: v.clone() if hasattr(v, "clone") else v for k, v in t.items()} for t in self.t]


def _bias(b, t):
    """1 / (1 - b^t) with the C library's powf, as the host computes it."""
    powf = C.CDLL("libm.so.6").powf
    powf.restype, powf.argtypes = C.c_float, [C.c_float, C.c_float]
    one = np.float32(1.0)
    return float(one / (one - np.float32(powf(b, t))))


def _want(torch, t, c, lr, t_step, b1, b2, eps, wd, bits):
    """The step of one tensor, operation by operation in f32."""
    f = lambda x: float(np.float32(x))  # noqa: E731
    n = t["n"]
    fine = torch.isfinite(t["grad"].float() * c) & torch.isfinite(t["val"])
    if bits == 8:
        return _want8(torch, t, c, lr, t_step, b1, b2, eps, wd, fine)
    g = t["grad"].float() * c
    m, v = t["m"], t["v"]
    m1 = m * f(b1) + g * f(np.float32(1) - np.float32(b1))
    v1 = v * f(b2) + (g * f(np.float32(1) - np.float32(b2))) * g
    upd = (m1 * _bias(b1, t_step)) / (torch.sqrt(v1 * _bias(b2, t_step)) + f(eps))
    if t["decay"] and wd:
        upd = upd + t["val"] * f(wd)
    return {"val": torch.where(fine, t["val"] - upd * f(lr), t["val"]), "m": torch.where(fine, m1, m),
            "v": torch.where(fine, v1, v)}


def _want8(torch, t, c, lr, t_step, b1, b2, eps, wd, fine):
    """The step of a tensor with 8-bit moments in 64 bits, and what the kernel may be off by."""
    f = lambda x: float(np.float32(x))  # noqa: E731
    n, blocks = t["n"], -(-t["n"] // 256)

    def per(s):
        return s.double().repeat_interleave(256)[:n]

    g = torch.where(fine, t["grad"].double() * c, 0.0)
    m, r = t["m"].view(torch.float8_e4m3fn).double() * per(t["m_scale"]), t["v"].view(torch.float8_e4m3fn).double() * per(t["v_scale"])
    b1, b2 = f(b1), f(b2)
    m1, m_tol = b1 * m + (1 - b1) * g, 5 * U * (b1 * m.abs() + (1 - b1) * g.abs())
    v1 = b2 * r * r + (1 - b2) * g * g
    u = torch.sqrt(v1)
    den = u * _bias(b2, t_step) ** 0.5 + f(eps)
    upd = m1 * _bias(b1, t_step) / den
    val = t["val"].double()
    step = f(lr) * (upd + f(wd) * t["decay"] * val)
    tol = f(lr) * (16 * U * upd.abs() + m_tol * _bias(b1, t_step) / den + 4 * U * f(wd) * val.abs()) + 2 * U * step.abs()
    out = {"val": val - step, "val_tol": tol, "fine": fine, "before": t["val"].clone()}
    for k, x, x_tol in (("m", torch.where(fine, m1, m), m_tol), ("v", torch.where(fine, u, r), 6 * U * u)):
        rows = torch.zeros(2, blocks * 256, device="cuda", dtype=torch.float64)
        rows[0, :n], rows[1, :n] = x.abs(), x_tol
        out[k], out[k + "_tol"] = x, x_tol
        out[k + "_scale"] = rows[0].view(blocks, 256).amax(1) / 448.0
        out[k + "_top_tol"] = rows[1].view(blocks, 256).amax(1)
    return out


def _same(torch, got, want, copy=None):
    if "m_scale" in want:
        return _near(torch, got, want, copy)
    for k, v in want.items():
        assert torch.equal(got[k], v), (k, got["n"], (got[k].float() - v.float()).abs().max())
    if copy:
        assert torch.equal(got["copy"], want["val"].to(_dt(torch, copy)))


def _near(torch, got, want, copy):
    """8-bit moments: `want` holds 64-bit values."""
    n = got["n"]
    err = (got["val"].double() - want["val"]).abs()
    assert (err <= U * want["val"].abs() + want["val_tol"])[want["fine"]].all(), float(err.max())
    assert torch.equal(got["val"][~want["fine"]].view(torch.int32), want["before"][~want["fine"]].view(torch.int32))
    for k in ("m", "v"):
        top, x, tol = want[k + "_scale"] * 448.0, want[k], want[k + "_tol"]
        assert ((got[k + "_scale"].double() - want[k + "_scale"]).abs() <= 16 * U * want[k + "_scale"] + want[k + "_top_tol"] / 448).all()
        scale = got[k + "_scale"].double().repeat_interleave(256)[:n]
        y = x / scale.clamp(min=1e-300)  # where the value is on the grid
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)
        code = got[k].view(torch.float8_e4m3fn).double()
        room = step / 2 + 16 * U * y.abs() + tol / scale.clamp(min=1e-300)
        if k == "v":
            room = torch.where((x > 0) & (y < 2.0**-9), 2.0**-9, room)
            assert (code[(x > 0) & (scale > 0)] > 0).all() and (code >= 0).all()
        assert ((code - y).abs() <= room)[scale > 0].all(), (k, n)
        assert (code[scale == 0] == 0).all() and (top.repeat_interleave(256)[:n][scale == 0] < 1e-30).all()
    if copy:
        assert torch.equal(got["copy"], got["val"].to(_dt(torch, copy)))


@pytest.mark.parametrize("grad", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits,copy,shift", [(32, None, 0), (32, "f16", 0), (32, "bf16", 1), (8, None, 0), (8, "bf16", 0),
                                             (8, "f16", 3)])
def test_step(nb, torch, grad, bits, copy, shift):
    s = Tensors(torch, SIZES, grad, bits, copy, shift)
    before = s.clone()
    plan = s.plan(nb)
    plan.step(**HYPER)
    torch.cuda.synchronize()
    for t, b in zip(s.t, before):
        _same(torch, t, _want(torch, b, 1.0, HYPER["lr"], 7, 0.9, 0.95, 1e-8, 0.1, bits), copy)


@pytest.mark.parametrize("grad", ["f32", "bf16"])
def test_bytes_are_those_of_the_operations_one_by_one(nb, torch, grad):
    """A byte at the middle between two others goes the way that the formula goes when each of its
    operations is rounded; roots, one in a million of which the kernel rounds the other way, may
    move one byte in a hundred thousand."""
    s = Tensors(torch, [1 << 20, 3001], grad, 8, seed=12)
    before = s.clone()
    s.plan(nb).step(**HYPER)
    torch.cuda.synchronize()
    for t, b in zip(s.t, before):
        n, blocks = b["n"], -(-b["n"] // 256)

        def per(x):
            return x.repeat_interleave(256)[:n]

        g = b["grad"].float()
        m = b["m"].view(torch.float8_e4m3fn).float() * per(b["m_scale"])
        r = b["v"].view(torch.float8_e4m3fn).float() * per(b["v_scale"])
        m = m * float(np.float32(0.9)) + g * float(np.float32(1) - np.float32(0.9))
        v = r.square() * float(np.float32(0.95)) + (g * float(np.float32(1) - np.float32(0.95))) * g
        for k, x in (("m", m), ("v", torch.sqrt(v))):
            rows = torch.zeros(blocks * 256, device="cuda")
            rows[:n] = x
            top = rows.view(blocks, 256).abs().amax(1)
            assert torch.equal(t[k + "_scale"], top * float(np.float32(1) / np.float32(448)))
            y = x * per(torch.where(top > 0, (1.0 / top) * 448.0, 0.0))
            if k == "v":
                y = torch.where(x > 0, y.clamp(min=2.0**-9), y)
            code = y.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
            away = int((t[k] != code).sum())
            assert away <= (1e-5 * n if n > 1e5 else 0), (k, away)


def test_32_bits_are_nk_adamw_step(nb, torch):
    s = Tensors(torch, SIZES, seed=3)
    other = s.clone()
    plan = s.plan(nb)
    for step in range(1, 5):
        plan.step(**{**HYPER, "t": step})
        for t in other:
            cfg = nb.NkAdamwCfg(HYPER["lr"], 0.9, 0.95, 1e-8, 0.1, step, t["decay"])
            nb._check(nb.lib().nk_adamw_step_device(t["val"].data_ptr(), t["grad"].data_ptr(), t["m"].data_ptr(),
                                                    t["v"].data_ptr(), t["n"], C.byref(cfg), None))
    torch.cuda.synchronize()
    for t, o in zip(s.t, other):
        assert all(torch.equal(t[k], o[k]) for k in ("val", "m", "v"))


@pytest.mark.parametrize("bits,grad", [(32, "f32"), (8, "bf16"), (8, "f16")])
@pytest.mark.parametrize("scale", [1.0, 1 / 1024])
def test_norm_and_clip(nb, torch, bits, grad, scale):
    s = Tensors(torch, SIZES, grad, bits, seed=4)
    before = s.clone()
    plan = s.plan(nb)
    norm = torch.zeros(1, device="cuda")
    bad = torch.zeros(1, device="cuda", dtype=torch.int32)
    exact = sum(float(t["grad"].double().square().sum()) for t in before) ** 0.5 * scale
    for limit in (0.0, 2 * exact, exact / 3):
        plan.step(**HYPER, grad_scale=scale, max_norm=limit, norm=norm.data_ptr(), bad=bad.data_ptr())
        torch.cuda.synchronize()
        # Squares, and sums of four of them, in f32: 3 roundings of a square, 2 of the result.
        assert abs(float(norm) - exact) <= 4 * 2.0**-24 * exact and int(bad) == 0
        c = np.float32(scale)
        if limit and float(norm) > np.float32(limit):
            c = np.float32(scale) * (np.float32(limit) * (np.float32(1) / np.float32(norm.cpu().numpy()[0])))
        for t, b in zip(s.t, before):
            _same(torch, t, _want(torch, b, float(c), HYPER["lr"], 7, 0.9, 0.95, 1e-8, 0.1, bits))
        before = s.clone()


@pytest.mark.parametrize("grad", ["f32", "bf16"])
@pytest.mark.parametrize("factor", [1e25, 1e-25])
def test_norm_of_gradients_whose_squares_leave_f32(nb, torch, grad, factor):
    s = Tensors(torch, SIZES, grad, 32, seed=5)
    for t in s.t:
        t["grad"] *= factor
        t["grad"][::3] = 0.0
    before = s.clone()
    plan = s.plan(nb)
    norm = torch.zeros(1, device="cuda")
    bad = torch.zeros(1, device="cuda", dtype=torch.int32)
    exact = sum(float(t["grad"].double().square().sum()) for t in before) ** 0.5
    plan.step(**HYPER, max_norm=1.0, norm=norm.data_ptr(), bad=bad.data_ptr())
    torch.cuda.synchronize()
    assert abs(float(norm) - exact) <= 4 * U * exact and int(bad) == 0
    c = np.float32(1)
    if factor > 1:
        c = np.float32(1) / np.float32(norm.cpu().numpy()[0])
    for t, b in zip(s.t, before):
        _same(torch, t, _want(torch, b, float(c), HYPER["lr"], 7, 0.9, 0.95, 1e-8, 0.1, 32))


@pytest.mark.parametrize("bits", [32, 8])
def test_elements_that_are_not_finite_stay(nb, torch, bits):
    s = Tensors(torch, [1000, 4096, 5], bits=bits, seed=5)
    s.t[0]["grad"][3] = float("nan")
    s.t[1]["grad"][4095] = float("inf")
    s.t[2]["val"][0] = float("inf")
    before = s.clone()
    plan = s.plan(nb)
    bad = torch.zeros(1, device="cuda", dtype=torch.int32)
    plan.step(**HYPER, bad=bad.data_ptr())
    torch.cuda.synchronize()
    assert int(bad) == 1
    for t, b in zip(s.t, before):
        _same(torch, t, _want(torch, b, 1.0, HYPER["lr"], 7, 0.9, 0.95, 1e-8, 0.1, bits))
    # With a clip nothing changes.
    now = s.clone()
    bad.zero_()
    norm = torch.zeros(1, device="cuda")
    plan.step(**HYPER, max_norm=1.0, norm=norm.data_ptr(), bad=bad.data_ptr())
    torch.cuda.synchronize()
    assert int(bad) == 1 and not torch.isfinite(norm).any()
    for t, b in zip(s.t, now):
        assert all(torch.equal(t[k].view(torch.uint8), b[k].view(torch.uint8)) for k in t if k in ("val", "m", "v"))


def test_blocks_of_zeros_and_of_extremes(nb, torch):
    """Zero gradients and moments stay zero; v stays above zero beside a large one; the largest values do not overflow."""
    s = Tensors(torch, [1024], bits=8, seed=6)
    t = s.t[0]
    for k in ("m", "v", "m_scale", "v_scale"):
        t[k].zero_()
    t["grad"][:256] = 0.0
    t["grad"][256:512] = 1e-9
    t["grad"][300] = 1e3
    t["grad"][512:768] = 1e-38
    t["grad"][768:] = 3e38
    before = s.clone()[0]
    plan = s.plan(nb)
    plan.step(**{**HYPER, "wd": 0.0})
    torch.cuda.synchronize()
    assert torch.equal(t["val"][:256], before["val"][:256]) and (t["m"][:256] == 0).all() and (t["v"][:256] == 0).all()
    assert (t["v"][256:512] > 0).all() and float(t["v_scale"][0]) == 0.0
    assert all(torch.isfinite(t[k]).all() for k in ("val", "m_scale", "v_scale"))
    assert (t["m"] != 127).all() and (t["v"] != 127).all()
    for _ in range(20):
        plan.step(**{**HYPER, "wd": 0.0})
    torch.cuda.synchronize()
    # A step moves a value by lr |m^| / (sqrt(v^) + eps), and in this framework's moments m^2 <= 11 v
    # (sum of the weights' squares ratio, (1 - b1)^2 / ((1 - b2)(1 - b1^2 / b2)) < 2) with rounding
    # of 1/16 in each: far below 4 steps each.
    assert (t["val"] - before["val"]).abs().max() <= 21 * 4 * HYPER["lr"]


def test_8_bits_follow_32_bits(nb, torch):
    """Thirty steps on noisy gradients: the values part by a small share of the way."""
    a, b = Tensors(torch, [50000], seed=7), Tensors(torch, [50000], bits=8, seed=7)
    for s in (a, b):
        for k in ("m", "v", "m_scale", "v_scale"):
            if k in s.t[0]:
                s.t[0][k].zero_()
    b.t[0]["val"].copy_(a.t[0]["val"])
    start = a.t[0]["val"].clone()
    pa, pb = a.plan(nb), b.plan(nb)
    g = torch.Generator(device="cuda").manual_seed(0)
    base = a.t[0]["grad"].clone()
    for step in range(1, 31):
        now = base * (1 + 0.5 * torch.randn(50000, generator=g, device="cuda"))
        for s in (a, b):
            s.t[0]["grad"].copy_(now)
        pa.step(**{**HYPER, "t": step, "wd": 0.0})
        pb.step(**{**HYPER, "t": step, "wd": 0.0})
    torch.cuda.synchronize()
    way = (a.t[0]["val"] - start).norm()
    # m is off by 2^-4 of itself at most after each step and forgets a tenth of that a step, the
    # root of v by 2^-4 and half of a twentieth: independent errors of 2^-4 / sqrt(3) add to
    # at most 0.036 sqrt(1 / (1 - 0.81)) = 0.08 and 0.036 sqrt(1 / (1 - 0.95)) = 0.16 of the update.
    assert (a.t[0]["val"] - b.t[0]["val"]).norm() <= 0.25 * way


def test_empty_tensors_and_empty_models(nb, torch):
    s = Tensors(torch, [0, 300, 0])
    before = s.clone()
    s.plan(nb).step(**HYPER)
    _same(torch, s.t[1], _want(torch, before[1], 1.0, HYPER["lr"], 7, 0.9, 0.95, 1e-8, 0.1, 32))
    norm = torch.full((1,), 9.0, device="cuda")
    nb.train.AdamwMany([]).step(**HYPER, max_norm=1.0, norm=norm.data_ptr())
    torch.cuda.synchronize()
    assert float(norm) == 0.0


def test_both_kinds_of_moments_in_one_model(nb, torch):
    a, b = Tensors(torch, [700, 5000], "bf16", 32, seed=8), Tensors(torch, [300, 9001], "bf16", 8, seed=9)
    before = a.clone(), b.clone()
    ta, tb = a.plan, b.plan
    made = []

    class Take:
        train = type("t", (), {"AdamwTensor": nb.train.AdamwTensor, "AdamwMany": staticmethod(made.extend)})

    ta(Take), tb(Take)
    plan = nb.train.AdamwMany([made[2], made[0], made[3], made[1]])
    plan.step(**HYPER)
    torch.cuda.synchronize()
    for s, was, bits in ((a, before[0], 32), (b, before[1], 8)):
        for t, w in zip(s.t, was):
            _same(torch, t, _want(torch, w, 1.0, HYPER["lr"], 7, 0.9, 0.95, 1e-8, 0.1, bits))


def test_streams_and_graphs(nb, torch):
    """Two models on two streams, and a captured step replayed: each replay is one more step."""
    sets = [Tensors(torch, SIZES, "bf16", 8, "bf16", seed=10), Tensors(torch, SIZES, "f32", 32, seed=11)]
    ref = [Tensors(torch, SIZES, "bf16", 8, "bf16", seed=10), Tensors(torch, SIZES, "f32", 32, seed=11)]
    for r in ref:
        p = r.plan(nb)
        for _ in range(4):
            p.step(**HYPER, max_norm=0.5)
    torch.cuda.synchronize()
    plans, streams, graphs = [s.plan(nb) for s in sets], [torch.cuda.Stream(), torch.cuda.Stream()], []
    for p, st in zip(plans, streams):
        p.step(**HYPER, max_norm=0.5, stream=st.cuda_stream)
    torch.cuda.synchronize()
    for p, st in zip(plans, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            p.step(**HYPER, max_norm=0.5, stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for s, r in zip(sets, ref):
        for a, b in zip(s.t, r.t):
            assert all(torch.equal(a[k], b[k]) for k in a if hasattr(a[k], "clone"))


def test_host_form(nb, torch):
    rng = np.random.default_rng(0)
    val, grad = rng.standard_normal(600).astype(np.float32), rng.standard_normal(600).astype(np.float32)
    zero = np.zeros(600, np.float32)
    out, norm = nb.adamw_step_many([dict(val=val, grad=grad, m=zero, v=zero, copy="f16"),
                                    dict(val=val, grad=grad, m=np.zeros(600), v=np.zeros(600), m_scale=np.zeros(3),
                                         v_scale=np.zeros(3), decay=False)], lr=0.1, t=1, wd=0.01)
    v, m, vv = nb.adamw_step(val, grad, zero, zero, 0.1, 1, True, wd=0.01)
    assert np.array_equal(out[0]["val"], v) and np.array_equal(out[0]["m"], m) and np.array_equal(out[0]["v"], vv)
    assert np.array_equal(out[0]["copy"], v.astype(np.float16))
    # (The first step moves a value by 0.1: 18 U of that, and the value's rounding.)
    assert np.abs(out[1]["val"] - nb.adamw_step(val, grad, zero, zero, 0.1, 1, False)[0]).max() <= 18 * U * 0.1 + 4 * 2 * U
    assert out[1]["m"].dtype == np.uint8 and out[1]["m_scale"].shape == (3,) and (out[1]["m_scale"] > 0).all()
    assert abs(norm - np.sqrt(2 * (grad.astype(np.float64) ** 2).sum())) < 1e-5
    grad[7] = np.nan
    with pytest.raises(nb.NoeticError):
        nb.adamw_step_many([dict(val=val, grad=grad, m=zero, v=zero)], lr=0.1, t=1)


def test_host_form_leaves_everything_where_the_norm_is_not_finite(nb):
    rng = np.random.default_rng(1)
    a = {k: rng.standard_normal(700).astype(np.float32) for k in ("val", "grad", "m", "v")}
    a["copy"] = rng.integers(0, 1 << 16, 700).astype(np.uint16)
    a["grad"][5] = np.inf
    before = {k: v.copy() for k, v in a.items()}
    t = (nb.train.NkAdamwTensor * 1)(nb.train.NkAdamwTensor(
        a["val"].ctypes.data, a["grad"].ctypes.data, a["m"].ctypes.data, a["v"].ctypes.data, None, None,
        a["copy"].ctypes.data, 700, 0, 2, 32, 1))
    cfg, norm = nb.NkAdamwCfg(0.1, 0.9, 0.95, 1e-8, 0.0, 1, 1), C.c_float()
    assert nb.lib().nk_adamw_many_step(t, 1, C.byref(cfg), 1.0, 1.0, C.byref(norm), 0) == nb.NK_ERR_INVALID
    assert norm.value == np.inf
    for k, v in a.items():
        assert v.tobytes() == before[k].tobytes(), k


@pytest.mark.parametrize("grad,copy", [("f32", None), ("bf16", "bf16")])
def test_8_bits_do_not_depend_on_where_a_tensor_lies(nb, torch, grad, copy):
    """The same tensors on and off 16-byte boundaries, and one whose broken element sends its
    block through the careful form: the same numbers, bit for bit."""
    sets = [Tensors(torch, SIZES, grad, 8, copy, shift, seed=13) for shift in (0, 1, 0)]
    for i in range(4):
        for k, s in enumerate(sets):
            for t in s.t:
                if k == 2 and t["n"] > 9:
                    t["val"][9] = float("inf")
            s.plan(nb).step(**{**HYPER, "t": 7 + i})
        torch.cuda.synchronize()
        for a, b, c in zip(*(s.t for s in sets)):
            for k in ("val", "m", "v", "m_scale", "v_scale") + (("copy",) if copy else ()):
                assert torch.equal(a[k], b[k]), (k, a["n"])
            if i == 0 and a["n"] > 9:  # (whose moments stay, and may have been the block's largest)
                keep = torch.arange(a["n"], device="cuda") != 9
                assert torch.equal(a["val"][keep], c["val"][keep])


@pytest.mark.parametrize("shift", [0, 3])
def test_a_moment_that_is_not_finite_spoils_no_other(nb, torch, shift):
    """A byte that is no number, or a block whose scale is infinite: those elements stay as they
    are, `bad` says so, and all others go on as they would without them."""
    s, ref = (Tensors(torch, [1000, 512], bits=8, shift=shift, seed=14) for _ in range(2))
    for t in (s.t[0], ref.t[0]):
        t["m"][7], t["v"][300] = 0, 1  # (nothing to the blocks' largest)
    s.t[0]["m"][7] = 127
    s.t[0]["v"][300] = 127
    s.t[1]["m_scale"][1] = float("inf")
    before = s.clone()
    bad = torch.zeros(1, device="cuda", dtype=torch.int32)
    for x, b in ((s, bad.data_ptr()), (ref, None)):
        x.plan(nb).step(**HYPER, bad=b)
    torch.cuda.synchronize()
    assert int(bad) == 1
    t, r = s.t[0], ref.t[0]
    kept = torch.ones(1000, dtype=torch.bool, device="cuda")
    kept[[7, 300]] = False
    for k in ("val", "m", "v"):
        assert torch.equal(t[k][kept], r[k][kept]), k
    assert torch.equal(t["val"][~kept], before[0]["val"][~kept])
    assert int(t["m"][7]) & 127 == 127 and int(t["v"][300]) & 127 == 127
    assert torch.equal(t["m_scale"], r["m_scale"]) and torch.equal(t["v_scale"], r["v_scale"])
    t, r = s.t[1], ref.t[1]
    assert torch.equal(t["val"][:256], r["val"][:256]) and torch.equal(t["val"][256:], before[1]["val"][256:])


def _pair(torch, n, seed):
    """The same tensor with 32-bit and with 8-bit moments, all zero."""
    a, b = Tensors(torch, [n], seed=seed), Tensors(torch, [n], bits=8, seed=seed)
    for s in (a, b):
        for k in ("m", "v", "m_scale", "v_scale"):
            if k in s.t[0]:
                s.t[0][k].zero_()
    b.t[0]["val"].copy_(a.t[0]["val"])
    return a, b


def _stored(torch, t, k):
    return t[k].view(torch.float8_e4m3fn).double() * t[k + "_scale"].double().repeat_interleave(256)[:t["n"]]


@pytest.mark.parametrize("noise", [1.0, 0.0])
@pytest.mark.parametrize("b2,steps", [(0.98, 600), (0.99, 1200), (0.999, 5000)])
def test_8_bit_roots_follow_gradients_that_shrink(nb, torch, b2, steps, noise):
    """A third of the way in, half the elements' gradients fall to a tenth.  A stored v's mean
    is the formula's; one element's is off by the roundings that it remembers: each at most a
    step's square over 4, (1/8)^2 / 4 of v at a step that moves it that far, and a step's
    share is (1 - b2) and the scale's: 30% of v an element (measured: 0.32).  25600 of them:
    0.2%; 5% is far off that and far below what rounding to nearest does (4 to 90 times v)."""
    n = 51200
    a, b = _pair(torch, n, 20)
    pa, pb = a.plan(nb), b.plan(nb)
    g = torch.Generator(device="cuda").manual_seed(3)
    size = torch.exp(torch.randn(n, generator=g, device="cuda") - 6)
    half = torch.arange(n, device="cuda") % 2 == 0
    for step in range(1, steps + 1):
        now = size * (torch.randn(n, generator=g, device="cuda") if noise else 1.0)
        if step > steps // 3:
            now[half] *= 0.1
        for s, p in ((a, pa), (b, pb)):
            s.t[0]["grad"].copy_(now)
            p.step(**{**HYPER, "t": step, "b2": b2, "wd": 0.0})
    torch.cuda.synchronize()
    ratio = _stored(torch, b.t[0], "v").square() / a.t[0]["v"].double()
    for which in (half, ~half):
        assert abs(float(ratio[which].mean()) - 1) <= 0.05, (float(ratio[half].mean()), float(ratio[~half].mean()))


@pytest.mark.parametrize("b1", [0.98, 0.99])
def test_8_bit_means_follow_gradients_that_turn(nb, torch, b1):
    """Gradients without noise, half of which turn round.  A stored m's mean is the formula's:
    over 25600 elements the errors (at most 1/16 of m each, and 1 / sqrt(1 - b1^2) of that
    remembered: 0.44) average to 0.3%; to nearest, m had not turned at all."""
    n, steps = 51200, 1500
    a, b = _pair(torch, n, 21)
    pa, pb = a.plan(nb), b.plan(nb)
    g = torch.Generator(device="cuda").manual_seed(4)
    size = torch.exp(torch.randn(n, generator=g, device="cuda") - 6)
    half = torch.arange(n, device="cuda") % 2 == 0
    for step in range(1, steps + 1):
        for s, p in ((a, pa), (b, pb)):
            s.t[0]["grad"].copy_(torch.where(half & (step > steps // 2), -size, size))
            p.step(**{**HYPER, "t": step, "b1": b1, "wd": 0.0})
    torch.cuda.synchronize()
    ratio = _stored(torch, b.t[0], "m") / a.t[0]["m"].double()
    for which in (half, ~half):
        assert abs(float(ratio[which].mean()) - 1) <= 0.05, float(ratio[which].mean())


@pytest.mark.parametrize("grad", ["f32", "bf16"])
def test_rounding_by_chance_is_between_neighbours_in_proportion_and_repeats(nb, torch, grad):
    n = 1 << 18
    hyper = {**HYPER, "b1": 0.96, "b2": 0.97}
    sets = [Tensors(torch, [n, 1000], grad, 8, shift=shift, seed=22) for shift in (0, 0, 3)]
    for s in sets:
        s.t[0]["val"].copy_(sets[0].t[0]["val"])
        # (Roots that are not tiny: of those the floor moves the mean.  127 is no number.)
        s.t[0]["v"].copy_((s.t[0]["v"] | 8).clamp(max=126))
    before = sets[0].clone()
    for s in sets:
        s.plan(nb).step(**hyper)
    torch.cuda.synchronize()
    for i, t in enumerate(sets[0].t):
        for o in sets[1:]:
            assert all(torch.equal(t[k], o.t[i][k]) for k in ("val", "m", "v", "m_scale", "v_scale"))
    t, want = sets[0].t[0], _want(torch, before[0], 1.0, HYPER["lr"], 7, 0.96, 0.97, 1e-8, 0.1, 8)
    err = (t["val"].double() - want["val"]).abs()
    assert (err <= U * want["val"].abs() + want["val_tol"]).all()
    for k in ("m", "v"):
        scale = t[k + "_scale"].double().repeat_interleave(256)
        y, code = (want[k] / scale).abs(), t[k].view(torch.float8_e4m3fn).double()
        assert ((code == 0) | (torch.sign(code) == torch.sign(want[k]))).all()
        code = code.abs()
        slack = 32 * U * y + want[k + "_tol"] / scale
        # Within a step, and one of the two beside it where it is not on the grid itself.
        step = torch.exp2(torch.floor(torch.log2(torch.maximum(y, code).clamp(min=2.0**-6))) - 3)
        assert ((code - y).abs() < step + slack).all()
        # The further of the two takes its share (what lies near the middle left out).
        f = torch.frac(y / torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0**-6))) - 3))
        share = float(((code - y).abs() > step * 0.51).double().mean())
        assert share > 0.5 * float(torch.minimum(f, 1 - f).mean()) > 0.01
        # Its mean (the square's), over elements of one size: 6 deviations of at most half a step each.
        for lo in (2.0**-7, 0.5, 3.0, 40.0, 200.0):
            at = (y >= lo) & (y < 2 * lo)
            if int(at.sum()) <= 500 and lo < 3.0:  # (v: none so small)
                continue
            d = code[at] - y[at] if k == "m" else (code[at].square() - y[at].square()) / (2 * y[at])
            most = float(step[at].max()) / 2 * 1.1
            assert abs(float(d.mean())) <= 6 * most / int(at.sum()) ** 0.5, (k, lo, float(d.mean()), most)
