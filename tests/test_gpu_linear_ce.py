"""Cross entropy from hidden rows and its gradients (include/noetic/train.h) on
the GPU against their definitions in 64 bits.

Tolerances count roundings, U = 2^-24 being half a step of f32.  With A = sum_k
|x_k w_k| of a logit:
 - products of 16-bit elements are exact in f32.  A sum of d of them passes each
   through at most d additions that round (U each), or d / 16 + 5 of the tensor
   cores' that cut (2 U each): off by (d + 64) U A at most.
 - f32 elements are taken with 22 bits (2^-22 of each factor, and 2^-40 of the
   largest element of its matrix below that): 2^-21 A + 2^-39 d max|x| max|w|.
 - loss = (m - z_t) + log s: two logits, the sum's own error (a mean of the
   logits' errors, 2^-22 of the exponential, N / 32 + 64 additions) and the
   rounding of differences of the size of the spread: 2 max dz + (N / 32 + 80 +
   4 Y) U.
 - p comes with dz, the 2 U (|m| + log s) of the statistics and 2^-22; G with half a
   step of its type more (f32: 2^-22), and 2^-38 of the largest weight; the
   products add (K + 64) U of sum |G| |w| and the output's rounding.
"""

import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0**-24
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


def _matrix(torch, rows, width, dtype, pad=0, shift=0, scale=1.0, seed=0):
    """A [rows, width] view whose rows start `shift` elements into an array of
    row stride width + pad (NaN around the rows)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    whole = torch.full((shift + rows * (width + pad) + 8,), NAN, device="cuda", dtype=_dt(torch, dtype))
    v = whole[shift:shift + rows * (width + pad)].view(rows, width + pad)[:, :width]
    v.copy_(torch.randn(rows, width, generator=g, device="cuda") * scale)
    return v


class Case:
    """Inputs, and what the definitions give for them in 64 bits."""

    def __init__(self, torch, rows, width, vocab, dtype, ignored=0.0, pad=0, shift=0, seed=0, spread=2.0, weights=True):
        g = torch.Generator(device="cuda").manual_seed(seed + 7)
        self.torch, self.dtype, self.rows, self.width, self.vocab = torch, dtype, rows, width, vocab
        self.x = _matrix(torch, rows, width, dtype, pad, shift, 1.0, seed)
        self.w = _matrix(torch, vocab, width, dtype, pad, shift, spread / width**0.5, seed + 1)
        self.targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
        dead = torch.rand(rows, generator=g, device="cuda") < ignored
        self.targets[dead] = -1
        self.x[dead] = NAN  # (What stands in a row that does not count can be anything.)
        self.weight = torch.rand(rows, generator=g, device="cuda") + 0.5 if weights else None
        self.live = ~dead

    def workspace(self, nb, backward):
        n = nb.train.linear_ce_workspace(CODE[self.dtype], self.rows, self.width, self.vocab, self.w.data_ptr(),
                                         self.w.stride(0), backward)
        return self.torch.full((n + 64,), 255, device="cuda", dtype=self.torch.uint8)  # (NaN in every type)

    def forward(self, nb, room=None, targets=None):
        torch = self.torch
        room = self.workspace(nb, False) if room is None else room
        loss = torch.full((self.rows,), 5.0, device="cuda")
        stats = torch.full((self.rows, 2), 5.0, device="cuda")
        nb._check(nb.lib().nk_linear_ce_device(
            _p(self.x), CODE[self.dtype], self.rows, self.width, self.x.stride(0), _p(self.w), self.vocab,
            self.w.stride(0), _p(self.targets if targets is None else targets), _p(loss), _p(stats), _p(room),
            room.numel() - 64, _st(torch)))
        return loss, stats

    def backward(self, nb, stats, scale=1.0, dw_dtype=None, dw=None, dx=None, want_dx=True, want_dw=True, room=None):
        torch = self.torch
        room = self.workspace(nb, True) if room is None else room
        add = dw is not None
        dw_dtype = dw_dtype or self.dtype
        if want_dx and dx is None:
            dx = torch.full((self.rows, self.width), 5.0, device="cuda", dtype=_dt(torch, self.dtype))
        if want_dw and dw is None:
            dw = torch.full((self.vocab, self.width), 5.0, device="cuda", dtype=_dt(torch, dw_dtype))
        nb._check(nb.lib().nk_linear_ce_backward_device(
            _p(self.x), CODE[self.dtype], self.rows, self.width, self.x.stride(0), _p(self.w), self.vocab,
            self.w.stride(0), _p(self.targets), _p(stats), _p(self.weight), scale, _p(dx),
            0 if dx is None else dx.stride(0), _p(dw), CODE[dw_dtype], 0 if dw is None else dw.stride(0), int(add),
            _p(room), room.numel() - 64, _st(torch)))
        return dx, dw

    # ---- 64 bits
    def x64(self):
        return self.torch.where(self.live[:, None], self.x.double(), 0.0)

    def logits(self):
        return self.x64() @ self.w.double().T

    def dz(self):
        """The most that a logit can be off, for each logit."""
        x, w = self.x64().abs(), self.w.double().abs()
        tol = (self.width + 64) * U * (x @ w.T)
        if self.dtype == "f32":
            tol = tol * (1 + 8 / (self.width + 64)) + 2.0**-39 * self.width * float(x.max()) * float(w.max())
        return tol

    def check_forward(self, loss, stats):
        torch = self.torch
        z, dz = self.logits(), self.dz().max(-1).values
        lse, m = torch.logsumexp(z, -1), z.max(-1).values
        at = z.gather(1, self.targets.long().clamp(min=0)[:, None])[:, 0]
        y = (m - z.min(-1).values)
        own = (self.vocab / 32 + 80 + 4 * y) * U
        zero = torch.zeros((), device="cuda", dtype=torch.float64)
        err = (loss.double() - torch.where(self.live, lse - at, zero)).abs()
        assert (err <= torch.where(self.live, 2 * dz + own, zero)).all(), float(err.max())
        err = (stats.double() - torch.stack([m, lse - m], 1) * self.live[:, None]).abs()
        tol = torch.stack([dz + U * m.abs(), 2 * dz + own + U * (lse - m).abs()], 1) * self.live[:, None]
        assert (err <= tol).all(), float(err.max())

    def check_backward(self, stats, scale, dx=None, dw=None, base=None):
        torch = self.torch
        eps = {"f32": 2.0**-22, "f16": 2.0**-11, "bf16": 2.0**-8}[self.dtype]
        h = self.weight.double() if self.weight is not None else torch.ones(self.rows, device="cuda", dtype=torch.float64)
        h = torch.where(self.live, h * scale, 0.0)[:, None]
        x, w, st = self.x64(), self.w.double(), stats.double()
        p = torch.exp(self.logits() - st.sum(1, keepdim=True))
        hot = torch.zeros_like(p).scatter_(1, self.targets.long().clamp(min=0)[:, None], 1.0)
        G = h * (p - hot)
        dG = h.abs() * p * torch.expm1(self.dz() + 2 * U * (st.abs().sum(1, keepdim=True) + 4)) + 4 * U * h.abs() * hot
        dG = dG + eps * (G.abs() + dG) + 2.0**-38 * h.abs().max()
        dG = dG * (h != 0)
        for out, a, b, db in ((dx, G, w, dG), (dw, G.T, x, dG.T)):
            if out is None:
                continue
            ref = a @ b
            tol = db @ b.abs() + (b.shape[0] + 64) * U * (a.abs() @ b.abs()) * (1 + (8 / (b.shape[0] + 64) if self.dtype == "f32" else 0))
            if self.dtype == "f32":
                # The product's own factors: 2^-22 of each element, 2^-40 of the largest.
                tol = tol + a.abs().sum(1, keepdim=True) * float(b.abs().max()) * 2.0**-39
            if out is dw and base is not None:
                ref = ref + base.double()
            f = torch.finfo(out.dtype)
            tol = tol + (f.eps / 2) * (ref.abs() + tol) + f.smallest_normal * f.eps / 2
            err = (out.double() - ref).abs()
            assert (err <= tol).all(), (float(err.max()), float((err / tol.clamp(min=1e-300)).max()))


SIZES = [(1, 1, 1), (1, 64, 1000), (2, 3, 5), (7, 17, 300), (64, 192, 1024), (129, 100, 1003), (255, 72, 515),
         (257, 136, 769), (300, 767, 2003), (513, 64, 33), (1, 1024, 32768), (5, 4096, 259), (17, 65, 8192)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width,vocab", SIZES)
def test_forward(nb, torch, rows, width, vocab, dtype):
    c = Case(torch, rows, width, vocab, dtype)
    c.check_forward(*c.forward(nb))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width,vocab", SIZES)
def test_backward(nb, torch, rows, width, vocab, dtype):
    c = Case(torch, rows, width, vocab, dtype)
    _, stats = c.forward(nb)
    c.check_backward(stats, 0.25, *c.backward(nb, stats, 0.25))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad,shift,ignored", [(0, 0, 0.4), (1, 0, 0.0), (8, 0, 0.2), (3, 1, 0.2), (16, 5, 0.9)])
def test_strides_places_and_padded_batches(nb, torch, dtype, pad, shift, ignored):
    c = Case(torch, 333, 200, 1500, dtype, ignored=ignored, pad=pad, shift=shift, seed=3)
    loss, stats = c.forward(nb)
    c.check_forward(loss, stats)
    # Outputs with strides of their own; what lies between their rows stays.
    dx = torch.full((333, 207), 7.0, device="cuda", dtype=_dt(torch, dtype))
    dw = torch.full((1500, 203), 7.0, device="cuda", dtype=_dt(torch, dtype))
    room = c.workspace(nb, True)
    nb._check(nb.lib().nk_linear_ce_backward_device(
        _p(c.x), CODE[dtype], 333, 200, c.x.stride(0), _p(c.w), 1500, c.w.stride(0), _p(c.targets), _p(stats),
        _p(c.weight), 1e-3, _p(dx), 207, _p(dw), CODE[dtype], 203, 0, _p(room), room.numel() - 64, _st(torch)))
    c.check_backward(stats, 1e-3, dx[:, :200], dw[:, :200])
    assert (dx[:, 200:] == 7).all() and (dw[:, 200:] == 7).all()
    assert (dx[:, :200][~c.live] == 0).all()
    assert (room[-64:] == 255).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_no_row_counts(nb, torch, dtype):
    c = Case(torch, 70, 64, 300, dtype)
    c.targets[:] = -1
    c.live[:] = False
    c.x[:] = NAN
    loss, stats = c.forward(nb)
    assert (loss == 0).all() and (stats == 0).all()
    dx, dw = c.backward(nb, stats)
    assert (dx == 0).all() and (dw == 0).all()
    base = torch.ones(300, 64, device="cuda", dtype=_dt(torch, dtype))
    _, dw = c.backward(nb, stats, dw=base.clone())
    assert torch.equal(dw, base)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_ids_beyond_the_vocabulary_are_no_token_and_weights_of_zero_add_nothing(nb, torch, dtype):
    c = Case(torch, 90, 96, 700, dtype, seed=5)
    c.targets[::3] = 700
    c.targets[1::7] = 2**31 - 1
    c.live = (c.targets >= 0) & (c.targets < 700)
    dead = ~c.live
    loss, stats = c.forward(nb)
    c.targets[dead] = -1
    c.x[dead] = NAN
    c.check_forward(loss, stats)
    c.weight[::5] = 0.0
    off = c.live & (c.weight == 0)
    dx, dw = c.backward(nb, stats)
    c.check_backward(stats, 1.0, dx, dw)
    # Their rows are not read.
    c.x[off] = INF
    again = c.backward(nb, stats)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1]) and (dx[off] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_each_output_alone_f32_sums_and_accumulation(nb, torch, dtype):
    c = Case(torch, 270, 130, 900, dtype, ignored=0.1, seed=6)
    _, stats = c.forward(nb)
    dx, dw = c.backward(nb, stats, 0.5)
    alone_x, none = c.backward(nb, stats, 0.5, want_dw=False)
    assert none is None and torch.equal(alone_x, dx)
    none, alone_w = c.backward(nb, stats, 0.5, want_dx=False)
    assert none is None and torch.equal(alone_w, dw)
    _, wide = c.backward(nb, stats, 0.5, dw_dtype="f32")
    c.check_backward(stats, 0.5, None, wide)
    assert torch.equal(wide.to(dw.dtype), dw)
    base = torch.randn(900, 130, device="cuda")
    _, added = c.backward(nb, stats, 0.5, dw_dtype="f32", dw=base.clone())
    c.check_backward(stats, 0.5, None, added, base)
    low = base.to(_dt(torch, dtype))
    _, added = c.backward(nb, stats, 0.5, dw=low.clone())
    c.check_backward(stats, 0.5, None, added, low)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_several_pieces_of_the_vocabulary(nb, torch, dtype):
    c = Case(torch, 5000, 48, 60001, dtype, ignored=0.05, seed=8)
    loss, stats = c.forward(nb)
    c.check_forward(loss, stats)
    torch.cuda.empty_cache()
    c.check_backward(stats, 1 / 5000, *c.backward(nb, stats, 1 / 5000))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_many_rows_of_a_tiny_vocabulary(nb, torch, dtype):
    c = Case(torch, 70001, 24, 37, dtype, ignored=0.3, seed=9)
    loss, stats = c.forward(nb)
    c.check_forward(loss, stats)
    c.check_backward(stats, 1 / 70001, *c.backward(nb, stats, 1 / 70001))


def test_sure_tokens_and_far_logits(nb, torch):
    """Logits in the thousands: p is 0 or 1, and nothing overflows."""
    for dtype in ("f32", "f16", "bf16"):
        c = Case(torch, 40, 64, 500, dtype, spread=500.0, seed=10)
        loss, stats = c.forward(nb)
        c.check_forward(loss, stats)
        dx, dw = c.backward(nb, stats)
        assert torch.isfinite(dx).all() and torch.isfinite(dw).all()
        c.check_backward(stats, 1.0, dx, dw)


@pytest.mark.parametrize("scale", [1e-20, 1e15])
def test_f32_and_bf16_values_far_from_one(nb, torch, scale):
    for dtype in ("f32", "bf16"):
        c = Case(torch, 50, 80, 300, dtype, seed=11)
        c.x.mul_(scale)
        c.w.div_(scale)
        loss, stats = c.forward(nb)
        c.check_forward(loss, stats)
        c.check_backward(stats, 1.0, *c.backward(nb, stats))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_broken_rows_leave_the_others_alone(nb, torch, dtype):
    c = Case(torch, 300, 128, 600, dtype, seed=12)
    loss, stats = c.forward(nb)
    c.x[17, 3] = NAN
    c.x[211, 0] = INF
    bad = torch.zeros(300, dtype=torch.bool, device="cuda")
    bad[[17, 211]] = True
    broken, st = c.forward(nb)
    assert torch.isnan(broken[bad]).all() and torch.isnan(st[bad]).all()
    assert torch.equal(broken[~bad], loss[~bad]) and torch.equal(st[~bad], stats[~bad])
    c.w[5, 9] = NAN
    broken, _ = c.forward(nb)
    assert torch.isnan(broken).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_weights_that_are_not_finite_break_their_rows(nb, torch, dtype):
    c = Case(torch, 300, 128, 600, dtype, seed=13)
    _, stats = c.forward(nb)
    c.weight[[17, 211]] = 1.0
    dx, _ = c.backward(nb, stats)
    c.weight[17], c.weight[211] = INF, NAN
    bad = torch.zeros(300, dtype=torch.bool, device="cuda")
    bad[[17, 211]] = True
    broken, dw = c.backward(nb, stats)
    assert not torch.isfinite(broken[bad]).any() and torch.equal(broken[~bad], dx[~bad])
    assert torch.isnan(dw).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradients_against_differences(nb, torch, dtype):
    """Along random directions, central differences of the 64-bit loss."""
    c = Case(torch, 60, 40, 200, dtype, ignored=0.2, seed=13)
    _, stats = c.forward(nb)
    dx, dw = c.backward(nb, stats, 2.0, dw_dtype="f32")
    x, w, t = c.x64(), c.w.double(), c.targets.long().clamp(min=0)[:, None]

    def total(x, w):
        z = x @ w.T
        loss = torch.logsumexp(z, -1) - z.gather(1, t)[:, 0]
        return float((2.0 * c.weight.double() * torch.where(c.live, loss, 0.0)).sum())

    g = torch.Generator(device="cuda").manual_seed(1)
    half = {"f32": 2.0**-20, "bf16": 2.0**-8}[dtype]
    for out, v, f in ((dx, x, lambda u: total(x + u, w)), (dw, w, lambda u: total(x, w + u))):
        u = torch.randn(v.shape, generator=g, device="cuda", dtype=torch.float64) * 1e-4
        if out is dx:
            u *= c.live[:, None]
        want, got = (f(u) - f(-u)) / 2, float((out.double() * u).sum())
        # Each element of the gradient: its own rounding and those of the 200 or 60
        # terms of its sum; the differences: their second order, |u|^3.
        bound = 4 * half * float((out.double() * u).abs().sum()) + half * float(u.abs().sum()) + 1e-9
        assert abs(want - got) <= bound, (want, got, bound)


def test_calls_on_streams_and_graphs_side_by_side(nb, torch):
    cases = [Case(torch, 700, 256, 4000, "bf16", ignored=0.2, seed=20), Case(torch, 400, 192, 3000, "f32", seed=21)]
    want = []
    for c in cases:
        loss, stats = c.forward(nb)
        want.append((loss, stats, *c.backward(nb, stats, 0.1)))
    torch.cuda.synchronize()
    rooms = [(c.workspace(nb, False), c.workspace(nb, True)) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        got = []
        for c, s, room in zip(cases, streams, rooms):
            with torch.cuda.stream(s):
                loss, stats = c.forward(nb, room[0])
                got.append((loss, stats, *c.backward(nb, stats, 0.1, room=room[1])))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    graphs, outs = [], []
    for c, s, room in zip(cases, streams, rooms):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            loss, stats = c.forward(nb, room[0])
            outs.append((loss, stats, *c.backward(nb, stats, 0.1, room=room[1])))
        graphs.append(g)
    # Other inputs in the same arrays: the replay computes with them.
    for c in cases:
        c.targets.copy_(c.targets.flip(0))
        c.x.copy_(c.x.flip(0))
        c.live = c.live.flip(0)
        c.weight.copy_(c.weight.flip(0))
    torch.cuda.synchronize()
    for _ in range(2):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for c, (loss, stats, dx, dw) in zip(cases, outs):
        c.check_forward(loss, stats)
        c.check_backward(stats, 0.1, dx, dw)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_no_rows_set_dw_to_zero_and_negative_weights_count(nb, torch, dtype):
    c = Case(torch, 65, 40, 260, dtype, seed=14)
    _, stats = c.forward(nb)
    c.weight[::2] *= -3.0
    c.check_backward(stats, 0.5, *c.backward(nb, stats, 0.5))
    c.check_backward(stats, -0.5, *c.backward(nb, stats, -0.5))
    # grad_scale 0: zeros.
    dx, dw = c.backward(nb, stats, 0.0)
    assert (dx == 0).all() and (dw == 0).all()
    none = Case(torch, 1, 40, 260, dtype, seed=15)
    none.rows = 0
    none.x, none.targets, none.weight = none.x[:0], none.targets[:0], None
    _, dw = none.backward(nb, torch.zeros(0, 2, device="cuda"), want_dx=False)
    assert (dw == 0).all()


def test_f32_factors_far_apart(nb, torch):
    """x and w whose products are ordinary, and whose sizes are the ends of f32's range."""
    for rows in (40, 300):
        c = Case(torch, rows, 96, 5000, "f32", seed=16)
        for scale in (1e32, 1e-32):
            c.x.mul_(scale)
            c.w.div_(scale)
            c.check_forward(*c.forward(nb))
            c.x.div_(scale)
            c.w.mul_(scale)
        # Rows of very different sizes.
        c.x[::2] *= 1e-12
        c.w[::3] *= 1e-9
        c.check_forward(*c.forward(nb))


def test_two_host_threads_at_once(nb, torch):
    import threading

    cases = [Case(torch, 300 + 40 * i, 64 + 32 * i, 3000 + 500 * i, ["f32", "f16", "bf16", "bf16"][i], ignored=0.1, seed=40 + i)
             for i in range(4)]
    want = []
    for c in cases:
        loss, stats = c.forward(nb)
        want.append((loss, stats, *c.backward(nb, stats, 0.1)))
    rooms = [(c.workspace(nb, False), c.workspace(nb, True)) for c in cases]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            st = torch.cuda.Stream()
            for _ in range(20):
                with torch.cuda.stream(st):
                    loss, stats = cases[i].forward(nb, rooms[i][0])
                    got[i] = (loss, stats, *cases[i].backward(nb, stats, 0.1, room=rooms[i][1]))
            st.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_a_training_step_end_to_end(nb, torch):
    """Hidden rows, loss, gradients, a clipped AdamW step of the vocabulary matrix and its
    16-bit copy, which the next loss reads: as a training program runs them, beside the
    same steps in 64 bits with the copy rounded where the program rounds it."""
    rows, d, V = 256, 64, 500
    c = Case(torch, rows, d, V, "bf16", ignored=0.1, seed=50, weights=False)
    val = c.w.float().clone()
    w = val.to(torch.bfloat16)
    c.w = w
    dw = torch.zeros(V, d, device="cuda")
    m, v = torch.zeros_like(dw), torch.zeros_like(dw)
    norm = torch.zeros(1, device="cuda")
    plan = nb.train.AdamwMany([nb.train.AdamwTensor(val=val.data_ptr(), grad=dw.data_ptr(), m=m.data_ptr(), v=v.data_ptr(),
                                                    copy=w.data_ptr(), n=V * d, copy_dtype=2)])
    n = int(c.live.sum())
    v64, m64, s64 = val.double().clone(), m.double(), v.double()
    for t in range(1, 6):
        loss, stats = c.forward(nb)
        c.check_forward(loss, stats)
        dx, _ = c.backward(nb, stats, 1 / n, dw_dtype="f32", dw=dw.zero_())
        c.check_backward(stats, 1 / n, dx, dw)
        g = dw.double()
        plan.step(lr=1e-2, t=t, max_norm=0.05, norm=norm.data_ptr())
        g = g * min(1.0, 0.05 / float(g.norm()))
        m64, s64 = 0.9 * m64 + 0.1 * g, 0.95 * s64 + 0.05 * g * g
        v64 = v64 - 1e-2 * (m64 / (1 - 0.9**t)) / (torch.sqrt(s64 / (1 - 0.95**t)) + 1e-8)
        # Five steps of at most lr each, 16 U of each, and the values' rounding; 0.9 and 0.95 are
        # taken as f32, 2^-25 of them, which the corrections magnify by 1 / (1 - b) at most.
        assert (val.double() - v64).abs().max() <= t * (1e-2 * 64 * U + U * float(val.abs().max()))
        assert torch.equal(w, val.to(torch.bfloat16))


def test_host_form_and_python_mirror(nb):
    rng = np.random.default_rng(0)
    x, w = rng.standard_normal((30, 50), np.float32), rng.standard_normal((90, 50), np.float32) * 0.3
    t = rng.integers(0, 90, 30)
    t[4] = -1
    out = nb.linear_cross_entropy(x, w, t)
    z = x.astype(np.float64) @ w.T.astype(np.float64)
    lse = np.log(np.exp(z).sum(1))
    want = np.where(t >= 0, lse - z[np.arange(30), t], 0.0)
    assert np.abs(out["loss"] - want).max() < 2e-5  # (114 U A of two logits, A about 20)
    base = rng.standard_normal((90, 50)).astype(np.float32)
    dx, dw = nb.linear_cross_entropy_backward(x, w, t, out["stats"], grad_scale=0.5)
    dx2, dw2 = nb.linear_cross_entropy_backward(x, w, t, out["stats"], grad_scale=0.5, dw=base)
    G = 0.5 * np.exp(z - lse[:, None])
    G[np.arange(30), t] -= 0.5
    G[4] = 0
    assert np.abs(dx - G @ w).max() < 2e-5 and np.abs(dw - G.T @ x).max() < 4e-5
    assert np.array_equal(dx, dx2) and np.abs(dw2 - base - dw).max() < 1e-6
    with pytest.raises(nb.NoeticError):
        nb.linear_cross_entropy(x, w, np.full(30, 90))
    with pytest.raises(ValueError):
        nb.linear_cross_entropy(x, w.astype(np.float16), t)
    with pytest.raises(ValueError):
        nb.linear_cross_entropy_backward(x, w, t, out["stats"], dw=base[:5])


def test_the_loss_is_that_of_the_logits(nb, torch):
    """Beside nk_token_logprobs of the same logits, and its gradient."""
    c = Case(torch, 200, 64, 1000, "f32", seed=30, weights=False)
    loss, stats = c.forward(nb)
    z = c.logits().float()
    lp = torch.empty(200, device="cuda")
    nb._check(nb.lib().nk_token_logprobs_device(_p(z), 0, 200, 1000, 1000, _p(c.targets), 1.0, 0, _p(lp), None, None, None,
                                                None, _st(torch)))
    tol = 2 * c.dz().max() + (1000 / 32 + 200) * U + U * z.abs().max() * 4
    assert (loss + lp).abs().max() <= tol


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width,vocab", [(600, 320, 1500), (300, 40, 5000)])
def test_a_wait_that_runs_out_leaves_nan_and_never_a_part_of_a_sum(nb, torch, dtype, rows, width, vocab):
    """A copy that never comes (a test control; the waits end after 2 ms): what is not the
    right number is NaN, and the next calls are as they were."""
    c = Case(torch, rows, width, vocab, dtype, ignored=0.1, seed=60)
    loss, stats = c.forward(nb)
    dx, dw = c.backward(nb, stats, 0.5)
    hold = nb.lib().nk_linear_ce_withhold
    assert hold(4) == nb.NK_ERR_INVALID and hold(-1) == nb.NK_ERR_INVALID
    try:
        nb._check(hold(1))
        broken, _ = c.forward(nb)
        if rows * width * vocab <= 1e8:  # (few products: a kernel without such waits)
            assert torch.equal(broken, loss)
        else:
            assert torch.isnan(broken[c.live]).all() and (broken[~c.live] == 0).all()
        nb._check(hold(2))
        gx, gw = c.backward(nb, stats, 0.5)
        assert torch.isnan(gx[c.live]).all() and torch.isnan(gw).all()
        nb._check(hold(3))
        for want_dx in (True, False):
            for got, want in zip(c.backward(nb, stats, 0.5, want_dx=want_dx), (dx, dw)):
                if got is None:
                    continue
                gone = torch.isnan(got)
                assert torch.equal(got[~gone], want[~gone])
                if (got.shape[0] == rows) == want_dx:
                    # The first tile of the first product that is there.
                    first = torch.nonzero(c.live)[:256, 0] if want_dx else slice(256)
                    assert gone[first, :256].all()
    finally:
        nb._check(hold(0))
    again, st = c.forward(nb)
    assert torch.equal(again, loss) and torch.equal(st, stats)
    for got, want in zip(c.backward(nb, stats, 0.5), (dx, dw)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_f32_sums_of_many_rows_do_not_drift(nb, torch, dtype):
    """dw in f32 of 65536 rows whose terms have one sign and one G: w = 0, so every p is what
    the statistics say, a power of two.  A chain of 16 K-blocks passes a term through 64
    additions that cut, and 5 (2 U each); 64 chains are added with U each; 4 U for the way
    out.  (One chain over all rows cuts 4096 times: 2960 U of f16, all one way.)"""
    rows, width, vocab = 65536, 2048, 2048
    g = torch.Generator(device="cuda").manual_seed(0)
    x = (1 + torch.rand(rows, width, generator=g, device="cuda")).to(_dt(torch, dtype))
    w = torch.zeros(vocab, width, device="cuda", dtype=_dt(torch, dtype))
    targets = torch.zeros(rows, device="cuda", dtype=torch.int32)
    stats = torch.tensor([0.0, 11 * np.log(2.0)], device="cuda", dtype=torch.float32).repeat(rows, 1)
    dw = torch.empty(vocab, width, device="cuda")
    room = torch.empty(nb.train.linear_ce_workspace(CODE[dtype], rows, width, vocab, w.data_ptr(), width, True), device="cuda",
                       dtype=torch.uint8)
    nb._check(nb.lib().nk_linear_ce_backward_device(
        _p(x), CODE[dtype], rows, width, width, _p(w), vocab, width, _p(targets), _p(stats), None, 1.0, None, 0, _p(dw), 0,
        width, 0, _p(room), room.numel(), _st(torch)))
    want = x.double().sum(0) / 2048
    off = (dw[1:].double() - want) / want
    assert float(off.abs().max()) <= (2 * (64 + 5) + 64 + 4) * U, float(off.abs().max()) / U


@pytest.mark.parametrize("dtype,top", [("f16", 100.0), ("bf16", 256.0), ("f32", 100.0)])
def test_probabilities_of_logits_far_from_zero(nb, torch, dtype, top):
    """Rows of one number each, under logits that are all top^2, exactly; a row's log-sum is
    what its statistics say.  dw is then G x, which shows each p: exp(-log sum), with the
    roundings of log s (U of it) and of the exponential (2^-22), below 16 U, and G's own."""
    rows, vocab = 64, 40
    x = torch.diag(torch.full((rows,), top, device="cuda")).to(_dt(torch, dtype))
    w = torch.full((vocab, rows), top, device="cuda").to(x.dtype)
    ls = torch.linspace(1.0, 4.0, rows, device="cuda")
    stats = torch.stack([torch.full_like(ls, top * top), ls], 1).contiguous()
    targets = torch.zeros(rows, device="cuda", dtype=torch.int32)
    dw = torch.empty(vocab, rows, device="cuda")
    room = torch.empty(nb.train.linear_ce_workspace(CODE[dtype], rows, rows, vocab, w.data_ptr(), rows, True), device="cuda",
                       dtype=torch.uint8)
    nb._check(nb.lib().nk_linear_ce_backward_device(
        _p(x), CODE[dtype], rows, rows, rows, _p(w), vocab, rows, _p(targets), _p(stats), None, 1.0, None, 0, _p(dw), 0, rows, 0,
        _p(room), room.numel(), _st(torch)))
    off = (dw[1:].double() / top) / torch.exp(-ls.double()) - 1
    assert float(off.abs().max()) <= {"f16": 2.0**-11, "bf16": 2.0**-8, "f32": 2.0**-22}[dtype] + 20 * U, float(off.abs().max())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_w_off_128_bytes_in_a_workspace_for_one_on_them(nb, torch, dtype):
    """2100 rows, from which on such a w is copied where there is room: the same numbers without."""
    rows, width, vocab = 2100, 192, 1100
    c = Case(torch, rows, width, vocab, dtype, ignored=0.1, shift=8, seed=61)
    assert c.w.data_ptr() % 128 == 16
    room = [nb.train.linear_ce_workspace(CODE[dtype], rows, width, vocab, w, width, back) for w in (256, 272) for back in (False, True)]
    assert room[0] < room[2] and room[1] < room[3]
    loss, stats = c.forward(nb)
    c.check_forward(loss, stats)
    dx, dw = c.backward(nb, stats, 0.5)
    c.check_backward(stats, 0.5, dx, dw)
    small = [torch.full((n + 64,), 255, device="cuda", dtype=torch.uint8) for n in room[:2]]
    got = c.forward(nb, small[0]) + c.backward(nb, stats, 0.5, room=small[1])
    for a, b in zip(got, (loss, stats, dx, dw)):
        assert torch.equal(a, b)
    assert all((s[-64:] == 255).all() for s in small)


_TRIES = (1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64)


def _up(n, to):
    return -(-n // to) * to


def _deal(items0, cost0, items1, cost1, pairs):
    """How many items of the second product a pair with one more, or one less, of the first takes."""
    more, q = items0 % pairs, items0 // pairs
    high, low = (q + 1) * cost0, q * cost0
    level = (items0 * cost0 + items1 * cost1 + pairs - 1) // pairs
    while True:
        n = [max(0, level - high) // cost1, max(0, level - low) // cost1]
        if more * n[0] + (pairs - more) * n[1] >= items1:
            return more, n[0], max(n)
        a, b = high + (n[0] + 1) * cost1, low + (n[1] + 1) * cost1
        level = a if more and a < b else b


def _cuts(dtype, rows, width, vocab, pairs=74):
    """(tokens of a piece, pieces of K of dx, of dw): the rule of a gradient call, restated."""
    parts, segs = (2, 3) if dtype == "f32" else (1, 1)
    mp = _up(max(rows, 1), 256)
    piece = min(max((256 << 20) // 2 // parts // mp // 256 * 256, 1024), vocab)
    ldg, nt = _up(piece, 256), _up(width, 256) // 256
    tx, kx, tw, kw = mp // 256 * nt, ldg // 64 * segs, ldg // 256 * nt, mp // 64 * segs
    least, best = 1e300, (1, 1)
    for i in _TRIES:
        for j in _TRIES:
            if (i > 1 and (kx // i < 8 or tx * i > 4 * pairs)) or (j > 1 and (kw // j < 8 or tw * j > 4 * pairs)):
                continue
            cx, cw = max(-(-kx // i), 24) + 4 + 16 * (i > 1), max(-(-kw // j), 24) + 4 + 16 * (j > 1)
            more, n0, n1 = _deal(tx * i, cx, tw * j, cw, pairs)
            q = tx * i // pairs
            cost = max((q + 1) * cx + n0 * cw if more else 0, q * cx + n1 * cw)
            if cost < least * 0.97:
                least, best = cost, (i, j)
    return (piece, *best)


@pytest.mark.parametrize("dtype,rows,width,vocab,want", [
    ("bf16", 16384, 320, 19001, (8192, 1, 1)), ("f16", 12288, 768, 19001, (10752, 1, 1)), ("f32", 8192, 320, 19001, (8192, 1, 1)),
    ("bf16", 18944, 512, 13001, (6912, 1, 4))])
def test_pieces_whose_sums_stay_whole(nb, torch, dtype, rows, width, vocab, want):
    """Several pieces of the vocabulary, the last one short, several column tiles, w read where it
    stands (16 bits), and no piece of K for dx: its sums wait in one buffer and leave with the
    last piece, as those of a large training batch do."""
    assert _cuts(dtype, rows, width, vocab) == want and width % 64 == 0 and rows >= 1024
    c = Case(torch, rows, width, vocab, dtype, ignored=0.05, seed=70)
    assert c.w.data_ptr() % 128 == 0
    loss, stats = c.forward(nb)
    c.check_forward(loss, stats)
    torch.cuda.empty_cache()
    dx, dw = c.backward(nb, stats, 1 / rows)
    c.check_backward(stats, 1 / rows, dx, dw)
    base = torch.randn(vocab, width, device="cuda") / rows
    torch.cuda.empty_cache()
    dx, dw = c.backward(nb, stats, 1 / rows, dw_dtype="f32", dw=base.clone())
    c.check_backward(stats, 1 / rows, dx, dw, base)
    torch.cuda.empty_cache()
