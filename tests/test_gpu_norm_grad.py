"""The gradients of layer norm and RMSNorm (include/noetic/head.h) in every kernel
that makes them, against the definition in 64 bits.

Which kernel a call takes depends on its width and on where the rows of x, dy and
dx start: `path` restates that rule, and a test without a GPU holds the shapes
here to reach every one.

Tolerances count roundings, U = 2^-24 being half a step of f32.
 - h = (x - mean) rstd: two roundings.  c = dy gain: one.
 - A row's mean of n terms: a term passes through at most n / 256 + 48 additions, then
   one product with 1 / n, itself rounded.
 - A sum over rows: rows that share a chain are at most rows / 32 (the fewest chains
   are those of 32 clusters; rows that a block's groups share, and the 64 parts of the
   kernels for wider rows, are more); joining the chains takes at most 8 additions in a
   block, 296 / 16 over the partial rows and 16 at the end, and one for what was there.
 - A result of a narrower type is off by half a step more.
"""

import ctypes as C
import math

import pytest

from test_gpu_head import _matrix, _norm, _norm_grad, _out_tol, torch  # noqa: F401  (torch: the fixture)

U = 2.0**-24
SIZE = {"f32": 4, "f16": 2, "bf16": 2}

# Rows and widths.  Up to 8192 columns a group of 32 to 512 threads takes a row, several
# rows in turn: two turns and a part of a third at least.
GROUP = [(5003, 24), (5003, 41), (5003, 104), (5003, 200), (5001, 201), (4900, 504), (4803, 501), (2600, 704), (2601, 701),
         (2500, 1000), (2501, 1001), (1300, 1400), (1301, 1401), (1203, 2000), (1302, 2001), (700, 2800), (701, 2803), (650, 4000),
         (655, 4001), (400, 7000), (331, 7001), (310, 8192), (7, 1), (3, 5), (1, 1000), (1, 777), (9, 8185)]
# A cluster of three to eight CTAs, in several turns; one row, and one to a cluster.
CLUSTER = [(401, 8200), (380, 12288), (301, 16384), (300, 20000), (233, 24000), (131, 28000), (130, 32768), (1, 9000), (30, 32000)]
WIDE = [(70, 33000), (3, 65536), (130, 40000)]
ODD_WIDE = [(130, 8201), (67, 9001), (3, 33001)]
SHAPES = GROUP + CLUSTER + WIDE + ODD_WIDE
# Where the rows of (x, dy, dx) start: strides beyond the width, and elements before the
# first row.  "alike": the same everywhere; "padded": strides that keep the rows'
# places of a 16-byte unit; "dx apart": dx at other places; "dy apart".
LAYOUTS = {"alike": lambda n: ((0, 0), (0, 0), (0, 0)), "padded": lambda n: ((1, 3), (1 + n, 3), (1 + 2 * n, 3)),
           "dx apart": lambda n: ((0, 0), (0, 0), (3, 1)), "dy apart": lambda n: ((0, 0), (1, 0), (0, 0))}


def path(size, width, x, dy, dx):
    """The kernel of a gradient whose arrays are given as (stride, element of the first row)."""
    n = 16 // size
    like = (x[0] - dy[0]) % n == 0 and (x[1] - dy[1]) % n == 0
    same = dx is None or ((x[0] - dx[0]) % n == 0 and (x[1] - dx[1]) % n == 0)
    whole = like and same and width % n == 0 and x[0] % n == 0 and x[1] % n == 0
    edge_units = (width + 2 * (n - 1)) // n

    def group(units):
        loads = 16 // n
        for threads in (32, 64, 128, 256):
            if threads == 32:
                if units <= 32:
                    return 32, 1
                if 2 < loads and units <= 64:
                    return 32, 2
            elif loads > 3 and units <= threads * 3:
                return threads, 3
            if units <= threads * loads:
                return threads, loads
        return 512, loads

    if whole and width // n <= 512 * 16 // n:
        return ("group", *group(width // n))
    if like and edge_units <= 512 * 16 // n:
        return ("odd group", *group(edge_units), "in place" if same else "staged")
    if whole and width // n <= 8 * 256 * 16 // n:
        return ("cluster", math.ceil(width / 4096))
    return ("wide", "vectors" if whole else "elements")


def _layout(dtype, width, name):
    places = LAYOUTS[name](16 // SIZE[dtype])
    return [(width + pad, shift) for pad, shift in places]


def test_the_shapes_reach_every_kernel():
    reached = {s: {path(s, w, *_layout(t, w, name)) for _, w in SHAPES for name in LAYOUTS} for t, s in (("f32", 4), ("bf16", 2))}
    loads = {4: {32: (1, 2, 4), 64: (3, 4), 128: (3, 4), 256: (3, 4), 512: (4,)}, 2: {32: (1, 2), 64: (2,), 128: (2,), 256: (2,), 512: (2,)}}
    for size, groups in loads.items():
        want = {("cluster", n) for n in range(3, 9)} | {("wide", "vectors"), ("wide", "elements")}
        for threads, ls in groups.items():
            for n in ls:
                want |= {("group", threads, n), ("odd group", threads, n, "in place"), ("odd group", threads, n, "staged")}
        assert reached[size] == want


def _reference(torch, x, dy, gain, mean, rstd):
    """(dx, its bound, dgain, its bound, dbias, its bound) from the given statistics."""
    rows, d = x.shape
    g, r = dy.double(), rstd.double()[:, None]
    off = x.double() - (0.0 if mean is None else mean.double()[:, None])
    hh, c = off * r, g * gain
    h_tol = 3 * U * hh.abs()
    n_add = (d / 256 + 48) * U
    mc, a_c = (0.0, 0.0) if mean is None else (c.mean(-1, keepdim=True), c.abs().mean(-1, keepdim=True))
    mch, a_ch = (c * hh).mean(-1, keepdim=True), (c * hh).abs().mean(-1, keepdim=True)
    dx = r * (c - mc - hh * mch)
    # c; the two means; the product with h, whose own error counts; the last product.
    tol = r * (2 * U * c.abs() + (n_add + 4 * U) * a_c + hh.abs() * (n_add + 6 * U) * a_ch + (h_tol + 2 * U * hh.abs()) * mch.abs()) + 3 * U * dx.abs()
    adds = (rows / 32 + 64) * U
    terms = g * hh
    return (dx, tol, terms.sum(0), (adds + 4 * U) * terms.abs().sum(0), g.sum(0), adds * g.abs().sum(0))


@pytest.mark.gpu
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("rows,d", SHAPES)
def test_gradient_in_every_kernel(gpu, torch, rows, d, layout, dtype, rms):
    n = 16 // SIZE[dtype]
    (xp, xs), (yp, ys), (op, os_) = LAYOUTS[layout](n)
    x, _ = _matrix(torch, rows, d, dtype, xp, xs, scale=1.5, seed=d, offset=0.7)
    dy, _ = _matrix(torch, rows, d, dtype, yp, ys, scale=0.5, seed=d + 1, offset=0.1)
    out, around = _matrix(torch, rows, d, dtype, op, os_, seed=d + 2)
    g = torch.Generator(device="cuda").manual_seed(d + rows)
    gain = 1 + 0.3 * torch.randn(d, generator=g, device="cuda")
    _, mean, rstd = _norm(gpu, torch, x, gain, None, 1e-5, rms, dtype)
    ref, tol, rg, gtol, rb, btol = _reference(torch, x, dy, gain, mean, rstd)
    tol = tol + _out_tol(torch, dtype, ref)

    def close(dx, dg, db, before=0.0, dx_ref=ref, dx_tol=tol):
        if dx is not None:
            assert ((dx.double() - dx_ref).abs() <= dx_tol).all()
        for got, want, bound in ((dg, rg, gtol), (db, rb, btol)):
            if got is not None:
                assert ((got.double() - before - want).abs() <= bound + U * (want + before).abs()).all()

    first = _norm_grad(gpu, torch, x, dy, gain, mean, rstd, dtype, dx=out)
    close(*first)
    assert (first[2] is None) == rms
    gaps = torch.ones(around.numel(), dtype=torch.bool, device="cuda")
    gaps[os_:os_ + rows * (d + op)].view(rows, -1)[:, :d] = False
    assert torch.isnan(around[gaps]).all()
    # The same call gives the same bits.
    kept = [None if v is None else v.clone() for v in first]
    again = _norm_grad(gpu, torch, x, dy, gain, mean, rstd, dtype, dx=out)
    assert all(a is None or torch.equal(a, b) for a, b in zip(kept, again))
    # dx alone, the sums alone (added to what is there), one of them alone, no gain, dx on dy.
    close(*_norm_grad(gpu, torch, x, dy, gain, mean, rstd, dtype, dx=out, dgain=False, dbias=False))
    before = torch.randn(d, generator=g, device="cuda")
    close(*_norm_grad(gpu, torch, x, dy, gain, mean, rstd, dtype, dx=None, accumulate=1, before=before), before=before.double())
    if not rms:
        close(*_norm_grad(gpu, torch, x, dy, gain, mean, rstd, dtype, dx=None, dgain=False))
    plain, ptol, *_ = _reference(torch, x, dy, torch.ones_like(gain), mean, rstd)
    close(*_norm_grad(gpu, torch, x, dy, None, mean, rstd, dtype, dx=out), dx_ref=plain, dx_tol=ptol + _out_tol(torch, dtype, plain))
    close(*_norm_grad(gpu, torch, x, dy, gain, mean, rstd, dtype, dx=dy))


@pytest.mark.gpu
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("rows,d,layout", [(40, 104, "alike"), (9, 1001, "alike"), (9, 1001, "dx apart"), (5, 7000, "alike"),
                                           (5, 12288, "alike"), (3, 33000, "alike"), (5, 777, "dy apart")])
def test_gradient_along_a_direction_against_differences(gpu, torch, rows, d, layout, rms):
    (xp, xs), (yp, ys), (op, os_) = LAYOUTS[layout](4)
    x, _ = _matrix(torch, rows, d, "f32", xp, xs, scale=1.5, seed=d, offset=0.7)
    dy, _ = _matrix(torch, rows, d, "f32", yp, ys, scale=0.5, seed=d + 1)
    out, _ = _matrix(torch, rows, d, "f32", op, os_)
    g = torch.Generator(device="cuda").manual_seed(d)
    gain = 1 + 0.3 * torch.randn(d, generator=g, device="cuda")
    _, mean, rstd = _norm(gpu, torch, x, gain, None, 1e-5, rms, "f32")
    dx, dg, db = _norm_grad(gpu, torch, x, dy, gain, mean, rstd, "f32", dx=out)
    v, vg, vb = (torch.randn(*s, generator=g, device="cuda", dtype=torch.float64) for s in ((rows, d), (d,), (d,)))

    def f(t):
        xx, gg = x.double() + t * v, gain.double() + t * vg
        mu = 0.0 if rms else xx.mean(-1, keepdim=True)
        y = (xx - mu) * torch.rsqrt((xx - mu).square().mean(-1, keepdim=True) + 1e-5) * gg
        return (dy.double() * (y if rms else y + t * vb)).sum()

    # h^2 = 1e-8 of a third derivative of the terms' own size; the statistics that the call is given are f32,
    # off by up to d / 256 + 60 roundings as its own sums are.
    h = 1e-4
    num = (f(h) - f(-h)) / (2 * h)
    terms = (dx.double() * v).abs().sum() + (dg.double() * vg).abs().sum() + (0.0 if rms else (db.double() * vb).abs().sum())
    got = (dx.double() * v).sum() + (dg.double() * vg).sum() + (0.0 if rms else (db.double() * vb).sum())
    assert abs(num - got) <= (1e-6 + 4 * (d / 256 + 60) * U) * terms


def test_the_workspace_holds_one_row_per_block_and_no_more(nb):
    # 296 blocks, or for rows too wide for a cluster 64, of two f32 per column; never more than one per row.
    n = C.c_uint64()
    for rows in (0, 1, 63, 64, 65, 295, 296, 297, 1 << 20, 1 << 26):
        for width, most in ((1, 296), (100, 296), (8192, 296), (32768, 296), (32769, 64), (1 << 20, 64)):
            status = nb.lib().nk_layer_norm_backward_workspace(rows, width, C.byref(n))
            if rows * width > 1 << 37:  # beyond what a matrix may hold
                assert status == nb.NK_ERR_INVALID and n.value == 0
                continue
            assert status == 0 and n.value == min(max(rows, 1), most) * 2 * width * 4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("rows,d", [(5003, 104), (5003, 41), (1301, 1401), (700, 2800), (331, 7001), (310, 8192), (301, 16384),
                                    (130, 20000), (130, 32768), (70, 33000), (67, 9001)])
def test_a_broken_row_stays_alone(gpu, torch, rows, d, layout, dtype):
    # NaN and infinities in some rows: all other rows, and the parameters' sums that do not see
    # them, have the bits that they have without.
    (xp, xs), (yp, ys), (op, os_) = LAYOUTS[layout](16 // SIZE[dtype])
    x, _ = _matrix(torch, rows, d, dtype, xp, xs, scale=1.5, seed=d, offset=0.7)
    dy, _ = _matrix(torch, rows, d, dtype, yp, ys, scale=0.5, seed=d + 1)
    out, _ = _matrix(torch, rows, d, dtype, op, os_)
    gain = torch.linspace(0.5, 1.5, d, device="cuda")
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bad[[0, 1, rows // 2, rows - 1]] = True
    c = d // 3
    for rms in (False, True):
        y, mean, rstd = _norm(gpu, torch, x, gain, None, 1e-5, rms, dtype, out)
        y = y.clone()
        dx, dg, db = _norm_grad(gpu, torch, x, dy, gain, mean, rstd, dtype, dx=out)
        dx = dx.clone()
        kept = x[bad].clone()
        x[0, c], x[1, d - 1], x[rows // 2, 0], x[rows - 1, c] = float("nan"), float("inf"), -float("inf"), float("nan")
        y2, mean2, rstd2 = _norm(gpu, torch, x, gain, None, 1e-5, rms, dtype, out)
        assert torch.equal(y2[~bad], y[~bad]) and torch.equal(rstd2[~bad], rstd[~bad])
        assert torch.isnan(y2[[0, rows - 1]]).all() and not torch.isfinite(y2[1, d - 1]) and not torch.isfinite(y2[rows // 2, 0])
        x[bad] = kept
        kept = dy[bad].clone()
        dy[bad, c] = float("nan")
        dx2, dg2, db2 = _norm_grad(gpu, torch, x, dy, gain, mean, rstd, dtype, dx=out)
        assert torch.equal(dx2[~bad], dx[~bad]) and torch.isnan(dx2[bad]).all()
        others = torch.arange(d, device="cuda") != c
        for a, b in ((dg, dg2), (db, db2)):
            assert a is None or (torch.equal(a[others], b[others]) and torch.isnan(b[c]))
        dy[bad] = kept
