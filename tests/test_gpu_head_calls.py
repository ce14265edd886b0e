"""Calls of include/noetic/head.h that the operators' own tests do not make: two
host threads at once, sums over many rows, logits at the end of f32's range,
special rows in every kernel, texts longer than a block of logits, streams and
graphs side by side."""

import ctypes as C
import threading

import numpy as np
import pytest

from test_gpu_head import (CODE, INF, NAN, NONE, U, _check_logprobs, _distill, _dt, _grad, _logprobs, _matrix, _norm,  # noqa: F401
                           _norm_grad, _out_tol, _p, _ref_distill, _ref_grad, _span, _sum_rel, torch)  # (torch: the fixture)

pytestmark = pytest.mark.gpu


def _both(gpu, torch, calls, times=4000):
    """Each call by a host thread of its own on a stream of its own, again and
    again; returns the messages of those that failed."""
    torch.cuda.synchronize()
    failed, start = [], threading.Barrier(len(calls))

    def work(call):
        st = torch.cuda.Stream()
        s = C.c_void_p(st.cuda_stream)
        start.wait()
        for _ in range(times):
            if call(s) != 0:
                failed.append(gpu.lib().nk_last_error())
        st.synchronize()

    threads = [threading.Thread(target=work, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return failed


# Pairs of calls of one kernel that take different amounts of shared memory, both
# more than every kernel may have: neither makes the other fail.
def test_two_threads_with_teachers_of_other_lengths(gpu, torch):
    L, R, V = gpu.lib(), 512, 4096
    z, _ = _matrix(torch, R, V, "f32", seed=1)
    z = z.contiguous()

    def call(K):
        ids = torch.arange(K, device="cuda", dtype=torch.int32).repeat(R, 1).contiguous()
        t = torch.zeros(R, K, device="cuda")
        dz = torch.empty_like(z)
        return lambda s: L.nk_distill_device(_p(z), 0, R, V, V, _p(ids), _p(t), 0, K, 1.0, None, None, 1.0, _p(dz), V, s)

    assert _both(gpu, torch, [call(1), call(64)]) == []


def test_two_threads_with_other_numbers_of_alternatives(gpu, torch):
    L, R, V = gpu.lib(), 512, 300
    z, _ = _matrix(torch, R, V, "f32", seed=1)
    z = z.contiguous()

    def call(top):
        ids = torch.empty(R, top, device="cuda", dtype=torch.int32)
        return lambda s: L.nk_token_logprobs_device(_p(z), 0, R, V, V, None, 1.0, top, None, None, None, _p(ids), None, s)

    assert _both(gpu, torch, [call(110), call(128)]) == []


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_two_threads_with_norms_into_other_layouts(gpu, torch, dtype):
    L, R, d = gpu.lib(), 9000, 767 if dtype == "f32" else 1001
    x, _ = _matrix(torch, R, d, dtype, seed=1)
    code, gain = CODE[dtype], torch.ones(d, device="cuda")
    _, mean, rstd = _norm(gpu, torch, x, gain, None, 1e-5, False, dtype)

    def forward(out):
        return lambda s: L.nk_layer_norm_device(_p(x), code, R, d, d, _p(gain), None, 1e-5, 0, _p(out), out.stride(0), None, None, s)

    def backward(out):
        return lambda s: L.nk_layer_norm_backward_device(_p(x), code, R, d, d, _p(gain), _p(mean), _p(rstd), 0, _p(x), d, _p(out),
                                                         out.stride(0), None, None, 0, None, 0, s)

    for call in (forward, backward):
        alike, other = (_matrix(torch, R, d, dtype, shift=k)[0] for k in (0, 1))
        assert _both(gpu, torch, [call(alike), call(other)]) == []


def test_norm_gradient_sums_over_a_million_rows(gpu, torch):
    # Rows of dy that start elsewhere than those of x.  A term passes through 64 additions, one for
    # each 4096 rows, four over the partial rows of a lane, 16 at the end.  Column 0 is a constant
    # of 1023.499 steps of the binade that a sum over every 64th row ends in: added one by one, half of
    # these additions would round down by half a step, 4000 U in all.
    rows, d = 2**20 + 37, 8
    x, _ = _matrix(torch, rows, d, "f32", seed=1)
    dy, _ = _matrix(torch, rows, d, "f32", pad=1, seed=2, offset=1.0)
    dy[:, 0] = 1023.499 * 2.0**-13
    gain = torch.ones(d, device="cuda")
    _, mean, rstd = _norm(gpu, torch, x, gain, None, 1e-5, False, "f32")
    dx, dg, db = _norm_grad(gpu, torch, x, dy, gain, mean, rstd, "f32")
    hh = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    adds = (64 + rows / 4096 + 4 + 16) * U
    g = dy.double()
    assert ((db - g.sum(0)).abs() <= adds * g.abs().sum(0)).all()
    assert ((dg - (g * hh).sum(0)).abs() <= (adds + 3 * U) * (g * hh).abs().sum(0)).all()


@pytest.mark.parametrize("rows,V", [(4, 300), (600, 300), (3, 60000), (2000, 9000)])
@pytest.mark.parametrize("T", [1.0, 0.5, 0.03])
def test_distillation_of_a_student_masked_by_the_lowest_value(gpu, torch, rows, V, T):
    # (z - m) / T is beyond f32's range where the teacher wants what the student's mask forbids and T is below 1;
    # T^2 times it is not.
    low = torch.finfo(torch.float32).min
    z, _ = _matrix(torch, rows, V, "f32", seed=V)
    z[:, 40:80] = low
    z[:, V - 3:] = low
    ids = torch.tensor([7, 50, V - 1, 79, 20], device="cuda", dtype=torch.int32).repeat(rows, 1)
    ids[::2, 1:4] = torch.tensor([8, 9, 10], device="cuda", dtype=torch.int32)
    g = torch.Generator(device="cuda").manual_seed(rows)
    t = torch.randn(rows, 5, generator=g, device="cuda") * T
    ref, tol, rdz, ztol = _ref_distill(torch, z, ids, t, T, None, 1.0)
    for grad in (True, False):
        loss, dz = _distill(gpu, torch, z, ids, t, T, None, 1.0, "f32", "f32", grad=grad)
        assert torch.isfinite(loss).all() and (loss[1::2] > 1e30).all()
        assert ((loss.double() - ref).abs() <= tol).all()
        if grad:
            assert ((dz.double() - rdz).abs() <= ztol + _out_tol(torch, "f32", rdz)).all()


def test_scores_in_several_blocks_of_logits(gpu):
    # A vocabulary of which a block of logits (512 MiB) holds fewer rows than the texts have, so
    # that a block ends inside a text: every position against the logits of the loss call in 64 bits.
    V, batch, t, top = 300007, 3, 210, 4
    block = (512 << 20) // (4 * V)
    assert block < batch * t and block % t != 0
    gm = gpu.Model.new(gpu.LmConfig(vocab=V, d_model=16, n_layer=2, expand=2, conv_k=3, mlp_mult=2, eps=1e-5, tau_max=8.0), 4, device=0)
    rng = np.random.default_rng(3)
    ids = rng.integers(0, V, batch * t).astype(np.uint32)
    tg = np.roll(ids, -1)
    tg[::11] = 0xFFFFFFFF
    out = gm.score(ids, tg, batch, t, top)
    _, lg = gm.loss(ids, tg, batch, t, want_logits=True)
    rel = _sum_rel(V, _span(V))
    for r in range(batch * t):
        lp, ent, ti, tl = (out[k].reshape(batch * t, -1)[r] for k in ("logprob", "entropy", "top_ids", "top_logprobs"))
        if tg[r] == 0xFFFFFFFF:
            assert lp == 0 and ent == 0 and (ti == 0xFFFFFFFF).all() and np.isneginf(tl).all()
            continue
        z = lg[r].astype(np.float64)
        p = z - z.max() - np.log(np.exp(z - z.max()).sum())
        best = np.argsort(-lg[r], kind="stable")[:top]
        assert np.array_equal(ti, best.astype(np.uint32))
        assert abs(lp[0] - p[tg[r]]) <= rel + 16 * U * abs(p[tg[r]]) and (abs(tl - p[best]) <= rel + 16 * U * abs(p[best])).all()
        assert abs(ent[0] + (np.exp(p) * p).sum()) <= (rel + 8 * U) * (2 + 2 * np.log(V))
    # Alternatives asked for and not taken: the same scores.
    lp = np.empty(batch * t, np.float32)
    as_p = lambda a: a.ctypes.data_as(C.c_void_p)  # noqa: E731
    gpu._check(gpu.lib().nk_model_score(gm.h, as_p(ids), as_p(tg), batch, t, top, as_p(lp), None, None, None))
    assert np.array_equal(lp, out["logprob"].reshape(-1))


# Rows, vocabulary: one block or cluster to a row, a warp, blocks of 128 and of 256 threads, clusters.
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,V", [(9, 1000), (603, 1000), (603, 1003), (720, 40000), (1260, 70001), (5, 130000), (513, 9)])
def test_special_rows_in_every_kernel_of_the_log_probabilities(gpu, torch, dtype, rows, V):
    low, half = torch.finfo(_dt(torch, dtype)).min, V // 2
    z, _ = _matrix(torch, rows, V, dtype, seed=V)
    z = z.contiguous()
    t = torch.randint(0, half, (rows,), device="cuda", dtype=torch.int32, generator=torch.Generator(device="cuda").manual_seed(V))
    kind = torch.arange(rows, device="cuda") % 9
    rest = slice(half, V)
    z[kind == 0] = -INF                  # nothing left
    z[kind == 1] = low                   # the lowest value alone: uniform
    z[kind == 2, rest] = low
    z[kind == 3, rest] = -INF
    z[kind == 4, half - 1] = NAN
    z[kind == 5, V - 1] = INF
    z[kind == 6] = -INF                  # one token left, at the end
    z[kind == 6, V - 1] = 1.0
    t[kind == 6] = V - 1
    z[kind == 7] = NAN                   # not read
    t[kind == 7] = NONE
    broken, plain = (kind == 4) | (kind == 5), (kind == 1) | (kind == 2) | (kind == 3) | (kind == 6) | (kind == 8)
    for T, top in ((1.0, 0), (1.0, 20), (0.3, 5), (40.0, 128)):
        out = _logprobs(gpu, torch, z, t, T, top, dtype)
        _check_logprobs(torch, {k: None if v is None else v[plain] for k, v in out.items()}, z[plain], t[plain], T, top)
        none, gone = kind == 0, kind == 7
        assert (out["logprob"][none] == -INF).all() and (out["entropy"][none] == 0).all() and (out["stats"][none] == -INF).all()
        assert torch.isnan(out["logprob"][broken]).all() and torch.isnan(out["entropy"][broken]).all()
        for k in ("logprob", "entropy", "stats"):
            assert (out[k][gone] == 0).all()
        assert (out["logprob"][kind == 6] == 0).all() and (out["entropy"][kind == 6] == 0).all()
        if top:
            assert (out["top_ids"][none | gone] == NONE).all() and (out["top_logprobs"][none | gone] == -INF).all()
            assert (out["top_ids"][kind == 4] != half - 1).all() and (out["top_ids"][kind == 5, 0] == V - 1).all()
        gl = torch.ones(rows, device="cuda")
        fw = out if T != 40.0 else _logprobs(gpu, torch, z, t, T, 0, dtype)
        dz = _grad(gpu, torch, z, t, T, fw["stats"], fw["entropy"], gl, 0.5 * gl, dtype)
        assert (dz[none | gone] == 0).all() and torch.isnan(dz[broken]).all()
        ref, tol = _ref_grad(torch, z[plain], t[plain], T, fw["stats"][plain], fw["entropy"][plain], gl[plain], 0.5 * gl[plain])
        # A probability below 2^-126 counts as 0: at most that is lost, times |g_logprob| + |g_entropy| (|log p| + H),
        # log p = -126 log 2 there (the logarithm of a smaller one grows slower than it falls), over T.
        lost = 2.0**-126 * (1 + 0.5 * (126 * np.log(2) + np.log(V))) / T
        assert ((dz[plain].double() - ref).abs() <= tol + lost + _out_tol(torch, dtype, ref)).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,V", [(8, 500), (1003, 500), (1003, 1001), (5, 130000), (700, 30000), (130, 200001), (515, 9)])
def test_special_rows_in_every_kernel_of_the_distillation(gpu, torch, dtype, rows, V):
    z, _ = _matrix(torch, rows, V, dtype, seed=V)
    z = z.contiguous()
    kind = torch.arange(rows, device="cuda") % 8
    ids = torch.tensor([0, V // 2, V - 1, V // 2, 2], device="cuda", dtype=torch.int32).repeat(rows, 1)  # one of them twice
    t = torch.randn(rows, 5, device="cuda", generator=torch.Generator(device="cuda").manual_seed(V))
    w = torch.ones(rows, device="cuda")
    z[kind == 0] = NAN                   # no entries: not read
    ids[kind == 0] = NONE
    z[kind == 1, 3:V // 2] = -INF        # masked where no entry is
    z[kind == 2, V - 2] = NAN
    t[kind == 3] = -INF                  # no entries either
    z[kind == 4] = NAN                   # weight 0
    w[kind == 4] = 0.0
    z[kind == 5, V - 1] = -INF           # the teacher wants what the student cannot say
    z[kind == 6] = -INF                  # a student that can say nothing
    t[kind == 7, 0] = torch.finfo(torch.float32).min
    for T in (1.0, 2.5):
        loss, dz = _distill(gpu, torch, z, ids, t, T, w, 0.7, dtype, "f32")
        alone = _distill(gpu, torch, z, ids, t, T, w, 0.7, dtype, "f32", grad=False)[0]
        ref, tol, rdz, ztol = _ref_distill(torch, z, ids, t, T, w, 0.7)
        plain = (kind == 1) | (kind == 7)
        for got in (loss, alone):
            assert ((got[plain].double() - ref[plain]).abs() <= tol[plain]).all()
            assert (got[(kind == 0) | (kind == 3)] == 0).all()
            assert torch.isnan(got[(kind == 2) | (kind == 4)]).all()
            assert (got[(kind == 5) | (kind == 6)] == INF).all()
        right = plain | (kind == 5)
        assert ((dz[right].double() - rdz[right]).abs() <= ztol[right] + _out_tol(torch, dtype, rdz[right])).all()
        assert (dz[(kind == 0) | (kind == 3) | (kind == 4) | (kind == 6)] == 0).all() and torch.isnan(dz[kind == 2]).all()


def _mixed_calls(gpu, torch, seed):
    """Calls of the kernels of short, long and wide rows on buffers of their own: (a function of the
    stream, its outputs) each."""
    L, g = gpu.lib(), torch.Generator(device="cuda").manual_seed(seed)
    keep = []

    def rn(*n, dtype="f32"):
        keep.append(torch.randn(*n, generator=g, device="cuda").to(_dt(torch, dtype)))
        return keep[-1]

    def out(*n, dtype=None):
        keep.append(torch.zeros(*n, device="cuda", dtype=dtype or torch.float32))
        return keep[-1]

    def ids(*n, V):
        keep.append(torch.randint(0, V, n, generator=g, device="cuda", dtype=torch.int32))
        return keep[-1]

    calls = []
    for R, V, dtype, top in ((700, 1024, "f32", 128), (5, 130000, "bf16", 20), (700, 40000, "f16", 7)):
        z, t, lp, ti = 3 * rn(R, V, dtype=dtype), ids(R, V=V), out(R), out(R, top, dtype=torch.int32)
        keep.append(z)
        calls.append((lambda s, z=z, t=t, lp=lp, ti=ti, R=R, V=V, top=top, c=CODE[dtype]: L.nk_token_logprobs_device(
            _p(z), c, R, V, V, _p(t), 1.0, top, _p(lp), None, None, _p(ti), None, s), (lp, ti)))
    for R, V, dtype, K in ((600, 4000, "f32", 40), (300, 70000, "bf16", 33), (3, 131072, "f16", 200)):
        z, i, q, ls, dz = rn(R, V, dtype=dtype), ids(R, K, V=V), rn(R, K), out(R), out(R, V, dtype=_dt(torch, dtype))
        calls.append((lambda s, z=z, i=i, q=q, ls=ls, dz=dz, R=R, V=V, K=K, c=CODE[dtype]: L.nk_distill_device(
            _p(z), c, R, V, V, _p(i), _p(q), 0, K, 2.0, _p(ls), None, 1.0, _p(dz), V, s), (ls, dz)))
    for R, d, dtype in ((700, 1001, "bf16"), (200, 20000, "f32"), (300, 16384, "bf16"), (70, 33001, "f16"), (900, 104, "f16")):
        x, dy, gain = rn(R, d, dtype=dtype), rn(R, d, dtype=dtype), rn(d)
        y, dx = (out(R * d + 1, dtype=_dt(torch, dtype))[1:] for _ in range(2))
        mean, rstd, dg, db = out(R), out(R), out(d), out(d)
        n = C.c_uint64()
        gpu._check(L.nk_layer_norm_backward_workspace(R, d, C.byref(n)))
        ws = out(n.value // 4)

        def both(s, x=x, dy=dy, gain=gain, y=y, dx=dx, mean=mean, rstd=rstd, dg=dg, db=db, ws=ws, n=n.value, R=R, d=d, c=CODE[dtype]):
            return L.nk_layer_norm_device(_p(x), c, R, d, d, _p(gain), None, 1e-5, 0, _p(y), d, _p(mean), _p(rstd), s) or \
                L.nk_layer_norm_backward_device(_p(x), c, R, d, d, _p(gain), _p(mean), _p(rstd), 0, _p(dy), d, _p(dx), d, _p(dg),
                                                _p(db), 0, _p(ws), n, s)

        calls.append((both, (y, dx, mean, rstd, dg, db)))
    return calls, keep


def test_large_calls_on_two_streams_and_in_graphs(gpu, torch):
    sets = [_mixed_calls(gpu, torch, k) for k in (1, 2)]

    def run(calls):
        s = C.c_void_p(torch.cuda.current_stream().cuda_stream)
        for f, _ in calls:
            assert f(s) == 0, gpu.lib().nk_last_error()

    want = []
    for calls, _ in sets:
        run(calls)
        torch.cuda.synchronize()
        want.append([o.clone() for _, outs in calls for o in outs])

    def clear():
        torch.cuda.synchronize()
        for calls, _ in sets:
            for _, outs in calls:
                for o in outs:
                    o.zero_()
        torch.cuda.synchronize()

    def same():
        torch.cuda.synchronize()
        return all(torch.equal(a, b) for (calls, _), w in zip(sets, want) for a, b in zip((o for _, outs in calls for o in outs), w))

    streams = [torch.cuda.Stream() for _ in sets]
    clear()
    for _ in range(3):
        for (calls, _), st in zip(sets, streams):
            with torch.cuda.stream(st):
                run(calls)
    assert same()
    graphs = []
    for calls, _ in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(calls)
        graphs.append(g)
    clear()
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    assert same()
    del graphs
