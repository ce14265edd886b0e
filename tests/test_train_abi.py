"""The operators at a training step's end (include/noetic/train.h) on CPU: the
header, the library and the Python mirror declare the same calls, and every bad
argument is refused with a status before any device work."""

import ctypes as C
import os
import re

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def buf():
    """Host memory to point at: no call below gets as far as reading it."""
    return C.create_string_buffer(1 << 14)


def _header():
    text = open(os.path.join(ROOT, "include", "noetic", "train.h")).read()
    return re.sub(r"/\*.*?\*/", "", text, flags=re.S)


def test_header_library_and_mirror_agree(nb):
    text = _header()
    names = set(re.findall(r"^(?:nk_status|void)\s+(nk_\w+)\s*\(", text, flags=re.M))
    assert names == set(nb.train.SIGNATURES)
    assert all(hasattr(C.CDLL(nb.LIB_PATH), n) for n in names)
    assert not names & set(nb.SIGNATURES) and not names & set(nb.head.SIGNATURES)
    for n in names:
        args = re.search(r"\b%s\s*\((.*?)\);" % n, text, flags=re.S).group(1)
        assert len(args.split(",")) == len(nb.train.SIGNATURES[n][1]), n
    assert int(re.search(r"NK_ADAMW_BLOCK (\d+)u", text).group(1)) == nb.train.NK_ADAMW_BLOCK
    # The structure: its fields in order, and their sizes.
    body = re.search(r"typedef struct nk_adamw_tensor \{(.*?)\}", text, flags=re.S).group(1)
    fields = re.findall(r"(\w+)\s*(?=[,;])", body)
    assert fields == [f[0] for f in nb.train.NkAdamwTensor._fields_]
    assert C.sizeof(nb.train.NkAdamwTensor) == 8 * 8 + 4 * 4


# Arguments of a call that would be taken, by name; p is some address.
def _calls(p):
    p = (p + 255) // 256 * 256
    return {
        "nk_linear_ce_device": dict(x=p, dtype=0, rows=2, width=8, x_stride=8, w=p + 256, vocab=4, w_stride=8,
                                    targets=p + 512, loss=p + 768, stats=p + 1024, workspace=p + 4096,
                                    workspace_bytes=1 << 30, stream=None),
        "nk_linear_ce_backward_device": dict(x=p, dtype=2, rows=2, width=8, x_stride=8, w=p + 256, vocab=4, w_stride=8,
                                             targets=p + 512, stats=p + 768, row_weight=p + 1024, grad_scale=1.0,
                                             dx=p + 1280, dx_stride=8, dw=p + 1536, dw_dtype=2, dw_stride=8,
                                             accumulate=0, workspace=p + 4096, workspace_bytes=1 << 30, stream=None),
    }


COMMON = [dict(x=None), dict(w=None), dict(targets=None), dict(dtype=3), dict(dtype=-1), dict(width=0), dict(vocab=0),
          dict(x_stride=7), dict(w_stride=7), dict(rows=(1 << 26) + 1), dict(vocab=(1 << 26) + 1),
          dict(width=(1 << 24) + 1, x_stride=1 << 25, w_stride=1 << 25), dict(rows=1 << 20, vocab=1 << 20),
          dict(x_stride=1 << 62), dict(w_stride=1 << 62), dict(x="+1"), dict(w="+1"), dict(targets="+2"),
          dict(workspace=None), dict(workspace="+128"), dict(workspace_bytes=0), dict(stats="+2")]
REFUSALS = {
    "nk_linear_ce_device": COMMON + [
        dict(loss=None, stats=None), dict(loss="+2"), dict(stats="-1024"), dict(loss="-768"), dict(loss="-512"),
        dict(stats="-252"), dict(workspace="-4096")],
    "nk_linear_ce_backward_device": COMMON + [
        dict(stats=None), dict(grad_scale=NAN), dict(grad_scale=INF), dict(dx=None, dw=None), dict(dx_stride=7),
        dict(dw_stride=7), dict(dx="+1"), dict(dw="+1"), dict(dw_dtype=1), dict(dw_dtype=3), dict(dw="-256"),
        dict(dx="-1280"), dict(dw="-1264"), dict(dx="-1024"), dict(row_weight="+1"), dict(workspace="-4096")],
}


def _call(nb, name, args):
    return getattr(nb.lib(), name)(*[v for v in args.values()])


@pytest.mark.parametrize("name,i", [(n, i) for n in REFUSALS for i in range(len(REFUSALS[n]))])
def test_refusals(nb, buf, name, i):
    args = dict(_calls(C.addressof(buf))[name])
    for k, v in REFUSALS[name][i].items():
        args[k] = args[k] + int(v) if isinstance(v, str) else v
    st = _call(nb, name, args)
    assert st == nb.NK_ERR_INVALID, (REFUSALS[name][i], st)
    msg = nb.lib().nk_last_error().decode()
    assert msg.startswith(name.replace("_device", "")) and len(msg) > len(name) and "cuda" not in msg.lower(), msg


def test_no_rows_is_no_work(nb, buf):
    c = _calls(C.addressof(buf))
    for name, args in c.items():
        args.update(rows=0, x=None, targets=None, stats=None, workspace=None)
        if "backward" in name:
            args.update(accumulate=1, row_weight=None)
        assert _call(nb, name, args) == nb.NK_OK, nb.lib().nk_last_error()


def test_workspace(nb):
    f, n = nb.lib().nk_linear_ce_workspace, C.c_uint64()
    assert f(2, 100, 64, 1000, 256, 64, 0, None) == nb.NK_ERR_INVALID
    for bad in [(3, 100, 64, 1000, 256, 64), (2, 1 << 27, 64, 1000, 256, 64), (2, 100, 0, 1000, 256, 64),
                (2, 100, 64, 0, 256, 64), (2, 100, 64, 1000, None, 64), (2, 100, 64, 1000, 256, 63)]:
        n.value = 7
        assert f(*bad, 1, C.byref(n)) == nb.NK_ERR_INVALID and n.value == 0
    for dtype in range(3):
        for rows, width, vocab in [(0, 1, 1), (1, 1, 1), (1000, 64, 1000), (8192, 1024, 32768), (1 << 20, 64, 1 << 16)]:
            for back in (0, 1):
                a = nb.train.linear_ce_workspace(dtype, rows, width, vocab, backward=back)
                odd = nb.train.linear_ce_workspace(dtype, rows, width, vocab, w=258 if dtype else 260, backward=back)
                assert a <= odd
                # Far from the logits of a large call.
                assert rows * vocab < 1 << 34 or a < rows * vocab


def _tensor(nb, p, **kw):
    args = dict(val=p, grad=p + 1024, m=p + 2048, v=p + 3072, m_scale=None, v_scale=None, copy=p + 4096, n=16, grad_dtype=0,
                copy_dtype=2, state_bits=32, decay=1)
    args.update(kw)
    return nb.train.NkAdamwTensor(*[args[f[0]] for f in nb.train.NkAdamwTensor._fields_])


def test_adamw_refusals(nb, buf):
    p = (C.addressof(buf) + 255) // 256 * 256
    L, h = nb.lib(), C.c_void_p()
    cfg = nb.NkAdamwCfg(1e-3, 0.9, 0.95, 1e-8, 0.0, 1, 1)

    def both(*tensors, count=None):
        t = (nb.train.NkAdamwTensor * max(1, len(tensors)))(*tensors)
        n = len(tensors) if count is None else count
        out = [L.nk_adamw_many_create(t, n, C.byref(h)), L.nk_adamw_many_step(t, n, C.byref(cfg), 1.0, 0.0, None, 0)]
        assert h.value is None
        assert out[0] == out[1]
        return out[0]

    for bad in [dict(val=None), dict(grad=None), dict(m=None), dict(v=None), dict(val=p + 2), dict(grad=p + 1025),
                dict(m=p + 2049), dict(v=p + 3074), dict(copy=p + 4097), dict(grad_dtype=3), dict(copy_dtype=0),
                dict(state_bits=16), dict(state_bits=8), dict(state_bits=8, m_scale=p + 5000), dict(m_scale=p + 5120),
                dict(state_bits=8, m_scale=p + 5121, v_scale=p + 5376), dict(n=(1 << 37) + 1), dict(m=p + 32), dict(grad=p),
                dict(grad=p + 60), dict(copy=p + 3072 + 60), dict(v=p + 2048 + 60)]:
        assert both(_tensor(nb, p, **bad)) == nb.NK_ERR_INVALID, bad
    # Two tensors that share an output, or one's output the other's gradient; a gradient may be shared.
    q = p + 8192
    assert both(_tensor(nb, p), _tensor(nb, q, m=p + 2048)) == nb.NK_ERR_INVALID
    assert both(_tensor(nb, p), _tensor(nb, q, grad=p)) == nb.NK_ERR_INVALID
    assert both(count=2 ** 25) == nb.NK_ERR_INVALID
    assert L.nk_adamw_many_create(None, 1, C.byref(h)) == nb.NK_ERR_INVALID
    assert L.nk_adamw_many_create(None, 0, None) == nb.NK_ERR_INVALID
    L.nk_adamw_many_free(None)
    assert L.nk_adamw_many_step_device(None, C.byref(cfg), 1.0, 0.0, None, None, None) == nb.NK_ERR_INVALID


def test_adamw_hyper_parameters(nb):
    t = (nb.train.NkAdamwTensor * 1)()
    good = dict(lr=1e-3, b1=0.9, b2=0.95, eps=1e-8, wd=0.0, t=1, grad_scale=1.0, max_norm=0.0)
    for bad in [dict(lr=NAN), dict(lr=-1.0), dict(b1=1.0), dict(b1=-0.1), dict(b2=NAN), dict(b2=1.5), dict(eps=0.0),
                dict(wd=-1.0), dict(wd=INF), dict(t=0), dict(grad_scale=NAN), dict(grad_scale=INF), dict(max_norm=-1.0),
                dict(max_norm=NAN), dict(max_norm=INF)]:
        a = {**good, **bad}
        cfg = nb.NkAdamwCfg(a["lr"], a["b1"], a["b2"], a["eps"], a["wd"], a["t"], 1)
        st = nb.lib().nk_adamw_many_step(t, 0, C.byref(cfg), a["grad_scale"], a["max_norm"], None, 0)
        assert st == nb.NK_ERR_INVALID, bad
    assert nb.lib().nk_adamw_many_step(t, 0, None, 1.0, 0.0, None, 0) == nb.NK_ERR_INVALID


def test_python_mirror_refuses_shapes(nb):
    x, w = np.zeros((3, 4), np.float32), np.zeros((5, 4), np.float32)
    for bad in [lambda: nb.linear_cross_entropy(x, w[:, :3], [0, 1, 2]), lambda: nb.linear_cross_entropy(x, w, [0, 1]),
                lambda: nb.linear_cross_entropy(x[0], w, [0]),
                lambda: nb.linear_cross_entropy_backward(x, w, [0, 1, 2], np.zeros(5)),
                lambda: nb.linear_cross_entropy_backward(x, w, [0, 1, 2], np.zeros((3, 2)), row_weight=np.zeros(2)),
                lambda: nb.linear_cross_entropy(x, w, [0, 1, 2**32 + 1]),
                lambda: nb.adamw_step_many([dict(val=np.zeros(4), grad=np.zeros(3), m=np.zeros(4), v=np.zeros(4))], 0.1, 1),
                lambda: nb.adamw_step_many([dict(val=np.zeros(4), grad=np.zeros(4), m=np.zeros(4), v=np.zeros(4),
                                                 m_scale=np.zeros(2), v_scale=np.zeros(1))], 0.1, 1)]:
        with pytest.raises(ValueError):
            bad()


def _far(nb, name, rows, width, vocab, dtype, w, room):
    """Whether a call is refused for its workspace.  (At these addresses there is nothing, and no
    call gets as far as looking.)"""
    a = dict(_calls(1 << 40)[name], dtype=dtype, rows=rows, width=width, x_stride=width, x=2 << 40, w=(3 << 40) + w, vocab=vocab,
             w_stride=width, targets=4 << 40, stats=5 << 40, workspace=6 << 40, workspace_bytes=room)
    a.update(dict(loss=7 << 40) if "loss" in a else dict(row_weight=None, dx=8 << 40, dx_stride=width, dw=9 << 40, dw_dtype=dtype,
                                                         dw_stride=width))
    st = _call(nb, name, a)
    assert st != nb.NK_OK
    return st == nb.NK_ERR_INVALID and "workspace" in nb.lib().nk_last_error().decode()


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("rows,width,vocab", [(8192, 1024, 32768), (2048, 768, 16384), (1024, 72, 3000), (100, 64, 1000)])
def test_a_workspace_serves_every_place_of_w_on_16_bytes(nb, dtype, rows, width, vocab):
    for name, back in (("nk_linear_ce_device", False), ("nk_linear_ce_backward_device", True)):
        n = [nb.train.linear_ce_workspace(dtype, rows, width, vocab, w=w, backward=back) for w in (256, 272, 320, 384)]
        assert n[0] == n[3] <= n[1] == n[2]  # (its place within 128 bytes)
        for w in (0, 16, 64, 112):
            assert not _far(nb, name, rows, width, vocab, dtype, w, n[0])
        assert _far(nb, name, rows, width, vocab, dtype, 16, 4096)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("width,vocab", [(768, 16384), (333, 131072), (24, 37), (1, 1), (64, 1000), (2048, 131072), (4097, 5000),
                                         (1024, 32768), (192, 300), (2304, 2048)])
def test_a_workspace_serves_any_fewer_rows(nb, dtype, width, vocab):
    rng = np.random.default_rng(width)
    most = min(1 << 17, (1 << 37) // vocab)
    sizes = sorted({1, 4, 5, 8, 9, 255, 256, 257, 1023, 1024, 2048, 4096, 4411, 5419, most,
                    *np.exp(rng.uniform(0, np.log(most), 40)).astype(int).tolist()})
    for name, back in (("nk_linear_ce_device", False), ("nk_linear_ce_backward_device", True)):
        for w in (0, 16, 4):
            n = [nb.train.linear_ce_workspace(dtype, rows, width, vocab, w=(3 << 40) + w, backward=back) for rows in sizes]
            assert n == sorted(n)
            for i, rows in enumerate(sizes):
                for fewer in {rows, *sizes[max(0, i - 6):i], *rng.integers(1, rows + 1, 6).tolist()}:
                    assert not _far(nb, name, fewer, width, vocab, dtype, w, n[i]), (rows, fewer, n[i])


def test_python_mirror_refuses_moments_of_another_kind_than_their_scales(nb):
    """Values taken as codes lost their fractions, and codes taken as values their scales."""
    def step(m, v, **scales):
        z = np.zeros(4, np.float32)
        return nb.adamw_step_many([dict(val=z, grad=z, m=m, v=v, **scales)], 0.1, 1)

    values, codes, one = np.full(4, 0.3, np.float32), np.full(4, 90, np.uint8), np.ones(1, np.float32)
    for m, v, scales in [(values, codes, True), (codes, values, True), (np.full(4, 300.0), codes, True), (-codes.astype(int), codes, True),
                         (codes, values, False), (values, codes, False)]:
        with pytest.raises(ValueError, match="codes"):
            step(m, v, **(dict(m_scale=one, v_scale=one) if scales else {}))
