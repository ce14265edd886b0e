"""The operators at the model's end (include/noetic/head.h) on CPU: the header,
the library and the Python mirror declare the same calls, and every bad argument
is refused with a status before any device work."""

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
    return C.create_string_buffer(1 << 12)


def test_header_library_and_mirror_agree(nb):
    text = open(os.path.join(ROOT, "include", "noetic", "head.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = set(re.findall(r"^nk_status\s+(nk_\w+)\s*\(", text, flags=re.M))
    assert names == set(nb.head.SIGNATURES)
    assert all(hasattr(C.CDLL(nb.LIB_PATH), n) for n in names)
    assert not names & set(nb.SIGNATURES)
    # The number of arguments, too.
    for n in names:
        args = re.search(r"\b%s\s*\((.*?)\);" % n, text, flags=re.S).group(1)
        assert len(args.split(",")) == len(nb.head.SIGNATURES[n][1]), n
    assert int(re.search(r"NK_MAX_TOP (\d+)u", text).group(1)) == nb.head.NK_MAX_TOP
    assert int(re.search(r"NK_MAX_TEACHER (\d+)u", text).group(1)) == nb.head.NK_MAX_TEACHER


# Arguments of a call that would be taken, by name; p is some address.
def _calls(p):
    return {
        "nk_token_logprobs_device": dict(logits=p, dtype=0, rows=2, vocab=8, row_stride=8, targets=p + 1024,
                                         temperature=1.0, top=2, logprob=p + 1280, entropy=p + 1536, stats=p + 1792,
                                         top_ids=p + 2048, top_logprobs=p + 2304, stream=None),
        "nk_token_logprobs_backward_device": dict(logits=p, dtype=0, rows=2, vocab=8, row_stride=8, targets=p + 1024,
                                                  temperature=1.0, stats=p + 1280, entropy=p + 1536, g_logprob=p + 1792,
                                                  g_entropy=p + 1792, dlogits=p, dlogits_stride=8, stream=None),
        "nk_distill_device": dict(logits=p, dtype=0, rows=2, vocab=8, row_stride=8, teacher_ids=p + 1024,
                                  teacher_logits=p + 1280, teacher_dtype=0, n_teacher=2, temperature=1.0, loss=p + 1536,
                                  row_weight=p + 1792, grad_scale=1.0, dlogits=p, dlogits_stride=8, stream=None),
        "nk_layer_norm_device": dict(x=p, dtype=0, rows=2, width=8, x_stride=8, gain=p + 1024, bias=p + 1024, eps=1e-5,
                                     rms=0, y=p, y_stride=8, mean=p + 1280, rstd=p + 1536, stream=None),
        "nk_layer_norm_backward_device": dict(x=p, dtype=0, rows=2, width=8, x_stride=8, gain=p + 256, mean=p + 512,
                                              rstd=p + 768, rms=0, dy=p + 1024, dy_stride=8, dx=p + 2048, dx_stride=8,
                                              dgain=p + 1280, dbias=p + 1536, accumulate=0, workspace=p + 2304,
                                              workspace_bytes=1 << 20, stream=None),
    }


REFUSALS = {
    "nk_token_logprobs_device": [
        dict(logits=None), dict(logits=2), dict(dtype=3), dict(dtype=-1), dict(vocab=0), dict(row_stride=7),
        dict(rows=(1 << 26) + 1), dict(vocab=1 << 31, row_stride=1 << 31), dict(row_stride=1 << 61),
        dict(rows=1 << 20, row_stride=1 << 20), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=NAN),
        dict(temperature=INF), dict(top=129), dict(top=0), dict(targets=None), dict(targets=2), dict(stats=1)],
    "nk_token_logprobs_backward_device": [
        dict(logits=None), dict(dtype=7), dict(vocab=0), dict(dlogits=None), dict(stats=None), dict(targets=None),
        dict(g_logprob=None, g_entropy=None), dict(entropy=None), dict(dlogits_stride=7), dict(dlogits_stride=9),
        dict(dlogits="+4"), dict(dlogits="+1"), dict(temperature=0.0), dict(dlogits_stride=1 << 40)],
    "nk_distill_device": [
        dict(logits=None), dict(dtype=5), dict(teacher_dtype=5), dict(vocab=0), dict(teacher_ids=None),
        dict(teacher_logits=None), dict(n_teacher=257), dict(loss=None, dlogits=None), dict(grad_scale=NAN),
        dict(grad_scale=INF), dict(temperature=NAN), dict(dlogits_stride=7), dict(dlogits="+4"),
        dict(teacher_logits="+2"), dict(row_weight=3)],
    "nk_layer_norm_device": [
        dict(x=None), dict(y=None), dict(dtype=3), dict(width=0), dict(x_stride=7), dict(y_stride=7), dict(eps=-1e-5),
        dict(eps=NAN), dict(eps=INF), dict(rms=1), dict(rms=1, bias=None), dict(rms=1, mean=None), dict(y="+4"),
        dict(x="+2"), dict(rows=(1 << 26) + 1), dict(gain=2)],
    "nk_layer_norm_backward_device": [
        dict(x=None), dict(dy=None), dict(rstd=None), dict(mean=None), dict(dtype=3), dict(width=0), dict(x_stride=7),
        dict(dy_stride=7), dict(dx_stride=7), dict(rms=1), dict(rms=1, mean=None), dict(workspace=None),
        dict(workspace_bytes=8), dict(workspace="+4"), dict(dx="-1020"), dict(dx="+1"), dict(dgain=2)],
}


@pytest.mark.parametrize("name,change", [(n, c) for n, cs in REFUSALS.items() for c in cs])
def test_bad_arguments_are_refused(nb, buf, name, change):
    p = C.addressof(buf)
    args = _calls(p)[name]
    for k, v in change.items():
        assert k in args
        args[k] = args[k] + int(v) if isinstance(v, str) else v
    assert getattr(nb.lib(), name)(*args.values()) == nb.NK_ERR_INVALID, nb.lib().nk_last_error()
    assert nb.lib().nk_last_error()


def test_dx_on_the_array_of_x_is_refused(nb, buf):
    p = C.addressof(buf)
    args = _calls(p)["nk_layer_norm_backward_device"]
    args["dx"] = args["x"]
    assert nb.lib().nk_layer_norm_backward_device(*args.values()) == nb.NK_ERR_INVALID


def test_columns_of_one_wide_array_do_not_overlap(nb, buf):
    # Refused for another reason (there is no device here, or the memory is the
    # host's), not as an overlap.
    p = C.addressof(buf)
    args = _calls(p)["nk_token_logprobs_backward_device"]
    args.update(row_stride=16, dlogits_stride=16, dlogits=p + 32)
    assert nb.lib().nk_token_logprobs_backward_device(*args.values()) != 0
    assert b"overlap" not in nb.lib().nk_last_error()
    args.update(dlogits=p + 28)
    assert nb.lib().nk_token_logprobs_backward_device(*args.values()) == nb.NK_ERR_INVALID
    assert b"overlap" in nb.lib().nk_last_error()


# An output on an input's place, or on another output's, other than in place.
@pytest.mark.parametrize("name,out,on", [
    ("nk_token_logprobs_device", "logprob", "targets"), ("nk_token_logprobs_device", "stats", "logits"),
    ("nk_token_logprobs_device", "entropy", "logprob"), ("nk_token_logprobs_device", "top_ids", "top_logprobs"),
    ("nk_token_logprobs_backward_device", "dlogits", "stats"), ("nk_token_logprobs_backward_device", "dlogits", "g_entropy"),
    ("nk_distill_device", "loss", "row_weight"), ("nk_distill_device", "loss", "dlogits"),
    ("nk_distill_device", "dlogits", "teacher_ids"), ("nk_layer_norm_device", "y", "gain"),
    ("nk_layer_norm_device", "mean", "x"), ("nk_layer_norm_device", "mean", "rstd"),
    ("nk_layer_norm_backward_device", "dgain", "gain"), ("nk_layer_norm_backward_device", "dbias", "dgain"),
    ("nk_layer_norm_backward_device", "workspace", "dy"), ("nk_layer_norm_backward_device", "dx", "rstd")])
def test_outputs_on_top_of_other_arrays_are_refused(nb, buf, name, out, on):
    args = _calls(C.addressof(buf))[name]
    getattr(nb.lib(), name)(*args.values())
    assert b"overlap" not in nb.lib().nk_last_error()
    for shift in (0, 4):
        assert getattr(nb.lib(), name)(*dict(args, **{out: args[on] + (0 if out == "workspace" else shift)}).values()) == nb.NK_ERR_INVALID
        assert b"overlap" in nb.lib().nk_last_error()


@pytest.mark.parametrize("temperature", [9e-5, 1.1e4, 1e30])
def test_distillation_refuses_temperatures_that_leave_the_loss_no_digits(nb, buf, temperature):
    args = _calls(C.addressof(buf))["nk_distill_device"]
    args["temperature"] = temperature
    assert nb.lib().nk_distill_device(*args.values()) == nb.NK_ERR_INVALID
    assert b"temperature" in nb.lib().nk_last_error()


@pytest.mark.parametrize("name", list(REFUSALS))
def test_no_rows_is_no_work(nb, name):
    args = _calls(0)[name]
    args = {k: (None if k in ("logits", "targets", "stats", "entropy", "logprob", "g_logprob", "g_entropy", "dlogits",
                              "top_ids", "top_logprobs", "teacher_ids", "teacher_logits", "loss", "row_weight", "x", "y",
                              "gain", "bias", "mean", "rstd", "dy", "dx", "dgain", "dbias", "workspace") else v)
            for k, v in args.items()}
    args["rows"] = 0
    assert getattr(nb.lib(), name)(*args.values()) == 0, nb.lib().nk_last_error()


def test_host_forms_refuse_null_arrays_and_bad_ids(nb):
    L = nb.lib()
    z = np.zeros((2, 4), np.float32)
    bad = np.array([1, 4], np.uint32)
    p = lambda a: a.ctypes.data_as(C.c_void_p)  # noqa: E731
    out = np.zeros(8, np.float32)
    assert L.nk_token_logprobs(None, 0, 2, 4, None, 1.0, 0, None, p(out), None, None, None, 0) == nb.NK_ERR_INVALID
    assert L.nk_token_logprobs(p(z), 0, 2, 4, p(bad), 1.0, 0, p(out), None, None, None, None, 0) == nb.NK_ERR_INVALID
    assert b"out of range" in L.nk_last_error()
    assert L.nk_token_logprobs_backward(p(z), 0, 2, 4, p(bad), 1.0, p(out), None, p(out), None, p(z), 0) == nb.NK_ERR_INVALID
    assert L.nk_distill(p(z), 0, 2, 4, p(bad), p(out), 0, 1, 1.0, p(out), None, 1.0, None, 0) == nb.NK_ERR_INVALID
    assert L.nk_layer_norm(None, 0, 2, 4, None, None, 1e-5, 0, p(z), None, None, 0) == nb.NK_ERR_INVALID
    assert L.nk_layer_norm_backward(p(z), 0, 2, 4, None, None, None, 1, p(z), p(z), None, None, 0, 0) == nb.NK_ERR_INVALID
    assert L.nk_layer_norm_backward_workspace(1, 1, None) == nb.NK_ERR_INVALID
    assert L.nk_layer_norm_backward_workspace(1, 1 << 31, C.byref(C.c_uint64())) == nb.NK_ERR_INVALID
    assert L.nk_model_score(None, None, None, 1, 1, 0, None, None, None, None) == nb.NK_ERR_INVALID


def test_python_mirror_checks_shapes(nb):
    z = np.zeros((2, 4), np.float32)
    with pytest.raises(ValueError):
        nb.token_logprobs(z[0], [0])
    with pytest.raises(ValueError):
        nb.token_logprobs(z, [0, 1, 2])
    with pytest.raises(ValueError):
        nb.distill(z, np.zeros((2, 3)), np.zeros((2, 2)))
    with pytest.raises(ValueError):
        nb.distill(z, np.zeros((3, 2)), np.zeros((3, 2)))
    with pytest.raises(ValueError):
        nb.layer_norm(z, gain=np.ones(3))
    with pytest.raises(ValueError):
        nb.layer_norm_backward(z, z.astype(np.float16), None, None, np.ones(2))


def test_workspace_grows_no_further_than_its_limit(nb):
    n = C.c_uint64()
    sizes = []
    for rows in (0, 1, 7, 1000, 1 << 20, 1 << 26):
        assert nb.lib().nk_layer_norm_backward_workspace(rows, 100, C.byref(n)) == 0
        sizes.append(n.value)
    assert sizes == sorted(sizes) and 0 < sizes[0] and sizes[-1] <= 2048 * 100 * 4
    # Nor do wide rows ask for more than a few sums of the parameters.
    assert nb.lib().nk_layer_norm_backward_workspace(1 << 10, 1 << 20, C.byref(n)) == 0
    assert n.value <= 64 * 2 * (1 << 20) * 4


def test_python_mirror_refuses_ids_beyond_32_bits(nb):
    # 2^32 + 1 is not token 1.
    z, far = np.zeros((2, 4), np.float32), np.array([0, (1 << 32) + 1])
    with pytest.raises(ValueError, match="32 bits"):
        nb.token_logprobs(z, far)
    with pytest.raises(ValueError, match="32 bits"):
        nb.token_logprobs_backward(z, -far, np.zeros((2, 2)), g_logprob=np.ones(2))
    with pytest.raises(ValueError, match="32 bits"):
        nb.distill(z, far[:, None], np.zeros((2, 1)))
    with pytest.raises(ValueError, match="32 bits"):
        nb.head.model_score(None, far, far, 1, 2)


def test_python_mirror_refuses_transposed_teacher_ids(nb):
    # As many ids as logits, but another row's.
    with pytest.raises(ValueError, match="shape"):
        nb.distill(np.zeros((2, 4), np.float32), np.zeros((3, 2), np.uint32), np.zeros((2, 3)))
