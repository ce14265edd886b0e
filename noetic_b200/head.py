"""Operators at the model's end (``include/noetic/head.h``): log probabilities
of given tokens, distillation from a teacher's top logits, layer norm and
RMSNorm, with their gradients.

The functions here take numpy arrays and run on ``device``, as the other ops of
the package do.  float32 and float16 arrays are passed as they are; a uint16
array holds bfloat16 bits.  Arrays that already live on a GPU go to the
``nk_*_device`` calls of :func:`noetic_b200.lib` instead (pointers, row strides
and a CUDA stream).
"""

from __future__ import annotations

import ctypes as C

import numpy as np

_P, _u32, _u64, _i32, _f32 = C.c_void_p, C.c_uint32, C.c_uint64, C.c_int, C.c_float

NK_F32, NK_F16, NK_BF16 = range(3)
NK_MAX_TOP, NK_MAX_TEACHER = 128, 256
NO_TOKEN = 0xFFFFFFFF

# Every entry point of include/noetic/head.h: name -> (restype, argtypes).
SIGNATURES = {
    "nk_token_logprobs_device": (_i32, [_P, _i32, _u64, _u64, _u64, _P, _f32, _u32, _P, _P, _P, _P, _P, _P]),
    "nk_token_logprobs": (_i32, [_P, _i32, _u64, _u64, _P, _f32, _u32, _P, _P, _P, _P, _P, _i32]),
    "nk_token_logprobs_backward_device": (_i32, [_P, _i32, _u64, _u64, _u64, _P, _f32, _P, _P, _P, _P, _P, _u64, _P]),
    "nk_token_logprobs_backward": (_i32, [_P, _i32, _u64, _u64, _P, _f32, _P, _P, _P, _P, _P, _i32]),
    "nk_distill_device": (_i32, [_P, _i32, _u64, _u64, _u64, _P, _P, _i32, _u32, _f32, _P, _P, _f32, _P, _u64, _P]),
    "nk_distill": (_i32, [_P, _i32, _u64, _u64, _P, _P, _i32, _u32, _f32, _P, _P, _f32, _P, _i32]),
    "nk_layer_norm_device": (_i32, [_P, _i32, _u64, _u64, _u64, _P, _P, _f32, _i32, _P, _u64, _P, _P, _P]),
    "nk_layer_norm": (_i32, [_P, _i32, _u64, _u64, _P, _P, _f32, _i32, _P, _P, _P, _i32]),
    "nk_layer_norm_backward_workspace": (_i32, [_u64, _u64, C.POINTER(_u64)]),
    "nk_layer_norm_backward_device": (_i32, [_P, _i32, _u64, _u64, _u64, _P, _P, _P, _i32, _P, _u64, _P, _u64, _P, _P,
                                             _i32, _P, _u64, _P]),
    "nk_layer_norm_backward": (_i32, [_P, _i32, _u64, _u64, _P, _P, _P, _i32, _P, _P, _P, _P, _i32, _i32]),
    "nk_model_score": (_i32, [_P, _P, _P, _u32, _u32, _u32, _P, _P, _P, _P]),
}


def _nb():
    import noetic_b200

    return noetic_b200


def _ptr(a):
    return None if a is None else a.ctypes.data_as(C.c_void_p)


def _matrix(a, what: str):
    """A contiguous matrix of a type the library takes, and its nk_dtype."""
    a = np.asarray(a)
    if a.ndim != 2:
        raise ValueError(f"{what} must be a matrix")
    codes = {np.dtype(np.float32): NK_F32, np.dtype(np.float16): NK_F16, np.dtype(np.uint16): NK_BF16}
    if a.dtype not in codes:
        a = a.astype(np.float32)
    return np.ascontiguousarray(a), codes[a.dtype]


def _vector(a, n: int, what: str, dtype=np.float32):
    if a is None:
        return None
    a = np.asarray(a)
    # (-1 in a signed array is 0xFFFFFFFF; the library looks at what is left.)
    if dtype == np.uint32 and a.dtype.itemsize > 4 and a.size and (a.max() > NO_TOKEN or a.min() < -(1 << 31)):
        raise ValueError(f"{what} must fit 32 bits")
    a = np.ascontiguousarray(a, dtype=dtype).reshape(-1)
    if a.size != n:
        raise ValueError(f"{what} must hold {n} values")
    return a


def token_logprobs(logits, targets=None, temperature: float = 1.0, top: int = 0, device: int = 0) -> dict:
    """Log probabilities of ``targets`` [rows] under ``logits`` [rows, vocab], with
    each row's ``entropy``, the ``stats`` of :func:`token_logprobs_backward` and
    its ``top`` most probable tokens (``top_ids``, ``top_logprobs``)."""
    nb = _nb()
    z, code = _matrix(logits, "logits")
    rows, vocab = z.shape
    t = _vector(targets, rows, "targets", np.uint32)
    out = {"logprob": None if t is None else np.empty(rows, np.float32), "entropy": np.empty(rows, np.float32),
           "stats": np.empty((rows, 2), np.float32)}
    if top:
        out.update(top_ids=np.empty((rows, top), np.uint32), top_logprobs=np.empty((rows, top), np.float32))
    nb._check(nb.lib().nk_token_logprobs(_ptr(z), code, rows, vocab, _ptr(t), temperature, top, _ptr(out["logprob"]),
                                         _ptr(out["entropy"]), _ptr(out["stats"]), _ptr(out.get("top_ids")),
                                         _ptr(out.get("top_logprobs")), device))
    return out


def token_logprobs_backward(logits, targets, stats, entropy=None, g_logprob=None, g_entropy=None,
                            temperature: float = 1.0, device: int = 0) -> np.ndarray:
    """The gradient of ``sum(g_logprob * logprob + g_entropy * entropy)`` for the
    logits, from what :func:`token_logprobs` returned."""
    nb = _nb()
    z, code = _matrix(logits, "logits")
    rows, vocab = z.shape
    t = _vector(targets, rows, "targets", np.uint32)
    st = _vector(stats, 2 * rows, "stats")
    en = _vector(entropy, rows, "entropy")
    gl, ge = _vector(g_logprob, rows, "g_logprob"), _vector(g_entropy, rows, "g_entropy")
    dz = np.empty_like(z)
    nb._check(nb.lib().nk_token_logprobs_backward(_ptr(z), code, rows, vocab, _ptr(t), temperature, _ptr(st), _ptr(en),
                                                  _ptr(gl), _ptr(ge), _ptr(dz), device))
    return dz


def distill(logits, teacher_ids, teacher_logits, temperature: float = 1.0, row_weight=None, grad_scale: float = 1.0,
            want_grad: bool = True, device: int = 0):
    """Distillation from a teacher's top logits [rows, n] at ``teacher_ids``:
    the loss of each row and, with ``want_grad``, the gradient of ``grad_scale *
    sum(row_weight * loss)`` for the logits.  Returns (loss, dlogits or None)."""
    nb = _nb()
    z, code = _matrix(logits, "logits")
    tl, t_code = _matrix(teacher_logits, "teacher_logits")
    rows, vocab = z.shape
    if tl.shape[0] != rows:
        raise ValueError("teacher_logits must have a row for each row of the logits")
    if np.ndim(teacher_ids) > 1 and np.shape(teacher_ids) != tl.shape:
        raise ValueError("teacher_ids must have the shape of teacher_logits")
    ids = _vector(teacher_ids, tl.size, "teacher_ids", np.uint32)
    w = _vector(row_weight, rows, "row_weight")
    loss = np.empty(rows, np.float32)
    dz = np.empty_like(z) if want_grad else None
    nb._check(nb.lib().nk_distill(_ptr(z), code, rows, vocab, _ptr(ids), _ptr(tl), t_code, tl.shape[1], temperature,
                                  _ptr(loss), _ptr(w), grad_scale, _ptr(dz), device))
    return loss, dz


def layer_norm(x, gain=None, bias=None, eps: float = 1e-5, rms: bool = False, device: int = 0) -> dict:
    """Layer norm of the rows of ``x`` (``rms``: RMSNorm, without mean and bias):
    ``y``, and the ``mean`` and ``rstd`` of :func:`layer_norm_backward`."""
    nb = _nb()
    x, code = _matrix(x, "x")
    rows, width = x.shape
    g, b = _vector(gain, width, "gain"), _vector(bias, width, "bias")
    y = np.empty_like(x)
    mean = None if rms else np.empty(rows, np.float32)
    rstd = np.empty(rows, np.float32)
    nb._check(nb.lib().nk_layer_norm(_ptr(x), code, rows, width, _ptr(g), _ptr(b), eps, int(rms), _ptr(y), _ptr(mean),
                                     _ptr(rstd), device))
    return {"y": y, "mean": mean, "rstd": rstd}


def layer_norm_backward(x, dy, gain, mean, rstd, dgain=None, dbias=None, device: int = 0):
    """The gradients of :func:`layer_norm` (``mean`` None: of its RMSNorm).
    Returns (dx, dgain, dbias); given ``dgain`` and ``dbias`` are added to."""
    nb = _nb()
    x, code = _matrix(x, "x")
    dy, dy_code = _matrix(dy, "dy")
    rows, width = x.shape
    if dy.shape != x.shape or dy_code != code:
        raise ValueError("dy must have the shape and type of x")
    rms = mean is None
    g, m, r = _vector(gain, width, "gain"), _vector(mean, rows, "mean"), _vector(rstd, rows, "rstd")
    dx = np.empty_like(x)
    dg = np.zeros(width, np.float32) if dgain is None else np.array(dgain, np.float32).reshape(-1)
    db = None if rms else np.zeros(width, np.float32) if dbias is None else np.array(dbias, np.float32).reshape(-1)
    if dg.size != width or (db is not None and db.size != width):
        raise ValueError("dgain and dbias must hold one value for each column")
    nb._check(nb.lib().nk_layer_norm_backward(_ptr(x), code, rows, width, _ptr(g), _ptr(m), _ptr(r), int(rms), _ptr(dy),
                                              _ptr(dx), _ptr(dg), _ptr(db), 1, device))
    return dx, dg, db


def model_score(model, ids, targets, batch: int, t: int, top: int = 0) -> dict:
    """``Model.score``: the log probability and entropy of every position of
    ``batch`` sequences of ``t`` tokens, and the ``top`` most probable tokens."""
    nb = _nb()
    ids = _vector(ids, batch * t, "ids", np.uint32)
    targets = _vector(targets, batch * t, "targets", np.uint32)
    out = {"logprob": np.empty((batch, t), np.float32), "entropy": np.empty((batch, t), np.float32)}
    if top:
        out.update(top_ids=np.empty((batch, t, top), np.uint32), top_logprobs=np.empty((batch, t, top), np.float32))
    nb._check(nb.lib().nk_model_score(model.h, _ptr(ids), _ptr(targets), batch, t, top, _ptr(out["logprob"]),
                                      _ptr(out["entropy"]), _ptr(out.get("top_ids")), _ptr(out.get("top_logprobs"))))
    return out
