"""The end of a training step (``include/noetic/train.h``): cross entropy straight
from hidden rows and the vocabulary matrix, its gradients, and AdamW over all of
a model's tensors at once.

:func:`linear_cross_entropy`, :func:`linear_cross_entropy_backward` and
:func:`adamw_step_many` take numpy arrays and run on ``device``, as the other ops
of the package do (a uint16 array holds bfloat16 bits).  Arrays that already live
on a GPU go to the ``nk_linear_ce*_device`` calls of :func:`noetic_b200.lib` and
to :class:`AdamwMany`.
"""

from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import numpy as np

from .head import NK_BF16, NK_F16, NK_F32, _matrix, _nb, _ptr, _vector

_P, _u32, _u64, _i32, _f32 = C.c_void_p, C.c_uint32, C.c_uint64, C.c_int, C.c_float

NK_ADAMW_BLOCK = 256


class NkAdamwTensor(C.Structure):
    _fields_ = [("val", _P), ("grad", _P), ("m", _P), ("v", _P), ("m_scale", _P), ("v_scale", _P), ("copy", _P),
                ("n", _u64), ("grad_dtype", _i32), ("copy_dtype", _i32), ("state_bits", _i32), ("decay", _i32)]


# Every entry point of include/noetic/train.h: name -> (restype, argtypes).
SIGNATURES = {
    "nk_linear_ce_device": (_i32, [_P, _i32, _u64, _u64, _u64, _P, _u64, _u64, _P, _P, _P, _P, _u64, _P]),
    "nk_linear_ce": (_i32, [_P, _i32, _u64, _u64, _P, _u64, _P, _P, _P, _i32]),
    "nk_linear_ce_workspace": (_i32, [_i32, _u64, _u64, _u64, _P, _u64, _i32, C.POINTER(_u64)]),
    "nk_linear_ce_backward_device": (_i32, [_P, _i32, _u64, _u64, _u64, _P, _u64, _u64, _P, _P, _P, _f32, _P, _u64, _P,
                                            _i32, _u64, _i32, _P, _u64, _P]),
    "nk_linear_ce_backward": (_i32, [_P, _i32, _u64, _u64, _P, _u64, _P, _P, _P, _f32, _P, _P, _i32, _i32, _i32]),
    "nk_linear_ce_withhold": (_i32, [_i32]),
    "nk_adamw_many_create": (_i32, [C.POINTER(NkAdamwTensor), _u64, C.POINTER(_P)]),
    "nk_adamw_many_free": (None, [_P]),
    "nk_adamw_many_step_device": (_i32, [_P, _P, _f32, _f32, _P, _P, _P]),
    "nk_adamw_many_step": (_i32, [C.POINTER(NkAdamwTensor), _u64, _P, _f32, _f32, _P, _i32]),
}


def linear_ce_workspace(dtype: int, rows: int, width: int, vocab: int, w: int = 256, w_stride: int | None = None,
                        backward: bool = False) -> int:
    """Bytes of workspace that ``nk_linear_ce_device`` (``backward``:
    ``nk_linear_ce_backward_device``) needs for up to ``rows`` rows; ``w`` is the address of the
    vocabulary matrix, of which the place within 128 bytes counts."""
    nb = _nb()
    n = _u64()
    nb._check(nb.lib().nk_linear_ce_workspace(dtype, rows, width, vocab, w, width if w_stride is None else w_stride,
                                              int(backward), C.byref(n)))
    return n.value


def _pair(x, w):
    x, code = _matrix(x, "x")
    w, w_code = _matrix(w, "w")
    if w_code != code or w.shape[1] != x.shape[1]:
        raise ValueError("x and w must have the same type and width")
    return x, w, code


def linear_cross_entropy(x, w, targets, device: int = 0) -> dict:
    """The ``loss`` of each row of ``x`` [rows, width] under the logits ``x @ w.T``
    (``w`` [vocab, width]), which are not kept, and the ``stats`` of
    :func:`linear_cross_entropy_backward`."""
    nb = _nb()
    x, w, code = _pair(x, w)
    rows, width = x.shape
    t = _vector(targets, rows, "targets", np.uint32)
    out = {"loss": np.empty(rows, np.float32), "stats": np.empty((rows, 2), np.float32)}
    nb._check(nb.lib().nk_linear_ce(_ptr(x), code, rows, width, _ptr(w), w.shape[0], _ptr(t), _ptr(out["loss"]),
                                    _ptr(out["stats"]), device))
    return out


def linear_cross_entropy_backward(x, w, targets, stats, row_weight=None, grad_scale: float = 1.0, dw=None,
                                  device: int = 0):
    """The gradients (dx, dw) of ``grad_scale * sum(row_weight * loss)``, from what
    :func:`linear_cross_entropy` returned.  dw has the type of ``w``; a given
    ``dw`` (of that type, or float32) is added to."""
    nb = _nb()
    x, w, code = _pair(x, w)
    rows, width = x.shape
    t = _vector(targets, rows, "targets", np.uint32)
    st, rw = _vector(stats, 2 * rows, "stats"), _vector(row_weight, rows, "row_weight")
    dx, dw_code, add = np.empty_like(x), code, dw is not None
    if add:
        dw, dw_code = _matrix(np.array(dw), "dw")
        if dw.shape != w.shape:
            raise ValueError("dw must have the shape of w")
    else:
        dw = np.empty_like(w)
    nb._check(nb.lib().nk_linear_ce_backward(_ptr(x), code, rows, width, _ptr(w), w.shape[0], _ptr(t), _ptr(st), _ptr(rw),
                                             grad_scale, _ptr(dx), _ptr(dw), dw_code, int(add), device))
    return dx, dw


@dataclass
class AdamwTensor:
    """One parameter tensor of :class:`AdamwMany`: device addresses, ``n`` elements
    and the types of ``nk_adamw_tensor``."""

    val: int
    grad: int
    m: int
    v: int
    n: int
    m_scale: int | None = None
    v_scale: int | None = None
    copy: int | None = None
    grad_dtype: int = NK_F32
    copy_dtype: int = NK_BF16
    state_bits: int = 32
    decay: int = 1


class AdamwMany:
    """AdamW over all of a model's tensors in one launch, on arrays that live on a
    GPU.  They stay where they are until :meth:`close`."""

    def __init__(self, tensors):
        nb = _nb()
        self.h, self._nb = None, None
        table = (NkAdamwTensor * len(tensors))(*[
            NkAdamwTensor(t.val, t.grad, t.m, t.v, t.m_scale, t.v_scale, t.copy, t.n, t.grad_dtype, t.copy_dtype,
                          t.state_bits, t.decay) for t in tensors])
        h = _P()
        nb._check(nb.lib().nk_adamw_many_create(table, len(tensors), C.byref(h)))
        self.h, self._nb = h, nb

    def step(self, lr: float, t: int, b1: float = 0.9, b2: float = 0.95, eps: float = 1e-8, wd: float = 0.0,
             grad_scale: float = 1.0, max_norm: float = 0.0, norm: int | None = None, bad: int | None = None,
             stream: int | None = None):
        """One step on ``stream``; t is the step counter after its increment.  ``norm``
        and ``bad`` are device addresses of a float32 and a uint32."""
        nb = self._nb
        cfg = nb.NkAdamwCfg(lr, b1, b2, eps, wd, t, 1)
        nb._check(nb.lib().nk_adamw_many_step_device(self.h, C.byref(cfg), grad_scale, max_norm, norm, bad, stream))

    def close(self):
        if self.h:
            self._nb.lib().nk_adamw_many_free(self.h)
            self.h = None

    def __del__(self):
        if self._nb is not None and self._nb.lib is not None:  # (None as the interpreter ends)
            self.close()


def _moment(a, kind, what):
    """A copy of a moment: float32, or codes of 8 bits, which no other numbers stand for."""
    a = np.asarray(a)
    new = np.array(a, kind).reshape(-1)
    if a.dtype != kind and (a.dtype == np.uint8 or (kind == np.uint8 and not np.array_equal(new, a.reshape(-1)))):
        raise ValueError(f"{what}: codes of 8 bits need m_scale and v_scale, and scales need codes")
    return new


def adamw_step_many(tensors, lr: float, t: int, b1: float = 0.9, b2: float = 0.95, eps: float = 1e-8, wd: float = 0.0,
                    grad_scale: float = 1.0, max_norm: float = 0.0, device: int = 0):
    """One AdamW step over copies of all ``tensors``, each a dict of arrays ``val``,
    ``grad``, ``m``, ``v`` (float32, or uint8 codes with ``m_scale`` and
    ``v_scale``, one for each 256 elements), with ``decay`` (default True) and
    ``copy`` ("f16" or "bf16": also return val rounded to it).  Returns (list of
    dicts of the new arrays, the gradients' norm)."""
    nb = _nb()
    table, out, keep = (NkAdamwTensor * len(tensors))(), [], []
    for i, t_in in enumerate(tensors):
        val = np.array(t_in["val"], np.float32).reshape(-1)
        grad = np.asarray(t_in["grad"])
        codes = {np.dtype(np.float32): NK_F32, np.dtype(np.float16): NK_F16, np.dtype(np.uint16): NK_BF16}
        grad = np.ascontiguousarray(grad if grad.dtype in codes else grad.astype(np.float32)).reshape(-1)
        bits = 8 if t_in.get("m_scale") is not None else 32
        kind = np.uint8 if bits == 8 else np.float32
        new = {"val": val, "m": _moment(t_in["m"], kind, "m"), "v": _moment(t_in["v"], kind, "v")}
        if bits == 8:
            blocks = -(-val.size // NK_ADAMW_BLOCK)
            for k in ("m_scale", "v_scale"):
                new[k] = np.array(_vector(t_in[k], blocks, k))
        if t_in.get("copy"):
            new["copy"] = np.empty(val.size, {"f16": np.float16, "bf16": np.uint16}[t_in["copy"]])
        if not grad.size == val.size == new["m"].size == new["v"].size:
            raise ValueError("val, grad, m and v must have the same size")
        table[i] = NkAdamwTensor(*[None if a is None else a.ctypes.data for a in
                                   (val, grad, new["m"], new["v"], new.get("m_scale"), new.get("v_scale"), new.get("copy"))],
                                 val.size, codes[grad.dtype], NK_F16 if t_in.get("copy") == "f16" else NK_BF16, bits,
                                 int(t_in.get("decay", True)))
        keep.append(grad)
        out.append(new)
    norm = C.c_float()
    cfg = nb.NkAdamwCfg(lr, b1, b2, eps, wd, t, 1)
    nb._check(nb.lib().nk_adamw_many_step(table, len(tensors), C.byref(cfg), grad_scale, max_norm, C.byref(norm), device))
    return out, norm.value
