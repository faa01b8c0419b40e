"""Torch-facing wrappers of the GLM C ABI.

Tensors follow the reference's Tensor3D memory layout
(``include/common/types/tensor3d.hpp:107-112``), written as C-contiguous
torch shapes ``[sheet, row, col]``:

* ``X``           ``(nobs, ntasks, nfeatures)``
* ``Y``, ``Yhat``  ``(nobs, ntasks, ntargets)``
* ``M``, ``grad``  ``(ntasks, ntargets, nfeatures)``

Every call launches asynchronously on ``stream`` (default: torch's current
stream) and goes to ``libglm_b200.so``; there is no host or torch fallback.

The whole-matrix operators at the end (:func:`orthogonalize`,
:func:`orthogonal_step`, :func:`quantize_q4`, :func:`dequantize_q4`,
:func:`predict_q4`; float32, float16 and bfloat16) also launch on the tensors'
own device where that is not the current one, and allocate what they return
on ``stream``.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import capi

SUFFIX = {
    torch.float16: "f16",
    torch.bfloat16: "bf16",
    torch.float32: "f32",
    torch.float64: "f64",
    torch.int8: "i8",
    torch.int16: "i16",
    torch.int32: "i32",
    torch.int64: "i64",
    torch.uint8: "u8",
    torch.uint16: "u16",
    torch.uint32: "u32",
    torch.uint64: "u64",
}


def _stream(stream) -> int:
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _need(t: torch.Tensor, name: str, shape, dtype) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _dims(X: torch.Tensor, M: torch.Tensor):
    nobs, ntasks, nf = X.shape
    ntasks2, nt, nf2 = M.shape
    if ntasks2 != ntasks or nf2 != nf:
        raise ValueError(f"X {tuple(X.shape)} and M {tuple(M.shape)} disagree")
    return nf, nt, ntasks, nobs


def predict(X, M, out=None, stream=None):
    """Yhat[obs, task, t] = sum_f M[task, t, f] X[obs, task, f]."""
    sfx = SUFFIX[X.dtype]
    nf, nt, ntasks, nobs = _dims(X, M)
    _need(X, "X", (nobs, ntasks, nf), X.dtype)
    _need(M, "M", (ntasks, nt, nf), X.dtype)
    if out is None:
        out = torch.empty((nobs, ntasks, nt), dtype=X.dtype, device=X.device)
    _need(out, "out", (nobs, ntasks, nt), X.dtype)
    capi.call(f"glmb_predict_{sfx}", _ptr(X), _ptr(M), _ptr(out), nf, nt, ntasks, nobs, _stream(stream))
    return out


def workspace_bytes(dtype, nf: int, nt: int, ntasks: int, nobs: int) -> int:
    return int(getattr(capi.lib(), f"glmb_gradient_workspace_size_{SUFFIX[dtype]}")(nf, nt, ntasks, nobs))


def gradient(X, M, Y, lam: float = 0.0, alpha: float = 0.0, regularize: bool = True,
             yhat_out=None, out=None, workspace=None, stream=None, logistic: bool = False):
    """Fused prediction + gradient (+ elastic-net term when ``regularize``).

    ``Y=None`` means an all-zero Y.  ``yhat_out`` (optional) receives the
    predictions.  ``workspace`` is an optional CUDA uint8 tensor of at least
    :func:`workspace_bytes` bytes.  ``logistic``: logistic link (mu =
    sigmoid(X M), gradient sum (mu - Y) X of the log-likelihood; predictions mu).
    """
    sfx = SUFFIX[X.dtype]
    nf, nt, ntasks, nobs = _dims(X, M)
    _need(X, "X", (nobs, ntasks, nf), X.dtype)
    _need(M, "M", (ntasks, nt, nf), X.dtype)
    flags = capi.GRAD_REGULARIZE if regularize else 0
    if logistic:
        flags |= capi.GRAD_LOGISTIC
    if Y is None:
        flags |= capi.GRAD_Y_ZERO
    else:
        _need(Y, "Y", (nobs, ntasks, nt), X.dtype)
    if yhat_out is not None:
        _need(yhat_out, "yhat_out", (nobs, ntasks, nt), X.dtype)
        flags |= capi.GRAD_WRITE_YHAT
    if out is None:
        out = torch.empty((ntasks, nt, nf), dtype=X.dtype, device=X.device)
    _need(out, "out", (ntasks, nt, nf), X.dtype)
    ws_ptr, ws_bytes = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel() * workspace.element_size())
    capi.call(f"glmb_gradient_{sfx}", _ptr(X), _ptr(M), _ptr(Y), _ptr(out), _ptr(yhat_out),
              nf, nt, ntasks, nobs, float(lam), float(alpha), flags, ws_ptr, ws_bytes, _stream(stream))
    return out


def loss(M, Y, Yhat, lam: float = 0.0, alpha: float = 0.0, out=None, workspace=None, stream=None):
    """sum (Yhat - Y)^2 + lam * (alpha * sum|M| + (1 - alpha) * sum M^2), as a
    one-element tensor of M's dtype (``Y=None``: zeros)."""
    sfx = SUFFIX[M.dtype]
    ntasks, nt, nf = M.shape
    nobs = Yhat.shape[0]
    _need(Yhat, "Yhat", (nobs, ntasks, nt), M.dtype)
    if Y is not None:
        _need(Y, "Y", (nobs, ntasks, nt), M.dtype)
    if out is None:
        out = torch.empty((1,), dtype=M.dtype, device=M.device)
    ws_ptr, ws_bytes = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel() * workspace.element_size())
    capi.call(f"glmb_loss_{sfx}", _ptr(M), _ptr(Y), _ptr(Yhat), _ptr(out), nf, nt, ntasks, nobs,
              float(lam), float(alpha), ws_ptr, ws_bytes, _stream(stream))
    return out


def gradient_loss(X, M, Y, lam: float = 0.0, alpha: float = 0.0, regularize: bool = True,
                  yhat_out=None, out=None, loss_out=None, workspace=None, stream=None):
    """Gradient (as :func:`gradient`) and loss (as :func:`loss`, always with
    the elastic-net term) from one call; returns (grad, loss, yhat).  On the
    rows path the squared residuals are summed in the gradient's own pass."""
    sfx = SUFFIX[X.dtype]
    nf, nt, ntasks, nobs = _dims(X, M)
    _need(X, "X", (nobs, ntasks, nf), X.dtype)
    _need(M, "M", (ntasks, nt, nf), X.dtype)
    flags = capi.GRAD_REGULARIZE if regularize else 0
    if Y is None:
        flags |= capi.GRAD_Y_ZERO
    else:
        _need(Y, "Y", (nobs, ntasks, nt), X.dtype)
    if yhat_out is None:
        yhat_out = torch.empty((nobs, ntasks, nt), dtype=X.dtype, device=X.device)
    _need(yhat_out, "yhat_out", (nobs, ntasks, nt), X.dtype)
    if out is None:
        out = torch.empty((ntasks, nt, nf), dtype=X.dtype, device=X.device)
    if loss_out is None:
        loss_out = torch.empty((1,), dtype=X.dtype, device=X.device)
    ws_ptr, ws_bytes = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel() * workspace.element_size())
    capi.call(f"glmb_gradient_loss_{sfx}", _ptr(X), _ptr(M), _ptr(Y), _ptr(out), _ptr(yhat_out), _ptr(loss_out),
              nf, nt, ntasks, nobs, float(lam), float(alpha), flags, ws_ptr, ws_bytes, _stream(stream))
    return out, loss_out, yhat_out


def gradient_partial(X, M, Y, out=None, yhat_out=None, workspace=None, stream=None):
    """sum_obs (Yhat - Y) X as float64 (no factor 2, no elastic-net term)."""
    sfx = SUFFIX[X.dtype]
    nf, nt, ntasks, nobs = _dims(X, M)
    flags = 0
    if Y is None:
        flags |= capi.GRAD_Y_ZERO
    else:
        _need(Y, "Y", (nobs, ntasks, nt), X.dtype)
    if yhat_out is not None:
        flags |= capi.GRAD_WRITE_YHAT
    if out is None:
        out = torch.empty((ntasks, nt, nf), dtype=torch.float64, device=X.device)
    _need(out, "out", (ntasks, nt, nf), torch.float64)
    ws_ptr, ws_bytes = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel() * workspace.element_size())
    capi.call(f"glmb_gradient_partial_{sfx}", _ptr(X), _ptr(M), _ptr(Y), _ptr(out), _ptr(yhat_out),
              nf, nt, ntasks, nobs, flags, ws_ptr, ws_bytes, _stream(stream))
    return out


def gradient_finalize(partial, M, lam: float = 0.0, alpha: float = 0.0, regularize: bool = True,
                      out=None, stream=None):
    """grad = 2*partial + lam*(alpha*sign(M) + 2*(1-alpha)*M)."""
    sfx = SUFFIX[M.dtype]
    ntasks, nt, nf = M.shape
    _need(partial, "partial", (ntasks, nt, nf), torch.float64)
    if out is None:
        out = torch.empty_like(M)
    capi.call(f"glmb_gradient_finalize_{sfx}", _ptr(partial), _ptr(M), _ptr(out), nf, nt, ntasks,
              float(lam), float(alpha), capi.GRAD_REGULARIZE if regularize else 0, _stream(stream))
    return out


def prox_step(beta, grad_smooth, inv_L: float, l1: float, stream=None):
    sfx = SUFFIX[beta.dtype]
    capi.call(f"glmb_prox_step_{sfx}", _ptr(beta), _ptr(grad_smooth), beta.numel(), float(inv_L),
              float(l1), _stream(stream))
    return beta


def prox_update(partial, beta, lipschitz, lambda1: float, lambda2: float, stream=None):
    sfx = SUFFIX[beta.dtype]
    ntasks, nt, nf = beta.shape
    capi.call(f"glmb_prox_update_{sfx}", _ptr(partial), _ptr(beta), _ptr(lipschitz), nf, nt, ntasks,
              float(lambda1), float(lambda2), _stream(stream))
    return beta


def power_init(v, seed: int, stream=None):
    """v: (ntasks, 1, nfeatures) start vector of the power iteration."""
    sfx = SUFFIX[v.dtype]
    ntasks, _, nf = v.shape
    capi.call(f"glmb_power_init_{sfx}", _ptr(v), nf, ntasks, int(seed) & (2**64 - 1), _stream(stream))
    return v


def power_step(partial, v, norm, lipschitz, lambda2: float, stream=None):
    sfx = SUFFIX[v.dtype]
    ntasks, _, nf = v.shape
    capi.call(f"glmb_power_step_{sfx}", _ptr(partial), _ptr(v), _ptr(norm), _ptr(lipschitz), nf,
              ntasks, float(lambda2), _stream(stream))
    return v


def fit_elastic_net(X, Y, lambda1: float, lambda2: float, n_power: int = 20, n_iter: int = 200,
                    seed: int = 42, beta=None, lipschitz=None, workspace=None, stream=None):
    """Single-GPU ISTA fit; returns (beta, lipschitz per task)."""
    sfx = SUFFIX[X.dtype]
    nobs, ntasks, nf = X.shape
    nt = Y.shape[2]
    if beta is None:
        beta = torch.empty((ntasks, nt, nf), dtype=X.dtype, device=X.device)
    if lipschitz is None:
        lipschitz = torch.empty((ntasks,), dtype=torch.float64, device=X.device)
    ws_ptr, ws_bytes = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel() * workspace.element_size())
    capi.call(f"glmb_fit_elastic_net_{sfx}", _ptr(X), _ptr(Y), _ptr(beta), _ptr(lipschitz), nf, nt,
              ntasks, nobs, float(lambda1), float(lambda2), int(n_power), int(n_iter),
              int(seed) & (2**64 - 1), ws_ptr, ws_bytes, _stream(stream))
    return beta, lipschitz


# ---- whole-matrix operators: orthogonalised updates, models in 4 bits ----------------

MATRIX_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _matrix_suffix(dtype) -> str:
    if dtype not in MATRIX_DTYPES:
        raise ValueError(f"dtype {dtype} is not one of float32, float16, bfloat16")
    return SUFFIX[dtype]


def _refuse(t, name: str, shape, dtype, device) -> None:
    _need(t, name, shape, dtype)
    raise ValueError(f"{name} is on {t.device}, expected {device}")


def _need_on(t: torch.Tensor, name: str, shape, dtype, device) -> None:
    # the checks of _need, in the order that costs a good call least
    if t.dtype != dtype or t.device != device or t.shape != shape or not t.is_cuda or not t.is_contiguous():
        _refuse(t, name, shape, dtype, device)


def _on(device, stream):
    """A context in which the tensors' device and the call's stream are
    current, allocations included; None where they are already."""
    if stream is None:
        return None if device.index == torch.cuda.current_device() else torch.cuda.device(device)
    if stream.device != device:
        raise ValueError(f"stream is on {stream.device}, the tensors are on {device}")
    return torch.cuda.stream(stream)


def _run(name: str, sfx: str, device, args) -> None:
    """One call of the library on the current stream of ``device``."""
    f = _entry.get((name, sfx))
    if f is None:
        f = _entry[(name, sfx)] = getattr(capi.lib(), f"{name}_{sfx}")
    st = f(*args, _raw_stream(device.index))
    if st != capi.GLMB_OK:
        capi.check(st, f"{name}_{sfx}")


_entry: dict = {}
# the current stream's handle without building a Stream object around it (2 us of a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                      lambda index: torch.cuda.current_stream(index).cuda_stream)


def _workspace(workspace, device):
    if workspace is None:
        return None, 0
    if workspace.device != device:
        raise ValueError(f"workspace is on {workspace.device}, expected {device}")
    if not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    return workspace.data_ptr(), workspace.nbytes


def _model_dims(M: torch.Tensor, name: str):
    if M.dim() != 3:
        raise ValueError(f"{name} has shape {tuple(M.shape)}, expected (ntasks, ntargets, nfeatures)")
    return M.shape


def _coefficients(coefficients, steps: int):
    """A host array of 3*steps doubles, or None for the library's own."""
    if coefficients is None:
        return None  # the library checks `steps`
    rows = list(coefficients)
    if len(rows) == 3 and all(isinstance(v, (int, float)) for v in rows):
        rows = [rows] * steps
    if len(rows) != steps or any(len(r) != 3 for r in rows):
        raise ValueError(f"coefficients must be one (a, b, c) or {steps} of them")
    return (ctypes.c_double * (3 * steps))(*[float(v) for r in rows for v in r])


def orthogonal_workspace_bytes(dtype, nf: int, nt: int, ntasks: int) -> int:
    """Workspace of :func:`orthogonalize` and :func:`orthogonal_step`."""
    return int(getattr(capi.lib(), f"glmm_orthogonal_workspace_size_{_matrix_suffix(dtype)}")(nf, nt, ntasks))


def orthogonalize(G, steps: int = 5, coefficients=None, out=None, workspace=None, stream=None):
    """Newton-Schulz orthogonalisation of every task's matrix of ``G``
    ``(ntasks, ntargets, nfeatures)``: X = G/|G|_F (zero stays zero), then
    ``steps`` times X <- aX + (bA + cA^2)X with A = X X^T on the shorter side.

    ``coefficients``: one (a, b, c) or one per step (any iterable of them), by default (3.4445,
    -4.7750, 2.0315), which brings the singular values near 1 in five steps.
    ``out`` may be ``G``."""
    sfx, device = _matrix_suffix(G.dtype), G.device
    _model_dims(G, "G")
    _need_on(G, "G", G.shape, G.dtype, device)
    steps = int(steps)
    coef = _coefficients(coefficients, steps)
    on = _on(device, stream)
    if on is not None:
        with on:
            return _orthogonalize(G, sfx, device, steps, coef, out, workspace)
    return _orthogonalize(G, sfx, device, steps, coef, out, workspace)


def _orthogonalize(G, sfx, device, steps, coef, out, workspace):
    # (on the current stream of `device`; coefficients may be an iterator, so they come as the array made of them)
    ntasks, nt, nf = G.shape
    if out is None:
        out = torch.empty_like(G)
    else:
        _need_on(out, "out", G.shape, G.dtype, device)
    ws_ptr, ws_bytes = _workspace(workspace, device)
    _run("glmm_orthogonalize", sfx, device,
         (G.data_ptr(), out.data_ptr(), nf, nt, ntasks, coef, steps, ws_ptr, ws_bytes))
    return out


def orthogonal_step(M, grad, momentum, lr: float, mu: float = 0.95, nesterov: bool = True,
                    weight_decay: float = 0.0, scale: float | None = None, steps: int = 5, coefficients=None,
                    workspace=None, stream=None):
    """One update of the model ``M`` by its orthogonalised momentum, in place:

        momentum <- mu*momentum + grad             (float32, M's shape)
        U = grad + mu*momentum if nesterov else momentum
        M <- (1 - lr*weight_decay)*M - lr*scale*orthogonalize(U)

    ``grad`` has M's type (as :func:`gradient` returns it); ``scale`` is
    sqrt(max(1, ntargets/nfeatures)) by default.  Returns ``M``."""
    sfx, device = _matrix_suffix(M.dtype), M.device
    ntasks, nt, nf = _model_dims(M, "M")
    _need_on(M, "M", M.shape, M.dtype, device)
    _need_on(grad, "grad", M.shape, M.dtype, device)
    _need_on(momentum, "momentum", M.shape, torch.float32, device)
    if scale is None:
        scale = math.sqrt(max(1.0, nt / nf)) if nf > 0 else 1.0
    steps = int(steps)
    coef = _coefficients(coefficients, steps)
    ws_ptr, ws_bytes = _workspace(workspace, device)
    args = (M.data_ptr(), grad.data_ptr(), momentum.data_ptr(), nf, nt, ntasks, float(lr), float(mu),
            float(weight_decay), float(scale), capi.STEP_NESTEROV if nesterov else 0, coef, steps, ws_ptr, ws_bytes)
    on = _on(device, stream)
    if on is not None:
        with on:
            _run("glmm_orthogonal_step", sfx, device, args)
    else:
        _run("glmm_orthogonal_step", sfx, device, args)
    return M


class Q4Model:
    """A model in 4 bits: codes and one scale per target and group of
    features, in the library's layout (``glm_matrix_b200.h``).  Made by
    :func:`quantize_q4`; ``shape`` is ``(ntasks, ntargets, nfeatures)``."""

    def __init__(self, shape, dtype, group: int, device):
        ntasks, nt, nf = self.shape = tuple(int(v) for v in shape)
        self.dtype, self.group = dtype, int(group)
        _matrix_suffix(dtype)
        if self.group not in (64, 128):
            raise ValueError(f"group is {group}, expected 64 or 128")
        codes, count = _q4_sizes(nf, nt, ntasks, self.group)
        # one allocation; the scales follow the codes, which are a multiple of 512 bytes
        self._held = torch.empty(codes + count * dtype.itemsize, dtype=torch.uint8, device=device)
        self._codes_bytes = codes

    def _pointers(self):
        # (asked of the tensor every time: a copied or unpickled model has another one)
        codes = self._held.data_ptr()
        return codes, codes + self._codes_bytes

    @property
    def device(self):
        return self._held.device

    @property
    def codes(self):
        return self._held[:self._codes_bytes]

    @property
    def scales(self):
        return self._held[self._codes_bytes:].view(self.dtype)


@functools.lru_cache(maxsize=256)
def _q4_sizes(nf: int, nt: int, ntasks: int, group: int):
    """Bytes of codes and number of scales, as the library lays them out."""
    L = capi.lib()
    return L.glmm_q4_codes_bytes(nf, nt, ntasks), L.glmm_q4_scales_count(nf, nt, ntasks, group)


def quantize_q4(M, group: int = 128, out=None, stream=None) -> Q4Model:
    """``M`` in 4 bits: per target and group of 64 or 128 features a scale
    s = max|w|/7 (rounded to M's type) and codes q = w/s rounded to the nearest
    of -7..7, ties to even.  ``out``: a Q4Model of the same shape to overwrite."""
    sfx, device = _matrix_suffix(M.dtype), M.device
    ntasks, nt, nf = _model_dims(M, "M")
    _need_on(M, "M", M.shape, M.dtype, device)
    on = _on(device, stream)
    if on is not None:
        with on:
            return quantize_q4(M, group, out)
    if out is None:
        out = Q4Model(M.shape, M.dtype, group, device)
    elif (out.shape, out.dtype, out.group, out.device) != (tuple(M.shape), M.dtype, group, device):
        raise ValueError("out was made for another shape, dtype, group or device")
    _run("glmm_quantize_q4", sfx, device,
         (M.data_ptr(), *out._pointers(), nf, nt, ntasks, out.group))
    return out


def dequantize_q4(model: Q4Model, out=None, stream=None):
    """The weights q*s of a :class:`Q4Model`, rounded to its dtype."""
    ntasks, nt, nf = model.shape
    device = model.device
    if device.type != "cuda":
        raise ValueError("model must be on a CUDA device")
    on = _on(device, stream)
    if on is not None:
        with on:
            return dequantize_q4(model, out)
    if out is None:
        out = torch.empty(model.shape, dtype=model.dtype, device=device)
    else:
        _need_on(out, "out", model.shape, model.dtype, device)
    _run("glmm_dequantize_q4", SUFFIX[model.dtype], device,
         (*model._pointers(), out.data_ptr(), nf, nt, ntasks, model.group))
    return out


def predict_q4_workspace_bytes(dtype, nf: int, nt: int, ntasks: int, nobs: int, group: int) -> int:
    """Workspace of :func:`predict_q4`."""
    return int(getattr(capi.lib(), f"glmm_predict_q4_workspace_size_{_matrix_suffix(dtype)}")(nf, nt, ntasks, nobs,
                                                                                            int(group)))


def predict_q4(X, model: Q4Model, out=None, workspace=None, stream=None):
    """:func:`predict` from a :class:`Q4Model`: Yhat[obs, task, t] = sum_f
    q[task, t, f]*s X[obs, task, f], from one observation to many; the products
    are those of the exact weights q*s, sums are float32."""
    ntasks, nt, nf = model.shape
    dtype, device = model.dtype, model.device
    if X.dim() != 3:
        raise ValueError(f"X has shape {tuple(X.shape)}, expected (nobs, ntasks, nfeatures)")
    nobs = X.shape[0]
    _need_on(X, "X", (nobs, ntasks, nf), dtype, device)
    on = _on(device, stream)
    if on is not None:
        with on:
            return predict_q4(X, model, out, workspace)
    if out is None:
        out = torch.empty((nobs, ntasks, nt), dtype=dtype, device=device)
    else:
        _need_on(out, "out", (nobs, ntasks, nt), dtype, device)
    ws_ptr, ws_bytes = _workspace(workspace, device)
    _run("glmm_predict_q4", SUFFIX[dtype], device,
         (X.data_ptr(), *model._pointers(), out.data_ptr(), nf, nt, ntasks, nobs,
          model.group, ws_ptr, ws_bytes))
    return out
