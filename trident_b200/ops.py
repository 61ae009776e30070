"""Operators of a trainable query encoder: embedding lookup and layer norm, with their gradients.

An encoder in front of an index turns token ids into the vectors that the index searches: it looks up a
row of a table for each token, scales it, normalises it and pools the rows of a query. These functions are
the forward and backward passes of the first two steps (trident_b200.optim.AdamW takes the training step),
on the CUDA kernels of libtrident_b200.so; there is no CPU fallback.

Tensors are float32, float16 or bfloat16 CUDA tensors; sums and statistics are held in float32 and every
result is rounded once. Work is queued on the current stream and nothing is read back. Two calls with the
same inputs give the same bits. Inputs may have a row stride; one without unit stride in its last dim (a
transposed or broadcast tensor) is copied first.
"""
import ctypes
import functools
from typing import Optional

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _dtype(t, name: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, not {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return code


def _rows(t, D: int):
    """(tensor, row stride) of t seen as rows of D elements, copied if its strides do not allow that."""
    if t.is_contiguous():
        return t, D
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= D:
        return t, t.stride(0)
    return t.contiguous(), D


def _out_rows(t, D: int, name: str) -> int:
    if t.is_contiguous():
        return D
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= D:
        return t.stride(0)
    raise ValueError(f"{name} must be contiguous, or 2-D with unit stride in its last dim")


# The current stream's handle by device index. torch's own accessor builds a Stream object, 2 us of a call
# that takes 7; the raw one is used where this torch has it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(dev, fn, *args) -> None:
    """fn(*args, current stream) with dev as the current device."""
    index = dev.index
    if index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(rc)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(name: str, device_index: int, *sizes) -> int:
    """Workspace bytes of an operator (a function of its sizes and the device alone)."""
    need = ctypes.c_size_t(0)
    with torch.cuda.device(device_index):
        _lib.check(getattr(_lib.lib(), name)(*sizes, ctypes.byref(need)))
    return need.value


def _p(t):
    return None if t is None else t.data_ptr()


def _ids(ids, dev):
    if ids.dtype == torch.int64:
        bits = 64
    elif ids.dtype == torch.int32:
        bits = 32
    else:
        raise ValueError(f"ids must be int32 or int64, not {ids.dtype}")
    if ids.get_device() != dev.index:
        raise ValueError(f"ids are on {ids.device}, not on {dev}")
    return (ids if ids.is_contiguous() else ids.contiguous()), bits


def _status(status, dev) -> None:
    if status is not None and (status.dtype != torch.int32 or status.numel() != 1 or status.device != dev):
        raise ValueError(f"status must be one int32 on {dev}")


def embedding_lookup(table, ids, scale: float = 1.0, out=None, status=None):
    """out[..., :] = scale * table[ids[...], :], of the table's dtype.

    table: [V, D]; ids: int32 or int64 of any shape. An id of -1 (a padded token, or a missing result of a
    search) gives zeros. Any other id outside [0, V) gives a row of NaN and sets _lib.STATUS_BAD_ID in
    `status` (one int32 on the device, optional). out: [*ids.shape, D], optional."""
    code, dev = _dtype(table, "table"), table.device
    if table.dim() != 2:
        raise ValueError("table must be [V, D]")
    V, D = table.shape
    table, ld = _rows(table, D)
    ids, bits = _ids(ids, dev)
    _status(status, dev)
    shape = (*ids.shape, D)
    if out is None:
        out, ld_out = table.new_empty(shape), D
    else:
        if out.shape != shape or out.dtype != table.dtype or out.device != dev:
            raise ValueError(f"out must be a {table.dtype} tensor of shape {shape} on {dev}")
        ld_out = _out_rows(out, D, "out")
    _call(dev, _lib.lib().trident_embed_lookup, table.data_ptr(), code, V, D, ld, ids.data_ptr(), bits, ids.numel(),
          scale, out.data_ptr(), ld_out, _p(status))
    return out


def embedding_grad(grad_out, ids, num_rows: int, scale: float = 1.0, out=None, accumulate: bool = False,
                   dtype: Optional[torch.dtype] = None, status=None):
    """The gradient of embedding_lookup with respect to its table: [num_rows, D], row v being scale times the
    sum of grad_out's rows whose id is v, in an order that the ids alone fix.

    grad_out: [*ids.shape, D]. Ids outside [0, num_rows) give nothing (all but -1 set `status`, as in the
    lookup). dtype: that of grad_out (default) or float32. out: a tensor to write to; with accumulate=True
    the sums are added to it and rows that no id names are not touched."""
    code, dev = _dtype(grad_out, "grad_out"), grad_out.device
    if grad_out.dim() != ids.dim() + 1 or grad_out.shape[:-1] != ids.shape:
        raise ValueError(f"grad_out must be [*ids.shape, D], not {tuple(grad_out.shape)}")
    V, D = int(num_rows), grad_out.shape[-1]
    grad_out, ld = _rows(grad_out, D)
    ids, bits = _ids(ids, dev)
    _status(status, dev)
    if out is None:
        if accumulate:
            raise ValueError("accumulate=True needs out")
        out, ld_out = grad_out.new_empty((V, D), dtype=dtype), D
    else:
        if out.shape != (V, D) or out.device != dev or (dtype is not None and out.dtype != dtype):
            raise ValueError(f"out must be a {dtype or ''} tensor of shape {(V, D)} on {dev}")
        ld_out = _out_rows(out, D, "out")
    out_code, T = _dtype(out, "out"), ids.numel()
    need = _workspace_bytes("trident_embed_grad_workspace_size", dev.index, T, V, D)
    ws = grad_out.new_empty(need, dtype=torch.uint8) if need else None
    _call(dev, _lib.lib().trident_embed_grad, grad_out.data_ptr(), code, ld, ids.data_ptr(), bits, T, V, D, scale,
          int(accumulate), out.data_ptr(), out_code, ld_out, _p(ws), need, _p(status))
    return out


def _norm_param(t, name, D, x):
    if t is None:
        return
    if t.dim() != 1 or t.numel() != D or not t.is_contiguous() or t.get_device() != x.get_device():
        raise ValueError(f"{name} must be contiguous, of shape ({D},), on {x.device}")


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, out=None, stats: bool = True):
    """Layer norm over the last dim: y = (x - mean) * rstd * weight + bias with rstd = 1/sqrt(var + eps).

    x: [..., D]; weight, bias: [D] of x's dtype or float32 (both the same), or None. Returns (y, mean, rstd)
    with float32 statistics of shape x.shape[:-1] for layer_norm_grad, or y alone with stats=False. out: a
    tensor for y, which may be x itself."""
    code, dev = _dtype(x, "x"), x.device
    D = x.shape[-1] if x.dim() else 0
    if D < 1:
        raise ValueError("x must have a last dim of at least 1")
    _norm_param(weight, "weight", D, x)
    _norm_param(bias, "bias", D, x)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("weight and bias must have the same dtype")
    param = weight if weight is not None else bias
    pcode = code if param is None else _dtype(param, "weight")
    shape, rows = x.shape, x.numel() // D
    if out is None:
        x, ld = _rows(x, D)
        out, ld_out = x.new_empty(shape), D
    else:
        if out.shape != shape or out.dtype != x.dtype or out.device != dev:
            raise ValueError(f"out must be a {x.dtype} tensor of shape {tuple(shape)} on {dev}")
        ld_out = _out_rows(out, D, "out")
        x, ld = _rows(x, D)
    mean = rstd = None
    if stats:
        mean = x.new_empty(shape[:-1], dtype=torch.float32)
        rstd = torch.empty_like(mean)
    _call(dev, _lib.lib().trident_layer_norm, x.data_ptr(), code, rows, D, ld, _p(weight), _p(bias), pcode, eps,
          out.data_ptr(), ld_out, _p(mean), _p(rstd))
    return (out, mean, rstd) if stats else out


def layer_norm_grad(grad_out, x, weight, mean, rstd, out=None, param_grads: bool = True):
    """The backward pass of layer_norm: (dx, dweight, dbias).

    grad_out, x: [..., D] of one dtype; weight as in the forward pass (None: 1); mean, rstd: the statistics
    that layer_norm returned. dweight and dbias have weight's dtype (x's where it is None);
    param_grads=False leaves them out (None). out: a tensor for dx, which may be grad_out itself."""
    code, dev = _dtype(x, "x"), x.device
    D = x.shape[-1] if x.dim() else 0
    if D < 1:
        raise ValueError("x must have a last dim of at least 1")
    if grad_out.shape != x.shape or grad_out.dtype != x.dtype or grad_out.device != dev:
        raise ValueError("grad_out must have x's shape, dtype and device")
    _norm_param(weight, "weight", D, x)
    for s, name in ((mean, "mean"), (rstd, "rstd")):
        if s.shape != x.shape[:-1] or s.dtype != torch.float32 or not s.is_contiguous() or s.device != dev:
            raise ValueError(f"{name} must be contiguous float32 of shape {tuple(x.shape[:-1])} on {dev}")
    pcode = code if weight is None else _dtype(weight, "weight")
    shape, rows = x.shape, x.numel() // D
    if out is None:
        out, ld_out = x.new_empty(shape), D
    else:
        if out.shape != shape or out.dtype != x.dtype or out.device != dev:
            raise ValueError(f"out must be a {x.dtype} tensor of shape {tuple(shape)} on {dev}")
        ld_out = _out_rows(out, D, "out")
    x, ld_x = _rows(x, D)
    grad_out, ld_dy = _rows(grad_out, D)
    need = _workspace_bytes("trident_layer_norm_grad_workspace_size", dev.index, rows, D)
    ws = x.new_empty(need, dtype=torch.uint8)
    dw = db = None
    if param_grads:
        dw = x.new_empty(D) if weight is None else torch.empty_like(weight)
        db = torch.empty_like(dw)
    _call(dev, _lib.lib().trident_layer_norm_grad, grad_out.data_ptr(), ld_dy, x.data_ptr(), ld_x, code, rows, D, _p(weight),
          pcode, mean.data_ptr(), rstd.data_ptr(), out.data_ptr(), ld_out, _p(dw), _p(db), ws.data_ptr(), need)
    return out, dw, db
