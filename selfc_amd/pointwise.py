"""Norm and products of per-pixel (or per-token) rows on the kernels of csrc/rmsnorm.hip and csrc/linear.hip.

    y, h = rms_norm(x, weight, residual=r)            h = x + r,  y = h / rms(h) * weight            (differentiable)
    q, s, h = rms_norm_q8(x, weight, residual=r)      the same with y as e4m3 and a scale per row
    y = linear(x, w, bias, act="gelu", residual=r)    y = act(x w^T + bias) + r                      (differentiable)
    y = linear_q8(q, s, wq, ws, ...)                  the same on e4m3 rows and an e4m3 weight (quantize_rows)

The last axis is the row; leading axes may be any.  Rows may have any length, pitch and offset: rows that the kernels cannot read
in 16-byte pieces are laid out again first (one more launch; widths that are multiples of 8 - of 16 in 8 bits - avoid it; 16-bit layers
of up to 256 values each way, and products of up to 16 rows of up to 8 KiB without gradients, read any layout in place).
Everything runs on the current stream of the tensors' device, allocates from torch's allocator only, and may be captured into a
graph.  As for every torch module, a backward pass is captured only when no eager graph over the same leaves is alive any more
(drop the losses of the eager steps first); such a capture is refused here (autograd would end the process).
Refused with an exception: tensors that are not on one GPU, types other than the ones named, shapes that do not match, second and
forward-mode derivatives.
"""
from __future__ import annotations

from contextlib import nullcontext
from typing import Optional, Tuple

import torch

from . import _lib, runtime as rt

#: activations of `linear`, by their number in the C ABI
ACTS = {"none": 0, None: 0, "relu": 1, "lrelu": 2, "gelu": 3, "silu": 4}
_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.float8_e4m3fn: 3}
_NAMES = {torch.float32: "float32", torch.bfloat16: "bfloat16", torch.float16: "float16", torch.float8_e4m3fn: "float8_e4m3fn"}
MAX_NORM_COLS = 16384
MAX_LINEAR = 1 << 20
E4M3_MAX = 448.0

_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_HERE = nullcontext()


def on_device(t: torch.Tensor):
    """The tensor's device as the current one for the duration of a launch."""
    return _HERE if t.get_device() == _current_device() else torch.cuda.device(t.device)


def _stream(t: torch.Tensor) -> int:
    """hipStream_t of the current stream of the tensor's device."""
    return _raw_stream(t.get_device())


def _bad(what: str):
    raise RuntimeError("selfc_amd: " + what)


def _elsewhere(first, **others):
    _lib.require_gpu(first)
    for name, t in others.items():
        if t is not None and t.device != first.device:
            _bad(f"{name} is on {t.device}, the rows are on {first.device}")


def _bad_type(name: str, t: torch.Tensor, *dtypes):
    _bad(f"{name} is {t.dtype}, expected {' or '.join(_NAMES[d] for d in dtypes)}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """(..., C) as a matrix whose rows are contiguous and do not overlap (a view where one exists)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.is_contiguous():
        return t
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


# -- captured backward passes ----------------------------------------------------------------------------------------------------
_MARK = "selfc_amd_graph_of"


def _watch(out: torch.Tensor):
    """A leaf's gradient accumulator lives as long as a graph that reaches it and remembers the stream it was made on.  If an eager
    graph is still alive when a captured backward pass reaches the same leaf, autograd waits for that stream inside the capture and
    the process ends; if a captured graph's outputs are still alive when another pass does, eager or captured, and the capture's stream is
    gone (runtime.graph_capture destroys its own), it ends as well.  So: the accumulators that a call reaches are marked with the stream
    and with whether it was being captured, and a call that meets such a mark refuses."""
    here = _raw_stream(out.get_device())
    capturing = torch.cuda.is_current_stream_capturing()
    for node, _ in out.grad_fn.next_functions:
        if node is None:
            continue
        for _ in range(4):                               # views and copies of a leaf in between: its rows, its transpose
            if hasattr(node, "variable"):
                break
            before = [n for n, _ in node.next_functions if n is not None]
            if len(before) != 1:
                break
            node = before[0]
        if not hasattr(node, "variable"):
            continue
        meta = node.metadata
        made, captured = meta.setdefault(_MARK, (here, capturing))
        if capturing and not captured and made != here:
            _bad("a graph of an earlier eager call over the same parameters is still alive; its gradients cannot be accumulated inside a "
                 "capture - drop that call's outputs and losses first")
        if captured and made != here and made in rt.CLOSED_STREAMS:
            _bad("a captured call's outputs over the same parameters still hold their graph, whose stream is gone - keep detached outputs of a "
                 "capture")


# -- norm ------------------------------------------------------------------------------------------------------------------------
def _norm_args(x, weight, residual, eps):
    dt, shape, dev = x.dtype, x.shape, x.device
    if not x.is_cuda or weight.device != dev or (residual is not None and residual.device != dev):
        _elsewhere(x, weight=weight, residual=residual)
    if dt is not torch.bfloat16 and dt is not torch.float16 and dt is not torch.float32:
        _bad_type("x", x, torch.bfloat16, torch.float16, torch.float32)
    if weight.dtype is not dt and weight.dtype is not torch.float32:
        _bad_type("weight", weight, *{dt, torch.float32})
    if not shape or not 1 <= shape[-1] <= MAX_NORM_COLS:
        _bad(f"rms_norm takes rows of 1 to {MAX_NORM_COLS} values, got {tuple(shape)}")
    if weight.dim() != 1 or weight.shape[0] != shape[-1]:
        _bad(f"weight has shape {tuple(weight.shape)}, the rows have {shape[-1]} values")
    if not eps >= 0:
        _bad(f"eps is {eps}")
    if residual is not None:
        if residual.dtype is not dt:
            _bad_type("residual", residual, dt)
        if residual.shape != shape:
            _bad(f"residual has shape {tuple(residual.shape)}, x {tuple(shape)}")


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, h): h = x + residual rounded to x's type (x itself without a residual), y = h / sqrt(mean(h^2) + eps) * weight.

    x: bf16, f16 or fp32 rows of up to 16,384 values; weight: x's type or fp32.  Statistics and the weight's gradient are summed in
    fp32 in a fixed order.  Gradients flow to x, residual and weight, from y and h."""
    _norm_args(x, weight, residual, eps)
    x2, r2, weight = _rows(x), None if residual is None else _rows(residual), weight.contiguous()
    grad = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad))
    with on_device(x):
        y, _, h = _lib.host().norm(x2, r2, weight, eps, False, grad, _stream(x))
        if grad:
            _watch(y)
    if x.dim() == 2:
        return y, (x if h is None else h)
    return y.view(x.shape), (x if h is None else h.view(x.shape))


def _no_grad_only(what: str, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise NotImplementedError(f"selfc_amd: {what} serves only - call it under torch.no_grad() (its 16-bit form has gradients)")


def rms_norm_q8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """(q, scale, h): rms_norm with y as float8_e4m3fn, y = q * scale[row] (fp32; the row's largest |y| is 448 steps, a row of zeros has
    scale 1).  For serving: no gradients."""
    _norm_args(x, weight, residual, eps)
    _no_grad_only("rms_norm_q8", x, weight, residual)
    with on_device(x):
        q, scale, h = _lib.host().norm(_rows(x), None if residual is None else _rows(residual), weight.contiguous(), eps, True, False, _stream(x))
    if x.dim() == 2:
        return q, scale, (x if h is None else h)
    return q.view(x.shape), scale.view(x.shape[:-1]), (x if h is None else h.view(x.shape))


# -- product ---------------------------------------------------------------------------------------------------------------------
def _linear_args(x, weight, bias, act, residual, out_dtype):
    """checks what `linear` and `linear_q8` share; the rows' type is the caller's to check"""
    dev, shape = x.device, x.shape
    if not x.is_cuda or weight.device != dev or (bias is not None and bias.device != dev) or (residual is not None and residual.device != dev):
        _elsewhere(x, weight=weight, bias=bias, residual=residual)
    if weight.dtype is not x.dtype:
        _bad_type("weight", weight, x.dtype)
    if weight.dim() != 2 or not shape or weight.shape[1] != shape[-1] or not 1 <= shape[-1] <= MAX_LINEAR or not 1 <= weight.shape[0] <= MAX_LINEAR:
        _bad(f"x {tuple(shape)} does not go with weight {tuple(weight.shape)}: (out, in) of 1 to {MAX_LINEAR}")
    if act not in ACTS:
        _bad(f"act is {act!r}, expected one of {sorted(k for k in ACTS if k)}")
    if bias is not None:
        if bias.dtype is not out_dtype:
            _bad_type("bias", bias, out_dtype)
        if bias.dim() != 1 or bias.shape[0] != weight.shape[0]:
            _bad(f"bias has shape {tuple(bias.shape)}, expected ({weight.shape[0]},)")
    if residual is not None:
        if residual.dtype is not out_dtype:
            _bad_type("residual", residual, out_dtype)
        if residual.shape != shape[:-1] + weight.shape[:1]:
            _bad(f"residual has shape {tuple(residual.shape)}, expected {tuple(shape[:-1] + weight.shape[:1])}")


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, act: str = "none",
           residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x weight^T + bias) + residual; x (..., in), weight (out, in), both bf16 or both f16, bias (out,) and residual (..., out) of the
    same type.  act: "none", "relu", "lrelu" (0.2), "gelu" (erf), "silu".  Sums, bias, activation and residual in fp32, one rounding at the end;
    in the backward pass dy act'(z) is rounded to x's type once, as the operand of both products; the bias's gradient is the sum of that operand
    (without the weight's gradient: of the numbers before their rounding).  act' of GELU and SiLU is kept in steps of 2^-15.  Gradients are of
    x's type: in f16 a loss has to be scaled so that they fit (FFNet does).  Wide weights stream through a kernel of
    their own for up to 16 rows; layers of up to 256 values each way keep theirs in shared memory.  Sums are added in a fixed order."""
    dt = x.dtype
    if dt is not torch.bfloat16 and dt is not torch.float16:
        _lib.require_gpu(x)
        _bad_type("x", x, torch.bfloat16, torch.float16)
    _linear_args(x, weight, bias, act, residual, dt)
    x2, w2 = _rows(x), _rows(weight)
    b = None if bias is None else bias.contiguous()
    r2 = None if residual is None else _rows(residual)
    grad = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                        or (residual is not None and residual.requires_grad))
    with on_device(x):
        y = _lib.host().linear(x2, w2, b, r2, ACTS[act], grad, _stream(x))
        if grad:
            _watch(y)
    return y if x.dim() == 2 else y.view(x.shape[:-1] + weight.shape[:1])


def quantize_rows(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, scale) of a weight (out, in): float8_e4m3fn rows with one fp32 scale each, for linear_q8.  Done once per weight."""
    if w.dim() != 2 or not w.is_floating_point():
        _bad(f"quantize_rows expects a float matrix, got {w.dtype} {tuple(w.shape)}")
    w = w.detach().float()
    most = w.abs().amax(1) if w.shape[1] else w.new_zeros(w.shape[0])
    scale = torch.where(most > 0, (most / E4M3_MAX).clamp_(min=2.0 ** -126), torch.ones_like(most))
    return (w / scale[:, None]).to(torch.float8_e4m3fn), scale


def linear_q8(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
              act: str = "none", residual: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """act(x_scale w_scale (x weight^T) + bias) + residual for float8_e4m3fn x (..., in) with a scale per row (rms_norm_q8) and weight
    (out, in) with a scale per output (quantize_rows); bias and residual of out_dtype (bf16, f16 or fp32).  For serving: no gradients.
    The matrix unit cuts products below 2^-13 of the largest among eight neighbours; everything behind that is summed in fp32."""
    if out_dtype not in (torch.bfloat16, torch.float16, torch.float32):
        _bad(f"out_dtype is {out_dtype}")
    if x.dtype is not torch.float8_e4m3fn:
        _bad_type("x", x, torch.float8_e4m3fn)
    _linear_args(x, weight, bias, act, residual, out_dtype)
    _no_grad_only("linear_q8", bias, residual, x_scale, w_scale)
    if x_scale.device != x.device or w_scale.device != x.device:
        _elsewhere(x, x_scale=x_scale, w_scale=w_scale)
    for name, t, shape in (("x_scale", x_scale, x.shape[:-1]), ("w_scale", w_scale, weight.shape[:1])):
        if t.dtype is not torch.float32:
            _bad_type(name, t, torch.float32)
        if t.shape != shape:
            _bad(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    with on_device(x):
        y = _lib.host().linear_q8(_rows(x), x_scale.reshape(-1).contiguous(), _rows(weight), w_scale.contiguous(), None if bias is None else bias.contiguous(),
                                  None if residual is None else _rows(residual), ACTS[act], _DTYPE[out_dtype], _stream(x))
    return y if x.dim() == 2 else y.view(x.shape[:-1] + weight.shape[:1])
