"""Norm and products of per-pixel (or per-token) rows on the kernels of csrc/rmsnorm.hip and csrc/linear.hip.

    y, h = rms_norm(x, weight, residual=r)            h = x + r,  y = h / rms(h) * weight            (differentiable)
    q, s, h = rms_norm_q8(x, weight, residual=r)      the same with y as e4m3 and a scale per row
    y = linear(x, w, bias, act="gelu", residual=r)    y = act(x w^T + bias) + r                      (differentiable)
    y = linear_q8(q, s, wq, ws, ...)                  the same on e4m3 rows and an e4m3 weight (quantize_rows)

The last axis is the row; leading axes may be any.  Rows may have any length, pitch and offset: rows that the kernels cannot read
in 16-byte pieces are laid out again first (one more launch; widths that are multiples of 8 - of 16 in 8 bits - avoid it; 16-bit layers
of up to about 200 values each way read any layout in place).
Everything runs on the current stream of the tensors' device, allocates from torch's allocator only, and may be captured into a
graph.  As for every torch module, a backward pass is captured only when no eager graph over the same leaves is alive any more
(drop the losses of the eager steps first); such a capture is refused here (autograd would end the process).
Refused with an exception: tensors that are not on one GPU, types other than the ones named, shapes that do not match.
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


def _pitch(t: torch.Tensor) -> int:
    rows, cols = t.shape
    return t.stride(0) if rows > 1 else max(cols, 1)


def _pieces(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """(matrix, pitch) that the product's kernels can read: 16-byte aligned rows of whole 16-byte pieces."""
    es, (rows, cols) = t.element_size(), t.shape
    per = 16 // es
    ld = t.stride(0) if rows > 1 else cols
    if not t.data_ptr() % 16 and not cols % per and not ld % per and ld < (1 << 21):
        return t, ld
    ldd = -(-cols // per) * per
    out = torch.empty((rows, ldd), dtype=t.dtype, device=t.device)
    rt.call("selfc_pack_rows", t.data_ptr(), ld, out.data_ptr(), rows, cols, ldd, es, _stream(t))
    return out, ldd


def _ws(rows: int, cols: int, total: int, es: int, device) -> Optional[torch.Tensor]:
    n = _lib.lib().selfc_linear_ws_floats(rows, cols, total, es)
    return torch.empty(n, dtype=torch.float32, device=device) if n else None


_ptr = rt._ptr

# -- captured backward passes ----------------------------------------------------------------------------------------------------
_EAGER = "selfc_amd_eager_graph"


def _watch(out: torch.Tensor):
    """A leaf's gradient accumulator lives as long as a graph that reaches it and remembers the stream it was made on.  If an eager
    graph is still alive when a captured backward pass reaches the same leaf, autograd waits for that stream inside the capture and
    the process ends.  So: the accumulators that an eager call reaches are marked with its stream, and a call under capture that meets
    another stream's mark refuses."""
    here = _raw_stream(out.get_device())
    capturing = torch.cuda.is_current_stream_capturing()
    for node, _ in out.grad_fn.next_functions:
        if node is None:
            continue
        if not hasattr(node, "variable"):                # rows of a leaf with more axes: a view in between
            node = next((n for n, _ in node.next_functions if n is not None and hasattr(n, "variable")), None)
            if node is None:
                continue
        meta = node.metadata
        if not capturing:
            meta[_EAGER] = here
        elif meta.get(_EAGER, here) != here:
            _bad("a graph of an earlier eager call over the same parameters is still alive; its gradients cannot be accumulated inside a "
                 "capture - drop that call's outputs and losses first")


def _no_second(ctx):
    if torch.is_grad_enabled():
        _bad("no second derivatives (create_graph=True)")


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


def _run_norm(x2, r2, weight, eps, q8: bool):
    rows, cols = x2.shape
    dev, dt = x2.device, x2.dtype
    y = torch.empty((rows, cols), dtype=torch.float8_e4m3fn if q8 else dt, device=dev)
    scale = torch.empty(rows, dtype=torch.float32, device=dev) if q8 else None
    h = torch.empty((rows, cols), dtype=dt, device=dev) if r2 is not None else None
    if rows:
        rt.call("selfc_rmsnorm", x2.data_ptr(), _pitch(x2), _ptr(r2), 0 if r2 is None else _pitch(r2), weight.data_ptr(),
                weight.dtype is torch.float32, _ptr(h), y.data_ptr(), _ptr(scale), rows, cols, _DTYPE[dt], eps, _stream(x2))
    return y, scale, h


class RMSNormFn(torch.autograd.Function):
    """rms_norm on matrices; the gradient needs h and the weight only (the row's statistic is recomputed)."""

    @staticmethod
    def forward(ctx, x2, r2, weight, eps):
        with on_device(x2):
            y, _, h = _run_norm(x2, r2, weight, eps, False)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x2 if h is None else h, weight)
        return (y,) if h is None else (y, h)

    @staticmethod
    def backward(ctx, dy, dh=None):
        _no_second(ctx)
        h, weight = ctx.saved_tensors
        to_x, to_r, want_w, _ = ctx.needs_input_grad
        want_x = to_x or to_r
        if dy is None:                     # only h was used
            return (dh if to_x else None), (dh if to_r else None), None, None
        rows, cols = h.shape
        dy = dy.contiguous()
        dh = dh.contiguous() if dh is not None else None
        with on_device(h):
            dx = torch.empty((rows, cols), dtype=h.dtype, device=h.device) if want_x else None
            dw = torch.empty_like(weight, memory_format=torch.contiguous_format) if want_w else None
            part = torch.empty(_lib.lib().selfc_rmsnorm_bwd_floats(rows, cols), dtype=torch.float32, device=h.device) if want_w else None
            if rows:
                rt.call("selfc_rmsnorm_bwd", h.data_ptr(), _pitch(h), weight.data_ptr(), weight.dtype is torch.float32, dy.data_ptr(), _ptr(dh),
                        _ptr(dx), _ptr(dw), _ptr(part), rows, cols, _DTYPE[h.dtype], ctx.eps, _stream(h))
            elif dw is not None:
                dw.zero_()
        return (dx if to_x else None), (dx if to_r else None), dw, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, h): h = x + residual rounded to x's type (x itself without a residual), y = h / sqrt(mean(h^2) + eps) * weight.

    x: bf16, f16 or fp32 rows of up to 16,384 values; weight: x's type or fp32.  Statistics and the weight's gradient are summed in
    fp32 in a fixed order.  Gradients flow to x, residual and weight, from y and h."""
    _norm_args(x, weight, residual, eps)
    x2, r2, weight = _rows(x), None if residual is None else _rows(residual), weight.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
        out = RMSNormFn.apply(x2, r2, weight, float(eps))
        _watch(out[0])
        y, h = out if r2 is not None else (out[0], None)
    else:
        with on_device(x):
            y, _, h = _run_norm(x2, r2, weight, float(eps), False)
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
        q, scale, h = _run_norm(_rows(x), None if residual is None else _rows(residual), weight.contiguous(), float(eps), True)
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


def _run_linear(xp, ldx, k, wp, ldw, n, xs, ws_, bias, act, r2, out_dtype, want_slope):
    rows, dev = xp.shape[0], xp.device
    y = torch.empty((rows, n), dtype=out_dtype, device=dev)
    slope = torch.empty((rows, -(-n // 8) * 8), dtype=torch.int16, device=dev) if want_slope else None
    if rows:
        es = xp.element_size()
        k = -(-k * es // 16) * 16 // es
        work = _ws(rows, n, k, es, dev) if rows > 16 else None
        rt.call("selfc_linear", xp.data_ptr(), ldx, wp.data_ptr(), ldw, _ptr(xs), _ptr(ws_), _ptr(bias), act, _ptr(r2),
                0 if r2 is None else _pitch(r2), y.data_ptr(), _ptr(slope), _ptr(work), rows, n, k, _DTYPE[xp.dtype], _DTYPE[out_dtype], _stream(xp))
    return y, slope


def _narrow(n: int, k: int) -> bool:
    return n <= 256 and k <= 256 and bool(_lib.lib().selfc_linear_rows_ok(n, k))


def _run_rows(x2, w2, bias, act, r2, want_slope, want_pieces):
    """(y, slope, x as whole pieces) of a narrow layer: one launch, any layout of x and the weight."""
    (rows, k), n = x2.shape, w2.shape[0]
    dev, dt = x2.device, x2.dtype
    y = torch.empty((rows, n), dtype=dt, device=dev)
    slope = torch.empty((rows, -(-n // 8) * 8), dtype=torch.int16, device=dev) if want_slope else None
    xp = None
    if want_pieces:
        whole = k % 8 == 0 and x2.data_ptr() % 16 == 0 and _pitch(x2) % 8 == 0 and _pitch(x2) < (1 << 21)
        xp = x2 if whole else torch.empty((rows, -(-k // 8) * 8), dtype=dt, device=dev)
    if rows:
        rt.call("selfc_linear_rows", x2.data_ptr(), _pitch(x2), w2.data_ptr(), _pitch(w2), _ptr(bias), act, _ptr(r2), 0 if r2 is None else _pitch(r2),
                y.data_ptr(), _ptr(slope), None if xp is None or xp is x2 else xp.data_ptr(), rows, n, k, _DTYPE[dt], _stream(x2))
    return y, slope, xp


class LinearFn(torch.autograd.Function):
    """linear on matrices.  Kept for the backward pass: x as the kernels read it, the weight, and the activation's derivative as 16-bit
    fixed point."""

    @staticmethod
    def forward(ctx, x2, weight, bias, r2, act):
        n, k = weight.shape
        need = ctx.needs_input_grad
        slope = act != 0 and any(need[:3])
        ctx.narrow = _narrow(n, k)
        with on_device(x2):
            if ctx.narrow:
                y, slope, xp = _run_rows(x2, weight, bias, act, r2, slope, need[1])
                wp, ldw = weight, _pitch(weight)
            else:
                xp, ldx = _pieces(x2)
                wp, ldw = _pieces(weight)
                y, slope = _run_linear(xp, ldx, k, wp, ldw, n, None, None, bias, act, r2, x2.dtype, slope)
        ctx.dims = (x2.shape[0], n, k, ldw)
        ctx.save_for_backward(xp if need[1] else None, wp if need[0] else None, slope)
        ctx.dtype = x2.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        _no_second(ctx)
        xp, wp, slope = ctx.saved_tensors
        rows, n, k, ldw = ctx.dims
        want_x, want_w, want_b, want_r, _ = ctx.needs_input_grad
        dev, dt, code, stream = dy.device, ctx.dtype, _DTYPE[ctx.dtype], _stream(dy)
        dx = dw = db = None
        if rows == 0:
            return (torch.empty((0, k), dtype=dt, device=dev) if want_x else None, torch.zeros((n, k), dtype=dt, device=dev) if want_w else None,
                    torch.zeros(n, dtype=dt, device=dev) if want_b else None, (dy if want_r else None), None)
        L = _lib.lib()
        with on_device(dy):
            g = _rows(dy)
            ldg, up = _pitch(g), -(-n // 8) * 8
            as_is = slope is None and n % 8 == 0 and g.data_ptr() % 16 == 0 and ldg % 8 == 0 and ldg < (1 << 21)
            rows_kernel = want_x and ctx.narrow
            make_dz = not as_is and (want_w or (want_x and not rows_kernel))
            dz, lddz = (torch.empty((rows, up), dtype=dt, device=dev), up) if make_dz else (g, ldg)
            if want_b:                              # with dW it comes out of that product
                db = torch.empty(n, dtype=dt, device=dev)
            if want_x:
                dx = torch.empty((rows, k), dtype=dt, device=dev)
            if rows_kernel:
                rt.call("selfc_linear_rows_bwd", g.data_ptr(), ldg, _ptr(slope), wp.data_ptr(), ldw, dx.data_ptr(), dz.data_ptr() if make_dz else None,
                        rows, n, k, code, stream)
            alone = want_b and not want_w
            if alone or (make_dz and not rows_kernel):
                part = torch.empty(L.selfc_linear_dz_floats(rows, n), dtype=torch.float32, device=dev) if alone else None
                rt.call("selfc_linear_dz", g.data_ptr(), ldg, _ptr(slope), dz.data_ptr() if make_dz and not rows_kernel else None, up,
                        db.data_ptr() if alone else None, _ptr(part), rows, n, code, stream)
            if want_x and not rows_kernel:
                work = _ws(rows, k, n, 2, dev)
                rt.call("selfc_linear_dx", dz.data_ptr(), lddz, wp.data_ptr(), ldw, dx.data_ptr(), _ptr(work), rows, n, k, code, stream)
            if want_w:
                dw = torch.empty((n, k), dtype=dt, device=dev)
                floats = L.selfc_linear_dw_floats(rows, n, k)
                work = torch.empty(floats, dtype=torch.float32, device=dev) if floats else None
                rt.call("selfc_linear_dw", dz.data_ptr(), lddz, xp.data_ptr(), _pitch(xp), dw.data_ptr(), _ptr(db), _ptr(work), rows, n, k, code, stream)
        return dx, dw, db, (dy if want_r else None), None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, act: str = "none",
           residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x weight^T + bias) + residual; x (..., in), weight (out, in), both bf16 or both f16, bias (out,) and residual (..., out) of the
    same type.  act: "none", "relu", "lrelu" (0.2), "gelu" (erf), "silu".  Sums, bias, activation and residual in fp32, one rounding at the end;
    in the backward pass dy act'(z) is rounded to x's type once, as the operand of both products.  Wide weights
    stream through a kernel of its own for up to 16 rows; layers of up to about 200 values each way keep theirs in shared memory.  Sums are added in a fixed order."""
    dt = x.dtype
    if dt is not torch.bfloat16 and dt is not torch.float16:
        _lib.require_gpu(x)
        _bad_type("x", x, torch.bfloat16, torch.float16)
    _linear_args(x, weight, bias, act, residual, dt)
    x2, w2 = _rows(x), _rows(weight)
    b = None if bias is None else bias.contiguous()
    r2 = None if residual is None else _rows(residual)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        y = LinearFn.apply(x2, w2, b, r2, ACTS[act])
        _watch(y)
    else:
        with on_device(x):
            n, k = w2.shape
            if _narrow(n, k):
                y = _run_rows(x2, w2, b, ACTS[act], r2, False, False)[0]
            else:
                xp, ldx = _pieces(x2)
                wp, ldw = _pieces(w2)
                y, _ = _run_linear(xp, ldx, k, wp, ldw, n, None, None, b, ACTS[act], r2, dt, False)
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
    (out, in) with a scale per output (quantize_rows); bias and residual of out_dtype (bf16, f16 or fp32).  For serving: no gradients."""
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
        x2 = _rows(x)
        xp, ldx = _pieces(x2)
        wp, ldw = _pieces(_rows(weight))
        y, _ = _run_linear(xp, ldx, x2.shape[1], wp, ldw, weight.shape[0], x_scale.reshape(-1).contiguous(), w_scale.contiguous(),
                           None if bias is None else bias.contiguous(), ACTS[act], None if residual is None else _rows(residual), out_dtype, False)
    return y if x.dim() == 2 else y.view(x.shape[:-1] + weight.shape[:1])
