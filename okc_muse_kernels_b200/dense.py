"""The dense operators around the expert block, over the C ABI.

``block_norm`` is the residual stream at a block's two ends: the norm after the block, its gate and scale, the residual
sum, and the norm before the next block, in one kernel (the reference's layer does this step around its experts in
`_boundary`, muse_decode_layer/layer.py).  ``int8_linear`` and ``int8_gated`` are products of 8-bit integers with a scale
per token and per weight row, for the dense projections of a layer and for feed-forwards without experts;
``quantize_rows`` makes such rows, of weights once and of tokens on the way in.

As in ``moe.py``: CUDA tensors only, work is enqueued on the current stream of the tensors' device, no host
synchronisation, capturable in a CUDA graph, wrong arguments raise ValueError before anything is launched.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import _lib
from ._lib import BlockNormArgs, Int8Args

__all__ = ["QuantRows", "quantize_rows", "int8_rows", "int8_linear", "int8_gated", "int8_ffn", "block_norm", "int8_status"]

BLOCK_NORM_MAX_HIDDEN = 16384
INT8_MAX_K = 131071           # the integer sums stay in 32 bits
_ROWS_KIND = {torch.bfloat16: 0, torch.float32: 1, torch.int8: 2}
_OUT = {"bf16": (0, torch.bfloat16), "f32": (1, torch.float32), "int8": (2, torch.int8)}


class QuantRows(NamedTuple):
    """Rows of int8 values and what they stand for: row r is ``q[r] * scale[r]``.  ``q`` int8 [R, C] with rows 16 bytes
    aligned, ``scale`` f32 [R]."""
    q: torch.Tensor
    scale: torch.Tensor


def _device(first: torch.Tensor, *others: torch.Tensor | None) -> torch.device:
    if not first.is_cuda:
        raise ValueError("okc_muse_kernels_b200 runs on CUDA tensors only (there is no CPU path)")
    dev = first.device
    for t in others:
        if t is not None and t.device != dev:
            raise ValueError(f"tensors on {dev} and {t.device}: all have to be on one device")
    return dev


def _call(fn, name: str, dev: torch.device, *args) -> None:
    """The C entry on the tensors' device (made current for the call if it is not) and its current stream."""
    if torch.cuda.current_device() == dev.index:
        rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    if rc:
        _lib.check(rc, name)


def _rows(t: torch.Tensor, what: str) -> torch.Tensor:
    if t.dim() != 2 or (t.dtype is not torch.bfloat16 and t.dtype is not torch.float32):
        raise ValueError(f"{what} must be bf16 or f32 [rows, columns]")
    if t.stride(1) != 1 or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


def _vector(t: torch.Tensor | None, n: int, what: str) -> torch.Tensor | None:
    if t is None:
        return None
    if t.dtype is not torch.float32 or t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{what} must be f32 [{n}]")
    return t.contiguous()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory from a's first to its last element touches b's."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    def span(t):
        n = sum((s - 1) * st for s, st in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (n + 1) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _out_rows(out: torch.Tensor | None, shape: tuple[int, int], dtype: torch.dtype, dev: torch.device, what: str, *inputs) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=dtype, device=dev)
    if tuple(out.shape) != shape or out.dtype != dtype or out.device != dev:
        raise ValueError(f"{what} must be {dtype} {list(shape)} on {dev}")
    if (shape[1] > 1 and out.stride(1) != 1) or (shape[0] > 1 and out.stride(0) < shape[1]):
        raise ValueError(f"{what} needs contiguous columns and rows that do not overlap")
    for t in inputs:
        if t is not None and _overlap(out, t):
            raise ValueError(f"{what} overlaps an input")
    return out


# ------------------------------------------------------------------------------------------------ int8 rows
def _empty_rows(rows: int, cols: int, dev: torch.device) -> torch.Tensor:
    pad = (cols + 15) // 16 * 16
    q = torch.empty((rows, pad), dtype=torch.int8, device=dev)
    return q if pad == cols else q[:, :cols]


def quantize_rows(x: torch.Tensor) -> QuantRows:
    """bf16 or f32 [R, C] -> int8 rows with a scale each.  With a = max|x| of a row: scale = a / 127 and
    q = rint(x * (127 / a)), halves to even, quotients and product in f32.  A row whose a is below 2**-120 becomes zeros
    with scale 0; a row that holds an infinity or a NaN becomes zeros with scale NaN, so that it makes NaN of every product.
    Weights are quantised with the same call once, a row per output channel.  C <= 131071."""
    x = _rows(x, "x")
    R, cols = x.shape
    if cols < 1 or cols > INT8_MAX_K:
        raise ValueError(f"rows of 1 to {INT8_MAX_K} columns, got {cols}")
    dev = _device(x)
    q = _empty_rows(R, cols, dev)
    scale = torch.empty(R, dtype=torch.float32, device=dev)
    if R:
        _call(_lib.lib().okc_moe_quantize_rows, "okc_moe_quantize_rows", dev, x.data_ptr(), _ROWS_KIND[x.dtype],
              max(x.stride(0), cols), R, cols, q.data_ptr(), max(q.stride(0), cols), scale.data_ptr())
    return QuantRows(q, scale)


def int8_rows(q: torch.Tensor, scale: torch.Tensor) -> QuantRows:
    """int8 [R, C] values and f32 [R] scales that come from elsewhere (a checkpoint), laid out as the products want them:
    rows 16 bytes aligned.  Once, at load time."""
    if q.dtype is not torch.int8 or q.dim() != 2 or scale.dtype is not torch.float32 or scale.shape != q.shape[:1]:
        raise ValueError("int8_rows wants int8 [R, C] and f32 [R]")
    dev = _device(q, scale)
    rows = _empty_rows(q.shape[0], q.shape[1], dev)
    rows.copy_(q)
    return QuantRows(rows, scale.contiguous())


def _check_quant(rows, what: str) -> tuple[torch.Tensor, torch.Tensor, int]:
    """The int8 tensor, its scales and the row stride to pass on."""
    q, scale = rows
    if q.dtype is not torch.int8 or q.dim() != 2 or scale.dtype is not torch.float32 or scale.dim() != 1 or scale.shape[0] != q.shape[0]:
        raise ValueError(f"{what} must be int8 [rows, columns] with f32 [rows] scales")
    R, cols = q.shape
    stride = q.stride(0)
    if R <= 1:
        stride = (cols + 15) // 16 * 16
    if (cols > 1 and q.stride(1) != 1) or stride < cols or stride % 16 or q.data_ptr() % 16:
        raise ValueError(f"{what} needs rows that start on 16-byte boundaries: lay them out with int8_rows() once")
    return q, scale.contiguous(), stride


def _product(fn, name: str, x, weight, bias, out_f32: bool, out, halves: int) -> torch.Tensor:
    w, w_scale, w_stride = _check_quant(weight, "weight")
    rows, K = w.shape
    if rows < halves or rows % halves:
        raise ValueError("a gated weight holds the gate rows and then as many up rows" if halves == 2 else "weight has no rows")
    N = rows // halves
    if isinstance(x, tuple):
        xt, x_scale, x_stride = _check_quant(x, "x")
    else:
        xt, x_scale = _rows(x, "x"), None
        x_stride = max(xt.stride(0), K)
    T = xt.shape[0]
    if xt.shape[1] != K or K < 1 or K > INT8_MAX_K:
        raise ValueError(f"x has {xt.shape[1]} columns and weight {K}; 1 to {INT8_MAX_K}, and as many in both")
    dev = _device(xt, x_scale, w, w_scale, bias, out)
    bias = _vector(bias, N, "bias")
    out = _out_rows(out, (T, N), torch.float32 if out_f32 else torch.bfloat16, dev, "out", xt, x_scale, w, w_scale, bias)
    if T == 0:
        return out
    lib = _lib.lib()
    kind = _ROWS_KIND[xt.dtype]
    n = lib.okc_moe_int8_scratch_bytes(kind, T, K)
    scratch = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    _call(getattr(lib, fn), name, dev, Int8Args(
        xt.data_ptr(), None if x_scale is None else x_scale.data_ptr(), w.data_ptr(), w_scale.data_ptr(),
        None if bias is None else bias.data_ptr(), out.data_ptr(), None if scratch is None else scratch.data_ptr(),
        x_stride, w_stride, max(out.stride(0), N), kind, int(out_f32), T, K, N))
    return out


def int8_linear(x, weight, *, bias: torch.Tensor | None = None, out_f32: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight.T`` in 8-bit integers: bf16 [T, N] (f32 with ``out_f32``).

    ``weight``: ``QuantRows`` (or a tuple) int8 [N, K] and f32 [N], one scale per output channel.  ``x``: bf16 or f32
    [T, K], quantised a row at a time as ``quantize_rows`` does, or ``QuantRows`` [T, K].  ``bias`` f32 [N].
    y[t, n] = (sum_k x.q[t, k] * weight.q[n, k]) * (x.scale[t] * weight.scale[n]) + bias[n]; the sum is exact, the rest is
    f32 and rounded once, so a token's bits do not depend on the other tokens of the call.  T may be 0; K <= 131071.
    ``out``: a tensor to write, which may not overlap an input."""
    return _product("okc_moe_int8_linear", "okc_moe_int8_linear", x, weight, bias, out_f32, out, 1)


def int8_gated(x, weight, *, out_f32: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """The first half of a gated feed-forward in one kernel: ``silu(x @ gate.T) * (x @ up.T)`` -> bf16 [T, I].

    ``weight``: int8 [2 I, K] and f32 [2 I], the gate rows first (the order of the experts' ``w13``).  Otherwise as
    ``int8_linear``."""
    return _product("okc_moe_int8_gated", "okc_moe_int8_gated", x, weight, None, out_f32, out, 2)


def int8_ffn(x, w13, w2, *, bias: torch.Tensor | None = None, out_f32: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """A dense gated feed-forward, the block of a layer without experts (or a shared expert held in 8 bits):
    ``int8_linear(int8_gated(x, w13), w2)``; the activations between the two products are bf16."""
    return int8_linear(int8_gated(x, w13), w2, bias=bias, out_f32=out_f32, out=out)


def int8_status() -> tuple[int, int]:
    """(status, detail) of the int8 products on the current device since the last call: (0, 0), or (OKC_ERR_TIMEOUT, code)
    when a bounded device wait ran out.  Synchronises the current stream."""
    detail = C.c_int32(0)
    rc = _lib.lib().okc_moe_int8_status(torch.cuda.current_stream().cuda_stream, C.byref(detail))
    return rc, detail.value


# ------------------------------------------------------------------------------------------------ norms
def block_norm(residual: torch.Tensor, block: torch.Tensor | None = None, *, post_gain: torch.Tensor | None = None,
               gate: torch.Tensor | None = None, gate_sigmoid: bool = False, residual_scale: float = 1.0,
               block_scale: float = 1.0, pre_gain: torch.Tensor | None = None, eps: float = 1e-5, out: str = "bf16",
               residual_out: torch.Tensor | None = None):
    """The residual stream behind a block and the input of the next one, in one kernel.  Returns ``(r', x)``:

        z  = block * rsqrt(mean(block**2) + eps) * post_gain     (``post_gain`` None: z = block)
        r' = residual_scale * residual + block_scale * g * z     (g = ``gate``, or its sigmoid with ``gate_sigmoid``)
        x  = r' * rsqrt(mean(r'**2) + eps) * pre_gain            (``pre_gain`` None: x is None)

    ``residual`` and ``block``: bf16 or f32 [T, H], each in its own type; ``r'`` has the residual's type, and
    ``residual_out=residual`` updates the stream in place.  Gains f32 [H] (a layer that stores w passes 1 + w).  ``gate``
    bf16 or f32: [H] (or [1, H]) per channel, [T, 1] per token, [T, H] per element.  ``out``: the type of x, "bf16", "f32"
    or "int8" (``QuantRows``, quantised as ``quantize_rows`` does, ready for ``int8_linear``).  All arithmetic is f32; x is
    made from r' before its rounding.  ``block`` None: the norm before a first block alone, r' is ``residual`` itself.
    H <= 16384; T may be 0."""
    if out not in _OUT:
        raise ValueError('out is "bf16", "f32" or "int8"')
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    res = _rows(residual, "residual")
    T, H = res.shape
    if H < 1 or H > BLOCK_NORM_MAX_HIDDEN:
        raise ValueError(f"rows of 1 to {BLOCK_NORM_MAX_HIDDEN} columns, got {H}")
    dev = _device(res, block, post_gain, gate, pre_gain, residual_out)
    post_gain, pre_gain = _vector(post_gain, H, "post_gain"), _vector(pre_gain, H, "pre_gain")
    kind, gate_stride = 0, 0
    if block is None:
        if post_gain is not None or gate is not None or residual_out is not None or residual_scale != 1.0 or block_scale != 1.0:
            raise ValueError("post_gain, gate, residual_out and the scales belong to a block's output")
        if pre_gain is None:
            raise ValueError("nothing to do: neither block nor pre_gain is given")
        new, blk = residual, None
    else:
        blk = _rows(block, "block")
        if blk.shape != res.shape:
            raise ValueError(f"block must be [{T}, {H}] like residual")
        if gate is not None:
            if gate.dtype is not torch.bfloat16 and gate.dtype is not torch.float32:
                raise ValueError("gate must be bf16 or f32")
            shape = tuple(gate.shape)
            if shape == (H,) or shape == (1, H):
                kind = 1
            elif shape == (T, 1):
                kind = 2
            elif shape == (T, H):
                kind = 3
            else:
                raise ValueError(f"gate must be [{H}], [{T}, 1] or [{T}, {H}]")
            if kind != 2 and H > 1 and gate.stride(-1) != 1 or kind == 3 and T > 1 and gate.stride(0) < H:
                gate = gate.contiguous()
            if kind != 1:
                gate_stride = gate.stride(0)
        # a thread reads its elements of every tensor before it writes r': the same memory element for element is fine
        apart = (t for t in (res, blk, gate, post_gain, pre_gain) if t is not None and not (
            residual_out is not None and t.data_ptr() == residual_out.data_ptr() and t.dtype == residual_out.dtype
            and t.shape == residual_out.shape and t.stride() == residual_out.stride()))
        new = _out_rows(residual_out, (T, H), res.dtype, dev, "residual_out", *apart)
    x = scale = None
    code, dtype = _OUT[out]
    if pre_gain is not None:
        if code == 2:
            x, scale = _empty_rows(T, H, dev), torch.empty(T, dtype=torch.float32, device=dev)
        else:
            x = torch.empty((T, H), dtype=dtype, device=dev)
    if T:
        f32 = torch.float32
        _call(_lib.lib().okc_moe_block_norm, "okc_moe_block_norm", dev, BlockNormArgs(
            res.data_ptr(), None if blk is None else blk.data_ptr(), gate.data_ptr() if kind else None,
            None if post_gain is None else post_gain.data_ptr(), None if pre_gain is None else pre_gain.data_ptr(),
            None if blk is None else new.data_ptr(), None if x is None else x.data_ptr(), None if scale is None else scale.data_ptr(),
            T, max(res.stride(0), H), H if blk is None else max(blk.stride(0), H), gate_stride, max(new.stride(0), H),
            H if x is None else max(x.stride(0), H), H, res.dtype is f32, blk is not None and blk.dtype is f32,
            kind != 0 and gate.dtype is f32, kind, gate_sigmoid, code, residual_scale, block_scale, eps))
    return new, (QuantRows(x, scale) if scale is not None else x)
