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
from ._lib import pack_block_norm as _pack_block_norm, pack_int8 as _pack_int8

__all__ = ["QuantRows", "quantize_rows", "int8_rows", "int8_linear", "int8_gated", "int8_ffn", "block_norm", "dense_status"]

BLOCK_NORM_MAX_HIDDEN = 16384
INT8_MAX_K = 131071           # the integer sums stay in 32 bits
MAX_ROWS = (1 << 31) - 1      # rows of a call
INT8_MAX_ROWS = 1 << 30       # tokens, and outputs, of a product
INT8_ONE_MAX_K = 16384        # up to here the product of one token quantises it itself and needs no scratch
_BF16, _F32, _I8 = torch.bfloat16, torch.float32, torch.int8
_ROWS_KIND = {_BF16: 0, _F32: 1, _I8: 2}
_OUT = {"bf16": (0, _BF16), "f32": (1, _F32), "int8": (2, _I8)}


class QuantRows(NamedTuple):
    """Rows of int8 values and what they stand for: row r is ``q[r] * scale[r]``.  ``q`` int8 [R, C] with rows 16 bytes
    aligned, ``scale`` f32 [R]."""
    q: torch.Tensor
    scale: torch.Tensor


# A decode step makes these calls by the hundred and its kernels take a few microseconds, so the checks below are written
# to cost little: each property is read once, and what can be compared as an integer is.
def _device(first: torch.Tensor, *others: torch.Tensor | None) -> int:
    """The index of the CUDA device that all tensors are on."""
    dev = first.get_device()
    if dev < 0:
        raise ValueError("okc_muse_kernels_b200 runs on CUDA tensors only (there is no CPU path)")
    for t in others:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"tensors on {first.device} and {t.device}: all have to be on one device")
    return dev


_empty = torch.empty_strided                         # the cheapest of torch's ways to uninitialised memory
# A torch without CUDA lacks the names below.  The package imports all the same (the layouts and synthetic weights need no
# GPU), and no call gets to them: each refuses tensors that are not on a CUDA device first.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)     # the current stream of a device as an integer
_current_device = getattr(torch._C, "_cuda_getDevice", None)           # (a CUDA tensor is at hand: CUDA is initialised)
# Memory of torch's caching allocator without a tensor around it (0.5 us, an empty tensor 1.5): on the current device, for
# work on the given stream; after the free it goes to later work on that stream, as a tensor's would.
_alloc = getattr(torch._C, "_cuda_cudaCachingAllocator_raw_alloc", None)
_free = getattr(torch._C, "_cuda_cudaCachingAllocator_raw_delete", None)


def _call(fn, name: str, dev: int, args) -> None:
    """The C entry on the tensors' device (made current for the call if it is not) and its current stream."""
    if _current_device() == dev:
        rc = fn(args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(args, _raw_stream(dev))
    if rc:
        _lib.check(rc, name)


def _rows(t: torch.Tensor, what: str) -> tuple[torch.Tensor, int, int, int]:
    """bf16 or f32 rows with contiguous columns (a copy if need be): tensor, rows, columns, row stride."""
    dtype = t.dtype
    if (dtype is not _BF16 and dtype is not _F32) or t.dim() != 2:
        raise ValueError(f"{what} must be bf16 or f32 [rows, columns]")
    R, cols = t.shape
    stride, one = t.stride()
    if one != 1 or stride < cols:
        if R > 1 or (one != 1 and cols > 1):
            t = t.contiguous()
        stride = cols
    return t, R, cols, stride


def _vector(t: torch.Tensor | None, n: int, what: str) -> torch.Tensor | None:
    if t is None:
        return None
    if t.dtype is not _F32 or t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{what} must be f32 [{n}]")
    return t if t.is_contiguous() else t.contiguous()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory from a's first to its last element touches b's; of rows that are equally far apart, whether the
    rows themselves do (columns side by side in one buffer do not)."""
    if a.data_ptr() > b.data_ptr():
        a, b = b, a
    gap = b.data_ptr() - a.data_ptr()
    if gap >= a.untyped_storage().nbytes() or not a.numel() or not b.numel():
        return False
    if gap >= (1 + sum((n - 1) * st for n, st in zip(a.shape, a.stride()))) * a.element_size():
        return False
    (rows_a, apart_a, len_a), (rows_b, apart_b, len_b) = _row_bytes(a), _row_bytes(b)
    apart = apart_a if rows_a > 1 else apart_b
    if rows_a == rows_b == 1 or (rows_a > 1 and rows_b > 1 and apart_a != apart_b) or apart <= 0:
        return True
    return gap % apart < len_a or gap % apart + len_b > apart


def _row_bytes(t: torch.Tensor) -> tuple[int, int, int]:
    """Rows, how many bytes they are apart, and the bytes from a row's first to its last column."""
    size = t.element_size()
    if t.dim() != 2:
        return 1, 0, (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride()))) * size
    return t.shape[0], t.stride(0) * size, (1 + (t.shape[1] - 1) * t.stride(1)) * size


def _check_out(out: torch.Tensor, R: int, cols: int, dtype: torch.dtype, what: str, inputs) -> int:
    """Checks a caller's output rows; returns their stride."""
    if tuple(out.shape) != (R, cols) or out.dtype is not dtype:
        raise ValueError(f"{what} must be {dtype} [{R}, {cols}]")
    stride, one = out.stride()
    if (cols > 1 and one != 1) or (R > 1 and stride < cols):
        raise ValueError(f"{what} needs contiguous columns and rows that do not overlap")
    for t in inputs:
        if t is not None and _overlap(out, t):
            raise ValueError(f"{what} overlaps an input")
    return max(stride, cols)


# ------------------------------------------------------------------------------------------------ int8 rows
def _empty_rows(like: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    pad = (cols + 15) // 16 * 16
    q = _empty((rows, pad), (pad, 1), dtype=_I8, device=like.device)
    return q if pad == cols else q[:, :cols]


def quantize_rows(x: torch.Tensor) -> QuantRows:
    """bf16 or f32 [R, C] -> int8 rows with a scale each.  With a = max|x| of a row: scale = a / 127 and
    q = rint(x * (127 / a)), halves to even, quotients and product in f32.  A row whose a is below 2**-120 becomes zeros
    with scale 0; a row that holds an infinity or a NaN becomes zeros with scale NaN, so that it makes NaN of every product.
    Weights are quantised with the same call once, a row per output channel.  C <= 131071."""
    x, R, cols, stride = _rows(x, "x")
    if cols < 1 or cols > INT8_MAX_K:
        raise ValueError(f"rows of 1 to {INT8_MAX_K} columns, got {cols}")
    if R > MAX_ROWS:
        raise ValueError(f"at most {MAX_ROWS} rows, got {R}")
    dev = _device(x)
    q = _empty_rows(x, R, cols)
    scale = _empty((R,), (1,), dtype=_F32, device=x.device)
    if R:
        args = x.data_ptr(), _ROWS_KIND[x.dtype], stride, R, cols, q.data_ptr(), max(q.stride(0), cols), scale.data_ptr()
        _call(lambda a, stream: _lib.lib().okc_moe_quantize_rows(*a, stream), "okc_moe_quantize_rows", dev, args)
    return QuantRows(q, scale)


def int8_rows(q: torch.Tensor, scale: torch.Tensor) -> QuantRows:
    """int8 [R, C] values and f32 [R] scales that come from elsewhere (a checkpoint), laid out as the products want them:
    rows 16 bytes aligned.  Once, at load time."""
    if q.dtype is not torch.int8 or q.dim() != 2 or scale.dtype is not torch.float32 or scale.shape != q.shape[:1]:
        raise ValueError("int8_rows wants int8 [R, C] and f32 [R]")
    _device(q, scale)
    rows = _empty_rows(q, *q.shape)
    rows.copy_(q)
    return QuantRows(rows, scale.contiguous())


def _check_quant(rows, what: str) -> tuple:
    """int8 tensor, its device, address, rows, columns and row stride to pass on, scales, their address."""
    q, scale = rows
    try:
        R, cols = q.shape
        n, = scale.shape
        ok = n == R and q.dtype is _I8 and scale.dtype is _F32
    except ValueError:
        ok = False
    if not ok:
        raise ValueError(f"{what} must be int8 [rows, columns] with f32 [rows] scales")
    stride, one = q.stride()
    if R <= 1:
        stride = cols + 15 & -16
    ptr = q.data_ptr()
    if (one != 1 and cols > 1) or stride < cols or (stride | ptr) & 15:
        raise ValueError(f"{what} needs rows that start on 16-byte boundaries: lay them out with int8_rows() once")
    dev = q.get_device()
    if scale.get_device() != dev:
        raise ValueError(f"{what}: int8 values on {q.device} and scales on {scale.device}")
    if not scale.is_contiguous():
        scale = scale.contiguous()
    return q, dev, ptr, R, cols, stride, scale, scale.data_ptr()


def _product(name: str, x, weight, bias, out_f32: bool, out, halves: int) -> torch.Tensor:
    w, dev, w_ptr, N, K, w_stride, w_scale, ws_ptr = _check_quant(weight, "weight")
    if N < halves or N % halves:
        raise ValueError("a gated weight holds the gate rows and then as many up rows" if halves == 2 else "weight has no rows")
    N //= halves
    if isinstance(x, tuple):
        x, x_dev, x_ptr, T, cols, x_stride, x_scale, xs_ptr = _check_quant(x, "x")
        kind, scratch = 2, 0
    else:
        x, T, cols, x_stride = _rows(x, "x")
        x_dev, x_ptr, kind, x_scale, xs_ptr, scratch = x.get_device(), x.data_ptr(), _ROWS_KIND[x.dtype], None, 0, T > 1 or K > INT8_ONE_MAX_K
    if cols != K or K < 1 or K > INT8_MAX_K:
        raise ValueError(f"x has {cols} columns and weight {K}; 1 to {INT8_MAX_K}, and as many in both")
    if T > INT8_MAX_ROWS or N > INT8_MAX_ROWS:
        raise ValueError(f"at most {INT8_MAX_ROWS} tokens and outputs, got {T} and {N}")
    if x_dev != dev or dev < 0 or bias is not None or out is not None:
        _device(x, w, bias, out)
    device, bias_ptr = x.device, 0
    if bias is not None:
        bias = _vector(bias, N, "bias")
        bias_ptr = bias.data_ptr()
    if out is None:
        out, out_stride = _empty((T, N), (N, 1), dtype=_F32 if out_f32 else _BF16, device=device), N
    else:
        out_stride = _check_out(out, T, N, _F32 if out_f32 else _BF16, "out", (x, x_scale, w, w_scale, bias))
    if T == 0:
        return out
    if scratch and _current_device() != dev:
        with torch.cuda.device(dev):
            return _product(name, x, weight, bias, out_f32, out, halves)
    fn, scratch_ptr = getattr(_lib.lib(), name), 0
    if scratch:      # int8 rows and scales of the tokens, for the call alone: okc_moe_int8_scratch_bytes
        scratch_ptr = _alloc(T * ((K + 15 & -16) + 4), _raw_stream(dev))
    try:
        _call(fn, name, dev, _pack_int8(
            x_ptr, xs_ptr, w_ptr, ws_ptr, bias_ptr, out.data_ptr(), scratch_ptr, x_stride, w_stride, out_stride, kind, out_f32, T, K, N))
    finally:
        if scratch_ptr:
            _free(scratch_ptr)
    return out


def int8_linear(x, weight, *, bias: torch.Tensor | None = None, out_f32: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight.T`` in 8-bit integers: bf16 [T, N] (f32 with ``out_f32``).

    ``weight``: ``QuantRows`` (or a tuple) int8 [N, K] and f32 [N], one scale per output channel.  ``x``: bf16 or f32
    [T, K], quantised a row at a time as ``quantize_rows`` does, or ``QuantRows`` [T, K].  ``bias`` f32 [N].
    y[t, n] = (sum_k x.q[t, k] * weight.q[n, k]) * (x.scale[t] * weight.scale[n]) + bias[n]; the sum is exact, the rest is
    f32 and rounded once, so a token's bits do not depend on the other tokens of the call.  T may be 0; K <= 131071.
    ``out``: a tensor to write, which may not overlap an input."""
    return _product("okc_moe_int8_linear", x, weight, bias, out_f32, out, 1)


def int8_gated(x, weight, *, out_f32: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """The first half of a gated feed-forward in one kernel: ``silu(x @ gate.T) * (x @ up.T)`` -> bf16 [T, I].

    ``weight``: int8 [2 I, K] and f32 [2 I], the gate rows first (the order of the experts' ``w13``).  Otherwise as
    ``int8_linear``."""
    return _product("okc_moe_int8_gated", x, weight, None, out_f32, out, 2)


def int8_ffn(x, w13, w2, *, bias: torch.Tensor | None = None, out_f32: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """A dense gated feed-forward, the block of a layer without experts (or a shared expert held in 8 bits):
    ``int8_linear(int8_gated(x, w13), w2)``; the activations between the two products are bf16."""
    return int8_linear(int8_gated(x, w13), w2, bias=bias, out_f32=out_f32, out=out)


def dense_status() -> tuple[int, int]:
    """(status, detail) of this module's operators on the current device since the last report: (0, 0), or (OKC_ERR_TIMEOUT, code)
    when a bounded device wait ran out (a product's first; a norm's is reported by the next call).  Synchronises the current
    stream."""
    detail = C.c_int32(0)
    rc = _lib.lib().okc_moe_dense_status(torch.cuda.current_stream().cuda_stream, C.byref(detail))
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
    A row's result depends on that row alone, but the order of its sums goes by the number of rows and their alignment, so
    its last bits may differ between batches of different sizes.  H <= 16384; T may be 0."""
    new, x, dev, args, held = check_norm(residual, block, post_gain, gate, gate_sigmoid, residual_scale, block_scale, pre_gain, eps, out, residual_out)
    if args is not None:
        _call(_lib.lib().okc_moe_block_norm, "okc_moe_block_norm", dev, args)
    return new, x


def check_norm(residual, block, post_gain, gate, gate_sigmoid, residual_scale, block_scale, pre_gain, eps, out, residual_out) -> tuple:
    """``block_norm`` up to its launch: its two results, the device, the arguments of the C entry (None without rows), and the
    tensors that they point into."""
    if out not in _OUT:
        raise ValueError('out is "bf16", "f32" or "int8"')
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    res, T, H, res_stride = _rows(residual, "residual")
    if H < 1 or H > BLOCK_NORM_MAX_HIDDEN:
        raise ValueError(f"rows of 1 to {BLOCK_NORM_MAX_HIDDEN} columns, got {H}")
    if T > MAX_ROWS:
        raise ValueError(f"at most {MAX_ROWS} rows, got {T}")
    dev = _device(res, block, post_gain, gate, pre_gain, residual_out)
    post_gain, pre_gain = _vector(post_gain, H, "post_gain"), _vector(pre_gain, H, "pre_gain")
    dtype = res.dtype
    blk = None
    kind = gate_stride = gate_f32 = blk_stride = new_stride = blk_ptr = blk_f32 = 0
    if block is None:
        if post_gain is not None or gate is not None or residual_out is not None or residual_scale != 1.0 or block_scale != 1.0:
            raise ValueError("post_gain, gate, residual_out and the scales belong to a block's output")
        if pre_gain is None:
            raise ValueError("nothing to do: neither block nor pre_gain is given")
        new = residual
    else:
        blk, rows, cols, blk_stride = _rows(block, "block")
        if rows != T or cols != H:
            raise ValueError(f"block must be [{T}, {H}] like residual")
        blk_ptr, blk_f32 = blk.data_ptr(), blk.dtype is _F32
        if gate is not None:
            gate, kind, gate_stride = _gate(gate, T, H)
            gate_f32 = gate.dtype is _F32
        if residual_out is None:
            new, new_stride = _empty((T, H), (H, 1), dtype=dtype, device=res.device), H
        else:
            # a thread reads its elements of every tensor before it writes r': the same memory element for element is fine
            new, new_stride = residual_out, _check_out(residual_out, T, H, dtype, "residual_out", (
                t for t in (res, blk, gate, post_gain, pre_gain) if t is not None and not (
                    t.data_ptr() == residual_out.data_ptr() and t.dtype is dtype and t.shape == residual_out.shape
                    and t.stride() == residual_out.stride())))
    x = scale = None
    x_stride = 0
    code, kind_of_x = _OUT[out]
    if pre_gain is not None:
        if code == 2:
            x, scale = _empty_rows(res, T, H), _empty((T,), (1,), dtype=_F32, device=res.device)
            x_stride = max(x.stride(0), H)
        else:
            x, x_stride = _empty((T, H), (H, 1), dtype=kind_of_x, device=res.device), H
    args = None
    if T:
        args = _pack_block_norm(
            res.data_ptr(), blk_ptr, gate.data_ptr() if kind else 0,
            0 if post_gain is None else post_gain.data_ptr(), 0 if pre_gain is None else pre_gain.data_ptr(),
            new.data_ptr() if blk_ptr else 0, 0 if x is None else x.data_ptr(), 0 if scale is None else scale.data_ptr(),
            T, res_stride, blk_stride, gate_stride, new_stride, x_stride, H, dtype is _F32, blk_f32, gate_f32, kind,
            bool(gate_sigmoid), code, residual_scale, block_scale, eps)
    return new, x if scale is None else QuantRows(x, scale), dev, args, (res, blk, gate, post_gain, pre_gain)


def launch_norm(norm: tuple) -> tuple:
    """Launches what ``check_norm`` returned; returns its results."""
    new, x, dev, args, _ = norm
    if args is not None:
        _call(_lib.lib().okc_moe_block_norm, "okc_moe_block_norm", dev, args)
    return new, x


def _gate(gate: torch.Tensor, T: int, H: int) -> tuple[torch.Tensor, int, int]:
    """A gate with contiguous columns, its kind (1 per channel, 2 per token, 3 per element) and its row stride."""
    if gate.dtype is not _BF16 and gate.dtype is not _F32:
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
    if (kind != 2 and H > 1 and gate.stride(-1) != 1) or (kind == 3 and T > 1 and gate.stride(0) < H):
        gate = gate.contiguous()
    return gate, kind, 0 if kind == 1 else gate.stride(0)
