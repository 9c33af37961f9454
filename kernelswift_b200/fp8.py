"""Dense block-scaled fp8 for the layers around the routed experts: the
quantisers, the product of e4m3 matrices with one scale per 128 columns of a
row and per 128x128 block of the weights, and the SwiGLU MLP that chains them
(the shared expert of an MoE layer).

Formats: scale_format "fp32" (scale = absmax / 448) or "ue8m0" (uint8 bytes b
meaning the power of two 2^(b - 127), applied by the tensor core). A scale
tensor's dtype says which it is. The grouped GEMMs of fused_moe take the same
formats per expert.

Everything runs in libmoe_b200.so on the current stream of the operands'
device; nothing allocates but the outputs, and a call can be captured in a
CUDA graph. There is no CPU path and no gradient: these are serving operators.
Activations, scales, addends and outputs that need one are refused (e4m3 operands
and the weights of quantize_blocks are taken as constants), and so is anything that
carries a tangent.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd import forward_ad

from . import _lib
from .fused_moe import _check_cuda, _DTYPE_CODE, _enqueue, _refuse_tangents

_FORMAT = {"fp32": 0, "ue8m0": 1}
_SCALE_FORMAT = {torch.float32: 0, torch.uint8: 1}
_FLOAT = (torch.float32, torch.float16, torch.bfloat16)
_FLOAT_CODE = {t: _DTYPE_CODE[t] for t in _FLOAT}


def _round_up(n: int, m: int) -> int:
    return -(-n // m) * m


def _empty_fp8(rows: int, cols: int, device) -> torch.Tensor:
    """[rows, cols] e4m3 whose rows start on 16-byte boundaries."""
    q = torch.empty(rows, _round_up(cols, 16), dtype=torch.float8_e4m3fn, device=device)
    return q if cols % 16 == 0 else q[:, :cols]


def _no_grad_needed(name: str, t: torch.Tensor) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient; the fp8 operators have none "
                         "(call them under torch.no_grad())")


def _rows_of(t: torch.Tensor) -> torch.Tensor:
    """A 2-D tensor whose rows are dense: `t`, or a dense copy."""
    pitch, step = t.stride()
    if step == 1 and pitch >= t.shape[1] or t.numel() == 0:
        return t
    return t.contiguous()


def _fp8_rows(name: str, t: torch.Tensor) -> torch.Tensor:
    """An e4m3 matrix whose rows start on 16-byte boundaries: `t`, or a copy
    with its row pitch padded."""
    if t.dtype != torch.float8_e4m3fn or t.dim() != 2:
        raise ValueError(f"{name} must be a 2-D float8_e4m3fn tensor")
    rows, cols = t.shape
    pitch, step = t.stride()
    if step == 1 and pitch % 16 == 0 and pitch >= cols and t.data_ptr() % 16 == 0:
        return t
    q = _empty_fp8(rows, cols, t.device)
    q.view(torch.uint8).copy_(t.view(torch.uint8))
    return q


def _check_out(out: torch.Tensor, rows: int, cols: int, dtype: torch.dtype, index: int) -> None:
    if (out.shape != (rows, cols) or out.get_device() != index or out.dtype != dtype
            or dtype not in _FLOAT or out.stride(1) != 1 and cols > 1
            or out.stride(0) < cols and rows > 1):
        raise ValueError(f"out must be a bf16, f16 or f32 [{rows}, {cols}] tensor with dense rows "
                         "on the operands' device")
    _no_grad_needed("out", out)


def _addend(addend: torch.Tensor, rows: int, cols: int, dtype: torch.dtype, index: int,
            out: torch.Tensor | None):
    """(pointer, row stride) of the addend; `out` where the caller gave one."""
    _no_grad_needed("addend", addend)
    if addend.shape != (rows, cols) or addend.dtype != dtype or addend.get_device() != index:
        raise ValueError(f"addend must be a {dtype} [{rows}, {cols}] tensor on the operands' "
                         "device")
    if addend.numel() and (addend.stride(1) != 1 and cols > 1
                           or addend.stride(0) < cols and rows > 1):
        raise ValueError("addend must have dense rows")
    if out is not None:
        _check_apart(out, addend)
    return addend.data_ptr(), max(addend.stride(0), cols)


def _check_apart(out: torch.Tensor, addend: torch.Tensor) -> None:
    """out and addend are the same elements or share none: an element is read by
    the thread that writes it, and only just before. Strides of a single row or
    column mean nothing."""
    size, (rows, cols) = out.element_size(), out.shape
    apart = (addend.data_ptr() - out.data_ptr()) // size
    pitch, add_pitch = (out.stride(0), addend.stride(0)) if rows > 1 else (cols, cols)
    if not out.numel() or apart == 0 and pitch == add_pitch:
        return
    if apart >= (rows - 1) * pitch + cols or -apart >= (rows - 1) * add_pitch + cols:
        return
    # columns of one wider matrix
    if add_pitch == pitch and cols <= apart % pitch <= pitch - cols:
        return
    raise ValueError("out and addend overlap without being the same elements")


def _status_ptr(status: torch.Tensor | None, index: int) -> int | None:
    if status is None:
        return None
    if status.dtype != torch.int32 or status.get_device() != index or status.numel() < 1:
        raise ValueError("status must be an int32 tensor on the operands' device")
    return status.data_ptr()


def quantize_rows(x: torch.Tensor, scale_format: str = "ue8m0", gated: bool = False
                  ) -> tuple[torch.Tensor, torch.Tensor]:
    """Quantises x [T, K] (f32/f16/bf16) to e4m3 with one scale per row and
    128 columns (moe_fp8_quantize_rows). gated: x is [T, 2K], gate then up, and
    silu(gate) * up [T, K] is quantised. Returns (q float8_e4m3fn [T, K], scale
    [T, ceil(K / 128)], float32 or uint8), the operands of block_matmul: views
    whose row pitch is padded to 16 bytes (q) and 4 (scale bytes); fp32 scales
    lie column by column."""
    index = x.get_device()
    if index < 0:
        _check_cuda("x", x)
    fmt = _FORMAT.get(scale_format)
    if fmt is None:
        raise ValueError(f"scale_format must be one of {sorted(_FORMAT)}")
    code = _FLOAT_CODE.get(x.dtype)
    if x.dim() != 2 or code is None or (gated and x.shape[1] % 2):
        raise ValueError("x must be a 2-D f32/f16/bf16 tensor, of an even width when gated")
    if x.requires_grad:
        _no_grad_needed("x", x)
    if forward_ad._current_level >= 0:
        _refuse_tangents(x=x)
    x = _rows_of(x)
    T, wide = x.shape
    K = wide // 2 if gated else wide
    if K < 1:
        raise ValueError("x has no columns")
    dev, kb = x.device, (K + 127) // 128
    q = _empty_fp8(T, K, dev)
    if fmt == 0:
        strides, dtype = (1, (T + 3) // 4 * 4), torch.float32
    else:
        strides, dtype = ((kb + 3) // 4 * 4, 1), torch.uint8
    scale = torch.empty_strided((T, kb), strides, dtype=dtype, device=dev)
    _enqueue("moe_fp8_quantize_rows", index, x.data_ptr(), code, T, K, max(x.stride(0), wide),
             gated, fmt, q.data_ptr(), (K + 15) // 16 * 16, scale.data_ptr(), *strides)
    return q, scale


def quantize_blocks(w: torch.Tensor, scale_format: str = "ue8m0"
                    ) -> tuple[torch.Tensor, torch.Tensor]:
    """Quantises weights w [N, K] (f32/f16/bf16) to e4m3 with one scale per
    128x128 block (moe_fp8_quantize_blocks), once per weight version. Returns
    (q float8_e4m3fn [N, K] of a row pitch padded to 16 bytes, scale
    [ceil(N / 128), ceil(K / 128)], float32 or uint8)."""
    _check_cuda("w", w)
    if scale_format not in _FORMAT:
        raise ValueError(f"scale_format must be one of {sorted(_FORMAT)}")
    if w.dim() != 2 or w.dtype not in _FLOAT or w.numel() == 0:
        raise ValueError("w must be a 2-D f32/f16/bf16 tensor")
    if forward_ad._current_level >= 0:
        _refuse_tangents(w=w)
    w = _rows_of(w.detach())
    N, K = w.shape
    dev = w.device
    q = _empty_fp8(N, K, dev)
    scale = torch.empty(-(-N // 128), -(-K // 128), device=dev,
                        dtype=torch.float32 if scale_format == "fp32" else torch.uint8)
    _enqueue("moe_fp8_quantize_blocks", w.get_device(), w.data_ptr(), _DTYPE_CODE[w.dtype], N, K,
             max(w.stride(0), K), _FORMAT[scale_format], q.data_ptr(), _round_up(K, 16),
             scale.data_ptr())
    return q, scale


def block_matmul(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                 out_dtype: torch.dtype = torch.bfloat16, addend: torch.Tensor | None = None,
                 out: torch.Tensor | None = None, status: torch.Tensor | None = None
                 ) -> torch.Tensor:
    """out [T, N] = x w^T (+ addend) for block-scaled e4m3 operands
    (moe_fp8_matmul).

    x float8_e4m3fn [T, K] with x_scale [T, ceil(K / 128)], w [N, K] with
    w_scale [ceil(N / 128), ceil(K / 128)]; both scales float32 or both uint8
    (UE8M0). Rows that do not start on 16-byte boundaries are copied first
    (quantize_rows and quantize_blocks pad them). addend [T, N] has out's
    dtype and may be out itself. Summed in fp32, rounded once to out_dtype
    (bf16, f16 or f32; out's own dtype where it is given). status: optional
    int32 device word (moe_read_status).
    """
    index = x.get_device()
    if not index == w.get_device() == x_scale.get_device() == w_scale.get_device() or index < 0:
        for name, t in (("x", x), ("x_scale", x_scale), ("w", w), ("w_scale", w_scale)):
            _check_cuda(name, t)
        raise ValueError("x, x_scale, w and w_scale must be on one device")
    if forward_ad._current_level >= 0:
        _refuse_tangents(x=x, x_scale=x_scale, w=w, w_scale=w_scale, addend=addend, out=out)
    x, w = _fp8_rows("x", x), _fp8_rows("w", w)
    (T, K), (N, w_cols) = x.shape, w.shape
    kb, nb = (K + 127) // 128, (N + 127) // 128
    if w_cols != K or K < 1 or N < 1:
        raise ValueError(f"w {tuple(w.shape)} does not match x {tuple(x.shape)}")
    fmt = _SCALE_FORMAT.get(x_scale.dtype)
    if fmt is None or w_scale.dtype != x_scale.dtype:
        raise ValueError("x_scale and w_scale must both be float32 or both uint8 (UE8M0)")
    if x_scale.shape != (T, kb) or w_scale.shape != (nb, kb):
        raise ValueError(f"scales must be [{T}, {kb}] and [{nb}, {kb}], got "
                         f"{tuple(x_scale.shape)} and {tuple(w_scale.shape)}")
    if out is not None:
        out_dtype = out.dtype
        _check_out(out, T, N, out_dtype, index)
    elif out_dtype not in _FLOAT_CODE:
        raise ValueError("out_dtype must be bf16, f16 or f32")
    add_ptr, add_ld = (None, 0) if addend is None else _addend(addend, T, N, out_dtype, index, out)
    if out is None:
        out, ld_out = torch.empty(T, N, dtype=out_dtype, device=x.device), N
    else:
        ld_out = max(out.stride(0), N)
    if x_scale.requires_grad or w_scale.requires_grad:
        _no_grad_needed("x_scale", x_scale)
        _no_grad_needed("w_scale", w_scale)
    if not w_scale.is_contiguous():
        w_scale = w_scale.contiguous()
    pitch = (K + 15) // 16 * 16
    _enqueue("moe_fp8_matmul", index, x.data_ptr(), max(x.stride(0), pitch), x_scale.data_ptr(),
             *x_scale.stride(), w.data_ptr(), max(w.stride(0), pitch), w_scale.data_ptr(), fmt, T,
             N, K, add_ptr, add_ld, out.data_ptr(), ld_out, _FLOAT_CODE[out_dtype],
             _status_ptr(status, index))
    return out


def block_matmul_plan(num_rows: int, out_cols: int, inner: int, scale_format: str = "ue8m0"
                      ) -> dict:
    """How block_matmul runs these sizes (moe_fp8_matmul_plan; no GPU needed)."""
    info = (ctypes.c_int32 * 4)()
    _lib.call("moe_fp8_matmul_plan", num_rows, out_cols, inner, _FORMAT[scale_format], info)
    return dict(zip(("cta_pairs", "tile_cols", "splits", "ctas"), list(info)))


@functools.lru_cache(maxsize=256)
def _mlp_workspace_bytes(T: int, H: int, inter: int, dtype: int, fmt: int) -> int:
    n = ctypes.c_size_t(0)
    _lib.call("moe_fp8_swiglu_mlp_workspace_size", T, H, inter, dtype, fmt, ctypes.byref(n))
    return n.value


def swiglu_mlp(x: torch.Tensor, w13: torch.Tensor, w13_scale: torch.Tensor, w2: torch.Tensor,
               w2_scale: torch.Tensor, addend: torch.Tensor | None = None,
               out: torch.Tensor | None = None, status: torch.Tensor | None = None
               ) -> torch.Tensor:
    """The SwiGLU MLP of a shared expert on block-scaled e4m3 weights
    (moe_fp8_swiglu_mlp): w2 (silu(g) * u) (+ addend), [g | u] = w13 x, for
    x [T, H] (f32/f16/bf16), w13 [2I, H] (gate rows, then up rows) and w2 [H, I]
    with their scales, all float32 or all uint8 (UE8M0). Activations are
    quantised per token and 128 columns in the weights' scale format; [g | u] is
    held in x's dtype. addend [T, H] in x's dtype (the routed experts' output; it
    may be out) is added before the one rounding of the result. Four launches."""
    index = x.get_device()
    if (not index == w13.get_device() == w13_scale.get_device() == w2.get_device()
            == w2_scale.get_device() or index < 0):
        for name, t in (("x", x), ("w13", w13), ("w13_scale", w13_scale), ("w2", w2),
                        ("w2_scale", w2_scale)):
            _check_cuda(name, t)
        raise ValueError("x and the weights with their scales must be on one device")
    if forward_ad._current_level >= 0:
        _refuse_tangents(x=x, w13=w13, w13_scale=w13_scale, w2=w2, w2_scale=w2_scale,
                         addend=addend, out=out)
    for name, t in (("x", x), ("w13_scale", w13_scale), ("w2_scale", w2_scale)):
        if t.requires_grad:
            _no_grad_needed(name, t)
    if x.dim() != 2 or x.dtype not in _FLOAT or x.shape[1] < 1:
        raise ValueError("x must be a 2-D f32/f16/bf16 tensor")
    w13, w2 = _fp8_rows("w13", w13), _fp8_rows("w2", w2)
    (T, H), inter = x.shape, w2.shape[1]
    if w13.shape != (2 * inter, H) or w2.shape[0] != H or inter < 1:
        raise ValueError(f"w13 {tuple(w13.shape)} and w2 {tuple(w2.shape)} must be [2I, {H}] and "
                         f"[{H}, I]")
    fmt = _SCALE_FORMAT.get(w13_scale.dtype)
    if fmt is None or w2_scale.dtype != w13_scale.dtype:
        raise ValueError("w13_scale and w2_scale must both be float32 or both uint8 (UE8M0)")
    hb, ib, gb = (H + 127) // 128, (inter + 127) // 128, (2 * inter + 127) // 128
    if w13_scale.shape != (gb, hb) or w2_scale.shape != (hb, ib):
        raise ValueError(f"scales must be [{gb}, {hb}] and [{hb}, {ib}], got "
                         f"{tuple(w13_scale.shape)} and {tuple(w2_scale.shape)}")
    x = _rows_of(x)
    if out is not None:
        _check_out(out, T, H, x.dtype, index)
    add_ptr, add_ld = (None, 0) if addend is None else _addend(addend, T, H, x.dtype, index, out)
    if out is None:
        out = torch.empty(T, H, dtype=x.dtype, device=x.device)
    code = _DTYPE_CODE[x.dtype]
    # of its own: a workspace kept by stream would be shared by captured graphs
    ws = torch.empty(_mlp_workspace_bytes(T, H, inter, code, fmt), dtype=torch.uint8,
                     device=x.device)
    w13_scale, w2_scale = w13_scale.contiguous(), w2_scale.contiguous()
    _enqueue("moe_fp8_swiglu_mlp", index, x.data_ptr(), max(x.stride(0), H), code, T, H, inter,
             w13.data_ptr(), max(w13.stride(0), _round_up(H, 16)), w13_scale.data_ptr(),
             w2.data_ptr(), max(w2.stride(0), _round_up(inter, 16)), w2_scale.data_ptr(), fmt,
             add_ptr, add_ld, out.data_ptr(), max(out.stride(0), H), ws.data_ptr(), ws.numel(),
             _status_ptr(status, index))
    return out
