"""Products grouped by expert in bf16 / fp16: the forward product over contiguous
token rows and its two gradients, with the group offsets on the device.

The reference operator's M-grouped layout (one concatenated activation tensor,
kernels/gemm/fp4_grouped_gemm/b200/kernel.py:10-37) for experts that stay in 16
bits, and for their training.  Like every call of this package they run on the
current CUDA stream of the tensors' device, never synchronise the host, and
record no autograd graph: the gradients are calls of their own.
"""
from __future__ import annotations

import torch

from . import _lib, ops

_DTYPES = {torch.bfloat16: 1, torch.float16: 2}
_I32_MAX = 2**31 - 1


def _check(name: str, t: torch.Tensor, shape, dtype, dev) -> None:
    if (t.dtype is not dtype or tuple(t.shape) != tuple(shape) or t.device != dev
            or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous {dtype} {list(shape)} tensor on {dev}, got "
                         f"{t.dtype} {list(t.shape)} on {t.device}")


def _offsets(offsets: torch.Tensor, dev) -> int:
    if (offsets.dtype is not torch.int32 or offsets.dim() != 1 or offsets.shape[0] < 2
            or offsets.device != dev or not offsets.is_contiguous()):
        raise ValueError(f"offsets must be a contiguous int32 [G + 1] tensor on {dev}")
    return int(offsets.shape[0]) - 1


def _tokens(name: str, t: torch.Tensor):
    if t.dim() != 2 or t.dtype not in _DTYPES or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 2-D bf16 or fp16 CUDA tensor")
    if max(t.shape) > _I32_MAX:
        raise ValueError(f"{name} {list(t.shape)} is too large")
    return int(t.shape[0]), int(t.shape[1])


def _run(direction: int, a, b, out, offsets, G, n, k, rows, accumulate=False) -> None:
    L = _lib.lib()
    dev = a.device
    if max(n, k) > _I32_MAX:
        raise ValueError(f"N={n}, K={k} too large")
    prob = _lib.FggF16RowsProblem(G, n, k, rows, _DTYPES[a.dtype], _DTYPES.get(out.dtype, 0),
                                  1 if accumulate else 0, offsets.data_ptr(), a.data_ptr(),
                                  b.data_ptr(), out.data_ptr())
    nbytes = int(L.fgg_f16_rows_workspace_bytes(prob, direction))
    if nbytes == 0:
        _lib.check(L.fgg_f16_grouped_gemm_rows(prob, direction, None, 0, None), "grouped_gemm_rows")
    if ops._is_current(dev):
        stream = ops._stream_ptr(dev)
        ws = ops._workspace(dev, stream, nbytes)
        rc = L.fgg_f16_grouped_gemm_rows(prob, direction, ws.data_ptr(), nbytes, stream)
    else:
        with torch.cuda.device(dev):
            stream = ops._stream_ptr(dev)
            ws = ops._workspace(dev, stream, nbytes)
            rc = L.fgg_f16_grouped_gemm_rows(prob, direction, ws.data_ptr(), nbytes, stream)
    _lib.check(rc, "grouped_gemm_rows")
    ops._set_last_ws(ws, stream)


def _weights(w: torch.Tensor, dtype, dev, G: int):
    if w.dim() != 3:
        raise ValueError(f"w must be [G, N, K], got {list(w.shape)}")
    _check("w", w, (G, w.shape[1], w.shape[2]), dtype, dev)
    return int(w.shape[1]), int(w.shape[2])


def grouped_gemm_rows(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, *,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """out[r, :] = W_g x_r for the rows r of every group g.

    x       [R, K] bf16 or fp16, token rows, group by group
    w       [G, N, K] of the same type (N and K multiples of 8)
    offsets int32 CUDA tensor [G + 1] (nondecreasing, offsets[G] <= R): group g
            owns rows [offsets[g], offsets[g+1]); it may be written by an earlier
            kernel on the stream -- the host never reads it
    out     optional contiguous [R, N] of the same type; rows outside every
            group are left as they are (in a new tensor they are undefined)
    Sums are held in fp32 and rounded once.  A call's results do not vary; a call of
    few tiles splits its sums over the GPU, so that the same rows may differ in the
    last bits between calls whose other groups have other rows (empty groups and
    spare rows change nothing).  Malformed offsets write
    nothing and make last_status() raise."""
    rows, k = _tokens("x", x)
    G = _offsets(offsets, x.device)
    n, kw = _weights(w, x.dtype, x.device, G)
    if kw != k:
        raise ValueError(f"x has K={k}, w has K={kw}")
    if out is None:
        out = torch.empty((rows, n), dtype=x.dtype, device=x.device)
    else:
        _check("out", out, (rows, n), x.dtype, x.device)
        ops._disjoint(out, x, w)
    _run(0, x, w, out, offsets, G, n, k, rows)
    return out


def grouped_gemm_rows_dgrad(dy: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, *,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of grouped_gemm_rows' x: out[r, :] = W_g^T dy_r, [R, K].

    dy [R, N] bf16 or fp16; w [G, N, K] as it lies in memory for the forward
    product (nothing is transposed); offsets, out as there."""
    rows, n = _tokens("dy", dy)
    G = _offsets(offsets, dy.device)
    nw, k = _weights(w, dy.dtype, dy.device, G)
    if nw != n:
        raise ValueError(f"dy has N={n}, w has N={nw}")
    if out is None:
        out = torch.empty((rows, k), dtype=dy.dtype, device=dy.device)
    else:
        _check("out", out, (rows, k), dy.dtype, dy.device)
        ops._disjoint(out, dy, w)
    _run(1, dy, w, out, offsets, G, n, k, rows)
    return out


def grouped_gemm_rows_wgrad(dy: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor, *,
                            out: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float32,
                            accumulate: bool = False) -> torch.Tensor:
    """The gradient of grouped_gemm_rows' w: out[g] = sum_r dy_r x_r^T, [G, N, K].

    dy [R, N] and x [R, K] of one 16-bit type; out_dtype fp32 or that type (an
    `out` given sets it).  An empty group's gradient is zero.  accumulate=True
    adds to `out` instead (fp32, gradient accumulation over microbatches): every
    element gets one addition in a fixed order, so results do not vary."""
    rows, n = _tokens("dy", dy)
    G = _offsets(offsets, dy.device)
    if x.dim() != 2:
        raise ValueError(f"x must be [R, K], got {list(x.shape)}")
    k = int(x.shape[1])
    _check("x", x, (rows, k), dy.dtype, dy.device)
    if out is None:
        if accumulate:
            raise ValueError("accumulate=True needs the gradient to add to: give out=")
        if out_dtype not in (torch.float32, dy.dtype):
            raise ValueError(f"out_dtype {out_dtype} must be float32 or {dy.dtype}")
        out = torch.empty((G, n, k), dtype=out_dtype, device=dy.device)
    else:
        if out.dtype not in (torch.float32, dy.dtype):
            raise ValueError(f"out dtype {out.dtype} must be float32 or {dy.dtype}")
        _check("out", out, (G, n, k), out.dtype, dy.device)
        ops._disjoint(out, dy, x)
        if accumulate and out.dtype is not torch.float32:
            raise ValueError("accumulate=True needs a float32 out")
    _run(2, dy, x, out, offsets, G, n, k, rows, accumulate)
    return out
