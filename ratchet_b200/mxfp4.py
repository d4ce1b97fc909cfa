"""MXFP4: quantisation, its inverse, and the grouped product of two MXFP4 operands.

E2M1 elements, two to a byte (the even one in the low half), with one
power-of-two scale per 32 of them along K, stored as an UE8M0 byte
(torch.float8_e8m0fnu): the weight format of the reference operator
(kernels/gemm/fp4_grouped_gemm/b200/kernel.py:14-26), whose scales as fp32 are
`sf.float()`.  It needs no per-tensor scale, so quantising is one pass.
"""
from __future__ import annotations

import torch

from . import _lib, ops

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_SF_DTYPES = (torch.float8_e8m0fnu, torch.uint8)
_I32_MAX = 2**31 - 1


def _sf_u8(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dtype not in _SF_DTYPES:
        raise ValueError(f"{name}: dtype {t.dtype} must be float8_e8m0fnu or uint8")
    return t if t.dtype == torch.uint8 else t.view(torch.uint8)


def quantize_mxfp4(x: torch.Tensor):
    """Quantise a contiguous CUDA tensor [..., K] (fp32, bf16 or fp16, K a multiple
    of 32, 16-byte aligned) to (codes uint8 [..., K/2], sf float8_e8m0fnu
    [..., K/32]): x ~ e2m1 * sf.

    A block's scale is 2^(floor(log2 max|x|) - 2), at least 2^-127; elements round
    to the nearest code, ties to the even one, and saturate at 6 scales.  A block
    with a NaN or an infinity has a NaN scale."""
    if x.dtype not in _DTYPES or not x.is_cuda or not x.is_contiguous() or x.dim() < 1:
        raise ValueError("x must be a contiguous fp32, bf16 or fp16 CUDA tensor")
    if x.shape[-1] % 32 != 0 or x.shape[-1] == 0:
        raise ValueError(f"K={x.shape[-1]} must be a positive multiple of 32")
    dev = x.device
    if ops._is_current(dev):
        return _quantize_on(x, dev)
    with torch.cuda.device(dev):
        return _quantize_on(x, dev)


def _quantize_on(x, dev):
    *lead, k = x.shape
    codes = torch.empty((*lead, k // 2), dtype=torch.uint8, device=dev)
    sf = torch.empty((*lead, k // 32), dtype=torch.float8_e8m0fnu, device=dev)
    _lib.check(_lib.lib().fgg_mxfp4_quantize(x.data_ptr(), _DTYPES[x.dtype], x.numel(),
                                             codes.data_ptr(), sf.data_ptr(),
                                             ops._stream_ptr(dev)), "quantize_mxfp4")
    return codes, sf


def dequantize_mxfp4(codes: torch.Tensor, sf: torch.Tensor,
                     dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [..., K] of codes [..., K/2] and scales [..., K/32], rounded once
    to dtype (bf16 holds each of them exactly down to its subnormals)."""
    if dtype not in _DTYPES:
        raise ValueError(f"dtype {dtype} must be float32, bfloat16 or float16")
    if codes.dtype not in ops._U8_DTYPES or sf.dtype not in _SF_DTYPES:
        raise ValueError(f"codes {codes.dtype} / sf {sf.dtype} must be codes and UE8M0 scales as bytes")
    if codes.dim() < 1 or codes.shape[-1] % 16 != 0 or codes.shape[-1] == 0:
        raise ValueError(f"codes {list(codes.shape)} must be [..., K/2] with K a multiple of 32")
    *lead, kh = codes.shape
    if list(sf.shape) != [*lead, kh // 16]:
        raise ValueError(f"sf {list(sf.shape)} does not match codes {list(codes.shape)}")
    dev = codes.device
    if not (codes.is_cuda and sf.device == dev and codes.is_contiguous() and sf.is_contiguous()):
        raise ValueError("codes and sf must be contiguous tensors on one CUDA device")
    if ops._is_current(dev):
        return _dequantize_on(codes, sf, dtype, (*lead, 2 * kh), dev)
    with torch.cuda.device(dev):
        return _dequantize_on(codes, sf, dtype, (*lead, 2 * kh), dev)


def _dequantize_on(codes, sf, dtype, shape, dev):
    x = torch.empty(shape, dtype=dtype, device=dev)
    _lib.check(_lib.lib().fgg_mxfp4_dequantize(codes.data_ptr(), sf.data_ptr(), x.numel(),
                                               x.data_ptr(), _DTYPES[dtype],
                                               ops._stream_ptr(dev)), "dequantize_mxfp4")
    return x


class Mxfp4WeightPack:
    """Device-side packed MXFP4 weights: the scales in the MMA's 512-byte SF atoms.
    The codes are read where they lie (the pack keeps them alive); pack again after
    changing scales in place."""

    def __init__(self, w: torch.Tensor, w_sf: torch.Tensor):
        codes, sf = ops._as_u8(w, "w"), _sf_u8(w_sf, "w_sf")
        if codes.dim() != 3:
            raise ValueError(f"w must be [G, N, K/2], got {list(codes.shape)}")
        G, n, kh = (int(v) for v in codes.shape)
        k = 2 * kh
        if tuple(sf.shape) != (G, n, k // 32) or k % 128 != 0:
            raise ValueError(f"w_sf {list(sf.shape)} must be [{G}, {n}, K/32] with K={k} a "
                             "multiple of 128")
        if not (codes.is_cuda and sf.device == codes.device and codes.is_contiguous()
                and sf.is_contiguous() and codes.data_ptr() % 16 == 0):
            raise ValueError("w (16-byte aligned) and w_sf must be contiguous tensors on one CUDA "
                             "device")
        if max(G, n, k) > _I32_MAX:
            raise ValueError(f"weights {list(codes.shape)} are too large")
        self.G, self.n, self.k = G, n, k
        self.device = codes.device
        self.sources = (w, w_sf)
        L = _lib.lib()
        nbytes = int(L.fgg_mxfp4_weight_pack_bytes(G, n, k))
        if nbytes == 0:
            raise ValueError(f"unsupported weight geometry G={G} N={n} K={k}: 1 to "
                             f"{_lib.FGG_MAX_GROUPS} groups, N and K multiples of 128")
        with ops._on(self.device):
            self.buf = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            _lib.check(L.fgg_mxfp4_pack_weights(sf.data_ptr(), G, n, k, self.buf.data_ptr(), nbytes,
                                                ops._stream_ptr(self.device)),
                       "pack_mxfp4_weights")


def pack_mxfp4_weights(w: torch.Tensor, w_sf: torch.Tensor) -> Mxfp4WeightPack:
    """Pack quantised weights, codes [G, N, K/2] and scales [G, N, K/32] (as
    quantize_mxfp4 returns them for [G, N, K]; N and K multiples of 128), for
    mxfp4_grouped_gemm_rows."""
    return Mxfp4WeightPack(w, w_sf)


def mxfp4_grouped_gemm_rows(a: torch.Tensor, a_sf: torch.Tensor, offsets: torch.Tensor,
                            pack: Mxfp4WeightPack, *, alpha: torch.Tensor | None = None,
                            out: torch.Tensor | None = None,
                            row_scale: torch.Tensor | None = None,
                            b_index: torch.Tensor | None = None,
                            max_group_rows: int = 0) -> torch.Tensor:
    """out[r, :] = bf16(alpha_g * row_scale_r * deq(a_r) deq(W_g)^T), [R, N].

    a [R, K/2] codes and a_sf [R, K/32] scales (quantize_mxfp4 of the token rows);
    offsets int32 CUDA [G + 1]: group g owns rows [offsets[g], offsets[g+1]); rows
    outside every group are left as they are.  pack: pack_mxfp4_weights; alpha
    fp32 [G], row_scale fp32 [R] (default 1); b_index int32 [G] names each group's
    packed weight group; max_group_rows: a host bound on every group's rows (<= 16
    selects the decode tiles).  All as in nvfp4_grouped_gemm_rows."""
    if not isinstance(pack, Mxfp4WeightPack):
        raise ValueError("pack must come from pack_mxfp4_weights")
    n, k, dev = pack.n, pack.k, pack.device
    if a.dtype not in ops._U8_DTYPES or a_sf.dtype not in _SF_DTYPES:
        raise ValueError(f"a {a.dtype} / a_sf {a_sf.dtype} must be codes and UE8M0 scales as bytes")
    if (a.dim() != 2 or a.shape[1] != k // 2 or a_sf.dim() != 2 or a_sf.shape[0] != a.shape[0]
            or a_sf.shape[1] != k // 32):
        raise ValueError(f"a {list(a.shape)} / a_sf {list(a_sf.shape)} do not match "
                         f"[R, {k // 2}] / [R, {k // 32}] for K={k}")
    if offsets.dtype is not torch.int32 or offsets.dim() != 1 or offsets.shape[0] < 2:
        raise ValueError("offsets must be int32 [G + 1]")
    rows, G = int(a.shape[0]), int(offsets.shape[0]) - 1
    if b_index is None and G != pack.G:
        raise ValueError(f"{G} groups but {pack.G} packed weight groups (pass b_index to map them)")
    if rows > _I32_MAX or not 0 <= max_group_rows <= _I32_MAX:
        raise ValueError(f"{rows} rows / max_group_rows={max_group_rows} out of range")
    for name, t, dt, shape in (("alpha", alpha, torch.float32, (G,)),
                               ("out", out, torch.bfloat16, (rows, n)),
                               ("row_scale", row_scale, torch.float32, (rows,)),
                               ("b_index", b_index, torch.int32, (G,))):
        if t is not None and (t.dtype is not dt or tuple(t.shape) != shape):
            raise ValueError(f"{name} must be {dt} {list(shape)}, got {t.dtype} {list(t.shape)}")
    di = dev.index  # on the host: -1
    for t in (a, a_sf, offsets, alpha, out, row_scale, b_index):
        if t is not None and (t.get_device() != di or not t.is_contiguous()):
            raise ValueError(f"every tensor must be contiguous and on {dev}")
    if out is not None:
        ops._disjoint(out, a, a_sf, pack.sources[0])
    if ops._is_current(dev):
        return _product_on(a, a_sf, offsets, pack, alpha, out, row_scale, b_index, max_group_rows)
    with torch.cuda.device(dev):
        return _product_on(a, a_sf, offsets, pack, alpha, out, row_scale, b_index, max_group_rows)


def _product_on(a, a_sf, offsets, pack, alpha, out, row_scale, b_index, max_group_rows):
    rows, n, dev = a.shape[0], pack.n, pack.device
    if out is None:
        out = torch.empty((rows, n), dtype=torch.bfloat16, device=dev)
    L = _lib.lib()
    ptr = lambda t: None if t is None else t.data_ptr()
    prob = _lib.FggMxfp4RowsProblem(
        (offsets.shape[0] - 1, n, pack.k, rows, offsets.data_ptr(), a.data_ptr(), a_sf.data_ptr(),
         ptr(alpha), out.data_ptr(), ptr(row_scale), ptr(b_index), pack.G, int(max_group_rows)),
        pack.sources[0].data_ptr())
    nbytes = int(L.fgg_mxfp4_rows_workspace_bytes(prob))
    if nbytes == 0:
        _lib.check(L.fgg_mxfp4_grouped_gemm_rows(prob, None, None, 0, None),
                   "mxfp4_grouped_gemm_rows")
    stream = ops._stream_ptr(dev)
    ws = ops._workspace(dev, stream, nbytes)
    _lib.check(L.fgg_mxfp4_grouped_gemm_rows(prob, pack.buf.data_ptr(), ws.data_ptr(), nbytes,
                                             stream), "mxfp4_grouped_gemm_rows")
    ops._set_last_ws(ws, stream)
    return out
