"""Refusals of the router, the 16-bit grouped products and MXFP4, without a GPU: the
C entries check their arguments before any device call, the Python ones before that."""
import pytest
import torch

import ratchet_b200 as rb
from ratchet_b200 import _lib

P = 1 << 20  # a pointer that is never followed


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


# ------------------------------------------------------------------ 16-bit products
def _f16(G=2, n=64, k=128, rows=16, dtype=1, out_dtype=1, acc=0, off=P, a=P, b=P, out=P):
    return _lib.FggF16RowsProblem(G, n, k, rows, dtype, out_dtype, acc, off, a, b, out)


@pytest.mark.parametrize("change,direction,code", [
    (dict(G=0), 0, _lib.FGG_EINVAL),
    (dict(G=_lib.FGG_MAX_GROUPS + 1), 0, _lib.FGG_EINVAL),
    (dict(n=60), 0, _lib.FGG_EBADSHAPE),
    (dict(k=4), 1, _lib.FGG_EBADSHAPE),
    (dict(n=0), 2, _lib.FGG_EBADSHAPE),
    (dict(n=256 * 65536), 0, _lib.FGG_EBADSHAPE),
    (dict(rows=-1), 0, _lib.FGG_EINVAL),
    (dict(dtype=0), 0, _lib.FGG_EINVAL),
    (dict(out_dtype=0), 0, _lib.FGG_EINVAL),       # fp32 results: weight gradients only
    (dict(out_dtype=2), 2, _lib.FGG_EINVAL),
    (dict(acc=1), 2, _lib.FGG_EINVAL),             # adding needs fp32
    (dict(acc=1), 0, _lib.FGG_EINVAL),
    (dict(), 3, _lib.FGG_EINVAL),
    (dict(), -1, _lib.FGG_EINVAL),
])
def test_f16_bad_problems(L, change, direction, code):
    p = _f16(**change)
    assert L.fgg_f16_rows_workspace_bytes(p, direction) == 0
    assert L.fgg_f16_grouped_gemm_rows(p, direction, P, 1 << 30, None) == code
    assert L.fgg_last_error_detail()


@pytest.mark.parametrize("direction", [0, 1, 2])
def test_f16_bad_buffers(L, direction):
    p = _f16()
    need = L.fgg_f16_rows_workspace_bytes(p, direction)
    assert need > 0
    call = lambda q, ws=P, size=need: L.fgg_f16_grouped_gemm_rows(q, direction, ws, size, None)
    assert call(p, None) == _lib.FGG_EINVAL
    assert call(p, P + 64) == _lib.FGG_EALIGN
    assert call(p, P, need - 1) == _lib.FGG_EWORKSPACE
    assert call(_f16(off=None)) == _lib.FGG_EINVAL
    assert call(_f16(a=None)) == _lib.FGG_EINVAL
    assert call(_f16(b=None)) == _lib.FGG_EINVAL
    assert call(_f16(out=None)) == _lib.FGG_EINVAL
    assert call(_f16(a=P + 8)) == _lib.FGG_EALIGN
    assert call(_f16(b=P + 2)) == _lib.FGG_EALIGN
    assert call(_f16(out=P + 4)) == _lib.FGG_EALIGN
    assert call(_f16(off=P + 2)) == _lib.FGG_EALIGN
    assert L.fgg_f16_grouped_gemm_rows(None, direction, P, need, None) == _lib.FGG_EINVAL


def test_f16_workspace_bytes(L):
    """Tile list: 12 bytes per tile of at most rows / 256 + G (and rows) token tiles;
    wgrad: the groups' order and 16 rows of both operands per group."""
    up = lambda x: (x + 255) // 256 * 256
    tiles = min(1000 // 256 + 3, 1000) * 2
    assert L.fgg_f16_rows_workspace_bytes(_f16(3, 264, 520, 1000), 0) == 256 + up(8 * tiles) + 4 * tiles
    tiles = min(1000 // 256 + 3, 1000) * 3
    assert L.fgg_f16_rows_workspace_bytes(_f16(3, 264, 520, 1000), 1) == 256 + up(8 * tiles) + 4 * tiles
    assert (L.fgg_f16_rows_workspace_bytes(_f16(3, 264, 520, 1000), 2)
            == 512 + up(3 * 16 * 264 * 2) + 3 * 16 * 520 * 2)


@pytest.mark.parametrize("groups,n,k,rows,direction,units", [
    (1, 256, 4096, 1, 0, 2),          # one tile of 64 steps: two slices of 32
    (1, 256, 8192, 256, 0, 8),        # of at most 256 / 256 + 1 token tiles
    (4, 264, 4096, 300, 0, 20),       # at most 5 token tiles x 2
    (1, 256, 32768, 1, 0, 16),        # at most 16 slices
    (9, 256, 65536, 4000, 0, 96),     # at most 96 units
    (1, 256, 4032, 1, 0, 0),          # 63 steps
    (1, 48 * 256 + 8, 8192, 1, 0, 0),  # 49 tiles or more in every call
    (1, 4096, 256, 1, 1, 2),
    (1, 64, 64, 30000, 2, 14),
    (1, 2056, 1288, 30000, 2, 0),     # 54 tiles
])
def test_f16_workspace_of_split_tiles(L, groups, n, k, rows, direction, units):
    """What units of 256 KB each, their list and the joins' counters add."""
    up = lambda x: (x + 255) // 256 * 256
    if direction == 2:
        base = 256 + up(4 * groups) + up(groups * 16 * n * 2) + groups * 16 * k * 2
    else:
        tiles = min(rows // 256 + groups, rows) * -(-(n if direction == 0 else k) // 256)
        base = 256 + up(8 * tiles) + 4 * tiles
    want = base if units == 0 else up(base) + up(96 * 4) + 96 * 16 * 4 + units * 256 * 1024
    assert L.fgg_f16_rows_workspace_bytes(_f16(groups, n, k, rows), direction) == want


def test_f16_python_refusals():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    w = torch.zeros(2, 32, 64, dtype=torch.bfloat16)
    off = torch.tensor([0, 2, 4], dtype=torch.int32)
    for call in (lambda: rb.grouped_gemm_rows(x, w, off),          # on the host
                 lambda: rb.grouped_gemm_rows_dgrad(x, w, off),
                 lambda: rb.grouped_gemm_rows_wgrad(x, x, off)):
        with pytest.raises(ValueError):
            call()


# -------------------------------------------------------------------------- router
@pytest.mark.parametrize("dtype,t,e,k,score,code", [
    (3, 4, 8, 2, 0, _lib.FGG_EINVAL),
    (0, 4, 8, 2, 2, _lib.FGG_EINVAL),
    (0, -1, 8, 2, 0, _lib.FGG_EINVAL),
    (0, 4, 0, 1, 0, _lib.FGG_EBADSHAPE),
    (0, 4, 1025, 2, 0, _lib.FGG_EBADSHAPE),
    (0, 4, 8, 0, 0, _lib.FGG_EBADSHAPE),
    (0, 4, 8, 9, 0, _lib.FGG_EBADSHAPE),
    (0, 4, 64, 33, 0, _lib.FGG_EBADSHAPE),
])
def test_router_bad_problems(L, dtype, t, e, k, score, code):
    assert L.fgg_moe_router(P, dtype, t, e, k, score, None, 1, 1.0, P, P, None) == code
    assert L.fgg_moe_router_backward(P, P, dtype, P, t, e, k, score, 1, 1.0, P, None) == code


def test_router_bad_buffers(L):
    fwd = lambda l=P, bias=None, ids=P, w=P: L.fgg_moe_router(l, 0, 4, 8, 2, 0, bias, 1, 1.0, ids, w, None)
    assert fwd(l=None) == _lib.FGG_EINVAL
    assert fwd(l=P + 2) == _lib.FGG_EALIGN
    assert fwd(ids=None) == _lib.FGG_EINVAL
    assert fwd(w=None) == _lib.FGG_EINVAL
    assert fwd(bias=P + 1) == _lib.FGG_EALIGN
    assert fwd(w=P + 2) == _lib.FGG_EALIGN
    bwd = lambda dw=P, l=P, ids=P, d=P: L.fgg_moe_router_backward(dw, l, 1, ids, 4, 8, 2, 0, 1, 1.0, d, None)
    assert bwd(dw=None) == _lib.FGG_EINVAL
    assert bwd(ids=None) == _lib.FGG_EINVAL
    assert bwd(d=None) == _lib.FGG_EINVAL
    assert bwd(l=P + 1) == _lib.FGG_EALIGN
    assert bwd(d=P + 1) == _lib.FGG_EALIGN
    assert bwd(dw=P + 2) == _lib.FGG_EALIGN
    # no tokens: nothing to do, whatever the other buffers
    assert L.fgg_moe_router(None, 0, 0, 8, 2, 0, None, 1, 1.0, None, None, None) == _lib.FGG_OK


def test_router_python_refusals():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        rb.moe_router(x, 2)
    with pytest.raises(ValueError):
        rb.moe_router_backward(torch.zeros(4, 2), x, torch.zeros(4, 2, dtype=torch.int32))


# --------------------------------------------------------------------------- MXFP4
def test_mxfp4_quantise_refusals(L):
    q = lambda x=P, dt=0, n=64, c=P, s=P: L.fgg_mxfp4_quantize(x, dt, n, c, s, None)
    d = lambda x=P, dt=0, n=64, c=P, s=P: L.fgg_mxfp4_dequantize(c, s, n, x, dt, None)
    for f in (q, d):
        assert f(dt=3) == _lib.FGG_EINVAL
        assert f(n=48) == _lib.FGG_EBADSHAPE
        assert f(n=-32) == _lib.FGG_EBADSHAPE
        assert f(x=None) == _lib.FGG_EINVAL
        assert f(c=None) == _lib.FGG_EINVAL
        assert f(s=None) == _lib.FGG_EINVAL
        assert f(x=P + 8) == _lib.FGG_EALIGN
        assert f(c=P + 2) == _lib.FGG_EALIGN
        assert f(x=None, c=None, s=None, n=0) == _lib.FGG_OK
        assert f(n=(1 << 31) * 8 * 256) == _lib.FGG_EBADSHAPE


def _rows(G=2, n=256, k=512, rows=300, wg=2, most=0, off=P, a=P, sf=P, alpha=P, out=P, idx=None,
          b=P):
    return _lib.FggMxfp4RowsProblem((G, n, k, rows, off, a, sf, alpha, out, None, idx, wg, most), b)


@pytest.mark.parametrize("change,code", [
    (dict(G=0), _lib.FGG_EINVAL),
    (dict(n=200), _lib.FGG_EBADSHAPE),
    (dict(k=64), _lib.FGG_EBADSHAPE),              # NVFP4 takes it, MXFP4 does not
    (dict(k=192), _lib.FGG_EBADSHAPE),
    (dict(rows=-1), _lib.FGG_EINVAL),
    (dict(idx=P, wg=0), _lib.FGG_EINVAL),
])
def test_mxfp4_bad_problems(L, change, code):
    p = _rows(**change)
    assert L.fgg_mxfp4_rows_workspace_bytes(p) == 0
    assert L.fgg_mxfp4_grouped_gemm_rows(p, P, P, 1 << 30, None) == code


def test_mxfp4_bad_buffers(L):
    p = _rows()
    need = L.fgg_mxfp4_rows_workspace_bytes(p)
    nv = L.fgg_nvfp4_rows_workspace_bytes(p.rows)
    assert 0 < need < nv                           # half the scale atoms
    call = lambda q, pack=P, ws=P, size=need: L.fgg_mxfp4_grouped_gemm_rows(q, pack, ws, size, None)
    assert call(p, ws=None) == _lib.FGG_EINVAL
    assert call(p, size=need - 1) == _lib.FGG_EWORKSPACE
    assert call(p, pack=None) == _lib.FGG_EINVAL
    assert call(_rows(off=None)) == _lib.FGG_EINVAL
    assert call(_rows(a=P + 8)) == _lib.FGG_EALIGN
    assert call(_rows(b=None)) == _lib.FGG_EINVAL
    assert call(_rows(b=P + 4)) == _lib.FGG_EALIGN
    # alpha is optional here, and only here
    nvfp4 = L.fgg_nvfp4_grouped_gemm_rows(_rows(alpha=None).rows, P, P, nv, None)
    assert nvfp4 == _lib.FGG_EINVAL and b"alpha" in L.fgg_last_error_detail()


def test_mxfp4_weight_pack_bytes(L):
    """A header and two 512-byte scale atoms per 128 rows and 256 K."""
    for g, n, k in ((1, 128, 128), (3, 256, 640), (8, 4096, 7168)):
        want = 256 + g * (n // 128) * ((k + 255) // 256) * 2 * 512
        assert L.fgg_mxfp4_weight_pack_bytes(g, n, k) == want
    for bad in ((0, 128, 128), (1, 100, 128), (1, 128, 64), (_lib.FGG_MAX_GROUPS + 1, 128, 128)):
        assert L.fgg_mxfp4_weight_pack_bytes(*bad) == 0
    pack = lambda sf=P, g=1, n=128, k=128, to=P, size=1 << 20: L.fgg_mxfp4_pack_weights(
        sf, g, n, k, to, size, None)
    assert pack(k=64) == _lib.FGG_EBADSHAPE
    assert pack(n=64) == _lib.FGG_EBADSHAPE
    assert pack(g=0) == _lib.FGG_EINVAL
    assert pack(sf=None) == _lib.FGG_EINVAL
    assert pack(to=None) == _lib.FGG_EINVAL
    assert pack(sf=P + 2) == _lib.FGG_EALIGN
    assert pack(to=P + 8) == _lib.FGG_EALIGN
    assert pack(size=1279) == _lib.FGG_EWORKSPACE


def test_mxfp4_python_refusals():
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError):
        rb.quantize_mxfp4(x)                       # on the host
    codes = torch.zeros(4, 32, dtype=torch.uint8)
    sf = torch.zeros(4, 2, dtype=torch.uint8)
    for bad in (lambda: rb.dequantize_mxfp4(codes, sf),
                lambda: rb.dequantize_mxfp4(codes, sf, torch.float64),
                lambda: rb.dequantize_mxfp4(codes, sf[:, :1]),
                lambda: rb.dequantize_mxfp4(codes[:, :5], sf),
                lambda: rb.dequantize_mxfp4(codes, sf.float()),
                lambda: rb.pack_mxfp4_weights(codes, sf),
                lambda: rb.pack_mxfp4_weights(torch.zeros(1, 128, 64, dtype=torch.uint8),
                                              torch.zeros(1, 128, 4, dtype=torch.uint8)),
                lambda: rb.mxfp4_grouped_gemm_rows(codes, sf, torch.zeros(2, dtype=torch.int32), None)):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------------- sources
def test_arrivals_in_another_cta_release_at_cluster_scope():
    """An arrival on another CTA's barrier orders this CTA's accesses before what the other
    does next only if it releases at cluster scope (a scope left out is the CTA's)."""
    import re
    from pathlib import Path

    csrc = Path(rb.__file__).resolve().parent / "csrc"
    found = []
    for f in sorted(csrc.glob("*.cu*")):
        found += [(f.name, m) for m in re.findall(r"mbarrier\.arrive[a-z0-9_.:]*shared::cluster[a-z0-9_.]*",
                                                  f.read_text())]
    assert found
    for name, op in found:
        assert ".release.cluster." in op, (name, op)


def test_no_descriptor_is_edited_on_the_device():
    """TMA descriptors are encoded on the host: the kernels that edited them on the device
    are the only ones that ever faulted."""
    from pathlib import Path

    csrc = Path(rb.__file__).resolve().parent / "csrc"
    for f in sorted(csrc.glob("*.cu*")):
        text = f.read_text()
        assert "tensormap.replace" not in text and "tensormap.cp_fenceproxy" not in text, f.name


def test_what_the_prepare_kernels_write_is_not_read_as_constant():
    """The products start while their prepare kernel runs, and that one while the kernel
    before it finishes: neither reads global memory as data that is constant for its life."""
    from pathlib import Path

    csrc = Path(rb.__file__).resolve().parent / "csrc"
    for name in ("fgg_engine.cuh", "fgg_nvfp4.cu", "fgg_mx.cu", "fgg_f16.cu"):
        text = (csrc / name).read_text()
        assert "griddep_wait()" in text
        assert "__ldg(" not in text and "ld.global.nc" not in text, name
