"""MXFP4: quantize_mxfp4 and dequantize_mxfp4 against the format's definition (every
value has to be equal), mxfp4_grouped_gemm_rows against the product in 64 bits.

Tolerance of the product: operands are exact, products of two of them and their
scales exact in fp32; the sum of K of them is held in fp32, off by at most K 2^-23
of the sum of their magnitudes (the tensor core may truncate), then scaled by alpha
and the row factor (2^-24 each) and rounded once to bf16 (half a step, 2^-8).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _quant_ref(x):
    """(values fp64, scale bytes) of [..., K]."""
    b = x.double().cpu().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    e = torch.where((top > 0) & ~bad, torch.frexp(top)[1].long() - 3, torch.full_like(top, -127).long())
    e = e.clamp(min=-127)
    y = torch.where(bad.unsqueeze(-1), torch.zeros_like(b), torch.ldexp(b, -e.unsqueeze(-1)))
    a = y.abs()
    step = 0.5 + 0.5 * (a >= 2) + (a >= 4)
    q = torch.sign(y) * (torch.round(a / step) * step).clamp(max=6.0)
    v = torch.where(bad.unsqueeze(-1), torch.full_like(b, float("nan")), torch.ldexp(q, e.unsqueeze(-1)))
    return v.flatten(-2), torch.where(bad, 255, e + 127).to(torch.uint8)


def _same(got, want):
    g, w = got.double().cpu(), want
    assert torch.equal(torch.isnan(g), torch.isnan(w))
    assert torch.equal(torch.nan_to_num(g), torch.nan_to_num(w))


DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.mark.parametrize("dtype", list(DTYPES))
# the last fills the GPU: several pieces per thread, the last block of them in part
@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (17, 2048), (2, 5, 160), (64,), (303, 32032)])
def test_quantize(cuda_device, dtype, shape):
    import ratchet_b200 as rb

    g = torch.Generator("cuda").manual_seed(sum(shape))
    x = torch.randn(*shape, generator=g, device=cuda_device)
    x = (x * torch.randn(*shape[:-1], 1, generator=g, device=cuda_device).exp()).to(DTYPES[dtype])
    codes, sf = rb.quantize_mxfp4(x)
    assert codes.shape == (*shape[:-1], shape[-1] // 2) and codes.dtype is torch.uint8
    assert sf.shape == (*shape[:-1], shape[-1] // 32) and sf.dtype is torch.float8_e8m0fnu
    v, s = _quant_ref(x)
    assert torch.equal(sf.view(torch.uint8).cpu(), s)
    _same(rb.dequantize_mxfp4(codes, sf, torch.float32), v)
    _same(rb.dequantize_mxfp4(codes, sf, DTYPES[dtype]), v.to(DTYPES[dtype]).double())


def test_every_tie_and_edge(cuda_device):
    """All thresholds of E2M1 with both neighbours, saturation, both signs."""
    import ratchet_b200 as rb

    grid = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.9375]
    vals = [n for g in grid for n in (g, g * (1 - 2.0**-20), g * (1 + 2.0**-20))]
    rows = []
    for v in vals:
        for s in (1.0, -1.0):
            row = [0.0] * 32
            row[0] = 4.0          # the largest of its block: the scale is 1
            row[7] = s * v if v < 8 else 4.0
            rows.append(row)
    x = torch.tensor(rows, device=cuda_device)
    codes, sf = rb.quantize_mxfp4(x)
    v, s = _quant_ref(x)
    assert torch.equal(sf.view(torch.uint8).cpu(), s)
    _same(rb.dequantize_mxfp4(codes, sf, torch.float32), v)


def test_extreme_blocks(cuda_device):
    """Zeros, subnormals, the largest numbers, NaN and infinity; only the block that
    holds one is lost."""
    import ratchet_b200 as rb

    x = torch.zeros(9, 64, device=cuda_device)
    x[1] = 2.0**-149
    x[2] = 2.0**-126
    x[3] = 2.0**-125 * 1.5
    x[4] = torch.finfo(torch.float32).max
    x[5, 40] = float("nan")
    x[5, 3] = 1.0
    x[6, 0] = float("inf")
    x[7, 63] = -float("inf")
    x[8] = -0.0
    codes, sf = rb.quantize_mxfp4(x)
    v, s = _quant_ref(x)
    assert torch.equal(sf.view(torch.uint8).cpu(), s)
    _same(rb.dequantize_mxfp4(codes, sf, torch.float32), v.float().double())
    assert bool(torch.isfinite(rb.dequantize_mxfp4(codes, sf)[5, :32]).all())


def test_every_code_and_scale_reads_back(cuda_device):
    import ratchet_b200 as rb

    sf = torch.arange(256, dtype=torch.uint8, device=cuda_device)
    codes = (torch.arange(16, device=cuda_device) | (15 - torch.arange(16, device=cuda_device)) << 4)
    codes = codes.to(torch.uint8).repeat(256, 1)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
    grid = torch.cat((grid, -grid))
    pair = torch.stack((grid, grid.flip(0)), -1).flatten()
    want = torch.ldexp(pair.repeat(256, 1), torch.arange(256).unsqueeze(1) - 127)
    want[255] = float("nan")
    got = rb.dequantize_mxfp4(codes, sf.unsqueeze(1), torch.float32)
    _same(got, want.float().double())          # past fp32's largest: infinite in both
    _same(rb.dequantize_mxfp4(codes, sf.unsqueeze(1), torch.bfloat16),
          want.float().to(torch.bfloat16).double())


def test_weights_serve_the_reference_operator(cuda_device):
    """quantize_mxfp4's weights are fp4_grouped_gemm's: codes as they are, scales as fp32."""
    import ratchet_b200 as rb

    g = torch.Generator("cuda").manual_seed(1)
    w = torch.randn(2, 128, 256, generator=g, device=cuda_device) * 0.05
    codes, sf = rb.quantize_mxfp4(w)
    a = torch.randn(448, 256, generator=g, device=cuda_device).to(torch.float8_e4m3fn)
    a_sf = torch.ones(448, 2, device=cuda_device)
    idx = torch.arange(448, device=cuda_device, dtype=torch.int32) // 224
    c = rb.fp4_grouped_gemm(a, a_sf, codes, sf.float(), idx)
    rb.last_status()
    W = rb.dequantize_mxfp4(codes, sf, torch.float32).double()
    A = a.double()
    for i in range(2):
        want = A[224 * i:224 * (i + 1)] @ W[i].T
        mag = A[224 * i:224 * (i + 1)].abs() @ W[i].abs().T
        err = (c[224 * i:224 * (i + 1)].double() - want).abs()
        acc = 256 * 2.0**-23 * mag
        assert bool((err <= acc + 2.0**-8 * (want.abs() + acc)).all())


def _product(dev, sizes, n, k, spare, seed, wgroups=None):
    import ratchet_b200 as rb

    g = torch.Generator("cuda").manual_seed(seed)
    rows = sum(sizes) + spare
    x = torch.randn(rows, k, generator=g, device=dev) * torch.randn(rows, 1, generator=g, device=dev).exp()
    w = torch.randn(wgroups or len(sizes), n, k, generator=g, device=dev) * 0.02
    off = [0]
    for s in sizes:
        off.append(off[-1] + s)
    qx, qw = rb.quantize_mxfp4(x), rb.quantize_mxfp4(w)
    X = rb.dequantize_mxfp4(*qx, torch.float32).double()
    W = rb.dequantize_mxfp4(*qw, torch.float32).double()
    return qx, rb.pack_mxfp4_weights(*qw), torch.tensor(off, dtype=torch.int32, device=dev), off, X, W


def _check(out, off, X, W, k, factor=None, index=None):
    for g, (a, b) in enumerate(zip(off, off[1:])):
        if a == b:
            continue
        w = W[index[g] if index else g]
        f = torch.ones(b - a, 1, dtype=torch.float64, device=X.device) if factor is None else factor(g, a, b)
        want, mag = f * (X[a:b] @ w.T), f.abs() * (X[a:b].abs() @ w.abs().T)
        acc = (k + 4) * 2.0**-23 * mag
        err = (out[a:b].double() - want).abs()
        bound = acc + 2.0**-8 * (want.abs() + acc)
        assert bool((err <= bound).all()), (g, float((err / bound).max()))


@pytest.mark.parametrize("sizes,n,k,spare,most", [
    ([1], 128, 128, 0, 0),                         # the smallest call: decode tiles
    ([3, 0, 16, 1], 256, 384, 2, 16),              # decode tiles, K tail
    ([3, 0, 16, 1], 256, 512, 2, 0),
    ([300, 0, 17, 224, 1, 225], 256, 640, 40, 0),  # CTA pairs, tile edges, K tail
    ([5, 130, 0, 225], 384, 896, 3, 0),            # one CTA per tile (N % 256 != 0)
    ([700, 64], 512, 2048, 0, 0),
])
def test_product(cuda_device, sizes, n, k, spare, most):
    import ratchet_b200 as rb

    qx, pack, offsets, off, X, W = _product(cuda_device, sizes, n, k, spare, seed=n + k)
    out = torch.full((X.shape[0], n), 7.0, dtype=torch.bfloat16, device=cuda_device)
    got = rb.mxfp4_grouped_gemm_rows(*qx, offsets, pack, out=out, max_group_rows=most)
    assert got is out
    rb.last_status()
    _check(out, off, X, W, k)
    assert bool((out[off[-1]:] == 7.0).all())      # rows behind the last group


def test_product_factors_and_index(cuda_device):
    """alpha per group, a factor per row, and six groups over three weight groups."""
    import ratchet_b200 as rb

    sizes, index = [40, 0, 230, 17, 300, 9], [2, 0, 1, 2, 0, 1]
    qx, pack, offsets, off, X, W = _product(cuda_device, sizes, 256, 512, 11, 77, wgroups=3)
    alpha = torch.linspace(0.5, 3.0, 6, device=cuda_device)
    rs = torch.linspace(-2.0, 2.0, X.shape[0], device=cuda_device)
    out = rb.mxfp4_grouped_gemm_rows(*qx, offsets, pack, alpha=alpha, row_scale=rs,
                                     b_index=torch.tensor(index, dtype=torch.int32, device=cuda_device))
    rb.last_status()
    _check(out, off, X, W, 512, lambda g, a, b: alpha[g].double() * rs[a:b].double().unsqueeze(1), index)


def test_a_nan_stays_in_its_row(cuda_device):
    """A NaN token makes its own row NaN (through the NaN scale), no other."""
    import ratchet_b200 as rb

    g = torch.Generator("cuda").manual_seed(5)
    x = torch.randn(60, 256, generator=g, device=cuda_device)
    x[7, 100] = float("nan")
    w = rb.quantize_mxfp4(torch.randn(1, 128, 256, generator=g, device=cuda_device))
    off = torch.tensor([0, 60], dtype=torch.int32, device=cuda_device)
    y = rb.mxfp4_grouped_gemm_rows(*rb.quantize_mxfp4(x), off, rb.pack_mxfp4_weights(*w))
    rb.last_status()
    bad = torch.isnan(y).any(1)
    assert bool(torch.isnan(y[7]).all()) and int(bad.sum()) == 1


def test_packs_of_the_other_format_are_refused(cuda_device):
    """An NVFP4 pack given to the MXFP4 call, and the other way round, ends with status
    0x201 and writes nothing."""
    import ratchet_b200 as rb
    from ratchet_b200 import _lib

    g = torch.Generator("cuda").manual_seed(5)
    w = torch.randn(1, 256, 512, generator=g, device=cuda_device)
    x = torch.randn(64, 512, generator=g, device=cuda_device)
    off = torch.tensor([0, 64], dtype=torch.int32, device=cuda_device)
    mx = rb.pack_mxfp4_weights(*rb.quantize_mxfp4(w))
    nc, ns, _ = rb.quantize_nvfp4(w[0])
    nv = rb.pack_weights([nc], [ns])
    out = torch.full((64, 256), 7.0, dtype=torch.bfloat16, device=cuda_device)
    with pytest.raises(ValueError):
        rb.mxfp4_grouped_gemm_rows(*rb.quantize_mxfp4(x), off, nv, out=out)
    L = _lib.lib()
    qx, sx = rb.quantize_mxfp4(x)
    alpha = torch.ones(1, device=cuda_device)
    wc, ws_ = rb.quantize_mxfp4(w)
    prob = _lib.FggMxfp4RowsProblem((1, 256, 512, 64, off.data_ptr(), qx.data_ptr(), sx.data_ptr(),
                                     alpha.data_ptr(), out.data_ptr(), None, None, 1, 0),
                                    wc.data_ptr())
    stream = torch.cuda.current_stream(cuda_device).cuda_stream
    # the larger (NVFP4) pack holds every byte that the MXFP4 call could read
    ws = torch.empty(int(L.fgg_mxfp4_rows_workspace_bytes(prob)), dtype=torch.uint8, device=cuda_device)
    assert nv.buf.numel() >= mx.buf.numel()
    _lib.check(L.fgg_mxfp4_grouped_gemm_rows(prob, nv.buf.data_ptr(), ws.data_ptr(), ws.numel(), stream),
               "rows")
    assert L.fgg_read_device_status(ws.data_ptr(), stream) == _lib.FGG_ETIMEOUT
    assert int(ws[:4].view(torch.int32).item()) == 0x201
    assert bool((out == 7.0).all())
