"""grouped_gemm_rows and its two gradients against plain products in 64 bits.

Tolerance.  Operands are exact in bf16 / fp16, products of two of them exact in
fp32; a sum of L products is held in fp32, each addition off by at most 2^-23 of
the magnitudes added so far (the tensor core may truncate), so the sum is off by
at most L 2^-23 S with S the sum of the products' magnitudes; it is then rounded
once to the output type, by at most half a step of it (2^-8 bf16, 2^-11 fp16) of
the value, or of the type's smallest normal number below it (fp16 2^-14).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def _problem(dev, sizes, n, k, dtype, spare=0, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    rows = sum(sizes) + spare
    x = torch.randn(rows, k, generator=g, device=dev).to(dtype)
    dy = torch.randn(rows, n, generator=g, device=dev).to(dtype)
    w = (torch.randn(len(sizes), n, k, generator=g, device=dev) * k**-0.5).to(dtype)
    off = [0]
    for s in sizes:
        off.append(off[-1] + s)
    return x, dy, w, torch.tensor(off, dtype=torch.int32, device=dev), off


def _close(got, want, mags, length, where):
    """|got - want| <= half a step of the output type + the sum's own error."""
    half = HALF[got.dtype]
    tiny = torch.finfo(got.dtype).tiny
    acc = length * 2.0**-23 * mags
    bound = (want.abs() + acc).clamp(min=tiny) * half + acc
    err = (got.double() - want).abs()
    bad = err > bound
    assert not bool(bad.any()), (where, float((err / bound).max()), bad.nonzero()[:4].tolist())


def _spans(off):
    return [(g, a, b) for g, (a, b) in enumerate(zip(off, off[1:]))]


def _check_fwd(x, w, out, off):
    for g, a, b in _spans(off):
        if b > a:
            X, W = x[a:b].double(), w[g].double()
            _close(out[a:b], X @ W.T, X.abs() @ W.abs().T, x.shape[1], ("fwd", g))


def _check_dgrad(dy, w, out, off):
    for g, a, b in _spans(off):
        if b > a:
            D, W = dy[a:b].double(), w[g].double()
            _close(out[a:b], D @ W, D.abs() @ W.abs(), dy.shape[1], ("dgrad", g))


def _check_wgrad(dy, x, out, off, start=None):
    for g, a, b in _spans(off):
        D, X = dy[a:b].double(), x[a:b].double()
        want, mags = D.T @ X, D.abs().T @ X.abs()
        if start is not None:
            want, mags = want + start[g].double(), mags + start[g].double().abs()
        _close(out[g], want, mags, b - a + 1, ("wgrad", g))


CASES = [
    # sizes, n, k, spare rows
    ([1], 8, 8, 0),                                # the smallest call
    ([1, 0, 2, 31, 33], 264, 520, 5),              # ragged against every tile edge
    ([0, 255, 256, 257, 0, 300], 256, 64, 3),      # token tile edges
    ([17, 64], 128, 1024, 0),                      # half a pair tile of weights
    ([5, 700, 0, 90], 520, 328, 11),               # several token tiles
    ([40] * 9, 1032, 72, 0),                       # contraction a little over a step
    ([3] * 100, 64, 200, 40),                      # many small groups
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_forward_and_gradients(cuda_device, case, dtype):
    import ratchet_b200 as rb

    sizes, n, k, spare = CASES[case]
    x, dy, w, offsets, off = _problem(cuda_device, sizes, n, k, dtype, spare, seed=case)
    y = torch.full((x.shape[0], n), 7.0, dtype=dtype, device=cuda_device)
    assert rb.grouped_gemm_rows(x, w, offsets, out=y) is y
    rb.last_status()
    _check_fwd(x, w, y, off)
    assert bool((y[off[-1]:] == 7.0).all())        # rows behind the last group
    dx = torch.full((x.shape[0], k), 7.0, dtype=dtype, device=cuda_device)
    rb.grouped_gemm_rows_dgrad(dy, w, offsets, out=dx)
    rb.last_status()
    _check_dgrad(dy, w, dx, off)
    assert bool((dx[off[-1]:] == 7.0).all())
    for dt in (torch.float32, dtype):
        dw = rb.grouped_gemm_rows_wgrad(dy, x, offsets, out_dtype=dt)
        rb.last_status()
        assert dw.dtype is dt
        _check_wgrad(dy, x, dw, off)
        for g, a, b in _spans(off):
            if a == b:
                assert bool((dw[g] == 0).all())
