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


@pytest.mark.parametrize("rows", [496, 512, 513, 1024, 1039, 4100])
def test_wgrad_chunks(cuda_device, rows):
    """Groups around and past the rows that one accumulator sums; the others of the
    same call are short."""
    import ratchet_b200 as rb

    sizes, n, k = [3, rows, 0, 70], 72, 136
    x, dy, w, offsets, off = _problem(cuda_device, sizes, n, k, torch.bfloat16, seed=rows)
    dw = rb.grouped_gemm_rows_wgrad(dy, x, offsets)
    rb.last_status()
    _check_wgrad(dy, x, dw, off)


SPLIT = [
    # sizes, n, k, spare rows: calls of few tiles, or of a few long ones, in which tiles
    # are cut along the contraction.  A slice's sum has fewer additions than the whole,
    # and at most four join it to the others: the bound above still holds.
    ([1], 256, 4096, 0),                 # one token, one tile
    ([0, 1, 0, 0], 4096, 2056, 3),       # contraction not a multiple of a step
    ([33, 0, 256], 264, 5128, 0),        # tiles over the output's edge, all columns
    ([300], 520, 2048, 2),               # several token tiles
    ([5000], 64, 64, 0),                 # one small gradient over many rows
    ([4999, 0, 3, 70], 136, 264, 7),     # one of four, with rows left over a sixteen
    ([2100, 9000, 2099], 72, 8, 1),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("case", range(len(SPLIT)))
def test_few_tiles(cuda_device, case, dtype):
    """Right, and the same bits however the slices' ends fall: again and again, and in
    a captured graph."""
    import ratchet_b200 as rb

    sizes, n, k, spare = SPLIT[case]
    x, dy, w, offsets, off = _problem(cuda_device, sizes, n, k, dtype, spare, seed=case)
    start = torch.randn(len(sizes), n, k, device=cuda_device)
    outs = [torch.full((x.shape[0], n), 7.0, dtype=dtype, device=cuda_device),
            torch.full((x.shape[0], k), 7.0, dtype=dtype, device=cuda_device),
            torch.empty(len(sizes), n, k, device=cuda_device),
            torch.empty(len(sizes), n, k, dtype=dtype, device=cuda_device), start.clone()]

    def run():
        rb.grouped_gemm_rows(x, w, offsets, out=outs[0])
        rb.grouped_gemm_rows_dgrad(dy, w, offsets, out=outs[1])
        rb.grouped_gemm_rows_wgrad(dy, x, offsets, out=outs[2])
        rb.grouped_gemm_rows_wgrad(dy, x, offsets, out=outs[3])
        outs[4].copy_(start)
        rb.grouped_gemm_rows_wgrad(dy, x, offsets, out=outs[4], accumulate=True)

    run()
    rb.last_status()
    _check_fwd(x, w, outs[0], off)
    _check_dgrad(dy, w, outs[1], off)
    _check_wgrad(dy, x, outs[2], off)
    _check_wgrad(dy, x, outs[3], off)
    _check_wgrad(dy, x, outs[4], off, start)
    for o in outs[:2]:
        assert bool((o[off[-1]:] == 7.0).all())
    first = [o.clone() for o in outs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for i in range(20):
        for o in outs:
            o.fill_(float("nan"))
        if i < 10:
            run()
        else:
            graph.replay()
        rb.last_status()
        for o, f, r in zip(outs, first, [off[-1], off[-1], None, None, None]):
            assert torch.equal(o[:r], f[:r])


def test_few_tiles_on_two_streams(cuda_device):
    """Two streams' calls at once, each with sums of its own; then offsets that are
    malformed in a call whose tiles would be split."""
    import ratchet_b200 as rb

    cases = [_problem(cuda_device, [2000 + 900 * i, 0, 3], 72, 328, torch.bfloat16, seed=i)
             for i in range(2)]
    want = [rb.grouped_gemm_rows_wgrad(dy, x, off) for x, dy, _, off, _ in cases]
    rb.last_status()
    for (x, dy, _, _, off), w in zip(cases, want):
        _check_wgrad(dy, x, w, off)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i, (st, (x, dy, _, off, _)) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(st):
                got[i].append(rb.grouped_gemm_rows_wgrad(dy, x, off))
    torch.cuda.synchronize()
    for gs, w in zip(got, want):
        assert all(torch.equal(g, w) for g in gs)
    x, dy = cases[0][:2]
    out = torch.full((3, 72, 328), 7.0, device=cuda_device)
    bad = torch.tensor([0, 2000, 1000, x.shape[0]], dtype=torch.int32, device=cuda_device)
    rb.grouped_gemm_rows_wgrad(dy, x, bad, out=out)
    with pytest.raises(rb.FggError):
        rb.last_status()
    assert bool((out == 7.0).all())
    assert torch.equal(rb.grouped_gemm_rows_wgrad(dy, x, cases[0][3]), want[0])
    rb.last_status()


def test_wgrad_long_sums_do_not_drift(cuda_device):
    """16384 rows of one sign, where truncating additions would lose the most: 16384 / 16
    of them 2^-24 each on average, 6e-5 of the sum.  With 512 rows to a chunk it is at
    most 32 truncations of 2^-23 and 32 roundings of 2^-24 of the sum: 6e-6."""
    import ratchet_b200 as rb

    g = torch.Generator("cuda").manual_seed(1)
    rows, n, k = 16384, 64, 64
    x = torch.rand(rows, k, generator=g, device=cuda_device).bfloat16()
    dy = torch.rand(rows, n, generator=g, device=cuda_device).bfloat16()
    off = torch.tensor([0, rows], dtype=torch.int32, device=cuda_device)
    dw = rb.grouped_gemm_rows_wgrad(dy, x, off)
    rb.last_status()
    want = dy.double().T @ x.double()
    assert float(((dw[0].double() - want).abs() / want).max()) <= 32 * 2.0**-23 + 32 * 2.0**-24


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_wgrad_accumulates(cuda_device, dtype):
    """Two microbatches into one fp32 gradient; an empty group's is left as it is."""
    import ratchet_b200 as rb

    sizes, n, k = [33, 0, 300, 5], 264, 72
    x, dy, w, offsets, off = _problem(cuda_device, sizes, n, k, dtype, seed=3)
    start = torch.randn(4, n, k, device=cuda_device)
    dw = start.clone()
    got = rb.grouped_gemm_rows_wgrad(dy, x, offsets, out=dw, accumulate=True)
    rb.last_status()
    assert got is dw
    _check_wgrad(dy, x, dw, off, start)
    assert torch.equal(dw[1], start[1])
    # the same call twice from the same start gives the same bits
    again = start.clone()
    rb.grouped_gemm_rows_wgrad(dy, x, offsets, out=again, accumulate=True)
    assert torch.equal(dw, again)


def test_infinities_stay_in_their_group(cuda_device):
    """Infinities and NaN in the rows of one group, in the rows behind the last and in
    the neighbours of a ragged tile reach no other group's results."""
    import ratchet_b200 as rb

    sizes, n, k, spare = [37, 21, 50], 128, 192, 20
    x, dy, w, offsets, off = _problem(cuda_device, sizes, n, k, torch.bfloat16, spare, seed=8)
    bad = torch.tensor([float("inf"), float("nan"), -float("inf")], device=cuda_device).bfloat16()
    for t in (x, dy):
        t[37:58] = bad[torch.arange(t.shape[1], device=cuda_device) % 3]
        t[108:] = float("nan")
    y = rb.grouped_gemm_rows(x, w, offsets)
    dx = rb.grouped_gemm_rows_dgrad(dy, w, offsets)
    dw = rb.grouped_gemm_rows_wgrad(dy, x, offsets)
    rb.last_status()
    for a, b, g in ((0, 37, 0), (58, 108, 2)):
        assert bool(torch.isfinite(y[a:b]).all()) and bool(torch.isfinite(dx[a:b]).all())
        D, X, W = dy[a:b].double(), x[a:b].double(), w[g].double()
        _close(y[a:b], X @ W.T, X.abs() @ W.abs().T, k, ("fwd", g))
        _close(dx[a:b], D @ W, D.abs() @ W.abs(), n, ("dgrad", g))
        _close(dw[g], D.T @ X, D.abs().T @ X.abs(), b - a + 1, ("wgrad", g))
    assert not bool(torch.isfinite(y[37:58]).any()) and not bool(torch.isfinite(dw[1]).any())
