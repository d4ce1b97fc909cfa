"""Tiles of the 16-bit grouped products that are cut along the contraction.

The workspace's words 4 and 5 tell how many tiles a call cut and into how many units,
and each case states its own, so that a case that no longer splits fails.  Tolerances
are test_gpu_f16's: a slice's sum has fewer additions than the whole, and at most four
joins follow, so the bound of a sum of as many products still holds.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
FWD, DGRAD, WGRAD = 0, 1, 2


def _close(got, want, mags, length, where):
    acc = length * 2.0**-23 * mags
    bound = (want.abs() + acc).clamp(min=torch.finfo(got.dtype).tiny) * HALF[got.dtype] + acc
    bad = (got.double() - want).abs() > bound
    assert not bool(bad.any()), (where, bad.nonzero()[:4].tolist())


class _Problem:
    """Operands of groups of the given sizes, with `spare` rows behind the last."""

    def __init__(self, dev, sizes, n, k, dtype, spare=0, seed=0):
        g = torch.Generator("cuda").manual_seed(seed)
        rows = sum(sizes) + spare
        rand = lambda *s: torch.randn(*s, generator=g, device=dev)
        self.x, self.dy = rand(rows, k).to(dtype), rand(rows, n).to(dtype)
        self.w = (rand(len(sizes), n, k) * k**-0.5).to(dtype)
        self.cut = [0]
        for s in sizes:
            self.cut.append(self.cut[-1] + s)
        self.off = torch.tensor(self.cut, dtype=torch.int32, device=dev)
        self.G, self.n, self.k, self.rows = len(sizes), n, k, rows

    def call(self, direction, out=None, off=None, accumulate=False):
        """(result, workspace) of one call of the C entry on a workspace of its own."""
        from ratchet_b200 import _lib, ops

        dev = self.x.device
        a = self.x if direction == FWD else self.dy
        b = self.x if direction == WGRAD else self.w
        if out is None:
            shape = {FWD: (self.rows, self.n), DGRAD: (self.rows, self.k),
                     WGRAD: (self.G, self.n, self.k)}[direction]
            out = torch.full(shape, 7.0, device=dev,
                             dtype=torch.float32 if direction == WGRAD else self.x.dtype)
        code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
        off = self.off if off is None else off
        p = _lib.FggF16RowsProblem(self.G, self.n, self.k, self.rows, code[a.dtype],
                                   code[out.dtype], int(accumulate), off.data_ptr(), a.data_ptr(),
                                   b.data_ptr(), out.data_ptr())
        L = _lib.lib()
        nbytes = L.fgg_f16_rows_workspace_bytes(p, direction)
        assert nbytes > 0
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        rc = L.fgg_f16_grouped_gemm_rows(p, direction, ws.data_ptr(), nbytes, ops._stream_ptr(dev))
        _lib.check(rc, "grouped_gemm_rows")
        return out, ws

    def check(self, direction, out, start=None):
        for g, (lo, hi) in enumerate(zip(self.cut, self.cut[1:])):
            X, D, W = self.x[lo:hi].double(), self.dy[lo:hi].double(), self.w[g].double()
            if direction == FWD:
                _close(out[lo:hi], X @ W.T, X.abs() @ W.abs().T, self.k, ("fwd", g))
            elif direction == DGRAD:
                _close(out[lo:hi], D @ W, D.abs() @ W.abs(), self.n, ("dgrad", g))
            else:
                want, mags = D.T @ X, D.abs().T @ X.abs()
                if start is not None:
                    want, mags = want + start[g].double(), mags + start[g].double().abs()
                _close(out[g], want, mags, hi - lo + 1, ("wgrad", g))
        if direction != WGRAD:
            assert bool((out[self.cut[-1]:] == 7.0).all())


def _split(ws):
    """(status, tiles cut, their units)"""
    words = ws[:24].view(torch.int32).tolist()
    return words[0], words[4], words[5]


CASES = [
    # direction, sizes, n, k, spare rows, tiles cut, units
    (FWD, [1], 256, 4096, 0, 1, 2),               # one token, one tile of 64 steps
    (FWD, [33], 256, 6144, 2, 1, 3),
    (FWD, [1, 0, 200], 264, 8192, 0, 4, 16),      # a second tile of 8 columns
    (FWD, [250], 520, 10240, 5, 3, 15),
    (FWD, [3], 8, 14336, 0, 1, 7),
    (FWD, [256, 70], 256, 32768, 0, 2, 32),
    (DGRAD, [1], 4096, 256, 0, 1, 2),
    (DGRAD, [9], 6144, 520, 3, 3, 9),
    (DGRAD, [0, 31, 200], 10248, 264, 0, 4, 20),  # the contraction ends inside a step
    (DGRAD, [2], 14336, 72, 0, 1, 7),
    (DGRAD, [130], 32776, 8, 1, 1, 16),
    (WGRAD, [4096], 64, 64, 0, 1, 2),             # a gradient of one tile
    (WGRAD, [6150], 72, 8, 0, 1, 3),
    (WGRAD, [10247], 264, 8, 4, 2, 10),
    (WGRAD, [7, 14336, 0], 136, 72, 0, 1, 7),
    (WGRAD, [33001], 8, 520, 0, 3, 48),
    (WGRAD, [9000, 100, 9001], 72, 136, 0, 2, 8),  # two of three groups
]


def _pairs(dev):
    return torch.cuda.get_device_properties(dev).multi_processor_count // 2


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_split_tiles(cuda_device, case, dtype):
    """Cut as stated, right, and the same bits in every run and in a replayed graph."""
    if _pairs(cuda_device) != 74:
        pytest.skip("the counts are those of 148 SMs")
    direction, sizes, n, k, spare, tiles, units = CASES[case]
    q = _Problem(cuda_device, sizes, n, k, dtype, spare, seed=case)
    first, ws = q.call(direction)
    assert _split(ws) == (0, tiles, units)
    q.check(direction, first)
    out = torch.empty_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = q.call(direction, out)
    for i in range(12):
        out.fill_(7.0)
        if i < 6:
            ws = q.call(direction, out)[1]
        else:
            graph.replay()
            ws = kept[1]
        assert _split(ws) == (0, tiles, units)
        assert torch.equal(out, first)
    if direction == WGRAD:
        start = torch.randn(first.shape, device=cuda_device)
        got = start.clone()
        q.call(direction, got, accumulate=True)
        assert torch.equal(got, start + first)     # one addition per element
        half = torch.empty(first.shape, dtype=dtype, device=cuda_device)
        q.call(direction, half)
        assert torch.equal(half, first.to(dtype))  # the same sums, rounded once


@pytest.mark.parametrize("direction,m,n,k", [
    (FWD, 200, 256, 4096), (FWD, 1, 520, 6144), (DGRAD, 40, 4096, 72), (WGRAD, 4097, 64, 64),
    (WGRAD, 5000, 264, 72)])
def test_spare_rows_and_empty_groups_change_nothing(cuda_device, direction, m, n, k):
    """The same bits from a group alone, with rows behind it, and among empty groups."""
    q = _Problem(cuda_device, [m], n, k, torch.bfloat16, seed=m)
    want = q.call(direction)[0]
    q.check(direction, want)
    for sizes, spare in (([m], 1), ([m], 900), ([0, m, 0, 0], 0), ([m, 0], 4000)):
        r = _Problem(cuda_device, sizes, n, k, torch.bfloat16, spare, seed=m)
        g = sizes.index(m)
        r.x[:m], r.dy[:m], r.w[g] = q.x, q.dy, q.w[0]
        got = r.call(direction)[0]
        assert torch.equal(got[g] if direction == WGRAD else got[:m],
                           want[0] if direction == WGRAD else want)


def test_split_calls_on_two_streams(cuda_device):
    """Two streams' split calls at once, each on its own sums."""
    if _pairs(cuda_device) != 74:
        pytest.skip("the counts are those of 148 SMs")
    cases = [_Problem(cuda_device, [9000 + 900 * i, 0, 3], 72, 328, torch.bfloat16, seed=i)
             for i in range(2)]
    want = []
    for q in cases:
        out, ws = q.call(WGRAD)
        assert _split(ws) == (0, 2, 8)
        q.check(WGRAD, out)
        want.append(out)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i, (st, q) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(st):
                got[i].append(q.call(WGRAD))
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        for o, ws in outs:
            assert _split(ws) == (0, 2, 8) and torch.equal(o, w)


def test_malformed_offsets_of_a_call_that_would_split(cuda_device):
    q = _Problem(cuda_device, [9000, 0, 3], 72, 328, torch.bfloat16)
    bad = torch.tensor([0, 9000, 8000, 9003], dtype=torch.int32, device=cuda_device)
    out, ws = q.call(WGRAD, off=bad)
    assert _split(ws) == (0x203, 0, 0) and bool((out == 7.0).all())
    q.check(WGRAD, q.call(WGRAD)[0])
