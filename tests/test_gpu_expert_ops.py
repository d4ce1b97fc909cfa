"""The router, the 16-bit grouped products and MXFP4 as they are used: together, with
the layer, on other streams, in graphs, from two threads, over long buffers."""
import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rand(dev, *shape, seed=0, std=1.0, dtype=torch.bfloat16):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * std).to(dtype)


def _plan(ids, experts):
    """Routes grouped by expert: (order of the routes, offsets); absent routes last."""
    flat = ids.reshape(-1).long()
    key = torch.where(flat < 0, experts, flat)
    order = torch.argsort(key, stable=True)
    counts = torch.bincount(key, minlength=experts + 1)[:experts]
    off = torch.zeros(experts + 1, dtype=torch.int32, device=ids.device)
    off[1:] = counts.cumsum(0)
    return order, off


def _bound(got, want, mags, length):
    """As in test_gpu_f16: fp32 sums of exact products, one rounding."""
    half = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}[got.dtype]
    acc = length * 2.0**-23 * mags
    err = (got.double() - want).abs()
    return bool((err <= half * (want.abs() + acc) + acc + 2.0**-126).all())


def test_a_training_step(cuda_device):
    """Router, grouped products, their gradients and the router's, as a layer's step
    uses them; every call against 64 bits on the inputs that it got, and the logits'
    gradient against autograd through the whole step in 64 bits."""
    import ratchet_b200 as rb

    dev = cuda_device
    T, E, topk, H, I = 150, 12, 3, 136, 72
    x = _rand(dev, T, H, seed=1)
    logits = _rand(dev, T, E, seed=2, std=1.5, dtype=torch.float32)
    logits[:, 4] = -float("inf")                       # an expert that gets no tokens
    w1 = _rand(dev, E, 2 * I, H, seed=3, std=H**-0.5)
    w2 = _rand(dev, E, H, I, seed=4, std=I**-0.5)
    dout = _rand(dev, T, H, seed=5, dtype=torch.float32)

    ids, gate = rb.moe_router(logits, topk)
    order, off = _plan(ids, E)
    token = order // topk
    xs = x[token]
    u = rb.grouped_gemm_rows(xs, w1, off)
    a, b = u.float().chunk(2, 1)
    h = (torch.nn.functional.silu(a) * b).bfloat16()
    y = rb.grouped_gemm_rows(h, w2, off)
    wr = gate.reshape(-1)[order]
    # backward
    dy = (dout[token] * wr[:, None]).bfloat16()
    dgate = torch.zeros(T * topk, device=dev)
    dgate[order] = (dout[token] * y.float()).sum(1)
    dh = rb.grouped_gemm_rows_dgrad(dy, w2, off)
    dw2 = rb.grouped_gemm_rows_wgrad(dy, h, off)
    s = torch.sigmoid(a)
    da = dh.float() * b * s * (1 + a * (1 - s))
    db = dh.float() * a * s
    du = torch.cat((da, db), 1).bfloat16()
    dxs = rb.grouped_gemm_rows_dgrad(du, w1, off)
    dw1 = rb.grouped_gemm_rows_wgrad(du, xs, off)
    dl = rb.moe_router_backward(dgate.view(T, topk), logits, ids)
    rb.last_status()

    bounds = off.tolist()
    assert bounds[-1] == T * topk
    for g in range(E):
        lo, hi = bounds[g], bounds[g + 1]
        assert (lo == hi) == (g == 4)
        r = slice(lo, hi)
        for got, A, B in ((u[r], xs[r], w1[g].T), (y[r], h[r], w2[g].T), (dh[r], dy[r], w2[g]),
                          (dxs[r], du[r], w1[g]), (dw2[g], dy[r].T, h[r]), (dw1[g], du[r].T, xs[r])):
            A, B = A.double(), B.double()
            assert _bound(got, A @ B, A.abs() @ B.abs(), A.shape[1] + 1), g

    # the step in 64 bits: gradient of the logits through softmax over the chosen
    l64 = logits.double().requires_grad_()
    p = torch.softmax(l64, 1).gather(1, ids.long())
    g64 = (p / p.sum(1, keepdim=True)).reshape(-1)
    (dgate.double() * g64).sum().backward()
    # relative to the row's shares: expf, its argument, sums and quotients in fp32
    # (test_gpu_router's bound with span 30 and 12 experts)
    mags = (g64.detach().view(T, topk) * (2 * dgate.double().abs().view(T, topk).max(1).values[:, None])).max(1).values
    assert bool(((dl.double() - l64.grad).abs() <= (32 + 8 * 30 + 4 * E) * 2.0**-24 * mags[:, None]).all())
    assert bool((dl[:, 4] == 0).all())


def test_the_layer_takes_the_routers_output(cuda_device):
    """ExpertParallelMoE on moe_router's ids and weights, absent routes among them: the
    same bits as with the ids and weights that 64-bit arithmetic on the host gives."""
    import ratchet_b200 as rb
    from ratchet_b200.moe import ExpertParallelMoE

    dev = cuda_device
    T, E, topk, n, k = 60, 8, 3, 128, 256
    logits = _rand(dev, T, E, seed=7, dtype=torch.float32)
    logits[5, 2:] = -float("inf")                      # two experts for three routes
    logits[9] = -float("inf")                          # none
    ids, w = rb.moe_router(logits, topk)
    assert ids[5, 2].item() == -1 and ids[9].tolist() == [-1] * 3
    wq = [rb.quantize_nvfp4(_rand(dev, n, k, seed=20 + e, dtype=torch.float32)) for e in range(E)]
    xq = rb.quantize_nvfp4(_rand(dev, T, k, seed=8, dtype=torch.float32))
    layer = ExpertParallelMoE([q[0] for q in wq], [q[1] for q in wq], [q[2] for q in wq],
                              np.zeros(E, np.int32), np.arange(E, dtype=np.int32))
    y = layer.forward(xq[0], xq[1], xq[2], ids, w)
    layer.check()
    assert bool((y[9] == 0).all())
    # each token's weighted sum of its experts' rows
    L = [rb.nvfp4_grouped_gemm([xq[0]], [xq[1]], [q[0]], [q[1]], alpha=(xq[2] * q[2]).reshape(1))[0]
         for q in wq]
    rows = torch.stack(L).double()
    for t in range(T):
        live = [(int(e), float(v)) for e, v in zip(ids[t], w[t]) if e >= 0]
        assert len(live) == (0 if t == 9 else 2 if t == 5 else 3)
        want = sum((v * rows[e, t] for e, v in live), torch.zeros(n, dtype=torch.float64, device=dev))
        mag = sum((abs(v) * rows[e, t].abs() for e, v in live), torch.zeros(n, dtype=torch.float64, device=dev))
        # the layer scales rows by xq's factor apart from alpha (one more rounding of
        # the bf16 row: 2^-8 of it on either side), sums in fp32, rounds once
        assert bool(((y[t].double() - want).abs() <= 2.0**-8 * (3 * mag + want.abs()) + 2.0**-20).all())


def test_serving_in_mxfp4(cuda_device):
    """Route, quantise, one grouped product with the router's weights as row factors."""
    import ratchet_b200 as rb

    dev = cuda_device
    T, E, topk, n, k = 90, 6, 2, 256, 384
    ids, gate = rb.moe_router(_rand(dev, T, E, seed=1), topk, score="sigmoid",
                              bias=torch.zeros(E, device=dev), scale=2.0)
    order, off = _plan(ids, E)
    xs = _rand(dev, T, k, seed=2)[order // topk].contiguous()
    wq = rb.quantize_mxfp4(_rand(dev, E, n, k, seed=3, std=0.05))
    xq = rb.quantize_mxfp4(xs)
    f = gate.reshape(-1)[order].contiguous()
    y = rb.mxfp4_grouped_gemm_rows(*xq, off, rb.pack_mxfp4_weights(*wq), row_scale=f)
    rb.last_status()
    X = rb.dequantize_mxfp4(*xq, torch.float32).double() * f.double()[:, None]
    W = rb.dequantize_mxfp4(*wq, torch.float32).double()
    b = off.tolist()
    for g in range(E):
        A = X[b[g]:b[g + 1]]
        assert _bound(y[b[g]:b[g + 1]], A @ W[g].T, A.abs() @ W[g].abs().T, k + 2)


def _calls(dev, seed=0):
    """One call of each entry on its own inputs: name -> (inputs in place, call)."""
    import ratchet_b200 as rb

    sizes = [40, 0, 300, 7]
    off = torch.tensor([0, 40, 40, 340, 347], dtype=torch.int32, device=dev)
    x, dy = _rand(dev, 347, 128, seed=seed), _rand(dev, 347, 256, seed=seed + 1)
    w = _rand(dev, 4, 256, 128, seed=seed + 2, std=0.1)
    logits = _rand(dev, 347, 40, seed=seed + 3, dtype=torch.float32)
    ids, gate = rb.moe_router(logits, 4)
    pack = rb.pack_mxfp4_weights(*rb.quantize_mxfp4(w))

    def product():
        return (rb.mxfp4_grouped_gemm_rows(*rb.quantize_mxfp4(x), off, pack),)

    return {
        "fwd": ([x], lambda: (rb.grouped_gemm_rows(x, w, off),)),
        "dgrad": ([dy], lambda: (rb.grouped_gemm_rows_dgrad(dy, w, off),)),
        "wgrad": ([x, dy], lambda: (rb.grouped_gemm_rows_wgrad(dy, x, off),)),
        "router": ([logits], lambda: rb.moe_router(logits, 4, score="sigmoid",
                                                   bias=torch.zeros(40, device=dev))),
        "router backward": ([logits], lambda: (rb.moe_router_backward(gate, logits, ids),)),
        "mxfp4": ([x], product),
    }


def test_other_streams(cuda_device):
    """Each call on a stream of its own that waits for its inputs: the same bits."""
    import ratchet_b200 as rb

    calls = _calls(cuda_device)
    want = {n: [t.clone() for t in f()] for n, (_, f) in calls.items()}
    rb.last_status()
    torch.cuda.synchronize()
    streams = {n: torch.cuda.Stream() for n in calls}
    got = {}
    for _ in range(3):
        for n, (_, f) in calls.items():
            streams[n].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(streams[n]):
                got[n] = f()
    torch.cuda.synchronize()
    for n in calls:
        for a, b in zip(got[n], want[n]):
            assert torch.equal(a, b), n


def test_captured_and_replayed(cuda_device):
    """Graphs of every call, replayed in turn on changed inputs, with eager calls of
    the same entries between: each sees what its inputs hold then."""
    import ratchet_b200 as rb

    dev = cuda_device
    calls = _calls(dev)
    for _, f in calls.values():
        f()
    torch.cuda.synchronize()
    graphs = {}
    for n, (_, f) in calls.items():
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f()
        graphs[n] = (g, out)
    for step in range(3):
        for n, (inputs, f) in calls.items():
            for i, t in enumerate(inputs):
                t.copy_(_rand(dev, *t.shape, seed=100 * step + i, dtype=t.dtype))
        for n in graphs:
            graphs[n][0].replay()
        eager = {n: f() for n, (_, f) in calls.items()}
        torch.cuda.synchronize()
        for n in calls:
            for a, b in zip(graphs[n][1], eager[n]):
                assert torch.equal(a, b), (n, step)


def test_offsets_of_an_earlier_kernel(cuda_device):
    """Group sizes that a kernel on the stream has just written, other ones each time,
    without a synchronisation."""
    import ratchet_b200 as rb

    dev = cuda_device
    x, w, dy = _rand(dev, 600, 64, seed=1), _rand(dev, 5, 72, 64, seed=2), _rand(dev, 600, 72, seed=3)
    off = torch.zeros(6, dtype=torch.int32, device=dev)
    sizes = [[600, 0, 0, 0, 0], [0, 1, 599, 0, 0], [100, 200, 50, 100, 150], [0, 0, 0, 0, 17]]
    sizes = torch.tensor(sizes, dtype=torch.int32, device=dev)
    got = []
    for s in sizes:
        off[1:] = s.cumsum(0)
        out = torch.zeros(600, 72, dtype=torch.bfloat16, device=dev)
        got.append((rb.grouped_gemm_rows(x, w, off, out=out), rb.grouped_gemm_rows_wgrad(dy, x, off)))
    rb.last_status()
    for s, (y, dw) in zip(sizes.tolist(), got):
        lo = 0
        for g, m in enumerate(s):
            X, D = x[lo:lo + m].double(), dy[lo:lo + m].double()
            assert _bound(y[lo:lo + m], X @ w[g].double().T, X.abs() @ w[g].double().abs().T, 64)
            assert _bound(dw[g], D.T @ X, D.abs().T @ X.abs(), m + 1)
            lo += m
        assert bool((y[lo:] == 0).all())


@pytest.mark.parametrize("bad", [[0, 10, 5, 20], [-1, 3, 5, 20], [0, 3, 5, 65], [2**30, 2**30, 2**30, 20]])
def test_malformed_offsets_write_nothing(cuda_device, bad):
    import ratchet_b200 as rb

    dev = cuda_device
    x, dy, w = _rand(dev, 64, 64), _rand(dev, 64, 32), _rand(dev, 3, 32, 64)
    off = torch.tensor(bad, dtype=torch.int32, device=dev)
    y = torch.full((64, 32), 7.0, dtype=torch.bfloat16, device=dev)
    dx = torch.full((64, 64), 7.0, dtype=torch.bfloat16, device=dev)
    dw = torch.full((3, 32, 64), 7.0, device=dev)
    for call, out in ((lambda: rb.grouped_gemm_rows(x, w, off, out=y), y),
                      (lambda: rb.grouped_gemm_rows_dgrad(dy, w, off, out=dx), dx),
                      (lambda: rb.grouped_gemm_rows_wgrad(dy, x, off, out=dw), dw)):
        call()
        with pytest.raises(rb.FggError, match="0x203"):
            rb.last_status()
        assert bool((out == 7.0).all())
    # the next call is clean
    good = torch.tensor([0, 3, 3, 64], dtype=torch.int32, device=dev)
    rb.grouped_gemm_rows(x, w, good, out=y)
    rb.last_status()


def test_calls_without_rows(cuda_device):
    import ratchet_b200 as rb

    dev = cuda_device
    x, dy = torch.empty(0, 64, dtype=torch.bfloat16, device=dev), torch.empty(0, 32, dtype=torch.bfloat16, device=dev)
    w, off = _rand(dev, 2, 32, 64), torch.zeros(3, dtype=torch.int32, device=dev)
    assert rb.grouped_gemm_rows(x, w, off).shape == (0, 32)
    assert rb.grouped_gemm_rows_dgrad(dy, w, off).shape == (0, 64)
    assert bool((rb.grouped_gemm_rows_wgrad(dy, x, off) == 0).all())
    kept = torch.ones(2, 32, 64, device=dev)
    rb.grouped_gemm_rows_wgrad(dy, x, off, out=kept, accumulate=True)
    assert bool((kept == 1).all())
    codes, sf = rb.quantize_mxfp4(torch.empty(0, 128, device=dev))
    assert rb.dequantize_mxfp4(codes, sf).shape == (0, 128)
    pack = rb.pack_mxfp4_weights(*rb.quantize_mxfp4(_rand(dev, 2, 128, 128)))
    assert rb.mxfp4_grouped_gemm_rows(codes, sf, off, pack).shape == (0, 128)
    rb.last_status()


def test_two_threads_on_one_stream(cuda_device):
    """Host threads issue calls of different geometry on the same stream: their launches
    interleave, their workspaces do not."""
    import ratchet_b200 as rb

    dev = cuda_device
    sets = [_calls(dev, seed=50), _calls(dev, seed=60)]
    x = _rand(dev, 900, 72, seed=9)
    w = _rand(dev, 3, 520, 72, seed=10)
    off = torch.tensor([0, 500, 501, 900], dtype=torch.int32, device=dev)
    sets[1]["fwd"] = ([x], lambda: (rb.grouped_gemm_rows(x, w, off),))
    want = [{n: [t.clone() for t in f()] for n, (_, f) in c.items()} for c in sets]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            with torch.cuda.device(dev):
                for _ in range(40):
                    got = {n: f() for n, (_, f) in sets[i].items()}
                    torch.cuda.current_stream().synchronize()
                    for n, out in got.items():
                        for a, b in zip(out, want[i][n]):
                            if not torch.equal(a, b):
                                failed.append((i, n))
        except Exception as e:  # noqa: BLE001
            failed.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed[:5]


def test_long_buffers(cuda_device):
    """Element offsets past 2^31: the last rows of token tensors of 4.3 GB."""
    import ratchet_b200 as rb

    dev = cuda_device
    k, n = 4104, 8
    rows = 2**31 // k + 300
    x = torch.empty(rows, k, dtype=torch.bfloat16, device=dev)
    x.normal_(generator=torch.Generator("cuda").manual_seed(1))
    w = _rand(dev, 3, n, k, seed=2, std=k**-0.5)
    cut = [0, 5, rows - 270, rows]
    off = torch.tensor(cut, dtype=torch.int32, device=dev)
    y = rb.grouped_gemm_rows(x, w, off)
    rb.last_status()
    for lo, hi, g in ((0, 5, 0), (rows - 700, rows - 270, 1), (rows - 270, rows, 2)):
        X, W = x[lo:hi].double(), w[g].double()
        assert _bound(y[lo:hi], X @ W.T, X.abs() @ W.abs().T, k)
    dy = _rand(dev, rows, n, seed=3)
    dw = rb.grouped_gemm_rows_wgrad(dy, x, off)
    dx = rb.grouped_gemm_rows_dgrad(dy, w, off)
    rb.last_status()
    lo, hi = cut[2], cut[3]
    D, X = dy[lo:hi].double(), x[lo:hi].double()
    assert _bound(dw[2], D.T @ X, D.abs().T @ X.abs(), hi - lo + 1)
    assert _bound(dx[lo:hi], D @ w[2].double(), D.abs() @ w[2].double().abs(), n)
    del y, dx, dw, dy
    m = x.view(-1)[: x.numel() // 32 * 32]
    codes, sf = rb.quantize_mxfp4(m)
    v = rb.dequantize_mxfp4(codes, sf)
    tail = m[-4096:].contiguous()
    c2, s2 = rb.quantize_mxfp4(tail)
    assert torch.equal(codes[-2048:], c2) and torch.equal(sf[-128:].view(torch.uint8), s2.view(torch.uint8))
    assert torch.equal(v[-4096:], rb.dequantize_mxfp4(c2, s2))


def test_rows_before_the_first_group(cuda_device):
    """offsets[0] need not be 0: the rows before it are left as they are."""
    import ratchet_b200 as rb

    dev = cuda_device
    x, dy, w = _rand(dev, 90, 64, seed=1), _rand(dev, 90, 40, seed=2), _rand(dev, 2, 40, 64, seed=3)
    off = torch.tensor([13, 50, 83], dtype=torch.int32, device=dev)
    y = torch.full((90, 40), 7.0, dtype=torch.bfloat16, device=dev)
    rb.grouped_gemm_rows(x, w, off, out=y)
    dw = rb.grouped_gemm_rows_wgrad(dy, x, off)
    rb.last_status()
    assert bool((y[:13] == 7.0).all()) and bool((y[83:] == 7.0).all())
    for g, (lo, hi) in enumerate(((13, 50), (50, 83))):
        X, D, W = x[lo:hi].double(), dy[lo:hi].double(), w[g].double()
        assert _bound(y[lo:hi], X @ W.T, X.abs() @ W.abs().T, 64)
        assert _bound(dw[g], D.T @ X, D.abs().T @ X.abs(), hi - lo + 1)


def test_waits_that_run_out(cuda_device):
    """With the test hook that arms no load, every wait of the 16-bit kernels runs out
    after about a second: a status, nothing written, and a clean call after it."""
    import ratchet_b200 as rb
    from ratchet_b200 import _lib

    dev = cuda_device
    x, dy, w = _rand(dev, 700, 1024), _rand(dev, 700, 520), _rand(dev, 2, 520, 1024)
    off = torch.tensor([0, 300, 700], dtype=torch.int32, device=dev)
    y = torch.full((700, 520), 7.0, dtype=torch.bfloat16, device=dev)
    dw = torch.full((2, 520, 1024), 7.0, device=dev)
    L = _lib.lib()
    for call, out in ((lambda: rb.grouped_gemm_rows(x, w, off, out=y), y),
                      (lambda: rb.grouped_gemm_rows_wgrad(dy, x, off, out=dw), dw)):
        L.fgg_debug_set_flags(_lib.FGG_DEBUG_NO_LOADS)
        try:
            call()
            torch.cuda.synchronize()
        finally:
            L.fgg_debug_set_flags(0)
        with pytest.raises(rb.FggError, match="0x10"):
            rb.last_status()
        assert bool((out == 7.0).all())
        call()
        rb.last_status()
        assert not bool((out == 7.0).all())


def test_first_calls_inside_a_capture(cuda_device):
    """A process whose very first calls are captured: no warm-up is needed."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch, ratchet_b200 as rb
d = "cuda"
x = torch.randn(50, 64, device=d).bfloat16(); dy = torch.randn(50, 40, device=d).bfloat16()
w = torch.randn(2, 40, 64, device=d).bfloat16()
off = torch.tensor([0, 20, 50], dtype=torch.int32, device=d)
l = torch.randn(50, 9, device=d); q = torch.randn(50, 128, device=d)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = (rb.grouped_gemm_rows(x, w, off), rb.grouped_gemm_rows_dgrad(dy, w, off),
           rb.grouped_gemm_rows_wgrad(dy, x, off), *rb.moe_router(l, 2), *rb.quantize_mxfp4(q))
g.replay(); torch.cuda.synchronize()
again = (rb.grouped_gemm_rows(x, w, off), rb.grouped_gemm_rows_dgrad(dy, w, off),
         rb.grouped_gemm_rows_wgrad(dy, x, off), *rb.moe_router(l, 2), *rb.quantize_mxfp4(q))
rb.last_status()
for a, b in zip(out, again):
    a, b = (t.view(torch.uint8) if t.element_size() == 1 else t for t in (a, b))
    assert torch.equal(a, b)
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=180,
                       cwd=Path(__file__).resolve().parents[1])
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_every_group_empty(cuda_device):
    """Rows, but none in a group: nothing is written, gradients are zero."""
    import ratchet_b200 as rb

    dev = cuda_device
    x, dy, w = _rand(dev, 20, 64), _rand(dev, 20, 40), _rand(dev, 3, 40, 64)
    for at in (0, 20):
        off = torch.full((4,), at, dtype=torch.int32, device=dev)
        y = torch.full((20, 40), 7.0, dtype=torch.bfloat16, device=dev)
        dx = torch.full((20, 64), 7.0, dtype=torch.bfloat16, device=dev)
        rb.grouped_gemm_rows(x, w, off, out=y)
        rb.grouped_gemm_rows_dgrad(dy, w, off, out=dx)
        assert bool((y == 7.0).all()) and bool((dx == 7.0).all())
        assert bool((rb.grouped_gemm_rows_wgrad(dy, x, off) == 0).all())
        rb.last_status()


def test_views_at_odd_places(cuda_device):
    """Tensors that start 16 bytes (the router: an element) into their storage give the
    bits of those that start it."""
    import ratchet_b200 as rb

    dev = cuda_device

    def shift(t, by):
        buf = torch.zeros(t.numel() + by, dtype=t.dtype, device=dev)
        buf[by:].copy_(t.reshape(-1))
        return buf[by:].view(t.shape)

    off = torch.tensor([0, 33, 90], dtype=torch.int32, device=dev)
    x, dy, w = _rand(dev, 90, 72, seed=1), _rand(dev, 90, 40, seed=2), _rand(dev, 2, 40, 72, seed=3)
    xs, ds, ws = shift(x, 8), shift(dy, 8), shift(w, 8)
    assert torch.equal(rb.grouped_gemm_rows(x, w, off), rb.grouped_gemm_rows(xs, ws, off))
    assert torch.equal(rb.grouped_gemm_rows_dgrad(dy, w, off), rb.grouped_gemm_rows_dgrad(ds, ws, off))
    for dt, by in ((torch.float32, 4), (torch.bfloat16, 8)):
        want = rb.grouped_gemm_rows_wgrad(dy, x, off, out_dtype=dt)
        out = shift(torch.zeros_like(want), by)
        rb.grouped_gemm_rows_wgrad(ds, xs, off, out=out)
        assert torch.equal(out, want)
        if dt is torch.float32:
            rb.grouped_gemm_rows_wgrad(ds, xs, off, out=out, accumulate=True)
            assert torch.equal(out, want + want)
    rb.last_status()
    for dt in (torch.float32, torch.bfloat16):
        logits = _rand(dev, 70, 64, seed=4, dtype=dt)
        moved = shift(logits, 1)
        a, b = rb.moe_router(logits, 6, renormalize=False), rb.moe_router(moved, 6, renormalize=False)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        assert torch.equal(rb.moe_router_backward(a[1], logits, a[0], renormalize=False),
                           rb.moe_router_backward(a[1], moved, a[0], renormalize=False))
    q = rb.quantize_mxfp4(_rand(dev, 5, 96, seed=5))
    assert torch.equal(rb.dequantize_mxfp4(*q), rb.dequantize_mxfp4(shift(q[0], 4), shift(
        q[1].view(torch.uint8), 1)))


def test_an_index_outside_the_weights(cuda_device):
    """A device b_index that names no packed group stops the product with status 0x202
    before any load of that tile; the next call is clean."""
    import ratchet_b200 as rb

    dev = cuda_device
    pack = rb.pack_mxfp4_weights(*rb.quantize_mxfp4(_rand(dev, 2, 256, 256)))
    q = rb.quantize_mxfp4(_rand(dev, 40, 256))
    off = torch.tensor([0, 20, 40], dtype=torch.int32, device=dev)
    for bad in ([0, 2], [-1, 1]):
        rb.mxfp4_grouped_gemm_rows(*q, off, pack, b_index=torch.tensor(bad, dtype=torch.int32, device=dev))
        with pytest.raises(rb.FggError, match="0x202"):
            rb.last_status()
    rb.mxfp4_grouped_gemm_rows(*q, off, pack, b_index=torch.tensor([1, 0], dtype=torch.int32, device=dev))
    rb.last_status()


def test_outputs_that_share_memory_are_refused(cuda_device):
    import ratchet_b200 as rb

    dev = cuda_device
    off = torch.tensor([0, 4, 16], dtype=torch.int32, device=dev)
    buf = torch.zeros(4 * 16 * 64, dtype=torch.bfloat16, device=dev)
    x, w = buf[:1024].view(16, 64), _rand(dev, 2, 64, 64)
    with pytest.raises(ValueError, match="shares"):
        rb.grouped_gemm_rows(x, w, off, out=x)
    with pytest.raises(ValueError, match="shares"):
        rb.grouped_gemm_rows(x, w, off, out=buf[512:1536].view(16, 64))
    with pytest.raises(ValueError, match="shares"):
        rb.grouped_gemm_rows_dgrad(x, w, off, out=w[0, :16])
    rb.grouped_gemm_rows(x, w, off, out=buf[1024:2048].view(16, 64))
    rb.last_status()


def test_python_refusals_on_the_device(cuda_device):
    import ratchet_b200 as rb

    dev = cuda_device
    x, dy, w = _rand(dev, 16, 64), _rand(dev, 16, 32), _rand(dev, 2, 32, 64)
    off = torch.tensor([0, 4, 16], dtype=torch.int32, device=dev)
    bf, f32 = torch.bfloat16, torch.float32
    bad = [
        lambda: rb.grouped_gemm_rows(x.float(), w, off),
        lambda: rb.grouped_gemm_rows(x.half(), w, off),                   # types differ
        lambda: rb.grouped_gemm_rows(x[:, ::2], w, off),                  # strided
        lambda: rb.grouped_gemm_rows(x, w[:, :, :56].contiguous(), off),  # K differs
        lambda: rb.grouped_gemm_rows(x, w, off[:2]),                      # one group
        lambda: rb.grouped_gemm_rows(x, w, off.long()),
        lambda: rb.grouped_gemm_rows(x, w, off.cpu()),
        lambda: rb.grouped_gemm_rows(x, w, off, out=torch.empty(15, 32, dtype=bf, device=dev)),
        lambda: rb.grouped_gemm_rows(x, w, off, out=torch.empty(16, 32, dtype=f32, device=dev)),
        lambda: rb.grouped_gemm_rows(_rand(dev, 16, 60), _rand(dev, 2, 32, 60), off),
        lambda: rb.grouped_gemm_rows(_rand(dev, 16 * 64 + 1)[1:].view(16, 64), w, off),  # 2 bytes off
        lambda: rb.grouped_gemm_rows_dgrad(x, w, off),
        lambda: rb.grouped_gemm_rows_wgrad(dy, x[:15], off),
        lambda: rb.grouped_gemm_rows_wgrad(dy, x, off, out_dtype=torch.float16),
        lambda: rb.grouped_gemm_rows_wgrad(dy, x, off, accumulate=True),
        lambda: rb.grouped_gemm_rows_wgrad(dy, x, off, out=torch.empty(2, 32, 64, dtype=bf, device=dev),
                                           accumulate=True),
        lambda: rb.moe_router(x, 65),
        lambda: rb.moe_router(x, 0),
        lambda: rb.moe_router(x, 2, score="tanh"),
        lambda: rb.moe_router(x.double(), 2),
        lambda: rb.moe_router(x.t(), 2),
        lambda: rb.moe_router(x, 2, bias=torch.zeros(64, dtype=bf, device=dev)),
        lambda: rb.moe_router(x, 2, bias=torch.zeros(63, device=dev)),
        lambda: rb.moe_router(x, 2, bias=torch.zeros(64)),
        lambda: rb.moe_router_backward(torch.zeros(16, 2, device=dev), x, torch.zeros(16, 3, dtype=torch.int32, device=dev)),
        lambda: rb.moe_router_backward(torch.zeros(16, 2, device=dev), x, torch.zeros(16, 2, device=dev)),
        lambda: rb.quantize_mxfp4(x[:, :48].contiguous()),
        lambda: rb.quantize_mxfp4(x.t()),
        lambda: rb.quantize_mxfp4(x.double()),
        lambda: rb.quantize_mxfp4(_rand(dev, 65)[1:]),                    # 2 bytes off
    ]
    codes, sf = rb.quantize_mxfp4(_rand(dev, 16, 128))
    pack = rb.pack_mxfp4_weights(*rb.quantize_mxfp4(_rand(dev, 2, 128, 128)))
    bad += [
        lambda: rb.mxfp4_grouped_gemm_rows(codes, sf[:, :2], off, pack),
        lambda: rb.mxfp4_grouped_gemm_rows(codes, sf.float(), off, pack),
        lambda: rb.mxfp4_grouped_gemm_rows(codes.float(), sf, off, pack),
        lambda: rb.mxfp4_grouped_gemm_rows(codes, sf, off[:2], pack),
        lambda: rb.mxfp4_grouped_gemm_rows(codes, sf, off.cpu(), pack),
        lambda: rb.mxfp4_grouped_gemm_rows(codes, sf, off, pack, alpha=torch.ones(3, device=dev)),
        lambda: rb.mxfp4_grouped_gemm_rows(codes, sf, off, pack, max_group_rows=-1),
        lambda: rb.mxfp4_grouped_gemm_rows(codes, sf, off, pack, out=torch.empty(16, 128, device=dev)),
        lambda: rb.dequantize_mxfp4(codes, sf, torch.int32),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
    # nothing that was refused left a mark
    rb.grouped_gemm_rows(x, w, off)
    rb.last_status()


def test_status_of_a_call_on_another_stream(cuda_device):
    """last_status waits for a call on another stream than the current one."""
    import ratchet_b200 as rb

    dev = cuda_device
    x, w = _rand(dev, 64, 64), _rand(dev, 3, 32, 64)
    good = torch.tensor([0, 3, 3, 64], dtype=torch.int32, device=dev)
    bad = torch.tensor([0, 10, 5, 20], dtype=torch.int32, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rb.grouped_gemm_rows(x, w, good)
        rb.last_status()
        torch.cuda._sleep(100_000_000)               # about 50 ms
        rb.grouped_gemm_rows(x, w, bad)
    with pytest.raises(rb.FggError, match="0x203"):
        rb.last_status()


def test_status_of_two_threads(cuda_device):
    """Malformed offsets of one thread raise there, and nowhere else."""
    import ratchet_b200 as rb

    dev = cuda_device
    x, w = _rand(dev, 64, 64), _rand(dev, 3, 32, 64)
    offsets = {"good": [0, 3, 3, 64], "bad": [0, 10, 5, 20]}
    offsets = {n: torch.tensor(v, dtype=torch.int32, device=dev) for n, v in offsets.items()}
    torch.cuda.synchronize()
    called, seen = threading.Barrier(2, timeout=30), {}

    def work(name):
        with torch.cuda.device(dev):
            wrong = 0
            for _ in range(20):
                called.wait()
                rb.grouped_gemm_rows(x, w, offsets[name])
                called.wait()
                try:
                    rb.last_status()
                except rb.FggError:
                    wrong += 1
            seen[name] = wrong

    threads = [threading.Thread(target=work, args=(n,)) for n in offsets]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert seen == {"good": 0, "bad": 20}
    rb.grouped_gemm_rows(x, w, offsets["good"])
    rb.last_status()


@pytest.mark.parametrize("bad", [[0, 5, 5], [1, 1, 1], [0, 3, 0], [-1, 0, 0]])
def test_malformed_offsets_without_rows(cuda_device, bad):
    """Offsets past zero rows are malformed like any others: nothing is written, and the
    status tells."""
    import ratchet_b200 as rb

    dev = cuda_device
    x, dy = _rand(dev, 0, 64), _rand(dev, 0, 32)
    w, off = _rand(dev, 2, 32, 64), torch.tensor(bad, dtype=torch.int32, device=dev)
    good = torch.zeros(3, dtype=torch.int32, device=dev)
    dw = torch.full((2, 32, 64), 7.0, device=dev)
    for call in (lambda o: rb.grouped_gemm_rows(x, w, o),
                 lambda o: rb.grouped_gemm_rows_dgrad(dy, w, o),
                 lambda o: rb.grouped_gemm_rows_wgrad(dy, x, o, out=dw)):
        call(off)
        with pytest.raises(rb.FggError, match="0x203"):
            rb.last_status()
        assert bool((dw == 7.0).all())
        if call(good) is dw:
            assert bool((dw == 0).all())
        rb.last_status()
