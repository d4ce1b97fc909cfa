"""moe_router and moe_router_backward against their definitions in 64 bits.

Ids have to be equal.  Tolerance of the weights: expf is off by at most 2 steps
(2^-22 of its value), its argument by half a step of the difference it is taken of
(|l - m| 2^-24, which expf turns into a relative error), a sum of E terms by E 2^-24,
a quotient by 2^-24: with X the largest |l - m| a weight is off by at most
(16 + 4 X + 2 E) 2^-24 of its value.  A gradient is a sum of products of those with
dw: the same share of the sum of their magnitudes, and half a step of its type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
INF = float("inf")


def _logits(dev, t, e, dtype, seed, std=1.5):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(t, e, generator=g, device=dev) * std).to(dtype)


def _scores(l, score):
    """fp64 scores of one row as a list; masked experts have 0."""
    l = [float(v) for v in l]
    if score == "sigmoid":
        return [0.0 if v == -INF else (1 / (1 + math.exp(-v)) if v > -700 else 0.0) for v in l]
    m = max(l)
    if m == -INF:
        return [0.0] * len(l)
    z = [math.exp(v - m) for v in l]
    s = math.fsum(z)
    return [v / s for v in z]


def _route(l, bias, topk, score):
    s = _scores(l, score)
    key = [float(v) for v in l] if bias is None else [
        -INF if float(v) == -INF else p + float(b) for v, p, b in zip(l, s, bias)]
    order = sorted((e for e in range(len(key)) if key[e] > -INF), key=lambda e: (-key[e], e))
    return (order + [-1] * topk)[:topk], s


def _check(logits, topk, score, bias, renorm, scale, ids, weights):
    x = logits.double().cpu()
    b = None if bias is None else bias.double().cpu().tolist()
    for t in range(x.shape[0]):
        l = x[t].tolist()
        want, s = _route(l, b, topk, score)
        assert ids[t].tolist() == want, (t, ids[t].tolist(), want)
        live = [v for v in l if v > -INF]
        span = max(abs(v) for v in live) + max(live) - min(live) if live else 0.0
        tol = (16 + 4 * span + 2 * len(l)) * 2.0**-24
        chosen = [s[e] if e >= 0 else 0.0 for e in want]
        total = math.fsum(chosen) if renorm else 1.0
        for j, c in enumerate(chosen):
            w = scale * c / total if total > 0 else 0.0
            got = float(weights[t, j])
            assert abs(got - w) <= tol * abs(w) + 2.0**-126, (t, j, got, w)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True], ids=["plain", "bias"])
@pytest.mark.parametrize("t,e,topk,dtype", [
    (1, 1, 1, torch.float32),
    (3, 7, 7, torch.bfloat16),
    (33, 64, 8, torch.float16),
    (17, 65, 2, torch.bfloat16),
    (9, 256, 8, torch.float32),
    (5, 500, 32, torch.bfloat16),
    (6, 1024, 16, torch.float32),
    (21, 60, 32, torch.float32),      # more routes than a token has lanes
    (4, 128, 17, torch.float16),
    (3, 512, 9, torch.bfloat16),
])
def test_forward(cuda_device, score, biased, t, e, topk, dtype):
    import ratchet_b200 as rb

    logits = _logits(cuda_device, t, e, dtype, seed=e + t)
    bias = _logits(cuda_device, 1, e, torch.float32, seed=5, std=0.05)[0] if biased else None
    for renorm, scale in ((True, 1.0), (False, 2.5)):
        ids, w = rb.moe_router(logits, topk, score=score, bias=bias, renormalize=renorm, scale=scale)
        assert ids.dtype is torch.int32 and w.dtype is torch.float32
        _check(logits, topk, score, bias, renorm, scale, ids.cpu(), w.cpu())


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_ties_go_to_the_lowest_index(cuda_device, score):
    """Whole-number logits tie often; -0 equals +0; equal biases keep the ties."""
    import ratchet_b200 as rb

    g = torch.Generator("cuda").manual_seed(3)
    logits = torch.randint(-2, 3, (40, 96), generator=g, device=cuda_device).float()
    logits[::2] *= -1.0  # makes -0
    bias = torch.full((96,), 0.25, device=cuda_device)
    for b in (None, bias):
        ids, w = rb.moe_router(logits, 8, score=score, bias=b)
        _check(logits, 8, score, b, True, 1.0, ids.cpu(), w.cpu())


def test_orders_that_32_bits_cannot_tell(cuda_device):
    """Scores plus biases that differ by less than a step of fp32: the order is the
    one in 64 bits."""
    import ratchet_b200 as rb

    e = 48
    g = torch.Generator("cuda").manual_seed(11)
    logits = torch.randn(64, e, generator=g, device=cuda_device)
    # biases that level the scores of row 0 up to fp32 rounding
    s = torch.sigmoid(logits[0].double())
    bias = (1.0 - s).float()
    logits[1:] = logits[0] + 1e-6 * torch.randn(63, e, generator=g, device=cuda_device)
    ids, w = rb.moe_router(logits, 8, score="sigmoid", bias=bias)
    _check(logits, 8, "sigmoid", bias, True, 1.0, ids.cpu(), w.cpu())


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True], ids=["plain", "bias"])
def test_masked_experts(cuda_device, score, biased):
    """-inf logits are never chosen, whatever their bias; rows with fewer experts than
    routes, and with none; the type's lowest value is a number like others."""
    import ratchet_b200 as rb

    logits = _logits(cuda_device, 6, 40, torch.float32, seed=8)
    logits[0, 3:] = -INF           # three experts for eight routes
    logits[1, :] = -INF            # none
    logits[2, ::2] = -INF
    logits[3, :36] = torch.finfo(torch.float32).min
    bias = None
    if biased:
        bias = torch.zeros(40, device=cuda_device)
        bias[20:] = 5.0            # larger than any score
        bias[39] = -INF            # a bias masks too
    ids, w = rb.moe_router(logits, 8, score=score, bias=bias)
    # sigmoid scores of the lowest value vanish: their weights are zero
    _check(logits, 8, score, bias, True, 1.0, ids.cpu(), w.cpu())
    assert ids[1].tolist() == [-1] * 8 and w[1].tolist() == [0.0] * 8


def test_small_sigmoid_scores_keep_their_ratio(cuda_device):
    """exp(-120) is no fp32 number, but the normalised weights are."""
    import ratchet_b200 as rb

    logits = torch.tensor([[-120.0, -121.0, -119.0, -150.0]], device=cuda_device)
    ids, w = rb.moe_router(logits, 3, score="sigmoid")
    assert ids[0].tolist() == [2, 0, 1]
    z = [math.exp(-119 + 119), math.exp(-1), math.exp(-2)]
    for j in range(3):
        assert abs(float(w[0, j]) - z[j] / sum(z)) <= 600 * 2.0**-24 * z[j]


def test_rows_without_numbers(cuda_device):
    """A NaN logit (softmax: +inf too) makes its row's weights NaN, no other's; ids
    stay in range."""
    import ratchet_b200 as rb

    base = _logits(cuda_device, 4, 33, torch.float32, seed=9)
    for score in ("softmax", "sigmoid"):
        for bias in (None, torch.zeros(33, device=cuda_device)):
            logits = base.clone()
            logits[1, 5] = float("nan")
            logits[2, 7] = INF
            ids, w = rb.moe_router(logits, 4, score=score, bias=bias)
            assert bool(torch.isnan(w[1]).all())
            assert bool(torch.isnan(w[2]).all()) == (score == "softmax")
            assert bool(((ids >= -1) & (ids < 33)).all())
            ok = torch.tensor([0, 3], device=cuda_device)
            _check(logits[ok], 4, score, bias, True, 1.0, ids[ok].cpu(), w[ok].cpu())


# ------------------------------------------------------------------ gradient
def _grad(l, ids, dw, score, renorm, scale):
    """(dl, magnitudes) of one row in 64 bits, from the formula."""
    s = _scores(l, score)
    E = len(l)
    d = [0.0] * E
    mag = [0.0] * E
    live = [(j, e) for j, e in enumerate(ids) if 0 <= e < E]
    total = math.fsum(s[e] for _, e in live)
    dp = [0.0] * E
    dpm = [0.0] * E
    for j, e in live:
        if renorm:
            dot = math.fsum(dw[i] * s[f] / total for i, f in live)
            dots = math.fsum(abs(dw[i]) * s[f] / total for i, f in live)
            dp[e] += scale * (dw[j] - dot) / total
            dpm[e] += abs(scale) * (abs(dw[j]) + dots) / total
        else:
            dp[e] += scale * dw[j]
            dpm[e] += abs(scale * dw[j])
    if score == "softmax":
        # over the chosen, sum_j s_j (dw_j - dot) / total = dot - dot = 0: the formula's sum
        # would be its own rounding, against which an expert that was not chosen is compared
        whole = 0.0 if renorm else math.fsum(p * v for p, v in zip(s, dp))
        wholem = math.fsum(p * v for p, v in zip(s, dpm))
        for e in range(E):
            d[e] = s[e] * (dp[e] - whole)
            mag[e] = s[e] * (dpm[e] + (0.0 if renorm else wholem))
    else:
        for e in range(E):
            d[e] = dp[e] * s[e] * (1 - s[e])
            mag[e] = dpm[e] * s[e] * (1 - s[e])
    return d, mag


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("t,e,topk,dtype", [
    (1, 1, 1, torch.float32),
    (5, 9, 3, torch.bfloat16),
    (19, 64, 8, torch.float32),
    (7, 130, 5, torch.float16),
    (4, 512, 32, torch.bfloat16),
    (3, 1000, 9, torch.float32),
    (18, 61, 32, torch.bfloat16),     # more routes than a token has lanes, odd rows
    (5, 128, 17, torch.float16),
])
def test_backward(cuda_device, score, renorm, t, e, topk, dtype):
    import ratchet_b200 as rb

    logits = _logits(cuda_device, t, e, dtype, seed=100 + e)
    ids, _ = rb.moe_router(logits, topk, score=score)
    if t > 1 and topk > 1:
        ids[1, 0] = -1                 # an absent route
        ids[0, 1] = ids[0, 0]          # the same expert twice
        ids[t - 1, topk - 1] = e + 5   # out of range: absent
    g = torch.Generator("cuda").manual_seed(4)
    dw = torch.randn(t, topk, generator=g, device=cuda_device)
    got = rb.moe_router_backward(dw, logits, ids, score=score, renormalize=renorm, scale=1.5)
    assert got.dtype is dtype and got.shape == logits.shape
    x = logits.double().cpu()
    for r in range(t):
        l = x[r].tolist()
        d, mag = _grad(l, ids[r].tolist(), dw[r].double().tolist(), score, renorm, 1.5)
        span = 2 * max(abs(v) for v in l)
        tol = (32 + 8 * span + 4 * e) * 2.0**-24
        tiny = torch.finfo(dtype).tiny
        for i in range(e):
            bound = tol * mag[i] + HALF[dtype] * max(abs(d[i]) + tol * mag[i], tiny)
            assert abs(float(got[r, i]) - d[i]) <= bound, (r, i, float(got[r, i]), d[i])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_backward_against_differences(cuda_device, score, renorm):
    """Central differences of the definition in 64 bits, at fixed ids."""
    import ratchet_b200 as rb

    e, topk, h = 24, 4, 1e-4
    logits = _logits(cuda_device, 2, e, torch.float32, seed=21)
    ids, _ = rb.moe_router(logits, topk, score=score)
    g = torch.Generator("cuda").manual_seed(6)
    dw = torch.randn(2, topk, generator=g, device=cuda_device)
    got = rb.moe_router_backward(dw, logits, ids, score=score, renormalize=renorm).cpu()

    def loss(l, r):
        s = _scores(l, score)
        c = [s[i] for i in ids[r].tolist()]
        total = math.fsum(c) if renorm else 1.0
        return math.fsum(float(dw[r, j]) * v / total for j, v in enumerate(c))

    for r in range(2):
        l = logits[r].double().tolist()
        for i in range(e):
            up, down = list(l), list(l)
            up[i] += h
            down[i] -= h
            want = (loss(up, r) - loss(down, r)) / (2 * h)
            # third derivatives are at most a few times |dw|: h^2 of them, and fp32
            assert abs(float(got[r, i]) - want) <= 1e-6, (r, i)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_gradient_where_one_route_has_nearly_all_the_weight(cuda_device, score):
    """Weights 1 - 1e-5 and 1e-5: the gradient w_0 w_1 (dw_0 - dw_1) keeps its relative
    accuracy, which the difference dw_0 - (w_0 dw_0 + w_1 dw_1) would lose."""
    import ratchet_b200 as rb

    logits = torch.tensor([[-2.0, -14.0, -30.0]], device=cuda_device)
    ids = torch.tensor([[0, 1]], dtype=torch.int32, device=cuda_device)
    dw = torch.tensor([[1.25, 0.5]], device=cuda_device)
    d = rb.moe_router_backward(dw, logits, ids, score=score).double().cpu()[0]
    s = _scores(logits[0].double().tolist(), score)
    w = [s[0] / (s[0] + s[1]), s[1] / (s[0] + s[1])]
    for i, sign in ((0, 1), (1, -1)):
        want = sign * w[0] * w[1] * 0.75 * (1.0 if score == "softmax" else 1 - s[i])
        # expf of up to 28 twice, quotients, products: test_backward's share of the value
        assert abs(float(d[i]) - want) <= (32 + 8 * 28 + 12) * 2.0**-24 * abs(want)
    assert float(d[2]) == 0.0


def test_masked_rows_have_no_gradient(cuda_device):
    import ratchet_b200 as rb

    logits = _logits(cuda_device, 3, 12, torch.float32, seed=2)
    logits[0, 2:] = -INF
    logits[1, :] = -INF
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            ids, _ = rb.moe_router(logits, 4, score=score, renormalize=renorm)
            d = rb.moe_router_backward(torch.ones(3, 4, device=cuda_device), logits, ids,
                                       score=score, renormalize=renorm)
            assert bool(torch.isfinite(d).all())
            assert bool((d[1] == 0).all()) and bool((d[0, 2:] == 0).all())


def test_no_tokens(cuda_device):
    import ratchet_b200 as rb

    ids, w = rb.moe_router(torch.empty(0, 8, device=cuda_device), 2)
    assert ids.shape == (0, 2) and w.shape == (0, 2)
    d = rb.moe_router_backward(w, torch.empty(0, 8, device=cuda_device), ids)
    assert d.shape == (0, 8)


@pytest.mark.parametrize("e", [3, 64, 130, 300, 700])
@pytest.mark.parametrize("lead", [2.0, 18.0, 25.0, 60.0])
@pytest.mark.parametrize("chosen", [[0], [0, 2], [2, 0], [1, 2], [0, 0, 2], [0, 1, 2]])
def test_whole_softmax_gradient_where_one_expert_has_nearly_all_the_score(cuda_device, e, lead,
                                                                         chosen):
    """dl_i = s_i [ D_i (1 - S) + sum_f s_f (D_i - D_f) ] of a chosen expert (S the chosen
    ones' score, D an expert's summed dw), -s_i sum_f s_f D_f of another, to a share of the
    magnitudes of these terms: a score's error twice (its own and that of s_f or 1 - S),
    a step for each addition over the routes, one for each difference and product."""
    import ratchet_b200 as rb

    logits = _logits(cuda_device, 2, e, torch.float32, seed=e, std=0.5)
    logits[:, 0] = logits[:, 1:].max(1).values + lead
    topk = len(chosen)
    ids = torch.tensor([chosen, chosen[::-1]], dtype=torch.int32, device=cuda_device)
    dw = torch.tensor([[1.25, -0.5, 2.0][:topk], [0.75, 0.5, 1.0][:topk]], device=cuda_device)
    got = rb.moe_router_backward(dw, logits, ids, renormalize=False, scale=0.5).cpu()
    for r in range(2):
        l = logits[r].double().tolist()
        m = max(l)
        z = [math.exp(v - m) for v in l]
        total = math.fsum(z)
        D = {}
        for f, v in zip(ids[r].tolist(), dw[r].tolist()):
            D[f] = D.get(f, 0.0) + 0.5 * v
        rest = math.fsum(v for i, v in enumerate(z) if i not in D) / total
        tol = (48 + 8 * (m - min(l)) + 4 * e + topk) * 2.0**-24
        for i in range(e):
            s = z[i] / total
            if i in D:
                terms = [D[i] * rest] + [z[f] / total * (D[i] - D[f]) for f in D]
            else:
                terms = [-z[f] / total * D[f] for f in D]
            want, mag = s * math.fsum(terms), s * math.fsum(abs(v) for v in terms)
            assert abs(float(got[r, i]) - want) <= tol * mag + 2.0**-126, (r, i, float(got[r, i]), want)


def test_whole_softmax_gradient_of_masked_routes(cuda_device):
    """A route to a masked expert is absent, whatever its dw."""
    import ratchet_b200 as rb

    logits = _logits(cuda_device, 2, 12, torch.float32, seed=3)
    logits[:, 5] = -INF
    ids = torch.tensor([[1, 5, 2], [1, -1, 2]], dtype=torch.int32, device=cuda_device)
    dw = torch.tensor([[1.0, INF, -2.0]] * 2, device=cuda_device)
    logits[1] = logits[0]
    d = rb.moe_router_backward(dw, logits, ids, renormalize=False)
    assert bool(torch.isfinite(d).all()) and torch.equal(d[0], d[1]) and float(d[0, 5]) == 0.0
