"""The language-model operators beside the FP4 grouped GEMM, as cases to be measured.

Three operators of a mixture-of-experts model, each in the directions that a program calls:

* route: the router.  Scores of each token's logits over the experts, the top-k experts, their
  combine weights ("fwd"), and the gradient of the logits from that of the weights ("bwd").
* experts: products grouped by expert over contiguous token rows in bf16 or fp16, with the group
  offsets on the device: y = x W_g^T ("fwd"), dx = dy W_g ("dgrad"), dW_g = dy_g^T x_g ("wgrad").
* mxfp4: 4-bit microscaled floating point (E2M1 elements, one power-of-two scale per 32):
  quantisation and its inverse ("quant"), and the product grouped by expert of freshly quantised
  activations with weights that are held quantised ("product").

`run` computes them in plain torch where `own` is false, with the framework's entry points where it is true.
"""
import math
import random

import torch

own = False  # set from outside: False = the plain forms, True = the framework's operators

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ cases
def _route(name, tokens, experts, topk, score, bias, renorm, scale, dtype, way):
    return {"name": name, "op": "route", "way": way, "tokens": tokens, "experts": experts,
            "topk": topk, "score": score, "bias": bias, "renorm": renorm, "scale": scale,
            "dtype": dtype}


def _experts(name, way, groups, rows, n, k, dtype, skew, spare=0, out="same"):
    return {"name": name, "op": "experts", "way": way, "groups": groups, "rows": rows, "n": n,
            "k": k, "dtype": dtype, "skew": skew, "spare": spare, "out": out}


def _quant(name, rows, k, dtype):
    return {"name": name, "op": "mxfp4", "way": "quant", "rows": rows, "k": k, "dtype": dtype}


def _product(name, groups, rows, n, k, skew):
    return {"name": name, "op": "mxfp4", "way": "product", "groups": groups, "rows": rows, "n": n,
            "k": k, "skew": skew}


def listed():
    return [
        # one decode step of a small batch: latency is all there is
        _route("route decode", 24, 64, 8, "softmax", False, True, 1.0, "fp32", "fwd"),
        # a prompt of 4096 tokens over many experts, sigmoid scores with a balancing bias
        _route("route prompt", 4096, 256, 8, "sigmoid", True, True, 2.5, "fp32", "fwd"),
        # a training step's router gradient, whole softmax kept in the weights
        _route("route train", 32768, 64, 8, "softmax", False, False, 1.0, "bf16", "bwd"),
        # decode: 64 experts with a handful of tokens each, weights read once (down projection)
        _experts("experts decode", "fwd", 64, 544, 7168, 2048, "bf16", 0.0),
        # the eight-group prefill shape (fused gate and up projection)
        _experts("experts prefill", "fwd", 8, 4352, 4096, 7168, "bf16", 0.0, spare=37),
        # training, skewed loads: gradient of the tokens through the gate and up projection
        _experts("experts dgrad", "dgrad", 64, 16384, 4096, 7168, "bf16", 1.1),
        # training, skewed loads: fp32 gradient of the down projection's weights
        _experts("experts wgrad", "wgrad", 64, 32768, 7168, 2048, "bf16", 1.1, out="fp32"),
        # a small model's odd sizes in fp16, empty groups among them
        _experts("experts wgrad odd", "wgrad", 5, 333, 264, 520, "fp16", 2.0),
        # activations of 16384 tokens to MXFP4 and back
        _quant("mxfp4 quant", 16384, 7168, "bf16"),
        # a decode batch's activations from fp32
        _quant("mxfp4 quant small", 17, 2048, "fp32"),
        # serving, prefill: quantise the tokens, multiply with the quantised gate and up weights
        _product("mxfp4 prefill", 8, 4352, 4096, 7168, 0.0),
        # serving, decode: 64 experts with a handful of tokens each
        _product("mxfp4 decode", 64, 544, 7168, 2048, 0.0),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["route", "route", "experts", "experts", "experts", "quant", "product"])
    if op == "route":
        e = _log(rng, 2, 512)
        c = _route("", _log(rng, 1, 32768), e, rng.randint(1, min(16, e)),
                   rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5, rng.random() < 0.6,
                   rng.choice([1.0, 2.5]), rng.choice(["fp32", "bf16", "fp16"]),
                   rng.choice(["fwd", "bwd"]))
        if c["tokens"] * e > 32768 * 128:
            c["tokens"] = 32768 * 128 // e
        # one renormalised route has the weight 1 whatever the logits: no gradient to compare
        c["renorm"] = c["renorm"] and c["topk"] > 1
    elif op == "experts":
        way = rng.choice(["fwd", "dgrad", "wgrad"])
        g = _log(rng, 1, 96)
        n, k = 8 * _log(rng, 1, 896), 8 * _log(rng, 1, 896)
        while g * n * k > 64 * 7168 * 2048:
            g = max(1, g // 2)
            n = max(8, n // 16 * 8)
        rows = _log(rng, 1, 32768)
        rows = max(1, min(rows, 32768 * 4096 * 3584 // (n * k)))
        c = _experts("", way, g, rows, n, k, rng.choice(["bf16", "fp16"]),
                     rng.choice([0.0, 0.6, 1.1, 2.0]),
                     spare=rng.choice([0, 0, rng.randint(1, 300)]) if way != "wgrad" else 0,
                     out=rng.choice(["same", "fp32"]) if way == "wgrad" else "same")
    elif op == "quant":
        k = 32 * _log(rng, 1, 256)
        c = _quant("", max(1, min(_log(rng, 1, 32768), 16384 * 7168 // k)), k,
                   rng.choice(["fp32", "bf16", "fp16"]))
    else:
        g = _log(rng, 1, 64)
        n, k = 128 * _log(rng, 1, 56), 128 * _log(rng, 1, 56)
        while g * n * k > 64 * 7168 * 2048:
            g = max(1, g // 2)
        rows = max(1, min(_log(rng, 1, 16384), 16384 * 4096 * 2048 // (n * k)))
        c = _product("", g, rows, n, k, rng.choice([0.0, 1.1]))
    del c["name"]
    return c


# ----------------------------------------------------------------- inputs
def _sizes(groups, rows, skew, seed):
    """Rows of each group: every row goes to a group drawn with weight rank^-skew."""
    g = torch.Generator().manual_seed(seed)
    p = (torch.arange(groups, dtype=torch.float64) + 1.0) ** -skew
    p = p[torch.randperm(groups, generator=g)]
    got = torch.multinomial(p, rows, replacement=True, generator=g)
    return torch.bincount(got, minlength=groups).tolist()


def _offsets(sizes):
    off = [0]
    for s in sizes:
        off.append(off[-1] + s)
    return torch.tensor(off, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32, std=1.0):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype).mul_(std)

    s = {"case": case}
    if case["op"] == "route":
        t, e, k = case["tokens"], case["experts"], case["topk"]
        # trained routers are peaked: logits of a few units, some experts ahead of the others
        s["logits"] = (normal(t, e, std=1.5) + normal(e, std=0.7)).to(DTYPES[case["dtype"]])
        s["bias"] = normal(e, std=0.05) if case["bias"] else None
        if case["way"] == "bwd":
            s["ids"] = _route_plain(s["logits"], k, case["score"], s["bias"], case["renorm"],
                                    case["scale"])[0]
            s["dweights"] = normal(t, k, std=0.1)
    elif case["op"] == "experts":
        g, n, k, dt = case["groups"], case["n"], case["k"], DTYPES[case["dtype"]]
        rows = case["rows"] + case["spare"]  # spare rows lie behind the last group
        s["sizes"] = _sizes(g, case["rows"], case["skew"], seed)
        s["offsets"] = _offsets(s["sizes"])
        if case["way"] != "dgrad":
            s["x"] = normal(rows, k, dtype=dt)
        if case["way"] != "fwd":
            s["dy"] = normal(rows, n, dtype=dt)
        if case["way"] != "wgrad":
            s["w"] = normal(g, n, k, dtype=dt, std=k ** -0.5)
            # the program's own output buffer: rows behind the last group stay as they are
            s["out"] = torch.zeros(rows, n if case["way"] == "fwd" else k, dtype=dt, device="cuda")
    elif case["way"] == "quant":
        # rows of different size, as hidden states have
        s["x"] = (normal(case["rows"], case["k"]) * normal(case["rows"], 1).exp()).to(
            DTYPES[case["dtype"]])
    else:
        g, n, k = case["groups"], case["n"], case["k"]
        s["sizes"] = _sizes(g, case["rows"], case["skew"], seed)
        s["offsets"] = _offsets(s["sizes"])
        s["x"] = normal(case["rows"], k, dtype=torch.bfloat16)
        # E2M1 codes of normal values as their own quantiser leaves them, scales around 2^-7
        s["w_codes"] = torch.empty(g, n, k // 2, dtype=torch.uint8, device="cuda")
        s["w_sf"] = torch.empty(g, n, k // 32, dtype=torch.uint8, device="cuda")
        for i in range(g):
            q, e = _quant_plain(normal(n, k, std=0.02))
            s["w_codes"][i], s["w_sf"][i] = _codes_of(q), (e + 127).to(torch.uint8)
        if own:  # a serving program packs its weights once
            import ratchet_b200

            s["pack"] = ratchet_b200.pack_mxfp4_weights(s["w_codes"], s["w_sf"])
    return s


# ------------------------------------------------------------ plain forms
def _route_plain(logits, topk, score, bias, renorm, scale):
    """Scores in 64 bits (the top-k borders lie close together), ids by score and lowest index."""
    x = logits.double()
    p = torch.softmax(x, 1) if score == "softmax" else torch.sigmoid(x)
    # without a bias the order of the scores is the order of the logits
    key = x if bias is None else p + bias.double()
    ids = torch.sort(key, dim=1, descending=True, stable=True)[1][:, :topk]
    w = p.gather(1, ids)
    if renorm:
        w = w / w.sum(1, keepdim=True)
    return ids.to(torch.int32), (w * scale).float()


def _route_backward_plain(dw, logits, ids, score, renorm, scale):
    x, ids, dw = logits.float(), ids.long(), dw * scale
    p = torch.softmax(x, 1) if score == "softmax" else torch.sigmoid(x)
    s = p.gather(1, ids)
    if renorm:
        total = s.sum(1, keepdim=True)
        ds = (dw - (dw * s).sum(1, keepdim=True) / total) / total
    else:
        ds = dw
    dp = torch.zeros_like(p).scatter_(1, ids, ds)
    if score == "softmax":
        dx = p * (dp - (dp * p).sum(1, keepdim=True))
    else:
        dx = dp * p * (1.0 - p)
    return dx.to(logits.dtype)


def _quant_plain(x):
    """x [.., K] -> (elements [.., K] on the E2M1 grid, exponents [.., K/32]) in fp32."""
    x = x.float().unflatten(-1, (-1, 32))
    amax = x.abs().amax(-1, keepdim=True)
    # amax = m 2^e with m in [1, 2): frexp gives m/2 and e+1; the largest E2M1 exponent is 2
    e = torch.where(amax > 0, torch.frexp(amax)[1] - 3, -127).clamp(min=-127)
    y = torch.ldexp(x, -e)
    a = y.abs()
    q = torch.zeros_like(a)
    # round to nearest: each threshold lies half way, ties go to the even code
    q = torch.where(a > 0.25, 0.5, q)
    q = torch.where(a >= 0.75, 1.0, q)
    q = torch.where(a > 1.25, 1.5, q)
    q = torch.where(a >= 1.75, 2.0, q)
    q = torch.where(a > 2.5, 3.0, q)
    q = torch.where(a >= 3.5, 4.0, q)
    q = torch.where(a > 5.0, 6.0, q)
    return torch.copysign(q, y).flatten(-2), e.squeeze(-1)


def _codes_of(q):
    """E2M1 codes of values on the grid, two to a byte, the first in the low half."""
    a = q.abs()
    c = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    c = c | (torch.signbit(q).to(torch.uint8) << 3)
    c = c.unflatten(-1, (-1, 2))
    return c[..., 0] | (c[..., 1] << 4)


_GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def _values_of(codes, sf):
    """Codes [.., K/2] and scale bytes [.., K/32] -> fp32 values [.., K]."""
    grid = torch.tensor(_GRID, device=codes.device)
    v = torch.stack((grid[(codes & 15).int()], grid[(codes >> 4).int()]), -1).flatten(-2)
    return torch.ldexp(v.unflatten(-1, (-1, 32)), sf.int().unsqueeze(-1) - 127).flatten(-2)


def _run_plain(s):
    case = s["case"]
    if case["op"] == "route":
        if case["way"] == "fwd":
            ids, w = _route_plain(s["logits"], case["topk"], case["score"], s["bias"],
                                  case["renorm"], case["scale"])
            return {"ids": ids, "weights": w}
        return {"dlogits": _route_backward_plain(s["dweights"], s["logits"], s["ids"],
                                                 case["score"], case["renorm"], case["scale"])}
    if case["op"] == "experts":
        sizes, rows = s["sizes"], case["rows"]
        if case["way"] == "fwd":
            y = [a.float() @ w.float().T for a, w in zip(s["x"][:rows].split(sizes), s["w"])]
            s["out"][:rows] = torch.cat(y).to(s["out"].dtype)
            return {"y": s["out"]}
        if case["way"] == "dgrad":
            dx = [a.float() @ w.float() for a, w in zip(s["dy"][:rows].split(sizes), s["w"])]
            s["out"][:rows] = torch.cat(dx).to(s["out"].dtype)
            return {"dx": s["out"]}
        dt = torch.float32 if case["out"] == "fp32" else DTYPES[case["dtype"]]
        return {"dw": torch.stack([(a.float().T @ b.float()).to(dt) for a, b in
                                   zip(s["dy"].split(sizes), s["x"].split(sizes))])}
    if case["way"] == "quant":
        q, e = _quant_plain(s["x"])
        v = torch.ldexp(q.unflatten(-1, (-1, 32)), e.unsqueeze(-1)).flatten(-2)
        return {"values": v.to(s["x"].dtype), "scales": torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)}
    q, e = _quant_plain(s["x"])
    a = torch.ldexp(q.unflatten(-1, (-1, 32)), e.unsqueeze(-1)).flatten(-2)
    y = [r @ _values_of(c, f).T for r, c, f in zip(a.split(s["sizes"]), s["w_codes"], s["w_sf"])]
    return {"y": torch.cat(y).to(torch.bfloat16)}


# --------------------------------------------------- the framework's calls
def _run_own(s):
    import ratchet_b200 as rb

    case = s["case"]
    if case["op"] == "route":
        if case["way"] == "fwd":
            ids, w = rb.moe_router(s["logits"], case["topk"], score=case["score"], bias=s["bias"],
                                   renormalize=case["renorm"], scale=case["scale"])
            return {"ids": ids, "weights": w}
        return {"dlogits": rb.moe_router_backward(s["dweights"], s["logits"], s["ids"],
                                                  score=case["score"], renormalize=case["renorm"],
                                                  scale=case["scale"])}
    if case["op"] == "experts":
        if case["way"] == "fwd":
            return {"y": rb.grouped_gemm_rows(s["x"], s["w"], s["offsets"], out=s["out"])}
        if case["way"] == "dgrad":
            return {"dx": rb.grouped_gemm_rows_dgrad(s["dy"], s["w"], s["offsets"], out=s["out"])}
        dt = torch.float32 if case["out"] == "fp32" else DTYPES[case["dtype"]]
        return {"dw": rb.grouped_gemm_rows_wgrad(s["dy"], s["x"], s["offsets"], out_dtype=dt)}
    codes, sf = rb.quantize_mxfp4(s["x"])
    if case["way"] == "quant":
        return {"values": rb.dequantize_mxfp4(codes, sf, dtype=s["x"].dtype),
                "scales": sf.to(torch.float32)}
    return {"y": rb.mxfp4_grouped_gemm_rows(codes, sf, s["offsets"], s["pack"])}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------- work
def _bytes(dtype):
    return 4 if dtype == "fp32" else 2


def work(case):
    if case["op"] == "route":
        t, e, k = case["tokens"], case["experts"], case["topk"]
        logits = t * e * _bytes(case["dtype"])
        if case["way"] == "fwd":
            return {"bytes": logits + 8 * t * k + (4 * e if case["bias"] else 0), "flops": 4 * t * e}
        return {"bytes": 2 * logits + 8 * t * k, "flops": 6 * t * e}
    if case["way"] == "quant":
        count = case["rows"] * case["k"]
        # the values, their scales in fp32, and the codes and scale bytes between the two calls
        return {"bytes": count * (2 * _bytes(case["dtype"]) + 1 + 6 / 32), "flops": 4 * count}
    g, rows, n, k = case["groups"], case["rows"], case["n"], case["k"]
    flops = 2 * rows * n * k
    held = min(g, rows)  # groups without rows need no weights
    if case["op"] == "mxfp4":
        return {"bytes": rows * (2 * k + 2 * n) + 17 * held * n * k // 32, "flops": flops}
    out = 4 if case["out"] == "fp32" else 2
    if case["way"] == "wgrad":
        return {"bytes": 2 * rows * (n + k) + out * g * n * k, "flops": flops}
    return {"bytes": 2 * rows * (n + k) + 2 * held * n * k, "flops": flops}


# ------------------------------------------------- the definitions in 64 bits
def _two_to(e):
    """2^e in 64 bits, from its bits (a power function may be off in the last place)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _grid_exact(y):
    """Nearest E2M1 value: steps of 1/2 below 2, of 1 below 4, of 2 above, ties to even."""
    a = y.abs()
    step = 0.5 + 0.5 * (a >= 2).double() + (a >= 4).double()
    return torch.sign(y) * (torch.round(a / step) * step).clamp(max=6.0)


def _mx_exact(x):
    """Values after quantisation and the scales, of x in 64 bits."""
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    top = b.abs().max(-1, keepdim=True).values
    # floor(log2) without a logarithm's rounding: 64-bit values keep their exponent in bits 52..62
    bits = (top.view(torch.int64) >> 52) & 0x7FF
    e = torch.where(top > 0, bits - 1023 - 2, torch.full_like(bits, -127)).clamp(min=-127)
    scale = _two_to(e)
    return (_grid_exact(b / scale) * scale).reshape(x.shape), scale.squeeze(-1)


def _weights_exact(codes, sf):
    c = torch.stack((codes % 16, codes // 16), -1).reshape(*codes.shape[:-1], -1).double()
    sign = torch.where(c >= 8, -1.0, 1.0).double()
    m, half = torch.div(c % 8, 2, rounding_mode="floor"), c % 2
    v = torch.where(m == 0, 0.5 * half, (1 + 0.5 * half) * _two_to(m - 1))
    scale = _two_to(sf.long() - 127).repeat_interleave(32, -1)
    return sign * v * scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        x = s["logits"].double()
        if case["score"] == "softmax":
            z = torch.exp(x - x.max(1, keepdim=True).values)
            p = z / z.sum(1, keepdim=True)
        else:
            p = 1.0 / (1.0 + torch.exp(-x))
        if case["way"] == "fwd":
            key = x if s["bias"] is None else p + s["bias"].double()
            chosen = torch.argsort(-key, dim=1, stable=True)[:, :case["topk"]]
            w = torch.take_along_dim(p, chosen, 1)
            if case["renorm"]:
                w = w / w.sum(1, keepdim=True)
            return {"ids": None, "weights": case["scale"] * w}
        # the gradient by the Jacobian of the chosen weights, one row of it per expert
        ids, dw = s["ids"].long(), s["dweights"].double() * case["scale"]
        t = torch.take_along_dim(p, ids, 1)
        if case["renorm"]:
            total = t.sum(1, keepdim=True)
            g = dw / total - (dw * t).sum(1, keepdim=True) / total ** 2
        else:
            g = dw
        if case["score"] == "softmax":
            dx = -p * (g * t).sum(1, keepdim=True)
            dx.scatter_add_(1, ids, g * t)
        else:
            dx = torch.zeros_like(p)
            dx.scatter_add_(1, ids, g * t * (1 - t))
        return {"dlogits": dx}
    if case["way"] == "quant":
        v, scale = _mx_exact(s["x"])
        return {"values": v, "scales": scale}
    bounds = [int(v) for v in s["offsets"].tolist()]
    spans = [(g, a, b) for g, (a, b) in enumerate(zip(bounds, bounds[1:])) if b > a]
    if case["op"] == "mxfp4":
        a = _mx_exact(s["x"])[0]
        y = torch.zeros(case["rows"], case["n"], dtype=torch.float64, device="cuda")
        for g, lo, hi in spans:
            y[lo:hi] = torch.mm(a[lo:hi], _weights_exact(s["w_codes"][g], s["w_sf"][g]).t())
        return {"y": y}
    if case["way"] == "wgrad":
        dw = torch.zeros(case["groups"], case["n"], case["k"], dtype=torch.float64, device="cuda")
        for g, lo, hi in spans:
            torch.mm(s["dy"][lo:hi].double().t(), s["x"][lo:hi].double(), out=dw[g])
        return {"dw": dw}
    src = s["x"] if case["way"] == "fwd" else s["dy"]
    y = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    for g, lo, hi in spans:
        w = s["w"][g].double()
        y[lo:hi] = torch.mm(src[lo:hi].double(), w.t() if case["way"] == "fwd" else w)
    return {"y" if case["way"] == "fwd" else "dx": y}
