"""What stands beside the products of this library as it is measured on it: the product with bias, activation and residual
for any number of rows on GGUF-quantized weights, its backward pass with the weights frozen, and the mixture-of-experts
layer of a few tokens (router, choice of experts, their gated feed-forward products, weighted sum).

Shapes are those of an 8B decoder (hidden 4096, key/value 1024, feed-forward 14336), as in the benchmark and the tests, the
same as eight experts of that size, many small experts, plus odd and ragged ones.  `draw` spreads sizes, formats and types
over the same ranges.
"""
import math
import os
import sys

import torch

own = False

ELEMS = {"q4_0": 32, "q8_0": 32, "q4_k": 256, "q6_k": 256}
BYTES = {"q4_0": 18, "q8_0": 34, "q4_k": 144, "q6_k": 210}
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
LARGEST = 2048 * 14336 * 4096  # multiply-adds of the largest listed product
EXPERTS = 8 * 14336 * 4096     # weights of the largest listed expert tensor


def _gq():
    path = os.path.join(os.getcwd(), "gretacore-v3_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import gq
    return gq


def listed():
    return [
        # key projection of one token with its bias: the smallest call of a decode step
        {"name": "linear_kv_token", "kind": "linear", "fmt": "q8_0", "m": 1, "n": 1024, "k": 4096, "dt": "bf16",
         "bias": "bf16"},
        # down projection of one token, added to the hidden state
        {"name": "linear_down_token", "kind": "linear", "fmt": "q4_k", "m": 1, "n": 4096, "k": 14336, "dt": "bf16",
         "resid": True},
        # the same of twelve sequences decoded together, with a bias in f32
        {"name": "linear_down_batch", "kind": "linear", "fmt": "q6_k", "m": 12, "n": 4096, "k": 14336, "dt": "f16",
         "bias": "f32", "resid": True},
        # first product of an ungated feed-forward block on a ragged prompt, odd row count of the weights, kept for a
        # backward pass
        {"name": "linear_ragged_train", "kind": "linear", "fmt": "q8_0", "m": 509, "n": 8191, "k": 4096, "dt": "f16",
         "bias": "f16", "act": "gelu", "save": True},
        # down projection of a full 2048-token chunk of a prompt
        {"name": "linear_down_prompt", "kind": "linear", "fmt": "q4_k", "m": 2048, "n": 4096, "k": 14336, "dt": "bf16",
         "resid": True},
        # backward of a short ragged sequence
        {"name": "linear_bwd_ragged", "kind": "bwd", "fmt": "q6_k", "m": 203, "n": 5003, "k": 4096, "dt": "f16",
         "act": "gelu"},
        # backward of a full 2048-token step
        {"name": "linear_bwd", "kind": "bwd", "fmt": "q4_0", "m": 2048, "n": 14336, "k": 4096, "dt": "bf16", "act": "relu"},
        # one token, many small experts: the smallest expert layer, where latency counts
        {"name": "moe_token_small", "kind": "moe", "fmt": "q4_k", "down": "q4_k", "m": 1, "e": 64, "top": 8, "n": 1024,
         "k": 2048, "dt": "bf16", "router": "f32"},
        # one token, two of eight experts of the 8B decoder's size, the mixed formats of a k-quant file
        {"name": "moe_token", "kind": "moe", "fmt": "q4_k", "down": "q6_k", "m": 1, "e": 8, "top": 2, "n": 14336,
         "k": 4096, "dt": "bf16", "router": "f32", "resid": True},
        # sixteen sequences decoded together on the same experts
        {"name": "moe_batch_16", "kind": "moe", "fmt": "q4_0", "down": "q4_0", "m": 16, "e": 8, "top": 2, "n": 14336,
         "k": 4096, "dt": "f16", "router": "f16"},
        # odd counts: 37 tokens, 61 experts, sizes of whole 32-blocks only; sigmoid scores with a selection bias
        {"name": "moe_batch_ragged", "kind": "moe", "fmt": "q8_0", "down": "q4_0", "m": 37, "e": 61, "top": 5, "n": 1376,
         "k": 2080, "dt": "bf16", "router": "bf16", "score": "sigmoid", "resid": True},
        # the most tokens of one call, every expert taken
        {"name": "moe_batch_64", "kind": "moe", "fmt": "q4_k", "down": "q6_k", "m": 64, "e": 128, "top": 8, "n": 768,
         "k": 2048, "dt": "bf16", "router": "f32"},
    ]


def _size(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "bwd", "moe", "moe"])
    case = {"kind": kind, "fmt": rng.choice(sorted(ELEMS)), "dt": rng.choice(["bf16", "f16"])}
    if kind == "moe":
        down = rng.choice([case["fmt"], rng.choice(sorted(ELEMS))])
        e = _size(rng, 2, 128)
        unit_n, unit_k = ELEMS[down], ELEMS[case["fmt"]]
        n = max(1, _size(rng, 256, 14336) // unit_n) * unit_n
        k = max(1, _size(rng, 512, 4096) // unit_k) * unit_k
        n = max(1, min(n, EXPERTS // (e * k)) // unit_n) * unit_n
        case.update(down=down, m=_size(rng, 1, 64), e=e, top=rng.randint(1, min(8, e)), n=n, k=k,
                    router=rng.choice(["f32", "f32", "bf16", "f16"]), score=rng.choice(["softmax", "softmax", "sigmoid"]),
                    resid=rng.random() < 0.5)
        return case
    m, n = _size(rng, 1, 2048), _size(rng, 64, 14336)
    k = max(1, _size(rng, 512, 14336) // ELEMS[case["fmt"]]) * ELEMS[case["fmt"]]
    n = max(1, min(n, LARGEST // (m * k)))
    case.update(m=m, n=n, k=k, act=rng.choice(["none", "none", "relu", "silu", "gelu"]))
    if kind == "linear":
        case.update(save=rng.random() < 0.3, resid=rng.random() < 0.5)
        if rng.random() < 0.6:
            case["bias"] = rng.choice(["f32", case["dt"]])
    return case


# ---- inputs -------------------------------------------------------------------
def _half_bytes(t):
    return t.to(torch.float16).reshape(-1, 1).view(torch.uint8)


def _codes(nb, per, mean, std, lo, hi, g):
    return torch.randn(nb, per, generator=g, device="cuda").mul_(std).add_(mean).round_().clamp_(lo, hi).to(torch.uint8)


def _blocks(fmt, n, k, g):
    """GGUF blocks of an n x k tensor of roughly normal weights of size 0.02."""
    nb = n * (k // ELEMS[fmt])
    u = 0.75 + 0.5 * torch.rand(nb, generator=g, device="cuda")
    if fmt == "q4_0":
        q = _codes(nb, 32, 8.0, 2.7, 0, 15, g)
        sign = 1 - 2 * torch.randint(0, 2, (nb,), generator=g, device="cuda")
        return torch.cat([_half_bytes(0.0074 * u * sign), q[:, :16] | (q[:, 16:] << 4)], 1)
    if fmt == "q8_0":
        q = _codes(nb, 32, 128.0, 42.0, 1, 255, g) ^ 128  # (two's complement)
        return torch.cat([_half_bytes(0.00048 * u), q], 1)
    if fmt == "q4_k":  # (d, dmin, 12 B of 6-bit scales and mins, 128 B of nibble pairs)
        sc = torch.randint(20, 60, (nb, 8), generator=g, device="cuda")
        mn = (sc + torch.randint(-3, 4, (nb, 8), generator=g, device="cuda")).clamp(0, 63)
        q = _codes(nb, 256, 7.5, 3.2, 0, 15, g)

        def six(v):  # four codes with the low 2 bits of the next four on top, then those codes' high nibbles
            top = v[:, 4:] >> 2
            return [v[:, :4] | ((v[:, 4:] & 3) << 6), top[:, 0:1] | (top[:, 1:2] << 4),
                    top[:, 2:3] | (top[:, 3:4] << 4)]

        d = (0.00016 * u).to(torch.float16)
        return torch.cat([_half_bytes(d), _half_bytes(d.float() * 7.5),
                          torch.cat(six(sc) + six(mn), 1).to(torch.uint8), q[:, 0::2] | (q[:, 1::2] << 4)], 1)
    q = _codes(nb, 256, 32.0, 11.0, 0, 63, g)
    lo, hi = q & 15, q >> 4
    sc = torch.randint(24, 100, (nb, 16), generator=g, device="cuda")
    sc = (sc * (1 - 2 * torch.randint(0, 2, (nb, 16), generator=g, device="cuda"))).to(torch.int8)
    return torch.cat([lo[:, 0::2] | (lo[:, 1::2] << 4),
                      hi[:, 0::4] | (hi[:, 1::4] << 2) | (hi[:, 2::4] << 4) | (hi[:, 3::4] << 6),
                      sc.view(torch.uint8), _half_bytes(0.00003 * u)], 1)


def _x(m, k, g):
    """Activations: normal, with a spread of channel sizes as a normalised hidden state has."""
    return torch.randn(m, k, generator=g, device="cuda") * torch.exp(0.5 * torch.randn(k, generator=g, device="cuda"))


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, m, n, k, dt = case["kind"], case["m"], case["n"], case["k"], DTYPE[case["dt"]]
    if kind == "moe":
        e = case["e"]
        # an expert's tensors behind the last one's, as in the three-dimensional tensors of a GGUF file
        s = {"gate": _blocks(case["fmt"], e * n, k, g), "up": _blocks(case["fmt"], e * n, k, g),
             "down": _blocks(case["down"], e * k, n, g)}
        s["x"] = _x(m, k, g).to(dt)
        # logits of size 1.2
        s["router"] = (torch.randn(e, k, generator=g, device="cuda") * (0.9 / k ** 0.5)).to(DTYPE[case["router"]])
        if case.get("score") == "sigmoid":
            s["rbias"] = 0.1 * torch.randn(e, generator=g, device="cuda")
        if case.get("resid"):
            s["resid"] = (2 * torch.randn(m, k, generator=g, device="cuda")).to(dt)
        return s
    s = {"w": _blocks(case["fmt"], n, k, g)}
    if kind == "linear":
        s["x"] = _x(m, k, g).to(dt)
        if "bias" in case:
            s["bias"] = (0.5 * torch.randn(n, generator=g, device="cuda")).to(DTYPE[case["bias"]])
        if case.get("resid"):
            s["resid"] = (2 * torch.randn(m, n, generator=g, device="cuda")).to(dt)
        return s
    # the kept products of a forward pass, and gradients of a mean over tokens: sizes differ from token to token, and
    # one token in eight (prompts, padding) has none
    s["z"] = (1.5 * torch.randn(m, n, generator=g, device="cuda")).to(dt)
    tok = torch.exp(torch.randn(m, 1, generator=g, device="cuda"))
    tok = tok * (torch.rand(m, 1, generator=g, device="cuda") >= 0.125)
    s["dy"] = (1e-2 * tok * torch.randn(m, n, generator=g, device="cuda")).to(dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # the weights as a program keeps them: laid out once when they are loaded
        gq = _gq()
        n, k = case["n"], case["k"]
        if case["kind"] == "moe":
            e = case["e"]
            for name in ("gate", "up"):
                s[name] = gq.repack(gq.FORMATS[case["fmt"]], s[name], e * n, k)
            s["down"] = gq.repack(gq.FORMATS[case["down"]], s["down"], e * k, n)
        else:
            s["w"] = gq.repack(gq.FORMATS[case["fmt"]], s["w"], n, k)
        s["ws"] = gq.Workspace("cuda")
    s["case"] = case
    return s


# ---- the operators ---------------------------------------------------------------
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    gq, c = _gq(), s["case"]
    kind, n, k, fmt = c["kind"], c["n"], c["k"], gq.FORMATS[c["fmt"]]
    if kind == "moe":
        score = {"softmax": gq.SCORE_SOFTMAX, "sigmoid": gq.SCORE_SIGMOID}[c.get("score", "softmax")]
        y, ids, weights = gq.moe_layer(fmt, s["gate"], s["up"], gq.FORMATS[c["down"]], s["down"], s["router"], s["x"], n, k,
                                       c["e"], c["top"], score=score, router_bias=s.get("rbias"), resid=s.get("resid"),
                                       save=True, workspace=s["ws"])
        return {"y": y, "ids": ids, "weights": weights}
    act = {"none": gq.ACT_NONE, "relu": gq.ACT_RELU, "silu": gq.ACT_SILU, "gelu": gq.ACT_GELU_TANH}[c.get("act", "none")]
    if kind == "linear":
        out = gq.linear(fmt, s["w"], s["x"], n, k, bias=s.get("bias"), act=act, resid=s.get("resid"),
                        save=c.get("save", False), workspace=s["ws"])
        return dict(zip("yz", out)) if c.get("save") else out
    return gq.linear_bwd(fmt, s["w"], s["dy"], s["z"], n, k, act=act, want_dbias=True, workspace=s["ws"])


def _plain_blocks(fmt, b, n, k):
    """GGUF blocks -> f32 [n][k]."""
    def half(col):
        return b[:, col:col + 2].contiguous().view(torch.float16).float()

    if fmt == "q4_0":
        q = b[:, 2:]
        w = (torch.cat([q & 15, q >> 4], 1).float() - 8) * half(0)
    elif fmt == "q8_0":
        w = b[:, 2:].contiguous().view(torch.int8).float() * half(0)
    elif fmt == "q4_k":
        s = b[:, 4:16].int()

        def six(v):
            hi = torch.stack([v[:, 4] & 15, v[:, 4] >> 4, v[:, 5] & 15, v[:, 5] >> 4], 1)
            return torch.cat([v[:, :4] & 63, (v[:, :4] >> 6) | (hi << 2)], 1).float()

        sc, mn = six(s[:, :6]) * half(0), six(s[:, 6:]) * half(2)
        q = b[:, 16:]
        q = torch.stack([q & 15, q >> 4], 2).reshape(-1, 8, 32).float()
        w = q * sc[:, :, None] - mn[:, :, None]
    else:
        ql, qh = b[:, :128], b[:, 128:192]
        lo = torch.stack([ql & 15, ql >> 4], 2).reshape(-1, 256)
        hi = torch.stack([(qh >> (2 * j)) & 3 for j in range(4)], 2).reshape(-1, 256)
        sc = b[:, 192:208].contiguous().view(torch.int8).float() * half(208)
        w = ((lo | (hi << 4)).float() - 32).reshape(-1, 16, 16) * sc[:, :, None]
    return w.reshape(n, k)


def _plain_act(act, z):
    """act(z) and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z * (z > 0), (z > 0).float()
    if act == "silu":
        sg = 1 / (1 + torch.exp(-z))
        return z * sg, sg * (1 + z * (1 - sg))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def _plain_route(s, c):
    """Experts and their weights: the choice in 64 bits, where two experts may lie close."""
    logits = s["x"].double() @ s["router"].double().t()
    if c.get("score") == "sigmoid":
        p = 1 / (1 + torch.exp(-logits))
        key = p + s["rbias"].double()
    else:
        p = torch.exp(logits - logits.amax(1, keepdim=True))
        key = logits
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :c["top"]]
    w = p.gather(1, ids)
    return ids.int(), (w / w.sum(1, keepdim=True)).float()


def _plain_moe(s, c):
    n, k, e = c["n"], c["k"], c["e"]
    ids, weights = _plain_route(s, c)
    x = s["x"].float()
    y = s["resid"].float() if c.get("resid") else torch.zeros_like(x)
    wide, narrow = n * (k // ELEMS[c["fmt"]]), k * (n // ELEMS[c["down"]])  # blocks of an expert
    for i in sorted(set(ids.flatten().tolist())):
        tok, slot = (ids == i).nonzero(as_tuple=True)
        gate = _plain_blocks(c["fmt"], s["gate"][i * wide:(i + 1) * wide], n, k)
        up = _plain_blocks(c["fmt"], s["up"][i * wide:(i + 1) * wide], n, k)
        xi = x[tok]
        h = _plain_act("silu", xi @ gate.t())[0] * (xi @ up.t())
        out = h @ _plain_blocks(c["down"], s["down"][i * narrow:(i + 1) * narrow], k, n).t()
        y = y.index_add(0, tok, out * weights[tok, slot][:, None])
    return {"y": y.to(DTYPE[c["dt"]]), "ids": ids, "weights": weights}


def _run_plain(s):
    c = s["case"]
    kind, n, k, dt = c["kind"], c["n"], c["k"], DTYPE[c["dt"]]
    if kind == "moe":
        return _plain_moe(s, c)
    w, act = _plain_blocks(c["fmt"], s["w"], n, k), c.get("act", "none")
    if kind == "bwd":
        dz = s["dy"].float() * _plain_act(act, s["z"].float())[1]
        return {"dx": (dz @ w).to(dt), "dz": dz.to(dt), "dbias": dz.double().sum(0).float()}
    z = s["x"].float() @ w.t()
    if "bias" in s:
        z = z + s["bias"].float()
    y = _plain_act(act, z)[0]
    if "resid" in s:
        y = y + s["resid"].float()
    return {"y": y.to(dt), "z": z.to(dt)} if c.get("save") else y.to(dt)


# ---- what a pass cannot do without ----------------------------------------------
def work(case):
    kind, m, n, k = case["kind"], case["m"], case["n"], case["k"]
    b = SIZE[case["dt"]]
    w = n * (k // ELEMS[case["fmt"]]) * BYTES[case["fmt"]]
    if kind == "moe":
        e, top = case["e"], case["top"]
        # experts that m tokens take, each `top` of them at random
        taken = e * (1 - (1 - top / e) ** m)
        down = k * (n // ELEMS[case["down"]]) * BYTES[case["down"]]
        rows = m * k * (3 if case.get("resid") else 2) * b + m * top * 8
        return {"bytes": int(taken * (2 * w + down)) + e * k * SIZE[case["router"]] + rows,
                "flops": 2 * m * k * (3 * top * n + e)}
    if kind == "bwd":
        return {"bytes": w + b * m * (3 * n + k) + 4 * n, "flops": 2 * m * n * k}
    outs = n * (1 + bool(case.get("save")) + bool(case.get("resid")))
    return {"bytes": w + b * m * (k + outs) + (n * SIZE[case["bias"]] if "bias" in case else 0), "flops": 2 * m * n * k}


# ---- the same in 64 bits ---------------------------------------------------------
def _gather(b, byte, shift, mask):
    """Code e of every block: bits `mask` of byte[e] >> shift[e]."""
    return (b[:, byte.cuda()].long() >> shift.cuda()) & mask


def _exact_rows(fmt, b, k, r0, r1):
    """Rows r0 .. r1 of the weight matrix, from each element's place in its block."""
    per = k // ELEMS[fmt]
    b = b[r0 * per:r1 * per]
    e = torch.arange(ELEMS[fmt])

    def f16(col):
        return (b[:, col].int() | (b[:, col + 1].int() << 8)).to(torch.int16).view(torch.float16).double()[:, None]

    if fmt == "q4_0":
        w = f16(0) * (_gather(b, 2 + e % 16, 4 * (e // 16), 15) - 8)
    elif fmt == "q8_0":
        v = b[:, 2:].long()
        w = f16(0) * (v - 256 * (v >= 128))
    elif fmt == "q4_k":
        j = e // 32

        def six(base):
            low = _gather(b, base + j % 4, torch.where(j < 4, 0, 6), 255)
            high = _gather(b, base + 4 + (j % 4) // 2, 4 * (j % 2), 15)
            return torch.where((j < 4).cuda(), low & 63, (low & 3) | (high << 2))

        w = f16(0) * six(4) * _gather(b, 16 + e // 2, 4 * (e % 2), 15) - f16(2) * six(10)
    else:
        code = _gather(b, e // 2, 4 * (e % 2), 15) + 16 * _gather(b, 128 + e // 4, 2 * (e % 4), 3)
        sc = b[:, (192 + e // 16).cuda()].long()
        w = f16(208) * (sc - 256 * (sc >= 128)) * (code - 32)
    return w.reshape(r1 - r0, k)


def _exact_act(act, z):
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.clamp(z, min=0), torch.where(z > 0, 1.0, 0.0).double()
    if act == "silu":
        sg = torch.sigmoid(z)
        return z * sg, sg + z * sg * torch.sigmoid(-z)
    p = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    dp = math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z ** 2)
    return z * torch.sigmoid(2 * p), torch.sigmoid(2 * p) + z * 2 * dp * torch.sigmoid(2 * p) * torch.sigmoid(-2 * p)


STEP = 2048  # rows of weights taken at a time


def _exact_product(fmt, b, x, n, k, first=0):
    """x W^T over rows first .. first + n of the blocks."""
    return torch.cat([x @ _exact_rows(fmt, b, k, first + r, first + min(r + STEP, n)).t().contiguous()
                      for r in range(0, n, STEP)], 1)


def _exact_moe(s, c):
    n, k, top = c["n"], c["k"], c["top"]
    x = s["x"].double()
    logits = torch.stack([(x * r.double()).sum(1) for r in s["router"]], 1)
    sigmoid = c.get("score") == "sigmoid"
    left = torch.sigmoid(logits) + s["rbias"].double() if sigmoid else logits.clone()
    ids = []
    for _ in range(top):  # (the largest left, of equal ones the first)
        at = (left == left.amax(1, keepdim=True)).int().argmax(1)
        ids.append(at)
        left[torch.arange(c["m"], device=x.device), at] = -math.inf
    ids = torch.stack(ids, 1)
    chosen = logits.gather(1, ids)
    weights = torch.sigmoid(chosen) if sigmoid else torch.softmax(chosen, 1)
    weights = weights / weights.sum(1, keepdim=True)
    y = s["resid"].double() if c.get("resid") else torch.zeros_like(x)
    for i in range(c["e"]):
        share = (weights * (ids == i)).sum(1)
        rows = share.nonzero()[:, 0]
        if len(rows) == 0:
            continue
        g = _exact_product(c["fmt"], s["gate"], x[rows], n, k, i * n)
        h = _exact_act("silu", g)[0] * _exact_product(c["fmt"], s["up"], x[rows], n, k, i * n)
        y[rows] += share[rows, None] * _exact_product(c["down"], s["down"], h, k, n, i * k)
    return {"y": y, "ids": ids.int(), "weights": weights}


def exact(case, seed):
    s = _inputs(case, seed)
    kind, n, k, act = case["kind"], case["n"], case["k"], case.get("act", "none")
    if kind == "moe":
        return _exact_moe(s, case)
    if kind == "bwd":
        dz = s["dy"].double() * _exact_act(act, s["z"].double())[1]
        dx = torch.zeros(case["m"], k, dtype=torch.float64, device="cuda")
        for r in range(0, n, STEP):
            dx += dz[:, r:r + STEP].contiguous() @ _exact_rows(case["fmt"], s["w"], k, r, min(r + STEP, n))
        return {"dx": dx, "dz": dz, "dbias": dz.sum(0)}
    z = _exact_product(case["fmt"], s["w"], s["x"].double(), n, k)
    if "bias" in s:
        z = z + s["bias"].double()
    y = _exact_act(act, z)[0]
    if "resid" in s:
        y = y + s["resid"].double()
    return {"y": y, "z": z} if case.get("save") else y
