"""The operators for training in 8 bits and for a language model's last product, as one measures them.

Four operators: the quantisation of a tensor in blocks of 128 with a scale for each block, the contraction of two
such tensors, the softmax cross entropy of a linear head whose logits are not kept, and its gradient. `own = False`
computes them in elementary torch operations in 32 bits, `own = True` by the library's entry points.
"""
import math

import torch

own = False

BLOCK = 128
FLOOR = 2.0 ** -100  # the smallest block maximum that a scale is made from
FP8 = {"e4m3": (torch.float8_e4m3fn, 448.0, 3, -6), "e5m2": (torch.float8_e5m2, 57344.0, 2, -14)}  # type, largest, mantissa bits, least exponent
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
IGNORE = -100


def listed():
    return [
        # one token's activations on their way into a linear layer while answering: nothing but latency
        dict(name="quantize one token", op="quantize", rows=1, cols=4096, type="bf16", to="e4m3", block="row", transposed=False),
        # the activations of a training step, a scale for 128 values of each token
        dict(name="quantize activations", op="quantize", rows=16384, cols=8192, type="bf16", to="e4m3", block="row", transposed=False),
        # the gradient of an odd number of tokens for the weight gradient: blocks along the tokens, tokens fastest
        dict(name="quantize gradient by tokens", op="quantize", rows=5001, cols=4104, type="bf16", to="e5m2", block="col", transposed=True),
        # 32-bit master weights after an optimiser's step, blocks of 128 x 128
        dict(name="quantize weights", op="quantize", rows=8192, cols=4096, type="f32", to="e4m3", block="both", transposed=False),
        # one token through a linear layer: the weights' bytes
        dict(name="scaled one token", op="scaled", m=1, n=4096, k=4096, a="e4m3", b="e4m3", rowB=False, out="bf16", add=False),
        # a ragged batch through an odd layer
        dict(name="scaled ragged", op="scaled", m=777, n=2056, k=1000, a="e4m3", b="e4m3", rowB=False, out="bf16", add=False),
        # a training step's forward product
        dict(name="scaled forward", op="scaled", m=8192, n=8192, k=8192, a="e4m3", b="e4m3", rowB=False, out="bf16", add=False),
        # the weight gradient, added to a 32-bit accumulator: the contracted mode is the tokens, a scale per row on both sides
        dict(name="scaled weight gradient", op="scaled", m=4096, n=4096, k=8192, a="e5m2", b="e4m3", rowB=True, out="f32", add=True),
        # scoring a few tokens against a vocabulary: the head's bytes
        dict(name="loss few tokens", op="loss", tokens=17, vocab=32001, width=2048, type="bf16"),
        # a training step's loss
        dict(name="loss training", op="loss", tokens=8192, vocab=128000, width=4096, type="bf16"),
        # 32-bit fine-tuning of a small head
        dict(name="gradient small head f32", op="gradient", tokens=300, vocab=10007, width=512, type="f32"),
        # a training step's gradient of the head and of what it reads
        dict(name="gradient training", op="gradient", tokens=4096, vocab=128000, width=4096, type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "scaled", "loss", "gradient"])
    if op == "quantize":
        return dict(op=op, rows=_log(rng, 1, 16384), cols=_log(rng, 32, 8192), type=rng.choice(["bf16", "f16", "f32"]),
                    to=rng.choice(["e4m3", "e5m2"]), block=rng.choice(["row", "col", "both"]), transposed=rng.random() < 0.5)
    if op == "scaled":
        out = rng.choice(["bf16", "f16", "f32"])
        return dict(op=op, m=_log(rng, 1, 8192), n=_log(rng, 16, 8192), k=_log(rng, 32, 8192), a=rng.choice(["e4m3", "e5m2"]),
                    b=rng.choice(["e4m3", "e5m2"]), rowB=rng.random() < 0.5, out=out, add=out == "f32" and rng.random() < 0.5)
    tokens = _log(rng, 1, 4096 if op == "gradient" else 8192)
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    vocab, width = _log(rng, 1000, 128000), _log(rng, 64, 4096)
    if kind == "f32":  # a 32-bit head is a small one
        tokens, vocab, width = min(tokens, 1024), min(vocab, 32000), min(width, 1024)
    elif rng.random() < 0.75:
        width = max(64, width // 8 * 8)
    return dict(op=op, tokens=tokens, vocab=vocab, width=width, type=kind)


def _pad(n, to=16):
    return (n + to - 1) // to * to


def _inputs(case, seed):
    """The call's inputs alone, from the seed."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    if case["op"] == "quantize":
        # activations: channels of different size, and a few large values
        x = rnd(case["rows"], case["cols"])
        x *= torch.exp(rnd(1, case["cols"]))
        x[:, :: 97] *= 20
        return dict(x=x.to(TYPES[case["type"]]))
    if case["op"] == "scaled":
        m, n, k = case["m"], case["n"], case["k"]
        kb, nb = -(-k // BLOCK), n if case["rowB"] else -(-n // BLOCK)

        def operand(rows, kind):  # rows of whole 16-byte words, as a program lays 8-bit operands out
            t = torch.zeros(rows, _pad(k), device="cuda", dtype=torch.float8_e4m3fn if kind == "e4m3" else torch.float8_e5m2)
            v = rnd(rows, k) * (FP8[kind][1] / 4.5)
            t[:, :k] = v.clamp(-FP8[kind][1], FP8[kind][1]).to(t.dtype)
            return t[:, :k]

        s = dict(a=operand(m, case["a"]), b=operand(n, case["b"]), sa=torch.exp(0.5 * rnd(m, kb)) * 4.5 / FP8[case["a"]][1],
                 sb=torch.exp(0.5 * rnd(nb, kb)) * 0.2 / FP8[case["b"]][1])
        if case["add"]:
            s["c"] = rnd(m, n) * 0.01
        return s
    t, v, d = case["tokens"], case["vocab"], case["width"]
    kind = TYPES[case["type"]]
    s = dict(h=rnd(t, d).to(kind), w=(rnd(v, d) * (2.0 / math.sqrt(d))).to(kind))
    s["target"] = torch.randint(0, v, (t,), generator=g, device="cuda")
    s["target"][torch.rand(t, generator=g, device="cuda") < 0.1] = IGNORE  # prompts and padding count for nothing
    if case["op"] == "gradient":
        n = max(1, int((s["target"] >= 0).sum()))
        s["g"] = torch.full((t,), 1.0 / n, device="cuda") * (0.5 + torch.rand(t, generator=g, device="cuda"))
        if kind == torch.float16:
            s["g"] *= 1024  # the loss is scaled where gradients have so few exponents
        step = max(1, (1 << 28) // v)
        s["lse"] = torch.cat([torch.logsumexp(s["h"][i: i + step].float() @ s["w"].float().T, 1) for i in range(0, t, step)])
    return s


def prepare(case, seed):
    s = dict(case=case, **_inputs(case, seed))
    if not own:
        return s
    import hiptensor_b200 as ht

    s["handle"] = h = ht.Handle()
    kinds = {"bf16": ht.R_16BF, "f16": ht.R_16F, "f32": ht.R_32F, "e4m3": ht.R_8F_E4M3, "e5m2": ht.R_8F_E5M2}
    new = lambda *shape, dtype=torch.float32: torch.empty(shape, device="cuda", dtype=dtype)  # noqa: E731
    if case["op"] == "quantize":
        r, c = case["rows"], case["cols"]
        s["block"] = (1 if case["block"] == "row" else BLOCK, 1 if case["block"] == "col" else BLOCK)
        s["scale"] = new(-(-r // s["block"][0]), -(-c // s["block"][1]))
        if case["transposed"]:
            s["q"] = new(c, _pad(r), dtype=FP8[case["to"]][0])[:, :r]
        else:
            s["q"] = new(r, _pad(c), dtype=FP8[case["to"]][0])[:, :c]
        s["modes"] = (0, 1), ((1, 0) if case["transposed"] else (0, 1))
        s["descs"] = (h.tensor_descriptor((r, c), (c, 1), kinds[case["type"]]),
                      h.tensor_descriptor(s["q"].shape, s["q"].stride(), kinds[case["to"]]),
                      h.tensor_descriptor(s["scale"].shape, s["scale"].stride(), ht.R_32F))
    elif case["op"] == "scaled":
        desc = lambda x, kind: h.tensor_descriptor(x.shape, x.stride(), kinds[kind])  # noqa: E731
        s["d"] = new(case["m"], case["n"], dtype=TYPES[case["out"]])
        dD = desc(s["d"], case["out"])
        s["plan"] = h.scaled_contraction_plan(desc(s["a"], case["a"]), (0, 2), desc(s["sa"], "f32"), (1, BLOCK),
                                              desc(s["b"], case["b"]), (1, 2), desc(s["sb"], "f32"),
                                              (1 if case["rowB"] else BLOCK, BLOCK), dD if case["add"] else None, dD, (0, 1),
                                              ht.COMPUTE_32F)
    else:
        t, v, d = case["tokens"], case["vocab"], case["width"]
        kind = kinds[case["type"]]
        s["plan"] = h.cross_entropy_plan(h.tensor_descriptor((t, d), None, kind), (0, 2), h.tensor_descriptor((v, d), None, kind),
                                         (1, 2), IGNORE, ht.COMPUTE_32F)
        size = h.cross_entropy_workspace_size(s["plan"], case["op"] == "gradient", ht.WORKSPACE_RECOMMENDED)
        s["workspace"] = new(size, dtype=torch.uint8)
        if case["op"] == "gradient":
            s["dh"], s["dw"] = torch.empty_like(s["h"]), torch.empty_like(s["w"])
        else:
            s["loss"], s["lse"] = new(t), new(t)
    return s


def _over(scale, block, rows, cols):
    """A scale for each element from one for each block."""
    for i, n in enumerate((rows, cols)):
        if block[i] > 1:
            scale = scale.repeat_interleave(block[i], i).narrow(i, 0, n)
    return scale


def _quantize(s):
    case, x = s["case"], s["x"].float()
    kind, largest, bits, least = FP8[case["to"]]
    rows, cols = x.shape
    br, bc = (1 if case["block"] == "row" else BLOCK), (1 if case["block"] == "col" else BLOCK)
    p = torch.nn.functional.pad(x.abs(), (0, -cols % bc, 0, -rows % br))
    a = p.view(p.shape[0] // br, br, p.shape[1] // bc, bc).amax((1, 3)).clamp(min=FLOOR)
    top = torch.full_like(a, largest)  # a tensor: by a number torch multiplies with its reciprocal, and that rounds twice
    # next to a border between two 8-bit values 32 bits are too few: the product is exact in 64, and rounded once
    y = x.double() * _over(top / a, (br, bc), rows, cols).double()
    e = torch.frexp(y)[1].sub(1).clamp(min=least)
    step = torch.exp2((e - bits).double())
    q = (torch.round(y / step) * step).float().clamp(-largest, largest).to(kind)
    return (q.T.contiguous() if case["transposed"] else q), a / top


def _scaled(s):
    case = s["case"]
    m, n, k = case["m"], case["n"], case["k"]
    a = s["a"].float() * _over(s["sa"], (1, BLOCK), m, k)
    b = s["b"].float() * _over(s["sb"], (1 if case["rowB"] else BLOCK, BLOCK), n, k)
    d = a @ b.T
    if case["add"]:
        d = d + s["c"]
    return d.to(TYPES[case["out"]])


def _loss(s):
    z = s["h"].float() @ s["w"].float().T
    top = z.amax(1)
    lse = top + torch.log(torch.exp(z - top[:, None]).sum(1))
    counts = s["target"] >= 0
    at = z.gather(1, s["target"].clamp(min=0)[:, None])[:, 0]
    return torch.where(counts, lse - at, torch.zeros_like(lse)), lse


def _gradient(s):
    h, w = s["h"].float(), s["w"].float()
    p = torch.exp(h @ w.T - s["lse"][:, None])
    counts = s["target"] >= 0
    p.scatter_add_(1, s["target"].clamp(min=0)[:, None], -torch.ones_like(s["g"])[:, None])
    p *= torch.where(counts, s["g"], torch.zeros_like(s["g"]))[:, None]
    return (p @ w).to(s["h"].dtype), (p.T @ h).to(s["w"].dtype)


def run(s):
    case = s["case"]
    if not own:
        return {"quantize": _quantize, "scaled": _scaled, "loss": _loss, "gradient": _gradient}[case["op"]](s)
    h, stream = s["handle"], torch.cuda.current_stream()
    if case["op"] == "quantize":
        (modeA, modeQ), (dA, dQ, dS) = s["modes"], s["descs"]
        h.block_quantize(s["x"], dA, modeA, s["block"], s["q"], dQ, modeQ, s["scale"], dS, stream)
        return s["q"], s["scale"]
    if case["op"] == "scaled":
        h.scaled_contraction(s["plan"], 1.0, s["a"], s["sa"], s["b"], s["sb"], 1.0 if case["add"] else 0.0, s.get("c"), s["d"],
                             stream)
        return s["d"]
    if case["op"] == "loss":
        h.cross_entropy(s["plan"], 1.0, s["h"], s["w"], s["target"], s["loss"], s["lse"], s["workspace"], s["workspace"].numel(),
                        stream)
        return s["loss"], s["lse"]
    h.cross_entropy_gradient(s["plan"], 1.0, s["h"], s["w"], s["target"], s["lse"], s["g"], s["dh"], s["dw"], s["workspace"],
                             s["workspace"].numel(), stream)
    return s["dh"], s["dw"]


def work(case):
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        blocks = math.prod(-(-case[x] // (1 if case["block"] == b else BLOCK)) for x, b in (("rows", "row"), ("cols", "col")))
        return {"bytes": n * (5 if case["type"] == "f32" else 3) + 4 * blocks, "flops": 3 * n}
    if case["op"] == "scaled":
        m, n, k = case["m"], case["n"], case["k"]
        kb = -(-k // BLOCK)
        scales = 4 * kb * (m + (n if case["rowB"] else -(-n // BLOCK)))
        return {"bytes": (m + n) * k + scales + m * n * ((4 if case["out"] == "f32" else 2) + (4 if case["add"] else 0)),
                "flops": 2 * m * n * k}
    t, v, d = case["tokens"], case["vocab"], case["width"]
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "loss":  # the logits; targets in, losses and normalisers out
        return {"bytes": (t + v) * d * size + 16 * t, "flops": 2 * t * v * d}
    # the logits again, and two products with them; targets, normalisers and the losses' gradients in
    return {"bytes": 2 * (t + v) * d * size + 16 * t, "flops": 6 * t * v * d}


def exact(case, seed):
    """From the definitions, in 64 bits, block by block."""
    s = _inputs(case, seed)
    if case["op"] == "quantize":
        _, largest, bits, least = FP8[case["to"]]
        x = s["x"].double()
        rows, cols = x.shape
        br, bc = (1 if case["block"] == "row" else BLOCK), (1 if case["block"] == "col" else BLOCK)
        down, over = torch.arange(rows, device="cuda") // br, torch.arange(cols, device="cuda") // bc
        top = torch.zeros(int(down[-1]) + 1, cols, device="cuda", dtype=torch.float64)
        top.scatter_reduce_(0, down[:, None].expand(rows, cols), x.abs(), "amax")
        a = torch.zeros(top.shape[0], int(over[-1]) + 1, device="cuda", dtype=torch.float64)
        a.scatter_reduce_(1, over[None].expand(top.shape), top, "amax")
        a = torch.maximum(a, torch.full_like(a, FLOOR))
        # the factor is a 32-bit number by definition: the nearest to largest / a
        y = x * (largest / a).float().double()[down][:, over]
        # values of 2^e to 2^(e+1) lie 2^(e - bits) apart, those below 2^least as far apart as there
        size = y.abs()
        e = torch.floor(torch.log2(torch.where(size > 0, size, torch.ones_like(size))))
        e = e + (torch.exp2(e + 1) <= size).double() - (torch.exp2(e) > size).double()
        gap = torch.exp2(torch.maximum(e, torch.full_like(e, least)) - bits)
        low = torch.floor(size / gap)
        rest = size / gap - low
        low = low + ((rest > 0.5) | ((rest == 0.5) & (low % 2 == 1))).double()
        q = torch.sign(y) * torch.minimum(low * gap, torch.full_like(gap, largest))
        return (q.T.contiguous() if case["transposed"] else q), a / largest
    if case["op"] == "scaled":
        m, n, k = case["m"], case["n"], case["k"]
        d = torch.zeros(m, n, device="cuda", dtype=torch.float64)
        cols = torch.arange(n, device="cuda") // (1 if case["rowB"] else BLOCK)
        for j in range(-(-k // BLOCK)):
            part = s["a"][:, j * BLOCK: (j + 1) * BLOCK].double() @ s["b"][:, j * BLOCK: (j + 1) * BLOCK].double().T
            d += part * s["sa"][:, j].double()[:, None] * s["sb"][:, j].double()[cols][None]
        return d + s["c"].double() if case["add"] else d
    t, v = case["tokens"], case["vocab"]
    w = s["w"].double()
    step = max(1, (1 << 28) // v)
    if case["op"] == "loss":
        loss, lse = [], []
        for i in range(0, t, step):
            z = s["h"][i: i + step].double() @ w.T
            lse.append(torch.logsumexp(z, 1))
            target = s["target"][i: i + step]
            at = z[torch.arange(len(target), device="cuda"), target.clamp(min=0)]
            loss.append((lse[-1] - at) * (target >= 0))
        return torch.cat(loss), torch.cat(lse)
    dh, dw = [], torch.zeros_like(w)
    for i in range(0, t, step):
        h, target = s["h"][i: i + step].double(), s["target"][i: i + step]
        p = torch.exp(h @ w.T - s["lse"][i: i + step].double()[:, None])
        p[torch.arange(len(target), device="cuda"), target.clamp(min=0)] -= 1
        p *= (s["g"][i: i + step].double() * (target >= 0))[:, None]
        dh.append(p @ w)
        dw += p.T @ h
    return torch.cat(dh), dw
