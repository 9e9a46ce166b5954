"""What is measured of the operators for classifiers with many classes and little
memory: softmax cross-entropy straight from the last layer's inputs, group norm
with an activation, and activations kept in 8 bits for the backward pass.

``listed()`` gives the measured cases and ``draw()`` further ones of the same
ranges; ``prepare()`` makes a case's inputs on the GPU from a seed, ``run()`` takes
them through one pass, ``exact()`` says what the pass computes and ``work()`` what
it has to read, write and calculate.  With ``own`` false, ``run()`` computes in
elementary torch operations, with ``own`` true it calls the library.

Everything is fp64, as in the whole library, so the plain form computes in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 64          # columns that share a scale in the 8-bit form
EPS = 1e-5          # group norm
NONE, RELU, SILU = 0, 1, 2
# flags of the C ABI: the gradient destinations hold nothing yet
STORE_A, STORE_B, STORE_C = 1, 2, 4


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # Linear layer + softmax cross-entropy over many classes.
        # The per-sample trainer's step, where launches and the weights' bytes count.
        dict(name="xent one row", op="xent", rows=1, width=128, classes=8192, grad=True),
        # Evaluation: the loss alone, on a class count that no tile divides.
        dict(name="xent loss odd", op="xent", rows=1000, width=784, classes=10007, grad=False),
        # A training batch on a medium layer and a class count that is odd: rows of the weight
        # matrix start on 8-byte boundaries only.
        dict(name="xent train odd", op="xent", rows=777, width=300, classes=50257, grad=True),
        # A training batch behind a 1024-wide hidden layer.
        dict(name="xent train", op="xent", rows=4096, width=1024, classes=32768, grad=True),
        # Group norm with an activation, channels last.
        # One image's feature map at inference: latency.
        dict(name="norm one image", op="norm", batch=1, positions=196, groups=8, per_group=8, act=SILU, backward=False),
        # A hidden layer's output rows: a full training batch of vectors.
        dict(name="norm rows", op="norm", batch=65536, positions=1, groups=16, per_group=64, act=RELU, backward=False),
        # Gradients of a batch of feature maps.
        dict(name="norm images back", op="norm", batch=128, positions=784, groups=32, per_group=8, act=SILU, backward=True),
        # The same with odd counts, five channels a group, no activation.
        dict(name="norm odd back", op="norm", batch=33, positions=197, groups=30, per_group=5, act=NONE, backward=True),
        # Activations in 8 bits.
        # A small odd activation, stored and read back: latency and ragged blocks.
        dict(name="q8 store odd", op="q8 store", rows=33, width=785),
        # The hidden activation of the large training step, stored and read back.
        dict(name="q8 store", op="q8 store", rows=65536, width=1024),
        # Backward of the ten-class layer on that activation: bound by memory.
        dict(name="q8 back ten", op="q8 back", rows=65536, width=1024, features=10),
        # Backward of a hidden layer on it: bound by arithmetic.
        dict(name="q8 back", op="q8 back", rows=65536, width=1024, features=1024),
    ]


def _between(rng, lo, hi):
    """A whole number from lo to hi, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["xent", "xent", "norm", "norm", "q8 store", "q8 back"])
    if op == "xent":
        while True:
            c = dict(op=op, rows=_between(rng, 1, 4096), width=_between(rng, 16, 1024),
                     classes=_between(rng, 500, 100000), grad=rng.random() < 0.7)
            if c["rows"] * c["width"] * c["classes"] <= 4096 * 1024 * 32768:
                return c
    if op == "norm":
        while True:
            c = dict(op=op, batch=_between(rng, 1, 4096), positions=_between(rng, 1, 1024), groups=_between(rng, 1, 64),
                     per_group=_between(rng, 1, 128), act=rng.choice([NONE, RELU, SILU]), backward=rng.random() < 0.6)
            # (a group of one or two values is normalised to signs: its gradient is rounding alone)
            if c["positions"] * c["per_group"] >= 4 and c["batch"] * c["positions"] * c["groups"] * c["per_group"] <= 128 * 784 * 256:
                return c
    if op == "q8 store":
        while True:
            c = dict(op=op, rows=_between(rng, 1, 65536), width=_between(rng, 1, 4096))
            if c["rows"] * c["width"] <= 65536 * 1024:
                return c
    while True:
        c = dict(op=op, rows=_between(rng, 16, 65536), width=_between(rng, 10, 1024), features=_between(rng, 1, 1024))
        if c["rows"] * c["width"] * c["features"] <= 65536 * 1024 * 1024:
            return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _blocks(width):
    return -(-width // BLOCK)


def _spread(values, width):
    """[rows, width] as [rows, blocks, BLOCK], the last block filled up with zeros."""
    rows, full = values.shape[0], _blocks(width) * BLOCK
    padded = torch.zeros(rows, full, dtype=values.dtype, device=values.device)
    padded[:, :width] = values
    return padded.view(rows, -1, BLOCK)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, dtype=torch.float64, device="cuda")

    def room(*shape, dtype=torch.float64):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    s = dict(case)
    if case["op"] == "xent":
        rows, width, classes = case["rows"], case["width"], case["classes"]
        s["x"] = normal(rows, width).clamp_(min=0.0)  # what a ReLU layer hands on
        s["w"] = normal(width, classes) / math.sqrt(width)
        s["b"] = 0.1 * normal(classes)
        labels = torch.randint(0, classes, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        if rows > 1:  # a few rows are padding of the batch
            pad = torch.rand(rows, generator=gen, device="cuda") < 0.04
            labels = torch.where(pad, torch.full_like(labels, -1), labels)
        s["labels"] = labels
        s["gloss"] = 1.0 + 0.25 * torch.rand(1, generator=gen, dtype=torch.float64, device="cuda")
        s["out"] = dict(loss=room(1))
        if case["grad"]:
            s["out"].update(gx=room(rows, width), gw=room(width, classes), gb=room(classes))
    elif case["op"] == "norm":
        n, p, g, d = case["batch"], case["positions"], case["groups"], case["per_group"]
        c = g * d
        s["x"] = (normal(n, p, c) * (0.5 + torch.rand(c, generator=gen, dtype=torch.float64, device="cuda")) + normal(c)).contiguous()
        s["gamma"] = 1.0 + 0.1 * normal(c)
        s["beta"] = 0.1 * normal(c)
        if case["backward"]:
            mean, rstd = _group_stats(s)
            s.update(mean=mean, rstd=rstd, gy=normal(n, p, c))
            s["out"] = dict(gx=room(n, p, c), ggamma=room(c), gbeta=room(c))
        else:
            s["out"] = dict(y=room(n, p, c), mean=room(n, g), rstd=room(n, g))
    else:
        rows, width = case["rows"], case["width"]
        h = (normal(rows, width) * torch.exp(normal(rows, 1))).clamp_(min=0.0)
        if case["op"] == "q8 store":
            s["x"] = h
            s["codes"], s["scales"] = room(rows, width, dtype=torch.int8), room(rows, _blocks(width))
            s["out"] = dict(values=room(rows, width))
        else:
            s["codes"], s["scales"] = _encode(h)
            s["g"] = normal(rows, case["features"]) / rows
            s["w"] = normal(width, case["features"]) / math.sqrt(width)
            s["out"] = dict(dw=room(width, case["features"]), dx=room(rows, width))
    torch.cuda.synchronize()  # the library works on a stream of its own
    return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _plain_xent(s):
    rows = s["rows"]
    z = s["x"] @ s["w"] + s["b"]
    top = z.amax(dim=1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(dim=1, keepdim=True)
    keep = (s["labels"] >= 0).to(z.dtype)
    at = s["labels"].clamp(min=0).long()[:, None]
    logp = (z.gather(1, at) - top - torch.log(total))[:, 0]
    loss = -(logp * keep).sum().view(1) / rows
    if not s["grad"]:
        return dict(loss=loss)
    g = e / total
    g.scatter_add_(1, at, torch.full_like(logp, -1.0)[:, None])
    g *= (keep * (s["gloss"] / rows))[:, None]
    return dict(loss=loss, gx=g @ s["w"].t(), gw=s["x"].t() @ g, gb=g.sum(dim=0))


def _group_stats(s):
    n, p, g, d = s["batch"], s["positions"], s["groups"], s["per_group"]
    x = s["x"].view(n, p, g, d)
    mean = x.sum(dim=(1, 3)) / (p * d)
    var = (x - mean[:, None, :, None]).square().sum(dim=(1, 3)) / (p * d)
    return mean, 1.0 / torch.sqrt(var + EPS)


def _plain_norm(s):
    n, p, g, d = s["batch"], s["positions"], s["groups"], s["per_group"]
    mean, rstd = (s["mean"], s["rstd"]) if s["backward"] else _group_stats(s)
    unit = (s["x"].view(n, p, g, d) - mean[:, None, :, None]) * rstd[:, None, :, None]
    z = unit.view(n, p, g * d) * s["gamma"] + s["beta"]
    if not s["backward"]:
        y = z.clamp(min=0.0) if s["act"] == RELU else z / (1.0 + torch.exp(-z)) if s["act"] == SILU else z
        return dict(y=y, mean=mean, rstd=rstd)
    if s["act"] == RELU:
        gz = s["gy"] * (z > 0)
    elif s["act"] == SILU:
        sig = 1.0 / (1.0 + torch.exp(-z))
        gz = s["gy"] * (sig * (1.0 + z * (1.0 - sig)))
    else:
        gz = s["gy"]
    ggamma, gbeta = (gz * unit.view(n, p, g * d)).sum(dim=(0, 1)), gz.sum(dim=(0, 1))
    gu = (gz * s["gamma"]).view(n, p, g, d)
    m1 = gu.sum(dim=(1, 3), keepdim=True) / (p * d)
    m2 = (gu * unit).sum(dim=(1, 3), keepdim=True) / (p * d)
    gx = rstd[:, None, :, None] * (gu - m1 - unit * m2)
    return dict(gx=gx.reshape(n, p, g * d), ggamma=ggamma, gbeta=gbeta)


def _encode(x):
    """Codes and scales of the 8-bit form: the nearest of 127 steps of a block's largest
    magnitude, except that what is not zero keeps its sign in the code."""
    rows, width = x.shape
    blocks = _spread(x, width)
    top = blocks.abs().amax(dim=2)
    inverse = torch.where(top > 0, 127.0 / top, torch.zeros_like(top))
    code = torch.round(blocks * inverse[:, :, None])
    code = torch.where((code == 0) & (blocks != 0), torch.sign(blocks), code)
    return code.to(torch.int8).view(rows, -1)[:, :width].contiguous(), top / 127.0


def _decode(codes, scales):
    width = codes.shape[1]
    return codes.to(torch.float64) * scales.repeat_interleave(BLOCK, dim=1)[:, :width]


def _plain_q8(s):
    if s["op"] == "q8 store":
        return dict(values=_decode(*_encode(s["x"])))
    dw = _decode(s["codes"], s["scales"]).t() @ s["g"]
    dx = (s["g"] @ s["w"].t()) * (s["codes"] > 0)
    return dict(dw=dw, dx=dx)


# ---------------------------------------------------------------------------
# The library's calls
# ---------------------------------------------------------------------------
def _library():
    import micrograd_b200
    return micrograd_b200.load_abi()


def _own_xent(s):
    abi, out = _library(), s["out"]
    x, w, b, labels = (s[k].data_ptr() for k in ("x", "w", "b", "labels"))
    sizes = (s["rows"], s["width"], s["classes"], float(s["rows"]))
    if not s["grad"]:
        abi.mg_linear_xent_fwd(x, w, b, labels, out["loss"].data_ptr(), *sizes)
    else:
        abi.mg_linear_xent_fwd_bwd(x, w, b, labels, s["gloss"].data_ptr(), out["loss"].data_ptr(),
                                   out["gx"].data_ptr(), out["gw"].data_ptr(), out["gb"].data_ptr(),
                                   *sizes, STORE_A | STORE_B | STORE_C)
    return out


def _own_norm(s):
    abi, out = _library(), s["out"]
    x, gamma, beta = (s[k].data_ptr() for k in ("x", "gamma", "beta"))
    sizes = (s["batch"], s["positions"], s["groups"] * s["per_group"], s["groups"])
    if not s["backward"]:
        abi.mg_group_norm_fwd(x, gamma, beta, out["y"].data_ptr(), out["mean"].data_ptr(), out["rstd"].data_ptr(),
                              *sizes, EPS, s["act"])
    else:
        abi.mg_group_norm_bwd(x, gamma, beta, s["mean"].data_ptr(), s["rstd"].data_ptr(), s["gy"].data_ptr(),
                              out["gx"].data_ptr(), out["ggamma"].data_ptr(), out["gbeta"].data_ptr(),
                              *sizes, s["act"], STORE_A | STORE_B | STORE_C)
    return out


def _own_q8(s):
    abi = _library()
    codes, scales = s["codes"].data_ptr(), s["scales"].data_ptr()
    rows, width = s["rows"], s["width"]
    if s["op"] == "q8 store":
        abi.mg_q8_pack(s["x"].data_ptr(), codes, scales, rows, width)
        abi.mg_q8_unpack(codes, scales, s["out"]["values"].data_ptr(), rows, width)
        return s["out"]
    g, w, dw, dx = (t.data_ptr() for t in (s["g"], s["w"], s["out"]["dw"], s["out"]["dx"]))
    abi.mg_gemm_tn_q8(codes, scales, g, dw, rows, s["features"], width, 0)
    abi.mg_gemm_nt_q8(g, w, dx, rows, s["features"], width, 0, codes)
    return s["out"]


def run(state):
    if state["op"] == "xent":
        return _own_xent(state) if own else _plain_xent(state)
    if state["op"] == "norm":
        return _own_norm(state) if own else _plain_norm(state)
    return _own_q8(state) if own else _plain_q8(state)


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_xent(s):
    leaves = [s[k].clone().requires_grad_(s["grad"]) for k in ("x", "w", "b")]
    logits = torch.addmm(leaves[2], leaves[0], leaves[1])
    loss = torch.nn.functional.cross_entropy(logits, s["labels"].long(), ignore_index=-1, reduction="sum") / s["rows"]
    if not s["grad"]:
        return dict(loss=loss.view(1))
    gx, gw, gb = torch.autograd.grad(loss, leaves, s["gloss"].view(()))
    return dict(loss=loss.detach().view(1), gx=gx, gw=gw, gb=gb)


def _exact_norm(s):
    n, p, g, d = s["batch"], s["positions"], s["groups"], s["per_group"]
    leaves = [s[k].clone().requires_grad_(s["backward"]) for k in ("x", "gamma", "beta")]
    x, gamma, beta = leaves
    rows = x.view(n, p, g, d).permute(0, 2, 1, 3).reshape(n, g, p * d)
    var, mean = torch.var_mean(rows, dim=2, correction=0)
    rstd = torch.rsqrt(var + EPS)
    unit = ((rows - mean[..., None]) * rstd[..., None]).view(n, g, p, d).permute(0, 2, 1, 3).reshape(n, p, g * d)
    z = torch.addcmul(beta, unit, gamma)
    y = torch.relu(z) if s["act"] == RELU else z * torch.sigmoid(z) if s["act"] == SILU else z
    if not s["backward"]:
        return dict(y=y, mean=mean, rstd=rstd)
    gx, ggamma, gbeta = torch.autograd.grad(y, leaves, s["gy"])
    return dict(gx=gx, ggamma=ggamma, gbeta=gbeta)


def _exact_q8(s):
    width, fill = s["width"], (0, -s["width"] % BLOCK)
    pad = torch.nn.functional.pad
    if s["op"] == "q8 store":
        x = pad(s["x"], fill).unflatten(1, (-1, BLOCK))
        top = torch.linalg.vector_norm(x, ord=math.inf, dim=2, keepdim=True)
        steps = (x * (127.0 / top)).nan_to_num(nan=0.0).round()
        steps = torch.where((steps == 0) & (x != 0), x.sign(), steps)
        return dict(values=(steps * (top / 127.0)).flatten(1)[:, :width])
    x = (pad(s["codes"].double(), fill).unflatten(1, (-1, BLOCK)) * s["scales"][:, :, None]).flatten(1)[:, :width]
    dx = torch.einsum("ro,wo->rw", s["g"], s["w"])
    return dict(dw=torch.einsum("rw,ro->wo", x, s["g"]), dx=torch.where(s["codes"] > 0, dx, torch.zeros_like(dx)))


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_xent(s) if case["op"] == "xent" else _exact_norm(s) if case["op"] == "norm" else _exact_q8(s)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "xent":
        rows, width, classes = case["rows"], case["width"], case["classes"]
        once = rows * width + width * classes + classes
        return dict(bytes=8 * once * (2 if case["grad"] else 1) + 4 * rows + 8,
                    flops=(6 if case["grad"] else 2) * rows * width * classes)
    if case["op"] == "norm":
        c, stats = case["groups"] * case["per_group"], case["batch"] * case["groups"]
        n = case["batch"] * case["positions"] * c
        if case["backward"]:
            return dict(bytes=8 * (3 * n + 4 * c + 2 * stats), flops=16 * n)
        return dict(bytes=8 * (2 * n + 2 * c + 2 * stats), flops=8 * n)
    rows, width = case["rows"], case["width"]
    kept = rows * width + 8 * rows * _blocks(width)  # bytes of the 8-bit form
    if case["op"] == "q8 store":
        return dict(bytes=16 * rows * width + 2 * kept, flops=6 * rows * width)
    out = case["features"]
    return dict(bytes=kept + 8 * (rows * out + 2 * width * out + rows * width), flops=4 * rows * width * out)
