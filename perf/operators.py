"""Timing cases of the operators over rows: layer norm, dropout and the two joined by a residual sum.

    norm      y = (x - mean) / sqrt(var + eps) * weight + bias over the last axis, each row by itself
    dropout   y = x / keep where the element is kept and 0 where not; which are kept follows from a
              state of two integers and the element's number, so no mask is stored
    addnorm   s = residual + dropout(x), rounded to the inputs' type, and y = norm(s): the join between
              two layers of a residual network; both are returned

The generator is Philox-4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, "Parallel random numbers:
as easy as 1, 2, 3", 2011).  ``state`` holds (seed, offset) as two int64.  Element i of the tensor in
row-major order belongs to counter (i // 8, offset), each 64 bits as two words, under key seed; its
16 bits are the (i % 8)-th halves of the four words that come out, low half first.  It is kept if they
are at least t = floor(65536 p + 1/2), and keep = 1 - t / 65536.

A case is a dict of plain values: ``op``, ``rows``, ``width``, ``dtype``, ``ld`` (elements between the
first elements of two rows of x, ``width`` for rows one after the other), ``train`` (forward and the
gradients under a given upstream gradient, or forward alone), ``p``, ``affine`` (whether there are a
weight and a bias), ``mean`` (of the values of x, which have a standard deviation of about one).
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
EPS = 1e-5
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _case(name, op, rows, width, dtype, **more):
    return dict({"name": name, "op": op, "rows": rows, "width": width, "dtype": dtype, "ld": width,
                 "train": True, "p": 0.0, "affine": True, "mean": 0.3}, **more)


def listed():
    return [
        # hidden radial features of the few edges of one atom: the call itself is what counts
        _case("norm_8x128_fp32", "norm", 8, 128, "fp32", train=False),
        # the l = 0 rows of the node embeddings [N, 25, 128] of a large structure, as they lie there
        _case("norm_scalars_48668x128_fp32", "norm", 48668, 128, "fp32", ld=3200, train=False),
        # hidden layer of the radial MLP over the edges of the benchmark graph, in training
        _case("norm_train_60000x128_fp32", "norm", 60000, 128, "fp32"),
        # a wide model in training: 16384 positions of 4096 channels
        _case("norm_train_16384x4096_bf16", "norm", 16384, 4096, "bf16"),
        # rows that start at any address: a width that nothing divides
        _case("norm_train_30011x1001_fp16", "norm", 30011, 1001, "fp16"),
        # hidden features of some edges
        _case("dropout_64x128_fp32", "dropout", 64, 128, "fp32", p=0.1, train=False),
        # the benchmark graph's hidden radial features
        _case("dropout_train_60000x128_fp32", "dropout", 60000, 128, "fp32", p=0.1),
        # activations of a wide hidden layer
        _case("dropout_train_16384x8192_bf16", "dropout", 16384, 8192, "bf16", p=0.1),
        # an odd number of columns of a wider array
        _case("dropout_train_20011x1023_fp16", "dropout", 20011, 1023, "fp16", p=0.25, ld=1030),
        # sixteen sequences, one position each, in evaluation: nothing is dropped
        _case("addnorm_16x4096_bf16", "addnorm", 16, 4096, "bf16", train=False),
        # residual layer over the benchmark graph's hidden radial features
        _case("addnorm_train_60000x128_fp32", "addnorm", 60000, 128, "fp32", p=0.1),
        # residual layer of a wide model
        _case("addnorm_train_16384x4096_bf16", "addnorm", 16384, 4096, "bf16", p=0.1),
    ]


def _most(op):
    return max(work(c)["bytes"] for c in listed() if c["op"] == op)


def draw(rng):
    op = rng.choice(["norm", "norm", "dropout", "addnorm"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    train = rng.random() < 0.7
    width = round(math.exp(rng.uniform(math.log(16), math.log(16384))))
    if rng.random() < 0.7:
        width = -(-width // 8) * 8
    ld = width + (rng.choice([1, 8, 24, 129]) if rng.random() < 0.25 else 0)
    affine = op != "dropout" and rng.random() < 0.85
    some = op == "dropout" or op == "addnorm" and train and rng.random() < 0.7
    p = rng.choice([0.05, 0.1, 0.2, 0.5]) if some else 0.0
    case = _case("", op, 1, width, dtype, ld=ld, train=train, p=p, affine=affine,
                 mean=rng.choice([0.0, 0.3, -2.0]))
    del case["name"]
    rows = math.exp(rng.uniform(0.0, math.log(400000)))
    most = _most(op) - work(case)["bytes"]
    per_row = work(dict(case, rows=2))["bytes"] - work(case)["bytes"]
    # (the strided array is made whole)
    case["rows"] = max(1, min(round(rows), int(most / per_row), 2 ** 28 // ld))
    return case


def work(case):
    """Bytes: every input and output once.  Operations: of the norm's two sums and its line per
    element, and of the VJP's; a choice and a product per dropped-out element."""
    n, w, train = case["rows"] * case["width"], case["width"], case["train"]
    size = 4 if case["dtype"] == "fp32" else 2
    arrays = {"norm": 2, "dropout": 2, "addnorm": 4}[case["op"]] * (2 if train else 1)
    params = (w * size * 2 * (2 if train else 1)) if case["affine"] and case["op"] != "dropout" else 0
    per = {"norm": 7, "dropout": 2, "addnorm": 8}[case["op"]]
    per += {"norm": 12, "dropout": 2, "addnorm": 14}[case["op"]] if train else 0
    return {"bytes": n * size * arrays + params, "flops": n * per}


def prepare(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    dt, (r, w) = TYPES[case["dtype"]], (case["rows"], case["width"])
    new = lambda *s: torch.randn(*s, generator=g, device=DEVICE, dtype=torch.float32)     # noqa: E731
    x = (new(r, case["ld"]) + case["mean"]).to(dt)[:, :w]
    s = {"op": case["op"], "train": case["train"], "p": case["p"], "x": x}
    s["state"] = torch.randint(0, 2 ** 62, (2,), generator=g, device=DEVICE)
    if case["op"] != "dropout":
        s["weight"] = (1 + 0.2 * new(w)).to(dt) if case["affine"] else None
        s["bias"] = (0.2 * new(w)).to(dt) if case["affine"] else None
    if case["op"] == "addnorm":
        s["residual"] = (new(r, w) - 0.5 * case["mean"]).to(dt)
    if case["train"]:
        s["grad_y"] = new(r, w).to(dt)
        if case["op"] == "addnorm":
            s["grad_s"] = new(r, w).to(dt)
        for k in ("x", "weight", "bias", "residual"):
            if s.get(k) is not None:
                s[k].requires_grad_(True)
    return s


# ---- the framework's calls ---------------------------------------------------------------------


def _own(s):
    from zippel_b200.blocks import rowwise
    x, train, p = s["x"], s["train"], s["p"]
    ins = [t for t in (x, s.get("residual"), s.get("weight"), s.get("bias")) if t is not None]
    if s["op"] == "norm":
        out, up = (rowwise.layer_norm(x, s["weight"], s["bias"], EPS),), ("grad_y",)
    elif s["op"] == "dropout":
        out, up = (rowwise.dropout(x, p, s["state"]),), ("grad_y",)
    else:
        out = rowwise.dropout_add_layer_norm(x, s["residual"], s["weight"], s["bias"], p, s["state"], EPS)
        up = ("grad_y", "grad_s")
    if train:
        out = [t.detach() for t in out] + list(torch.autograd.grad(out, ins, [s[k] for k in up]))
    return list(out)


# ---- the plain form ----------------------------------------------------------------------------


def _low(v):
    return v & 0xFFFFFFFF


def _kept(shape, p, state):
    """Which elements are kept, and one over the share that is."""
    t = math.floor(65536 * p + 0.5)
    n = math.prod(shape)
    group = torch.arange((n + 7) // 8, device=state.device)
    c0, c1 = _low(group), group >> 32
    c2, c3 = (_low(state[1]).expand_as(c0), _low(state[1] >> 32).expand_as(c0))
    k0, k1 = _low(state[0]), _low(state[0] >> 32)
    for _ in range(10):                        # each round works on what the last one left
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57                 # (64 bits; the sign bit is one of them)
        c0, c1, c2, c3 = _low(b >> 32) ^ c1 ^ k0, _low(b), _low(a >> 32) ^ c3 ^ k1, _low(a)
        k0, k1 = _low(k0 + 0x9E3779B9), _low(k1 + 0xBB67AE85)
    words = torch.stack([c0, c1, c2, c3], -1)
    halves = torch.stack([words & 0xFFFF, words >> 16], -1).view(-1)[:n]
    return (halves >= t).view(shape), 65536 / (65536 - t) if t < 65536 else 0.0


def _drop(v, mask, scale):
    return torch.where(mask, v * scale, 0.0)


def _norm_vjp(xc, rstd, w, gy):
    """Gradients of the normalised input (xc: centred), the weight and the bias."""
    z = xc * rstd
    gz = gy if w is None else gy * w
    gx = (gz - gz.mean(1, keepdim=True) - z * (gz * z).mean(1, keepdim=True)) * rstd
    return gx, None if w is None else (gy * z).sum(0), None if w is None else gy.sum(0)


def _plain(s):
    up = lambda k: None if s.get(k) is None else s[k].float()                              # noqa: E731
    dt, x = s["x"].dtype, up("x")
    mask, scale = (_kept(x.shape, s["p"], s["state"]) if s["p"] > 0 else
                   (torch.ones((), dtype=torch.bool, device=x.device), 1.0))
    if s["op"] == "dropout":
        out = [_drop(x, mask, scale)]
        return [t.to(dt) for t in (out + [_drop(up("grad_y"), mask, scale)] if s["train"] else out)]
    w, b = up("weight"), up("bias")
    total = x
    if s["op"] == "addnorm":
        total = (up("residual") + _drop(x, mask, scale)).to(dt).float()      # an output: as it is returned
    xc = total - total.mean(1, keepdim=True)
    rstd = torch.rsqrt((xc * xc).mean(1, keepdim=True) + EPS)
    y = xc * rstd if w is None else xc * rstd * w + b
    out = [y] + ([total] if s["op"] == "addnorm" else [])
    if s["train"]:
        gx, gw, gb = _norm_vjp(xc, rstd, w, up("grad_y"))
        if s["op"] == "addnorm":
            gx = gx + up("grad_s")
            out += [_drop(gx, mask, scale), gx]
        else:
            out += [gx]
        out += [] if w is None else [gw, gb]
    return [t.to(dt) for t in out]


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


# ---- in 64 bits --------------------------------------------------------------------------------


def _factors(shape, p, state):
    """Factor of each element, 0 or 1 / keep, with the generator in numpy's unsigned integers."""
    t, n = int(p * 65536 + 0.5), math.prod(shape)
    seed, offset = (int(v) % 2 ** 64 for v in state.tolist())
    u, mask = np.uint64, np.uint64(0xFFFFFFFF)
    out, step = np.empty((n + 7) // 8 * 8, np.bool_), 1 << 16
    for first in range(0, (n + 7) // 8, step):
        g = np.arange(first, min(first + step, (n + 7) // 8), dtype=np.uint64)
        c = [g & mask, g >> u(32), np.full_like(g, offset & 0xFFFFFFFF), np.full_like(g, offset >> 32)]
        for i in range(10):
            k = [(seed + i * 0x9E3779B9) & 0xFFFFFFFF, ((seed >> 32) + i * 0xBB67AE85) & 0xFFFFFFFF]
            lo, hi = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
            c = [(hi >> u(32)) ^ c[1] ^ u(k[0]), hi & mask, (lo >> u(32)) ^ c[3] ^ u(k[1]), lo & mask]
        bits = np.stack(c, 1).astype(np.uint32).view(np.uint16)          # (little-endian: low half first)
        out[8 * first:8 * (first + len(g))] = (bits >= t).reshape(-1) if t < 65536 else False
    keep = torch.from_numpy(out[:n]).to(DEVICE).view(shape)
    return keep.double() * (65536 / (65536 - t) if t < 65536 else 0.0)


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    x, w, b = d["x"], d.get("weight"), d.get("bias")
    factor = _factors(x.shape, s["p"], s["state"]) if s["p"] > 0 else None
    if s["op"] == "dropout":
        return [x * factor, d["grad_y"] * factor] if s["train"] else [x * factor]
    out, total = [], x
    if s["op"] == "addnorm":
        total = d["residual"] + (x if factor is None else x * factor)
        total = total.to(s["x"].dtype).double()
        out = [total]
    leaves = [t.requires_grad_(True) for t in (total, w, b) if t is not None]
    y = torch.nn.functional.layer_norm(total, x.shape[1:], w, b, EPS)
    out = [y.detach(), *(t.detach() for t in out)]
    if s["train"]:
        gx, *params = torch.autograd.grad(y, leaves, d["grad_y"])
        if s["op"] == "addnorm":
            gx = gx + d["grad_s"]
            out += [gx if factor is None else gx * factor, gx, *params]
        else:
            out += [gx, *params]
    return out
