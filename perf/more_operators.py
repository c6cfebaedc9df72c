"""Performance cases of what a deep stack of attention layers over a large scene takes: attention in which each Gaussian sees its
neighbours along the scene's order, the norms between the layers, and the clipping of a training step's gradients.

A case is a dict of plain values: the operator ("op"), "dtype" and

    window  gaussian_attention with a window: scenes "b", queries "nq" and keys "nk" of each scene (the queries are the last of the
            keys' places), heads "hq" and "hkv" (each key head serves hq / hkv query heads), head width "d"; a query at place p sees
            the places up to p + "right" that are not before p - "left" or are among the first "sinks"; each scene keeps the fraction
            "keep" of its keys (1: no mask); "empty": its first scene none
    norm    layer_norm: scenes "b" of "n" rows of "c" channels; "residual": the sum with a second tensor before it
    clip    clip_grad_norm_: the gradients of "gaussians" Gaussians (means, opacity, scales, rotations, features of "c"
            channels; none if 0) and of "layers" attention layers of "c" channels, clipped to "max_norm" into the float32 gradients
            that the optimizer takes

window and norm forward alone, or with "train" forward and backward with the gradients of all inputs.
"""
import math
import os
import sys

import torch

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for _p in (_ROOT, os.path.join(_ROOT, "shelfgaussian-cudagaussianvoxelizer_amd")):
    if _p not in sys.path:
        sys.path.insert(0, _p)

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5
CLIP_EPS = 1e-6


def _window(name, train, b, nq, nk, hq, hkv, d, dtype, left, right, sinks, keep=1.0, empty=False):
    c = {"op": "window", "train": train, "b": b, "nq": nq, "nk": nk, "hq": hq, "hkv": hkv, "d": d, "dtype": dtype, "left": left,
         "right": right, "sinks": sinks, "keep": keep, "empty": empty}
    return dict(c, name=name) if name else c


def _norm(name, train, b, n, c, dtype, residual):
    c = {"op": "norm", "train": train, "b": b, "n": n, "c": c, "dtype": dtype, "residual": residual}
    return dict(c, name=name) if name else c


def _clip(name, gaussians, layers, c, dtype, max_norm=1.0):
    c = {"op": "clip", "gaussians": gaussians, "layers": layers, "c": c, "dtype": dtype, "max_norm": max_norm}
    return dict(c, name=name) if name else c


def listed():
    return [
        # a token that arrives at the end of a streamed scene: latency
        _window("window_step_1x18000_h16d64_bf16", False, 1, 1, 18000, 16, 16, 64, "bf16", 4096, 0, 4),
        # a batch of sparse scenes padded to 300 Gaussians, one of them empty
        _window("window_infer_6x300_h8d32", False, 6, 300, 300, 8, 8, 32, "f32", 32, 32, 1, 0.7, True),
        # new Gaussians of streamed scenes that look back, shared key heads, a width between two tiles', pruned keys
        _window("window_train_ragged_d72_bf16", True, 2, 2999, 7001, 12, 4, 72, "bf16", 1000, 0, 8, 0.8),
        # float32 inference over a large scene
        _window("window_infer_n60000_h8d64", False, 1, 60000, 60000, 8, 8, 64, "f32", 128, 128, 4),
        # the headline scene's 1024 channels as 16 heads, one training step
        _window("window_train_n18000_h16d64_bf16", True, 1, 18000, 18000, 16, 16, 64, "bf16", 512, 512, 16),
        # the largest scene of the published configurations
        _window("window_train_n200000_h8d64_bf16", True, 1, 200000, 200000, 8, 8, 64, "bf16", 256, 256, 16),
        # a few hundred Gaussians, no gradients: one launch
        _norm("norm_n300_c256", False, 1, 300, 256, "f32", False),
        # rows that no vector divides, float32 training
        _norm("norm_train_ragged_c771", True, 2, 2999, 771, "f32", True),
        # the headline scene, one training step with the residual sum
        _norm("norm_train_n18000_c1024_bf16", True, 1, 18000, 1024, "bf16", True),
        # a small model: latency
        _clip("clip_n2000_c64_2layers", 2000, 2, 64, "f32"),
        # the headline scene's Gaussians: few tensors, one of them large
        _clip("clip_n18000_c1024", 18000, 0, 1024, "f32"),
        # a deep stack's weights, bfloat16 gradients into float32 ones
        _clip("clip_12layers_c1024_bf16", 0, 12, 1024, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges, none of more work than the largest listed one of its operator."""
    dtype = rng.choice(["bf16", "bf16", "f32"])
    kind = rng.random()
    if kind < 0.2:
        while True:
            case = _norm(None, rng.random() < 0.7, rng.choice([1, 1, 2, 6]), _log_int(rng, 1, 100000), _log_int(rng, 16, 4096), dtype,
                         rng.random() < 0.6)
            if case["b"] * case["n"] * case["c"] <= 18000 * 1024:
                return case
    if kind < 0.35:
        while True:
            case = _clip(None, rng.choice([0, _log_int(rng, 100, 50000)]), rng.choice([0, 1, rng.randint(1, 24)]),
                         _log_int(rng, 16, 1024), dtype, rng.choice([0.1, 1.0, 35.0, 1e6]))
            if case["gaussians"] + case["layers"] > 0 and sum(_clip_numels(case)) <= 12 * 12 * 1024 * 1024:
                return case
    train = rng.random() < 0.6
    b = rng.choice([1, 1, 1, 2, 3, 6])
    d = rng.choice([32, 64, 64, 96, 128, rng.randint(16, 128), rng.randint(16, 128)])
    hkv, group = rng.randint(1, 8), rng.choice([1, 1, 2, 3, 4])
    hkv = max(1, min(hkv, 1024 // (group * d)))
    nk = _log_int(rng, 64, 200000)
    nq = nk if rng.random() < 0.6 else min(nk, rng.choice([1, _log_int(rng, 1, nk)]))
    left = _log_int(rng, 8, 4096)
    right = rng.choice([0, left, left, _log_int(rng, 8, 4096)])
    sinks = rng.choice([0, 1, 4, rng.randint(1, 64)])
    keep = rng.choice([1.0, 1.0, round(rng.uniform(0.1, 0.95), 3)])
    empty = b > 1 and keep < 1.0 and rng.random() < 0.5
    most = 7.5e11 if dtype == "bf16" else 6.0e10   # float32 products run at a sixteenth of the bfloat16 ones' rate
    while True:
        case = _window(None, train, b, nq, nk, hkv * group, hkv, d, dtype, left, right, sinks, keep, empty)
        w = work(dict(case, keep=1.0, empty=False))
        if w["flops"] <= most and w["bytes"] <= 2.3e9 and b * hkv * group * nk * d <= 200000 * 512:
            return case
        nq, nk = max(1, int(nq * 0.8)), max(64, int(nk * 0.8))


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _clip_shapes(case):
    """Shapes of the gradients: those of the Gaussians, those of each layer."""
    n, c = case["gaussians"], case["c"]
    each = [[(n, 3), (n,), (n, 3), (n, 4), (n, c)]] if n else []
    layer = [(c,), (c,), (c, c), (2 * c, c), (64,), (64,), (c, c), (c,), (c,), (4 * c, c), (4 * c,), (c, 4 * c), (c,)]
    return each + [layer] * case["layers"]


def _clip_numels(case):
    return [math.prod(s) for bucket in _clip_shapes(case) for s in bucket]


def _kept(case):
    """Valid keys of each scene."""
    n = [case["nk"]] * case["b"]
    if case["keep"] < 1.0:
        n = [int(case["nk"] * case["keep"])] * case["b"]
    if case["empty"]:
        n[0] = 0
    return n


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def leaf(t):
        return t.detach().requires_grad_(case["train"])

    s = {"case": dict(case)}
    if case["op"] == "clip":
        # each bucket's gradients are views of one allocation, as all-reduced gradients are
        s["flat"], s["grads"], s["out_flat"], s["out"] = [], [], [], []
        for bucket in _clip_shapes(case):
            sizes = [math.prod(shape) for shape in bucket]
            at = [0]
            for n in sizes:
                at.append(at[-1] + -(-n // 8) * 8)
            flat, out = torch.zeros(at[-1], dtype=dt, device=dev), torch.zeros(at[-1], device=dev)
            for shape, n, a in zip(bucket, sizes, at):
                scale = 10.0 ** (-3.0 + 2.0 * float(torch.rand((), generator=torch.Generator().manual_seed(seed + a))))
                flat[a:a + n] = (scale * rand(n)).to(dt)
                s["grads"].append(flat[a:a + n].view(shape))
                s["out"].append(out[a:a + n].view(shape))
            s["flat"].append(flat)
            s["out_flat"].append(out)
        return s
    if case["op"] == "norm":
        b, n, c = case["b"], case["n"], case["c"]
        s["x"] = leaf((rand(b, n, c) + 0.3 * rand(c)).to(dt))
        s["residual"] = leaf((2.0 * rand(b, n, c) + 0.5 * rand(c)).to(dt)) if case["residual"] else None
        s["w"], s["b"] = leaf(1.0 + 0.2 * rand(c)), leaf(0.1 * rand(c))
        if case["train"]:
            s["g"] = rand(b, n, c).to(dt)
            s["gs"] = rand(b, n, c).to(dt) if case["residual"] else None
        return s
    b, nq, nk, hq, hkv, d = (case[k] for k in ("b", "nq", "nk", "hq", "hkv", "d"))

    def rows(n, heads):   # normed rows that vary slowly along the scene's order, plus what is each Gaussian's own
        slow = rand(b, n // 64 + 2, hkv, 1, d).expand(b, n // 64 + 2, hkv, heads // hkv, d).reshape(b, -1, heads, d)
        x = slow[:, torch.arange(n, device=dev) // 64].add_(rand(b, n, heads, d))
        return x.mul_(1.3 * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)).to(dt)

    s["k"] = leaf(rows(nk, hkv))
    s["q"] = leaf(rows(nq, hq))
    s["v"] = leaf(rand(b, nk, 2 * hkv, d).to(dt)[:, :, hkv:])   # a slice of the keys' fused projection
    s["mask"] = None
    if case["keep"] < 1.0 or case["empty"]:
        order = torch.rand(b, nk, generator=g, device=dev).argsort(1).argsort(1)
        s["mask"] = order < torch.tensor(_kept(case), device=dev)[:, None]
    if case["train"]:
        s["g"] = rand(b, nq, hq, d).to(dt)
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if own:
        return {"window": _own_window, "norm": _own_norm, "clip": _own_clip}[op](s)
    with torch.no_grad():
        return {"window": _plain_window, "norm": _plain_norm, "clip": _plain_clip}[op](s)


def _own_window(s):
    from CudaGaussianVoxelizer import gaussian_attention
    c = s["case"]
    out = gaussian_attention(s["q"], s["k"], s["v"], key_mask=s["mask"], window=(c["left"], c["right"]), sinks=c["sinks"])
    if not c["train"]:
        return {"out": out}
    return {"out": out, "grads": torch.autograd.grad(out, [s["q"], s["k"], s["v"]], s["g"])}


def _own_norm(s):
    from CudaGaussianVoxelizer import layer_norm
    if s["residual"] is None:
        y = layer_norm(s["x"], s["w"], s["b"], eps=EPS)
        if not s["case"]["train"]:
            return {"y": y}
        return {"y": y, "grads": torch.autograd.grad(y, [s["x"], s["w"], s["b"]], s["g"])}
    y, total = layer_norm(s["x"], s["w"], s["b"], residual=s["residual"], eps=EPS)
    if not s["case"]["train"]:
        return {"y": y, "sum": total}
    # the sum's two terms have the same gradient
    return {"y": y, "sum": total, "grads": torch.autograd.grad([y, total], [s["x"], s["w"], s["b"]], [s["g"], s["gs"]])}


def _own_clip(s):
    from CudaGaussianVoxelizer import clip_grad_norm_
    norm = clip_grad_norm_(s["grads"], s["case"]["max_norm"], out=s["out"])
    return {"norm": norm, "out": s["out_flat"]}


def _plain_window(s):
    """Blocks of queries with the keys that any of them sees: the sinks, then a slice."""
    c, dt = s["case"], s["q"].dtype
    (b, nq, hq, d), (nk, hkv) = s["q"].shape, s["k"].shape[1:3]
    dev, group, scale, shift = s["q"].device, hq // hkv, 1.0 / math.sqrt(d), nk - nq
    q, k, v = (s[n].float().transpose(1, 2).contiguous() for n in ("q", "k", "v"))
    out = torch.zeros(b, hq, nq, d, device=dev)
    if c["train"]:
        g = s["g"].float().transpose(1, 2).contiguous()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    step = 1024
    for i0 in range(0, nq, step):
        i1 = min(nq, i0 + step)
        hi = max(0, min(nk, i1 - 1 + shift + c["right"] + 1))
        lo = max(0, min(hi, i0 + shift - c["left"]))
        ns = min(c["sinks"], lo)

        def keys(x):
            return torch.cat([x[:, :, :ns], x[:, :, lo:hi]], 2)

        if ns + hi - lo == 0:
            continue
        j = torch.cat([torch.arange(ns, device=dev), torch.arange(lo, hi, device=dev)])
        p = torch.arange(i0, i1, device=dev)[:, None] + shift
        see = ((j <= p + c["right"]) & ((j >= p - c["left"]) | (j < c["sinks"])))[None, None, None]
        if s["mask"] is not None:
            see = see & s["mask"][:, j][:, None, None, None]
        m, kb, vb = i1 - i0, keys(k), keys(v)
        qb = q[:, :, i0:i1].reshape(b, hkv, group * m, d)
        w = torch.matmul(qb, kb.mT).mul_(scale).view(b, hkv, group, m, len(j))
        w = w.masked_fill_(~see, -math.inf).view(b, hkv, group * m, len(j))
        top = w.amax(-1, keepdim=True)
        w.sub_(torch.where(top.isinf(), torch.zeros_like(top), top)).exp_()
        total = w.sum(-1, keepdim=True)
        w.div_(torch.where(total > 0, total, torch.ones_like(total)))
        o = torch.matmul(w, vb)
        out[:, :, i0:i1] = o.view(b, hq, m, d)
        if not c["train"]:
            continue
        gb = g[:, :, i0:i1].reshape(b, hkv, group * m, d)
        dvb = torch.matmul(w.mT.contiguous(), gb)
        ds = torch.matmul(gb, vb.mT)
        ds.sub_((gb * o).sum(-1, keepdim=True)).mul_(w).mul_(scale)
        dq[:, :, i0:i1] = torch.matmul(ds, kb).view(b, hq, m, d)
        dkb = torch.matmul(ds.mT.contiguous(), qb)
        for total, part in ((dk, dkb), (dv, dvb)):
            total[:, :, :ns] += part[:, :, :ns]
            total[:, :, lo:hi] += part[:, :, ns:]

    def rows(x):
        return x.transpose(1, 2).to(dt, memory_format=torch.contiguous_format)

    return {"out": rows(out), "grads": (rows(dq), rows(dk), rows(dv))} if c["train"] else {"out": rows(out)}


def _plain_norm(s):
    dt, x, w = s["x"].dtype, s["x"].float(), s["w"]
    residual = s["residual"]
    if residual is not None:
        total = (x + residual.float()).to(dt)
        x = total.float()
    x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    x = x * r
    got = {"y": (x * w + s["b"]).to(dt)}
    if residual is not None:
        got["sum"] = total
    if not s["case"]["train"]:
        return got
    g = s["g"].float()
    t = g * w
    dx = r * (t - t.mean(-1, keepdim=True) - x * (t * x).mean(-1, keepdim=True))
    if residual is not None:
        dx = dx + s["gs"].float()
    got["grads"] = (dx.to(dt), (g * x).sum((0, 1)), g.sum((0, 1)))
    return got


def _plain_clip(s):
    total = torch.stack([g.float().square().sum() for g in s["grads"]]).sum()
    norm = total.sqrt()
    factor = (s["case"]["max_norm"] / (norm + CLIP_EPS)).clamp(max=1.0)
    for g, o in zip(s["grads"], s["out"]):
        o.copy_(g.float() * factor)
    return {"norm": norm, "out": s["out_flat"]}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _exact_norm(case, s):
    x, w, b = (s[n].detach().double().requires_grad_() for n in ("x", "w", "b"))
    total = x
    if case["residual"]:   # the rounding of the sum is part of the definition
        total = x + ((s["x"].detach().float() + s["residual"].detach().float()).to(s["x"].dtype).double() - x.detach())
    var, mean = torch.var_mean(total, -1, unbiased=False, keepdim=True)
    y = (total - mean) / (var + EPS).sqrt() * w + b
    got = {"y": y.detach()}
    if case["residual"]:
        got["sum"] = total.detach()
    if case["train"]:
        outs, gs = ([y, total], [s["g"].double(), s["gs"].double()]) if case["residual"] else ([y], [s["g"].double()])
        got["grads"] = torch.autograd.grad(outs, [x, w, b], gs)
    return got


def _exact_clip(case, s):
    norm = math.sqrt(sum(float(f.double().square().sum()) for f in s["flat"]))
    factor = min(1.0, case["max_norm"] / (norm + CLIP_EPS))
    return {"norm": torch.tensor(norm, dtype=torch.float64), "out": [f.double() * factor for f in s["flat"]]}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] != "window":
        return _exact_norm(case, s) if case["op"] == "norm" else _exact_clip(case, s)
    dev, group, train = s["q"].device, case["hq"] // case["hkv"], case["train"]
    nq, nk, left, right, sinks = (case[k] for k in ("nq", "nk", "left", "right", "sinks"))
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    out = torch.zeros_like(q)
    grads = [torch.zeros_like(t) for t in (q, k, v)]
    every = torch.arange(nk, device=dev)
    for i0 in range(0, nq, 4096):   # queries whose places are first .. last
        i1 = min(nq, i0 + 4096)
        first, last = i0 + nk - nq, i1 - 1 + nk - nq
        near = every[(every <= last + right) & ((every >= first - left) | (every < sinks))]
        place = torch.arange(first, last + 1, device=dev)[:, None]
        hidden = (near > place + right) | ((near < place - left) & (near >= sinks))
        for b in range(case["b"]):
            unseen = hidden if s["mask"] is None else hidden | ~s["mask"][b, near]
            alone = unseen.all(1, keepdim=True)
            for h in range(case["hq"]):
                qh, kh, vh = q[b, i0:i1, h], k[b, near, h // group], v[b, near, h // group]
                score = (qh @ kh.T / math.sqrt(case["d"])).masked_fill_(unseen, -1e300)
                p = torch.softmax(score, -1).masked_fill_(alone | unseen, 0.0)
                del score
                out[b, i0:i1, h] = p @ vh
                if train:
                    g = s["g"][b, i0:i1, h].double()
                    dp = g @ vh.T
                    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(case["d"])
                    grads[0][b, i0:i1, h] = ds @ kh
                    grads[1][b, :, h // group].index_add_(0, near, ds.T @ qh)
                    grads[2][b, :, h // group].index_add_(0, near, p.T @ g)
    return {"out": out, "grads": tuple(grads)} if train else {"out": out}


def _seen(case):
    """(pairs of a query and a key that it sees, keys that any query sees) of a scene without a mask."""
    nq, nk, left, right, sinks = (case[k] for k in ("nq", "nk", "left", "right", "sinks"))
    p = torch.arange(nk - nq, nk)
    hi = (p + right + 1).clamp(0, nk)
    lo = torch.minimum((p - left).clamp(0, nk), hi)
    pairs = int((hi - lo + torch.minimum(lo, torch.tensor(sinks))).sum())
    return pairs, nk - int(lo[0]) + min(sinks, int(lo[0]))


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "clip":   # read once; float32 written
        n = sum(_clip_numels(case))
        return {"bytes": n * (size + 4), "flops": 3 * n}
    if case["op"] == "norm":
        values, r = case["b"] * case["n"] * case["c"], case["residual"]
        if not case["train"]:
            return {"bytes": values * size * (4 if r else 2) + 8 * case["c"], "flops": 8 * values}
        # x (residual) in, y (sum) out; the gradients of y (and sum) in, that of x out
        return {"bytes": values * size * (7 if r else 4) + 16 * case["c"], "flops": 22 * values}
    b, nq, nk, hq, hkv, d = (case[k] for k in ("b", "nq", "nk", "hq", "hkv", "d"))
    pairs, keys = _seen(case)
    share = sum(_kept(case)) / (b * nk)
    queries = b * nq * hq * d * size
    flops = 4 * b * pairs * share * hq * d
    if not case["train"]:
        return {"bytes": 2 * queries + 2 * b * keys * share * hkv * d * size, "flops": flops}
    # forward: q, k, v in, the output out; backward: its gradient in, three gradients out
    return {"bytes": 4 * queries + 2 * b * keys * share * hkv * d * size + 2 * b * nk * hkv * d * size, "flops": 3.5 * flops}
