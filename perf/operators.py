"""Performance cases of the operators that run in front of the splat: Gaussian queries that attend to one another or to
image tokens, with norms and rotations by their positions.

A case is a dict of plain values: the operator ("op"), scenes "b", queries "nq" and keys "nk" of each scene, heads "hq" and
"hkv" (each key head serves hq / hkv query heads), head width "d", "dtype", and

    rotary     qk_norm_rotary: norms of queries and keys with the rotation by "axes" position coordinates; "shared": queries
               and keys are the same tokens
    attention  gaussian_attention: each scene keeps the fraction "keep" of its keys (1: no mask); "empty": its first scene none

each forward alone, or with "train" forward and backward with the gradients of all inputs.
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
EPS = 1e-6
RANGE = ((-40.0, 40.0), (-40.0, 40.0), (-1.0, 5.4), (0.0, 4.0))   # the scene of the published benchmark in metres; seconds
PLAIN_SCORES = 18000 * 18000 * 16   # scores that a drawn case may have: the plain form holds them


def _attention(name, train, b, nq, nk, hq, hkv, d, dtype, keep=1.0, empty=False):
    c = {"op": "attention", "train": train, "b": b, "nq": nq, "nk": nk, "hq": hq, "hkv": hkv, "d": d, "dtype": dtype,
         "keep": keep, "empty": empty}
    return dict(c, name=name) if name else c


def _rotary(name, train, b, nq, nk, hq, hkv, d, dtype, axes=3, shared=True):
    c = {"op": "rotary", "train": train, "b": b, "nq": nq, "nk": nk, "hq": hq, "hkv": hkv, "d": d, "dtype": dtype,
         "axes": axes, "shared": shared}
    return dict(c, name=name) if name else c


def listed():
    return [
        # a few hundred Gaussians before their first attention, no gradients: one launch
        _rotary("rotary_n300_h8d32", False, 1, 300, 300, 8, 8, 32, "f32"),
        # queries at Gaussians, keys at image tokens, shared key heads and a width that no vector divides, float32 training
        _rotary("rotary_train_ragged_d75", True, 2, 2999, 7001, 12, 4, 75, "f32", shared=False),
        # the headline scene's 1024 channels as 16 heads, one training step
        _rotary("rotary_train_n18000_h16d64_bf16", True, 1, 18000, 18000, 16, 16, 64, "bf16"),
        # one query that pools a whole scene (a planner's or a caption's token): bandwidth and latency
        _attention("pool_1x18000_h16d64_bf16", False, 1, 1, 18000, 16, 16, 64, "bf16"),
        # a batch of sparse scenes padded to 300 Gaussians, one of them empty
        _attention("infer_6x300_h8d32", False, 6, 300, 300, 8, 8, 32, "f32", 0.7, True),
        # a small float32 training step
        _attention("train_n2000_h8d32", True, 1, 2000, 2000, 8, 8, 32, "f32"),
        # float32 inference with a base backbone's 768 channels
        _attention("infer_n9000_h12d64", False, 1, 9000, 9000, 12, 12, 64, "f32"),
        # a training step with a fifth of the Gaussians pruned
        _attention("train_n9000_h12d64_bf16_masked", True, 1, 9000, 9000, 12, 12, 64, "bf16", 0.8),
        # Gaussians attending to image tokens, shared key heads, ragged sizes
        _attention("train_cross_ragged_d72_bf16", True, 2, 2999, 7001, 12, 4, 72, "bf16"),
        # wide heads
        _attention("train_n9000_h8d128_bf16", True, 1, 9000, 9000, 8, 8, 128, "bf16"),
        # the headline scene without gradients
        _attention("infer_n18000_h16d64_bf16", False, 1, 18000, 18000, 16, 16, 64, "bf16"),
        # the largest training step
        _attention("train_n18000_h8d64_bf16", True, 1, 18000, 18000, 8, 8, 64, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges; an attention takes no more products and a rotary moves no more bytes than the
    largest listed one."""
    train = rng.random() < 0.6
    dtype = rng.choice(["bf16", "bf16", "f32"])
    b = rng.choice([1, 1, 1, 2, 3, 6])
    d = rng.choice([32, 64, 64, 96, 128, rng.randint(16, 128), rng.randint(16, 128)])
    hkv, group = rng.randint(1, 8), rng.choice([1, 1, 2, 3, 4])
    hkv = max(1, min(hkv, 1024 // (group * d)))
    hq = hkv * group
    if rng.random() < 0.3:
        shared = rng.random() < 0.6
        axes = rng.choice([1, 2, 3, 3, 3, 4])
        nq = _log_int(rng, 300, 18000)
        if rng.random() < 0.3:
            nq = nq // 64 * 64
        nk = nq if shared else _log_int(rng, 300, 18000)
        while True:
            case = _rotary(None, train, b, nq, nk, hq, hkv, d, dtype, axes, shared)
            if work(case)["bytes"] <= 3.0e8:
                return case
            nq, nk = int(nq * 0.8), int(nk * 0.8)
    nk = _log_int(rng, 64, 18000)
    nq = nk if rng.random() < 0.5 else _log_int(rng, 1, 18000)
    keep = rng.choice([1.0, 1.0, round(rng.uniform(0.1, 0.95), 3)])
    empty = b > 1 and keep < 1.0 and rng.random() < 0.5
    most = 1.8e12 if dtype == "bf16" else 4.0e11   # float32 products run at a sixteenth of the bfloat16 ones' rate
    while True:
        case = _attention(None, train, b, nq, nk, hq, hkv, d, dtype, keep, empty)
        if work(dict(case, keep=1.0, empty=False))["flops"] <= most and b * hq * nq * nk <= PLAIN_SCORES:
            return case
        nq, nk = max(1, int(nq * 0.8)), max(64, int(nk * 0.8))


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _kept(case):
    """Valid keys of each scene."""
    n = [case["nk"]] * case["b"]
    if case["keep"] < 1.0:
        n = [int(case["nk"] * case["keep"])] * case["b"]
    if case["empty"]:
        n[0] = 0
    return n


def _normed(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)


def _tokens(g, b, n, mix, width):
    """Projected tokens (b, n, width): features of a scene vary along few directions ("mix"), plus what is each token's own."""
    dev = torch.device("cuda")
    return torch.randn(b, n, mix.shape[0], generator=g, device=dev) @ mix + 0.7 * torch.randn(b, n, width, generator=g, device=dev)


def _table(case):
    """(axes, pairs) angles per unit of each coordinate: an equal share of the pairs turns with each axis, wavelengths
    from two voxels to twice the scene."""
    axes, each = case["axes"], case["d"] // 2 // case["axes"]
    f = torch.zeros(axes, axes * each)
    for a in range(axes):
        step = torch.arange(each) / max(1, each - 1)
        f[a, a * each:(a + 1) * each] = 2 * math.pi / (0.8 * 200.0 ** step)
    return f.cuda()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    b, nq, nk, hq, hkv, d, dt = (case[k] for k in ("b", "nq", "nk", "hq", "hkv", "d", "dtype"))
    dt, train = DTYPES[dt], case["train"]

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def leaf(t):
        return t.detach().requires_grad_(train)

    group = hq // hkv
    mix = 0.4 * rand(16, hkv * d)
    mix_q = mix.view(16, hkv, 1, d).expand(16, hkv, group, d).reshape(16, hq * d)
    s = {"case": dict(case)}
    if case["op"] == "rotary":
        if case["shared"]:   # views of the tokens' fused projection
            qkv = torch.cat([_tokens(g, b, nq, mix_q, hq * d), _tokens(g, b, nq, mix, hkv * d), rand(b, nq, hkv * d)], -1)
            qkv = qkv.to(dt).view(b, nq, hq + 2 * hkv, d)
            s["q"], s["k"] = leaf(qkv[:, :, :hq]), leaf(qkv[:, :, hq:hq + hkv])
        else:
            s["q"] = leaf(_tokens(g, b, nq, mix_q, hq * d).to(dt).view(b, nq, hq, d))
            s["k"] = leaf(_tokens(g, b, nk, mix, hkv * d).to(dt).view(b, nk, hkv, d))
        lo = torch.tensor([r[0] for r in RANGE[:case["axes"]]], device=dev)
        hi = torch.tensor([r[1] for r in RANGE[:case["axes"]]], device=dev)

        def place(n):
            return leaf(lo + (hi - lo) * torch.rand(b, n, case["axes"], generator=g, device=dev))

        s["pos"] = place(nq)
        s["kpos"] = None if case["shared"] else place(nk)
        s["wq"], s["wk"] = (leaf(1.0 + 0.2 * rand(d)) for _ in range(2))
        s["freqs"] = _table(case)
        if train:
            s["gq"], s["gk"] = rand(b, nq, hq, d).to(dt), rand(b, nk, hkv, d).to(dt)
        return s
    q = _normed(_tokens(g, b, nq, mix_q, hq * d).view(b, nq, hq, d)) * 1.2
    k = _normed(_tokens(g, b, nk, mix, hkv * d).view(b, nk, hkv, d)) * 1.2
    s["q"], s["k"] = leaf(q.to(dt)), leaf(k.to(dt))
    # values are a slice of the keys' fused projection
    s["v"] = leaf(rand(b, nk, 2 * hkv, d).to(dt)[:, :, hkv:])
    s["mask"] = None
    if case["keep"] < 1.0 or case["empty"]:
        order = torch.rand(b, nk, generator=g, device=dev).argsort(1).argsort(1)
        s["mask"] = order < torch.tensor(_kept(case), device=dev)[:, None]
    if train:
        s["g"] = rand(b, nq, hq, d).to(dt)
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        return _own_rotary(s, c["train"]) if c["op"] == "rotary" else _own_attention(s, c["train"])
    with torch.no_grad():
        return _plain_rotary(s, c["train"]) if c["op"] == "rotary" else _plain_attention(s, c["train"])


def _own_rotary(s, train):
    from CudaGaussianVoxelizer import qk_norm_rotary
    q, k = qk_norm_rotary(s["q"], s["k"], s["pos"], s["freqs"], s["wq"], s["wk"], k_positions=s["kpos"], eps=EPS)
    if not train:
        return {"q": q, "k": k}
    wrt = [s["q"], s["k"], s["pos"], s["wq"], s["wk"]] + ([] if s["kpos"] is None else [s["kpos"]])
    return {"q": q, "k": k, "grads": torch.autograd.grad([q, k], wrt, [s["gq"], s["gk"]])}


def _own_attention(s, train):
    from CudaGaussianVoxelizer import gaussian_attention
    out = gaussian_attention(s["q"], s["k"], s["v"], key_mask=s["mask"])
    if not train:
        return {"out": out}
    return {"out": out, "grads": torch.autograd.grad(out, [s["q"], s["k"], s["v"]], s["g"])}


def _plain_rotate(x, cos, sin):
    """The first pairs of x (.., d) turned; what is left of d stays."""
    p = cos.shape[-1]
    x0, x1 = x[..., 0:2 * p:2], x[..., 1:2 * p:2]
    turned = torch.stack([x0 * cos - x1 * sin, x0 * sin + x1 * cos], -1).flatten(-2)
    return torch.cat([turned, x[..., 2 * p:]], -1)


def _plain_side(x, w, pos, freqs, g):
    """One of the two tensors: its output and, with g, the gradients of x, w and the angles."""
    dt, x = x.dtype, x.float()
    angle = (pos[..., :, None] * freqs).sum(-2)[:, :, None]
    cos, sin = angle.cos(), angle.sin()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    y = x * r * w
    out = _plain_rotate(y, cos, sin).to(dt)
    if g is None:
        return out, None
    dy = _plain_rotate(g.float(), cos, -sin)
    dw = (dy * x * r).sum((0, 1, 2))
    t = dy * w
    dx = r * t - x * r.pow(3) * (t * x).mean(-1, keepdim=True)
    p = freqs.shape[1]
    turn = (dy[..., 1:2 * p:2] * y[..., 0:2 * p:2] - dy[..., 0:2 * p:2] * y[..., 1:2 * p:2]).sum(2)
    return out, (dx.to(dt), dw, (turn[:, :, None, :] * freqs).sum(-1))


def _plain_rotary(s, train):
    kpos = s["pos"] if s["kpos"] is None else s["kpos"]
    q, dq = _plain_side(s["q"], s["wq"], s["pos"], s["freqs"], s["gq"] if train else None)
    k, dk = _plain_side(s["k"], s["wk"], kpos, s["freqs"], s["gk"] if train else None)
    if not train:
        return {"q": q, "k": k}
    shared = s["kpos"] is None
    grads = (dq[0], dk[0], dq[2] + dk[2] if shared else dq[2], dq[1], dk[1]) + (() if shared else (dk[2],))
    return {"q": q, "k": k, "grads": grads}


def _heads_first(x, hkv):
    """(b, n, h, d) as float32 (b, hkv, h / hkv, n, d): the query heads of each key head side by side."""
    b, n, h, d = x.shape
    return x.float().view(b, n, hkv, h // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, h // hkv * n, d)


def _tokens_first(x, n, dt):
    b, hkv, rows, d = x.shape
    return x.view(b, hkv, rows // n, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, hkv * (rows // n), d).to(dt)


def _plain_attention(s, train):
    dt, (b, nq, hq, d), (nk, hkv) = s["q"].dtype, s["q"].shape, s["k"].shape[1:3]
    scale = 1.0 / math.sqrt(d)
    q = _heads_first(s["q"], hkv)
    k, v = (s[n].float().permute(0, 2, 1, 3).contiguous() for n in ("k", "v"))
    p = torch.matmul(q, k.mT).mul_(scale)
    if s["mask"] is not None:
        p.masked_fill_(~s["mask"][:, None, None, :], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top.isinf(), torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    o = torch.matmul(p, v)
    out = _tokens_first(o, nq, dt)
    if not train:
        return {"out": out}
    g = _heads_first(s["g"], hkv)
    dv = torch.matmul(p.mT, g)
    ds = torch.matmul(g, v.mT)
    ds.sub_((g * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.mT, q)
    return {"out": out, "grads": (_tokens_first(dq, nq, dt), _tokens_first(dk, nk, dt), _tokens_first(dv, nk, dt))}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _exact_rotary(case, s):
    def side(x, w, pos):
        x = x.detach().double().requires_grad_()
        w = w.detach().double().requires_grad_()
        pos = pos.detach().double().requires_grad_()
        f = s["freqs"].double()
        y = w * x / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
        n = 2 * f.shape[1]
        z = torch.view_as_complex(y[..., :n].unflatten(-1, (-1, 2)).contiguous())
        angle = pos @ f
        z = z * torch.polar(torch.ones_like(angle), angle)[:, :, None]
        return (x, w, pos), torch.cat([torch.view_as_real(z).flatten(-2), y[..., n:]], -1)

    (q, wq, pos), oq = side(s["q"], s["wq"], s["pos"])
    (k, wk, kpos), ok = side(s["k"], s["wk"], s["pos"] if s["kpos"] is None else s["kpos"])
    if not case["train"]:
        return {"q": oq.detach(), "k": ok.detach()}
    dq, dwq, dpos = torch.autograd.grad(oq, [q, wq, pos], s["gq"].double())
    dk, dwk, dkpos = torch.autograd.grad(ok, [k, wk, kpos], s["gk"].double())
    shared = s["kpos"] is None
    grads = (dq, dk, dpos + dkpos if shared else dpos, dwq, dwk) + (() if shared else (dkpos,))
    return {"q": oq.detach(), "k": ok.detach(), "grads": grads}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, s)
    group = case["hq"] // case["hkv"]
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    out = torch.zeros_like(q)
    grads = [torch.zeros_like(t) for t in (q, k, v)]
    for b in range(case["b"]):   # one head at a time: its scores are held once
        keys = torch.arange(case["nk"], device=q.device)
        if s["mask"] is not None:
            keys = keys[s["mask"][b]]
        if not len(keys):
            continue
        for h in range(case["hq"]):
            qh, kh, vh = q[b, :, h], k[b, keys, h // group], v[b, keys, h // group]
            p = torch.softmax(qh @ kh.T / math.sqrt(case["d"]), -1)
            out[b, :, h] = p @ vh
            if case["train"]:
                g = s["g"][b, :, h].double()
                dp = g @ vh.T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(case["d"])
                grads[0][b, :, h] = ds @ kh
                grads[1][b, keys, h // group] += ds.T @ qh
                grads[2][b, keys, h // group] += p.T @ g
                del dp, ds
            del p
    return {"out": out, "grads": tuple(grads)} if case["train"] else {"out": out}


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    b, nq, nk, hq, hkv, d = (case[k] for k in ("b", "nq", "nk", "hq", "hkv", "d"))
    if case["op"] == "rotary":
        values = b * d * (nq * hq + nk * hkv)
        places = 4 * case["axes"] * b * (nq + (0 if case["shared"] else nk))
        if not case["train"]:
            return {"bytes": 2 * values * size + places, "flops": 8 * values}
        # q, k and both gradients in; outputs and gradients out; positions and their gradient
        return {"bytes": 4 * values * size + 2 * places, "flops": 28 * values}
    keys = sum(_kept(case))
    queries = b * nq * hq * d * size
    flops = 4 * nq * keys * hq * d
    if not case["train"]:
        return {"bytes": 2 * queries + 2 * keys * hkv * d * size, "flops": flops}
    # forward: q, k, v in, the output out; backward: its gradient in, three gradients out
    return {"bytes": 4 * queries + 2 * keys * hkv * d * size + 2 * b * nk * hkv * d * size, "flops": 3.5 * flops}
