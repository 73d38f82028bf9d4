"""Cases for the channel-last operators next to the DDPM: group norm with an
activation, the matrix product with bias, activation and residual, and dropout
from a counter-based generator.

``listed()`` names the measured cases, ``draw(rng)`` makes more of the same
ranges, ``prepare(case, seed)`` makes a case's inputs on the GPU, and
``run(state)`` makes one pass: elementary torch operations in 32 bits while
``own`` is false, the library's calls while it is true. ``exact(case, seed)``
is the same in 64 bits, written from the definitions apart from ``run``.

Definitions (z is the argument of the activation ``act``):

* group norm: per sample and group of C / G channels over all pixels,
  z = (x - mean) / sqrt(var + eps) * weight + bias, out = act(z)
* linear: z = x weight^T + bias, out = act(z) + residual
* dropout: the value at position q = offset + i is kept if
  philox4x32_10(counter = (q // 4, 0), key = seed)[q % 4] >= round(p * 2^32),
  out = x * kept / (1 - p) + residual
"""

import math

import numpy as np
import torch

own = False

EPS = 1e-5
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one small map of the decoder, inference: nothing but latency
        dict(name="norm_16x16_fp32", op="norm", n=1, c=64, h=16, w=16, groups=8, act="silu",
             dtype="fp32", train=False),
        # a ragged crop: odd rows and columns, groups of 12 channels
        dict(name="norm_odd_fp16_train", op="norm", n=3, c=60, h=37, w=53, groups=5, act="gelu",
             dtype="fp16", train=True),
        # training at half resolution, a batch of 8
        dict(name="norm_128_b8_bf16_train", op="norm", n=8, c=64, h=128, w=128, groups=8,
             act="silu", dtype="bf16", train=True),
        # the benchmark's own training batch: 64 maps of 256 x 256
        dict(name="norm_256_b64_bf16_train", op="norm", n=64, c=64, h=256, w=256, groups=8,
             act="silu", dtype="bf16", train=True),
        # one pooled vector or one token: the weight has to be read, nothing else counts
        dict(name="linear_one_row_bf16", op="linear", m=1, k=1024, n=4096, act="silu", bias=True,
             residual=True, dtype="bf16", train=False),
        # the taps of a 256 x 256 map from its 64 channels (3 x 64 x 9 outputs a pixel)
        dict(name="linear_taps_bf16", op="linear", m=65536, k=64, n=1728, act="none", bias=True,
             residual=False, dtype="bf16", train=False),
        # ragged rows and widths, a training step
        dict(name="linear_odd_fp16_train", op="linear", m=1999, k=200, n=333, act="silu",
             bias=True, residual=True, dtype="fp16", train=True),
        # 4C -> C projection of a 256 x 256 map onto its residual, in full precision
        dict(name="linear_project_fp32_train", op="linear", m=65536, k=256, n=64, act="none",
             bias=True, residual=True, dtype="fp32", train=True),
        # a wide expansion, a training step: bound by the matrix products
        dict(name="linear_expand_bf16_train", op="linear", m=16384, k=1024, n=4096, act="gelu",
             bias=True, residual=False, dtype="bf16", train=True),
        # one small map: latency
        dict(name="dropout_16x16_fp32", op="dropout", size=16384, p=0.1, offset=0, residual=False,
             dtype="fp32", train=False),
        # dropout onto a residual, a training step at half resolution with a batch of 8
        dict(name="dropout_128_b8_bf16_train", op="dropout", size=8388608, p=0.1, offset=0,
             residual=True, dtype="bf16", train=True),
        # the benchmark's own batch
        dict(name="dropout_256_b64_bf16", op="dropout", size=268435456, p=0.25, offset=0,
             residual=False, dtype="bf16", train=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "linear", "dropout"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    train = rng.random() < 0.5
    if op == "norm":
        while True:
            groups = rng.choice([1, 2, 3, 4, 5, 8, 16, 32])
            c = groups * rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 24])
            n, h, w = _log(rng, 1, 64), _log(rng, 1, 256), _log(rng, 1, 256)
            # groups of fewer than 64 values have next to no gradient left to compare
            if n * c * h * w <= 2 ** 26 and c // groups * h * w >= 64:
                break
        # a rounding turns a relu's gradient on or off at z = 0, which 32 bits show
        act = rng.choice(["none", "silu", "gelu"] + (["relu"] if dtype != "fp32" else []))
        return dict(op=op, n=n, c=c, h=h, w=w, groups=groups, act=act, dtype=dtype, train=train)
    if op == "linear":
        while True:
            m, k, n = _log(rng, 1, 65536), _log(rng, 1, 4096), _log(rng, 1, 4096)
            if m * k * n <= 2 ** 35 and m * max(k, n) <= 2 ** 27:
                break
        if rng.random() < 0.5:
            k = max(8, k // 8 * 8)
        if rng.random() < 0.5:
            n = max(8, n // 8 * 8)
        act = rng.choice(["none", "silu", "gelu"] + (["relu"] if dtype != "fp32" else []))
        return dict(op=op, m=m, k=k, n=n, act=act, bias=rng.random() < 0.75,
                    residual=rng.random() < 0.5, dtype=dtype, train=train)
    return dict(op=op, size=_log(rng, 1, 2 ** 26), p=rng.choice([0.05, 0.1, 0.25, 0.5]),
                offset=rng.choice([0, rng.randrange(2 ** 20), rng.randrange(2 ** 40)]),
                residual=rng.random() < 0.5, dtype=dtype, train=train)


# ---------------------------------------------------------------- inputs ----
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    s = dict(case)
    grad = case["train"]
    if case["op"] == "norm":
        n, c, h, w = (case[k] for k in ("n", "c", "h", "w"))
        # channels of different spread and mean, as a convolution leaves them
        x = normal(n, h, w, c).mul_(normal(c).abs_().add_(0.25)).add_(normal(c)).to(t)
        s["x"] = x.permute(0, 3, 1, 2).requires_grad_(grad)
        s["weight"] = normal(c).mul_(0.2).add_(1).to(t).requires_grad_(grad)
        s["bias"] = normal(c).mul_(0.2).to(t).requires_grad_(grad)
        if grad:
            s["dy"] = normal(n, h, w, c).to(t).permute(0, 3, 1, 2)
    elif case["op"] == "linear":
        m, k, n = (case[i] for i in ("m", "k", "n"))
        s["x"] = normal(m, k).to(t).requires_grad_(grad)
        s["weight"] = normal(n, k).div_(math.sqrt(k)).to(t).requires_grad_(grad)
        s["bias"] = normal(n).mul_(0.2).to(t).requires_grad_(grad) if case["bias"] else None
        s["residual"] = normal(m, n).to(t).requires_grad_(grad) if case["residual"] else None
        if grad:
            s["dy"] = normal(m, n).to(t)
    else:
        size = case["size"]
        s["seed"] = (seed * 0x9E3779B97F4A7C15 + 12345) % 2 ** 63
        s["x"] = normal(size).to(t).requires_grad_(grad)
        s["residual"] = normal(size).to(t).requires_grad_(grad) if case["residual"] else None
        if grad:
            s["dy"] = normal(size).to(t)
    return s


# ------------------------------------------------------------ plain forms ----
def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return z * (0.5 * (1 + torch.erf(z * math.sqrt(0.5))))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        e = 1 / (1 + torch.exp(-z))
        return e * (1 + z * (1 - e))
    if act == "gelu":
        return (0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
                + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi)))
    return torch.ones_like(z)


def _norm(s):
    n, c, h, w = s["x"].shape
    groups, t = s["groups"], s["x"].dtype

    def rows(v):  # [n, pixels, groups, channels of a group]
        return v.permute(0, 2, 3, 1).reshape(n, h * w, groups, c // groups).float()

    def image(v):
        return v.reshape(n, h, w, c).to(t).permute(0, 3, 1, 2)

    x = rows(s["x"])
    weight, bias = (s[k].float().reshape(groups, c // groups) for k in ("weight", "bias"))
    mean = x.mean((1, 3), keepdim=True)
    var = (x - mean).square().mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(var + EPS)
    xhat = (x - mean) * rstd
    z = xhat * weight + bias
    out = [image(_act(z, s["act"]))]
    if s["train"]:
        dz = rows(s["dy"]) * _act_grad(z, s["act"])
        dxhat = dz * weight
        dx = rstd * (dxhat - dxhat.mean((1, 3), keepdim=True)
                     - xhat * (dxhat * xhat).mean((1, 3), keepdim=True))
        out += [image(dx), (dz * xhat).sum((0, 1)).reshape(c).to(t),
                dz.sum((0, 1)).reshape(c).to(t)]
    return out


def _linear(s):
    t = s["x"].dtype
    x, weight = s["x"].float(), s["weight"].float()
    z = x @ weight.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    out = _act(z, s["act"])
    if s["residual"] is not None:
        out = out + s["residual"].float()
    out = [out.to(t)]
    if s["train"]:
        dz = s["dy"].float() * _act_grad(z, s["act"])
        out += [(dz @ weight).to(t), (dz.t() @ x).to(t)]
        if s["bias"] is not None:
            out.append(dz.sum(0).to(t))
        if s["residual"] is not None:
            out.append(s["dy"])
    return out


def _mul32(a, m):
    """High and low 32 bits of a * m; the 64-bit product wraps, its bits do not change."""
    p = a * m
    return (p >> 32) & 0xFFFFFFFF, p & 0xFFFFFFFF


def _kept(size, p, seed, offset, device):
    first = offset // 4
    block = torch.arange(first, (offset + size + 3) // 4, device=device, dtype=torch.int64)
    c = [block & 0xFFFFFFFF, block >> 32, torch.zeros_like(block), torch.zeros_like(block)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        hi0, lo0 = _mul32(c[0], 0xD2511F53)
        hi1, lo1 = _mul32(c[2], 0xCD9E8D57)
        c = [hi1 ^ c[1] ^ k0, lo1, hi0 ^ c[3] ^ k1, lo0]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    least = min(int(math.floor(p * 2 ** 32 + 0.5)), 2 ** 32)
    return (torch.stack(c, 1) >= least).reshape(-1)[offset - 4 * first:][:size]


def _dropout(s):
    t = s["x"].dtype
    kept = _kept(s["size"], s["p"], s["seed"], s["offset"], s["x"].device).float() * (1 / (1 - s["p"]))
    out = s["x"].float() * kept
    if s["residual"] is not None:
        out = out + s["residual"].float()
    out = [out.to(t)]
    if s["train"]:
        out.append((s["dy"].float() * kept).to(t))
        if s["residual"] is not None:
            out.append(s["dy"])
    return out


def _own(s):
    """The library's calls, as a user makes them."""
    from dynamicconvolutionoperator_b200 import dropout, group_norm_act, linear_act

    act = None if s.get("act") == "none" else s.get("act")

    def call():
        if s["op"] == "norm":
            return group_norm_act(s["x"], s["groups"], s["weight"], s["bias"], EPS, activation=act)
        if s["op"] == "linear":
            return linear_act(s["x"], s["weight"], s["bias"], activation=act,
                              residual=s["residual"])
        return dropout(s["x"], s["p"], s["seed"], offset=s["offset"], residual=s["residual"])

    if not s["train"]:
        with torch.no_grad():
            return [call()]
    leaves = [s[k] for k in ("x", "weight", "bias", "residual") if s.get(k) is not None]
    out = call()
    return [out.detach(), *torch.autograd.grad(out, leaves, s["dy"])]


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"norm": _norm, "linear": _linear, "dropout": _dropout}[state["op"]](state)


# ------------------------------------------------------------------ work ----
def work(case):
    """Each input read once and each output written once. Operations: two per
    multiply-add of the matrix products, a handful per value of the others."""
    size = 4 if case["dtype"] == "fp32" else 2
    train = case["train"]
    if case["op"] == "norm":
        values = case["n"] * case["c"] * case["h"] * case["w"]
        # x, out; dy, dx
        return {"bytes": values * size * (4 if train else 2) + case["c"] * size * (4 if train else 2),
                "flops": values * (30 if train else 12)}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        # x, weight, out, bias, residual; dy, dx, dweight, dbias (the residual's gradient is dy)
        values = m * k + n * k + m * n + n * case["bias"] + m * n * case["residual"]
        if train:
            values += m * n + m * k + n * k + n * case["bias"]
        return {"bytes": values * size, "flops": 2 * m * n * k * (3 if train else 1)}
    values = case["size"]
    # x, out, residual; dy, dx; the generator's ten rounds are about 15 operations a value
    return {"bytes": values * size * (2 + case["residual"] + 2 * train),
            "flops": values * 15 * (2 if train else 1)}


# ----------------------------------------------------------------- exact ----
def _sigma(z):
    return torch.sigmoid(z)


def _phi(z):
    return torch.special.ndtr(z)


_VALUE = {
    "none": lambda z: z,
    "relu": lambda z: torch.where(z > 0, z, torch.zeros_like(z)),
    "silu": lambda z: z * _sigma(z),
    "gelu": lambda z: z * _phi(z),
}
_SLOPE = {
    "none": lambda z: torch.ones_like(z),
    "relu": lambda z: torch.where(z > 0, torch.ones_like(z), torch.zeros_like(z)),
    "silu": lambda z: _sigma(z) + z * _sigma(z) * _sigma(-z),
    "gelu": lambda z: _phi(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi),
}


def _exact_norm(case, s):
    n, c, h, w = s["x"].shape
    groups = case["groups"]
    out, dx = [], []
    dweight = torch.zeros(c, dtype=torch.float64, device="cuda")
    dbias = torch.zeros_like(dweight)
    weight, bias = s["weight"].detach().double(), s["bias"].detach().double()
    for i in range(n):
        x = s["x"][i].detach().double().reshape(groups, -1)
        spread, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        scale = torch.rsqrt(spread + EPS)
        xhat = ((x - mean) * scale).reshape(c, h * w)
        z = torch.addcmul(bias[:, None], xhat, weight[:, None])
        out.append(_VALUE[case["act"]](z).reshape(c, h, w))
        if case["train"]:
            dz = s["dy"][i].double().reshape(c, h * w) * _SLOPE[case["act"]](z)
            dweight += torch.linalg.vecdot(dz, xhat)
            dbias += dz.sum(1)
            d = (dz * weight[:, None]).reshape(groups, -1)
            xg = xhat.reshape(groups, -1)
            along = torch.linalg.vecdot(d, xg)[:, None] / x.shape[1]
            dx.append(((d - d.mean(1, keepdim=True) - xg * along) * scale).reshape(c, h, w))
    return [torch.stack(out)] + ([torch.stack(dx), dweight, dbias] if case["train"] else [])


def _exact_linear(case, s):
    x, weight = s["x"].detach().double(), s["weight"].detach().double()
    z = torch.einsum("mk,nk->mn", x, weight)
    if case["bias"]:
        z += s["bias"].detach().double()
    y = _VALUE[case["act"]](z)
    if case["residual"]:
        y = y + s["residual"].detach().double()
    if not case["train"]:
        return [y]
    dz = s["dy"].double() * _SLOPE[case["act"]](z)
    got = [y, torch.einsum("mn,nk->mk", dz, weight), torch.einsum("mn,mk->nk", dz, x)]
    if case["bias"]:
        got.append(torch.einsum("mn->n", dz))
    if case["residual"]:
        got.append(s["dy"].double())
    return got


def _exact_words(q, seed):
    """The generator's word at each position, its products put together from
    factors of 32 and 16 bits, which do not pass 48."""
    def product(a, m):
        low, high = a * (m & 0xFFFF), a * (m >> 16)
        return ((low >> 16) + high) >> 16, (low + ((high & 0xFFFF) << 16)) & 0xFFFFFFFF

    block = torch.div(q, 4, rounding_mode="floor")
    a, b = block % 2 ** 32, torch.div(block, 2 ** 32, rounding_mode="floor")
    c = d = torch.zeros_like(a)
    keys = [[(k + i * step) % 2 ** 32 for i in range(10)]
            for k, step in ((seed % 2 ** 32, 0x9E3779B9), (seed // 2 ** 32, 0xBB67AE85))]
    for k, j in zip(*keys):
        (ah, al), (ch, cl) = product(a, 0xD2511F53), product(c, 0xCD9E8D57)
        a, b, c, d = torch.bitwise_xor(ch, b).bitwise_xor(torch.full_like(b, k)), cl, \
            torch.bitwise_xor(ah, d).bitwise_xor(torch.full_like(d, j)), al
    lane = q % 4
    return torch.where(lane == 0, a, torch.where(lane == 1, b, torch.where(lane == 2, c, d)))


def _exact_dropout(case, s):
    size, p = case["size"], case["p"]
    least = int(np.floor(np.float64(p) * 4294967296.0 + 0.5))
    out = s["x"].detach().double()
    dx = s["dy"].double() if case["train"] else None
    for at in range(0, size, 1 << 24):
        to = min(size, at + (1 << 24))
        q = torch.arange(case["offset"] + at, case["offset"] + to, device="cuda")
        drop = _exact_words(q, s["seed"]) < least
        for v in (out, dx):
            if v is not None:
                v[at:to] = torch.where(drop, torch.zeros_like(v[at:to]), v[at:to] / (1 - p))
    if case["residual"]:
        out += s["residual"].detach().double()
    got = [out]
    if case["train"]:
        got.append(dx)
        if case["residual"]:
            got.append(s["dy"].double())
    return got


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "linear": _exact_linear,
                "dropout": _exact_dropout}[case["op"]](case, s)
