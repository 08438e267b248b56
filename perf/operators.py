"""Cases for the 8-bit block operators of ``maggy_amd.ops``.

Four operators share one 8-bit format, OCP e4m3 codes with one power-of-two
scale for 128 neighbouring values:

``pack8`` / ``unpack8``  a tensor held in 8 bits and read back
``swiglu8``              silu(g) * u, whose backward pass reads g and u in
                         8 bits
``rms_norm8``            RMSNorm, whose backward pass reads x in 8 bits
``linear8``              x @ W^T of 8-bit operands, with both gradients, or
                         on weights that were packed once for serving

The format: for a block of 128 values with largest finite magnitude A, the
scale is 2^t with the smallest t >= -126 that has A <= 448 * 2^t; a code is
x * 2^-t rounded to e4m3, ties to even.  Activations and gradients have
blocks along the axis that the product sums over, weights have blocks of
128 x 128, so that a weight and its transpose stand for the same values.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16,
          "fp32": torch.float32}


def listed():
    return [
        # one decoded token through the 1B model's attention projections
        # (dim 2048): latency
        {"name": "serve-1x2048x2048", "op": "serve", "m": 1, "k": 2048,
         "n": 2048, "dtype": "bf16"},
        # a decode step of 8 sequences through the 8B feed-forward's way up
        {"name": "serve-8x4096x14336", "op": "serve", "m": 8, "k": 4096,
         "n": 14336, "dtype": "bf16"},
        # a prompt batch of 8 x 512 tokens through the 8B way down
        {"name": "serve-4096x14336x4096", "op": "serve", "m": 4096,
         "k": 14336, "n": 4096, "dtype": "bf16"},
        # the 8B benchmark's training step (6 x 4096 tokens), way up
        {"name": "train-24576x4096x14336", "op": "train", "m": 24576,
         "k": 4096, "n": "14336", "dtype": "bf16"},
        # gate and up of the 1B model from one packed input, 4096 tokens
        {"name": "train-4096x2048x8192+8192", "op": "train", "m": 4096,
         "k": 2048, "n": "8192+8192", "dtype": "bf16"},
        # nothing a multiple of a tile: a ragged batch, odd widths
        {"name": "train-1001x1111x777", "op": "train", "m": 1001, "k": 1111,
         "n": "777", "dtype": "bf16"},
        # the 8B feed-forward's gate, 6 x 4096 tokens
        {"name": "swiglu-24576x14336", "op": "swiglu", "m": 24576,
         "k": 14336, "dtype": "bf16"},
        # a short odd batch of a small model
        {"name": "swiglu-37x1000", "op": "swiglu", "m": 37, "k": 1000,
         "dtype": "fp16"},
        # the 8B model's norms, 6 x 4096 tokens
        {"name": "rms-24576x4096", "op": "rms", "m": 24576, "k": 4096,
         "dtype": "bf16"},
        # a handful of rows of an odd width: latency
        {"name": "rms-7x2050", "op": "rms", "m": 7, "k": 2050,
         "dtype": "fp32"},
        # a residual stream kept over a block, 6 x 4096 tokens
        {"name": "pack-24576x4096", "op": "pack", "m": 24576, "k": 4096,
         "dtype": "bf16"},
        # a small odd tensor kept
        {"name": "pack-333x517", "op": "pack", "m": 333, "k": 517,
         "dtype": "fp32"},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm, often odd."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    pick = rng.random()
    if pick < 0.3 and n >= 256:
        n = n // 128 * 128
    elif pick < 0.6:
        n |= 1
    return min(max(n, lo), hi)


def draw(rng):
    case = _any(rng)
    # no drawn case costs more than the largest listed one of its kind
    most = {c["op"]: work(c) for c in reversed(listed())
            if c["m"] >= 4096}
    while any(work(case)[w] > most[case["op"]][w]
              for w in ("bytes", "flops")):
        case["m"] = case["m"] * 3 // 4
    return case


def _any(rng):
    op = rng.choice(["serve", "serve", "train", "train", "swiglu", "rms",
                     "pack"])
    if op == "serve":
        return {"op": op, "m": _spread(rng, 1, 4096),
                "k": _spread(rng, 64, 14336), "n": _spread(rng, 64, 14336),
                "dtype": "bf16"}
    if op == "train":
        return {"op": op, "m": _spread(rng, 1, 24576),
                "k": _spread(rng, 64, 8192),
                "n": "+".join(str(_spread(rng, 32, 4096)) for _ in range(
                    rng.choice([1, 1, 2, 3]))),
                "dtype": "bf16"}
    return {"op": op, "m": _spread(rng, 1, 24576),
            "k": _spread(rng, 64, 14336 if op == "swiglu" else 8192),
            "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}


def _widths(case):
    return [int(n) for n in case["n"].split("+")]


# --------------------------------------------------------------- the inputs
class _Make:
    """Normal numbers from one seed, on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        t = torch.empty(shape, device="cuda", dtype=dtype)
        return t.normal_(0.0, std, generator=self.gen)

    def activation(self, m, k, dtype):
        """Rows of different size with a few loud channels, as a residual
        stream has them."""
        x = self.normal(m, k, dtype=dtype)
        x *= torch.exp(0.5 * self.normal(m, 1)).to(dtype)
        x *= torch.exp(self.normal(1, k).clamp_(max=3.0)).to(dtype)
        return x


def prepare(case, seed):
    mk = _Make(seed)
    dt = _TYPES[case["dtype"]]
    op, m, k = case["op"], case["m"], case["k"]
    if op == "serve":
        w = mk.normal(case["n"], k, std=0.02, dtype=dt)
        x = mk.activation(m, k, dt)
        if own:
            from maggy_amd import ops

            return {"op": op, "x": x, "w": ops.pack_weight8(w)}
        return {"op": op, "x": x, "w": _weight_values(w.float())}
    if op == "train":
        x = mk.activation(m, k, dt).requires_grad_(True)
        ws = [mk.normal(n, k, std=0.02, dtype=dt).requires_grad_(True)
              for n in _widths(case)]
        dys = [mk.normal(m, n, std=1e-3, dtype=dt) for n in _widths(case)]
        return {"op": op, "x": x, "ws": ws, "dys": dys}
    if op == "swiglu":
        return {"op": op, "g": mk.normal(m, k, dtype=dt).requires_grad_(True),
                "u": mk.normal(m, k, dtype=dt).requires_grad_(True),
                "dy": mk.normal(m, k, std=1e-3, dtype=dt)}
    if op == "rms":
        return {"op": op, "x": mk.activation(m, k, dt).requires_grad_(True),
                "w": (1.0 + 0.1 * mk.normal(k)).requires_grad_(True),
                "dy": mk.normal(m, k, std=1e-2, dtype=dt), "eps": 1e-5}
    return {"op": op, "x": mk.activation(m, k, dt)}


# ----------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


def _run_own(s):
    from maggy_amd import ops

    op = s["op"]
    if op == "serve":
        return ops.linear8(s["x"], s["w"])
    if op == "train":
        ys = ops.linear8(s["x"], *s["ws"])
        ys = ys if isinstance(ys, tuple) else (ys,)
        grads = torch.autograd.grad(ys, [s["x"], *s["ws"]], s["dys"])
        return [y.detach() for y in ys] + list(grads)
    if op == "swiglu":
        h = ops.swiglu8(s["g"], s["u"])
        return [h.detach(),
                *torch.autograd.grad(h, (s["g"], s["u"]), s["dy"])]
    if op == "rms":
        y = ops.rms_norm8(s["x"], s["w"], s["eps"])
        return [y.detach(),
                *torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])]
    return ops.unpack8(ops.pack8(s["x"]))


def _held(a):
    """The values that blocks of 128 along the last axis of ``a`` stand for
    in 8 bits (fp32 in, fp32 out)."""
    r, c = a.shape
    pad = -c % 128
    if pad:
        a = torch.nn.functional.pad(a, (0, pad))
    b = a.view(r, -1, 128)
    return (_rounded(b, b.abs().amax(-1, keepdim=True))
            .view(r, -1)[:, :c])


def _weight_values(w):
    """The same for blocks of 128 x 128."""
    n, k = w.shape
    w = torch.nn.functional.pad(w, (0, -k % 128, 0, -n % 128))
    b = w.view(w.shape[0] // 128, 128, w.shape[1] // 128, 128)
    v = _rounded(b, b.abs().amax((1, 3), keepdim=True))
    return v.view(w.shape)[:n, :k]


def _rounded(b, top):
    # top = frac * 2^e with frac in [1/2, 1); 448 = 7/8 * 2^9
    frac, e = torch.frexp(top)
    t = (e - 9 + (frac > 0.875)).clamp_(min=-126)
    t = torch.where(top == 0, -126, t)
    # 2^t by its bits: ldexp goes through pow, which is not exact
    scale = ((t.int() + 127) << 23).view(torch.float32)
    inverse = ((127 - t.int()) << 23).view(torch.float32)
    return (b * inverse).to(torch.float8_e4m3fn).float() * scale


@torch.no_grad()
def _run_plain(s):
    op = s["op"]
    if op == "serve":
        x = s["x"]
        return (_held(x.float()) @ s["w"].t()).to(x.dtype)
    if op == "train":
        x, ws, dys = s["x"], s["ws"], s["dys"]
        held = _held(x.float())
        over_rows = _held(held.t().contiguous())
        ys, dws, dx = [], [], None
        for w, dy in zip(ws, dys):
            wv, d = _weight_values(w.float()), dy.float()
            ys.append((held @ wv.t()).to(x.dtype))
            part = _held(d) @ wv
            dx = part if dx is None else dx + part
            dws.append((_held(d.t().contiguous()) @ over_rows.t())
                       .to(w.dtype))
        return [*ys, dx.to(x.dtype), *dws]
    if op == "swiglu":
        g, u, dy = s["g"], s["u"], s["dy"].float()
        gf, uf = g.float(), u.float()
        h = gf / (1.0 + torch.exp(-gf)) * uf
        gf, uf = _held(gf), _held(uf)
        sig = 1.0 / (1.0 + torch.exp(-gf))
        dg = dy * uf * sig * (1.0 + gf * (1.0 - sig))
        du = dy * gf * sig
        return [h.to(g.dtype), dg.to(g.dtype), du.to(u.dtype)]
    if op == "rms":
        x, w, dy = s["x"], s["w"], s["dy"].float()
        xf = x.float()
        inv = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + s["eps"])
        y = xf * inv * w
        n = _held(xf) * inv
        a = dy * w
        dx = inv * (a - n * (a * n).mean(-1, keepdim=True))
        dw = (dy.double() * n).sum(0)
        return [y.to(x.dtype), dx.to(x.dtype), dw.to(w.dtype)]
    x = s["x"]
    return _held(x.float()).to(x.dtype)


# ---------------------------------------------------------------- the floor
def work(case):
    op, m, k = case["op"], case["m"], case["k"]
    size = 4 if case["dtype"] == "fp32" else 2
    if op == "serve":
        # the weights are read in the 8 bits that they are kept in
        n = case["n"]
        return {"bytes": size * m * (k + n) + n * k + n * k // 128 ** 2,
                "flops": 2 * m * n * k}
    if op == "train":
        # x, W and dY in; Y, dX and dW out
        n = sum(_widths(case))
        return {"bytes": 2 * size * (m * k + n * k + m * n),
                "flops": 6 * m * n * k}
    # what is held between the passes is written once and read once: 8 bits
    # a value and one byte of scale for 128
    held = m * (2 * k + 2 * -(-k // 128))
    if op == "swiglu":
        return {"bytes": 6 * size * m * k + 2 * held, "flops": 30 * m * k}
    if op == "rms":
        return {"bytes": 4 * size * m * k + held + 8 * k,
                "flops": 20 * m * k}
    return {"bytes": 2 * size * m * k + held, "flops": 4 * m * k}


# --------------------------------------------------------- in 64 bits, apart
def _e4m3(v):
    """Round fp64 magnitudes of at most 448 to e4m3: steps of 2^(e-3) from
    2^-6 up, of 2^-9 below; ties to even."""
    _, e = torch.frexp(v)
    step = _two_to((e - 1).clamp(min=-6) - 3)
    return torch.round(v / step) * step


def _two_to(t):
    return ((t.long() + 1023) << 52).view(torch.float64)


def _value64(a, axis):
    """The 8-bit values of ``a`` in fp64, blocks of 128 along ``axis``."""
    a = a.movedim(axis, 0)
    out = torch.empty(a.shape, dtype=torch.float64, device=a.device)
    for i in range(0, a.shape[0], 128):
        out[i:i + 128] = _block64(a[i:i + 128].double(), (0,))
    return out.movedim(0, axis)


def _weight64(w):
    out = torch.empty(w.shape, dtype=torch.float64, device=w.device)
    for i in range(0, w.shape[0], 128):
        for j in range(0, w.shape[1], 128):
            b = w[i:i + 128, j:j + 128].double()
            out[i:i + 128, j:j + 128] = _block64(b, (0, 1))
    return out


def _block64(b, dims):
    top = b.abs().amax(dims, keepdim=True)
    t = torch.floor(torch.log2(top.clamp(min=1e-300))) - 8
    # the logarithm may be off next to a power of two: the smallest that fits
    t = t.clamp(min=-126)
    t = torch.where((t > -126) & (top <= 448 * _two_to(t - 1)), t - 1, t)
    t = torch.where(top > 448 * _two_to(t), t + 1, t)
    s = _two_to(t)
    return _e4m3(b / s) * s


@torch.no_grad()
def exact(case, seed):
    global own
    before, own = own, False
    try:
        op = case["op"]
        mk = _Make(seed) if op == "serve" else None
        if op == "serve":
            # the weights themselves; ``prepare`` keeps only their values
            dt = _TYPES[case["dtype"]]
            w = mk.normal(case["n"], case["k"], std=0.02, dtype=dt)
            x = mk.activation(case["m"], case["k"], dt)
            return _value64(x, 1) @ _weight64(w).t()
        s = prepare(case, seed)
    finally:
        own = before
    if op == "train":
        held = _value64(s["x"], 1)
        over_rows = _value64(held, 0)
        ys, dws, dx = [], [], 0.0
        for w, dy in zip(s["ws"], s["dys"]):
            wv = _weight64(w)
            ys.append(held @ wv.t())
            dx = dx + _value64(dy, 1) @ wv
            dws.append(_value64(dy, 0).t() @ over_rows)
        return [*ys, dx, *dws]
    if op == "swiglu":
        g, u, dy = (s[n].detach().double() for n in ("g", "u", "dy"))
        h = g * torch.sigmoid(g) * u
        g, u = _value64(g, 1), _value64(u, 1)
        sig = torch.sigmoid(g)
        return [h, dy * u * (sig + g * sig * (1 - sig)), dy * g * sig]
    if op == "rms":
        x, w, dy = (s[n].detach().double() for n in ("x", "w", "dy"))
        k = x.shape[1]
        inv = 1.0 / torch.sqrt((x ** 2).sum(1, keepdim=True) / k + s["eps"])
        y, n = x * inv * w, _value64(x, 1) * inv
        dn = dy * w
        dx = inv * dn - inv * n * ((dn * n).sum(1, keepdim=True) / k)
        return [y, dx, (dy * n).sum(0)]
    return _value64(s["x"], 1)
