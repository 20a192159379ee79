"""The dense layers beside the MoE layer as measurable cases: rows quantized to 8-bit floating point,
the linear layer and the gated feed-forward block on 8-bit weights with a scale per 128 x 128 block,
and the gated feed-forward block in bf16 and fp32 with its gradients.

A block that is trained in bf16 or fp32 and then served in 8 bits stands behind them: a training step
runs the block forward and backward on a batch of thousands of tokens, a server runs it and the
projections around it on one to some thousand rows. Sizes are those of the benchmark's layers (hidden
1024 to 7168, the small layer's 2.75 for a block's width) or plain ones; drawn cases add others, odd
ones among them.

``listed`` gives the fixed cases, ``draw`` more of the same ranges, ``prepare`` what a program has in
hand before the call, ``run`` one call (with ``own`` through the framework's entry points, otherwise
in elementary torch operations), ``work`` the bytes and operations that a call cannot do without,
``exact`` its result in 64 bits.
"""
import math

import torch

own = False

GROUP = 128      # values that share a scale
E4M3_MAX = 448.0
MIN_SCALE = 1e-12


def _quantize(name, rows, width, act="bf16"):
    c = {"op": "quantize", "rows": rows, "in": width, "act": act}
    return dict(c, name=name) if name else c


def _linear(name, rows, inf, outf, bias=False):
    c = {"op": "linear", "rows": rows, "in": inf, "out": outf, "act": "bf16", "bias": bias}
    return dict(c, name=name) if name else c


def _block(name, op, rows, hidden, ffn, act="bf16"):
    c = {"op": op, "rows": rows, "hidden": hidden, "ffn": ffn, "act": act}
    return dict(c, name=name) if name else c


def listed():
    return [
        # the rows of a batch of decoding sequences, before a product: a launch
        _quantize("quantize 64 x 4096", 64, 4096),
        # a prompt's rows: one pass over memory
        _quantize("quantize 16721 x 4096", 16721, 4096),
        # an attention projection, one sequence
        _linear("fp8 linear 1 x 4096 x 4096", 1, 4096, 4096),
        # widths that fill no block
        _linear("fp8 linear 7 x 5000 x 3001", 7, 5000, 3001, bias=True),
        # a prompt, the wide side of a block
        _linear("fp8 linear 8192 x 4096 x 8192", 8192, 4096, 8192),
        # one sequence's step: the block's weights once
        _block("fp8 block 1 x 4096 x 11264", "fp8 block", 1, 4096, 11264),
        # a batch of decoding sequences on a narrow block
        _block("fp8 block 48 x 5120 x 1536", "fp8 block", 48, 5120, 1536),
        # a prompt
        _block("fp8 block 4096 x 4096 x 11264", "fp8 block", 4096, 4096, 11264),
        # the block as it was trained, one sequence's step
        _block("block 1 x 4096 x 11264", "block", 1, 4096, 11264),
        # a training step in fp32 on the small layer
        _block("step 2052 x 1024 x 2816 f32", "step", 2052, 1024, 2816, act="f32"),
        # a training step on a short batch, sizes that fill no tile
        _block("step 333 x 1000 x 2730", "step", 333, 1000, 2730),
        # a training step on a full batch
        _block("step 4096 x 4096 x 11264", "step", 4096, 4096, 11264),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width: mostly a multiple of a block, else any number."""
    w = _log_int(rng, lo, hi)
    return max(lo, w // 128 * 128) if rng.random() < 0.6 else w


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "fp8 block", "fp8 block", "block", "step", "step"])
    act = rng.choice(["bf16", "bf16", "f32"])
    while True:
        rows = _log_int(rng, 1, 16384)
        if op == "quantize":
            c = _quantize(None, rows, _width(rng, 32, 16384), act)
            if c["rows"] * c["in"] * (2 if act == "f32" else 1) <= 16721 * 4096:
                return c
        elif op == "linear":
            c = _linear(None, rows, _width(rng, 32, 16384), _width(rng, 16, 65536), rng.random() < 0.5)
            if work(c)["flops"] <= 2 * 8192 * 4096 * 8192 and c["in"] * c["out"] <= 1 << 28:
                return c
        else:
            c = _block(None, op, rows, _width(rng, 32, 8192), _width(rng, 32, 16384),
                       "bf16" if op == "fp8 block" else act)
            most = 18 * 2052 * 4096 * 5632 if act == "f32" and op != "fp8 block" else 6 * 4096 * 4096 * 11264
            if work(c)["flops"] <= most and c["hidden"] * c["ffn"] <= 1 << 26:
                return c


# ---------------------------------------------------------------- inputs
def _dtype(c):
    return torch.float32 if c["act"] == "f32" else torch.bfloat16


def _rows(g, n, width):
    """Activations: rows of several sizes, a few channels larger than the others."""
    x = torch.randn(n, width, generator=g, device="cuda")
    x *= 0.5 + torch.rand(n, 1, generator=g, device="cuda")
    x[:, 5::61] *= 8.0
    return x


def _codes(g, outf, inf):
    """A weight in 8 bits: codes [out][in] (their bytes) and a scale per 128 x 128 block. About 1 /
    sqrt(in) in size, so that products stay about as large as their inputs."""
    q = torch.randn(outf, inf, generator=g, device="cuda").mul_(100).clamp_(-E4M3_MAX, E4M3_MAX)
    s = 0.75 + 0.5 * torch.rand(-(-outf // GROUP), -(-inf // GROUP), generator=g, device="cuda")
    return q.to(torch.float8_e4m3fn).view(torch.uint8), s * (0.01 / math.sqrt(inf))


def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _dtype(c)
    if c["op"] == "quantize":
        return {"x": _rows(g, c["rows"], c["in"]).to(dt)}
    if c["op"] == "linear":
        r = {"x": _rows(g, c["rows"], c["in"]).to(dt), "w": _codes(g, c["out"], c["in"]), "bias": None}
        if c["bias"]:
            r["bias"] = torch.randn(c["out"], generator=g, device="cuda").to(dt)
        return r
    N, H, F = c["rows"], c["hidden"], c["ffn"]
    r = {"x": _rows(g, N, H).to(dt)}
    for n, o, i in (("gate", F, H), ("up", F, H), ("down", H, F)):
        if c["op"] == "fp8 block":
            r[n] = _codes(g, o, i)
        else:
            r[n] = (torch.randn(o, i, generator=g, device="cuda") / math.sqrt(i)).to(dt)
    if c["op"] == "step":
        r["dy"] = torch.randn(N, H, generator=g, device="cuda").mul_(0.1).to(dt)
    return r


# ---------------------------------------------------------------- what a program has in hand
@torch.no_grad()
def prepare(case, seed):
    st = dict(_inputs(case, seed), case=case)
    if own:
        if case["op"] in ("linear", "fp8 block"):
            from pisceslx_amd import quant
            for n in ("w", "gate", "up", "down"):
                if n in st:
                    st[n] = quant.pack_fp8_linear_codes(*st[n], st[n][0].shape[1])
        elif case["op"] == "step":
            for n in ("x", "gate", "up", "down"):
                st[n].requires_grad_(True)
    return st


# ---------------------------------------------------------------- one call
def run(state):
    return _own(state) if own else _plain(state)


def _own(st):
    from pisceslx_amd import functional as yvf
    c = st["case"]
    if c["op"] == "quantize":
        q = yvf.quantize_fp8_rows(st["x"])
        return {"codes": q.codes[:, :c["in"]], "scales": q.scales}
    if c["op"] == "linear":
        return yvf.fp8_linear(st["x"], st["w"], st["bias"])
    if c["op"] == "fp8 block":
        return yvf.fp8_swiglu(st["x"], st["gate"], st["up"], st["down"])
    y = yvf.swiglu(st["x"], st["gate"], st["up"], st["down"])
    if c["op"] == "block":
        return y
    dx, dg, du, dd = torch.autograd.grad(y, [st["x"], st["gate"], st["up"], st["down"]], st["dy"])
    return {"y": y.detach(), "dx": dx, "dgate": dg, "dup": du, "ddown": dd}


def _plain_quantize(x):
    """Codes [rows][in] as 8-bit floats and scales [groups][rows] of 32-bit rows."""
    n, width = x.shape
    pad = -width % GROUP
    v = torch.cat([x, x.new_zeros(n, pad)], dim=1) if pad else x
    v = v.view(n, -1, GROUP)
    top = v.abs().amax(dim=2)  # divided by a tensor: torch multiplies by a number's reciprocal instead
    s = (top / torch.full_like(top, E4M3_MAX)).clamp(min=MIN_SCALE)
    q = (v / s[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.view(n, -1)[:, :width], s.t().contiguous()


def _spread(s, rows, cols):
    """Block scales as a factor for each value of a [rows][cols] weight."""
    return s.repeat_interleave(GROUP, 0)[:rows].repeat_interleave(GROUP, 1)[:, :cols]


def _plain_product(x, w):
    """32-bit rows x (quantized here) times a weight of codes and block scales, in 32 bits."""
    q, s = _plain_quantize(x)
    a = q.float() * s.t().repeat_interleave(GROUP, 1)[:, :x.shape[1]]
    codes, ws = w
    b = codes.view(torch.float8_e4m3fn).float() * _spread(ws, *codes.shape)
    return a @ b.t()


@torch.no_grad()
def _plain(st):
    c, x = st["case"], st["x"].float()
    dt = _dtype(c)
    if c["op"] == "quantize":
        q, s = _plain_quantize(x)
        return {"codes": q, "scales": s}
    if c["op"] == "linear":
        y = _plain_product(x, st["w"])
        return (y if st["bias"] is None else y + st["bias"].float()).to(dt)
    if c["op"] == "fp8 block":
        g, u = _plain_product(x, st["gate"]), _plain_product(x, st["up"])
        return _plain_product(g / (1.0 + torch.exp(-g)) * u, st["down"]).to(dt)
    wg, wu, wd = st["gate"].float(), st["up"].float(), st["down"].float()
    g, u = x @ wg.t(), x @ wu.t()
    s = 1.0 / (1.0 + torch.exp(-g))
    h = g * s * u
    y = (h @ wd.t()).to(dt)
    if c["op"] == "block":
        return y
    dy = st["dy"].float()
    dh = dy @ wd
    du = dh * g * s
    dg = dh * u * s * (1.0 + g * (1.0 - s))
    return {"y": y, "dx": (dg @ wg + du @ wu).to(dt), "dgate": (dg.t() @ x).to(dt),
            "dup": (du.t() @ x).to(dt), "ddown": (dy.t() @ h).to(dt)}


# ---------------------------------------------------------------- bytes and operations
def work(case):
    c = case
    b, n = (4 if c["act"] == "f32" else 2), c["rows"]
    if c["op"] == "quantize":
        return {"bytes": n * (c["in"] * (b + 1) + 4 * -(-c["in"] // GROUP)), "flops": 3 * n * c["in"]}

    def weight(o, i):
        return o * i + 4 * -(-o // GROUP) * -(-i // GROUP)

    if c["op"] == "linear":
        i, o = c["in"], c["out"]
        return {"bytes": weight(o, i) + b * (n * (i + o) + (o if c["bias"] else 0)), "flops": 2 * n * i * o}
    H, F = c["hidden"], c["ffn"]
    if c["op"] == "fp8 block":
        return {"bytes": 2 * weight(F, H) + weight(H, F) + 2 * n * H * b, "flops": 6 * n * H * F}
    if c["op"] == "block":
        return {"bytes": b * (3 * H * F + 2 * n * H), "flops": 6 * n * H * F}
    # x, dy, weights read; y, dx, gradients written
    return {"bytes": b * (6 * H * F + 4 * n * H), "flops": 18 * n * H * F}


# ---------------------------------------------------------------- 64-bit results
def _e4m3(v):
    """64-bit numbers rounded to the nearest that four exponent and three mantissa bits hold."""
    e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -20))).clamp(min=-6.0)
    step = torch.exp2(e - 3.0)
    return torch.round(v / step).mul_(step).clamp_(-E4M3_MAX, E4M3_MAX)


def _exact_rows(x):
    """(rounded x / s, s) of 64-bit rows: [rows][in] and [groups][rows]; a scale is a 32-bit number, and so
    is the quotient that is rounded to 8 bits (bf16 rows have many quotients halfway between two codes)."""
    v, s = torch.empty_like(x), []
    for k in range(0, x.shape[1], GROUP):
        part = x[:, k:k + GROUP]
        t = torch.clamp(part.abs().max(dim=1).values / E4M3_MAX, min=MIN_SCALE).float().double()
        v[:, k:k + GROUP] = _e4m3((part / t[:, None]).float().double())
        s.append(t)
    return v, torch.stack(s)


def _exact_weight(pair):
    q, s = pair
    w = q.view(torch.float8_e4m3fn).double()
    for k in range(s.shape[1]):
        w[:, k * GROUP:(k + 1) * GROUP] *= s[:, k].double().repeat_interleave(GROUP)[:w.shape[0], None]
    return w


def _exact_product(x, pair):
    v, s = _exact_rows(x)
    for k in range(s.shape[0]):
        v[:, k * GROUP:(k + 1) * GROUP] *= s[k][:, None]
    return torch.nn.functional.linear(v, _exact_weight(pair))


def exact(case, seed):
    c = case
    r = _inputs(c, seed)
    x = r["x"].double()
    if c["op"] == "quantize":
        v, s = _exact_rows(x)
        return {"codes": v, "scales": s}
    if c["op"] == "linear":
        y = _exact_product(x, r["w"])
        return y if r["bias"] is None else y + r["bias"].double()
    if c["op"] == "fp8 block":
        h = torch.nn.functional.silu(_exact_product(x, r["gate"])).mul_(_exact_product(x, r["up"]))
        return _exact_product(h, r["down"])
    wg, wu, wd = (r[n].double() for n in ("gate", "up", "down"))
    leaves = [x, wg, wu, wd]
    if c["op"] == "step":
        for t in leaves:
            t.requires_grad_(True)
    y = torch.nn.functional.linear(
        torch.nn.functional.silu(torch.nn.functional.linear(x, wg)) * torch.nn.functional.linear(x, wu), wd)
    if c["op"] == "block":
        return y
    grads = torch.autograd.grad(y, leaves, r["dy"].double())
    return {"y": y.detach(), "dx": grads[0], "dgate": grads[1], "dup": grads[2], "ddown": grads[3]}
