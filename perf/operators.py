"""The operators of single-token steps as measurable cases: the whole MoE layer for a few tokens,
its experts on a routing computed elsewhere, and the linear layer with 4-bit weights.

A decoder that serves one or a few sequences stands behind them: each step runs dense
projections and MoE layers on one to sixteen rows, and a prompt passes the same projections with
thousands of rows. Layer shapes are those of the benchmark's configurations; drawn cases add other
widths, expert counts and formats.

``listed`` gives the fixed cases, ``draw`` more of the same ranges, ``prepare`` what a program has
in hand before the call, ``run`` one call (with ``own`` through the framework's entry points,
otherwise in elementary torch operations), ``work`` the bytes and operations that a call cannot do
without, ``exact`` its result in 64 bits.
"""
import math

import torch

own = False

# hidden, experts, ffn, top_k, shared experts of the benchmark's layers
SHAPES = {
    "small": (1024, 8, 2816, 2, 1),
    "mid": (4096, 64, 1408, 6, 2),
    "wide": (5120, 128, 1536, 8, 1),
    "huge": (7168, 256, 2048, 8, 0),
}
MAX_TOKENS = 16
MIN_CAPACITY = 4
GROUP = 128  # weights of a row that share a scale (int4)


def _moe(name, op, shape, fmt, tokens, fixed=False):
    H, E, F, k, S = SHAPES[shape] if isinstance(shape, str) else shape
    c = {"op": op, "hidden": H, "experts": E, "ffn": F, "top_k": k, "shared": S, "format": fmt,
         "tokens": tokens, "fixed": fixed}
    return dict(c, name=name) if name else c


def _linear(name, rows, inf, outf, act="bf16", bias=False):
    c = {"op": "linear", "rows": rows, "in": inf, "out": outf, "act": act, "bias": bias}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one sequence on the small full-precision layer: launches and chains, hardly any bytes
        _moe("layer f32 1", "layer", "small", "f32", 1),
        # one sequence on the int8 layer, the plainest decode step there is
        _moe("layer int8 1", "layer", "mid", "int8", 1),
        # a few sequences on the 4-bit layer
        _moe("layer int4 3", "layer", "wide", "int4", 3),
        # eight sequences on the largest layer, fixed-shape routing with a skewed bias
        _moe("layer fp8 8", "layer", "huge", "fp8", 8, fixed=True),
        # the most rows the form takes: most experts are touched, several rows each
        _moe("layer bf16 16", "layer", "mid", "bf16", 16),
        # routing from another router, shared experts and the skip residual as in the layer
        _moe("experts int8 4", "experts", "mid", "int8", 4),
        # an external dispatch over an uneven layer: no shared experts, odd counts
        _moe("experts bf16 13", "experts", (1088, 40, 832, 5, 0), "bf16", 13),
        # an attention projection, one row
        _linear("linear 1 x 4096 x 4096", 1, 4096, 4096),
        # logits of a large vocabulary, one row, an odd count of outputs
        _linear("linear 1 x 4096 x 100003", 1, 4096, 100003),
        # fp32 activations, widths that fill no block
        _linear("linear 7 x 5000 x 3001 f32", 7, 5000, 3001, act="f32", bias=True),
        # a batch of decoding sequences
        _linear("linear 48 x 5120 x 8192", 48, 5120, 8192, bias=True),
        # a prompt
        _linear("linear 2048 x 4096 x 4096", 2048, 4096, 4096),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.4:
        rows = _log_int(rng, 1, 4096)
        act = rng.choice(["bf16", "bf16", "f32"])
        while True:
            inf, outf = _log_int(rng, 64, 16384), _log_int(rng, 64, 131072)
            if rng.random() < 0.5:  # most layers are multiples of a block wide
                inf, outf = max(128, inf // 128 * 128), max(16, outf // 16 * 16)
            # at most the prompt's operations (fp32 rows cost three times as many), the logits' bytes
            ops = rows * inf * outf * (3 if act == "f32" else 1)
            if ops <= 2048 * 4096 * 4096 and inf * outf <= 4096 * 100003:
                return _linear(None, rows, inf, outf, act, rng.random() < 0.5)
    op = rng.choice(["layer", "layer", "experts"])
    fmt = rng.choice(["int8", "int4", "fp8", "bf16", "f32"])
    step = 128 if fmt in ("int4", "fp8") else 64
    while True:
        H = _log_int(rng, 256, 7168) // step * step
        F = max(step, _log_int(rng, 128, 4096) // step * step)
        E = _log_int(rng, 2, 256)
        k = min(E, _log_int(rng, 1, 8 if E < 64 else 12))
        S = rng.choice([0, 0, 1, 1, 2, 3])
        c = _moe(None, op, (H, E, F, k, S), fmt, rng.randint(1, MAX_TOKENS),
                 fixed=op == "layer" and rng.random() < 0.4)
        weights = {"f32": 4, "bf16": 2, "int8": 1, "fp8": 1, "int4": 0.5}[fmt] * 3 * H * F * (E + S)
        # at most the largest listed call's bytes, and a state of a few GB
        if weights <= 4e9 and work(c)["bytes"] <= 1.8e9:
            return c


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _codes(g, fmt, outf, inf):
    """A weight matrix as its format stores it, row-major: (codes, scales or None). Values of
    about 0.02 throughout; int4 holds two codes a byte, the even column in the low half."""
    w = _randn(g, outf, inf)
    if fmt == "f32":
        return w.mul_(0.02), None
    if fmt == "bf16":
        return w.mul_(0.02).to(torch.bfloat16), None
    if fmt == "int8":
        s = 0.02 / 32 * (0.75 + 0.5 * torch.rand(outf, generator=g, device="cuda"))
        return torch.round(w.mul_(32)).clamp_(-127, 127).to(torch.int8), s.to(torch.bfloat16)
    if fmt == "fp8":
        s = 0.02 / 100 * (0.75 + 0.5 * torch.rand(outf // 128, inf // 128, generator=g, device="cuda"))
        return w.mul_(100).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), s
    q = torch.round(w.mul_(2.3)).add_(8).clamp_(0, 15).to(torch.uint8)
    groups = -(-inf // GROUP)
    if inf % GROUP:  # columns past the end hold the code of zero
        q = torch.nn.functional.pad(q, (0, groups * GROUP - inf), value=8)
    s = 0.02 / 2.3 * (0.75 + 0.5 * torch.rand(outf, groups, generator=g, device="cuda"))
    return q[:, 0::2] | (q[:, 1::2] << 4), s.to(torch.bfloat16)


def _expert_codes(c, seed):
    """(gate, up, down) of one expert after the other, routed first, then shared; each a pair."""
    g = _gen(seed + 7919)
    H, F = c["hidden"], c["ffn"]
    for _ in range(c["experts"] + c["shared"]):
        yield tuple(_codes(g, c["format"], o, i) for o, i in ((F, H), (F, H), (H, F)))


def _act_dtype(c):
    return torch.float32 if c.get("act", c.get("format")) == "f32" else torch.bfloat16


def _moe_inputs(c, seed):
    """x, skip and mix of the call, and the router's weights or the routing."""
    g = _gen(seed)
    N, H, E, k = c["tokens"], c["hidden"], c["experts"], c["top_k"]
    dt = _act_dtype(c)
    r = {"skip": _randn(g, N, H).to(dt) if c["shared"] else None,
         "mix": torch.softmax(_randn(g, c["shared"]), 0) if c["shared"] else None}
    if c["op"] == "experts":
        logits = _randn(g, N, E) * 1.3
        top = torch.topk(logits, k, dim=1)
        r.update(x=_randn(g, N, H).to(dt), indices=top.indices.contiguous(),
                 weights=torch.softmax(top.values, dim=1).contiguous())
        return r
    r["gate"] = (_randn(g, E, H) * 0.02).to(dt)
    if c["fixed"]:  # a skewed expert bias: Zipf shares over a shuffled order
        order = torch.randperm(E, generator=g, device="cuda")
        r["bias"] = torch.empty(E, device="cuda")
        r["bias"][order] = -1.2 * torch.log(torch.arange(1, E + 1, device="cuda").float())
    else:
        r["w1"], r["w2"] = _randn(g, 64, H) * 0.02, _randn(g, 1, 64) * 0.02
    # a token with two of its first logits closer than 32-bit sums in any order can tell has no one
    # right list of experts: the batch is made of the others
    x = _randn(g, N + 32, H).to(dt)
    z = x.double() @ r["gate"].double().t()
    if c["fixed"]:
        z = z + r["bias"].double()
    z = torch.sort(z, dim=1, descending=True).values[:, :k + 1]
    x = x[(z[:, :-1] - z[:, 1:]).amin(dim=1) > 2e-5] if z.shape[1] > 1 else x
    r["x"] = x[:N].contiguous()
    return r


def _linear_inputs(c, seed):
    g = _gen(seed)
    dt = _act_dtype(c)
    codes, scales = _codes(g, "int4", c["out"], c["in"])
    return {"x": _randn(g, c["rows"], c["in"]).to(dt), "codes": codes, "scales": scales,
            "bias": _randn(g, c["out"]).to(dt) if c["bias"] else None}


# ---------------------------------------------------------------- what a program has in hand
@torch.no_grad()
def prepare(case, seed):
    c = case
    if c["op"] == "linear":
        r = _linear_inputs(c, seed)
        st = {"case": c, "x": r["x"], "bias": r["bias"]}
        if own:
            from pisceslx_amd import quant
            st["weight"] = quant.pack_linear_codes(r["codes"], r["scales"], c["in"])
        else:
            st.update(codes=r["codes"], scales=r["scales"])
        return st
    st = dict(_moe_inputs(c, seed), case=c)
    n, H, F = c["experts"] + c["shared"], c["hidden"], c["ffn"]
    if not own:
        st["experts"] = None
        for e, parts in enumerate(_expert_codes(c, seed)):
            if st["experts"] is None:
                st["experts"] = [tuple(None if t is None else t.new_empty((n,) + t.shape) for t in m) for m in parts]
            for dst, src in zip(st["experts"], parts):
                for d, s in zip(dst, src):
                    if d is not None:
                        d[e] = s
        return st
    from pisceslx_amd import functional as yvf
    from pisceslx_amd import _lib
    from pisceslx_amd.gate import YvStableMoEGate
    from pisceslx_amd.quant import ExpertPacker, FORMAT_BY_NAME, block_matrix
    fmt = FORMAT_BY_NAME[c["format"]]
    pk = ExpertPacker(fmt, c["experts"], c["shared"], H, F, "cuda").packed
    for e, parts in enumerate(_expert_codes(c, seed)):
        for (q, s), w, ws in zip(parts, (pk.w_gate, pk.w_up, pk.w_down), (pk.s_gate, pk.s_up, pk.s_down)):
            w[e] = block_matrix(q, fmt)
            if s is not None:
                ws[e] = s
    st["experts"] = pk
    act = _lib.ACT_F32 if _act_dtype(c) == torch.float32 else _lib.ACT_BF16
    if c["op"] == "layer":
        gate = YvStableMoEGate(H, c["experts"], top_k=c["top_k"], device="cuda", dtype=_act_dtype(c),
                               min_capacity=MIN_CAPACITY, fixed_shape_mode=c["fixed"],
                               enable_dynamic_capacity=not c["fixed"]).eval()
        gate.gate.weight.copy_(st["gate"])
        if c["fixed"]:
            gate.expert_bias.copy_(st["bias"])
        else:
            gate.complexity_predictor[0].weight.copy_(st["w1"])
            gate.complexity_predictor[0].bias.zero_()
            gate.complexity_predictor[2].weight.copy_(st["w2"])
            gate.complexity_predictor[2].bias.zero_()
        st["gate"], st["act"] = gate, act
    nbytes = yvf.few_workspace_bytes(c["tokens"], act, c["top_k"], pk)
    st["workspace"] = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    return st


# ---------------------------------------------------------------- one call
@torch.no_grad()
def run(state):
    c = state["case"]
    if not own:
        return _plain_linear(state) if c["op"] == "linear" else _plain_moe(state)
    from pisceslx_amd import functional as yvf
    if c["op"] == "linear":
        return yvf.int4_linear(state["x"], state["weight"], state["bias"])
    if c["op"] == "experts":
        out, shared, _ = yvf.experts_few(state["x"], state["weights"], state["indices"], state["experts"],
                                         state["mix"], state["skip"], workspace=state["workspace"])
        return {"out": out} if shared is None else {"out": out, "shared": shared}
    out, shared, routing = yvf.moe_forward_few(state["x"], state["gate"].router_state(state["act"]),
                                               state["experts"], state["mix"], state["skip"],
                                               workspace=state["workspace"])
    res = {"out": out, "weights": routing.weights, "indices": routing.indices}
    if shared is not None:
        res["shared"] = shared
    return res


def _values(fmt, q, s):
    """The numbers that codes [..., out, in] stand for, in 32 bits."""
    if fmt in ("f32", "bf16"):
        return q.float()
    if fmt == "int8":
        return q.float() * s.float()[..., None]
    if fmt == "fp8":
        v = q.view(torch.float8_e4m3fn).float()
        return v * s.repeat_interleave(128, -2).repeat_interleave(128, -1)
    v = torch.stack([q & 15, q >> 4], dim=-1).flatten(-2).float() - 8.0
    return v * s.float().repeat_interleave(GROUP, -1)


def _plain_linear(st):
    c = st["case"]
    x = st["x"].float()
    w = _values("int4", st["codes"], st["scales"])[:, :c["in"]]
    y = x @ w.t()
    if st["bias"] is not None:
        y = y + st["bias"].float()
    return y.to(st["x"].dtype)


def _plain_routing(c, st):
    """Softmax, top-k, softmax of the k, and outside fixed mode the capacity trim; logits in 64
    bits (a near-tie decides which expert runs)."""
    x, N, E, k = st["x"].double(), c["tokens"], c["experts"], c["top_k"]
    z = x @ st["gate"].double().t()
    if c["fixed"]:
        z = z + st["bias"].double()
    p, idx = torch.sort(torch.softmax(z, dim=1), dim=1, descending=True, stable=True)
    p, idx = p[:, :k].contiguous(), idx[:, :k].contiguous()
    w = torch.exp(p - p[:, :1])
    w = w / w.sum(dim=1, keepdim=True)
    if c["fixed"]:
        return w.float(), idx
    hidden = torch.clamp(x @ st["w1"].double().t(), min=0.0)
    score = 1.0 / (1.0 + torch.exp(-(hidden @ st["w2"].double().t())))
    factor = (0.5 + 1.5 * score.mean()).clamp(0.5, 2.0)
    cap = torch.clamp((N * factor / E).floor(), min=MIN_CAPACITY)
    # slots of the same expert that come first: by probability, then by place
    e, q = idx.reshape(-1), p.reshape(-1)
    place = torch.arange(N * k, device=e.device)
    before = (q[None, :] > q[:, None]) | ((q[None, :] == q[:, None]) & (place[None, :] < place[:, None]))
    rank = (before & (e[None, :] == e[:, None])).sum(dim=1)
    w = w * (rank < cap).view(N, k)
    return (w / w.sum(dim=1, keepdim=True).clamp(min=1e-8)).float(), idx


def _plain_moe(st):
    c = st["case"]
    w, idx = (st["weights"], st["indices"]) if c["op"] == "experts" else _plain_routing(c, st)
    E, S, dt = c["experts"], c["shared"], st["x"].dtype
    x = st["x"].float()

    def ffn(sel, rows):
        """Outputs of the selected experts: expert i on rows[i] ([H] or [N, H])."""
        g, u, d = (_values(c["format"], q[sel], None if s is None else s[sel]) for q, s in st["experts"])
        rows = rows.unsqueeze(-1) if rows.dim() == 2 else rows.transpose(1, 2).contiguous()
        a = torch.matmul(g, rows)
        h = a / (1.0 + torch.exp(-a)) * torch.matmul(u, rows)
        return torch.matmul(d, h)

    out = []
    for t in range(c["tokens"]):
        y = ffn(idx[t], x[t].expand(c["top_k"], -1)).squeeze(-1)
        out.append((w[t, :, None] * y).sum(dim=0))
    out = torch.stack(out)
    res = {}
    if S:
        y = ffn(slice(E, E + S), x.expand(S, -1, -1))
        shared = (st["mix"][:, None, None] * y.transpose(1, 2)).sum(dim=0)
        out = out + shared + 0.1 * st["skip"].float()
        res["shared"] = shared.to(dt)
    res["out"] = out.to(dt)
    if c["op"] == "layer":
        res["weights"], res["indices"] = w, idx
        res = {n: res[n] for n in ("out", "weights", "indices", "shared") if n in res}
    return res


# ---------------------------------------------------------------- bytes and operations
def _touched(c):
    """Routed experts that a batch is expected to use: each token takes k of E, by their shares."""
    E, k, N = c["experts"], c["top_k"], c["tokens"]
    if not c["fixed"] or k == E:
        return E * (1.0 - (1.0 - k / E) ** N)
    # a normal logit (of the deviation that the inputs give) plus the bias, above the level that k
    # experts reach on average
    sd = 0.02 * math.sqrt(c["hidden"])
    bias = [-1.2 * math.log(i + 1) for i in range(E)]
    share = lambda level: [0.5 * math.erfc((level - b) / (sd * math.sqrt(2.0))) for b in bias]
    lo, hi = -40.0, 40.0
    for _ in range(60):
        mid = 0.5 * (lo + hi)
        lo, hi = (mid, hi) if sum(share(mid)) > k else (lo, mid)
    return sum(1.0 - (1.0 - q) ** N for q in share(lo))


def work(case):
    c = case
    if c["op"] == "linear":
        n, i, o = c["rows"], c["in"], c["out"]
        b = 4 if c["act"] == "f32" else 2
        return {"bytes": o * -(-i // 2) + 2 * o * -(-i // GROUP) + b * (n * (i + o) + (o if c["bias"] else 0)),
                "flops": 2 * n * i * o}
    N, H, F, E, k, S = (c[n] for n in ("tokens", "hidden", "ffn", "experts", "top_k", "shared"))
    b = 4 if c["format"] == "f32" else 2
    per = 3 * H * F
    expert = {"f32": 4 * per, "bf16": 2 * per, "int8": per + 2 * (2 * F + H),
              "int4": per // 2 + 2 * (per // GROUP), "fp8": per + 4 * (per // 16384)}[c["format"]]
    nbytes = (_touched(c) + S) * expert + 2 * N * H * b + N * k * 12 + (2 * N * H * b if S else 0)
    flops = 6 * H * F * N * (k + S)
    if c["op"] == "layer":
        nbytes += E * H * b
        flops += 2 * N * H * E
        if not c["fixed"]:
            nbytes += 64 * H * 4
            flops += 2 * N * H * 64
    return {"bytes": int(nbytes), "flops": int(flops)}


# ---------------------------------------------------------------- 64-bit results
def _dense64(fmt, pair):
    """A matrix of the inputs in 64 bits, from its definition."""
    q, s = pair
    if s is None:
        return q.double()
    if fmt == "int8":
        return torch.diag(s.double()) @ q.double() if q.shape[0] <= 64 else q.double().mul_(s.double().view(-1, 1))
    if fmt == "fp8":
        o, i = q.shape
        v = q.view(torch.float8_e4m3fn).double().view(o // 128, 128, i // 128, 128)
        return (v * s.double().view(o // 128, 1, i // 128, 1)).view(o, i)
    o = q.shape[0]
    v = torch.empty(o, 2 * q.shape[1], dtype=torch.float64, device=q.device)
    v[:, 0::2] = (q % 16).double() - 8
    v[:, 1::2] = torch.div(q, 16, rounding_mode="floor").double() - 8
    return (v.view(o, -1, GROUP) * s.double().unsqueeze(-1)).view(o, -1)


def _exact_routing(c, r):
    x = r["x"].double().cpu()
    N, E, k = c["tokens"], c["experts"], c["top_k"]
    z = torch.nn.functional.linear(x, r["gate"].double().cpu())
    if c["fixed"]:
        z += r["bias"].double().cpu()
    prob = torch.nn.functional.softmax(z, dim=-1)
    chosen = [sorted(range(E), key=lambda e: (-prob[t, e].item(), e))[:k] for t in range(N)]
    idx = torch.tensor(chosen)
    p = prob.gather(1, idx)
    w = torch.nn.functional.softmax(p, dim=-1)
    if not c["fixed"]:
        s = torch.sigmoid(torch.relu(x @ r["w1"].double().cpu().t()) @ r["w2"].double().cpu().t())
        cap = max(MIN_CAPACITY, int(N * min(2.0, max(0.5, 0.5 + 1.5 * s.mean().item())) / E))
        for e in range(E):
            slots = [(-p[t, j].item(), t, j) for t in range(N) for j in range(k) if chosen[t][j] == e]
            for _, t, j in sorted(slots)[cap:]:
                w[t, j] = 0.0
        w = w / w.sum(dim=1, keepdim=True).clamp(min=1e-8)
    return w.cuda(), idx.cuda()


@torch.no_grad()
def exact(case, seed):
    c = case
    if c["op"] == "linear":
        r = _linear_inputs(c, seed)
        y = torch.empty(c["rows"], c["out"], dtype=torch.float64, device="cuda")
        x = r["x"].double()
        for o in range(0, c["out"], 8192):
            w = _dense64("int4", (r["codes"][o:o + 8192], r["scales"][o:o + 8192]))[:, :c["in"]]
            y[:, o:o + 8192] = x @ w.t()
        return y if r["bias"] is None else y + r["bias"].double()
    r = _moe_inputs(c, seed)
    x = r["x"].double()
    w, idx = (r["weights"].double(), r["indices"]) if c["op"] == "experts" else _exact_routing(c, r)
    out, shared = torch.zeros_like(x), torch.zeros_like(x)
    for e, parts in enumerate(_expert_codes(c, seed)):
        if e < c["experts"]:
            t, j = torch.nonzero(idx == e, as_tuple=True)
            if t.numel() == 0:
                continue
        else:
            t = torch.arange(c["tokens"], device="cuda")
        g, u, d = (_dense64(c["format"], m) for m in parts)
        y = (torch.nn.functional.silu(x[t] @ g.t()) * (x[t] @ u.t())) @ d.t()
        if e < c["experts"]:
            out.index_add_(0, t, w[t, j, None] * y)
        else:
            shared += r["mix"][e - c["experts"]].double() * y
    res = {"out": out}
    if c["shared"]:
        res["out"] = out + shared + 0.1 * r["skip"].double()
        res["shared"] = shared
    if c["op"] == "layer":
        res = {"out": res["out"], "weights": w, "indices": idx, **({"shared": shared} if c["shared"] else {})}
    return res
