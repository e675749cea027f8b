"""The operators of a feed-forward block of experts over packed weights, as cases that can be timed.

Each of T tokens is sent to k of E experts, which makes T k pairs; pair t k + j is token t's j-th choice.

  route  softmax or sigmoid scores of a row of logits, the experts chosen (a bias and groups of experts may take part in
         the choice), their weights, and the pairs sorted by expert: `order` and the `offsets` of every expert in it
  gemm   products of the pairs' rows with their experts' packed matrices (W4 with group scales, with or without zero-points, or
         MXFP4), one packed matrix of E * R rows; "up": rows of x are tokens, the outputs lie in sorted order
         and act(gate) * up is taken of the two halves of an expert's rows; "down": rows of x lie in
         sorted order, the outputs at their pairs
  norm   the weighted sum of a token's k rows joined to the residual stream: a norm behind the block, its gate, the
         residual's scale, and the norm ahead of the next block

`own` chooses the library's entry points; without it `run` computes the same from elementary
torch operations.
"""
import math

import torch

own = False

DEV = "cuda"
F16_MAX, F32_MAX = 65504.0, torch.finfo(torch.float32).max


def listed():
    return [
        # one token of a decode loop
        _case("route_token", "route", T=1, E=128, k=8),
        # a decode step of 61 sequences; logits as the FP16 product of the router gives them
        _case("route_step", "route", T=61, E=64, k=6, renorm=False, f32=False),
        # a prompt: sigmoid scores, a bias that balances the load, four of eight groups kept
        _case("route_groups", "route", T=4099, E=256, k=8, score="sigmoid", bias=True, groups=8, top_groups=4, scale=2.5),
        # several prompts admitted at once, the token list padded as a captured step has it
        _case("route_prompts", "route", T=16384, E=128, k=8, pad=333),
        # one token: eight experts' matrices are read for a row each
        _case("up_token", "gemm", T=1, E=128, k=8, K=2048, width=1024, gs=128),
        # a decode step: most experts have a row or two, 16-bit scales under every 64, zero-points
        _case("up_step", "gemm", T=61, E=64, k=6, K=2048, width=1408, gs=64, zeros=True),
        # the way back of a decode step, MXFP4
        _case("down_step", "gemm", T=32, E=32, k=4, K=2048, width=4096, up=False, mx=True),
        # a prompt through many narrow experts
        _case("up_prompt", "gemm", T=4096, E=64, k=8, K=2048, width=1024, gs=128),
        # a prompt through few wide ones, MXFP4
        _case("down_prompt", "gemm", T=2053, E=8, k=2, K=14336, width=4096, up=False, mx=True),
        # one token's rows joined, no norm behind the block
        _case("norm_token", "norm", T=1, k=8, D=2048, post=False),
        # a prompt: a norm on either side, a gate per channel, the residual stream in FP32
        _case("norm_prompt", "norm", T=4096, k=8, D=2048, gate="channel", f32=True),
        # a block without experts, rows of an odd length, centred norms with biases and a gate per element
        _case("norm_ragged", "norm", T=777, k=1, D=4097, centred=True, gate="element", scale=0.22),
    ]


def _case(name, kind, **more):
    """route: T tokens and `pad` places behind them, E experts, k chosen.  gemm: rows of K, `width` outputs (up: each of a
    gate and an up row).  norm: rows of D, k of them per token."""
    rest = {
        "route": dict(pad=0, score="softmax", bias=False, groups=1, top_groups=1, renorm=True, scale=1.0, f32=True),
        "gemm": dict(up=True, act="silu", mx=False, gs=32, zeros=False),
        "norm": dict(centred=False, post=True, gate="none", scale=1.0, f32=False, shared=False),
    }[kind]
    return {"name": name, "kind": kind, **rest, **more}


# ---- draws ---------------------------------------------------------------------------------


def _log(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def _draw_once(rng):
    kind = rng.choice(["route", "gemm", "gemm", "norm"])
    if kind == "route":
        E = rng.choice([8, 16, 32, 60, 64, 128, 160, 256, 384])
        groups = rng.choice([g for g in (1, 1, 2, 4, 8) if E % g == 0 and E // g >= 4])
        keep = rng.randint(1, groups)
        return _case("", "route", T=_log(rng, 1, 16384), E=E, k=rng.randint(1, min(8, keep * (E // groups))),
                     pad=rng.choice([0, 0, _log(rng, 1, 500)]), score=rng.choice(["softmax", "sigmoid"]),
                     bias=rng.random() < 0.5, groups=groups, top_groups=keep, renorm=rng.random() < 0.7,
                     scale=rng.choice([1.0, 2.5]), f32=rng.random() < 0.6)
    if kind == "gemm":
        E = rng.choice([8, 16, 32, 60, 64, 128])
        up, mx = rng.random() < 0.5, rng.random() < 0.4
        return _case("", "gemm", T=_log(rng, 1, 4096), E=E, k=rng.randint(1, min(8, E)), up=up, mx=mx,
                     gs=32 if mx else rng.choice([32, 64, 128, 128]), zeros=not mx and rng.random() < 0.4,
                     K=64 * _log(rng, 8, 112), width=32 * _log(rng, 8, 128), act=rng.choice(["silu", "gelu"]))
    D = rng.choice([64 * _log(rng, 4, 128), _log(rng, 200, 8192)])
    return _case("", "norm", T=_log(rng, 1, 8192), k=rng.choice([1, 2, 4, 6, 8]), D=D, centred=rng.random() < 0.3,
                 post=rng.random() < 0.6, gate=rng.choice(["none", "channel", "element"]),
                 scale=rng.choice([1.0, 0.22]), f32=rng.random() < 0.5, shared=rng.random() < 0.3)


def _cost(case):
    w = work(case)
    return w["bytes"] / 5e12 + w["flops"] / 5e14


def draw(rng):
    most = {k: max(_cost(c) for c in listed() if c["kind"] == k) for k in ("route", "gemm", "norm")}
    while True:
        case = _draw_once(rng)
        codes = case["E"] * _rows(case) * case["K"] if case["kind"] == "gemm" else 0
        if _cost(case) <= most[case["kind"]] and codes <= 8 * 14336 * 4096:
            del case["name"]
            return case


# ---- inputs --------------------------------------------------------------------------------


def _rows(case):
    """Rows of an expert's matrix."""
    return case["width"] * (2 if case["up"] else 1)


def _randn(gen, *shape):
    return torch.randn(*shape, device=DEV, generator=gen)


def _logits(gen, T, E):
    """Rows near N(0, 1.5) over experts of which some are more popular than others."""
    return 1.5 * _randn(gen, T, E) + 0.7 * _randn(gen, E)


def _codes(gen, rows, K, signed):
    """Packed words of eight 4-bit codes, low first: offset codes as rounding of normal values leaves them, or (signed) E2M1."""
    q = torch.empty(rows, (K + 7) // 8, dtype=torch.int32, device=DEV)
    shift = torch.arange(0, 32, 4, device=DEV, dtype=torch.int32)
    step = max(1, (1 << 26) // K)
    for r in range(0, rows, step):
        n = min(step, rows - r)
        x = _randn(gen, n, q.shape[1], 8).half()
        if signed:
            mag = (x.abs() * 2.5).round().clamp(max=7).int()
            c = mag + 8 * (x < 0).int()
        else:
            c = (x * 2.7 + 8).round().clamp(0, 15).int()
        q[r:r + n] = (c << shift).sum(dim=2, dtype=torch.int32)
    return q


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = {"case": case}
    {"route": _prepare_route, "gemm": _prepare_gemm, "norm": _prepare_norm}[case["kind"]](case, gen, s)
    if own:
        _handles(s)
    return s


def _prepare_route(case, gen, s):
    T, E, P = case["T"] + case["pad"], case["E"], (case["T"] + case["pad"]) * case["k"]
    x = _logits(gen, T, E)
    s["logits"] = x if case["f32"] else x.half()
    s["bias"] = 0.1 * _randn(gen, E) if case["bias"] else None
    s["count"] = torch.tensor([case["T"]], dtype=torch.int32, device=DEV) if case["pad"] else None
    s["experts"] = torch.zeros(T, case["k"], dtype=torch.int32, device=DEV)
    s["weights"] = torch.zeros(T, case["k"], device=DEV)
    s["order"], s["offsets"] = (torch.zeros(n, dtype=torch.int32, device=DEV) for n in (P, E + 1))


def _prepare_gemm(case, gen, s):
    T, E, k, K, R = case["T"], case["E"], case["k"], case["K"], _rows(case)
    chosen = _logits(gen, T, E).topk(k, dim=1).indices.reshape(-1)
    s["order"] = chosen.sort(stable=True).indices.int()
    counts = torch.bincount(chosen, minlength=E)
    s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()
    s["counts"] = counts.tolist()
    s["q"] = _codes(gen, E * R, K, case["mx"])
    G = -(-K // case["gs"])
    if case["mx"]:
        s["scales"] = torch.randint(117, 122, (E * R, G), dtype=torch.uint8, device=DEV, generator=gen)
    else:
        s["scales"] = ((0.5 + torch.rand(E * R, G, device=DEV, generator=gen)) * (0.3 / math.sqrt(K))).half()
    s["zeros"] = _codes(gen, E * R, G, False) if case["zeros"] else None
    x = _randn(gen, T if case["up"] else T * k, K)
    s["x"] = (x if case["up"] else x * _randn(gen, T * k, K) * 0.5).half()
    s["out"] = torch.zeros(T * k, case["width"], dtype=torch.float16, device=DEV)


def _prepare_norm(case, gen, s):
    T, k, D = case["T"], case["k"], case["D"]
    s["y"] = _randn(gen, T, k, D).half()
    w = torch.rand(T, k, device=DEV, generator=gen) + 0.1
    s["weights"] = w / w.sum(dim=1, keepdim=True) if k > 1 else None
    s["shared"] = _randn(gen, T, D).half() if case["shared"] else None
    # a stream in which some channels are far larger than others
    r = 2.0 * _randn(gen, T, D) * (1.0 + 4.0 * (torch.rand(D, device=DEV, generator=gen) < 0.02))
    s["residual"] = r if case["f32"] else r.half()
    for name, there in (("post", case["post"]), ("pre", True)):
        s[name] = (1.0 + 0.2 * _randn(gen, D)).half() if there else None
        s[name + "_bias"] = (0.1 * _randn(gen, D)).half() if there and case["centred"] else None
    s["gate"] = {"none": lambda: None, "channel": lambda: _randn(gen, D).half(),
                 "element": lambda: torch.tanh(_randn(gen, T, D)).half()}[case["gate"]]()
    s["residual_out"] = torch.zeros_like(s["residual"])
    s["h"] = torch.zeros(T, D, dtype=torch.float16, device=DEV)


EPS = 1e-6


def _handles(s):
    """The views and the workspace that a program keeps from call to call."""
    import importlib

    capi = importlib.import_module("w4a16-dequant-gemm_amd").capi
    capi.load()
    case, at = s["case"], {k: v.data_ptr() if isinstance(v, torch.Tensor) else 0 for k, v in s.items()}
    s["capi"], s["at"] = capi, at
    if case["kind"] == "route":
        s["router"] = capi.router(case["E"], case["k"], score=1 if case["score"] == "sigmoid" else 0, groups=case["groups"],
                                  top_groups=case["top_groups"], group_best=2, renorm=case["renorm"], scale=case["scale"],
                                  bias=at["bias"])
        n = capi.route_experts_workspace(s["router"], s["logits"].shape[0])
        s["space"] = torch.zeros(n, dtype=torch.uint8, device=DEV)
    elif case["kind"] == "gemm":
        s["rows"] = capi.expert_rows(case["E"], case["T"], case["k"], at["offsets"], at["order"])
        N, K = s["q"].shape[0], case["K"]
        if case["mx"]:
            s["view"] = capi.PackedMxView(N, K, -(-K // 32), at["q"], at["scales"])
        else:
            s["view"] = capi.PackedView(N, K, case["gs"], -(-K // case["gs"]), 0 if case["zeros"] else 1, at["q"],
                                        at["scales"], at["zeros"])
        s["act"] = (1 if case["act"] == "silu" else 2) if case["up"] else 0
    else:
        s["norm"] = capi.block_norm(case["D"], centred=case["centred"], eps=EPS, residual_scale=case["scale"], post=at["post"],
                                    post_bias=at["post_bias"], gate=at["gate"],
                                    gate_stride=case["D"] if case["gate"] == "element" else 0, pre=at["pre"],
                                    pre_bias=at["pre_bias"])


# ---- the library's calls ---------------------------------------------------------------------


def _own_route(s):
    at, space = s["at"], s["space"]
    s["capi"].route_experts(s["router"], at["logits"], s["case"]["f32"], 0, s["logits"].shape[0], at["count"], at["experts"],
                            at["weights"], at["order"], at["offsets"], space.data_ptr(), space.numel())


def _own_gemm(s):
    case, at = s["case"], s["at"]
    call = s["capi"].gemm_experts_mx if case["mx"] else s["capi"].gemm_experts
    call(s["view"], s["rows"], s["act"], at["x"], case["up"], at["out"], not case["up"])


def _own_norm(s):
    case, at = s["case"], s["at"]
    s["capi"].residual_norm(s["norm"], case["T"], case["k"], at["y"], at["weights"], at["shared"], at["residual"], case["f32"],
                            at["residual_out"], at["h"])


# ---- the same from elementary operations -------------------------------------------------------


def _best(c, n):
    """Indices of the n largest of each row, descending, ties to the lowest index."""
    return c.sort(dim=1, descending=True, stable=True).indices[:, :n]


def _plain_route(s):
    case, l = s["case"], s["logits"]
    T, E = l.shape
    k, g = case["k"], case["groups"]
    x = l.float()
    if case["score"] == "softmax":
        p = (x - x.amax(dim=1, keepdim=True)).exp()
        p = p / p.sum(dim=1, keepdim=True)
    else:
        p = 1.0 / (1.0 + (-x).exp())
    c = l.double()  # the choice: both scores rise with the logit
    if s["bias"] is not None or g > 1:  # next to a border 32 bits would not tell experts apart
        if case["score"] == "softmax":
            c = (c - c.amax(dim=1, keepdim=True)).exp()
            c = c / c.sum(dim=1, keepdim=True)
        else:
            c = 1.0 / (1.0 + (-c).exp())
        if s["bias"] is not None:
            c = c + s["bias"].double()
    if g > 1:
        of = c.view(T, g, E // g).sort(dim=2, descending=True).values[:, :, :2].sum(dim=2)
        keep = torch.zeros(T, g, dtype=torch.bool, device=DEV).scatter_(1, _best(of, case["top_groups"]), True)
        c = torch.where(keep.repeat_interleave(E // g, dim=1), c, -math.inf)
    experts = _best(c, k)
    w = p.gather(1, experts)
    if case["renorm"]:
        w = w / w.sum(dim=1, keepdim=True)
    w = w * case["scale"]
    if s["count"] is not None:
        there = torch.arange(T, device=DEV)[:, None] < s["count"]
        experts, w = torch.where(there, experts, E), torch.where(there, w, 0.0)
    flat = experts.reshape(-1)
    order = flat.sort(stable=True).indices
    offsets = torch.zeros(E + 2, dtype=torch.long, device=DEV)
    offsets[1:].scatter_add_(0, flat, torch.ones_like(flat))
    offsets = offsets.cumsum(0)[:E + 1]
    s["experts"].copy_(torch.where(experts < E, experts, -1))
    s["weights"].copy_(w)
    s["order"].copy_(torch.where(torch.arange(T * k, device=DEV) < offsets[E], order, -1))
    s["offsets"].copy_(offsets)


def _nibbles(q, n):
    """Codes of packed words [rows][words] -> [rows][n]."""
    shift = torch.arange(0, 32, 4, device=DEV, dtype=torch.int32)
    return ((q[:, :, None] >> shift) & 15).view(q.shape[0], -1)[:, :n]


_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _weights(s, r0, r1):
    """Rows r0 .. r1 of the packed matrix, which are halves by definition, in FP32."""
    case, K, gs = s["case"], s["case"]["K"], s["case"]["gs"]
    code = _nibbles(s["q"][r0:r1], K)
    if case["mx"]:
        value = torch.tensor(_E2M1 + [-v for v in _E2M1], device=DEV)[code.long()]
        scale = torch.exp2(s["scales"][r0:r1].float() - 127.0)
    else:
        zero = _nibbles(s["zeros"][r0:r1], s["scales"].shape[1]).repeat_interleave(gs, dim=1)[:, :K] if case["zeros"] else 8
        value = (code - zero).float()
        scale = s["scales"][r0:r1].float()
    return (value * scale.repeat_interleave(gs, dim=1)[:, :K]).half().float()


def _act(name, x):
    if name == "silu":
        return x / (1.0 + (-x).exp())
    return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x * x * x)))


def _plain_gemm(s):
    case, R, I = s["case"], _rows(s["case"]), s["case"]["width"]
    order, at = s["order"].long(), 0
    for e, n in enumerate(s["counts"]):
        if n == 0:
            continue
        pairs = order[at:at + n]
        x = (s["x"][pairs // case["k"]] if case["up"] else s["x"][at:at + n]).float()
        y = torch.matmul(x, _weights(s, e * R, (e + 1) * R).T)
        if case["up"]:
            s["out"][at:at + n] = (_act(case["act"], y[:, :I]) * y[:, I:]).half()
        else:
            s["out"][pairs] = y.half()
        at += n


def _normed(x, weight, bias, centred):
    if centred:
        x = x - x.mean(dim=1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(dim=1, keepdim=True) + EPS) * weight.to(x.dtype)
    return x if bias is None else x + bias.to(x.dtype)


def _plain_norm(s):
    case = s["case"]
    b = s["y"].float()
    b = (b * s["weights"][:, :, None]).sum(dim=1) if s["weights"] is not None else b.sum(dim=1)
    if s["shared"] is not None:
        b = b + s["shared"].float()
    if s["post"] is not None:
        b = _normed(b, s["post"], s["post_bias"], case["centred"])
    if s["gate"] is not None:
        b = b * s["gate"].float()
    r = s["residual"].float() + case["scale"] * b
    s["residual_out"].copy_(r)
    s["h"].copy_(_normed(r, s["pre"], s["pre_bias"], case["centred"]))


def run(state):
    kind = state["case"]["kind"]
    if kind == "route":
        _own_route(state) if own else _plain_route(state)
        return {k: state[k] for k in ("experts", "weights", "order", "offsets")}
    if kind == "gemm":
        _own_gemm(state) if own else _plain_gemm(state)
        return {"out": state["out"]}
    _own_norm(state) if own else _plain_norm(state)
    return {k: state[k] for k in ("residual_out", "h")}


# ---- the definition in 64 bits ------------------------------------------------------------------


def _exact_route(s):
    """The weights; what is chosen is whole numbers."""
    case, l, k, g = s["case"], s["logits"].double(), s["case"]["k"], s["case"]["groups"]
    T, E = l.shape
    p = torch.softmax(l, dim=1) if case["score"] == "softmax" else torch.sigmoid(l)
    c = p + s["bias"].double() if s["bias"] is not None else p.clone()
    if g > 1:
        groups = c.view(T, g, E // g)
        value = groups.topk(2, dim=2).values.sum(dim=2)
        worst = value.topk(case["top_groups"], dim=1).values[:, -1:]
        groups.masked_fill_((value < worst)[:, :, None], -math.inf)
    chosen = c.topk(k, dim=1).indices
    w = p.gather(1, chosen)
    w = (w / w.sum(dim=1, keepdim=True) if case["renorm"] else w) * case["scale"]
    w[case["T"]:] = 0.0
    return {"experts": None, "weights": w, "order": None, "offsets": None}


def _exact_gemm(s):
    """Pair by pair's expert: out = x W^T of the definition's values, decoded digit by digit."""
    case, K, k, I = s["case"], s["case"]["K"], s["case"]["k"], s["case"]["width"]
    E, R, gs = case["E"], _rows(case), case["gs"]
    group = torch.arange(K, device=DEV) // gs
    word, place = torch.arange(K, device=DEV) // 8, 4 * (torch.arange(K, device=DEV) % 8)
    out = torch.zeros(case["T"] * k, I, dtype=torch.float64, device=DEV)
    bounds = s["offsets"].tolist()
    for e in range(E):
        lo, hi = bounds[e], bounds[e + 1]
        if lo == hi:
            continue
        rows = slice(e * R, (e + 1) * R)
        code = torch.bitwise_right_shift(s["q"][rows][:, word].long() & 0xFFFFFFFF, place) & 15
        if case["mx"]:
            mag, exponent = code & 1, (code >> 1) & 3
            value = torch.where(exponent == 0, 0.5 * mag, (1.0 + 0.5 * mag) * torch.exp2(exponent.double() - 1.0))
            value = torch.where(code >= 8, -value, value)
            scale = torch.ldexp(torch.ones((), dtype=torch.float64, device=DEV), s["scales"][rows].int() - 127)
        else:
            z = 8
            if s["zeros"] is not None:
                zw = s["zeros"][rows][:, group // 8].long() & 0xFFFFFFFF
                z = torch.bitwise_right_shift(zw, 4 * (group % 8)) & 15
            value, scale = (code - z).double(), s["scales"][rows].double()
        w = (value * scale[:, group]).half().double()
        pairs = s["order"][lo:hi].long()
        x = s["x"][torch.div(pairs, k, rounding_mode="floor")] if case["up"] else s["x"][lo:hi]
        y = x.double() @ w.T.contiguous()
        if not case["up"]:
            out[pairs] = y
            continue
        gate, up = y[:, :I], y[:, I:]
        if case["act"] == "silu":
            gate = gate * torch.sigmoid(gate)
        else:
            gate = torch.nn.functional.gelu(gate, approximate="tanh")
        out[lo:hi] = gate * up
    return {"out": out}


def _exact_norm(s):
    case = s["case"]

    def norm(x, name):
        rest = dict(weight=s[name].double(), eps=EPS)
        if case["centred"]:
            return torch.nn.functional.layer_norm(x, (case["D"],), bias=s[name + "_bias"].double(), **rest)
        return torch.nn.functional.rms_norm(x, (case["D"],), **rest)

    b = torch.zeros(case["T"], case["D"], dtype=torch.float64, device=DEV)
    for j in range(case["k"]):
        b += s["y"][:, j].double() * (1.0 if s["weights"] is None else s["weights"][:, j, None].double())
    if s["shared"] is not None:
        b += s["shared"].double()
    if s["post"] is not None:
        b = norm(b, "post")
    if s["gate"] is not None:
        b = s["gate"].double() * b
    r = s["residual"].double() + case["scale"] * b
    return {"residual_out": r, "h": norm(r, "pre")}


def exact(case, seed):
    if case["kind"] == "gemm" and work(case)["flops"] > 1e12:
        return None
    s = prepare(case, seed)
    return {"route": _exact_route, "gemm": _exact_gemm, "norm": _exact_norm}[case["kind"]](s)


# ---- what a pass cannot do without ----------------------------------------------------------------


def work(case):
    T, k = case["T"], case["k"]
    if case["kind"] == "route":
        T += case["pad"]
        # logits in; an expert, a weight and a place in the order per pair; offsets
        return {"bytes": case["T"] * case["E"] * (4 if case["f32"] else 2) + 12 * T * k + 4 * (case["E"] + 1),
                "flops": 10 * case["T"] * case["E"]}
    if case["kind"] == "gemm":
        E, K, R, P = case["E"], case["K"], _rows(case), T * k
        # the matrices of the experts that tokens are sent to, as many as evenly spread choices reach
        hit = E * (1.0 - (1.0 - k / E) ** T)
        per = K / 2 + (K / 32 if case["mx"] else -(-K // case["gs"]) * (2.5 if case["zeros"] else 2))
        x = T if case["up"] else P
        return {"bytes": int(hit * R * per + 2 * x * K + 2 * P * case["width"] + 4 * (P + E + 1)), "flops": 2 * P * R * K}
    D, r = case["D"], 4 if case["f32"] else 2
    vectors = 2 * D * ((1 + case["centred"]) * (1 + case["post"]) + (case["gate"] == "channel"))
    per = 2 * k * D + 2 * r * D + 2 * D + 2 * D * (case["gate"] == "element") + 2 * D * case["shared"] + 4 * k * (k > 1)
    return {"bytes": T * per + vectors, "flops": T * D * (2 * k + 12)}
