"""Timed cases of the routing and block-scaled fp8 operators.

Three operators, in their plain form (``own`` false: elementary torch
operations in 32 bits) and as a program calls the framework's kernels:

* ``route``: experts chosen from router logits, and the gradient;
* ``linear``: a projection in e4m3 with one scale per 128 values of an
  activation row and per 128 x 128 block of the weights, and its gradients;
* ``experts``: routing, then the routed experts' FFNs with such weights.

Quantisation is the same on both sides, step by step in fp32: with
``a = max(amax, 2^-100)`` of a block, ``scale = a / 448`` and
``q = e4m3(x * (448 / a))``.  (``448.0 / a`` of a tensor would be a reciprocal
and a product, two roundings; ``full_like(a, 448) / a`` is the one division.)
"""
import torch

own = False

BLOCK = 128
TINY = 2.0 ** -100


# ---------------------------------------------------------------- cases
def _route(name, n, e, k, score="softmax", dtype="float32", bias=False, groups=1, topk_groups=1,
           group_score="top2", renorm=True, scale=1.0, backward=False):
    c = dict(op="route", n=n, e=e, k=k, score=score, dtype=dtype, bias=bias, groups=groups, topk_groups=topk_groups,
             group_score=group_score, renorm=renorm, scale=scale, backward=backward)
    return c if name is None else dict(c, name=name)


def _linear(name, m, k, n, train=False):
    c = dict(op="linear", m=m, k=k, n=n, train=train)
    return c if name is None else dict(c, name=name)


def _experts(name, n, e, k, h, u, act="swiglu", score="softmax", groups=1, topk_groups=1):
    c = dict(op="experts", n=n, e=e, k=k, h=h, u=u, act=act, score=score, groups=groups, topk_groups=topk_groups)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # one decode step's routing: 64 requests, 128 experts
        _route("route_decode", 64, 128, 8),
        # a prefill with an odd token count and an expert count that is no multiple of 32
        _route("route_ragged", 8191, 60, 3, dtype="bfloat16", renorm=False),
        # a large prefill batch with balanced sigmoid routing limited to 4 of 8 groups
        _route("route_groups", 65536, 256, 8, score="sigmoid", bias=True, groups=8, topk_groups=4, scale=2.5),
        # a training step of the router: forward and gradient
        _route("route_train", 16384, 128, 8, dtype="bfloat16", backward=True),
        # a projection for one new token
        _linear("linear_token", 1, 2048, 4096),
        # a decode batch into an output width that ends inside a block
        _linear("linear_decode", 67, 2048, 1000),
        # a prefill chunk whose sizes all end inside a block
        _linear("linear_ragged", 4095, 1360, 2056),
        # a long prefill through a wide projection
        _linear("linear_prefill", 16384, 4096, 8192),
        # one training step of a projection: forward, input gradient, weight gradient
        _linear("linear_train", 8192, 2048, 4096, train=True),
        # the experts of a handful of tokens (GELU FFN)
        _experts("experts_few", 3, 64, 4, 2048, 1024, act="gelu"),
        # a decode batch over 128 experts
        _experts("experts_decode", 256, 128, 8, 2048, 768),
        # a prefill over 64 experts with grouped sigmoid routing
        _experts("experts_prefill", 4096, 64, 4, 2048, 1024, score="sigmoid", groups=8, topk_groups=4),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["route", "linear", "experts"])
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        e = groups * _log_int(rng, 8, 256) if groups == 1 else groups * _log_int(rng, 4, 32)
        k = rng.randint(1, min(8, e))
        topk_groups = rng.randint(1, groups)
        while topk_groups * (e // groups) < k:
            topk_groups += 1
        return _route(None, _log_int(rng, 1, 65536), e, k, score=rng.choice(["softmax", "sigmoid"]),
                      dtype=rng.choice(["float32", "bfloat16"]), bias=rng.random() < 0.5, groups=groups,
                      topk_groups=topk_groups, group_score=rng.choice(["top2", "max"]), renorm=rng.random() < 0.7,
                      scale=rng.choice([1.0, 2.5]), backward=rng.random() < 0.3)
    if op == "linear":
        return _linear(None, _log_int(rng, 1, 8192), _log_int(rng, 64, 4096), _log_int(rng, 64, 8192),
                       train=rng.random() < 0.3)
    groups = rng.choice([1, 4])
    e = groups * rng.randint(2, 24)
    k = rng.randint(1, min(8, e))
    topk_groups = rng.randint(1, groups)
    while topk_groups * (e // groups) < k:
        topk_groups += 1
    return _experts(None, _log_int(rng, 1, 3000), e, k, _log_int(rng, 128, 2048), _log_int(rng, 128, 1024),
                    act=rng.choice(["swiglu", "gelu"]), score=rng.choice(["softmax", "sigmoid"]), groups=groups,
                    topk_groups=topk_groups)


# ---------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)


def _quantize(x, block_rows):
    """(q as e4m3, scale): [.., R, C] -> q [.., R, C], scale [.., R / block_rows, C / 128], in plain torch steps."""
    *lead, r, c = x.shape
    rb, cb = -(-r // block_rows), -(-c // BLOCK)
    xp = torch.nn.functional.pad(x.float(), (0, cb * BLOCK - c, 0, rb * block_rows - r))
    xb = xp.view(*lead, rb, block_rows, cb, BLOCK)
    a = xb.abs().amax(dim=(-3, -1), keepdim=True).clamp_min(TINY)
    q = (xb * (torch.full_like(a, 448.0) / a)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(*lead, rb * block_rows, cb * BLOCK)
    return q[..., :r, :c], (a / 448.0).view(*lead, rb, cb)


def _dequantize(q, scale, block_rows, dtype=torch.float32):
    r, c = q.shape[-2:]
    s = scale.to(dtype).repeat_interleave(block_rows, -2)[..., :r, :].repeat_interleave(BLOCK, -1)[..., :c]
    return q.to(torch.float32).to(dtype) * s


def _weights(g, *shape):
    """Quantised weights as a checkpoint holds them: rows start on 16-byte boundaries."""
    w = _randn(g, *shape, std=shape[-1] ** -0.5)
    q, s = _quantize(w, BLOCK)
    c = shape[-1]
    store = torch.zeros(*shape[:-1], -(-c // 16) * 16, dtype=torch.uint8, device="cuda")
    store[..., :c] = q.view(torch.uint8) if q.is_contiguous() else q.contiguous().view(torch.uint8)
    return store.view(torch.float8_e4m3fn)[..., :c], s.contiguous()


def _logits(g, n, e, dtype):
    # projections of normalised hidden rows, with some experts liked by every token
    return (_randn(g, n, e) + 0.5 * _randn(g, 1, e)).to(dtype)


def _bias(g, e):
    # a balance bias after many small steps
    return (torch.randint(-100, 101, (e,), generator=g, device="cuda") * 1e-3).float()


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    if case["op"] == "route":
        st["logits"] = _logits(g, case["n"], case["e"], getattr(torch, case["dtype"]))
        st["bias"] = _bias(g, case["e"]) if case["bias"] else None
        if case["backward"]:
            st["grad"] = _randn(g, case["n"], case["k"])
            st["logits"].requires_grad_(own)
    elif case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        st["x"] = _randn(g, m, k, dtype=torch.bfloat16)
        if case["train"]:
            st["w"] = _randn(g, n, k, dtype=torch.bfloat16, std=k ** -0.5).requires_grad_(own)
            st["x"].requires_grad_(own)
            st["dy"] = _randn(g, m, n, dtype=torch.bfloat16, std=0.01)
        else:
            st["wq"], st["ws"] = _weights(g, n, k)
            if own:
                from spider_web_moe_b200.fp8_blocks import Fp8BlockTensor

                st["weight"] = Fp8BlockTensor(st["wq"], st["ws"], BLOCK)
    else:
        e, h, u = case["e"], case["h"], case["u"]
        st["logits"] = _logits(g, case["n"], e, torch.float32)
        st["bias"] = _bias(g, e) if case["score"] == "sigmoid" else None
        st["x"] = _randn(g, case["n"], h, dtype=torch.bfloat16)
        names = ["up", "down"] + (["gate"] if case["act"] == "swiglu" else [])
        for s in names:
            rows, cols = (h, u) if s == "down" else (u, h)
            st["q_" + s], st["s_" + s] = _weights(g, e, rows, cols)
            st["b_" + s] = _randn(g, e, rows, std=0.02)
        if own:
            from spider_web_moe_b200.fp8_blocks import Fp8BlockExperts, Fp8BlockTensor

            t = {s: Fp8BlockTensor(st["q_" + s], st["s_" + s], BLOCK) for s in names}
            st["experts"] = Fp8BlockExperts(t["up"], st["b_up"], t["down"], st["b_down"], t.get("gate"),
                                            st.get("b_gate"))
    return st


# ---------------------------------------------------------------- the framework's calls
def _route_args(case):
    if case["op"] == "route":
        return dict(score=case["score"], num_groups=case["groups"], topk_groups=case["topk_groups"],
                    group_score=case["group_score"], renormalize=case["renorm"], scale=case["scale"])
    return dict(score=case["score"], num_groups=case["groups"], topk_groups=case["topk_groups"])


def _run_own(st):
    case = st["case"]
    if case["op"] == "route":
        from spider_web_moe_b200.routing import route_experts

        idx, w = route_experts(st["logits"], case["k"], bias=st["bias"], **_route_args(case))
        if not case["backward"]:
            return idx, w
        (grad,) = torch.autograd.grad(w, st["logits"], st["grad"])
        return idx, w.detach(), grad
    if case["op"] == "linear":
        from spider_web_moe_b200.fp8_blocks import fp8_block_linear

        if not case["train"]:
            return fp8_block_linear(st["x"], st["weight"])
        y = fp8_block_linear(st["x"], st["w"])
        dx, dw = torch.autograd.grad(y, (st["x"], st["w"]), st["dy"])
        return y.detach(), dx, dw
    from spider_web_moe_b200.fp8_blocks import fp8_expert_delta
    from spider_web_moe_b200.routing import route_experts

    idx, w = route_experts(st["logits"], case["k"], bias=st["bias"], **_route_args(case))
    return idx, w, fp8_expert_delta(st["x"], idx, w, st["experts"])


# ---------------------------------------------------------------- plain forms
def _scores(logits, score):
    return torch.softmax(logits, -1) if score == "softmax" else 1.0 / (1.0 + torch.exp(-logits))


def _plain_route(logits, k, bias, score, num_groups, topk_groups, group_score="top2", renormalize=True, scale=1.0):
    # choices in 64 bits: two of them can lie closer than 32 bits resolve
    c = _scores(logits.double(), score)
    if bias is not None:
        c = c + bias.double()
    n, e = c.shape
    if num_groups > 1:
        per = c.view(n, num_groups, e // num_groups)
        srt = per.sort(dim=-1, descending=True).values
        gs = srt[..., : 2 if group_score == "top2" else 1].sum(-1)
        keep = gs.sort(dim=-1, descending=True, stable=True).indices[:, :topk_groups]
        dropped = torch.ones(n, num_groups, dtype=torch.bool, device=c.device).scatter_(1, keep, False)
        c = per.masked_fill(dropped.unsqueeze(-1), float("-inf")).view(n, e)
    idx = c.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    s = _scores(logits.float(), score)
    w = s.gather(1, idx)
    if renormalize:
        w = w / w.sum(-1, keepdim=True).clamp_min(1e-9)
    return idx.int(), w * scale


def _plain_route_grad(logits, idx, g, score, renormalize, scale):
    s = _scores(logits.float(), score)
    idx = idx.long()
    ss = s.gather(1, idx)
    if renormalize:
        d = ss.sum(-1, keepdim=True).clamp_min(1e-9)
        ds = scale * (g - (g * ss).sum(-1, keepdim=True) / d) / d
    else:
        ds = scale * g
    full = torch.zeros_like(s).scatter_(1, idx, ds)
    if score == "softmax":
        dl = s * (full - (full * s).sum(-1, keepdim=True))
    else:
        dl = full * s * (1.0 - s)
    return dl.to(logits.dtype)


def _plain_act(a, gate):
    if gate is not None:
        return gate / (1.0 + torch.exp(-gate)) * a
    return 0.5 * a * (1.0 + torch.erf(a * 0.7071067811865476))


def _rows(x):
    return _dequantize(*_quantize(x, 1), 1)


def _plain_experts(st, idx, w, dtype=torch.float32):
    """delta in `dtype` arithmetic; quantised values are formed in fp32 as the definition says."""
    case = st["case"]
    n, k, e = case["n"], case["k"], case["e"]
    x = _rows(st["x"]).to(dtype)
    flat = idx.reshape(-1).long()
    order = flat.sort(stable=True).indices
    ends = torch.bincount(flat, minlength=e).cumsum(0).tolist()
    y = torch.empty(n * k, case["h"], dtype=dtype, device="cuda")
    lo = 0
    for i, hi in enumerate(ends):
        if hi > lo:
            rows = order[lo:hi]
            deq = lambda s: _dequantize(st["q_" + s][i], st["s_" + s][i], BLOCK, dtype)  # noqa: E731
            xi = x[rows // k]
            up = xi @ deq("up").t() + st["b_up"][i].to(dtype)
            gate = xi @ deq("gate").t() + st["b_gate"][i].to(dtype) if case["act"] == "swiglu" else None
            a = _rows(_plain_act(up, gate)).to(dtype)
            y[rows] = a @ deq("down").t() + st["b_down"][i].to(dtype)
        lo = hi
    return (y.view(n, k, -1) * w.to(dtype).unsqueeze(-1)).sum(1)


def _run_plain(st):
    case = st["case"]
    if case["op"] == "route":
        idx, w = _plain_route(st["logits"], case["k"], st["bias"], **_route_args(case))
        if not case["backward"]:
            return idx, w
        return idx, w, _plain_route_grad(st["logits"], idx, st["grad"], case["score"], case["renorm"], case["scale"])
    if case["op"] == "linear":
        x = _rows(st["x"])
        if not case["train"]:
            return (x @ _dequantize(st["wq"], st["ws"], BLOCK).t()).bfloat16()
        w = _dequantize(*_quantize(st["w"], BLOCK), BLOCK)
        dw = _rows(st["dy"].t()) @ _rows(st["x"].t()).t()
        return (x @ w.t()).bfloat16(), (_rows(st["dy"]) @ w).bfloat16(), dw.bfloat16()
    idx, w = _plain_route(st["logits"], case["k"], st["bias"], **_route_args(case))
    return idx, w, _plain_experts(st, idx, w).bfloat16()


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "route":
        n, e, k = case["n"], case["e"], case["k"]
        item = 2 if case["dtype"] == "bfloat16" else 4
        nbytes = n * e * item + n * k * 8
        flops = 4 * n * e
        if case["backward"]:
            nbytes += n * k * 4 + n * e * item
            flops += 4 * n * e
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        if case["train"]:
            return {"bytes": 2 * (2 * m * k + 2 * n * k + 2 * m * n), "flops": 6 * m * n * k}
        return {"bytes": 2 * m * k + n * k + 2 * m * n, "flops": 2 * m * n * k}
    n, e, k, h, u = (case[s] for s in ("n", "e", "k", "h", "u"))
    mats = 3 if case["act"] == "swiglu" else 2
    touched = e * (1.0 - (1.0 - k / e) ** n)  # experts that some token chose, for even routing
    return {"bytes": int(touched * mats * h * u + n * h * 4 + n * e * 4 + n * k * 8), "flops": 2 * n * k * mats * h * u}


# ---------------------------------------------------------------- 64-bit values
def _exact_scores(logits, score):
    x = logits.double()
    if score == "sigmoid":
        return torch.sigmoid(x)
    z = torch.exp(x - x.amax(-1, keepdim=True))
    return z / z.sum(-1, keepdim=True)


def _exact_route(logits, k, bias, score, num_groups, topk_groups, group_score="top2", renormalize=True, scale=1.0):
    s = _exact_scores(logits, score)
    c = s if bias is None else s + bias.double()
    n, e = c.shape
    if num_groups > 1:
        per = c.reshape(n, num_groups, -1)
        take = min(2 if group_score == "top2" else 1, per.shape[-1])
        gs = per.topk(take, dim=-1).values.sum(-1)
        # rank of a group: how many groups come before it
        a, b = gs.unsqueeze(2), gs.unsqueeze(1)
        ahead = (b > a) | ((b == a) & torch.ones(num_groups, num_groups, device=c.device).tril(-1).bool())
        keep = ahead.sum(-1) < topk_groups
        c = torch.where(keep.unsqueeze(-1), per, torch.full_like(per, float("-inf"))).reshape(n, e)
    picked = []
    c = c.clone()
    for _ in range(k):
        best = c.amax(-1, keepdim=True)
        i = (c == best).to(torch.int8).argmax(-1, keepdim=True)  # lowest index of the largest
        picked.append(i)
        c.scatter_(1, i, float("-inf"))
    idx = torch.cat(picked, 1)
    w = s.gather(1, idx)
    if renormalize:
        w = w / w.sum(-1, keepdim=True).clamp_min(1e-9)
    return idx.int(), w * scale


def _exact_route_grad(logits, idx, g, score, renormalize, scale):
    with torch.enable_grad():
        x = logits.detach().double().requires_grad_(True)
        s = _exact_scores(x, score).gather(1, idx.long())
        if renormalize:
            s = s / s.sum(-1, keepdim=True).clamp_min(1e-9)
        (out,) = torch.autograd.grad(s * scale, x, g.double())
    return out


def _exact_rows(x):
    """Values of 1 x 128 blocks after quantisation, in 64 bits."""
    r, c = x.shape
    out = torch.empty(r, c, dtype=torch.float64, device=x.device)
    for c0 in range(0, c, BLOCK):
        b = x[:, c0:c0 + BLOCK].float()
        a = b.abs().max(dim=1, keepdim=True).values.clamp_min(TINY)
        q = (b * (torch.full_like(a, 448.0) / a)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
        out[:, c0:c0 + BLOCK] = q.double() * (a / 448.0).double()
    return out


def _exact_matrix(q, s):
    r, c = q.shape
    i = torch.arange(r, device=q.device) // BLOCK
    j = torch.arange(c, device=q.device) // BLOCK
    return q.to(torch.float32).double() * s.double()[i][:, j]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "route":
        logits = st["logits"].detach()
        idx, w = _exact_route(logits, case["k"], st["bias"], **_route_args(case))
        if not case["backward"]:
            return idx, w
        return idx, w, _exact_route_grad(logits, idx, st["grad"], case["score"], case["renorm"], case["scale"])
    if case["op"] == "linear":
        x = st["x"].detach()
        if not case["train"]:
            return _exact_rows(x) @ _exact_matrix(st["wq"], st["ws"]).t()
        w = _exact_matrix(*_quantize(st["w"].detach(), BLOCK))
        xr, dr = _exact_rows(x), _exact_rows(st["dy"])
        return xr @ w.t(), dr @ w, _exact_rows(st["dy"].t()) @ _exact_rows(x.t()).t()
    idx, w = _exact_route(st["logits"], case["k"], st["bias"], **_route_args(case))
    x = _exact_rows(st["x"])
    out = torch.zeros(case["n"], case["h"], dtype=torch.float64, device="cuda")
    for i in range(case["e"]):
        tok, slot = (idx == i).nonzero(as_tuple=True)
        if tok.numel() == 0:
            continue
        up = x[tok] @ _exact_matrix(st["q_up"][i], st["s_up"][i]).t() + st["b_up"][i].double()
        if case["act"] == "swiglu":
            gate = x[tok] @ _exact_matrix(st["q_gate"][i], st["s_gate"][i]).t() + st["b_gate"][i].double()
            up = gate * torch.sigmoid(gate) * up
        else:
            up = up * (torch.special.ndtr(up))
        y = _exact_rows(up) @ _exact_matrix(st["q_down"][i], st["s_down"][i]).t() + st["b_down"][i].double()
        out.index_add_(0, tok, y * w[tok, slot].unsqueeze(1))
    return idx, w, out
