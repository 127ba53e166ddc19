"""Performance cases of the layer's trainable front and of its weighted form.

Three operators, each in the calls that a user makes of it:

  norm     LayerNorm / RMSNorm of token rows and its backward pass, the parameters' gradients
           reduced over all tokens
  route    token-choice routing: softmax or sigmoid scores of the router's logits, a balance bias
           and expert groups in the choice, the k best, their weights; and its backward pass
  experts  the experts' products weighted by a routing: out = last_bias (+ x) + sum_j w_j FFN_{e_j}(x)

Where ``own`` is false the operators are computed in their plain form from elementary torch
operations in 32 bits (64 where experts are compared by sums of scores), rounded once at the end.
"""
from __future__ import annotations

import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp32": torch.float32}

# layer shapes: hidden width, expert width, experts, activation, gated (the benchmark's models, a
# MoE-fied attention projection, and one that no vector width divides)
SHAPES = {
    "vit": dict(d=768, H=128, E=24, act="relu", glu=False),
    "bert": dict(d=768, H=32, E=96, act="relu", glu=False),
    "geglu": dict(d=2048, H=128, E=128, act="gelu", glu=True),
    "proj": dict(d=768, H=32, E=12, act="gelu", glu=False),
    "odd": dict(d=130, H=20, E=7, act="gelu", glu=False),
}


def _norm(name, n, d, dtype="bf16", params="same", kind="layer", call="train", strided=False):
    c = dict(op="norm", n=n, d=d, dtype=dtype, params=params, kind=kind, call=call, strided=strided)
    return dict(c, name=name) if name else c


def _route(name, n, E, k, dtype="bf16", scores="softmax", renormalise=True, bias=False, groups=1,
           top_groups=1, scale=1.0, call="forward"):
    c = dict(op="route", n=n, E=E, k=k, dtype=dtype, scores=scores, renormalise=renormalise,
             bias=bias, groups=groups, top_groups=top_groups, scale=scale, call=call)
    return dict(c, name=name) if name else c


def _experts(name, shape, n, k, dtype="bf16", residual=False):
    c = dict(op="experts", shape=shape, n=n, k=k, dtype=dtype, residual=residual)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one generation step of 37 sequences: the normalisation in front of a gated layer, latency
        _norm("norm_decode_37", 37, 2048, kind="rms", call="forward"),
        # finetuning the ViT on the headline batch: bf16 activations, parameters kept in fp32
        _norm("norm_vit_train", 50432, 768, params="fp32"),
        # the backward pass alone of the gated layer's norm, 32768 tokens
        _norm("norm_rms_backward", 32768, 2048, kind="rms", call="backward"),
        # fp32 rows of an odd width, cut out of a wider tensor
        _norm("norm_odd_fp32_train", 4099, 1023, dtype="fp32", strided=True),
        # one token of one sequence: latency
        _route("route_token", 1, 128, 8),
        # prefill of 64 x 2048 tokens over the gated layer's 128 experts
        _route("route_prefill_128k", 131072, 128, 8),
        # sigmoid scores with a balance bias, four of eight groups of experts, fp32 logits
        _route("route_groups_16k", 16384, 256, 8, dtype="fp32", scores="sigmoid", bias=True,
               groups=8, top_groups=4, scale=2.5),
        # router training over BERT's 96 experts: weights as they are, and their gradient
        _route("route_train_64k", 65536, 96, 4, dtype="fp32", renormalise=False, call="train"),
        # one token of one sequence through the gated layer: latency
        _experts("experts_token", "geglu", 1, 8),
        # a generation step of 37 sequences
        _experts("experts_decode_37", "geglu", 37, 8),
        # the fp32 layer on 8 images
        _experts("experts_vit_fp32_8", "vit", 1576, 4, dtype="fp32"),
        # the headline batch with four weighted experts per token and the residual inside
        _experts("experts_vit_256", "vit", 50432, 4, residual=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "route", "experts"])
    if op == "norm":
        d = rng.choice([768, 1024, 2048, _log(rng, 16, 8192)])
        return _norm("", _log(rng, 1, min(131072, (1 << 26) // d)), d, dtype=rng.choice(["bf16", "bf16", "fp32"]),
                     params=rng.choice(["same", "fp32"]), kind=rng.choice(["layer", "rms"]),
                     call=rng.choice(["forward", "backward", "train"]), strided=rng.random() < 0.25)
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        E = rng.choice([24, 96, 128, 256]) if groups > 1 else rng.choice([24, 96, 128, _log(rng, 2, 512)])
        top = rng.randint(1, groups)
        renormalise = rng.random() < 0.6        # (a single renormalised weight is the scale itself)
        return _route("", _log(rng, 1, 131072 * 128 // max(E, 128)), E,
                      rng.randint(2 if renormalise else 1, min(16, E // groups * top)),
                      dtype=rng.choice(["bf16", "fp32"]),
                      scores=rng.choice(["softmax", "sigmoid"]), renormalise=renormalise,
                      bias=rng.random() < 0.5, groups=groups, top_groups=top,
                      scale=rng.choice([1.0, 2.5]), call=rng.choice(["forward", "train"]))
    shape = rng.choice(["vit", "bert", "geglu", "geglu", "proj", "odd"])
    s = SHAPES[shape]
    dtype = "fp32" if shape != "geglu" and rng.random() < 0.3 else "bf16"
    k = rng.randint(1, min(8, s["E"]))
    most = (1 if dtype == "bf16" and shape != "odd" else 0.1) * 50432 * 4 * 768 * 128 * 2
    n = _log(rng, 1, int(min(50432, most / (k * s["d"] * s["H"] * (3 if s["glu"] else 2)))))
    return _experts("", shape, n, k, dtype=dtype, residual=rng.random() < 0.5)


class State:
    pass


def _prepare_norm(c, st, rn):
    n, d, dt = c["n"], c["d"], DT[c["dtype"]]
    pt = dt if c["params"] == "same" else torch.float32
    st.eps, st.offset = (1e-6, 1.0) if c["kind"] == "rms" else (1e-5, 0.0)
    wide = torch.empty(n, d + 9 if c["strided"] else d, dtype=dt, device="cuda")
    st.x = wide[:, :d]
    # channels of different sizes, rows off centre, as a residual stream has them
    st.x.copy_(rn(n, d) * (0.5 + rn(d).abs()) + 0.3 * rn(n, 1))
    st.w = ((0.0 if c["kind"] == "rms" else 1.0) + 0.1 * rn(d)).to(pt)
    st.b = (0.1 * rn(d)).to(pt) if c["kind"] == "layer" else None
    st.dy = (0.01 * rn(n, d)).to(dt)
    if c["call"] == "backward":
        # what the forward pass has kept
        xd = st.x.double()
        st.mean = xd.mean(1) if c["kind"] == "layer" else torch.zeros(n, device="cuda", dtype=torch.float64)
        st.rstd = torch.rsqrt((xd - st.mean[:, None]).square().mean(1) + st.eps).float()
        st.mean = st.mean.float() if c["kind"] == "layer" else None
    if c["call"] == "train":
        st.x.requires_grad_(True)
        st.w.requires_grad_(True)
        if st.b is not None:
            st.b.requires_grad_(True)


def _prepare_route(c, st, rn):
    # experts of different popularity, tokens of different sureness
    st.logits = (rn(c["n"], c["E"]) * (1.0 + 0.5 * rn(c["n"], 1).abs()) + 0.5 * rn(c["E"])).to(DT[c["dtype"]])
    st.bias = (0.05 * rn(c["E"])) if c["bias"] else None
    st.dw = rn(c["n"], c["k"])
    if c["call"] == "train":
        st.logits.requires_grad_(True)


def _prepare_experts(c, st, rn):
    s, dt = SHAPES[c["shape"]], DT[c["dtype"]]
    n, k, d, H, E = c["n"], c["k"], s["d"], s["H"], s["E"]
    x = rn(n, d)
    st.x = (x * torch.rsqrt(x.pow(2).mean(1, keepdim=True) + 1e-6)).to(dt)
    logits = rn(n, E) + 0.5 * rn(E)                      # some experts are wanted more than others
    top, st.experts = logits.topk(k, dim=1)
    st.experts = st.experts.int()
    st.weights = torch.softmax(top, dim=1)
    st.w1, st.w2 = (0.05 * rn(E, d, H)).to(dt), (0.05 * rn(E, H, d)).to(dt)
    st.w_up = (0.05 * rn(E, d, H)).to(dt) if s["glu"] else None
    st.b1 = None if s["glu"] else (0.1 * rn(E, H)).to(dt)
    st.last_bias = None if s["glu"] else (0.1 * rn(d)).to(dt)
    st.act = s["act"]
    st.residual = c["residual"]
    if own:                                              # the module, with its weights laid out once
        import d2dmoe_b200 as D
        cls = D.B200GluExperts if s["glu"] else D.B200KernelExperts
        act = {"relu": torch.nn.ReLU, "gelu": torch.nn.GELU}[s["act"]]
        with torch.device("cuda"):
            st.ex = cls(d, E, expert_dim=H, bias=False if s["glu"] else "without_last",
                        activation=act, intermediate_gating=s["glu"]).to(dt)
        with torch.no_grad():
            if s["glu"]:
                st.ex.layers[0].w.copy_(st.w1)
                st.ex.layers[1].w.copy_(st.w2)
                st.ex.layers[2].w.copy_(st.w_up)
            else:
                st.ex.w1.copy_(st.w1)
                st.ex.b1.copy_(st.b1)
                st.ex.w2.copy_(st.w2)
        st.ex.packed()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    st = State()
    st.c = dict(case)
    {"norm": _prepare_norm, "route": _prepare_route, "experts": _prepare_experts}[case["op"]](case, st, rn)
    return st


# -- the framework's calls ------------------------------------------------------------------------
def _own_norm(c, st):
    import d2dmoe_b200 as D
    how = dict(kind=c["kind"], weight_offset=st.offset)
    if c["call"] == "backward":
        dx, dw, db = D.ops.layer_norm_backward(st.dy, st.x, st.w, st.mean, st.rstd, bias=st.b is not None, **how)
        return {"dx": dx, "dw": dw, "db": db}
    y = D.layer_norm(st.x, st.w, st.b, st.eps, **how)
    if c["call"] == "forward":
        return {"y": y}
    leaves = (st.x, st.w) if st.b is None else (st.x, st.w, st.b)
    return {"y": y, "grads": torch.autograd.grad(y, leaves, st.dy)}


def _own_route(c, st):
    import d2dmoe_b200 as D
    w, e = D.route_tokens(st.logits, c["k"], scores=c["scores"], bias=st.bias, groups=c["groups"],
                          top_groups=c["top_groups"], renormalise=c["renormalise"], scale=c["scale"])
    if c["call"] == "forward":
        return {"weights": w, "experts": e}
    return {"weights": w, "experts": e, "dlogits": torch.autograd.grad(w, st.logits, st.dw)[0]}


def _own_experts(c, st):
    return st.ex.forward_weighted(st.x, st.experts, st.weights, last_bias=st.last_bias,
                                  add_residual=st.residual)


# -- plain forms ----------------------------------------------------------------------------------
@torch.no_grad()
def _plain_norm(c, st):
    x, dy = st.x.float(), st.dy.float()
    w = st.offset + st.w.float()
    if c["call"] == "backward":
        mean, rstd = st.mean[:, None] if c["kind"] == "layer" else 0.0, st.rstd[:, None]
    else:
        mean = x.mean(1, keepdim=True) if c["kind"] == "layer" else 0.0
        rstd = torch.rsqrt((x - mean).square().mean(1, keepdim=True) + st.eps)
    xh = (x - mean) * rstd
    y = xh * w
    if st.b is not None:
        y = y + st.b.float()
    y = y.to(st.x.dtype)
    if c["call"] == "forward":
        return {"y": y}
    g = dy * w
    dx = g - xh * (g * xh).mean(1, keepdim=True)
    if c["kind"] == "layer":
        dx = dx - g.mean(1, keepdim=True)
    dx = (dx * rstd).to(st.x.dtype)
    dw = (dy * xh).sum(0).to(st.w.dtype)
    db = dy.sum(0).to(st.w.dtype) if st.b is not None else None
    if c["call"] == "backward":
        return {"dx": dx, "dw": dw, "db": db}
    return {"y": y, "grads": (dx, dw) if db is None else (dx, dw, db)}


def _scores(c, logits):
    if c["scores"] == "softmax":
        p = torch.exp(logits - logits.amax(1, keepdim=True))
        return p / p.sum(1, keepdim=True)
    return 1.0 / (1.0 + torch.exp(-logits))


def _choice(c, logits, bias):
    """The k experts of each token, the best first, ties to the lowest index: without a bias in the
    order of the logits, which is that of their scores; with one, of score + bias; in 64 bits."""
    l64 = logits.double()
    s = _scores(c, l64)
    key = l64 if bias is None else s + bias.double()
    if c["groups"] > 1:
        n, G = key.shape[0], c["groups"]
        v = (s if bias is None else key).view(n, G, -1)
        v = v.sort(dim=2, descending=True).values[:, :, :2].sum(2)          # the two best of a group
        kept = v.sort(dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        out = torch.ones(n, G, dtype=torch.bool, device=v.device).scatter(1, kept, False)
        key = key.view(n, G, -1).masked_fill(out[:, :, None], -math.inf).view(n, -1)
    return key.sort(dim=1, descending=True, stable=True).indices[:, :c["k"]]


@torch.no_grad()
def _plain_route(c, st):
    l32 = st.logits.float()
    idx = _choice(c, l32, st.bias)
    s = _scores(c, l32)
    chosen = s.gather(1, idx)
    total = chosen.sum(1, keepdim=True)
    p = chosen / total if c["renormalise"] else chosen
    out = {"weights": p * c["scale"], "experts": idx.int()}
    if c["call"] == "forward":
        return out
    g = st.dw * c["scale"]
    if c["renormalise"]:
        g = (g - (p * g).sum(1, keepdim=True)) / total           # of the chosen scores
    ds = torch.zeros_like(s).scatter(1, idx, g)
    if c["scores"] == "softmax":
        dl = s * (ds - (s * ds).sum(1, keepdim=True))
    else:
        dl = ds * s * (1.0 / (1.0 + torch.exp(l32)))
    return {**out, "dlogits": dl.to(st.logits.dtype)}


def _activate(h, act):
    return torch.relu(h) if act == "relu" else 0.5 * h * (1.0 + torch.erf(h * math.sqrt(0.5)))


@torch.no_grad()
def _plain_experts(c, st):
    """Pairs (token, expert) sorted by expert, each used expert's rows padded to the longest list,
    three batched products, back to the tokens, weighted sum."""
    n, k = st.experts.shape
    used, place = st.experts.long().reshape(-1).unique(return_inverse=True)
    order = place.sort(stable=True).indices
    counts = torch.bincount(place, minlength=used.numel())
    first = counts.cumsum(0) - counts
    rank = torch.empty_like(order)
    rank[order] = torch.arange(n * k, device=order.device) - first[place[order]]
    rows = torch.zeros(used.numel(), int(counts.max()), dtype=torch.long, device=order.device)
    rows[place, rank] = torch.arange(n * k, device=order.device) // k
    xe = st.x.float()[rows]
    h = torch.bmm(xe, st.w1[used].float())
    if st.b1 is not None:
        h = h + st.b1[used].float()[:, None]
    h = _activate(h, st.act)
    if st.w_up is not None:
        h = h * torch.bmm(xe, st.w_up[used].float())
    y = torch.bmm(h, st.w2[used].float())[place, rank].view(n, k, -1)
    out = (y * st.weights[:, :, None]).sum(1)
    if st.last_bias is not None:
        out = out + st.last_bias.float()
    if st.residual:
        out = out + st.x.float()
    return out.to(st.x.dtype)


def run(state):
    c = state.c
    if own:
        return {"norm": _own_norm, "route": _own_route, "experts": _own_experts}[c["op"]](c, state)
    return {"norm": _plain_norm, "route": _plain_route, "experts": _plain_experts}[c["op"]](c, state)


def work(case):
    c, es = case, 4 if case["dtype"] == "fp32" else 2
    n = c["n"]
    if c["op"] == "norm":
        ps = 4 if c["params"] == "fp32" else es
        passes = {"forward": 2, "backward": 3, "train": 5}[c["call"]]
        params = (2 if c["kind"] == "layer" else 1) * c["d"] * ps * {"forward": 1, "backward": 2, "train": 2}[c["call"]]
        ops = {"forward": 7, "backward": 14, "train": 21}[c["call"]]
        return {"bytes": passes * n * c["d"] * es + params, "flops": ops * n * c["d"]}
    if c["op"] == "route":
        E, k = c["E"], c["k"]
        moved = n * (E * es + k * 8) + (4 * E if c["bias"] else 0)
        if c["call"] == "train":
            moved += n * (k * 4 + E * es)
        return {"bytes": moved, "flops": (16 if c["call"] == "train" else 8) * n * E}
    s = SHAPES[c["shape"]]
    d, H, E, k, m = s["d"], s["H"], s["E"], c["k"], 3 if s["glu"] else 2
    touched = E * (1.0 - (1.0 - k / E) ** n)                     # experts that any token wants
    return {"bytes": es * (2 * n * d + touched * (m * d * H + (0 if s["glu"] else H))) + 8 * n * k,
            "flops": 2.0 * n * k * d * H * m + 2.0 * n * k * d}


# -- 64 bits, from the definitions -----------------------------------------------------------------
def _exact_norm(c, st):
    x = st.x.detach().double().requires_grad_(True)
    w = st.w.detach().double().requires_grad_(True)
    b = None if st.b is None else st.b.detach().double().requires_grad_(True)
    m = x.mean(-1, keepdim=True) if c["kind"] == "layer" else torch.zeros_like(x[:, :1])
    var = ((x - m) ** 2).sum(-1, keepdim=True) / c["d"]
    y = (x - m) / torch.sqrt(var + st.eps) * (w + st.offset)
    y = y if b is None else y + b
    if c["call"] == "forward":
        return {"y": y.detach()}
    grads = torch.autograd.grad(y, (x, w) if b is None else (x, w, b), st.dy.double())
    if c["call"] == "backward":
        return {"dx": grads[0], "dw": grads[1], "db": None if b is None else grads[2]}
    return {"y": y.detach(), "grads": grads}


def _exact_route(c, st):
    logits = st.logits.detach().double().requires_grad_(True)
    with torch.no_grad():
        idx = _choice(c, st.logits.detach().float(), st.bias)
    s = torch.softmax(logits, 1) if c["scores"] == "softmax" else torch.sigmoid(logits)
    w = s.gather(1, idx)
    if c["renormalise"]:
        w = w / w.sum(1, keepdim=True)
    w = w * c["scale"]
    out = {"weights": w.detach(), "experts": idx.int()}
    if c["call"] == "forward":
        return out
    return {**out, "dlogits": torch.autograd.grad(w, logits, st.dw.double())[0]}


@torch.no_grad()
def exact(case, seed):
    c, st = case, prepare(case, seed)
    if c["op"] != "experts":
        with torch.enable_grad():
            return (_exact_norm if c["op"] == "norm" else _exact_route)(c, st)
    x, wt = st.x.double(), st.weights.double()
    out = torch.zeros_like(x)
    if st.last_bias is not None:
        out += st.last_bias.double()
    if st.residual:
        out += x
    for e in range(st.w1.shape[0]):
        t, j = (st.experts == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        h = x[t] @ st.w1[e].double()
        if st.b1 is not None:
            h = h + st.b1[e].double()
        h = torch.relu(h) if st.act == "relu" else torch.nn.functional.gelu(h)
        if st.w_up is not None:
            h = h * (x[t] @ st.w_up[e].double())
        out.index_add_(0, t, (h @ st.w2[e].double()) * wt[t, j][:, None])
    return out
