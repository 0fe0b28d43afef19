"""4-bit weights and routed experts, as timed cases:

  quantize  activations or weights to 4-bit blocks, and the values that these stand for
  product   y = x . w^T with 4-bit weights; x in 16 bits, or quantised to 4 bits too within the call
  route     scores of a router to the experts of each token and their weights
  experts   the SwiGLU FFN of the experts that the tokens chose, 16-bit or 4-bit weights

4 bits: 32 consecutive values of a row share a power of two 2^e (a byte, e + 127), the least with amax < 7 * 2^e,
e >= -110; each value is sign and magnitude of x / 2^e rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the
even code), two of them a byte, the first in its low half.

Routing: s = softmax or sigmoid of a token's logits; experts are chosen by c = s + bias, the `top_k` largest in descending
order, ties to the lowest index.  With groups only those of the `top_groups` best groups of experts are in question, a group
counting the sum of its `group_top` largest c.  Weights are s of the chosen, divided by their sum if renormalised, times scale.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# model width and FFN width
WIDTHS = {"llama": (4096, 14336), "falcon": (4544, 18176)}
# experts: number, chosen per token, model width, expert width.  Whole FFNs; and FFNs an eighth as wide, of either model
EXPERTS = {"llama8": (8, 2, 4096, 14336), "llama64": (64, 6, 4096, 1792), "falcon32": (32, 4, 4544, 2272)}
E_MIN = -110
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quantize(name, dtype, rows, k):
    return {"name": name, "kind": "quantize", "dtype": dtype, "rows": rows, "k": k}


def _product(name, dtype, rows, k, n, x4):
    return {"name": name, "kind": "product", "dtype": dtype, "rows": rows, "k": k, "n": n, "x4": x4}


def _route(name, dtype, tokens, experts, top_k, scores, bias=False, groups=1, top_groups=1, group_top=1, renormalize=True, scale=1.0):
    return {"name": name, "kind": "route", "dtype": dtype, "tokens": tokens, "experts": experts, "top_k": top_k, "scores": scores,
            "bias": bias, "groups": groups, "top_groups": top_groups, "group_top": group_top, "renormalize": renormalize,
            "scale": scale}


def _experts(name, config, dtype, tokens, w4):
    return {"name": name, "kind": "experts", "config": config, "dtype": dtype, "tokens": tokens, "w4": w4}


def listed():
    return [
        # the activations of a decode step over a small batch, ahead of a product: nothing but latency
        _quantize("quantize_falcon_16", "bf16", 16, 4544),
        # a weight matrix as it is loaded: bandwidth
        _quantize("quantize_llama_4096", "f16", 4096, 14336),
        # one token through the down projection: the weights' bytes
        _product("product_llama_1", "bf16", 1, 14336, 4096, False),
        # a chunk of a prompt or a large decode batch, ragged, over weights whose rows are no multiple of 128 values
        _product("product_falcon_333", "f16", 333, 4544, 18176, False),
        # a long prompt, both sides in 4 bits: the 4-bit matrix rate
        _product("product_llama_4096_x4", "bf16", 4096, 4096, 14336, True),
        # the routing of one token among a few experts
        _route("route_1x8", "bf16", 1, 8, 2, "softmax"),
        # a long prompt among many experts in groups, balanced by a bias
        _route("route_4096x256_groups", "f32", 4096, 256, 8, "sigmoid", bias=True, groups=8, top_groups=4, group_top=2, scale=2.5),
        # one token of one conversation through two whole FFNs
        _experts("experts_llama8_1", "llama8", "bf16", 1, False),
        # a decode batch: every expert has a few rows
        _experts("experts_llama8_32_w4", "llama8", "bf16", 32, True),
        # a ragged chunk over small experts of odd width, some 40 rows each
        _experts("experts_falcon32_333", "falcon32", "f16", 333, False),
        # a prompt over 4-bit weights
        _experts("experts_llama64_2048_w4", "llama64", "bf16", 2048, True),
        # a long prompt: the matrix rate
        _experts("experts_llama8_4096", "llama8", "f16", 4096, False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("quantize", "product", "product", "product", "route", "route", "experts", "experts", "experts"))
    dtype = rng.choice(("f16", "bf16"))
    if kind == "quantize":
        n, f = WIDTHS[rng.choice(tuple(WIDTHS))]
        c = _quantize("", dtype, _log_int(rng, 1, 4096), rng.choice((n, f)))
    elif kind == "product":
        n, f = WIDTHS[rng.choice(tuple(WIDTHS))]
        k, cols = rng.choice(((n, f), (f, n), (n, n)))
        c = _product("", dtype, _log_int(rng, 1, 4096), k, cols, rng.random() < 0.5)
    elif kind == "route":
        experts = rng.choice((8, 16, 32, 64, 128, 160, 256))
        top_k = rng.randint(1, 8)
        groups = rng.choice((1, 1, 4, 8)) if experts >= 32 else 1
        size = experts // groups
        top_groups = rng.randint(min(groups, (top_k + size - 1) // size), groups)
        bias = rng.random() < 0.5
        c = _route("", rng.choice(("f32", "f16", "bf16")), _log_int(rng, 1, 16384), experts, top_k, rng.choice(("softmax", "sigmoid")), bias,
                   groups, top_groups, 2 if bias else 1, rng.random() < 0.7, rng.choice((1.0, 2.5)))
    else:
        c = _experts("", rng.choice(tuple(EXPERTS)), dtype, _log_int(rng, 1, 4096), rng.random() < 0.5)
    del c["name"]
    return c


def work(case):
    kind = case["kind"]
    if kind == "quantize":
        values = case["rows"] * case["k"]
        # 16 bits in, 4 bits out and, for the values they stand for, back in, and those out
        return {"bytes": values * 2 * (2 + 17 / 32), "flops": values * 2}
    if kind == "product":
        m, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": n * k * 17 / 32 + m * k * 2 + m * n * 2, "flops": 2 * m * n * k}
    if kind == "route":
        t, e = case["tokens"], case["experts"]
        return {"bytes": t * e * (4 if case["dtype"] == "f32" else 2) + (4 * e if case["bias"] else 0) + t * case["top_k"] * 8,
                "flops": t * e * 8}
    e, k, n, f = EXPERTS[case["config"]]
    t = case["tokens"]
    chosen = e * (1.0 - (1.0 - k / e) ** t)  # experts that some token chose, if all are as likely
    return {"bytes": chosen * 3 * n * f * (17 / 32 if case["w4"] else 2) + 4 * t * n + 8 * t * k, "flops": 6 * t * k * n * f}


def _values(seed, dev):
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def make(*shape, std=1.0, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device=dev).normal_(0.0, std, generator=gen)

    def codes(*shape, lo=0, hi=256):
        return torch.randint(lo, hi, shape, dtype=torch.uint8, device=dev, generator=gen)

    return make, codes


def prepare(case, seed):
    dev = torch.device("cuda:0")
    make, codes = _values(seed, dev)
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    st = {"case": case}
    if kind == "quantize":
        # some channels larger than the others, as activations have them
        st["x"] = make(case["rows"], case["k"], dtype=dt).mul_(torch.exp(make(case["k"], std=0.7)).to(dt))
    elif kind == "product":
        m, k, n = case["rows"], case["k"], case["n"]
        st["x"] = make(m, k, dtype=dt).mul_(torch.exp(make(k, std=0.5)).to(dt))
        # much like normal weights of a deviation of 0.02
        st["w"], st["w_scales"] = codes(n, k // 2), codes(n, k // 32, lo=119, hi=121)
    elif kind == "route":
        st["logits"] = make(case["tokens"], case["experts"], std=1.5).to(dt)
        st["bias"] = make(case["experts"], std=0.1) if case["bias"] else None
    else:
        e, k, n, f = EXPERTS[case["config"]]
        t = case["tokens"]
        st["x"] = make(t, n, dtype=dt)
        top = (make(t, e) + make(e, std=0.2)).topk(k, dim=-1)  # (some experts are chosen more often)
        st["ids"], st["weights"] = top.indices.to(torch.int32), torch.softmax(top.values, -1)
        for name, rows, cols in (("gate", f, n), ("up", f, n), ("down", n, f)):
            if case["w4"]:
                st[name], st[name + "_scales"] = codes(e, rows, cols // 2), codes(e, rows, cols // 32, lo=119, hi=121)
            else:
                st[name], st[name + "_scales"] = make(e, rows, cols, std=0.02, dtype=dt), None
    return st


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(st):
    from trinity_amd import blocks

    c = st["case"]
    if c["kind"] == "quantize":
        codes, scales = blocks.Fp4Matmul.quantize(st["x"])
        return blocks.Fp4Matmul.dequantize(codes, scales, DTYPES[c["dtype"]])
    op = st.get("op")
    if c["kind"] == "product":
        if op is None:  # made once by a program
            op = st["op"] = blocks.Fp4Matmul(quantize_x=c["x4"])
        return op.run(st["x"], st["w"], st["w_scales"])
    if c["kind"] == "route":
        if op is None:
            op = st["op"] = blocks.Router(c["top_k"], scores=c["scores"], groups=c["groups"], top_groups=c["top_groups"],
                                          group_top=c["group_top"], renormalize=c["renormalize"], scale=c["scale"])
        return op.route(st["logits"], st["bias"])
    if op is None:
        op = st["op"] = blocks.ExpertsFfn()
    return op.run(st["x"], st["ids"], st["weights"], st["gate"], st["up"], st["down"], st["gate_scales"], st["up_scales"],
                  st["down_scales"])


# ------------------------------------------------------------------------------------------------------- the plain form
def _power(e):
    """2^e as fp32, exactly, for whole e in [-126, 127]."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _decode4(codes, scales):
    """fp32 values of rows [..., k]."""
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.float32, device=codes.device)
    both = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)
    x = level[both.int()]
    return (x.unflatten(-1, (-1, 32)) * _power(scales.int() - 127).unsqueeze(-1)).flatten(-2)


def _encode4(x):
    """codes and scales of fp32 rows [..., k]."""
    blk = x.unflatten(-1, (-1, 32))
    bits = blk.abs().amax(-1).view(torch.int32)
    e = (bits >> 23) - 127 - 2 + ((bits & 0x7FFFFF) >= 0x600000).int()  # (at least 1.75 times its power of two: one more)
    e = e.clamp(min=E_MIN)
    y = blk.abs() / _power(e).unsqueeze(-1)
    code = ((y > 0.25).int() + (y >= 0.75).int() + (y > 1.25).int() + (y >= 1.75).int() + (y > 2.5).int()
            + (y >= 3.5).int() + (y > 5.0).int())
    code = (code + 8 * torch.signbit(blk).int()).flatten(-2)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8), (e + 127).to(torch.uint8)


def _plain_quantize(st):
    codes, scales = _encode4(st["x"].float())
    return _decode4(codes, scales).to(st["x"].dtype)


def _plain_product(st):
    x = st["x"].float()
    if st["case"]["x4"]:
        x = _decode4(*_encode4(x))
    return torch.matmul(x, _decode4(st["w"], st["w_scales"]).T).to(st["x"].dtype)


def _plain_route(st):
    c = st["case"]
    t, e, k = c["tokens"], c["experts"], c["top_k"]
    # (in 64 bits: scores next to each other are told apart)
    z = st["logits"].double()
    if c["scores"] == "softmax":
        p = torch.exp(z - z.amax(-1, keepdim=True))
        s = p / p.sum(-1, keepdim=True)
    else:
        s = 1.0 / (1.0 + torch.exp(-z))
    choice = s if st["bias"] is None else s + st["bias"].double()
    if c["groups"] > 1:
        by_group = choice.view(t, c["groups"], -1)
        group = by_group.sort(dim=-1, descending=True).values[..., :c["group_top"]].sum(-1)
        best = group.sort(dim=-1, descending=True, stable=True).indices[:, :c["top_groups"]]
        stays = torch.zeros(t, c["groups"], dtype=torch.bool, device=z.device)
        stays.scatter_(1, best, True)
        choice = torch.where(stays[..., None], by_group, -math.inf).view(t, e)
    ids = choice.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    w = s.gather(1, ids)
    if c["renormalize"]:
        w = w / w.sum(-1, keepdim=True)
    return ids.to(torch.int32), (w * c["scale"]).float()


def _plain_experts(st):
    c = st["case"]
    e, k, n, f = EXPERTS[c["config"]]
    t = c["tokens"]
    # each expert's rows next to each other, as many for each as the busiest has; experts without rows are left out
    of, order = st["ids"].flatten().long().sort(dim=0, stable=True)
    counts = torch.bincount(of, minlength=e)
    present = counts.nonzero().flatten()
    place = (counts > 0).long().cumsum(0)[of] - 1
    at = torch.arange(t * k, device=of.device) - (counts.cumsum(0) - counts)[of]
    x = torch.zeros(present.numel(), int(counts.max()), n, dtype=torch.float32, device=of.device)
    x[place, at] = st["x"][order // k].float()

    def product(a, name):
        w = _decode4(st[name][present], st[name + "_scales"][present]) if c["w4"] else st[name][present].float()
        return torch.matmul(a, w.transpose(1, 2))

    g = product(x, "gate")
    y = product(g / (1.0 + torch.exp(-g)) * product(x, "up"), "down")
    back = torch.empty(t * k, n, dtype=torch.float32, device=of.device)
    back[order] = y[place, at]
    return (back.view(t, k, n) * st["weights"][..., None]).sum(1).to(st["x"].dtype)


def run(st):
    if own:
        return _own(st)
    kind = st["case"]["kind"]
    if kind == "quantize":
        return _plain_quantize(st)
    if kind == "product":
        return _plain_product(st)
    if kind == "route":
        return _plain_route(st)
    return _plain_experts(st)


# ------------------------------------------------------------------------------------------------------------ in 64 bits
def _exact_levels(x):
    """x in fp64, blocks of 32 in the last dimension, as the values that 4 bits hold."""
    blk = x.reshape(*x.shape[:-1], -1, 32)
    amax = blk.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(torch.where(amax > 0, amax, 1.0))  # amax = m 2^e, m in [0.5, 1)
    e = torch.where(m >= 0.875, e - 2, e - 3)
    e = torch.where(amax > 0, e, E_MIN).clamp(min=E_MIN)
    unit = torch.ldexp(torch.ones_like(amax), e)
    y = blk / unit
    # between 0 and 2 the levels are halves, up to 4 ones, beyond twos
    a = y.abs()
    r = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), (torch.round(a / 2) * 2).clamp(max=6.0)))
    return (torch.copysign(r, y) * unit).reshape(x.shape)


def _exact_values(codes, scales):
    lo, hi = (codes % 16).long(), (codes // 16).long()
    code = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.long, device=codes.device)
    code[..., 0::2], code[..., 1::2] = lo, hi
    mag = code % 8
    val = torch.where(mag < 2, mag * 0.5, (1 + (mag % 2) * 0.5).double() * torch.exp2((mag // 2 - 1).double()))
    val = torch.where(code >= 8, -val, val).double()
    return val * torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.int() - 127).repeat_interleave(32, -1)


def _exact_route(st, c):
    z = st["logits"].double()
    s = torch.softmax(z, -1) if c["scores"] == "softmax" else torch.sigmoid(z)
    choice = s.clone() if st["bias"] is None else s + st["bias"].double()
    if c["groups"] > 1:
        size = c["experts"] // c["groups"]
        group = torch.stack([choice[:, i * size:(i + 1) * size].topk(c["group_top"], -1).values.sum(-1) for i in range(c["groups"])], 1)
        for _ in range(c["groups"] - c["top_groups"]):
            worst = c["groups"] - 1 - group.flip(1).argmin(1)  # (of equal ones the last)
            group.scatter_(1, worst[:, None], math.inf)
            choice.masked_fill_((torch.arange(c["experts"], device=z.device) // size)[None] == worst[:, None], -math.inf)
    w = []
    for _ in range(c["top_k"]):
        i = choice.argmax(1, keepdim=True)
        w.append(s.gather(1, i))
        choice.scatter_(1, i, -math.inf)
    w = torch.cat(w, 1)
    return None, w / (w.sum(1, keepdim=True) if c["renormalize"] else 1.0) * c["scale"]


def _exact_experts(st, c):
    e, k, n, f = EXPERTS[c["config"]]
    x, out = st["x"].double(), torch.zeros(c["tokens"], n, dtype=torch.float64, device=st["x"].device)
    for i in range(e):
        t, j = (st["ids"] == i).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        w = [_exact_values(st[m][i], st[m + "_scales"][i]) if c["w4"] else st[m][i].double() for m in ("gate", "up", "down")]
        h = torch.nn.functional.silu(x[t] @ w[0].T) * (x[t] @ w[1].T)
        out.index_add_(0, t, (h @ w[2].T) * st["weights"][t, j].double()[:, None])
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "quantize":
        return _exact_levels(st["x"].double())
    if case["kind"] == "product":
        x = st["x"].double()
        return (_exact_levels(x) if case["x4"] else x) @ _exact_values(st["w"], st["w_scales"]).T
    if case["kind"] == "route":
        return _exact_route(st, case)
    return _exact_experts(st, case)
