"""The operators around a cache of keys and values that serves several sequences of different lengths, as timed cases:

  cache    new rows of k and v quantised to 4 bits as they are written to the cache, and rows of it read back
  kv4      attention of new tokens over such a cache: single tokens, a few, chunks of prompts; with and without a window
  window   attention over a 16-bit cache with a sliding window and a few first tokens that stay visible (sinks)

A sequence of length n has its keys in rows [0, n) of its cache, those of the call's `new` tokens among them: token i is at
position n - new + i.  A position below zero is padding (a sequence shorter than the call): it is not written, and its
output is zero, its log-sum-exp -inf.

4 bits: 32 consecutive channels of a row share a power of two 2^e (a byte, e + 127), the least with amax < 7 * 2^e,
e >= -110; each value is sign and magnitude of x / 2^e rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the
even code), two of them a byte, the first in its low half.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
# query heads, KV heads, head dimension
HEADS = {"llama": (32, 8, 128), "llama_mha": (32, 32, 128), "falcon": (71, 1, 64)}
E_MIN = -110
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _case(name, kind, heads, dtype, batch, new, keys, window=0, sinks=0, lse=False):
    """keys: length of the longest sequence, the new tokens among them."""
    return {"name": name, "kind": kind, "heads": heads, "dtype": dtype, "batch": batch, "new": new, "keys": keys,
            "window": window, "sinks": sinks, "lse": lse}


def listed():
    return [
        # the token of a decode step written to a conversation's cache, and its stored values looked at: nothing but latency
        _case("append_llama_1", "append", "llama", "f16", 1, 1, 1025),
        # a ragged batch of multi-query prompts written in one call; the shorter sequences are padded
        _case("append_falcon_3x333", "append", "falcon", "bf16", 3, 333, 333),
        # four long prompts written: bandwidth
        _case("append_llama_4x4096", "append", "llama", "f16", 4, 4096, 4096),
        # a long conversation's cache read back, as for handing it to another engine
        _case("read_llama_32752", "read", "llama", "bf16", 1, 0, 32752),
        # one decode step of one conversation
        _case("kv4_llama_1x1_4096", "kv4", "llama", "bf16", 1, 1, 4096),
        # one decode step over a long context
        _case("kv4_llama_1x1_32753", "kv4", "llama", "f16", 1, 1, 32753, lse=True),
        # one decode step of a batch of conversations of different lengths
        _case("kv4_llama_32x1_8192", "kv4", "llama", "bf16", 32, 1, 8192),
        # a few tokens of five sequences (speculative decoding), multi-query, in a window
        _case("kv4_falcon_5x3_5000_window", "kv4", "falcon", "f16", 5, 3, 5000, window=1024, sinks=4),
        # a chunk of a long prompt behind what is cached already
        _case("kv4_llama_1x512_16512", "kv4", "llama", "bf16", 1, 512, 16512),
        # a batch's decode step in a window: the length of the conversations no longer matters
        _case("window_llama_16x1_30000", "window", "llama", "bf16", 16, 1, 30000, window=4096, sinks=4),
        # two ragged multi-query prompts, one of them padded, in a narrow window
        _case("window_falcon_2x1000", "window", "falcon", "f16", 2, 1000, 1000, window=256, sinks=16, lse=True),
        # a long prompt in a window
        _case("window_llama_1x8192", "window", "llama", "f16", 1, 8192, 8192, window=1024, sinks=4),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("append", "read", "kv4", "kv4", "kv4", "window", "window"))
    heads, dtype = rng.choice(tuple(HEADS)), rng.choice(("f16", "bf16"))
    most = 4 if HEADS[heads][1] == 32 else 1  # (a KV head per query head: as many bytes in fewer keys)
    batch = _log_int(rng, 1, 32)
    window = sinks = 0
    if kind == "read":
        new, keys = 0, _log_int(rng, 1, max(1, 32768 // batch // most))
    elif kind == "append":
        new = _log_int(rng, 1, 16384 // batch // most)
        keys = new if rng.random() < 0.5 else new + _log_int(rng, 1, 4096)
    else:
        form = rng.choice(("decode", "decode", "chunk", "prompt"))
        if form == "decode":
            new, keys = _log_int(rng, 1, 16), _log_int(rng, 128, min(32768, 131072 // batch // most))
        elif form == "chunk":
            batch = _log_int(rng, 1, 4)
            new, keys = _log_int(rng, 17, 512), _log_int(rng, 600, 16384 // batch)
        else:
            batch = _log_int(rng, 1, 4)
            new = keys = _log_int(rng, 128, 4096 // batch)
        if kind == "window" or rng.random() < 0.4:
            window, sinks = _log_int(rng, 16, 4096), rng.choice((0, 1, 4, 16, 100))
    c = _case("", kind, heads, dtype, batch, new, max(keys, new), window, sinks, kind in ("kv4", "window") and rng.random() < 0.3)
    del c["name"]
    return c


def _lens(case):
    """Lengths of the sequences: from `keys` down to about half of it."""
    b, n = case["batch"], case["keys"]
    return [n - (i * n) // (2 * b) for i in range(b)]


def _visible(case):
    """(sum over the sequences of the keys that some token sees, of the pairs of a token and a key it sees)."""
    keys = pairs = 0
    s, w, sinks = case["new"], case["window"], case["sinks"]
    for n in _lens(case):
        first = max(0, n - s)
        if w == 0:
            keys += n
            pairs += sum(range(first + 1, n + 1))
            continue
        lo = max(0, first - w + 1)
        keys += n - lo + min(sinks, lo)
        for p in range(first, n):
            at = max(0, p - w + 1)
            pairs += p + 1 - at + min(sinks, at)
    return keys, pairs


def work(case):
    hq, hkv, d = HEADS[case["heads"]]
    b, s = case["batch"], case["new"]
    row16, row4 = 2 * d, d // 2 + d // 32
    if case["kind"] in ("append", "read"):
        rows = sum(min(s, n) for n in _lens(case)) if case["kind"] == "append" else sum(_lens(case))
        moved = 2 * hkv * rows
        # append: rows in, 4 bits out and, for their stored values, back in, and those out
        return {"bytes": moved * (2 * row16 + 2 * row4) if case["kind"] == "append" else moved * (row16 + row4),
                "flops": moved * d}
    keys, pairs = _visible(case)
    row = row4 if case["kind"] == "kv4" else row16
    return {"bytes": 2 * keys * hkv * row + 2 * b * s * hq * row16 + (4 * b * s * hq if case["lse"] else 0),
            "flops": 4 * d * hq * pairs}


def _values(seed, dev):
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def make(*shape, std=1.0, dtype=torch.float16):
        return torch.empty(*shape, dtype=dtype, device=dev).normal_(0.0, std, generator=gen)

    def codes(*shape, lo=0, hi=256):
        return torch.randint(lo, hi, shape, dtype=torch.uint8, device=dev, generator=gen)

    return make, codes


def prepare(case, seed):
    dev = torch.device("cuda:0")
    make, codes = _values(seed, dev)
    hq, hkv, d = HEADS[case["heads"]]
    b, s, dt = case["batch"], case["new"], DTYPES[case["dtype"]]
    rows = (case["keys"] // 64 + 1) * 64  # (a cache has room to grow)
    st = {"case": case, "lens": torch.tensor(_lens(case), dtype=torch.int32, device=dev)}
    if case["kind"] == "window":
        st["k_cache"] = make(b, hkv, rows, d, dtype=dt)
        st["v_cache"] = make(b, hkv, rows, d, dtype=dt)
    else:
        # much like a cache of normal values: blocks of up to 1.5 or 3
        for x in ("k", "v"):
            st[x + "_cache"] = codes(b, hkv, rows, d // 2)
            st[x + "_scales"] = codes(b, hkv, rows, d // 32, lo=125, hi=127)
    if case["kind"] == "append":
        # k and v as columns of one projection's output, next to q; some channels of k larger than the others
        qkv = make(b * s, (hq + 2 * hkv) * d, dtype=dt)
        st["k"], st["v"] = qkv[:, hq * d:(hq + hkv) * d], qkv[:, (hq + hkv) * d:]
        st["k"].mul_(torch.exp(make(hkv * d, std=0.7, dtype=torch.float32)).to(dt))
    elif case["kind"] != "read":
        st["q"] = make(b * s, hq * d, dtype=dt)
    return st


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(st):
    from trinity_amd import blocks

    c = st["case"]
    hq, hkv, d = HEADS[c["heads"]]
    op = st.get("op")
    if op is None:  # made once by a program, with the workspace that it keeps
        op = st["op"] = blocks.CachedAttention(hq, hkv, d, window=c["window"], sinks=c["sinks"])
    if c["kind"] in ("append", "read"):
        kw = {"lens": st["lens"], "kv_len": c["keys"]}
        cache = (st["k_cache"], st["v_cache"], st["k_scales"], st["v_scales"])
        if c["kind"] == "append":
            op.append(st["k"], st["v"], *cache, **kw)
        return op.read(*cache, DTYPES[c["dtype"]], rows=c["new"] or c["keys"], **kw)
    return op.attend(st["q"], st["k_cache"], st["v_cache"], st.get("k_scales"), st.get("v_scales"), lens=st["lens"],
                     kv_len=c["keys"], want_lse=c["lse"])


# ------------------------------------------------------------------------------------------------------- the plain form
def _power(e):
    """2^e as fp32, exactly, for whole e in [-126, 127]."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _decode4(codes, scales):
    """fp32 values of cache rows [..., d]."""
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.float32, device=codes.device)
    both = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)
    x = level[both.int()]
    return (x.unflatten(-1, (-1, 32)) * _power(scales.int() - 127).unsqueeze(-1)).flatten(-2)


def _encode4(x):
    """codes and scales of fp32 rows [..., d]."""
    blk = x.unflatten(-1, (-1, 32))
    amax = blk.abs().amax(-1)
    bits = amax.view(torch.int32)
    e = (bits >> 23) - 127 - 2 + ((bits & 0x7FFFFF) >= 0x600000).int()  # (at least 1.75 times its power of two: one more)
    e = e.clamp(min=E_MIN)
    y = blk.abs() / _power(e).unsqueeze(-1)
    code = ((y > 0.25).int() + (y >= 0.75).int() + (y > 1.25).int() + (y >= 1.75).int() + (y > 2.5).int()
            + (y >= 3.5).int() + (y > 5.0).int())
    code = (code + 8 * torch.signbit(blk).int()).flatten(-2)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8), (e + 127).to(torch.uint8)


def _plain_append(st):
    hq, hkv, d = HEADS[st["case"]["heads"]]
    b, s = st["case"]["batch"], st["case"]["new"]
    pos = st["lens"].long()[:, None] - s + torch.arange(s, device=st["lens"].device)
    row = torch.where(pos >= 0, pos, st["k_cache"].shape[2] - 1)  # (padding goes to the last row, which no sequence reaches)
    seq = torch.arange(b, device=pos.device)[:, None]
    for x in ("k", "v"):
        codes, scales = _encode4(st[x].float().view(b, s, hkv, d))
        st[x + "_cache"][seq, :, row] = codes
        st[x + "_scales"][seq, :, row] = scales


def _plain_read(st, rows):
    """The last `rows` rows of each sequence [b, hkv, rows, d] (zero where it has fewer)."""
    dt = DTYPES[st["case"]["dtype"]]
    b = st["case"]["batch"]
    row = st["lens"].long()[:, None] - rows + torch.arange(rows, device=st["lens"].device)
    seq, real = torch.arange(b, device=row.device)[:, None], (row >= 0)[:, None, :, None]
    out = []
    for x in ("k", "v"):
        codes = st[x + "_cache"].transpose(1, 2)[seq, row.clamp(min=0)].transpose(1, 2)
        scales = st[x + "_scales"].transpose(1, 2)[seq, row.clamp(min=0)].transpose(1, 2)
        out.append(torch.where(real, _decode4(codes, scales), 0.0).to(dt))
    return out


def _plain_attend(st):
    c = st["case"]
    hq, hkv, d = HEADS[c["heads"]]
    b, s, n, g = c["batch"], c["new"], c["keys"], hq // hkv
    if c["kind"] == "kv4":
        k, v = (_decode4(st[x + "_cache"][:, :, :n], st[x + "_scales"][:, :, :n]) for x in ("k", "v"))
    else:
        k, v = st["k_cache"][:, :, :n].float(), st["v_cache"][:, :, :n].float()
    q = st["q"].float().view(b, s, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * s, d)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(b, hkv, g, s, n) * d ** -0.5
    key = torch.arange(n, device=q.device)
    pos = (st["lens"].long()[:, None] - s + torch.arange(s, device=q.device))[..., None]
    seen = key <= pos
    if c["window"]:
        seen = seen & ((key > pos - c["window"]) | (key < c["sinks"]))
    seen, real = seen[:, None, None], (pos >= 0)[:, None, None]
    x = torch.where(seen, x, -math.inf)
    top = torch.where(real, x.amax(-1, keepdim=True), 0.0)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, hkv, g * s, n), v).view(b, hkv, g, s, d)
    o = torch.where(real, o / total, 0.0)
    out = o.permute(0, 3, 1, 2, 4).reshape(b * s, hq * d).to(DTYPES[c["dtype"]])
    if not c["lse"]:
        return out
    return out, (top + torch.log(total)).reshape(b, hq, s)


def run(st):
    if own:
        return _own(st)
    c = st["case"]
    if c["kind"] == "append":
        _plain_append(st)
    if c["kind"] in ("append", "read"):
        return _plain_read(st, c["new"] or c["keys"])
    return _plain_attend(st)


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


def _exact_cache(codes, scales):
    lo, hi = (codes % 16).long(), (codes // 16).long()
    code = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.long, device=codes.device)
    code[..., 0::2], code[..., 1::2] = lo, hi
    mag = code % 8
    val = torch.where(mag < 2, mag * 0.5, (1 + (mag % 2) * 0.5).double() * torch.exp2((mag // 2 - 1).double()))
    val = torch.where(code >= 8, -val, val).double()
    return val * torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.int() - 127).repeat_interleave(32, -1)


def exact(case, seed):
    st = prepare(case, seed)
    hq, hkv, d = HEADS[case["heads"]]
    b, s = case["batch"], case["new"]
    lens = _lens(case)
    dev = st["lens"].device
    if case["kind"] in ("append", "read"):
        rows = s or case["keys"]
        outs = []
        for x in ("k", "v"):
            out = torch.zeros(b, hkv, rows, d, dtype=torch.float64, device=dev)
            for i, n in enumerate(lens):
                m = min(rows, n)
                if case["kind"] == "read":
                    out[i, :, rows - m:] = _exact_cache(st[x + "_cache"][i, :, n - m:n], st[x + "_scales"][i, :, n - m:n])
                else:
                    new = st[x].double().view(b, s, hkv, d)[i, s - m:]
                    out[i, :, rows - m:] = _exact_levels(new).transpose(0, 1)
            outs.append(out)
        return outs
    out = torch.zeros(b, s, hq, d, dtype=torch.float64, device=dev)
    lse = torch.full((b, hq, s), -math.inf, dtype=torch.float64, device=dev)
    q = st["q"].double().view(b, s, hq, d)
    for i, n in enumerate(lens):
        for hk in range(hkv):
            if case["kind"] == "kv4":
                k, v = (_exact_cache(st[x + "_cache"][i, hk, :n], st[x + "_scales"][i, hk, :n]) for x in ("k", "v"))
            else:
                k, v = st["k_cache"][i, hk, :n].double(), st["v_cache"][i, hk, :n].double()
            for h in range(hk * (hq // hkv), (hk + 1) * (hq // hkv)):
                for i0 in range(max(0, s - n), s, 1024):
                    i1 = min(s, i0 + 1024)
                    pos = torch.arange(n - s + i0, n - s + i1, device=dev)[:, None]
                    key = torch.arange(n, device=dev)[None]
                    hidden = key > pos
                    if case["window"]:
                        hidden |= (key <= pos - case["window"]) & (key >= case["sinks"])
                    z = (q[i, i0:i1, h] @ k.T) / math.sqrt(d)
                    z.masked_fill_(hidden, -math.inf)
                    lse[i, h, i0:i1] = torch.logsumexp(z, -1)
                    out[i, i0:i1, h] = torch.softmax(z, -1) @ v
    out = out.reshape(b * s, hq * d)
    return (out, lse) if case["lse"] else out
