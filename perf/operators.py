"""Cases of the 4- and 8-bit KV cache: appending rows, reading them back, attending over them.

A row of `dim` values is held in blocks of 8 consecutive values.  A block has one power of two, 2**e,
the smallest with max|x| <= top * 2**e, and eight codes: 4 bits (0 .5 1 1.5 2 3 4 6 and negatives,
top = 7) or 8 bits (e4m3, largest 448, top = 464), x / 2**e rounded to the nearest, ties to even.
`inputs` makes the data of a case from its seed; `run` is the plain form or, with `own`, the calls
into recurrent_drafting_amd; `exact` is the definition in 64 bits.
"""

import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BLOCK = 8


def _package():
    path = os.path.join(os.getcwd(), "ml-recurrent-drafter_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from recurrent_drafting_amd import attention, kv_cache

    return attention, kv_cache


# ---- cases ---------------------------------------------------------------------------------------

def _case(name, op, batch, new, prev, heads, kv_heads, dim, bits, dtype, mask="token", ragged=False):
    return dict(name=name, op=op, batch=batch, new=new, prev=prev, heads=heads, kv_heads=kv_heads, dim=dim,
                bits=bits, dtype=dtype, mask=mask, ragged=ragged)


def listed():
    return [
        # one token of one sequence, grouped heads: the smallest call of a serving loop
        _case("append 1 token 8-bit f16", "append", 1, 1, 500, 32, 8, 128, 8, "f16"),
        # the verification step of the 7B shape: batch 8, a tree of 115 packed tokens
        _case("append tree 4-bit", "append", 8, 115, 1500, 32, 32, 128, 4, "bf16"),
        # a prompt: many tokens, grouped heads of 64
        _case("append prompt 4-bit d64", "append", 4, 1021, 0, 32, 8, 64, 4, "bf16"),
        # a layer's rows handed to code that wants them in 16 bits (View.slice)
        _case("read layer 4-bit", "read", 8, 0, 2548, 32, 32, 128, 4, "bf16"),
        _case("read odd 8-bit f16 d64", "read", 3, 0, 777, 8, 8, 64, 8, "f16"),
        # single tokens: the shortest cache, the 7B shape at full context, one long sequence of grouped heads
        _case("attend 1 token short", "attend", 1, 1, 32, 32, 8, 128, 4, "bf16"),
        _case("attend token 4-bit", "attend", 8, 1, 2547, 32, 32, 128, 4, "bf16", ragged=True),
        _case("attend token long 8-bit", "attend", 1, 1, 65536, 32, 8, 128, 8, "f16"),
        # trees: the 7B shape early in its trajectory, the wide tree of the 13B shape with ragged rows,
        # grouped heads of 64
        _case("attend tree 4-bit", "attend", 8, 115, 620, 32, 32, 128, 4, "bf16", mask="tree"),
        _case("attend tree ragged 8-bit", "attend", 16, 162, 1800, 40, 40, 128, 8, "bf16", mask="tree", ragged=True),
        _case("attend tree 4-bit gqa d64", "attend", 16, 46, 1211, 32, 8, 64, 4, "f16", mask="tree", ragged=True),
        # a prompt over the rows it has just appended, left-padded rows in the batch
        _case("attend prompt 4-bit gqa", "attend", 2, 1900, 0, 32, 8, 128, 4, "bf16", mask="prompt", ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend", "attend"])
    heads, kv_heads = rng.choice([(32, 32), (32, 8), (40, 40), (24, 4), (12, 12), (16, 1)])
    dim = rng.choice([64, 128, 128])
    bits = rng.choice([4, 4, 8])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    batch = _log(rng, 1, 16)
    if op == "append":
        new, prev, mask = _log(rng, 1, 900), rng.randint(0, 700), "token"
        batch = min(batch, max(1, 400000 // (new * (heads + 2 * kv_heads))))
    elif op == "read":
        new, prev, mask = 0, _log(rng, 1, 1200), "token"
    else:
        mask = rng.choice(["token", "tree", "tree", "prompt"])
        if mask == "token":
            new, prev = 1, _log(rng, 1, 12000 // batch)
        elif mask == "tree":
            new, prev = rng.randint(2, 225), _log(rng, 16, 1700)
            batch = min(batch, max(1, 160000000 // (new * (new + prev) * heads)))
        else:
            batch = min(batch, 3)
            new, prev = _log(rng, 2, 1300), 0
    return dict(op=op, batch=batch, new=new, prev=prev, heads=heads, kv_heads=kv_heads, dim=dim, bits=bits,
                dtype=dtype, mask=mask, ragged=rng.random() < 0.6)


# ---- inputs --------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _keys_and_values(case, g, tokens):
    """(batch, tokens, kv_heads * dim) keys, whose channels differ in size, and values."""
    shape = (case["batch"], tokens, case["kv_heads"] * case["dim"])
    dt = _DTYPES[case["dtype"]]
    gain = torch.exp(0.5 * torch.randn(shape[2], generator=g, device="cuda"))
    k = (torch.randn(shape, generator=g, device="cuda") * gain).to(dt)
    v = torch.randn(shape, generator=g, device="cuda").to(dt)
    return k, v


def _mask(case, g):
    """(batch, new, prev + new) bool: which keys each query attends to."""
    B, n, prev = case["batch"], case["new"], case["prev"]
    kv = prev + n
    key = torch.arange(kv, device="cuda")
    query = torch.arange(n, device="cuda")
    pads = torch.zeros(B, dtype=torch.long, device="cuda")
    if case["ragged"]:
        pads = torch.randint(0, (prev if prev else n) * 3 // 4 + 1, (B,), generator=g, device="cuda")
        pads[0] = 0  # the longest row has none
    if case["mask"] == "prompt":
        m = key <= prev + query[:, None]
        m = m.expand(B, n, kv)
    else:
        # a random tree: the parent of node t is one of the nodes before it, node 0 is the root
        m = torch.zeros((B, n, kv), dtype=torch.bool, device="cuda")
        m[:, :, :prev] = True
        parent = torch.rand((B, n), generator=g, device="cuda") * query
        parent = parent.long()
        up = torch.eye(n, dtype=torch.bool, device="cuda").repeat(B, 1, 1)
        rows = torch.arange(B, device="cuda")
        for t in range(1, n):
            up[:, t] |= up[rows, parent[:, t]]
        m[:, :, prev:] = up
    m = m & (key >= pads[:, None, None])
    # a row that attends to nothing (left padding) attends to everything, as the model arranges it
    return m | ~m.any(dim=2, keepdim=True)


def inputs(case, seed):
    g = _generator(seed)
    dt = _DTYPES[case["dtype"]]
    D, B, n = case["dim"], case["batch"], case["new"]
    x = {}
    if case["op"] == "append":
        x["q"] = torch.randn((B, n, case["heads"] * D), generator=g, device="cuda").to(dt)
        x["k"], x["v"] = _keys_and_values(case, g, n)
        angle = torch.outer(torch.arange(case["prev"] + n, device="cuda").float(),
                            1.0 / (10000.0 ** (torch.arange(0, D, 2, device="cuda").float() / D)))
        angle = torch.cat((angle, angle), dim=-1)
        x["cos"], x["sin"] = angle.cos().to(dt), angle.sin().to(dt)
        offset = torch.arange(n, device="cuda").expand(B, n)
        x["position_ids"] = (case["prev"] + offset -
                             torch.randint(0, case["prev"] + 1, (B, 1), generator=g, device="cuda"))
        x["position_ids"] = x["position_ids"].contiguous()
        return x
    x["k"], x["v"] = _keys_and_values(case, g, case["prev"] + n)
    if case["op"] == "attend":
        x["q"] = (2.0 * torch.randn((B, n, case["heads"] * D), generator=g, device="cuda")).to(dt)
        x["mask"] = _mask(case, g)
    return x


def _heads(x, dim):
    """(B, n, heads * dim) -> (B, heads, n, dim)"""
    return x.unflatten(2, (-1, dim)).transpose(1, 2)


# ---- plain form ----------------------------------------------------------------------------------

def _exponent_range(bits, dtype):
    top = 15 if dtype == torch.float16 else 127
    hi = top - (2 if bits == 4 else 8)
    lo = (-23 if bits == 4 else -15) if dtype == torch.float16 else -100
    return lo, hi


def _pow2(e):
    """2**e in float64, from the exponent field."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _encode(x, bits, dtype):
    """x (..., D) float64 -> codes (two 4-bit codes in a byte, or e4m3 bytes) and block exponents."""
    y = x.unflatten(-1, (-1, _BLOCK))
    amax = y.abs().amax(dim=-1)
    lo, hi = _exponent_range(bits, dtype)
    top, bias = (7.0, 3) if bits == 4 else (464.0, 9)
    e = torch.frexp(amax)[1] - bias
    e = e + (amax > top * _pow2(e)).to(e.dtype)
    e = torch.where(amax == 0, torch.full_like(e, lo), e).clamp(lo, hi)
    y = y * _pow2(-e).unsqueeze(-1)
    mag = y.abs()
    if bits == 4:
        step = torch.where(mag < 2, 0.5, torch.where(mag < 4, 1.0, 2.0))
        mag = (torch.round(mag / step) * step).clamp(max=6.0)
        # 0 .5 1 1.5 2 3 4 6 -> 0 .. 7
        code = torch.where(mag < 2, mag * 2, torch.where(mag < 4, mag + 2, mag / 2 + 4)).to(torch.uint8)
        code = (code | (torch.signbit(y).to(torch.uint8) << 3)).flatten(-2)
        code = code[..., 0::2] | (code[..., 1::2] << 4)
    else:
        binade = (torch.frexp(mag.clamp(min=2.0 ** -20))[1] - 1).clamp(min=-6)
        step = _pow2(binade - 3)
        mag = (torch.round(mag / step) * step).clamp(max=448.0)
        code = torch.copysign(mag, y).to(torch.float8_e4m3fn).view(torch.uint8).flatten(-2)
    return code, e.to(torch.int16)


def _decode(code, e, bits):
    """float32 values (..., D) of codes and block exponents."""
    if bits == 4:
        level = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=code.device)
        level = torch.cat((level, -level))
        pair = torch.stack((code & 15, code >> 4), dim=-1).flatten(-2)
        x = level[pair.int()]
    else:
        x = code.view(torch.float8_e4m3fn).float()
    x = x.unflatten(-1, (-1, _BLOCK)) * _pow2(e).float().unsqueeze(-1)
    return x.flatten(-2)


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    return x * cos + torch.cat((-x[..., half:], x[..., :half]), dim=-1) * sin


def _plain(state):
    case, x = state["case"], state["x"]
    dt, D, bits = _DTYPES[case["dtype"]], case["dim"], case["bits"]
    if case["op"] == "append":
        cos = x["cos"][x["position_ids"]].unsqueeze(1)
        sin = x["sin"][x["position_ids"]].unsqueeze(1)
        q = _rotate(_heads(x["q"], D).float(), cos.float(), sin.float()).to(dt)
        # (in 64 bits: a key next to the border of two codes)
        k = _encode(_rotate(_heads(x["k"], D).double(), cos.double(), sin.double()), bits, dt)
        v = _encode(_heads(x["v"], D).double(), bits, dt)
        return q, _decode(*k, bits).to(dt), _decode(*v, bits).to(dt)
    if case["op"] == "read":
        return _decode(*state["k"], bits).to(dt), _decode(*state["v"], bits).to(dt)
    B, H, Hkv, n = case["batch"], case["heads"], case["kv_heads"], case["new"]
    k, v = _decode(*state["k"], bits), _decode(*state["v"], bits)
    q = _heads(x["q"], D).float().reshape(B, Hkv, (H // Hkv) * n, D)
    s = torch.matmul(q, k.transpose(2, 3)).view(B, Hkv, H // Hkv, n, -1) / math.sqrt(D)
    s = s.masked_fill(~x["mask"][:, None, None], -math.inf)
    p = torch.exp(s - s.amax(dim=-1, keepdim=True))
    out = torch.matmul(p.view(B, Hkv, (H // Hkv) * n, -1), v) / p.sum(dim=-1).view(B, Hkv, -1, 1)
    return out.view(B, H, n, D).transpose(1, 2).reshape(B, n, H * D).to(dt)


# ---- the framework's calls -----------------------------------------------------------------------

def _own_state(case, x):
    attention, kv_cache = _package()
    cache = kv_cache.Cache(case["batch"], case["prev"] + case["new"], 1, case["kv_heads"], case["dim"],
                           _DTYPES[case["dtype"]], torch.device("cuda"), bits=case["bits"])
    views = cache.sliced[0]
    state = {"case": case, "x": x, "cache": cache, "views": views}
    if case["op"] != "append":
        for view, rows in zip(views, (x["k"], x["v"])):
            view.append(_heads(rows, case["dim"]))
    if case["op"] == "attend":
        state["q"] = _heads(x["q"], case["dim"])
        state["prepared"] = attention.prepare(x["mask"], n_heads=case["heads"])
    return state


def _own(state):
    attention, kv_cache = _package()
    case, x = state["case"], state["x"]
    key_view, value_view = state["views"]
    if case["op"] == "append":
        state["cache"].set_length(case["prev"])
        q, _, _ = kv_cache.rope_append(x["q"], x["k"], x["v"], x["cos"], x["sin"], x["position_ids"], state["views"])
        return q, key_view.slice(case["prev"]), value_view.slice(case["prev"])
    if case["op"] == "read":
        return key_view.slice(0), value_view.slice(0)
    return attention.masked_attention(state["q"], key_view.rows(), value_view.rows(), state["prepared"])


# ---- interface -----------------------------------------------------------------------------------

def prepare(case, seed):
    x = inputs(case, seed)
    if own:
        return _own_state(case, x)
    state = {"case": case, "x": x}
    if case["op"] != "append":
        dt, D = _DTYPES[case["dtype"]], case["dim"]
        for name in ("k", "v"):
            state[name] = _encode(_heads(x[name], D).double(), case["bits"], dt)
    return state


def run(state):
    return _own(state) if own else _plain(state)


def _attended(case):
    """(keys of the batch that some query attends to, (query, key) pairs), without the seed: ragged
    rows counted at the mean of their padding."""
    B, n, prev = case["batch"], case["new"], case["prev"]
    pads = ((prev if prev else n) * 3 // 4) / 2 * (B - 1) if case["ragged"] else 0
    keys = B * (prev + n) - pads
    if case["mask"] == "prompt":
        pairs = B * n * (n + 1) / 2 - pads * n / 2
    else:
        pairs = n * (B * prev - pads) + B * n * min(n, 8)
    return keys, pairs


def work(case):
    B, n, D, H, Hkv = case["batch"], case["new"], case["dim"], case["heads"], case["kv_heads"]
    es = _DTYPES[case["dtype"]].itemsize
    record = D * case["bits"] // 8 + D // _BLOCK
    if case["op"] == "append":
        rows = B * n
        table = 2 * min(case["prev"] + n, rows) * D * es
        moved = (2 * H + 2 * Hkv) * D * es + 2 * Hkv * (2 * record + D * es)
        return {"bytes": rows * moved + table + 8 * rows, "flops": rows * (H + Hkv) * D * 3 + rows * 2 * Hkv * D * 4}
    if case["op"] == "read":
        rows = 2 * B * Hkv * case["prev"]
        return {"bytes": rows * (record + D * es), "flops": rows * D}
    keys, pairs = _attended(case)
    bits = B * n * ((case["prev"] + n + 63) // 64) * 8
    return {"bytes": int(2 * Hkv * keys * record + 2 * B * n * H * D * es + bits), "flops": int(4 * H * D * pairs)}


# ---- the definition in 64 bits -------------------------------------------------------------------

def _held(x, bits, dtype):
    """What the cache holds for float64 x (..., D): nearest point of the block's grid."""
    if bits == 4:
        grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    else:
        grid = [(c % 8) * 2.0 ** -9 if c < 8 else (8 + c % 8) * 2.0 ** (c // 8 - 10) for c in range(127)]
    grid = torch.tensor(grid, dtype=torch.float64, device=x.device)
    top = 7.0 if bits == 4 else 464.0
    lo, hi = _exponent_range(bits, dtype)
    y = x.unflatten(-1, (-1, _BLOCK))
    amax = y.abs().amax(dim=-1, keepdim=True)
    e = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -400) / top))
    power = torch.tensor([2.0 ** i for i in range(-500, 500)], dtype=torch.float64, device=x.device)
    two = lambda i: power[i.long() + 500]
    for _ in range(2):  # (the logarithm may be off by one next to a power of two)
        e = torch.where(amax > top * two(e), e + 1, e)
        e = torch.where(amax <= top * two(e - 1), e - 1, e)
    unit = two(e.clamp(lo, hi))
    mag = y.abs() / unit
    below = (torch.searchsorted(grid, mag.contiguous(), right=True) - 1).clamp(max=len(grid) - 2)
    a, b = grid[below], grid[below + 1]
    up = (mag - a > b - mag) | ((mag - a == b - mag) & (below % 2 == 1))
    return (torch.where(up, b, a) * unit * torch.sign(y)).flatten(-2)


def exact(case, seed):
    x = inputs(case, seed)
    dt, D, bits = _DTYPES[case["dtype"]], case["dim"], case["bits"]
    if case["op"] == "append":
        cos = x["cos"].double()[x["position_ids"]][:, None]
        sin = x["sin"].double()[x["position_ids"]][:, None]

        def turned(t):
            t = _heads(t, D).double()
            a, b = t[..., : D // 2], t[..., D // 2 :]
            return torch.cat((a * cos[..., : D // 2] - b * sin[..., : D // 2],
                              b * cos[..., D // 2 :] + a * sin[..., D // 2 :]), dim=-1)

        return turned(x["q"]), _held(turned(x["k"]), bits, dt), _held(_heads(x["v"], D).double(), bits, dt)
    k, v = _held(_heads(x["k"], D).double(), bits, dt), _held(_heads(x["v"], D).double(), bits, dt)
    if case["op"] == "read":
        return k, v
    B, H, Hkv, n = case["batch"], case["heads"], case["kv_heads"], case["new"]
    q = _heads(x["q"], D).double()
    out = torch.empty((B, n, H, D), dtype=torch.float64, device="cuda")
    for b in range(B):
        for h in range(H):
            s = (q[b, h] @ k[b, h // (H // Hkv)].T) * D ** -0.5
            s[~x["mask"][b]] = -math.inf
            out[b, :, h] = torch.softmax(s, dim=-1) @ v[b, h // (H // Hkv)]
    return out.view(B, n, H * D)
