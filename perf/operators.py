"""Timed cases of the paged 8-bit KV cache: the append that fills it and the attention that reads it.

``own`` false: plain torch in 32 bits.  ``own`` true: the calls a program makes of the module
(yk_kv_append, yk_attention_e4m3 through ``yanaiengine_b200.abi``).

Page layout, as in every KV pool of the module: [block][layer][K|V][kv head][16 slots][head_dim].  An e4m3
pool holds codes of 8 bits and one scale byte for each (block, layer, K|V, kv head): value = code * 2^(byte - 127),
byte in 67..187; the append picks the smallest exponent whose largest finite code (448) covers the block.
"""
import math
import random

import torch

own = False

PAGE = 16
LAYERS = 2  # layers of every pool here; the calls use layer 1
BIAS, E_MIN, E_MAX = 127, -60, 60
WORKSPACE = 24 << 20  # bytes a program keeps for the attention's partial results

_DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def listed():
    def append(name, **kw):
        return dict(dict(name=name, op="append", src="float32", dst="bfloat16", cache="e4m3", heads=32, kv_heads=8,
                         head_dim=128, norm=True, rope=True), **kw)

    def attention(name, **kw):
        return dict(dict(name=name, op="attention", dtype="bfloat16", heads=32, kv_heads=8, head_dim=128, window=0,
                         cap=0.0), **kw)

    return [
        # one sequence decoding: the projections of one token, appended mid-page
        append("append_one_token", seqs=1, new=1, ctx_lo=600, ctx_hi=600),
        # the verify step of 32 sequences with 5 drafts each (the benchmark's target shape), fp32 GEMM results
        append("append_verify", seqs=32, new=6, ctx_lo=512, ctx_hi=2048),
        # ragged prompts of a fresh batch, bf16 projections
        append("append_prompts", src="bfloat16", seqs=7, new=1171, ctx_lo=1171, ctx_hi=3000),
        # a verify step of a head_dim 256 model without per-head norms
        append("append_wide_heads", seqs=64, new=5, ctx_lo=2048, ctx_hi=8192, heads=16, head_dim=256, norm=False),
        # per-head norms in front of an ordinary bf16 pool
        append("append_bf16_pool", cache="bfloat16", seqs=32, new=64, ctx_lo=64, ctx_hi=2048),
        # one sequence decoding
        attention("attend_one_token", seqs=1, new=1, ctx_lo=600, ctx_hi=600),
        # the draft model's decode step (1B shape)
        attention("attend_draft_decode", seqs=32, new=1, ctx_lo=512, ctx_hi=2048, head_dim=64),
        # the verify step of the benchmark's target shape
        attention("attend_verify", seqs=32, new=6, ctx_lo=512, ctx_hi=2048),
        # one long conversation, single tokens
        attention("attend_long_decode", seqs=1, new=1, ctx_lo=131000, ctx_hi=131000),
        # verify over long contexts, soft-capped scores, head_dim 256 (the 9B shape's global layers)
        attention("attend_capped_verify", seqs=64, new=5, ctx_lo=2048, ctx_hi=8192, heads=16, head_dim=256, cap=50.0),
        # a prompt chunk attending to itself and to what was cached before it
        attention("attend_prompt", seqs=3, new=1500, ctx_lo=1500, ctx_hi=5000),
        # the fp32 models' verify, sliding window
        attention("attend_fp32_window", dtype="float32", seqs=9, new=5, ctx_lo=300, ctx_hi=1900, heads=12, kv_heads=4,
                  head_dim=64, window=333),
    ]


def draw(rng):
    while True:
        case = _any(rng)
        w = work(case)
        if w["flops"] <= 2.0e11 and w["bytes"] <= 1.3e9:  # no more than the largest listed ones
            return case


def _any(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    dh = rng.choice([64, 128, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 8])
    if rng.random() < 0.4:
        new = rng.choice([1, rng.randint(2, 9), log(2, 1200)])
        seqs = min(log(1, 96), max(1, 9000 // new))
        hi = new + log(1, 4000)
        f32 = rng.random() < 0.3
        return dict(op="append", src="float32" if f32 or rng.random() < 0.5 else "bfloat16",
                    dst="float32" if f32 else "bfloat16",
                    cache=rng.choice(["e4m3", "e4m3", "e4m3", "float32" if f32 else "bfloat16"]), heads=heads,
                    kv_heads=kv, head_dim=dh, norm=rng.random() < 0.7, rope=rng.random() < 0.9, seqs=seqs, new=new,
                    ctx_lo=rng.randint(new, hi), ctx_hi=hi)
    kind = rng.random()
    new = 1 if kind < 0.35 else rng.randint(2, 9) if kind < 0.75 else log(10, 1200)
    seqs = log(1, 64) if new < 10 else log(1, 4)
    hi = new + log(1, min(120000, 300000 // seqs) if new < 10 else 4000)
    return dict(op="attention", dtype="float32" if rng.random() < 0.25 else "bfloat16", heads=heads, kv_heads=kv,
                head_dim=dh, window=rng.choice([0, 0, log(1, 4096)]), cap=rng.choice([0.0, 0.0, 30.0]), seqs=seqs,
                new=new, ctx_lo=rng.randint(new, hi), ctx_hi=hi)


def _lengths(case):
    """(new tokens, length after them) of each sequence: set by the case alone, spread over its range."""
    spread = [(b * 0.6180339887498949) % 1.0 for b in range(case["seqs"])]
    ctx = [case["ctx_hi"] - int(f * (case["ctx_hi"] - case["ctx_lo"] + 1)) for f in spread]
    # every third sequence of a ragged batch brings fewer new tokens
    new = [case["new"] if b % 3 or case["seqs"] == 1 else max(1, case["new"] - case["new"] // 3)
           for b in range(case["seqs"])]
    return [min(n, c) for n, c in zip(new, ctx)], [max(c, 1) for c in ctx]


def _visible(case):
    """(query, key) pairs that attend, and keys that any query of its sequence reads."""
    pairs = keys = 0
    w = case["window"]
    for n, c in zip(*_lengths(case)):
        for p in range(c - n, c):
            pairs += p + 1 if w <= 0 else min(p + 1, w)
        keys += c if w <= 0 else min(c, w + n - 1)
    return pairs, keys


def work(case):
    H, G, dh = case["heads"], case["kv_heads"], case["head_dim"]
    new, ctx = _lengths(case)
    T = sum(new)
    if case["op"] == "append":
        src, dst = _DT[case["src"]].itemsize, _DT[case["dst"]].itemsize
        cell = 1 if case["cache"] == "e4m3" else _DT[case["cache"]].itemsize
        pages = sum((c + 15) // 16 - (c - n) // 16 for n, c in zip(new, ctx))
        b = T * ((H + 2 * G) * dh * src + H * dh * dst + 2 * G * dh * cell + 4)
        b += T * dh * 4 if case["rope"] else 0
        b += 2 * dh * 4 if case["norm"] else 0
        b += pages * 2 * G if case["cache"] == "e4m3" else 0
        return {"bytes": b, "flops": T * dh * ((H + G) * (4 * case["norm"] + 3 * case["rope"]) + 2 * G * 3)}
    pairs, keys = _visible(case)
    es = _DT[case["dtype"]].itemsize
    return {"bytes": keys * 2 * G * dh + keys // 16 * (2 * G + 4) + 2 * T * H * dh * es + 12 * len(new),
            "flops": 4 * pairs * H * dh}


def _scale_exponent(amax):
    """Smallest e with amax <= 448 * 2^e, in E_MIN..E_MAX."""
    m, e = torch.frexp(amax)  # amax = m * 2^e, 0.5 <= m < 1
    e = e - 9 + (m > 0.875).to(e.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, E_MIN)).clamp(E_MIN, E_MAX)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed * 2 + 1)
    H, G, dh = case["heads"], case["kv_heads"], case["head_dim"]
    new, ctx = _lengths(case)
    B, T = len(new), sum(new)
    need = [(c + PAGE - 1) // PAGE for c in ctx]
    blocks = sum(need) + 3
    order = list(range(blocks))
    random.Random(seed).shuffle(order)  # a pool in use: pages lie anywhere
    width = max(need)
    rows, at = [], 0
    for k in need:
        rows.append(order[at:at + k] + [0] * (width - k))
        at += k
    tables = torch.tensor(rows, dtype=torch.int32)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    pos = torch.cat([torch.arange(c - n, c) for n, c in zip(new, ctx)])
    seq = torch.repeat_interleave(torch.arange(B), torch.tensor(new))
    slots = tables[seq, pos // PAGE] * PAGE + (pos % PAGE).to(torch.int32)
    s = dict(case=dict(case), T=T, B=B, longest=max(ctx), most=max(new), blocks=blocks, tables=tables.to(dev),
             starts=torch.tensor(starts, dtype=torch.int32, device=dev),
             ctx=torch.tensor(ctx, dtype=torch.int32, device=dev), slots=slots.to(torch.int32).to(dev),
             pos=pos.to(dev), err=torch.zeros(1, dtype=torch.int32, device=dev))
    # what the cache holds: channels of unequal size, blocks of unequal scale
    shape = (blocks, LAYERS, 2, G, PAGE, dh)
    cache = case.get("cache", "e4m3")
    gain = torch.rand(1, 1, 2, G, 1, dh, generator=g, device=dev) * 1.5 + 0.25
    size = torch.exp2(torch.randn(blocks, 1, 2, G, 1, 1, generator=g, device=dev)) if cache == "e4m3" else 1.0
    held = torch.randn(shape, generator=g, device=dev, dtype=torch.bfloat16)
    held.mul_(gain.to(torch.bfloat16))
    if cache == "e4m3":
        held.mul_(size.to(torch.bfloat16))
        e = _scale_exponent(held.abs().amax((4, 5)).float())
        held.mul_(torch.exp2(-e.float())[..., None, None].to(torch.bfloat16))
        s["pool"] = held.to(torch.float8_e4m3fn).view(torch.uint8)
        s["scales"] = (e + BIAS).to(torch.uint8)
    else:
        s["pool"], s["scales"] = held.to(_DT[cache]), None
    del held
    if case["op"] == "append":
        raw = torch.randn(T, (H + 2 * G) * dh, generator=g, device=dev)
        raw *= torch.rand(1, (H + 2 * G) * dh, generator=g, device=dev) * 2 + 0.1
        s["qkv"] = raw.to(_DT[case["src"]])
        s["q"] = torch.zeros(T, H, dh, dtype=_DT[case["dst"]], device=dev)
        s["q_gain"] = torch.rand(dh, generator=g, device=dev) + 0.5 if case["norm"] else None
        s["k_gain"] = torch.rand(dh, generator=g, device=dev) + 0.5 if case["norm"] else None
        s["eps"] = 1e-5
        if case["rope"]:  # (cos, sin) of the step's tokens, one table for every layer
            freq = 500000.0 ** (-torch.arange(0, dh, 2, dtype=torch.float64, device=dev) / dh)
            ang = s["pos"].double()[:, None] * freq
            s["rope"] = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
        else:
            s["rope"] = None
    else:
        dt = _DT[case["dtype"]]
        s["q"] = (torch.randn(T, H, dh, generator=g, device=dev) * 1.3).to(dt)
        s["out"] = torch.zeros(T, H, dh, dtype=dt, device=dev)
        s["workspace"] = torch.zeros(WORKSPACE, dtype=torch.uint8, device=dev)
    return s


def run(s):
    if own:
        return _own_append(s) if s["case"]["op"] == "append" else _own_attention(s)
    return _plain_append(s) if s["case"]["op"] == "append" else _plain_attention(s)


def _append_outputs(s):
    if s["scales"] is None:
        return {"q": s["q"], "cache": s["pool"]}
    # 8-bit cells and scale bytes as the numbers they stand for
    return {"q": s["q"], "cache": s["pool"].view(torch.float8_e4m3fn), "scales": s["scales"].view(torch.float8_e8m0fnu)}


def _own_append(s):
    from yanaiengine_b200 import abi

    c = s["case"]
    abi.kv_append(s["pool"], s["scales"], 1, s["qkv"], s["q"], s["slots"], s["rope"], s["q_gain"], s["k_gain"], s["eps"],
                  s["err"], c["heads"])
    return _append_outputs(s)


def _own_attention(s):
    from yanaiengine_b200 import abi

    c = s["case"]
    abi.attention_e4m3(s["q"], s["out"], s["pool"], s["scales"], 1, s["starts"], s["ctx"], s["tables"], s["workspace"],
                       s["err"], max_new=s["most"], window=c["window"], cap=c["cap"])
    return {"out": s["out"]}


def _plain_append(s):
    c = s["case"]
    H, G, dh, T = c["heads"], c["kv_heads"], c["head_dim"], s["T"]
    x = s["qkv"].float().view(T, H + 2 * G, dh)
    q, k, v = x[:, :H], x[:, H:H + G], x[:, H + G:]
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + s["eps"]) * s["q_gain"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + s["eps"]) * s["k_gain"]
    if c["rope"]:
        co, si = s["rope"][:, None, :, 0], s["rope"][:, None, :, 1]

        def turn(t):
            a, b = t[..., 0::2], t[..., 1::2]
            return torch.stack([a * co - b * si, a * si + b * co], -1).flatten(-2)

        q, k = turn(q), turn(k)
    s["q"].copy_(q)
    kv = torch.stack([k, v], 1)  # [T, K|V, kv head, dh]
    block, at = (s["slots"] // PAGE).long(), (s["slots"] % PAGE).long()
    if s["scales"] is None:
        s["pool"][block, 1, :, :, at] = kv.to(s["pool"].dtype)
        return _append_outputs(s)
    # one exponent for each touched block: it never shrinks while older tokens of the block stay
    first = torch.ones(T, dtype=torch.bool, device=block.device)
    first[1:] = block[1:] != block[:-1]
    group = first.cumsum(0) - 1
    cells = torch.zeros(T, 2, G, device=block.device)
    cells.index_reduce_(0, group, kv.abs().amax(-1), "amax")
    want = _scale_exponent(cells)
    lead = torch.zeros(T, dtype=torch.long, device=block.device).index_add_(0, group, torch.where(first, block, 0))
    kept = torch.zeros(T, dtype=torch.long, device=block.device).index_add_(0, group, torch.where(first, at, 0))
    had = s["scales"][lead, 1].to(torch.int32) - BIAS
    e = torch.where(kept[:, None, None] > 0, torch.maximum(want, had), want)
    # older tokens of the block move to the new exponent
    pages = s["pool"][lead, 1].view(torch.float8_e4m3fn).float()
    moved = (pages * torch.exp2((had - e).float())[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    old = torch.arange(PAGE, device=block.device) < kept[:, None]
    whole = torch.where(old[:, None, None, :, None], moved, s["pool"][lead, 1])
    code = (kv * torch.exp2(-e[group].float())[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    whole[group, :, :, at] = code
    # unused groups at the end repeat the last used one
    used = torch.minimum(torch.arange(T, device=block.device), group[-1])
    s["pool"][lead[used], 1] = whole[used]
    s["scales"][lead[used], 1] = (e[used] + BIAS).to(torch.uint8)
    return _append_outputs(s)


def _plain_attention(s):
    c = s["case"]
    H, G, dh, T, B = c["heads"], c["kv_heads"], c["head_dim"], s["T"], s["B"]
    N, S = s["most"], s["longest"]
    tables = s["tables"].long()
    scale = torch.exp2(s["scales"][:, 1].clamp(BIAS + E_MIN, BIAS + E_MAX).float() - BIAS)[tables]
    held = s["pool"][:, 1][tables].view(torch.float8_e4m3fn).float() * scale[..., None, None]
    held = held.permute(2, 0, 3, 1, 4, 5).reshape(2, B, G, -1, dh)[:, :, :, :S]  # [K|V, B, kv head, keys, dh]
    starts, ctx = s["starts"].long(), s["ctx"].long()
    new = starts[1:] - starts[:-1]
    token = torch.arange(T, device=tables.device)
    seq = torch.searchsorted(starts[1:], token, right=True)
    row = token - starts[seq]
    q = torch.zeros(B, N, H, dh, device=tables.device)
    q[seq, row] = s["q"].float()
    q = q.view(B, N, G, H // G, dh).permute(0, 2, 1, 3, 4).reshape(B, G, N * (H // G), dh)
    x = torch.matmul(q, held[0].transpose(-1, -2)) * (1.0 / math.sqrt(dh))
    if c["cap"] > 0:
        x = c["cap"] * torch.tanh(x / c["cap"])
    at = (ctx - new)[:, None] + torch.arange(N, device=tables.device)  # [B, N] positions
    key = torch.arange(S, device=tables.device)
    see = key <= at[..., None]
    if c["window"] > 0:
        see = see & (at[..., None] - key < c["window"])
    see = see[:, None, :, None].expand(B, 1, N, H // G, S).reshape(B, 1, N * (H // G), S)
    x = x.masked_fill(~see, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min))
    y = torch.matmul(x, held[1]) / x.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
    y = y.view(B, G, N, H // G, dh).permute(0, 2, 1, 3, 4).reshape(B, N, H, dh)
    s["out"].copy_(y[seq, row])
    return {"out": s["out"]}


def exact(case, seed):
    s = prepare(case, seed)
    H, G, dh = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        q = s["qkv"].double()[:, :H * dh].reshape(s["T"], H, dh)
        if case["norm"]:
            q = q / (q.pow(2).sum(-1, keepdim=True) / dh + s["eps"]).sqrt() * s["q_gain"].double()
        if case["rope"]:
            z = torch.view_as_complex(q.reshape(s["T"], H, dh // 2, 2).contiguous())
            q = torch.view_as_real(z * torch.view_as_complex(s["rope"].double())[:, None]).reshape(s["T"], H, dh)
        return {"q": q, "cache": None, "scales": None} if s["scales"] is not None else {"q": q, "cache": None}
    out = torch.zeros(s["T"], H, dh, dtype=torch.float64, device="cuda")
    t = 0
    for b, (n, c) in enumerate(zip(*_lengths(case))):
        ids = s["tables"][b, :(c + PAGE - 1) // PAGE].long()
        page = s["pool"][ids, 1].view(torch.float8_e4m3fn).double()
        page = page * 2.0 ** (s["scales"][ids, 1].double() - BIAS)[..., None, None]
        # [page, K|V, kv head, slot, dh] -> [K|V, kv head, key, dh]
        page = page.permute(1, 2, 0, 3, 4).reshape(2, G, -1, dh)[:, :, :c]
        for lo in range(0, n, 256):  # a few hundred queries at a time
            hi = min(n, lo + 256)
            p = torch.arange(c - n + lo, c - n + hi, device="cuda")[:, None]
            j = torch.arange(c, device="cuda")[None]
            off = j > p
            if case["window"] > 0:
                off |= p - j >= case["window"]
            for h in range(G):
                w = H // G
                qq = s["q"][t + lo:t + hi, h * w:(h + 1) * w].double().transpose(0, 1)
                x = qq @ page[0, h].T / dh ** 0.5
                if case["cap"] > 0:
                    x = torch.tanh(x / case["cap"]) * case["cap"]
                x[:, off] = -math.inf
                out[t + lo:t + hi, h * w:(h + 1) * w] = (torch.softmax(x, -1) @ page[1, h]).transpose(0, 1)
        t += n
    return {"out": out}
