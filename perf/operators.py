"""What the LLM backbone's rotary, append-attention and tree-verification
operators are measured on: the cases, their inputs, their plain forms and their
definitions in 64 bits.

Shapes come from the backbone's own configuration (12 query heads over 2 kv
heads, head dim 128, 256-position blocks), the FM head's (16 heads of 64,
16-row pages), and generic grouped-query ones.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "f32": 4}
THETA = 1.0e6
ORIGINAL = 32768      # positions a scaled rotary was first made for


# ------------------------------------------------------------------ cases
def _rotary(name, tokens, heads, kv_heads, dim, rot, layout, scaling, dtype, store, far, block=256):
    return {"name": name, "op": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "rot": rot, "layout": layout, "scaling": scaling, "dtype": dtype,
            "store": store, "far": far, "block": block}


def _verify(name, seqs, tree_lo, tree_hi, prior_lo, prior_hi, heads, kv_heads, dim, block, dtype,
            softcap=0.0):
    return {"name": name, "op": "verify", "seqs": seqs, "new_lo": tree_lo, "new_hi": tree_hi,
            "prior_lo": prior_lo, "prior_hi": prior_hi, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "block": block, "dtype": dtype, "softcap": softcap}


def _append(name, seqs, new_lo, new_hi, prior_lo, prior_hi, heads, kv_heads, dim, block, dtype,
            softcap=0.0, slopes=False, window=0, prefix=False, docs=False):
    return {"name": name, "op": "append", "seqs": seqs, "new_lo": new_lo, "new_hi": new_hi,
            "prior_lo": prior_lo, "prior_hi": prior_hi, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "block": block, "dtype": dtype, "softcap": softcap, "slopes": slopes,
            "window": window, "prefix": prefix, "docs": docs}


def listed():
    return [
        # one request generating alone: the smallest call of the rotary and cache store
        _rotary("rotary_one", 1, 12, 2, 128, 128, "half", "none", "bf16", True, 4096),
        # one decode step of the benchmark's 64 requests
        _rotary("rotary_step", 64, 12, 2, 128, 128, "half", "none", "bf16", True, 4096),
        # a long prompt's prefill past the trained length, stored into the paged cache
        _rotary("rotary_prefill", 16384, 12, 2, 128, 128, "half", "yarn", "bf16", True, 131072),
        # interleaved pairs over half of each head in fp32, no store
        _rotary("rotary_pairs", 8191, 16, 16, 64, 32, "interleaved", "bands", "f32", False, 1 << 20),
        # one request with a few drafted tokens: latency
        _verify("verify_one", 1, 8, 8, 300, 300, 12, 2, 128, 256, "bf16"),
        # the benchmark's batch, drafts of up to 16 tokens, ragged histories
        _verify("verify_batch", 64, 1, 16, 0, 2000, 12, 2, 128, 256, "bf16"),
        # wide trees over small pages, fp16, capped scores
        _verify("verify_wide", 16, 33, 63, 3000, 9000, 16, 4, 64, 16, "fp16", softcap=30.0),
        # few requests with very long caches: the key axis has to be split
        _verify("verify_long", 4, 25, 25, 40000, 60001, 12, 2, 128, 256, "bf16"),
        # single tokens under a cap and a sliding window: the serving form
        _append("append_step", 64, 1, 1, 0, 4000, 12, 2, 128, 256, "bf16", softcap=50.0, window=1024),
        # chunked prefill of a mixed batch; a bidirectional prompt prefix
        _append("append_chunks", 24, 1, 384, 0, 1100, 12, 2, 128, 256, "bf16", prefix=True),
        # packed documents with a distance bias, fp16, small pages
        _append("append_docs", 6, 700, 1300, 0, 500, 16, 16, 64, 16, "fp16", slopes=True, docs=True),
        # a long prompt's second half: compute-bound
        _append("append_long", 1, 8192, 8192, 8192, 8192, 12, 2, 128, 256, "bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("rotary", "verify", "append"))
    if op == "rotary":
        kv = rng.choice((1, 2, 4, 8))
        heads, dim = kv * rng.choice((1, 2, 4, 6)), rng.choice((64, 128))
        rot = dim if rng.random() < 0.5 else rng.choice((dim // 4, dim // 2, dim))
        c = _rotary("", _log(rng, 1, 16384), heads, kv, dim, rot, rng.choice(("half", "interleaved")),
                    rng.choice(("none", "linear", "ntk", "bands", "yarn")),
                    rng.choice(("bf16", "fp16", "f32")), rng.random() < 0.6, _log(rng, 128, 1 << 20),
                    rng.choice((16, 64, 256)))
        while c["tokens"] * heads * dim * BYTES[c["dtype"]] > 16384 * 16 * 128 * 2:
            c["tokens"] = max(1, c["tokens"] // 2)
    else:
        kv = rng.choice((1, 2, 4, 8))
        heads = kv * rng.choice((1, 2, 3, 4, 6, 8))
        dim, block = rng.choice((64, 128)), rng.choice((16, 48, 64, 256))
        dtype = rng.choice(("bf16", "fp16"))
        seqs = _log(rng, 1, 64)
        prior = 0 if rng.random() < 0.2 else _log(rng, 1, 60000)
        if op == "verify":
            hi = _log(rng, 1, 64)
            c = _verify("", seqs, rng.randint(1, hi), hi, rng.randint(0, prior), prior, heads, kv, dim,
                        block, dtype, rng.choice((0.0, 0.0, 30.0)))
        else:
            hi = _log(rng, 1, 8192)
            c = _append("", seqs, rng.randint(1, hi), hi, rng.randint(0, prior), prior, heads, kv, dim,
                        block, dtype, rng.choice((0.0, 0.0, 50.0)), rng.random() < 0.3,
                        rng.choice((0, 0, _log(rng, 1, 4096))), rng.random() < 0.3, rng.random() < 0.3)
        # no more than the largest listed case
        while c["seqs"] * heads * c["new_hi"] * (c["new_hi"] + c["prior_hi"]) > 5e8 and c["seqs"] > 1:
            c["seqs"] //= 2
        while heads * c["new_hi"] * (c["new_hi"] + c["prior_hi"]) > 1e9:
            c["new_hi"] = max(1, c["new_hi"] // 2)
            c["new_lo"] = min(c["new_lo"], c["new_hi"])
        while c["seqs"] * kv * dim * (c["new_hi"] + c["prior_hi"]) > 1e8:
            c["prior_hi"] //= 2
            c["prior_lo"] = min(c["prior_lo"], c["prior_hi"])
    del c["name"]
    return c


# ------------------------------------------------------------------ lengths
def _lengths(c):
    """New tokens and prior positions of each sequence: the case's, whatever the seed."""
    r = random.Random("%(seqs)d %(new_lo)d %(new_hi)d %(prior_lo)d %(prior_hi)d" % c)
    new = [r.randint(c["new_lo"], c["new_hi"]) for _ in range(c["seqs"])]
    prior = [r.randint(c["prior_lo"], c["prior_hi"]) for _ in range(c["seqs"])]
    new[-1], prior[0] = c["new_hi"], c["prior_hi"]
    return new, prior


def _intervals(c):
    """Per sequence the prefix length, and per token the first key of its document."""
    new, prior = _lengths(c)
    r = random.Random(len(new) + sum(new))
    prefix = [r.randint(0, p + m) if c.get("prefix") else 0 for m, p in zip(new, prior)]
    first = []
    for m, p in zip(new, prior):
        cuts = sorted({0} | {r.randint(0, m + p - 1) for _ in range(3)}) if c.get("docs") else [0]
        at = 0
        for j in range(m):
            while at + 1 < len(cuts) and cuts[at + 1] <= p + j:
                at += 1
            first.append(cuts[at])
    return prefix, first


def _span(c, p, j, m, prefix, first):
    """[lo, hi): the keys that new token j of a sequence may see."""
    lo, hi = first, max(p + j + 1, min(prefix, p + m))
    if c.get("window"):
        lo = max(lo, p + j + 1 - c["window"])
    return lo, hi


# ------------------------------------------------------------------ inputs
def _frequencies(c, dtype=torch.float64):
    """Radians a position of each rotated pair, and the factor on cos and sin."""
    rot, kind, f = c["rot"], c["scaling"], 4.0
    i = torch.arange(0, rot, 2, dtype=dtype)
    theta = THETA * f ** (rot / (rot - 2)) if kind == "ntk" else THETA
    inv = theta ** (-i / rot)
    if kind == "linear":
        return inv / f, 1.0
    if kind == "bands":     # short waves as they are, long ones stretched, a ramp between
        smooth = ((ORIGINAL * inv / (2 * math.pi) - 1.0) / 3.0).clamp(0, 1)
        return inv / f * (1 - smooth) + inv * smooth, 1.0
    if kind == "yarn":      # the ramp runs over the pairs' indices
        at = lambda turns: rot * math.log(ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(THETA))  # noqa: E731
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
        return inv / f * ramp + inv * (1 - ramp), 0.1 * math.log(f) + 1.0
    return inv, 1.0


def _inputs(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    dt, D, H, KVH, bs = DTYPES[c["dtype"]], c["dim"], c["heads"], c["kv_heads"], c["block"]
    randn = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    if c["op"] == "rotary":
        T = c["tokens"]
        # q, k and v as the packed projection leaves them: slices of one row
        qkv = (randn(T, (H + 2 * KVH) * D) * 2).to(dt)
        q, k, v = (t.view(T, -1, D) for t in qkv.split([H * D, KVH * D, KVH * D], dim=1))
        start = int(torch.randint(0, max(1, c["far"] - T), (1,), generator=cpu))
        st = {"q": q, "k": k, "v": v, "positions": torch.arange(start, start + T, dtype=torch.int32).to(DEV)}
        if c["store"]:
            blocks = -(-T // bs) + 2
            st["slots"] = torch.randperm(blocks * bs, generator=cpu)[:T].to(torch.int32).to(DEV)
            st["k_cache"] = torch.zeros(blocks, bs, KVH, D, dtype=dt, device=DEV)
            st["v_cache"] = torch.zeros(blocks, bs, KVH, D, dtype=dt, device=DEV)
        return st
    new, prior = _lengths(c)
    n, T = len(new), sum(new)
    ctx = [m + p for m, p in zip(new, prior)]
    need = [-(-x // bs) for x in ctx]
    blocks = sum(need) + 2
    order = torch.randperm(blocks, generator=cpu)
    table = torch.full((n, max(need)), -1, dtype=torch.int32)
    at = 0
    for i, b in enumerate(need):
        table[i, :b] = order[at:at + b].to(torch.int32)
        at += b
    q = (randn(T, H, D) * 2).to(dt)
    # keys share a direction, as trained heads' do; the values do not
    k_cache = (randn(blocks, bs, KVH, D) + 0.5 * randn(KVH, D)).to(dt)
    v_cache = randn(blocks, bs, KVH, D).to(dt)
    cu = [0]
    for m in new:
        cu.append(cu[-1] + m)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).to(DEV)  # noqa: E731
    st = {"q": q, "k_cache": k_cache, "v_cache": v_cache, "cu": i32(cu), "ctx": i32(ctx),
          "table": table.to(DEV), "M": max(new), "L": max(ctx)}
    if c["op"] == "verify":
        bits, r = [], random.Random(seed)
        for m in new:       # each drafted token continues one before it, or the history
            row = []
            for t in range(m):
                up = r.randint(max(-1, t - 4), t - 1)
                seen = (row[up] if up >= 0 else 0) | 1 << t
                row.append(seen)
            bits += [b - (1 << 64) if b >> 63 else b for b in row]
        st["tree"] = torch.tensor(bits, dtype=torch.int64).to(DEV)
        return st
    prefix, first = _intervals(c)
    st["prefix"] = i32(prefix) if c["prefix"] else None
    st["first"] = i32(first) if c["docs"] else None
    st["slopes"] = (torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)]).to(DEV)
                    if c["slopes"] else None)
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if own:
        c = case
        if c["op"] == "rotary":
            from nanovllm_dots_b200.llm_rotary import B200Rotary, RotaryScaling
            scaling = None if c["scaling"] == "none" else RotaryScaling(c["scaling"], 4.0, ORIGINAL)
            st["rotary"] = B200Rotary(c["dim"], theta=THETA, rot_dim=c["rot"], layout=c["layout"],
                                      scaling=scaling, device=DEV)
        else:
            from nanovllm_dots_b200.llm_append import B200AppendAttention
            st["attention"] = B200AppendAttention(
                c["heads"], c["dim"], c["dim"] ** -0.5, c["kv_heads"], max_tokens=st["q"].shape[0],
                max_seqs=c["seqs"], max_blocks=st["table"].shape[1], block_size=c["block"],
                dtype=DTYPES[c["dtype"]], softcap=c["softcap"], window=c.get("window", 0),
                slopes=st.get("slopes"), device=DEV)
    else:
        if case["op"] == "rotary":
            inv, factor = _frequencies(case)
            st["inv"], st["factor"] = inv.to(DEV), factor
    return st


# ------------------------------------------------------------------ plain forms
def _turn(x, cos, sin, rot, layout):
    """x [T, heads, D] with its first `rot` dims rotated, rounded once."""
    f = x.float()
    r, rest = f[..., :rot], f[..., rot:]
    cos, sin = cos[:, None], sin[:, None]
    if layout == "half":
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((r, rest), -1).to(x.dtype)


def _plain_rotary(st):
    c = st["case"]
    angle = st["positions"].double()[:, None] * st["inv"]
    cos, sin = (torch.cos(angle) * st["factor"]).float(), (torch.sin(angle) * st["factor"]).float()
    q = _turn(st["q"], cos, sin, c["rot"], c["layout"])
    if not c["store"]:
        return {"q": q}
    at = st["slots"].long()
    st["k_cache"].view(-1, c["kv_heads"], c["dim"])[at] = _turn(st["k"], cos, sin, c["rot"], c["layout"])
    st["v_cache"].view(-1, c["kv_heads"], c["dim"])[at] = st["v"]
    return {"q": q, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _plain_attention(st):
    c, q = st["case"], st["q"]
    H, KVH, D = c["heads"], c["kv_heads"], c["dim"]
    G, n, M, L = H // KVH, c["seqs"], st["M"], st["L"]
    cu, ctx = st["cu"].long(), st["ctx"].long()
    j, k = torch.arange(M, device=q.device), torch.arange(L, device=q.device)
    m = cu[1:] - cu[:-1]
    tok = (cu[:-1, None] + j).clamp(max=q.shape[0] - 1)             # [n, M]
    table = st["table"].long().clamp(min=0)
    K = st["k_cache"][table].view(n, -1, KVH, D)[:, :L].float().permute(0, 2, 3, 1)
    V = st["v_cache"][table].view(n, -1, KVH, D)[:, :L].float().permute(0, 2, 1, 3)
    Q = q[tok].float().view(n, M, KVH, G, D).permute(0, 2, 3, 1, 4).reshape(n, KVH, G * M, D)
    s = (Q @ K).view(n, KVH, G, M, L) * (D ** -0.5)
    if c["softcap"]:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    base = (ctx - m)[:, None]                                       # [n, 1]
    at = (base + j)[:, :, None]                                     # [n, M, 1]
    if c["op"] == "verify":
        d = (k - base).clamp(0, 63)[:, None, :]
        see = (k < base)[:, None, :] | ((st["tree"][tok][:, :, None] >> d) & 1).bool()
        see = see & (k < ctx[:, None])[:, None, :]
    else:
        see = k <= at
        if st["prefix"] is not None:
            see = see | (k < st["prefix"][:, None, None])
        see = see & (k < ctx[:, None, None])
        if c["window"]:
            see = see & (k > at - c["window"])
        if st["first"] is not None:
            see = see & (k >= st["first"][tok][:, :, None])
        if st["slopes"] is not None:
            s = s - st["slopes"].view(1, KVH, G, 1, 1) * (at - k).abs()[:, None, None].float()
    s = s.masked_fill(~see[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > float("-inf"), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    o = (p.view(n, KVH, G * M, L) @ V).view(n, KVH, G, M, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o.permute(0, 3, 1, 2, 4).reshape(n, M, H, D)
    # token t of the batch is row t - cu[seq] of its sequence
    t = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(cu[1:], t, right=True)
    return {"out": o[seq, t - cu[seq]].to(q.dtype)}


def run(state):
    if own:
        op = state["case"]["op"]
        if op == "rotary":
            if not state["case"]["store"]:
                return {"q": state["rotary"].rotate(state["q"], state["positions"])}
            q = state["rotary"].rotate_store(state["q"], state["k"], state["v"], state["positions"],
                                             state["slots"], state["k_cache"], state["v_cache"])
            return {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}
        if op == "verify":
            return {"out": state["attention"].verify(state["q"], state["k_cache"], state["v_cache"],
                                                     state["cu"], state["ctx"], state["table"],
                                                     state["tree"])}
        return {"out": state["attention"].append(state["q"], state["k_cache"], state["v_cache"],
                                                 state["cu"], state["ctx"], state["table"],
                                                 prefix_lens=state["prefix"],
                                                 first_keys=state["first"])}
    return _plain_rotary(state) if state["case"]["op"] == "rotary" else _plain_attention(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    D, H, KVH, e = c["dim"], c["heads"], c["kv_heads"], BYTES[c["dtype"]]
    if c["op"] == "rotary":
        T = c["tokens"]
        heads = H + 2 * KVH if c["store"] else H
        turned = H + KVH if c["store"] else H
        return {"bytes": T * (2 * heads * D * e + 8) + c["rot"] * 4, "flops": T * turned * c["rot"] * 3}
    new, prior = _lengths(c)
    pairs = keys = 0
    if c["op"] == "verify":
        for m, p in zip(new, prior):    # each token sees the history and, at the mean, half its path
            pairs += m * p + sum(min(t + 1, 1 + t // 3) for t in range(m))
            keys += m + p
    else:
        prefix, first = _intervals(c)
        t = 0
        for m, p, pre in zip(new, prior, prefix):
            a, b = m + p, 0
            for j in range(m):
                lo, hi = _span(c, p, j, m, pre, first[t])
                pairs += max(0, hi - lo)
                if hi > lo:
                    a, b = min(a, lo), max(b, hi)
                t += 1
            keys += max(0, b - a)
    T = sum(new)
    return {"bytes": 2 * T * H * D * e + 2 * keys * KVH * D * e + 8 * T,
            "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    c, st = case, _inputs(case, seed)
    D, H, KVH = c["dim"], c["heads"], c["kv_heads"]
    if c["op"] == "rotary":
        inv, factor = _frequencies(c)
        pos = st["positions"].double()
        unit = torch.polar(torch.full_like(pos, factor)[:, None].expand(-1, len(inv)).contiguous(),
                           pos[:, None] * inv.to(DEV))[:, None]

        def turned(x):
            x = x.double().clone()
            pair = (slice(0, c["rot"] // 2), slice(c["rot"] // 2, c["rot"]))
            if c["layout"] == "interleaved":
                pair = (slice(0, c["rot"], 2), slice(1, c["rot"], 2))
            z = torch.complex(x[..., pair[0]].contiguous(), x[..., pair[1]].contiguous()) * unit
            x[..., pair[0]], x[..., pair[1]] = z.real, z.imag
            return x

        if not c["store"]:
            return {"q": turned(st["q"])}
        kc, vc = st["k_cache"].double(), st["v_cache"].double()
        kc.view(-1, KVH, D).index_copy_(0, st["slots"].long(), turned(st["k"]))
        vc.view(-1, KVH, D).index_copy_(0, st["slots"].long(), st["v"].double())
        return {"q": turned(st["q"]), "k_cache": kc, "v_cache": vc}
    new, prior = _lengths(c)
    out = torch.zeros(sum(new), H, D, dtype=torch.float64, device=DEV)
    prefix, first = _intervals(c) if c["op"] == "append" else (None, None)
    table, t0 = st["table"].long().cpu(), 0
    for i, (m, p) in enumerate(zip(new, prior)):
        n = m + p
        key = torch.arange(n)
        rows = (table[i, key // c["block"]] * c["block"] + key % c["block"]).to(DEV)
        key = key.to(DEV)
        if c["op"] == "verify":
            tree = st["tree"][t0:t0 + m]
            bit = torch.bitwise_right_shift(tree[:, None], torch.arange(m, device=DEV)) & 1
            hidden = torch.cat((torch.zeros(m, p, dtype=torch.bool, device=DEV), bit == 0), 1)
        else:
            spans = [_span(c, p, j, m, prefix[i], first[t0 + j]) for j in range(m)]
            lo, hi = torch.tensor(spans, device=DEV).unbind(1)
            hidden = (key < lo[:, None]) | (key >= hi[:, None])
        for h in range(H):
            k = st["k_cache"].view(-1, KVH, D)[rows, h * KVH // H].double()
            v = st["v_cache"].view(-1, KVH, D)[rows, h * KVH // H].double()
            s = st["q"][t0:t0 + m, h].double() @ k.t() / math.sqrt(D)
            if c["softcap"]:
                s = (s / c["softcap"]).tanh_() * c["softcap"]
            if c["op"] == "append" and c["slopes"]:
                away = (torch.arange(p, n, device=DEV)[:, None] - key).abs()
                s -= float(st["slopes"][h]) * away.double()
            s.masked_fill_(hidden, float("-inf"))
            out[t0:t0 + m, h] = torch.nan_to_num(torch.softmax(s, 1), nan=0.0) @ v
        t0 += m
    return {"out": out}
