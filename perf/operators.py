"""The paged-cache operators whose speed is measured, through the framework's public entry points.

A server keeps the keys and values of many sequences in pages of one cache and steps them together:
`gsvk_op_paged_append` rotates the new tokens' queries and keys to their positions and writes keys and
values into the pages, `gsvk_op_attn_paged` lets the new tokens attend to what their sequences hold.
A step brings one token per sequence, a chunk of a prompt, a few drafted tokens, or a mix of these.

`listed` names the cases, `draw` makes more of the same ranges, `prepare` makes what a program holds
before a call, `run` is one call (in elementary torch operations, or with `own` on the framework's
kernels), `work` counts the bytes and operations it cannot do without, and `exact` computes the result
in 64 bits.
"""
import math
import os
import random
import sys

import torch

own = False   # set by the caller: the framework's kernels instead of the plain form

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- the cases ----------------------------------------------------------------------------
# B sequences, `ones` of them with one new token, the others with new_lo..new_hi; ctx_lo..ctx_hi keys
# before them; nh query heads of dim hd over nkv key/value heads; pages of `page` keys.

def _append(name, B, new, ctx, nh, nkv, hd, x, t, page, rot, style, ones=0):
    return {"name": name, "op": "append", "B": B, "ones": ones, "new_lo": new[0], "new_hi": new[1], "ctx_lo": ctx[0],
            "ctx_hi": ctx[1], "nh": nh, "nkv": nkv, "hd": hd, "x": x, "type": t, "page": page, "rot": rot, "style": style}


def _attn(name, B, new, ctx, nh, nkv, hd, t, page, ones=0, window=0, prefix=False):
    return {"name": name, "op": "attn", "B": B, "ones": ones, "new_lo": new[0], "new_hi": new[1], "ctx_lo": ctx[0],
            "ctx_hi": ctx[1], "nh": nh, "nkv": nkv, "hd": hd, "type": t, "page": page, "window": window,
            "prefix": prefix}


def listed():
    return [
        # one caller's next token, this framework's heads, fp32 projections: pure latency
        _append("append_step_b1", 1, (1, 1), (400, 400), 16, 16, 32, "f32", "f16", 16, 32, "pairs"),
        # a server's step: one token for each of 64 sequences, grouped heads
        _append("append_step_b64", 64, (1, 1), (100, 4000), 32, 8, 128, "bf16", "bf16", 16, 128, "halves"),
        # four long prompts of odd lengths, half of each head rotated
        _append("append_prompt_b4", 4, (3001, 4099), (0, 0), 32, 8, 128, "bf16", "bf16", 64, 64, "halves"),
        # one caller's next token over one spoken sentence, this framework's heads: latency
        _attn("step_b1", 1, (1, 1), (500, 500), 16, 16, 32, "f16", 16),
        # one layer of the benchmark's decode batch: 64 sequences of unequal length
        _attn("step_b64", 64, (1, 1), (255, 2047), 16, 16, 32, "f16", 32),
        # a server's step with grouped heads of 128 over contexts of 1 to 12 thousand keys
        _attn("step_b32_grouped", 32, (1, 1), (1000, 12000), 32, 8, 128, "bf16", 16),
        # two very long documents, one token each: the cache does not fit any on-chip memory
        _attn("step_b2_long", 2, (1, 1), (131070, 131070), 64, 8, 128, "bf16", 64),
        # five drafted tokens per sequence under a sliding window
        _attn("draft_b8_window", 8, (5, 5), (1700, 5000), 16, 4, 64, "f16", 16, window=1024),
        # this framework's prompts: text that sees itself in both directions, then causal codes
        _attn("prompt_b16_prefix", 16, (100, 400), (0, 0), 16, 16, 32, "f16", 32, prefix=True),
        # chunks of four long prompts
        _attn("chunk_b4", 4, (512, 512), (1000, 7600), 32, 8, 128, "bf16", 16),
        # a step of a server that mixes two chunks of prompts with 22 sequences' next tokens
        _attn("mixed_b24", 24, (700, 1000), (200, 4000), 32, 8, 128, "bf16", 16, ones=22),
        # a whole prompt at once, the largest product
        _attn("prompt_b1_8191", 1, (8191, 8191), (0, 0), 32, 8, 128, "bf16", 64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    w = work(c)
    return w["bytes"] / 5e12, w["flops"] / 1e15


def draw(rng):
    nkv = rng.choice([1, 2, 4, 8, 16])
    heads = {"nkv": nkv, "nh": nkv * rng.choice([1, 1, 2, 4, 5, 8]), "hd": rng.choice([32, 64, 128])}
    page, t = rng.choice([16, 32, 64, 128]), rng.choice(["f16", "bf16"])
    form = rng.choice(["step", "draft", "chunk", "prompt", "mixed"])
    B = _log(rng, 1, 64) if form in ("step", "draft") else _log(rng, 2, 32) if form == "mixed" else _log(rng, 1, 16)
    new_hi = {"step": 1, "draft": rng.randint(2, 9)}.get(form) or _log(rng, 20, 4100)
    new_lo = new_hi if form in ("step", "draft") else rng.randint(max(1, new_hi // 3), new_hi)
    ctx_hi = 0 if form == "prompt" else _log(rng, 20, 60000 if form == "step" else 12000)
    ctx_lo = rng.randint(ctx_hi // 8, ctx_hi)
    ones = rng.randint(1, B - 1) if form == "mixed" else 0
    if rng.random() < 0.3:
        c = _append("", B, (new_lo, new_hi), (ctx_lo, ctx_hi), heads["nh"], nkv, heads["hd"],
                    rng.choice(["f32", t]), t, page, rng.choice([heads["hd"], heads["hd"], heads["hd"] // 2]),
                    rng.choice(["halves", "pairs"]), ones)
    else:
        prefix = form == "prompt" and rng.random() < 0.3
        c = _attn("", B, (new_lo, new_hi), (ctx_lo, ctx_hi), heads["nh"], nkv, heads["hd"], t, page, ones,
                  0 if prefix or rng.random() < 0.7 else _log(rng, 16, 2000), prefix)
    del c["name"]
    top = [max(v) for v in zip(*(_cost(x) for x in listed()))]
    while any(v > m for v, m in zip(_cost(c), top)) or (c["op"] == "attn" and _scores(c) > 3e9):
        # fewer sequences, then shorter ones: a drawn case costs no more than the largest listed one
        if c["B"] > 2:
            c["B"] = (c["B"] + 1) // 2
            c["ones"] = min(c["ones"], c["B"] - 1)
        else:
            for k in ("new_lo", "new_hi", "ctx_lo", "ctx_hi"):
                c[k] = c[k] * 2 // 3 if c[k] > 2 else c[k]
    return c


def _lengths(c):
    """(new tokens, keys in all) of every sequence: a property of the case, the same for every seed."""
    rng = random.Random("%(B)d %(ones)d %(new_lo)d %(new_hi)d %(ctx_lo)d %(ctx_hi)d" % c)
    new = [1 if b < c["ones"] else rng.randint(c["new_lo"], c["new_hi"]) for b in range(c["B"])]
    old = [rng.randint(c["ctx_lo"], c["ctx_hi"]) for _ in range(c["B"])]
    order = list(range(c["B"]))
    rng.shuffle(order)
    return [(new[b], old[b] + new[b]) for b in order]


def _prefix(c, n, total):
    """The bidirectional part of a sequence: all but the last 64 keys (the codes of a reference recording)."""
    return max(1, total - 64) if c["prefix"] else 0


def _scores(c):
    """Scores that the plain form holds at once (every sequence padded to the longest)."""
    lens = _lengths(c)
    return c["B"] * c["nh"] * max(n for n, _ in lens) * max(t for _, t in lens)


def work(case):
    c = dict(case)
    lens = _lengths(c)
    T, es = sum(n for n, _ in lens), 2
    if c["op"] == "append":
        row = (c["nh"] + 2 * c["nkv"]) * c["hd"]
        xs = 4 if c["x"] == "f32" else 2
        return {"bytes": T * (row * (xs + es) + c["rot"] * 4 + 4),
                "flops": T * 3 * (c["nh"] + c["nkv"]) * c["rot"]}
    pairs = keys = 0
    for n, total in lens:
        pre, w = _prefix(c, n, total), c["window"]
        if not w:
            # rows total-n .. total-1 see max(p + 1, pre) keys
            a = min(max(pre - (total - n), 0), n)       # rows inside the prefix
            pairs += a * pre + sum(range(total - n + a + 1, total + 1))
            keys += total
        else:
            pairs += sum(min(p + 1, w) for p in range(total - n, total))
            keys += total - max(0, total - n - w + 1)
    return {"bytes": 2 * keys * c["nkv"] * c["hd"] * es + 2 * T * c["nh"] * c["hd"] * es + T * c["nh"] * 4,
            "flops": 4 * c["hd"] * c["nh"] * pairs}


# ---- what a program holds -----------------------------------------------------------------

def prepare(case, seed):
    c = dict(case)
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    lens = _lengths(c)
    B, P, hd, nkv, nh = c["B"], c["page"], c["hd"], c["nkv"], c["nh"]
    T = sum(n for n, _ in lens)
    cols = max(-(-t // P) for _, t in lens) + 1
    used = sum(-(-t // P) for _, t in lens)
    # the pages of a sequence lie anywhere in the cache; entries past its last page hold no page
    ids = list(range(used + 3))
    rng.shuffle(ids)
    rows, at = [], 0
    for _, t in lens:
        n = -(-t // P)
        rows.append(ids[at:at + n] + [-1] * (cols - n))
        at += n
    s = {"case": c, "table": torch.tensor(rows, dtype=torch.int32, device=dev),
         "seq_start": torch.tensor([sum(n for n, _ in lens[:b]) for b in range(B + 1)], dtype=torch.int32, device=dev),
         "kv_len": torch.tensor([t for _, t in lens], dtype=torch.int32, device=dev),
         "tokens": T, "max_new": max(n for n, _ in lens), "max_keys": max(t for _, t in lens)}
    t = DT[c["type"]]

    def normal(shape, dtype, scale=1.0, mean=0.0):
        return torch.empty(shape, dtype=dtype, device=dev).normal_(mean, scale, generator=g)

    # every slot holds something: a page was another sequence's before
    s["kc"] = normal((used + 3, nkv, P, hd), t)
    s["vc"] = normal((used + 3, nkv, P, hd), t, 1.0, 0.1)
    if c["op"] == "append":
        # one row of the fused projection per token: queries, keys, values side by side
        s["qkv"] = normal((T, (nh + 2 * nkv) * hd), DT[c["x"]], 1.5)
        half, top = c["rot"] // 2, max(t for _, t in lens)
        inv = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
        ang = torch.arange(top + 1, dtype=torch.float64, device=dev)[:, None] * inv
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    else:
        s["q"] = normal((T, nh, hd), t, 2.0)   # scores of a standard deviation of 2
        s["scale"] = 1.0 / math.sqrt(hd)
        s["prefix"] = None
        if c["prefix"]:
            s["prefix"] = torch.tensor([_prefix(c, n, t) for n, t in lens], dtype=torch.int32, device=dev)
    return s


# ---- one call -----------------------------------------------------------------------------

_module = None


def _gsvk():
    """The framework's Python binding, found once."""
    global _module
    if _module is None:
        package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gsv.cpp_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        import gsvk
        _module = gsvk
    return _module


def _split(s):
    c = s["case"]
    nq, nk = c["nh"] * c["hd"], c["nkv"] * c["hd"]
    return s["qkv"][:, :nq], s["qkv"][:, nq:nq + nk], s["qkv"][:, nq + nk:]


def _own(s):
    gsvk = _gsvk()
    c = s["case"]
    if "kv" not in s:   # the handle of the cache and its batch, which a program keeps with its buffers
        s["kv"] = gsvk.PagedKV(s["kc"], s["vc"], s["table"], s["seq_start"], s["kv_len"])
    if c["op"] == "append":
        q, k, v = _split(s)
        q_out = torch.empty((s["tokens"], c["nh"], c["hd"]), dtype=s["kc"].dtype, device=q.device)
        gsvk.op_paged_append(s["kv"], k, v, q=q, q_out=q_out, cos=s["cos"], sin=s["sin"],
                             pairs=c["style"] == "pairs")
        return {"q": q_out, "k": s["kc"], "v": s["vc"]}
    out = torch.empty_like(s["q"])
    lse = torch.empty((s["tokens"], c["nh"]), dtype=torch.float32, device=out.device)
    gsvk.op_attn_paged(s["kv"], s["q"], s["scale"], out, max_new=s["max_new"], max_keys=s["max_keys"], lse=lse,
                       window=c["window"], prefix=s["prefix"])
    return {"out": out, "lse": lse}


def _rows(s):
    """Sequence, index in its chunk and slot of every new token."""
    r = torch.arange(s["tokens"], device=s["table"].device)
    b = torch.searchsorted(s["seq_start"][1:].long(), r, right=True)
    i = r - s["seq_start"].long()[b]
    n = (s["seq_start"][1:] - s["seq_start"][:-1]).long()
    return b, i, s["kv_len"].long()[b] - n[b] + i


def _rotate(x, cos, sin, rot, style):
    if style == "halves":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1)
    a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _plain_append(s):
    c = s["case"]
    t, T = s["kc"].dtype, s["tokens"]
    b, _, slot = _rows(s)
    page = s["table"][b, slot // c["page"]].long()
    off = slot % c["page"]
    q, k, v = (x.float().view(T, -1, c["hd"]) for x in _split(s))
    cos, sin = s["cos"][slot][:, None], s["sin"][slot][:, None]
    s["kc"][page, :, off] = _rotate(k, cos, sin, c["rot"], c["style"]).to(t)
    s["vc"][page, :, off] = v.to(t)
    return {"q": _rotate(q, cos, sin, c["rot"], c["style"]).to(t), "k": s["kc"], "v": s["vc"]}


def _plain_attn(s):
    c = s["case"]
    B, nkv, hd, nh = c["B"], c["nkv"], c["hd"], c["nh"]
    G, n, L = nh // nkv, s["max_new"], s["max_keys"]
    b, i, slot = _rows(s)

    def gather(cache):   # [B, nkv, L, hd] of every sequence's pages in order
        x = cache[s["table"].clamp_min(0).long()]
        return x.permute(0, 2, 1, 3, 4).reshape(B, nkv, -1, hd)[:, :, :L].float()

    q = torch.zeros((B, n, nkv, G, hd), device=slot.device)
    q[b, i] = s["q"].float().view(-1, nkv, G, hd)
    q = q.permute(0, 2, 3, 1, 4).reshape(B, nkv, G * n, hd)
    keys = torch.arange(L, device=slot.device)
    new = (s["seq_start"][1:] - s["seq_start"][:-1]).long()
    p = (s["kv_len"] - new)[:, None] + torch.arange(n, device=slot.device)      # [B, n] positions
    end = p + 1 if s["prefix"] is None else torch.maximum(p + 1, s["prefix"][:, None])
    see = (keys < end[..., None]) & (keys < s["kv_len"][:, None, None])
    if c["window"]:
        see &= keys > p[..., None] - c["window"]
    x = torch.matmul(q, gather(s["kc"]).transpose(2, 3).contiguous()).mul_(s["scale"])
    x = x.view(B, nkv, G, n, L).masked_fill_(~see[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    x = x.sub_(m).exp_()
    z = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(B, nkv, G * n, L), gather(s["vc"])).view(B, nkv, G, n, hd)
    o = torch.where(z > 0, o / z, torch.zeros_like(o))
    lse = (m + z.log()).squeeze(-1)
    return {"out": o.permute(0, 3, 1, 2, 4)[b, i].reshape(-1, nh, hd).to(s["q"].dtype),
            "lse": lse.permute(0, 3, 1, 2)[b, i].reshape(-1, nh)}


def run(state):
    if own:
        return _own(state)
    return _plain_append(state) if state["case"]["op"] == "append" else _plain_attn(state)


# ---- the definition in 64 bits ---------------------------------------------------------------

def _exact_append(c, s, lens):
    out = [x.clone().double() for x in (s["kc"], s["vc"])]
    q_out = torch.empty((s["tokens"], c["nh"], c["hd"]), dtype=torch.float64, device=s["kc"].device)
    # each pair as a complex number times cos + i sin of its position
    first = 0
    for b, (n, total) in enumerate(lens):
        slots = torch.arange(total - n, total, device=s["kc"].device)
        turn = torch.complex(s["cos"].double()[slots], s["sin"].double()[slots])[:, None]
        x = s["qkv"][first:first + n].double().view(n, -1, c["hd"])
        part, rest = x[:, :c["nh"] + c["nkv"], :c["rot"]], x[:, :c["nh"] + c["nkv"], c["rot"]:]
        if c["style"] == "halves":
            z = torch.view_as_complex(part.unflatten(-1, (2, -1)).transpose(-1, -2).contiguous()) * turn
            part = torch.view_as_real(z).transpose(-1, -2).flatten(-2)
        else:
            part = torch.view_as_real(torch.view_as_complex(part.unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)
        y = torch.cat([part, rest], -1)
        q_out[first:first + n] = y[:, :c["nh"]]
        page, off = s["table"][b].long()[slots // c["page"]], slots % c["page"]
        for h in range(c["nkv"]):
            out[0][page, h, off] = y[:, c["nh"] + h]
            out[1][page, h, off] = x[:, c["nh"] + c["nkv"] + h]
        first += n
    return {"q": q_out, "k": out[0], "v": out[1]}


def _exact_attn(c, s, lens):
    G = c["nh"] // c["nkv"]
    out = torch.zeros((s["tokens"], c["nh"], c["hd"]), dtype=torch.float64, device=s["q"].device)
    lse = torch.full((s["tokens"], c["nh"]), -math.inf, dtype=torch.float64, device=s["q"].device)
    first = 0
    for b, (n, total) in enumerate(lens):
        pages = s["table"][b, :-(-total // c["page"])].long()
        key = torch.arange(total, device=out.device)
        for h in range(c["nkv"]):
            K = s["kc"][pages, h].reshape(-1, c["hd"])[:total].double()
            V = s["vc"][pages, h].reshape(-1, c["hd"])[:total].double()
            for r0 in range(0, n, 1024):
                r1 = min(n, r0 + 1024)
                p = torch.arange(total - n + r0, total - n + r1, device=out.device)[:, None]
                hide = key[None] > (torch.clamp_min(p, _prefix(c, n, total) - 1) if c["prefix"] else p)
                if c["window"]:
                    hide = hide | (key[None] <= p - c["window"])
                for g in range(h * G, h * G + G):
                    x = (s["q"][first + r0:first + r1, g].double() @ K.T) * s["scale"]
                    x = torch.where(hide, -math.inf, x)
                    z = torch.logsumexp(x, -1)
                    out[first + r0:first + r1, g] = torch.exp(x - z[:, None]) @ V
                    lse[first + r0:first + r1, g] = z
        first += n
    return {"out": out, "lse": lse}


def exact(case, seed):
    c = dict(case)
    s = prepare(c, seed)
    return (_exact_append if c["op"] == "append" else _exact_attn)(c, s, _lengths(c))
