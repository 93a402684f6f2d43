"""The work that users of flashmask_b200 have its operators around attention do, as cases that can be timed and compared.

A case is a dict of plain values.  ``use`` says which call it is:

* ``norm_train``   ``qk_norm_rotary`` and the gradients of q, k and both weights, before the attention of a training step;
* ``norm``         ``qk_norm_rotary`` without gradients: a prompt, or the one new token of every sequence;
* ``cache``        ``kv_cache_write`` of new tokens, ``kv_cache_read`` of the last tokens of every sequence;
* ``attention``    ``kv_cache_attention`` of one token, a few, or a chunk of a prompt for every sequence;
* ``step``         one layer's step of generation: norm and rotation, append to the cache, attention over it.

The cache holds pages of tokens in 8 bits (``e4m3`` or ``int8``) with a power of two as the scale of every page and kv head.  A
case fixes the LENGTHS of its sequences through ``layout``; their order, and which page is where, come from the seed.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
LARGEST = {"e4m3": 448.0, "int8": 127.0}
EXPONENTS = {"e4m3": (-64, 119), "int8": (-64, 121)}


# ------------------------------------------------------------------ cases
def _norm(use, B, S, Hq, Hkv, d, rot, dtype="bf16", interleaved=False, docs=True, layout=1, name=None):
    c = {"use": use, "B": B, "S": S, "Hq": Hq, "Hkv": Hkv, "d": d, "rot": rot, "dtype": dtype, "interleaved": interleaved,
         "docs": docs, "layout": layout}
    return {**c, "name": name} if name else c


def _cached(use, B, S, length, Hq, Hkv, d, dv, kind="e4m3", page=64, dtype="bf16", spread=0.0, window=0, sink=False, layout=1,
            name=None):
    c = {"use": use, "B": B, "S": S, "len": length, "Hq": Hq, "Hkv": Hkv, "d": d, "dv": dv, "kind": kind, "page": page,
         "dtype": dtype, "spread": spread, "window": window, "sink": sink, "layout": layout}
    return {**c, "name": name} if name else c


def listed():
    return [
        # packed fine-tuning at 8K tokens with grouped heads: what stands before the benchmark's headline attention
        _norm("norm_train", 2, 8192, 32, 8, 128, 128, name="norm_train_8k_gqa"),
        # a batch that is no round length, 96-wide heads of which two thirds rotate, neighbouring pairs
        _norm("norm_train", 2, 3001, 16, 4, 96, 64, dtype="fp16", interleaved=True, layout=2, name="norm_train_3001_d96"),
        # the new token of eight sequences: latency alone
        _norm("norm", 8, 1, 32, 8, 128, 128, docs=False, name="norm_decode_8"),
        # two prompts of 8K tokens written to the cache and read back
        _cached("cache", 2, 8192, 8192, 0, 8, 128, 128, name="cache_prompt_2x8k"),
        # one token appended to each of 64 sequences of any length, the pages that it went to read back
        _cached("cache", 64, 1, 2048, 0, 8, 128, 128, kind="int8", page=32, dtype="fp16", spread=0.9, layout=3,
                name="cache_append_64"),
        # the first answers of a short chat: one sequence, latency alone
        _cached("attention", 1, 1, 777, 32, 8, 128, 128, kind="int8", page=16, name="decode_1x777_int8"),
        # one more token for each of eight sequences
        _cached("attention", 8, 1, 8192, 32, 8, 128, 128, name="decode_8x8k"),
        # a full server: 64 sequences of very different lengths, 64-wide heads
        _cached("attention", 64, 1, 4096, 32, 8, 64, 64, kind="int8", page=32, dtype="fp16", spread=1.0, layout=4,
                name="decode_64_ragged_d64"),
        # five drafted tokens checked at once, window attention with a sink logit per head
        _cached("attention", 16, 5, 5000, 32, 8, 128, 128, spread=0.5, window=1024, sink=True, layout=5,
                name="draft_16x5_window"),
        # the longest context, one sequence
        _cached("attention", 1, 1, 131072, 32, 8, 128, 128, page=128, name="decode_1x128k"),
        # a chunk of a long prompt against everything before it
        _cached("attention", 1, 512, 16384, 32, 8, 128, 128, name="chunk_512_of_16k"),
        # one layer's step of generation for eight sequences
        _cached("step", 8, 1, 8192, 32, 8, 128, 128, spread=0.3, layout=6, name="step_8x8k"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above."""
    use = rng.choice(["norm_train", "norm_train", "norm", "cache", "cache", "attention", "attention", "attention", "attention", "step"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    layout = rng.randrange(1, 1 << 20)
    hkv = rng.choice([1, 2, 4, 8])
    hq = min(32, hkv * rng.choice([1, 2, 4, 4, 8]))
    if use in ("norm", "norm_train"):
        S = _log_int(rng, 1, 8192)
        d = rng.choice([64, 80, 96, 128, 128, 128, 192, 256])
        B = rng.randint(1, max(1, min(64, 16384 * 128 // (S * d))))
        rot = rng.choice([d, d, d // 2 // 16 * 16])
        return _norm(use, B, S, hq, hkv, d, rot, dtype, rng.random() < 0.3, rng.random() < 0.6, layout)
    kind, page = rng.choice(["e4m3", "e4m3", "int8"]), rng.choice([16, 32, 64, 64, 128])
    spread = rng.choice([0.0, 0.4, 0.9])
    if use == "cache":
        S = 1 if rng.random() < 0.4 else _log_int(rng, 2, 4096)
        B = rng.randint(1, max(1, min(64, 8192 // S)))
        d, dv = rng.choice([(64, 64), (80, 80), (96, 96), (128, 128), (128, 128), (192, 128), (256, 256)])
        return _cached(use, B, S, S + _log_int(rng, 1, 2048), 0, hkv, d, dv, kind, page, dtype, spread, layout=layout)
    d, dv = rng.choice([(64, 64), (80, 80), (96, 96), (128, 128), (128, 128), (128, 128), (192, 128), (256, 256)])
    window = rng.choice([0, 0, 0, _log_int(rng, 64, 4096)])
    sink = rng.random() < 0.3
    if use == "step":
        L = _log_int(rng, 32, 16384)
        B = rng.randint(1, max(1, min(64, 65536 // L)))
        return _cached(use, B, 1, L, hq, hkv, d, dv if d == dv else d, kind, page, dtype, spread, window, sink, layout)
    S = 1 if rng.random() < 0.5 else (_log_int(rng, 2, 8) if rng.random() < 0.6 else _log_int(rng, 9, 512))
    L = S + _log_int(rng, 1, 65536 if S == 1 else 7168)
    B = rng.randint(1, max(1, min(64, 65536 // L, 512 // S)))
    return _cached(use, B, S, L, hq, hkv, d, dv, kind, page, dtype, spread, window, sink, layout)


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """Lengths of the case's sequences with their new tokens: a function of the case alone, longest up to 4 x `len`."""
    B, S, L = case["B"], case["S"], case["len"]
    if not case["spread"]:
        return [L] * B
    r = np.random.default_rng(case["layout"])
    f = np.exp(case["spread"] * r.standard_normal(B))
    return [int(min(4 * L, max(S, round(L * x / f.mean())))) for x in f]


def _tables(case, length):
    """cos and sin of every position and frequency, as a model keeps them."""
    half = case["rot"] // 2
    inv = 10000.0 ** (-np.arange(half, dtype=np.float64) / half)
    angle = np.arange(length, dtype=np.float64)[:, None] * inv[None]
    return torch.from_numpy(np.cos(angle).astype(np.float32)).cuda(), torch.from_numpy(np.sin(angle).astype(np.float32)).cuda()


def _to_8_bits(x, e, kind):
    """x 2^-e rounded to the payload's grid; x fp32, e fp32 exponents."""
    y = torch.ldexp(x, -e)
    return y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn) if kind == "e4m3" else torch.round(y).clamp(-127.0, 127.0).to(torch.int8)


def _exponent(amax, kind):
    """The least e with amax <= M 2^e, within the range of the kind."""
    m, x = torch.frexp(amax / LARGEST[kind])          # amax / M = m 2^x with m in [0.5, 1)
    # the quotient is rounded: compare against the exact products on both sides
    e = (x - 1).float()
    for _ in range(2):
        e = torch.where(amax > torch.ldexp(torch.full_like(amax, LARGEST[kind]), e), e + 1, e)
    return torch.where(amax > 0, e, torch.full_like(e, -1e9)).clamp(*EXPONENTS[kind])


def _normal(g, dt, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dt)


def _norm_inputs(case, seed, B, S, positions):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, d, Hq, Hkv = DTYPES[case["dtype"]], case["d"], case["Hq"], case["Hkv"]
    # q and k are views of one projection's output, as a model with a fused projection has them
    x = _normal(g, dt, B, S, Hq + 2 * Hkv, d)
    s = {"q": x[:, :, :Hq], "k": x[:, :, Hq:Hq + Hkv], "v": x[:, :, Hq + Hkv:], "positions": positions,
         "q_weight": (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dt),
         "k_weight": (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dt)}
    return s, g


def _cache_inputs(case, seed):
    """The cache with every token before the new ones, its page table and lengths."""
    B, S, P, H, d, dv, kind = (case[k] for k in ("B", "S", "page", "Hkv", "d", "dv", "kind"))
    r = np.random.default_rng([seed, 7])
    lens = [int(n) for n in r.permutation(_lengths(case))]
    need = [-(-n // P) for n in lens]
    n_pages = sum(need) + 3
    order = r.permutation(n_pages)
    table, at = np.zeros((B, max(need)), np.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    s = {"table": torch.from_numpy(table).cuda(), "seqlens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "lens": lens}
    for name, w in (("k", d), ("v", dv)):
        pay = torch.empty(n_pages, H, P, w, device="cuda", dtype=torch.float8_e4m3fn if kind == "e4m3" else torch.int8)
        scale = torch.empty(n_pages, H, device="cuda")
        for p0 in range(0, n_pages, 512):
            x = torch.randn(min(512, n_pages - p0), H, P, w, generator=g, device="cuda")
            e = _exponent(x.abs().amax((2, 3)), kind)
            pay[p0:p0 + 512] = _to_8_bits(x, e[..., None, None], kind)
            scale[p0:p0 + 512] = torch.ldexp(torch.ones_like(e), e)
        s[name + "8"], s[name + "_scale"] = pay, scale
    return s, g


def _inputs(case, seed):
    use = case["use"]
    if use in ("norm", "norm_train"):
        B, S = case["B"], case["S"]
        pos = np.tile(np.arange(S, dtype=np.int32), (B, 1))
        if case["docs"]:
            r = np.random.default_rng([case["layout"], seed])
            for b in range(B):                       # documents start over at position 0
                at = 0
                while at < S:
                    n = int(min(S - at, max(16, r.lognormal(math.log(1024), 1.0))))
                    pos[b, at:at + n] = np.arange(n)
                    at += n
        else:
            pos += np.random.default_rng([case["layout"], seed]).integers(0, 8192, (B, 1)).astype(np.int32)
        s, g = _norm_inputs(case, seed, B, S, torch.from_numpy(pos).cuda())
        s["cos"], s["sin"] = _tables(case, 16384)
        if use == "norm_train":
            s["d_q"] = _normal(g, DTYPES[case["dtype"]], *s["q"].shape)
            s["d_k"] = _normal(g, DTYPES[case["dtype"]], *s["k"].shape)
        return s
    s, g = _cache_inputs(case, seed)
    dt, B, S = DTYPES[case["dtype"]], case["B"], case["S"]
    s["start"] = s["seqlens"] - S
    if use == "cache":
        s["key"] = _normal(g, dt, B, S, case["Hkv"], case["d"]) * 1.5
        s["value"] = _normal(g, dt, B, S, case["Hkv"], case["dv"]) * 1.5
    elif use == "attention":
        s["query"] = _normal(g, dt, B, S, case["Hq"], case["d"])
    else:
        more, g = _norm_inputs({**case, "rot": case["d"]}, seed + 2, B, 1, s["start"].view(B, 1))
        s.update(more)
        s["cos"], s["sin"] = _tables({"rot": case["d"]}, 4 * case["len"] + 1)
    s["sinks"] = torch.randn(case["Hq"], generator=g, device="cuda") if case["sink"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["use"] == "norm_train":
        # views of one buffer cannot be leaves of their own: the leaf is the projection's output, as in a model
        s["wrt"] = []
        for name in ("q", "k", "q_weight", "k_weight"):
            s[name] = s[name].detach().requires_grad_(True)
            s["wrt"].append(s[name])
    if case["use"] == "cache":
        s["last"] = case["S"] if case["S"] > 1 else case["page"]
        s["from"] = s["seqlens"] - s["last"]
    if own and "k8" in s:
        import flashmask_b200 as fm
        s["cache"] = fm.QuantizedKVCache(s["k8"], s["v8"], s["k_scale"], s["v_scale"])
    return s


# ------------------------------------------------------------------ plain forms
def _plain_norm(x, w, cos, sin, positions, interleaved):
    """x, w in 32 bits -> the rotated norm in 32 bits."""
    u = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
    c, s = cos[positions.long()][:, :, None], sin[positions.long()][:, :, None]
    half = cos.shape[1]
    if interleaved:
        a, b = u[..., 0:2 * half:2], u[..., 1:2 * half:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = u[..., :half], u[..., half:2 * half]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, u[..., 2 * half:]], -1)


def _plain_write(case, s, key, value):
    """The cache with `key` and `value` written at positions start .. start + S - 1, scales grown where they have to."""
    P, kind, B, S = case["page"], case["kind"], case["B"], case["S"]
    n_pages = (S - 1) // P + 2
    first = s["start"].long() // P
    j = torch.arange(n_pages, device="cuda")
    page_at = first[:, None] + j[None]                                               # [B, n]
    touched = page_at <= ((s["start"].long() + S - 1) // P)[:, None]
    page = s["table"].long().gather(1, page_at.clamp(max=s["table"].shape[1] - 1))
    slot = page_at[..., None] * P + torch.arange(P, device="cuda")                     # positions [B, n, P]
    token = slot - s["start"].long()[:, None, None]
    new = (token >= 0) & (token < S)
    old = (token < 0) & ((s["start"].long() % P) > 0)[:, None, None] & (j == 0)[None, :, None]
    pick = (torch.arange(B, device="cuda")[:, None, None], token.clamp(0, S - 1))
    done = {}
    for name, x in (("k", key), ("v", value)):
        pay, scale = s[name + "8"].clone(), s[name + "_scale"].clone()
        fresh = x.float()[pick].permute(0, 1, 3, 2, 4)                               # [B, n, H, P, w]
        keep = new[:, :, None, :, None]
        amax = torch.where(keep, fresh.abs(), torch.zeros_like(fresh)).amax((3, 4))
        e = _exponent(amax, kind)
        e_old = torch.frexp(scale[page])[1].float() - 1
        e = torch.where(old.any(-1)[..., None], torch.maximum(e, e_old), e)
        before = pay[page]
        again = _to_8_bits(before.float(), (e - e_old)[..., None, None], kind)
        fresh = _to_8_bits(fresh, e[..., None, None], kind)
        raw = lambda t: t.view(torch.uint8)
        merged = torch.where(keep, raw(fresh), torch.where(old[:, :, None, :, None], raw(again), raw(before)))
        raw(pay)[page[touched]] = merged[touched]
        scale[page[touched]] = torch.ldexp(torch.ones_like(e), e)[touched]
        done[name + "8"], done[name + "_scale"] = pay, scale
    return done


def _plain_read(c, name, table, b, lo, hi):
    """Positions lo .. hi - 1 of sequence b in 32 bits: [hi - lo, H, w]."""
    pay, scale = c[name + "8"], c[name + "_scale"]
    P = pay.shape[2]
    pages = table[b, lo // P:(hi - 1) // P + 1].long()
    x = pay[pages].float() * scale[pages][..., None, None]
    return x.permute(0, 2, 1, 3).flatten(0, 1)[lo - lo // P * P:][:hi - lo]


def _plain_attention(case, s, c, query):
    """(out, lse) over the cache c, sequence by sequence."""
    S, G, w = case["S"], case["Hq"] // case["Hkv"], case["window"]
    out = torch.empty(case["B"], S, case["Hq"], case["dv"], device="cuda", dtype=query.dtype)
    lse = torch.empty(case["B"], case["Hq"], S, device="cuda")
    for b, n in enumerate(s["lens"]):
        lo = max(0, n - S - w + 1) if w else 0
        k, v = (_plain_read(c, name, s["table"], b, lo, n) for name in ("k", "v"))
        p = torch.arange(n - S, n, device="cuda")[:, None]
        key = torch.arange(lo, n, device="cuda")[None]
        hidden = key > p
        if w:
            hidden |= key <= p - w
        for h in range(case["Hkv"]):
            q = query[b, :, h * G:(h + 1) * G].float().permute(1, 0, 2)                # [G, S, d]
            x = (q @ k[:, h].T) / math.sqrt(case["d"])
            x = x.masked_fill(hidden, -math.inf)
            m = x.amax(-1, keepdim=True)
            if s["sinks"] is not None:
                m = torch.maximum(m, s["sinks"][h * G:(h + 1) * G, None, None])
            e = torch.exp(x - m)
            l = e.sum(-1, keepdim=True)
            if s["sinks"] is not None:
                l = l + torch.exp(s["sinks"][h * G:(h + 1) * G, None, None] - m)
            out[b, :, h * G:(h + 1) * G] = ((e @ v[:, h]) / l).permute(1, 0, 2).to(query.dtype)
            lse[b, h * G:(h + 1) * G] = (m + torch.log(l))[..., 0]
    return out, lse


def _run_plain(s):
    case = s["case"]
    use, dt = case["use"], DTYPES[case["dtype"]]
    if use in ("norm", "norm_train"):
        back = use == "norm_train"
        x = [s[n].detach().float().requires_grad_(back) for n in ("q", "k", "q_weight", "k_weight")]
        with torch.set_grad_enabled(back):
            y = [_plain_norm(x[i], x[i + 2], s["cos"], s["sin"], s["positions"], case["interleaved"]) for i in (0, 1)]
        out = [t.detach().to(dt) for t in y]
        if back:
            out += [t.to(dt) for t in torch.autograd.grad(y, x, [s["d_q"].float(), s["d_k"].float()])]
        return out
    with torch.no_grad():
        if use == "cache":
            c = _plain_write(case, s, s["key"], s["value"])
            res = []
            for name in ("k", "v"):
                w = case["d"] if name == "k" else case["dv"]
                r = torch.zeros(case["B"], s["last"], case["Hkv"], w, device="cuda", dtype=dt)
                for b, n in enumerate(s["lens"]):
                    lo = max(0, n - s["last"])
                    r[b, s["last"] - (n - lo):] = _plain_read(c, name, s["table"], b, lo, n).to(dt)
                res.append(r)
            return res + [c["k_scale"], c["v_scale"]]
        if use == "attention":
            return list(_plain_attention(case, s, s, s["query"]))
        q, k = (_plain_norm(s[n].float(), s[n + "_weight"].float(), s["cos"], s["sin"], s["positions"], False).to(dt) for n in ("q", "k"))
        c = _plain_write(case, s, k, s["v"])
        return [q, k, *_plain_attention(case, s, c, q), c["k_scale"], c["v_scale"]]


# ------------------------------------------------------------------ the framework's calls
def _run_own(s):
    import flashmask_b200 as fm
    case = s["case"]
    use = case["use"]
    if use == "norm_train":
        q, k = fm.qk_norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["positions"],
                                 interleaved=case["interleaved"])
        return [q.detach(), k.detach(), *torch.autograd.grad([q, k], s["wrt"], [s["d_q"], s["d_k"]])]
    with torch.no_grad():
        if use == "norm":
            return list(fm.qk_norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["positions"],
                                          interleaved=case["interleaved"]))
        cache, table, seqlens = s["cache"], s["table"], s["seqlens"]
        window = case["window"] or None
        if use == "attention":
            return list(fm.kv_cache_attention(s["query"], cache, table, seqlens, window_size=window, sink=s["sinks"], return_lse=True))
        if use == "cache":
            fm.kv_cache_write(cache, s["key"], s["value"], table, s["start"])
            return [*fm.kv_cache_read(cache, table, s["from"], seqlens, s["last"], dtype=DTYPES[case["dtype"]]), cache.k_scale, cache.v_scale]
        q, k = fm.qk_norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["positions"])
        fm.kv_cache_write(cache, k, s["v"], table, s["start"])
        return [q, k, *fm.kv_cache_attention(q, cache, table, seqlens, window_size=window, sink=s["sinks"], return_lse=True),
                cache.k_scale, cache.v_scale]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ floors
def work(case):
    use = case["use"]
    if use in ("norm", "norm_train"):
        rows = case["B"] * case["S"] * (case["Hq"] + case["Hkv"])
        tables = case["B"] * case["S"] * (4 + 4 * case["rot"])
        n = rows * case["d"]
        if use == "norm":
            return {"bytes": 4 * n + tables, "flops": 8 * n}
        return {"bytes": 8 * n + tables, "flops": 24 * n}     # x and dy in, y and dx out, each once
    B, S, H, d, dv, P = (case[k] for k in ("B", "S", "Hkv", "d", "dv", "page"))
    lens = _lengths(case)
    if use == "cache":
        n = B * S * H * (d + dv)
        last = S if S > 1 else P
        m = sum(min(x, last) for x in lens) * H * (d + dv)
        return {"bytes": 3 * n + (m if S == 1 else 0) + 2 * B * last * H * (d + dv), "flops": 4 * n + 2 * m}
    keys = pairs = 0
    for n in lens:
        w = case["window"] or n
        keys += n - max(0, n - S - w + 1)
        lo = n - S + 1                                        # visible to the first row without a window
        pairs += sum(min(x, w) for x in range(lo, n + 1))
    nbytes = keys * H * (d + dv) + -(-keys // P) * (8 * H + 4) + B * S * case["Hq"] * (2 * d + 2 * dv + 4)
    flops = 2 * pairs * case["Hq"] * (d + dv)
    if use == "step":
        n = B * (case["Hq"] + H) * d
        nbytes += 4 * n + 3 * B * H * (d + dv)
        flops += 8 * n
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------ 64 bits, from the definitions
def _grid_e4m3(y):
    """Nearest value of 4 exponent bits (bias 7) and 3 mantissa bits, ties to even, at most 448."""
    a = y.abs().clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.sign(y) * (torch.round(a / step) * step).clamp(max=448.0)


def _values_of(payload, kind):
    """What payload bytes stand for before their scale, in 64 bits."""
    raw = payload.view(torch.uint8)
    if kind == "int8":
        table = [i if i < 128 else i - 256 for i in range(256)]
    else:
        table = []
        for i in range(256):
            x, m = i >> 3 & 15, i & 7
            v = m * 2.0 ** -9 if x == 0 else (8 + m) * 2.0 ** (x - 10)
            table.append(-v if i & 128 else v)
    return torch.tensor(table, dtype=torch.float64, device="cuda")[raw.int()]


def _exact_norm(case, s, name, rot):
    x = s[name].detach().double()
    w = s[name + "_weight"].detach().double()
    pos, half, d = s["positions"].long(), rot // 2, x.shape[-1]
    c, sn = s["cos"].double()[pos].unsqueeze(2), s["sin"].double()[pos].unsqueeze(2)
    i = torch.arange(half, device="cuda")
    first, second = (2 * i, 2 * i + 1) if case.get("interleaved") else (i, i + half)
    r = (x.square().sum(-1, keepdim=True) / d + 1e-6).pow(-0.5)
    xr = x * r
    y = xr * w
    a, b = y[..., first], y[..., second]
    y[..., first], y[..., second] = a * c - b * sn, a * sn + b * c
    dy = s.get("d_" + name)
    if dy is None:
        return y, None, None
    g = dy.double()
    a, b = g[..., first], g[..., second]
    g[..., first], g[..., second] = a * c + b * sn, b * c - a * sn
    dw = (g * xr).sum((0, 1, 2))
    g *= w
    return y, r * (g - xr * (g * xr).mean(-1, keepdim=True)), dw


def _exact_sequence(case, s, b, name, fresh):
    """The values that positions 0 .. len - 1 of sequence b stand for after the write of `fresh` [S, H, w] (None: no write), and
    {page: scales [H]} of the pages that the write touched."""
    P, kind, n, S = case["page"], case["kind"], s["lens"][b], case["S"]
    lo_e, hi_e = EXPONENTS[kind]
    pages = s["table"][b, :-(-n // P)].long()
    scales = s[name + "_scale"].double()[pages]                                      # [pages, H]
    units = _values_of(s[name + "8"][pages], kind)                                   # [pages, H, P, w]
    touched = {}
    if fresh is not None:
        fresh = fresh.double()
        at = n - S
        for j in range(at // P, (n - 1) // P + 1):
            lo, hi = max(at, j * P), min(n, (j + 1) * P)
            x = fresh[lo - at:hi - at].transpose(0, 1)                               # [H, tokens, w]
            amax = x.abs().amax((1, 2)).clamp(min=1e-300)
            e = torch.ceil(torch.log2(amax / LARGEST[kind]))
            e = torch.where(torch.exp2(e) * LARGEST[kind] < amax, e + 1, e)
            e = torch.where(torch.exp2(e - 1) * LARGEST[kind] >= amax, e - 1, e).clamp(lo_e, hi_e)
            grid = _grid_e4m3 if kind == "e4m3" else lambda y: torch.round(y).clamp(-127, 127)
            if lo > j * P:
                e = torch.maximum(e, torch.log2(scales[j]).round())
                units[j, :, :lo - j * P] = grid(units[j, :, :lo - j * P] * (scales[j] / torch.exp2(e))[:, None, None])
            units[j, :, lo - j * P:hi - j * P] = grid(x / torch.exp2(e)[:, None, None])
            scales[j] = torch.exp2(e)
            touched[int(pages[j])] = scales[j].clone()
    return (units * scales[..., None, None]).permute(0, 2, 1, 3).flatten(0, 1)[:n], touched


def _exact_attention(case, s, query, k_of, v_of):
    B, S, Hq, H, w = (case[k] for k in ("B", "S", "Hq", "Hkv", "window"))
    G = Hq // H
    out = torch.empty(B, S, Hq, case["dv"], dtype=torch.float64, device="cuda")
    lse = torch.empty(B, Hq, S, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"]):
        k, v = k_of(b), v_of(b)
        for h in range(Hq):
            x = query[b, :, h].double() @ k[:, h // G].T * case["d"] ** -0.5           # [S, n]
            p = torch.arange(S, device="cuda").unsqueeze(1) + (n - S)
            j = torch.arange(n, device="cuda").unsqueeze(0)
            seen = (j <= p) & (j > p - w) if w else j <= p
            x = torch.where(seen, x, torch.full_like(x, -math.inf))
            if s["sinks"] is not None:
                x = torch.cat([x, s["sinks"][h].double().expand(S, 1)], 1)
            lse[b, h] = torch.logsumexp(x, 1)
            out[b, :, h] = torch.softmax(x, 1)[:, :n] @ v[:, h // G]
    return out, lse


def exact(case, seed):
    s = _inputs(case, seed)
    use, dt = case["use"], DTYPES[case["dtype"]]
    if use in ("norm", "norm_train"):
        y, dx, dw = zip(*(_exact_norm(case, s, n, case["rot"]) for n in ("q", "k")))
        return list(y) if use == "norm" else [*y, *dx, *dw]
    if use == "attention":
        return list(_exact_attention(case, s, s["query"], *(lambda b, n=n: _exact_sequence(case, s, b, n, None)[0] for n in ("k", "v"))))
    scales = {n: s[n + "_scale"].double() for n in ("k", "v")}
    if use == "cache":
        new, last = {"k": s["key"], "v": s["value"]}, case["S"] if case["S"] > 1 else case["page"]
    else:
        q, k = (_exact_norm(case, s, n, case["d"])[0] for n in ("q", "k"))
        new = {"k": k.to(dt), "v": s["v"]}                    # the cache takes the key as the 16-bit type holds it
    read = {}
    for n in ("k", "v"):
        for b in range(case["B"]):
            read[n, b], touched = _exact_sequence(case, s, b, n, new[n][b])
            for page, sc in touched.items():
                scales[n][page] = sc
    if use == "step":
        return [q, k, *_exact_attention(case, s, q.to(dt), lambda b: read["k", b], lambda b: read["v", b]), scales["k"], scales["v"]]
    res = []
    for n in ("k", "v"):
        r = torch.zeros(case["B"], last, case["Hkv"], case["d"] if n == "k" else case["dv"], dtype=torch.float64, device="cuda")
        for b in range(case["B"]):
            x = read[n, b][-last:]
            r[b, last - x.shape[0]:] = x
        res.append(r)
    return [*res, scales["k"], scales["v"]]
