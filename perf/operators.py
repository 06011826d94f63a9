"""Operators over a key/value cache held in 8 bits: its writing, its reading back, the attention of new tokens over it,
and the same attention for a batch of sequences that share one prefix.

A cache row is one token of one kv head: D values as whole numbers c in -127 .. 127 and one fp32 scale, x = c * scale with
scale = max|x| / 127 and c = 127 x / max|x| rounded to the nearest, ties to even.  Token t of sequence b lies at position
starts[b] + t where t < counts[b]; later tokens are padding.  Query t sees the keys of the `window` positions up to its
own (0: all of them); with a prefix of P tokens, positions 0 .. P - 1 are the prefix's and a sequence's own follow.  A
padding query's output row, or a padding token read back, is zero.

Sizes are those of this repository's configurations, tests and benchmark (12 or 16 heads of 64 or 128, windows of 512,
1024 and 2048, sequences of up to 16384 tokens, ragged ones, grouped heads).  As in the model, q and k are RMS-normalised
rows and v is a strided view of the fused projection.
"""
import math
import os
import sys

import torch

own = False

_BF16 = torch.bfloat16


def _store(name, B, T, Hkv, D, capacity, first, ragged):
    """Write T tokens after `first` earlier ones (fewer in some sequences if ragged) and read them back."""
    return {"name": name, "kind": "store", "B": B, "T": T, "Hkv": Hkv, "D": D, "capacity": capacity, "first": first, "ragged": ragged}


def _read(name, B, T, Hkv, D, capacity, first):
    return {"name": name, "kind": "read", "B": B, "T": T, "Hkv": Hkv, "D": D, "capacity": capacity, "first": first}


def _attend(name, B, T, H, Hkv, D, capacity, lo, hi, window=0, prefix=0, ragged=False):
    """T new tokens per sequence (fewer in some if ragged), after lo .. hi cached ones, over `prefix` shared ones."""
    return {"name": name, "kind": "prefix" if prefix else "attend", "B": B, "T": T, "H": H, "Hkv": Hkv, "D": D,
            "capacity": capacity, "lo": lo, "hi": hi, "window": window, "prefix": prefix, "ragged": ragged}


def listed():
    return [
        # A generation step of a small batch: one token per sequence, each at a place of its own.
        _store("store_step", 16, 1, 12, 64, 2048, 1000, False),
        # The prompt of one sequence, grouped heads, an odd length.
        _store("store_prompt", 1, 1777, 4, 128, 2048, 0, False),
        # A chunk of a batch's prompts behind earlier chunks, some of them shorter.
        _store("store_batch", 8, 2048, 12, 64, 4096, 333, True),
        # A scored context taken out of its cache to be used elsewhere.
        _read("read_span", 1, 999, 12, 64, 2048, 77),
        # The deep model's whole batch, head dim 128.
        _read("read_long", 4, 4096, 12, 128, 8192, 4095),
        # One token of one sequence in a local layer: latency counts.
        _attend("decode_local", 1, 1, 12, 12, 64, 4096, 2047, 2047, window=512),
        # One token of one long sequence in a full layer.
        _attend("decode_long", 1, 1, 16, 16, 128, 16384, 16383, 16383),
        # A generation step of a large ragged batch.
        _attend("decode_batch", 64, 1, 12, 12, 64, 2048, 64, 2047),
        # Four drafted tokens per sequence, grouped heads of 128, a ragged batch.
        _attend("decode_drafts", 32, 4, 12, 4, 128, 4096, 500, 4092, ragged=True),
        # A chunk of two long prompts over what is cached already.
        _attend("chunk", 2, 500, 12, 12, 64, 4096, 1500, 2500),
        # Four continuations of one context scored in a local layer (multiple choice).
        _attend("prefix_choices", 4, 37, 12, 12, 64, 128, 0, 0, window=512, prefix=1000, ragged=True),
        # One token of each of 64 samples drawn from one long prompt.
        _attend("prefix_samples", 64, 1, 12, 4, 64, 512, 30, 511, prefix=8000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    D = rng.choice((64, 128))
    H = rng.choice((4, 6, 8, 12, 16))
    Hkv = H if rng.random() < 0.5 else rng.choice([g for g in (1, 2, 4) if H % g == 0])
    kind = rng.choice(("store", "read", "attend", "attend", "prefix"))
    if kind in ("store", "read"):
        T, B = _log(rng, 1, 4096), _log(rng, 1, 32)
        first = rng.randrange(0, 4096)
        capacity = first + T + rng.randrange(0, 500)
        return _store("", B, T, Hkv, D, capacity, first, rng.random() < 0.5) if kind == "store" else _read("", B, T, Hkv, D, capacity, first)
    T = 1 if rng.random() < 0.5 else _log(rng, 2, 500)
    B = _log(rng, 1, 64 if T < 16 else 4)
    hi = _log(rng, 1, 16000 if kind == "attend" else 1000)
    window = rng.choice((0, 0, 512, rng.randrange(1, 513), rng.randrange(513, 2049)))
    prefix = _log(rng, 16, 16000) if kind == "prefix" else 0
    return _attend("", B, T, H, Hkv, D, hi + T + rng.randrange(0, 500), rng.randrange(0, hi + 1), hi, window, prefix, rng.random() < 0.5)


def draw(rng):
    most = [work(c) for c in listed()]
    while True:
        case = _draw(rng)
        cost = work(case)
        if any(cost["bytes"] <= w["bytes"] and cost["flops"] <= w["flops"] for w in most):
            case.pop("name")
            return case


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, the last one hi."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)][::-1]


def _starts(case):
    if case["kind"] in ("store", "read"):
        return _spread(case["first"] // 2, case["first"], case["B"])
    return _spread(case["lo"], case["hi"], case["B"])


def _counts(case):
    T = case["T"]
    return _spread((T + 1) // 2, T, case["B"]) if case.get("ragged") else [T] * case["B"]


def _encode(x):
    """Whole numbers and scales of rows x."""
    top = x.float().abs().amax(dim=-1, keepdim=True)
    codes = torch.round(x.float() * 127.0 / torch.where(top > 0, top, 1.0))
    return codes.to(torch.int8), (top / torch.full_like(top, 127.0))[..., 0]


def _rms_rows(x):
    return (x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + 1e-6)).to(_BF16)


def _tokens(g, B, T, Hkv, D):
    """New k and v (B, T, Hkv, D): v a view of a fused projection."""
    k = _rms_rows(torch.randn((B, T, Hkv, D), generator=g, device="cuda"))
    fused = torch.empty((B, T, 3, Hkv * D), device="cuda", dtype=_BF16)
    fused[:, :, 2] = torch.randn((B, T, Hkv * D), generator=g, device="cuda").to(_BF16)
    return k, fused[:, :, 2].view(B, T, Hkv, D)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, T, Hkv, D = (case[x] for x in ("B", "T", "Hkv", "D"))
    order = torch.randperm(B, generator=g, device="cuda")
    s = {"case": case}
    for name, values in (("starts", _starts(case)), ("counts", _counts(case))):
        s[name] = torch.tensor(values, device="cuda", dtype=torch.int32)[order]
    if case["kind"] == "store":
        s["k"], s["v"] = _tokens(g, B, T, Hkv, D)
        return s
    # what earlier calls wrote: the whole cache, and the prefix's
    s["cached"] = _tokens(g, B, max(_starts(case)) + T, Hkv, D)
    if case["kind"] != "read":
        s["q"] = _rms_rows(torch.randn((B, T, case["H"], D), generator=g, device="cuda"))
        if case["prefix"]:
            s["shared"] = _tokens(g, 1, case["prefix"], Hkv, D)
    return s


def _hlm():
    if os.path.abspath("hackable-lm_amd") not in sys.path:
        sys.path.insert(0, os.path.abspath("hackable-lm_amd"))
    import hlm_attn

    return hlm_attn


def _cache_of(k, v, capacity):
    hlm = _hlm()
    cache = hlm.KVCache(k.shape[0], capacity, k.shape[2], k.shape[3], device=k.device)
    hlm.kv_cache_write_hip(cache, k, v, 0)
    return cache


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        if case["kind"] == "store":
            s["cache"] = _hlm().KVCache(case["B"], case["capacity"], case["Hkv"], case["D"], device="cuda")
        else:
            s["cache"] = _cache_of(*s.pop("cached"), case["capacity"])
        if "shared" in s:
            s["prefix"] = _cache_of(*s.pop("shared"), case["prefix"])
        return s
    for name in ("cached", "shared"):
        if name in s:
            s[name] = tuple((c.transpose(1, 2).contiguous(), x.transpose(1, 2).contiguous()) for c, x in map(_encode, s[name]))
    if case["kind"] == "store":
        shape = (case["B"], case["Hkv"], case["capacity"], case["D"])
        s["cached"] = tuple((torch.zeros(shape, device="cuda", dtype=torch.int8), torch.zeros(shape[:3], device="cuda")) for _ in "kv")
    return s


def _span(case, s):
    """(B, T) positions of the new tokens, and which of them are no padding."""
    t = torch.arange(case["T"], device="cuda")
    return s["starts"].long()[:, None] + t, t < s["counts"][:, None]


def _plain_read(case, s, rows, real):
    b = torch.arange(case["B"], device="cuda")[:, None]
    out = []
    for codes, scales in s["cached"]:
        x = codes[b, :, rows].float() * scales[b, :, rows][..., None]
        out.append(torch.where(real[..., None, None], x, 0.0).to(_BF16))
    return tuple(out)


def _plain_store(case, s):
    rows, real = _span(case, s)
    b, t = real.nonzero(as_tuple=True)
    for x, (codes, scales) in zip((s["k"], s["v"]), s["cached"]):
        c, f = _encode(x[b, t])
        codes[b, :, rows[b, t]] = c
        scales[b, :, rows[b, t]] = f
    return _plain_read(case, s, rows, real)


def _plain_attend(case, s):
    B, T, H, Hkv, D, P = (case[x] for x in ("B", "T", "H", "Hkv", "D", "prefix"))
    k, v = (codes.float() * scales[..., None] for codes, scales in s["cached"])
    if P:
        shared = [(codes.float() * scales[..., None]).expand(B, Hkv, P, D) for codes, scales in s["shared"]]
        k, v = torch.cat((shared[0], k), dim=2), torch.cat((shared[1], v), dim=2)
    rows, real = _span(case, s)
    lag = (rows + P)[:, :, None] - torch.arange(k.shape[2], device="cuda")
    seen = (lag >= 0) & real[:, :, None]
    if case["window"]:
        seen &= lag < case["window"]
    seen = seen[:, None, None]  # (B, 1, 1, T, keys)
    q = s["q"].float().view(B, T, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).view(B, Hkv, H // Hkv, T, -1) / math.sqrt(D)
    scores = torch.where(seen, scores, -torch.inf)
    top = scores.amax(dim=-1, keepdim=True)
    e = torch.exp(scores - torch.where(top > -torch.inf, top, 0.0))
    p = e / e.sum(dim=-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(p.view(B, Hkv, -1, k.shape[2]), v).view(B, Hkv, H // Hkv, T, D)
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(_BF16)


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        if kind == "store":
            return _plain_store(case, state)
        return _plain_read(case, state, *_span(case, state)) if kind == "read" else _plain_attend(case, state)
    hlm = _hlm()
    counts = state["counts"] if case.get("ragged") else None
    if kind == "store":
        hlm.kv_cache_write_hip(state["cache"], state["k"], state["v"], state["starts"], counts)
    if kind in ("store", "read"):
        return hlm.kv_cache_read_hip(state["cache"], state["starts"], case["T"], counts)
    return hlm.cached_attention_hip(
        state["q"], state["cache"], state["starts"], counts, window_size=case["window"] or None,
        prefix=state.get("prefix"), prefix_length=case["prefix"],
    )


def work(case):
    """Bytes: the keys and values that some query sees (a prefix's once), new tokens and queries in, results out.  Flops: 4 D
    per query, visible key and head; a few for each value written or read."""
    Hkv, D, kind = case["Hkv"], case["D"], case["kind"]
    row = Hkv * D
    if kind in ("store", "read"):
        real, out = sum(_counts(case)), case["B"] * case["T"]
        once = 2 * real * Hkv * (D + 4)
        return {"bytes": (4 * real * row + once if kind == "store" else 0) + once + 4 * out * row, "flops": 4 * real * row}
    P, W = case["prefix"], case["window"] or 1 << 62
    keys, pairs, seen_from = 0, 0, P
    for first, n in zip(_starts(case), _counts(case)):
        at = P + first
        keys += first + n - max(0, at - W + 1 - P)
        seen_from = min(seen_from, max(0, at - W + 1))
        full = max(0, min(n, W - at))  # queries whose window reaches position 0
        pairs += full * at + full * (full + 1) // 2 + (n - full) * min(W, at + n)
    keys += P - seen_from
    q = case["B"] * case["T"] * case["H"] * D
    return {"bytes": 2 * 2 * q + 2 * keys * Hkv * (D + 4), "flops": 4 * D * pairs * case["H"]}


def _exact_rows(x):
    """Rows in 64 bits as a cache holds them."""
    x = x.double()
    top = x.abs().amax(dim=-1, keepdim=True)
    return torch.where(top > 0, torch.round(127 * x / top.clamp(min=1e-300)) * (top / 127), torch.zeros_like(x))


def exact(case, seed):
    s = _inputs(case, seed)
    B, T, Hkv, D = (case[x] for x in ("B", "T", "Hkv", "D"))
    first, n = s["starts"].tolist(), s["counts"].tolist()
    if case["kind"] in ("store", "read"):
        out = [torch.zeros((B, T, Hkv, D), device="cuda", dtype=torch.float64) for _ in "kv"]
        for b in range(B):
            for to, x in zip(out, (s["k"], s["v"]) if case["kind"] == "store" else s["cached"]):
                at = 0 if case["kind"] == "store" else first[b]
                to[b, : n[b]] = _exact_rows(x[b, at : at + n[b]])
        return tuple(out)
    H, P = case["H"], case["prefix"]
    G, W = H // Hkv, case["window"] or 1 << 40
    o = torch.zeros((B, T, H, D), device="cuda", dtype=torch.float64)
    shared = [_exact_rows(x[0]) for x in s["shared"]] if P else None
    for b in range(B):
        own_rows = [_exact_rows(x[b, : first[b] + n[b]]) for x in s["cached"]]
        k, v = [torch.cat(pair) for pair in zip(shared, own_rows)] if P else own_rows
        at = P + first[b] + torch.arange(n[b], device="cuda")
        place = torch.arange(k.shape[0], device="cuda")
        hidden = (place > at[:, None]) | (place <= at[:, None] - W)
        for h in range(H):
            kh, vh = k[:, h // G].contiguous(), v[:, h // G].contiguous()
            logits = torch.mm(s["q"][b, : n[b], h].double(), kh.t().contiguous()) * D**-0.5
            o[b, : n[b], h] = torch.mm(torch.softmax(logits.masked_fill(hidden, -math.inf), dim=-1), vh)
    return o
