"""The 4-bit key/value cache at work, as cases that can be timed and checked.

Three operators: quantising keys and values into a paged cache as they are written, reading them back, and attention
over the cache.  A case is one pass:

* op "write": the new tokens' keys and values go into the cache (`w4a16_kv.kv4_write`) and what the cache
  then holds of them is read back (`w4a16_kv.kv4_read`): the values that the codes stand for;
* op "read": the keys and values of whole sequences come back out of the cache (`w4a16_kv.kv4_read`);
* op "attn": attention of a batch's queries over the cache (`w4a16_kv.kv4_attention`).

A group of G values of one token and KV head is held as s (q - z): codes q in 0..15, s in fp16, z a multiple of
1/8 in fp16.  The cache is one byte tensor [pages, KV heads, P (D + 8 D / G)]; the bytes of one page and head hold,
for its P tokens,
  key codes   [P][D/2]          byte j: the codes of values j (low four bits) and j + D/2
  value codes [P/16][D/2][16]   the same byte of token t of 16 at place PLACE[t % 4] of its four
  key scales, key zeros, value scales, value zeros, each fp16 [D/G][P].

Head counts and sizes are the Llama-3 layers' (32 query and 8 KV heads, 64 and 8, 128 values a head) and generic
ones.  Inputs are made on the GPU from the seed alone.
"""
import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_entry = None


def _kv():
    """The framework's entry points."""
    global _entry
    if _entry is None:
        sys.path.insert(0, os.path.join(_ROOT, "w4a16-gemm_amd"))
        import w4a16_kv
        _entry = w4a16_kv
    return _entry


# ------------------------------------------------------------------------------------------- cases


def listed():
    def write(name, T, B, start, D, G, P, dtype, fused):
        # T new tokens of B sequences (ragged: see _shares) that already hold about `start` tokens
        return {"name": name, "op": "write", "T": T, "B": B, "start": start, "Hq": 32, "Hkv": 8, "D": D, "G": G, "P": P,
                "dtype": dtype, "fused": fused}

    def read(name, T, B, Hkv, D, G, P, dtype):
        return {"name": name, "op": "read", "T": T, "B": B, "Hkv": Hkv, "D": D, "G": G, "P": P, "dtype": dtype}

    def attn(name, B, q, lo, hi, Hq, Hkv, D, G, P, dtype, window=0, idle=0):
        # B sequences whose lengths spread from lo to hi, the last q tokens of each asking (q = 0: all of them);
        # idle: every idle-th sequence of the batch is empty
        return {"name": name, "op": "attn", "B": B, "q": q, "lo": lo, "hi": hi, "Hq": Hq, "Hkv": Hkv, "D": D, "G": G, "P": P,
                "dtype": dtype, "window": window, "idle": idle}

    return [
        # generating one token for one request: its keys and values join the cache
        write("write-step-1", 1, 1, 1000, 128, 128, 64, "fp16", True),
        # a ragged prompt's keys and values, slices of the fused qkv projection's output
        write("write-prompt-513", 513, 1, 0, 128, 128, 64, "fp16", True),
        # several prompts at once that continue what their caches hold, at any offset; groups of 64
        write("write-prompts-8192", 8192, 5, 300, 128, 64, 16, "bf16", False),
        # a shared prefix of small heads is read back, and a long context
        read("read-prefix-1000", 1000, 1, 8, 64, 64, 32, "bf16"),
        read("read-context-32768", 32768, 3, 8, 128, 128, 64, "fp16"),
        # one token of one request: a short context, where latency counts, and a long one
        attn("step-1x100", 1, 1, 100, 100, 32, 8, 128, 128, 64, "fp16"),
        attn("step-1x131072", 1, 1, 131072, 131072, 32, 8, 128, 128, 64, "fp16"),
        # one token of each of 64 requests of ragged lengths, some slots of the batch idle
        attn("step-64-ragged", 64, 1, 40, 8192, 32, 8, 128, 128, 16, "fp16", 0, 16),
        # five draft tokens to verify for each of four requests, wider grouping of the query heads
        attn("draft-5x4", 4, 5, 1000, 4100, 64, 8, 128, 64, 32, "bf16"),
        # a chunk of a long prompt over what the cache already holds
        attn("chunk-512-over-16k", 1, 512, 16384, 16384, 32, 8, 128, 128, 64, "bf16"),
        # ragged prompts of a model with small heads, no grouping, that looks back 400 tokens
        attn("prompts-ragged-window", 6, 0, 70, 2000, 16, 16, 64, 64, 16, "fp16", 400),
        # a whole prompt of 8192 tokens
        attn("prompt-8192", 1, 0, 8192, 8192, 32, 8, 128, 128, 64, "fp16"),
    ]


def _log(rng, lo, hi):
    return int(lo * (hi / lo) ** rng.random())


def draw(rng):
    D, G = rng.choice([(128, 128), (128, 128), (128, 64), (64, 64)])
    P, dtype = rng.choice([16, 32, 64, 128]), rng.choice(["fp16", "bf16"])
    kind = rng.random()
    if kind < 0.15:
        T = _log(rng, 1, 8192)
        return {"op": "write", "T": T, "B": min(T, rng.choice([1, 1, 3, 8, 32])), "start": rng.choice([0, rng.randint(1, 2000)]),
                "Hq": 32, "Hkv": 8, "D": D, "G": G, "P": P, "dtype": dtype, "fused": rng.random() < 0.5}
    if kind < 0.3:
        T = _log(rng, 20, 32768)
        return {"op": "read", "T": T, "B": min(T, rng.choice([1, 2, 5])), "Hkv": rng.choice([4, 8]), "D": D, "G": G, "P": P, "dtype": dtype}
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (64, 8), (16, 16), (28, 4), (8, 1)])
    c = {"op": "attn", "Hq": Hq, "Hkv": Hkv, "D": D, "G": G, "P": P, "dtype": dtype,
         "window": rng.choice([0, 0, 0, rng.randint(1, 1500)]), "idle": rng.choice([0, 0, 7])}
    if kind < 0.7:                                                    # single tokens and drafts
        B = _log(rng, 1, 64)
        hi = _log(rng, 20, 131072 // (B * max(1, Hkv // 8)))
        return {**c, "B": B, "q": rng.choice([1, 1, 1, 2, 4, 8]), "lo": max(1, hi // rng.choice([1, 10, 100])), "hi": hi}
    B = _log(rng, 1, 8)
    if kind < 0.85:                                                   # whole prompts
        hi = _log(rng, 40, min(8192, 8192 * 32 // (B * Hq)))
        return {**c, "B": B, "q": 0, "lo": max(1, hi // rng.choice([1, 4])), "hi": hi}
    hi = _log(rng, 40, 16384 // B)
    return {**c, "B": B, "q": max(1, _log(rng, 9, 600) // B), "lo": max(1, hi // rng.choice([1, 4])), "hi": hi}


def _shares(T, B):
    """T tokens as B ragged runs (each at least one)."""
    even = T // B
    runs = [even - (i * even) // (2 * B) for i in range(1, B)]
    return runs + [T - sum(runs)]


def _lengths(c):
    """The sequences' lengths and numbers of queries."""
    B, lo, hi = c["B"], c["lo"], c["hi"]
    L = [max(1, round(lo * (hi / lo) ** ((0.6180339887 * i) % 1.0))) for i in range(1, B + 1)]
    L[B // 2] = hi
    if c["idle"]:
        L = [0 if i % c["idle"] == c["idle"] - 1 else n for i, n in enumerate(L)]
    return L, [n if not c["q"] else (1 if c["q"] == 1 else min(n, c["q"])) for n in L]


def _attended(c):
    """Keys that the queries attend to, summed over the queries, and keys that any of them does, over the sequences."""
    pairs = keys = 0
    for n, m in zip(*_lengths(c)):
        if n == 0:
            continue
        w = c["window"] or n
        first = n - m + 1                                             # keys up to the first query's own
        full = max(0, n - max(first, w) + 1) if w < n else 0          # queries that see w keys
        short = m - full
        pairs += full * w + short * first + short * (short - 1) // 2
        keys += min(n, w + m - 1)
    return pairs, keys


def work(case):
    c = case
    D, G, Hkv = c["D"], c["G"], c["Hkv"]
    row = D + 8 * D // G                                              # cache bytes of a token and KV head
    if c["op"] == "write":                                            # read k and v, write the cache, read it, write the values
        return {"bytes": c["T"] * Hkv * (2 * row + 8 * D) + 16 * c["T"], "flops": c["T"] * Hkv * 2 * D * 8}
    if c["op"] == "read":
        return {"bytes": c["T"] * Hkv * (row + 4 * D) + 8 * c["T"], "flops": c["T"] * Hkv * 2 * D * 2}
    pairs, keys = _attended(c)
    T = sum(_lengths(c)[1])
    return {"bytes": keys * Hkv * row + T * c["Hq"] * D * 4, "flops": 4 * pairs * c["Hq"] * D}


# ------------------------------------------------------------------------------------------ inputs

PLACE = (0, 2, 1, 3)


def _dtype(c):
    return torch.float16 if c["dtype"] == "fp16" else torch.bfloat16


def _keys_values(c, T, g):
    """Keys as projections give them (some channels offset, a few much larger than the rest) and values; for "fused"
    both are slices of one projection's output."""
    H, D = c["Hkv"], c["D"]
    Hq = c["Hq"] if c.get("fused") else 0
    x = torch.randn(T, Hq + 2 * H, D, device="cuda", generator=g)
    gain = 1 + 4 * (torch.rand(H, D, device="cuda", generator=g) > 0.97)
    x[:, Hq:Hq + H] = x[:, Hq:Hq + H] * gain + 0.5 * torch.randn(H, D, device="cuda", generator=g)
    x = x.to(_dtype(c))
    k, v = x[:, Hq:Hq + H], x[:, Hq + H:]
    return (k, v) if Hq else (k.contiguous(), v.contiguous())


def _tables(c, lengths, g):
    """Each sequence's pages, in an order of their own, and how many pages the cache has."""
    P = c["P"]
    width = max(1, max(-(-n // P) for n in lengths))
    pages = width * len(lengths) + 3
    return torch.randperm(pages, device="cuda", generator=g)[:width * len(lengths)].view(len(lengths), width).int(), pages


def _slots(c, table, starts, counts):
    """Where tokens starts[b] .. starts[b] + counts[b] - 1 of each sequence b lie: page * P + place in it."""
    P = c["P"]
    n = torch.tensor(counts, device="cuda")
    b = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), n)
    t = torch.arange(b.numel(), device="cuda") - (n.cumsum(0) - n)[b] + torch.tensor(starts, device="cuda")[b]
    return table[b, t // P].long() * P + t % P


def _inputs(c, seed):
    """What a case works on: keys, values, their slots, queries and tables."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    if c["op"] == "attn":
        L, nq = _lengths(c)
        starts, counts = [0] * len(L), L
    else:
        counts = _shares(c["T"], c["B"])
        starts = [c["start"] and (c["start"] * (3 + 2 * i)) // 5 for i in range(c["B"])] if c["op"] == "write" else [0] * c["B"]
    table, pages = _tables(c, [a + n for a, n in zip(starts, counts)], g)
    k, v = _keys_values(c, sum(counts), g)
    d = {"k": k, "v": v, "table": table, "pages": pages, "slots": _slots(c, table, starts, counts), "counts": counts}
    if c["op"] == "attn":
        d["q"] = torch.randn(sum(nq), c["Hq"], c["D"], device="cuda", generator=g).to(_dtype(c))
        d["lens"] = torch.tensor(L, dtype=torch.int32, device="cuda")
        d["q_start"] = None
        if c["q"] != 1:
            d["q_start"] = torch.tensor([sum(nq[:i]) for i in range(len(nq) + 1)], dtype=torch.int32, device="cuda")
        d["max_q"] = max(nq) if c["q"] != 1 else 1
    return d


def _empty_cache(c, pages):
    return torch.zeros(pages, c["Hkv"], c["P"] * (c["D"] + 8 * c["D"] // c["G"]), dtype=torch.uint8, device="cuda")


def prepare(case, seed):
    d = _inputs(case, seed)
    d["case"], d["cache"] = case, _empty_cache(case, d["pages"])
    if case["op"] != "write":
        _plain_write(case, d["cache"], d["k"], d["v"], d["slots"])
        del d["k"], d["v"]
    return d


# ------------------------------------------------------------------------------- the plain forms


def _parts(c, cache):
    """Views of the cache: key codes [pages, H, P, D/2], value codes [pages, H, P/16, D/2, 16] and the key scales, key
    zeros, value scales and value zeros [pages, H, D/G, P]."""
    P, D, G = c["P"], c["D"], c["G"]
    half, side = P * D // 2, (D // G) * P * 2
    codes_k = cache[:, :, :half].unflatten(-1, (P, D // 2))
    codes_v = cache[:, :, half:2 * half].unflatten(-1, (P // 16, D // 2, 16))
    rest = cache[:, :, 2 * half:].view(torch.float16).unflatten(-1, (4, D // G, P))
    return codes_k, codes_v, rest


def _quantised(c, x):
    """Codes [T, H, D], scales and zeros [T, H, D/G] of x [T, H, D]."""
    x = x.float().clamp(-65504, 65504).unflatten(-1, (c["D"] // c["G"], c["G"]))
    lo, hi = x.amin(-1), x.amax(-1)
    s = torch.maximum((hi - lo) / 15, torch.maximum(lo.abs(), hi.abs()) / 96).clamp_min(2.0 ** -14).half()
    z = torch.round(-lo / s.float() * 8) / 8
    q = torch.round(x / s.float().unsqueeze(-1) + z.unsqueeze(-1)).clamp(0, 15)
    return q.flatten(-2).to(torch.uint8), s, z.half()


def _places(c, slots):
    """Page, place in it, 16-token tile and place in the tile's bytes of each slot."""
    page, t = slots // c["P"], slots % c["P"]
    return page, t, t // 16, (t % 16) // 4 * 4 + (t & 1) * 2 + ((t >> 1) & 1)


def _plain_write(c, cache, k, v, slots):
    codes_k, codes_v, rest = _parts(c, cache)
    page, t, tile, place = _places(c, slots)
    half = c["D"] // 2
    q, s, z = _quantised(c, k)
    codes_k[page, :, t] = q[..., :half] | (q[..., half:] << 4)
    rest[page, :, 0, :, t], rest[page, :, 1, :, t] = s, z
    q, s, z = _quantised(c, v)
    codes_v[page, :, tile, :, place] = q[..., :half] | (q[..., half:] << 4)
    rest[page, :, 2, :, t], rest[page, :, 3, :, t] = s, z


def _values(c, codes, s, z):
    """s (q - z) in 32 bits of packed codes [..., D/2], scales and zeros [..., D/G]."""
    q = torch.cat([codes & 15, codes >> 4], -1).float().unflatten(-1, (c["D"] // c["G"], c["G"]))
    return ((q - z.float().unsqueeze(-1)) * s.float().unsqueeze(-1)).flatten(-2)


def _plain_read(c, cache, slots):
    codes_k, codes_v, rest = _parts(c, cache)
    page, t, tile, place = _places(c, slots)
    k = _values(c, codes_k[page, :, t], rest[page, :, 0, :, t], rest[page, :, 1, :, t])
    return k, _values(c, codes_v[page, :, tile, :, place], rest[page, :, 2, :, t], rest[page, :, 3, :, t])


def _plain_attention(c, d):
    P, H, D, rep = c["P"], c["Hkv"], c["D"], c["Hq"] // c["Hkv"]
    q, table, lens = d["q"], d["table"], d["lens"]
    B, T, L, M = table.shape[0], q.shape[0], table.shape[1] * P, d["max_q"]
    at = torch.arange(L, device="cuda")
    k, v = _plain_read(c, d["cache"], (table.long()[:, at // P] * P + at % P).flatten())
    k, v = (x.view(B, L, H, D).permute(0, 2, 1, 3) for x in (k, v))
    first = d["q_start"].long() if d["q_start"] is not None else torch.arange(B + 1, device="cuda")
    count = first[1:] - first[:-1]
    i = torch.arange(M, device="cuda")
    rows = q.float()[(first[:-1, None] + i).clamp_max(T - 1)]                          # [B, M, Hq, D]
    rows = rows.view(B, M, H, rep, D).permute(0, 2, 3, 1, 4).reshape(B, H, rep * M, D)
    pos = (lens.long() - count)[:, None] + i                                           # [B, M]: each query's place
    seen = (at <= pos[..., None]) & (at < lens.long()[:, None, None])
    if c["window"]:
        seen &= at > pos[..., None] - c["window"]
    x = torch.matmul(rows, k.transpose(-1, -2).contiguous()).view(B, H, rep, M, L) * (D ** -0.5)
    x = x.masked_fill_(~seen[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    out = torch.matmul(x.view(B, H, rep * M, L), v.contiguous()).view(B, H, rep, M, D)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).reshape(B, M, c["Hq"], D)
    token = torch.arange(T, device="cuda")
    b = torch.bucketize(token, first[1:], right=True)
    return out[b, token - first[b]].to(q.dtype)


def run(state):
    d = state
    c = d["case"]
    if own:
        kv = _kv()
        if c["op"] == "attn":
            return kv.kv4_attention(d["q"], d["cache"], d["table"], d["lens"], c["G"], q_start=d["q_start"], max_q=d["max_q"],
                                    window=c["window"])
        if c["op"] == "write":
            kv.kv4_write(d["cache"], d["k"], d["v"], d["slots"], c["G"])
        return kv.kv4_read(d["cache"], d["slots"], c["D"], c["G"], _dtype(c))
    if c["op"] == "attn":
        return _plain_attention(c, d)
    if c["op"] == "write":
        _plain_write(c, d["cache"], d["k"], d["v"], d["slots"])
    k, v = _plain_read(c, d["cache"], d["slots"])
    return k.to(_dtype(c)), v.to(_dtype(c))


# ------------------------------------------------------------------------------------ in 64 bits


def _held(c, x):
    """The values in 64 bits that the cache holds of x [T, H, D]: the format's definition, s rounded to fp16."""
    w = x.double().reshape(x.shape[0], x.shape[1], -1, c["G"])
    low, high = w.min(-1, keepdim=True)[0], w.max(-1, keepdim=True)[0]
    step = torch.stack([(high - low) / 15, low.abs() / 96, high.abs() / 96, torch.full_like(low, 2.0 ** -14)]).max(0)[0]
    step = step.to(torch.float16).double()
    zero = torch.round(-low / step * 8) / 8
    code = torch.round(w / step + zero)
    return (step * (torch.minimum(torch.maximum(code, torch.zeros_like(code)), torch.full_like(code, 15)) - zero)).reshape(x.shape)


def exact(case, seed):
    c, d = case, _inputs(case, seed)
    k, v = _held(c, d["k"]), _held(c, d["v"])
    if c["op"] != "attn":
        return k, v
    out = torch.zeros(d["q"].shape, dtype=torch.float64, device="cuda")
    L, nq = _lengths(c)
    rep, key, query = c["Hq"] // c["Hkv"], 0, 0
    for n, m in zip(L, nq):
        for h in range(c["Hkv"] if n else 0):
            kh, vh = k[key:key + n, h], v[key:key + n, h]
            for a in range(0, m, 1024):                               # queries a .. b - 1 of the sequence
                b = min(m, a + 1024)
                own_place = torch.arange(n - m + a, n - m + b, device="cuda")[:, None]
                place = torch.arange(n, device="cuda")[None]
                away = (place > own_place) | ((place <= own_place - c["window"]) if c["window"] else (place < 0))
                for r in range(h * rep, (h + 1) * rep):
                    y = d["q"][query + a:query + b, r].double() @ kh.t().contiguous() / math.sqrt(c["D"])
                    out[query + a:query + b, r] = torch.softmax(y.masked_fill(away, float("-inf")), -1) @ vh
        key, query = key + n, query + m
    return out
