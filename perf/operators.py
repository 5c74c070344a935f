"""Operators that serve requests of different lengths, for timing and for comparing outputs.

  append   ops.paged_append: keys and values of new tokens enter a paged cache, q and k rotated on the way
  decode   ops.paged_attention: one new token per sequence over its pages
  packed   ops.packed_attention: causal attention over whole prompts of different lengths, packed row after row
  sample   ops.sample_tokens: temperature, top-k, top-p and min-p from given uniform numbers

Sizes are those of this repository's decoders (32 query heads over 8 key/value heads of 128, bf16: Ninolorn 7b; 32 heads of 128
and 12 of 64, fp16: OPT 6.7b and 125m; a vocabulary of 50272) or generic. With `own` false the operators run in elementary torch
operations in 32 bits (angles and sampling in 64), else as a user calls them.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one interactive user: the new token's key and value
        {"name": "append_1", "op": "append", "form": "step", "batch": 1, "tokens": 2000, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "dtype": "bf16", "rot": 64, "interleaved": False, "shape": 1},
        # prompts of several requests, some continued, enter the cache together
        {"name": "append_prompts", "op": "append", "form": "prompts", "batch": 7, "tokens": 8191, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "dtype": "bf16", "rot": 64, "interleaved": False, "shape": 2},
        # a short conversation of one user, small model: latency
        {"name": "decode_1_short", "op": "decode", "batch": 1, "tokens": 137, "heads": 12, "kv_heads": 12, "dim": 64, "page": 16,
         "dtype": "fp16", "shape": 3},
        # a very long document of one user
        {"name": "decode_1_long", "op": "decode", "batch": 1, "tokens": 131071, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "dtype": "bf16", "shape": 4},
        # many users with contexts from nothing to long
        {"name": "decode_64_ragged", "op": "decode", "batch": 64, "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "dtype": "bf16", "shape": 5},
        # a batch of OPT 6.7b: no grouped heads, larger pages
        {"name": "decode_16_opt", "op": "decode", "batch": 16, "tokens": 2048, "heads": 32, "kv_heads": 32, "dim": 128, "page": 64,
         "dtype": "fp16", "shape": 6},
        # a handful of short prompts, small model: latency
        {"name": "packed_short", "op": "packed", "batch": 5, "tokens": 333, "heads": 12, "kv_heads": 12, "dim": 64, "dtype": "fp16",
         "shape": 7},
        # prompts of a busy server
        {"name": "packed_ragged", "op": "packed", "batch": 24, "tokens": 16384, "heads": 32, "kv_heads": 8, "dim": 128,
         "dtype": "bf16", "shape": 8},
        # one long document of odd length
        {"name": "packed_long", "op": "packed", "batch": 1, "tokens": 16001, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16",
         "shape": 9},
        # one interactive user with the usual settings
        {"name": "sample_1", "op": "sample", "batch": 1, "vocab": 50272, "dtype": "fp32", "temperature": 0.8, "top_k": 50,
         "top_p": 0.95, "min_p": 0.0, "mixed": False, "spread": 2.5},
        # users with settings of their own, greedy ones among them
        {"name": "sample_256_mixed", "op": "sample", "batch": 256, "vocab": 50272, "dtype": "fp32", "temperature": 1.0, "top_k": 0,
         "top_p": 0.9, "min_p": 0.05, "mixed": True, "spread": 2.5},
        # half-precision logits of a large vocabulary, nucleus only
        {"name": "sample_32_nucleus", "op": "sample", "batch": 32, "vocab": 151936, "dtype": "bf16", "temperature": 1.0, "top_k": 0,
         "top_p": 0.9, "min_p": 0.0, "mixed": False, "spread": 2.5},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    op = rng.choice(("append", "decode", "packed", "sample"))
    heads, kv_heads = rng.choice(((32, 8), (32, 32), (12, 12), (16, 2), (24, 8), (8, 1), (40, 10)))
    case = {"op": op, "heads": heads, "kv_heads": kv_heads, "shape": rng.randrange(10 ** 6)}
    if op == "sample":
        batch = log(1, 256)
        return {"op": op, "batch": batch, "vocab": log(1000, min(262144, 256 * 50272 // batch)),
                "dtype": rng.choice(("fp32", "bf16", "fp16")), "temperature": round(rng.uniform(0.3, 2.0), 3),
                "top_k": rng.choice((0, 0, 1, log(2, 1000))), "top_p": rng.choice((1.0, round(rng.uniform(0.05, 0.999), 3))),
                "min_p": rng.choice((0.0, round(rng.uniform(0.001, 0.3), 4))), "mixed": rng.random() < 0.3,
                "spread": round(rng.uniform(0.5, 4.0), 2)}
    if op == "packed":
        case.update(batch=log(1, 64), dim=rng.choice((64, 80, 96, 128)), dtype=rng.choice(("bf16", "fp16")))
        case["tokens"] = max(case["batch"], log(1, 16001 if heads <= 32 else 12000))
        return case
    case.update(dim=rng.choice((32, 64, 80, 96, 128, 256)), dtype=rng.choice(("bf16", "fp16", "fp32")),
                page=rng.choice((16, 24, 32, 64, 128)), batch=log(1, 64))
    most = 2 ** 30 // (2 * kv_heads * case["dim"] * BYTES[case["dtype"]])  # cached tokens in a gigabyte
    if op == "decode":
        case["tokens"] = log(1, max(1, min(131071, most // case["batch"])))
        return case
    form = rng.choice(("step", "prompts"))
    case.update(form=form, rot=rng.choice((0, case["dim"] // 2, case["dim"] // 4)), interleaved=rng.random() < 0.5)
    case["tokens"] = log(1, 4000) if form == "step" else max(case["batch"], log(1, 8192 * 32 // heads))
    return case


def _lengths(case):
    """Lengths of the sequences, the same for every seed. decode: cached tokens up to `tokens`, the first has them all, and of
    many one has none. packed and append: rows that add up to `tokens`, one sequence of several without any."""
    r, B, n = random.Random(case["shape"]), case["batch"], case["tokens"]
    if case["op"] == "decode" or case.get("form") == "step":
        out = [n] + [r.randint(1, n) for _ in range(B - 1)]
        if B >= 8 and case["op"] == "decode":
            out[B // 2] = 0
        return out
    if B == 1:
        return [n]
    share = [r.random() ** 2 + 0.02 for _ in range(B)]
    if B >= 4:
        share[1] = 0.0
    out = [int(n * s / sum(share)) for s in share]
    out[0] += n - sum(out)
    return out


def _past(case):
    """Tokens that each sequence of an append holds before."""
    if case["form"] == "step":
        return _lengths(case)
    r = random.Random(case["shape"] + 1)
    return [r.choice((0, r.randint(0, 500))) for _ in range(case["batch"])]


def _table(lengths, page, gen):
    """Pages dealt out in random order, and how many there are; entries behind a sequence's last page are -1."""
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device=DEV).int()
    table = torch.full((len(lengths), max(1, max(need))), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def rnd(*shape, dtype=None):
        return torch.randn(*shape, device=DEV, generator=gen).to(dtype or TYPES[case["dtype"]])

    state = {"case": case}
    if case["op"] == "sample":
        B, V = case["batch"], case["vocab"]
        x = torch.randn(B, V, device=DEV, generator=gen) * case["spread"]
        # a few tokens stand out, as a trained model's do, by as much as the row is sure
        peaks = torch.randint(0, V // 8, (B, 8), device=DEV, generator=gen) + torch.arange(8, device=DEV) * (V // 8)
        height = torch.rand(B, 8, device=DEV, generator=gen) * torch.rand(B, 1, device=DEV, generator=gen)
        x.scatter_(1, peaks, x.gather(1, peaks) + 6 * case["spread"] * height)
        x[:, V // 3:V // 3 + 16] = -math.inf  # ids that no token has
        state["logits"], state["uniform"] = x.to(TYPES[case["dtype"]]), torch.rand(B, device=DEV, generator=gen)
        state["temperature"], state["top_k"], state["top_p"], state["min_p"] = (case[n] for n in ("temperature", "top_k", "top_p", "min_p"))
        if case["mixed"]:  # a tensor of each setting, one entry per row
            r = random.Random(seed)
            rows = [(r.choice((0.0, 0.7, 1.0, 1.3)), r.choice((0, 1, 20, 50, 400)), r.choice((1.0, 0.95, 0.8, 0.5)), r.choice((0.0, 0.02, 0.1)))
                    for _ in range(B)]
            t, k, p, m = zip(*rows)
            state["temperature"], state["top_k"] = torch.tensor(t, device=DEV), torch.tensor(k, dtype=torch.int32, device=DEV)
            state["top_p"], state["min_p"] = torch.tensor(p, device=DEV), torch.tensor(m, device=DEV)
        return state
    H, G, D, lengths = case["heads"], case["kv_heads"], case["dim"], _lengths(case)
    state.update(lengths=lengths, scale=D ** -0.5)
    if case["op"] == "packed":
        # rows of the fused projection, q | k | v
        T = sum(lengths)
        state["qkv"] = rnd(T, (H + 2 * G) * D)
        state["cu"] = torch.tensor([0] + lengths, device=DEV).cumsum(0).int()
        return state
    S, dt = case["page"], TYPES[case["dtype"]]
    if case["op"] == "decode":
        state["table"], P = _table(lengths, S, gen)
        # nobody has written to what is behind a sequence's end
        pages = torch.full((2, P, G, S, D), math.nan, dtype=dt, device=DEV)
        for b, n in enumerate(lengths):
            if n:
                used = rnd(2, -(-n // S), G, S, D)
                if n % S:
                    used[:, -1, :, n % S:] = math.nan
                pages[:, state["table"][b, :-(-n // S)].long()] = used
        state["k_pages"], state["v_pages"] = pages[0], pages[1]
        state["q"] = rnd(len(lengths), H, D)
        state["pos"] = torch.tensor(lengths, device=DEV) - 1
        return state
    past = _past(case)
    rows = [1] * len(past) if case["form"] == "step" else lengths
    state["rows"], state["past"] = rows, past
    state["table"], P = _table([a + n for a, n in zip(past, rows)], S, gen)
    state["k_pages"], state["v_pages"] = rnd(P, G, S, D), rnd(P, G, S, D)
    state["qkv"] = rnd(sum(rows), (H + 2 * G) * D)
    state["pos"] = torch.tensor(past, device=DEV)
    state["cu"] = None if case["form"] == "step" else torch.tensor([0] + rows, device=DEV).cumsum(0).int()
    half = case["rot"]
    state["freqs"] = (10000.0 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)).float() if half else None
    return state


def _split(state):
    """q (T, H, D), k and v (T, G, D): views of the fused projection's rows."""
    H, G, D = (state["case"][n] for n in ("heads", "kv_heads", "dim"))
    q, k, v = state["qkv"].split((H * D, G * D, G * D), dim=1)
    return q.unflatten(1, (H, D)), k.unflatten(1, (G, D)), v.unflatten(1, (G, D))


# ---- the user's calls ------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _own_append(s):
    from dejavu_b200 import ops

    q, k, v = _split(s)
    prompts = s["cu"] is not None
    q_rot, k_rot = ops.paged_append(q, k, v, s["k_pages"], s["v_pages"], s["table"], s["pos"], cu_seqlens=s["cu"], freqs=s["freqs"],
                                    interleaved=s["case"]["interleaved"], keys=prompts)
    out = {"q": q_rot, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if prompts:
        out["k"] = k_rot
    return out


def _own_decode(s):
    from dejavu_b200 import ops

    return ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["pos"], s["scale"])


def _own_packed(s):
    from dejavu_b200 import ops

    q, k, v = _split(s)
    return ops.packed_attention(q, k, v, s["cu"], s["scale"])


def _own_sample(s):
    from dejavu_b200 import ops

    return ops.sample_tokens(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                             min_p=s["min_p"])


_OWN = {"append": _own_append, "decode": _own_decode, "packed": _own_packed, "sample": _own_sample}


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _rotated(x, positions, freqs, interleaved):
    """x (T, heads, D): pairs (i, i + half), or neighbours, of the first 2 * half dimensions; angles in 64 bits."""
    if freqs is None:
        return x.float()
    half = freqs.numel()
    angle = positions.double()[:, None] * freqs.double()
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = x.float()
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    ra, rb = a * c - b * s, b * c + a * s
    head = torch.stack((ra, rb), -1).flatten(-2) if interleaved else torch.cat((ra, rb), -1)
    return torch.cat((head, x[..., 2 * half:]), -1)


def _plain_append(s):
    q, k, v = _split(s)
    case, dt, rows, S = s["case"], s["qkv"].dtype, s["rows"], s["case"]["page"]
    if s["cu"] is None:
        b = torch.arange(len(rows), device=DEV)
        positions = s["pos"]
    else:
        cu = s["cu"].long()
        b = torch.repeat_interleave(cu[1:] - cu[:-1], output_size=q.shape[0])
        positions = s["pos"][b] + torch.arange(q.shape[0], device=DEV) - cu[:-1][b]
    q_rot = _rotated(q, positions, s["freqs"], case["interleaved"]).to(dt)
    k_rot = _rotated(k, positions, s["freqs"], case["interleaved"]).to(dt)
    page = s["table"][b, positions // S].long()
    s["k_pages"][page, :, positions % S] = k_rot
    s["v_pages"][page, :, positions % S] = v
    out = {"q": q_rot, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if s["cu"] is not None:
        out["k"] = k_rot
    return out


def _attend(q, k, v, scale, first=None):
    """q (G, R, n, D), k and v (G, L, D), fp32. first: the number of keys that the first of the n queries sees, the next ones see one
    more each; None: all."""
    G, R, n, D = q.shape
    scores = (q.reshape(G, R * n, D) @ k.transpose(1, 2)).view(G, R, n, -1) * scale
    if first is not None:
        unseen = torch.arange(k.shape[1], device=DEV) >= torch.arange(n, device=DEV)[:, None] + first
        scores.masked_fill_(unseen, -math.inf)
    w = torch.exp(scores - scores.amax(-1, keepdim=True))
    total = w.sum(-1, keepdim=True)
    return (w.view(G, R * n, -1) @ v).view(G, R, n, D) / total


def _plain_decode(s):
    q, (B, H, D), G = s["q"], s["q"].shape, s["case"]["kv_heads"]
    out = torch.zeros_like(q)
    for b, n in enumerate(s["lengths"]):
        if n == 0:
            continue
        pages = s["table"][b, :-(-n // s["case"]["page"])].long()
        k, v = (x[pages].float().transpose(0, 1).flatten(1, 2)[:, :n] for x in (s["k_pages"], s["v_pages"]))
        out[b] = _attend(q[b].float().view(G, H // G, 1, D), k, v, s["scale"]).view(H, D).to(q.dtype)
    return out


def _plain_packed(s, rows=1024):
    q, k, v = _split(s)
    (T, H, D), G = q.shape, k.shape[1]
    out = torch.empty(T, H, D, dtype=q.dtype, device=DEV)
    start = 0
    for n in s["lengths"]:
        for a in range(0, n, rows):
            e = min(n, a + rows)
            qs = q[start + a:start + e].float().transpose(0, 1).reshape(G, H // G, e - a, D)
            ks, vs = (x[start:start + e].float().transpose(0, 1) for x in (k, v))
            o = _attend(qs, ks, vs, s["scale"], first=a + 1)
            out[start + a:start + e] = o.view(H, e - a, D).transpose(0, 1).to(q.dtype)
        start += n
    return out


def _plain_sample(s):
    x = s["logits"]
    B, V = x.shape

    def column(value, dtype=torch.float64):
        return value.to(dtype)[:, None] if torch.is_tensor(value) else torch.full((B, 1), value, dtype=dtype, device=DEV)

    T, p, min_p, k = column(s["temperature"]), column(s["top_p"]), column(s["min_p"]), column(s["top_k"], torch.int64)
    x = torch.where(x.isnan(), -math.inf, x).double()
    greedy = T == 0
    z = x / torch.where(greedy, 1.0, T)
    w = torch.exp(z - z.amax(1, keepdim=True))
    ranked, order = torch.sort(w, dim=1, descending=True, stable=True)  # (of equal ones the lowest index first)
    rank = torch.arange(V, device=DEV)[None]
    kept = rank < torch.where(greedy, 1, torch.where(k <= 0, V, k))
    ranked = ranked * kept
    before = ranked.cumsum(1) - ranked
    kept &= (p >= 1) | (before < p * ranked.sum(1, keepdim=True)) | (rank == 0)
    kept &= ranked >= min_p
    w = w * torch.zeros_like(kept).scatter_(1, order, kept)
    run = w.cumsum(1)
    return (run > s["uniform"].double()[:, None] * run[:, -1:]).int().argmax(1)


_PLAIN = {"append": _plain_append, "decode": _plain_decode, "packed": _plain_packed, "sample": _plain_sample}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "sample":
        n = case["batch"] * case["vocab"]
        return {"bytes": n * e + 12 * case["batch"], "flops": 4 * n}
    H, G, D, lengths = case["heads"], case["kv_heads"], case["dim"], _lengths(case)
    if case["op"] == "decode":
        T = sum(lengths)
        entries = sum(-(-n // case["page"]) for n in lengths)
        return {"bytes": (2 * T * G * D + 2 * len(lengths) * H * D) * e + 4 * entries + 8 * len(lengths), "flops": 4 * T * H * D}
    if case["op"] == "packed":
        pairs = sum(n * (n + 1) // 2 for n in lengths)
        return {"bytes": sum(lengths) * (2 * H + 2 * G) * D * e, "flops": 4 * pairs * H * D}
    T = len(lengths) if case["form"] == "step" else sum(lengths)
    keys_out = G if case["form"] == "prompts" else 0
    return {"bytes": T * (2 * H + 4 * G + keys_out) * D * e, "flops": 6 * T * (H + G) * case["rot"]}


# ---- the operators from their definitions, in 64 bits ---------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "decode": _exact_decode, "packed": _exact_packed, "sample": _exact_sample}[case["op"]](s)


def _exact_append(s):
    case = s["case"]
    H, G, D, S = case["heads"], case["kv_heads"], case["dim"], case["page"]
    x = s["qkv"].double().view(-1, H + 2 * G, D)
    table = s["table"].tolist()
    where = [(table[b][p // S], p % S, p) for b, (a, n) in enumerate(zip(s["past"], s["rows"])) for p in range(a, a + n)]
    page, slot, p = torch.tensor(where, device=DEV).unbind(1)
    if s["freqs"] is not None:  # a rotation is a product with exp(i angle)
        half = s["freqs"].numel()
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), torch.outer(p.double(), s["freqs"].double()))[:, None]
        first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else (slice(0, half), slice(half, 2 * half))
        y = torch.complex(x[:, :H + G, first], x[:, :H + G, second]) * turn
        x = x.clone()
        x[:, :H + G, first], x[:, :H + G, second] = y.real, y.imag
    q, k, v = x.split((H, G, G), dim=1)
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    k_pages[page, :, slot], v_pages[page, :, slot] = k, v
    out = {"q": q, "k_pages": k_pages, "v_pages": v_pages}
    if s["cu"] is not None:
        out["k"] = k
    return out


def _exact_decode(s):
    q, G = s["q"].double() * s["scale"], s["case"]["kv_heads"]
    B, H, D = q.shape
    out = torch.zeros_like(q)
    for b, n in enumerate(s["lengths"]):
        for g in range(G if n else 0):
            pages = s["table"][b, :-(-n // s["case"]["page"])].long()
            k, v = (x[pages, g].double().reshape(-1, D)[:n] for x in (s["k_pages"], s["v_pages"]))
            heads = slice(g * (H // G), (g + 1) * (H // G))
            out[b, heads] = torch.softmax(q[b, heads] @ k.t(), 1) @ v
    return out


def _exact_packed(s):
    H, G, D = (s["case"][n] for n in ("heads", "kv_heads", "dim"))
    x = s["qkv"].double().view(-1, H + 2 * G, D)
    out, start = torch.empty(x.shape[0], H, D, dtype=torch.float64, device=DEV), 0
    for n in s["lengths"]:
        y = x[start:start + n]
        for h in range(H):
            k, v = y[:, H + h // (H // G)], y[:, H + G + h // (H // G)]
            for a in range(0, n, 4096):
                e = min(n, a + 4096)
                z = (y[a:e, h] * s["scale"]) @ k[:e].t()
                z += torch.full_like(z, -math.inf).triu_(a + 1)
                out[start + a:start + e, h] = torch.softmax(z, 1) @ v[:e]
        start += n
    return out


def _exact_sample(s):
    import numpy as np

    x, u = s["logits"].double().cpu().numpy(), s["uniform"].double().cpu().numpy()
    B, V = x.shape
    settings = [np.broadcast_to(v.cpu().numpy() if torch.is_tensor(v) else v, B) for v in (s["temperature"], s["top_k"], s["top_p"], s["min_p"])]
    out = []
    for row, r, T, k, p, m in zip(x, u, *settings):
        if T == 0:
            out.append(int(np.argmax(row)))
            continue
        order = np.argsort(-row, kind="stable")
        if k > 0:
            order = order[:k]
        w = np.exp((row[order] - row[order[0]]) / np.float64(T))
        if p < 1:
            w = w[:max(1, int(np.searchsorted(np.cumsum(w), np.float64(p) * w.sum(), side="left")) + 1)]
        w = w[w >= np.float64(m)]
        kept = np.sort(order[:len(w)])
        run = np.cumsum(np.exp((row[kept] - row[order[0]]) / np.float64(T)))
        out.append(int(kept[np.searchsorted(run, r * run[-1], side="right")]))
    return torch.tensor(out, device=DEV)
