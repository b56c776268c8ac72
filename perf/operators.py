"""The operators of a serving step over a paged key/value cache, as cases that can be timed and compared.

Four operators that a decoder needs once its requests have different lengths, come and go, and sample:

    tables   block table, slot map and positions of a step, built on the device from the requests' lengths
    write    rotary embedding of a prompt's (or a mixed batch's) q and k, k and v written into cache pages
    attend   one new token per request: rotary embedding, cache write, attention over the request's pages
    sample   the next token of every row: temperature, top-k, top-p, min-p, from given uniform numbers

With `own` false `run` computes each in plain torch operations; with `own` true it makes the calls of
`bitstack_b200.glue`.  Both take the same state."""
import math

import numpy as np
import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one decode step of a full server: every request grows by one token, a few are idle, some cross into a new page
        {"name": "tables-decode", "kind": "tables", "batch": 256, "page": 16, "max_len": 8191, "max_new": 1},
        # admission of a wave of prompts of very different lengths
        {"name": "tables-prompts", "kind": "tables", "batch": 64, "page": 16, "max_len": 4095, "max_new": 1024},
        # a prompt of the 8B head layout just below 2048 tokens
        {"name": "write-prompt", "kind": "write", "tokens": 2047, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "fp16"},
        # prompts and single tokens mixed in one batch, 70B head layout, with padding rows
        {"name": "write-mixed", "kind": "write", "tokens": 301, "q_heads": 64, "kv_heads": 8, "dim": 128, "page": 32, "dtype": "bf16"},
        # interactive use: one request, short context; latency counts
        {"name": "attend-one-short", "kind": "attend", "batch": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "max_len": 201, "dtype": "fp16"},
        # one request with a very long context
        {"name": "attend-one-long", "kind": "attend", "batch": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "max_len": 131071, "dtype": "fp16"},
        # the 70B head layout at batch 16, 256-token prompts and up to 128 decode steps
        {"name": "attend-70b-batch16", "kind": "attend", "batch": 16, "q_heads": 64, "kv_heads": 8, "dim": 128, "page": 16, "max_len": 384, "dtype": "fp16"},
        # a loaded server: 64 requests of ragged lengths, idle rows among them
        {"name": "attend-64-ragged", "kind": "attend", "batch": 64, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "max_len": 8192, "dtype": "fp16"},
        # many short requests of a small model
        {"name": "attend-128-small-heads", "kind": "attend", "batch": 128, "q_heads": 16, "kv_heads": 4, "dim": 64, "page": 24, "max_len": 1500, "dtype": "bf16"},
        # interactive use: one row of the 128256-token vocabulary
        {"name": "sample-one", "kind": "sample", "batch": 1, "vocab": 128256, "dtype": "fp16", "filters": "kp"},
        # a loaded server: rows with settings of their own, some masked, some greedy
        {"name": "sample-64-mixed", "kind": "sample", "batch": 64, "vocab": 128256, "dtype": "fp16", "filters": "mixed"},
        # 32-bit logits of a smaller vocabulary, nucleus sampling throughout
        {"name": "sample-256-nucleus", "kind": "sample", "batch": 256, "vocab": 32000, "dtype": "fp32", "filters": "p"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    kind = rng.choice(["tables", "write", "attend", "attend", "sample", "sample"])
    if kind == "tables":
        return {"kind": kind, "batch": _log(rng, 1, 600), "page": rng.choice([1, 8, 16, 24, 64, 128]), "max_len": _log(rng, 1, 20000),
                "max_new": rng.choice([1, 1, _log(rng, 2, 128)])}
    heads, kv = rng.choice([(32, 8), (64, 8), (8, 1), (16, 16), (12, 4), (24, 1), (5, 5)])
    if kind == "write":
        return {"kind": kind, "tokens": _log(rng, 1, 2047), "q_heads": heads, "kv_heads": kv, "dim": rng.choice([64, 128]),
                "page": rng.choice([8, 16, 24, 64]), "dtype": rng.choice(["fp16", "bf16"])}
    if kind == "attend":
        batch, dim = _log(rng, 1, 96), rng.choice([64, 128, 128])
        most = min(65536, int(5e8 / (batch * kv * dim * 4)))
        return {"kind": kind, "batch": batch, "q_heads": heads, "kv_heads": kv, "dim": dim, "page": rng.choice([1, 8, 16, 24, 64, 128]),
                "max_len": _log(rng, 1, most), "dtype": rng.choice(["fp16", "bf16"])}
    vocab = _log(rng, 100, 200000)
    return {"kind": kind, "batch": _log(rng, 1, min(256, max(1, 8000000 // vocab))), "vocab": vocab,
            "dtype": rng.choice(["fp16", "bf16", "fp32"]), "filters": rng.choice(["none", "k", "p", "kp", "mixed"])}


# ------------------------------------------------------------------------------------------------ inputs

def _lengths(batch, most):
    """Lengths from short to `most`, a third of `most` on average; which request has which goes by the seed."""
    return [most if i == batch - 1 else 1 + int((most - 1) * ((i + 0.5) / batch) ** 2) for i in range(batch)]


def _idle(batch):
    return batch // 16


def _tables_sizes(c):
    lens = _lengths(c["batch"], c["max_len"])
    if c["max_new"] == 1:
        new = [1] * (c["batch"] - _idle(c["batch"])) + [0] * _idle(c["batch"])
    else:
        new = _lengths(c["batch"], c["max_new"])
    return lens, new


def _rotary(max_len, dim, dtype, device):
    inv = 1.0 / (500000.0 ** (torch.arange(0, dim, 2, device=device, dtype=torch.float64) / dim))
    angle = torch.outer(torch.arange(max_len, device=device, dtype=torch.float64), inv)
    angle = torch.cat([angle, angle], dim=-1)
    return angle.cos().to(dtype), angle.sin().to(dtype)


def _normal(shape, dtype, gen):
    return torch.randn(shape, dtype=dtype, device="cuda", generator=gen)


def prepare(case, seed):
    c, dev = case, "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    if c["kind"] == "tables":
        lens, new = _tables_sizes(c)
        B, ps = c["batch"], c["page"]
        at = torch.randperm(B, device=dev, generator=gen)
        lens = torch.tensor(lens, dtype=torch.int32, device=dev)[at]
        new = torch.tensor(new, dtype=torch.int32, device=dev)[torch.randperm(B, device=dev, generator=gen)]
        held = (lens + ps - 1) // ps
        width = -(-(c["max_len"] + c["max_new"]) // ps)
        grow = int(((lens + new + ps - 1) // ps - held).sum())
        total = int(held.sum())
        pages = torch.randperm(total + grow + 7, device=dev, generator=gen).int()
        table = torch.full((B, width), -1, dtype=torch.int32, device=dev)
        mine = torch.arange(width, device=dev) < held[:, None]
        table[mine] = pages[:total]
        free = torch.full((total + grow + 7,), -1, dtype=torch.int32, device=dev)
        free[:grow + 7] = pages[total:]
        return {"kind": "tables", "lens": lens, "new": new, "table": table, "free": free,
                "count": torch.tensor([grow + 7], dtype=torch.int32, device=dev), "page": ps,
                "tokens": int(new.sum()) + 3, "lens_out": torch.empty_like(lens),
                "count_out": torch.empty(1, dtype=torch.int32, device=dev)}
    if c["kind"] == "sample":
        B, V, dtype = c["batch"], c["vocab"], _DTYPES[c["dtype"]]
        logits = _normal((B, V), torch.float32, gen) * 2.5
        top = torch.randint(0, V, (B, 24), device=dev, generator=gen)      # what a trained model's head gives: a few likely tokens
        logits.scatter_add_(1, top, 9.0 - 0.35 * torch.arange(24, device=dev, dtype=torch.float32).expand(B, 24))
        pick = lambda values, t: torch.tensor(values, dtype=t, device=dev)[torch.randint(0, len(values), (B,), device=dev, generator=gen)]  # noqa: E731
        s = {"kind": "sample", "temperature": pick([0.6, 0.7, 0.8, 1.0, 1.3], torch.float32), "top_k": None, "top_p": None, "min_p": None}
        if c["filters"] == "mixed":
            masked = torch.rand((B, 1), device=dev, generator=gen) < 0.25  # constrained decoding: tokens that may not come
            logits = torch.where(masked & (torch.rand((B, V), device=dev, generator=gen) < 0.3), -math.inf, logits)
            s["temperature"] = pick([0.0, 0.5, 0.7, 1.0, 1.0, 1.5], torch.float32)
            s["min_p"] = pick([0.0, 0.0, 0.02, 0.1], torch.float32)
        if c["filters"] in ("k", "kp", "mixed"):
            s["top_k"] = pick([0, 1, 20, 50, 50, 1000], torch.int32) if c["filters"] == "mixed" else pick([40, 50, 64], torch.int32)
        if c["filters"] in ("p", "kp", "mixed"):
            s["top_p"] = pick([1.0, 0.5, 0.9, 0.95], torch.float32) if c["filters"] == "mixed" else pick([0.8, 0.9, 0.95], torch.float32)
        s["logits"] = logits.to(dtype)
        s["uniforms"] = torch.rand((B,), device=dev, generator=gen)
        s["tokens"] = torch.zeros(B, dtype=torch.int64, device=dev)
        s["logprobs"] = torch.zeros(B, dtype=torch.float32, device=dev)
        return s
    dtype, ps, Hq, Hkv, D = _DTYPES[c["dtype"]], c["page"], c["q_heads"], c["kv_heads"], c["dim"]
    s = {"kind": c["kind"], "q_heads": Hq, "kv_heads": Hkv, "dim": D, "page": ps}
    if c["kind"] == "write":
        T = c["tokens"]
        pages = -(-T // ps) + 5
        s["cos"], s["sin"] = _rotary(4096, D, dtype, dev)
        first = int(torch.randint(0, 2000, (1,), device=dev, generator=gen))
        at = torch.arange(T, device=dev)
        s["positions"] = first + at
        order = torch.randperm(pages, device=dev, generator=gen)
        s["slots"] = order[(at + 3) // ps] * ps + (at + 3) % ps
        pad = T // 32                                                     # padding at the end of the batch
        if pad:
            s["positions"][T - pad:] = -1
            s["slots"][T - pad:] = -1
    else:
        T = c["batch"]
        lens = torch.tensor(_lengths(T, c["max_len"]), device=dev)
        if _idle(T):
            lens[1:1 + _idle(T)] = 0
        lens = lens[torch.randperm(T, device=dev, generator=gen)]
        s["positions"] = lens - 1                                          # idle rows: -1
        s["cos"], s["sin"] = _rotary(c["max_len"], D, dtype, dev)
        held = (lens + ps - 1) // ps
        total, width = int(held.sum()), -(-c["max_len"] // ps)
        pages = total + 3
        order = torch.randperm(pages, device=dev, generator=gen).int()
        s["table"] = torch.full((T, width), -1, dtype=torch.int32, device=dev)
        s["table"][torch.arange(width, device=dev) < held[:, None]] = order[:total]
    s["q"] = _normal((T, Hq * D), dtype, gen)
    s["k"] = _normal((T, Hkv * D), dtype, gen)
    s["v"] = _normal((T, Hkv * D), dtype, gen)
    s["k_pages"] = _normal((pages, Hkv, ps, D), dtype, gen)
    s["v_pages"] = _normal((pages, Hkv, ps, D), dtype, gen)
    return s


# ------------------------------------------------------------------------------------------------ the operators

def run(state):
    return _RUN[state["kind"]](state)


def _run_tables(s):
    if own:
        from bitstack_b200 import glue
        slots, positions, offsets, last = glue.page_tables(s["lens"], s["new"], s["table"], s["free"], s["count"], s["page"], s["tokens"],
                                                           lens_out=s["lens_out"], free_count_out=s["count_out"])
        return [s["table"], slots, positions, offsets, last, s["lens_out"], s["count_out"]]
    ps, lens, new, count = s["page"], s["lens"].long(), s["new"].long(), s["count"].long()
    B, width = s["table"].shape
    held, held_after = (lens + ps - 1) // ps, (lens + new + ps - 1) // ps
    fits = held_after <= width
    need = torch.where(fits, held_after - held, 0)
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= count))                        # pages go to the requests in their order, while there are any
    column = torch.arange(width, device=lens.device)
    fresh = served[:, None] & (column >= held[:, None]) & (column < held_after[:, None])
    source = count - 1 - ((upto - need)[:, None] + column - held[:, None])  # the free pages are a stack
    table = torch.where(fresh, s["free"][source.clamp(0, s["free"].numel() - 1)], s["table"])
    ends = new.cumsum(0)
    offsets = torch.cat([torch.zeros_like(ends[:1]), ends])
    token = torch.arange(s["tokens"], device=lens.device)
    row = torch.searchsorted(ends, token, right=True)
    real = row < B
    row = row.clamp(max=B - 1)
    real &= served[row]
    position = lens[row] + token - offsets[row]
    slot = table[row, (position // ps).clamp(0, width - 1)].long() * ps + position % ps
    last = torch.where(served & (new > 0), lens + new - 1, -1)
    return [table, torch.where(real, slot, -1), torch.where(real, position, -1), offsets.int(), last,
            torch.where(served, lens + new, lens).int(), (count - torch.where(served, need, 0).sum()).int()]


def _rotate(x, cos, sin):
    """x: [T, heads, D]; cos, sin: [T, D]; halves rotated against one another."""
    half = x.shape[-1] // 2
    return x * cos[:, None] + torch.cat([-x[..., half:], x[..., :half]], dim=-1) * sin[:, None]


def _run_write(s):
    Hq, Hkv, D, ps = s["q_heads"], s["kv_heads"], s["dim"], s["page"]
    if own:
        from bitstack_b200 import glue
        q = glue.rope_paged_cache(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["positions"], s["slots"], s["k_pages"], s["v_pages"], Hq, Hkv, D)
        return [q, s["k_pages"], s["v_pages"]]
    T, dtype = s["q"].shape[0], s["q"].dtype
    at = s["positions"].clamp(min=0)
    cos, sin = s["cos"][at].float(), s["sin"][at].float()
    q = _rotate(s["q"].view(T, Hq, D).float(), cos, sin)
    q = torch.where((s["positions"] >= 0)[:, None, None], q, 0.0).to(dtype).view(T, Hq * D)
    keep = torch.nonzero(s["slots"] >= 0).squeeze(1)
    page, row = s["slots"][keep] // ps, s["slots"][keep] % ps
    s["k_pages"][page, :, row] = _rotate(s["k"].view(T, Hkv, D).float(), cos, sin).to(dtype)[keep]
    s["v_pages"][page, :, row] = s["v"].view(T, Hkv, D)[keep]
    return [q, s["k_pages"], s["v_pages"]]


def _run_attend(s):
    Hq, Hkv, D, ps = s["q_heads"], s["kv_heads"], s["dim"], s["page"]
    if own:
        from bitstack_b200 import glue
        out = glue.paged_decode_attention(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["positions"], s["table"], s["k_pages"], s["v_pages"], Hq, Hkv, D)
        return [out, s["k_pages"], s["v_pages"]]
    B, dtype = s["q"].shape[0], s["q"].dtype
    live = s["positions"] >= 0
    at = s["positions"].clamp(min=0)
    cos, sin = s["cos"][at].float(), s["sin"][at].float()
    q = _rotate(s["q"].view(B, Hq, D).float(), cos, sin).view(B, Hkv, Hq // Hkv, D)
    busy = torch.nonzero(live).squeeze(1)
    page, row = s["table"][busy, at[busy] // ps].long(), at[busy] % ps
    s["k_pages"][page, :, row] = _rotate(s["k"].view(B, Hkv, D).float(), cos, sin).to(dtype)[busy]
    s["v_pages"][page, :, row] = s["v"].view(B, Hkv, D)[busy]
    table = s["table"].clamp(min=0).long()
    keys = s["k_pages"][table].transpose(1, 2).reshape(B, Hkv, -1, D).float()
    scores = q @ keys.transpose(2, 3) * (1.0 / math.sqrt(D))
    del keys
    seen = torch.arange(scores.shape[-1], device=q.device) <= s["positions"][:, None]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weight = torch.exp(scores - torch.where(live[:, None, None, None], top, 0.0))
    values = s["v_pages"][table].transpose(1, 2).reshape(B, Hkv, -1, D).float()
    out = (weight @ values) / weight.sum(-1, keepdim=True).clamp(min=1e-30)
    return [out.to(dtype).view(B, Hq * D), s["k_pages"], s["v_pages"]]


def _run_sample(s):
    if own:
        from bitstack_b200 import glue
        tokens = glue.sample_step(s["logits"], s["uniforms"], s["tokens"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], logprobs=s["logprobs"])
        return [tokens, s["logprobs"]]
    x = s["logits"].double()                                               # sums over a vocabulary, and borders between its tokens: 64 bits
    B, V = x.shape
    temperature = s["temperature"].double()[:, None]
    greedy = temperature <= 0
    order = torch.sort(x, dim=-1, descending=True, stable=True)            # ties: the lowest token first
    x, token = order.values, order.indices
    weight = torch.exp((x - x[:, :1]) / torch.where(greedy, 1.0, temperature))
    rank = torch.arange(V, device=x.device)
    keep = torch.ones_like(x, dtype=torch.bool)
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        keep &= (rank < k) | (k <= 0)
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        kept = torch.where(keep, weight, 0.0)
        before = kept.cumsum(-1) - kept
        keep &= (before < p * kept.sum(-1, keepdim=True)) | (p >= 1) | (rank == 0)
    if s["min_p"] is not None:
        keep &= weight >= s["min_p"].double()[:, None]
    keep &= ~greedy | (rank == 0)
    weight = torch.zeros_like(x).scatter_(1, token, torch.where(keep, weight, 0.0))   # back in the vocabulary's order
    upto = weight.cumsum(-1)
    total = upto[:, -1:]
    chosen = torch.searchsorted(upto, s["uniforms"].double()[:, None] * total, right=True).clamp(max=V - 1)
    return [chosen.squeeze(1), torch.log(weight.gather(1, chosen) / total).squeeze(1).float()]


_RUN = {"tables": _run_tables, "write": _run_write, "attend": _run_attend, "sample": _run_sample}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    c = case
    if c["kind"] == "tables":
        lens, new = _tables_sizes(c)
        tokens = sum(new) + 3
        # lengths and new counts in; offsets, lengths and last positions out; slot and position of every token; the pages that were taken
        return {"bytes": 4 * 2 * c["batch"] + (4 + 4 + 8) * c["batch"] + 16 * tokens + 8 * (tokens // c["page"] + 1), "flops": 8 * tokens}
    if c["kind"] == "sample":
        n = c["batch"] * c["vocab"]
        return {"bytes": n * (4 if c["dtype"] == "fp32" else 2) + 40 * c["batch"], "flops": 12 * n}
    Hq, Hkv, D = c["q_heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "write":
        T = c["tokens"]
        live = T - T // 32
        return {"bytes": live * (2 * (2 * Hq + 4 * Hkv) * D + 16 + 4 * D), "flops": 3 * live * (Hq + Hkv) * D}
    B = c["batch"]
    lens = _lengths(B, c["max_len"])
    lens[1:1 + _idle(B)] = [0] * _idle(B)
    rows = sum(lens)
    return {"bytes": rows * Hkv * D * 4 + B * (2 * Hq + 4 * Hkv) * D * 2 + 4 * sum(-(-n // c["page"]) for n in lens), "flops": 4 * rows * Hq * D}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return None if case["kind"] == "tables" else {"write": _exact_write, "attend": _exact_attend, "sample": _exact_sample}[case["kind"]](s)


def _turned(x, heads, D, cos, sin):
    """Each pair (x[i], x[i + D/2]) as a complex number, turned by its angle."""
    x = x.double().view(-1, heads, 2, D // 2)
    z = torch.complex(x[:, :, 0], x[:, :, 1])
    # the table may hold a cosine and a sine of its own for each half: they are rounded copies of one another
    turn = torch.complex(cos.double()[:, None, :D // 2], sin.double()[:, None, :D // 2])
    z = z * turn
    return torch.cat([z.real, z.imag], dim=-1)


def _exact_write(s):
    Hq, Hkv, D, ps = s["q_heads"], s["kv_heads"], s["dim"], s["page"]
    n = int((s["positions"] >= 0).sum())                                    # padding comes last
    cos, sin = s["cos"][s["positions"][:n]], s["sin"][s["positions"][:n]]
    q = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    q[:n] = _turned(s["q"][:n], Hq, D, cos, sin).view(n, Hq * D)
    k, v = s["k_pages"].double(), s["v_pages"].double()
    turned = _turned(s["k"][:n], Hkv, D, cos, sin)
    page, row = torch.div(s["slots"][:n], ps, rounding_mode="floor"), torch.remainder(s["slots"][:n], ps)
    k.permute(0, 2, 1, 3).index_put_((page, row), turned)
    v.permute(0, 2, 1, 3).index_put_((page, row), s["v"][:n].double().view(n, Hkv, D))
    return [q, k, v]


def _exact_attend(s):
    Hq, Hkv, D, ps = s["q_heads"], s["kv_heads"], s["dim"], s["page"]
    B = s["q"].shape[0]
    k, v = s["k_pages"].double(), s["v_pages"].double()
    out = torch.zeros((B, Hq, D), dtype=torch.float64, device="cuda")
    for b, p in enumerate(s["positions"].tolist()):
        if p < 0:
            continue
        cos, sin = s["cos"][p:p + 1], s["sin"][p:p + 1]
        q = _turned(s["q"][b], Hq, D, cos, sin)[0]
        pages = s["table"][b, :p // ps + 1].long()
        k[pages[-1], :, p % ps] = _turned(s["k"][b], Hkv, D, cos, sin)[0]
        v[pages[-1], :, p % ps] = s["v"][b].double().view(Hkv, D)
        for h in range(Hkv):
            keys, values = k[pages, h].reshape(-1, D)[:p + 1], v[pages, h].reshape(-1, D)[:p + 1]
            mine = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
            out[b, mine] = torch.softmax(q[mine] @ keys.t() / D ** 0.5, dim=-1) @ values
    return [out.view(B, Hq * D), k, v]


def _exact_sample(s):
    logits, u = s["logits"].double().cpu().numpy(), s["uniforms"].double().cpu().numpy()
    settings = {n: None if s[n] is None else s[n].cpu().numpy() for n in ("temperature", "top_k", "top_p", "min_p")}
    found = np.zeros(len(u))
    for b, x in enumerate(logits):
        t = float(settings["temperature"][b])
        if t <= 0:
            continue                                                         # a greedy row: its token has probability one
        order = np.argsort(-x, kind="stable")
        w = np.exp((x[order] - x[order[0]]) / t)
        n = len(x)
        if settings["top_k"] is not None and settings["top_k"][b] > 0:
            n = min(n, int(settings["top_k"][b]))
        if settings["top_p"] is not None and settings["top_p"][b] < 1:
            sums = np.cumsum(w[:n])
            n = min(n, 1 + int(np.searchsorted(sums, float(settings["top_p"][b]) * sums[-1], side="left")))
        if settings["min_p"] is not None:
            n = min(n, int(np.sum(w >= float(settings["min_p"][b]))))
        kept = np.sort(order[:n])
        w = np.exp((x[kept] - x[order[0]]) / t)
        sums = np.cumsum(w)
        at = min(int(np.searchsorted(sums, u[b] * sums[-1], side="right")), n - 1)
        found[b] = np.log(w[at] / sums[-1])
    return [None, torch.from_numpy(found)]
