"""Timed cases of the operators that stand between a block's projections when
many requests are served at once, on one GPU.

``listed()`` holds the fixed cases and ``draw(rng)`` makes one more of the
same ranges.  A case is a dict of plain values; its ``kind`` names the
operator:

  step    page_step: pages, slots and positions of a step's new tokens from
          the requests' lengths
  append  cache_append: rotary positions on q and k, k and v written to their
          slots of the paged cache
  attend  paged_attention: each new token's attention over its request's pages
  adapt   adapter_add: the requests' low-rank adapters beside a projection

``run`` computes them with elementary torch operations in 32 bits, or, where
``own`` is true, through the library's entry points.  Projection shapes and
heads are those of ``libortho_amd.workloads`` (4096 -> 4096 as 32 heads of
128, 4096 -> 11008, 11008 -> 4096) and generic ones beside them.
"""
import math
import random

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one decode step of a small server: 16 requests, a token each
        {"name": "step-16", "kind": "step", "requests": 16, "prompts": 0, "longest": 4096, "prompt": 0, "page": 16},
        # a large server's step: 448 requests decode, 64 bring prompts
        {"name": "step-512", "kind": "step", "requests": 512, "prompts": 64, "longest": 8192, "prompt": 1024,
         "page": 32},
        # q, k, v of four requests' tokens, heads of the 4096-wide block
        {"name": "append-4", "kind": "append", "tokens": 4, "heads": 32, "kv_heads": 32, "dim": 128, "rot": 128,
         "interleaved": False, "page": 16, "dtype": "bf16"},
        # a long prompt with shared key heads
        {"name": "append-2048", "kind": "append", "tokens": 2048, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "interleaved": False, "page": 32, "dtype": "fp16"},
        # one user, a short conversation: launch and latency count
        {"name": "attend-1-short", "kind": "attend", "requests": 1, "shortest": 190, "longest": 190, "context": 4096,
         "heads": 32, "kv_heads": 32, "dim": 128, "window": 0, "page": 16, "dtype": "fp16"},
        # one user, a long document, shared key heads: few rows, a long axis
        {"name": "attend-1-long", "kind": "attend", "requests": 1, "shortest": 32768, "longest": 32768,
         "context": 32768, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "page": 64, "dtype": "bf16"},
        # a serving batch of the 4096-wide block, ragged lengths
        {"name": "attend-32", "kind": "attend", "requests": 32, "shortest": 16, "longest": 4096, "context": 4096,
         "heads": 32, "kv_heads": 32, "dim": 128, "window": 0, "page": 16, "dtype": "fp16"},
        # heads of an odd width over a window of the cache
        {"name": "attend-40-window", "kind": "attend", "requests": 40, "shortest": 1, "longest": 6000,
         "context": 8192, "heads": 20, "kv_heads": 4, "dim": 80, "window": 1000, "page": 16, "dtype": "fp16"},
        # a large batch of long conversations: the largest call, memory-bound
        {"name": "attend-128", "kind": "attend", "requests": 128, "shortest": 2048, "longest": 16384,
         "context": 16384, "heads": 64, "kv_heads": 8, "dim": 128, "window": 0, "page": 32, "dtype": "bf16"},
        # one user's adapter beside one projection
        {"name": "adapt-1", "kind": "adapt", "tokens": 1, "adapters": 1, "bare": 0, "runs": False, "K": 4096,
         "N": 4096, "rank": 16, "dtype": "fp16"},
        # a decode batch whose requests share 24 adapters, some without one
        {"name": "adapt-48", "kind": "adapt", "tokens": 48, "adapters": 24, "bare": 5, "runs": False, "K": 4096,
         "N": 11008, "rank": 32, "dtype": "bf16"},
        # prompts of five requests in one pass
        {"name": "adapt-2048", "kind": "adapt", "tokens": 2048, "adapters": 5, "bare": 100, "runs": True, "K": 11008,
         "N": 4096, "rank": 64, "dtype": "fp16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


# the most of a drawn case: keys times key heads times width of an attention
# call, and tokens of a step
_MAX_KV = 128 * 6000 * 8 * 128
_MAX_STEP = 12000


def draw(rng):
    kind = rng.choices(["step", "append", "attend", "adapt"], [2, 3, 6, 5])[0]
    dtype = rng.choice(["fp16", "bf16"])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    if kind == "step":
        requests = _log_int(rng, 1, 1024)
        prompts = rng.choice([0, 0, rng.randrange(requests + 1)])
        return {"kind": kind, "requests": requests, "prompts": prompts, "longest": _log_int(rng, 16, 16384),
                "prompt": _log_int(rng, 1, max(1, min(2048, _MAX_STEP // max(1, prompts)))) if prompts else 0,
                "page": rng.choice([page, rng.randrange(1, 100)])}
    dim = rng.choice([128, 128, 128, 64, 64, 80, 96, 112, 256])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 8, 16, 32])
    heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 7, 8, 16) if g * kv_heads <= 64])
    if kind == "append":
        return {"kind": kind, "tokens": _log_int(rng, 1, max(1, min(4096, 2048 * 48 * 128 // ((heads + 2 * kv_heads) * dim)))),
                "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rng.choice([dim, dim, dim // 2]),
                "interleaved": rng.random() < 0.3, "page": page, "dtype": dtype}
    if kind == "attend":
        longest = _log_int(rng, 1, 32768)
        requests = _log_int(rng, 1, max(1, min(256, _MAX_KV // (longest * kv_heads * dim))))
        return {"kind": kind, "requests": requests, "shortest": rng.choice([1, max(1, longest // 8), longest]),
                "longest": longest, "context": -(-longest // page) * page * rng.choice([1, 1, 2]), "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "window": rng.choice([0, 0, 0, _log_int(rng, 1, longest)]),
                "page": page, "dtype": dtype}
    K, N = rng.choice([(4096, 4096), (4096, 11008), (11008, 4096), (4096, 14336), (2048, 2048), (5120, 5120),
                       (8192, 1024), (4000, 11008), (1000, 999)])
    rank = rng.choice([4, 8, 16, 16, 32, 64, 128, 20])
    adapters = _log_int(rng, 1, 64)
    most = 2048 * 64 * (11008 + 4096) // (rank * (K + N))
    return {"kind": kind, "tokens": _log_int(rng, 1, min(4096, most)), "adapters": adapters,
            "bare": rng.choice([0, 0, 3]), "runs": rng.random() < 0.5, "K": K, "N": N, "rank": rank, "dtype": dtype}


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, shape, sigma, dtype):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0, sigma, generator=g)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _step_counts(case):
    """(cached, new) tokens of each request: prompts start from nothing."""
    rng = random.Random(case["requests"] * 7919 + case["longest"])
    cached, new = [], []
    first = set(rng.sample(range(case["requests"]), case["prompts"]))
    for r in range(case["requests"]):
        cached.append(0 if r in first else _log_int(rng, 1, case["longest"]))
        new.append(_log_int(rng, 1, case["prompt"]) if r in first else 1)
    return cached, new


def _lengths(case):
    """Keys of each request, spread over the logarithm of the range."""
    rng = random.Random(case["requests"] * 7919 + case["longest"])
    lens = [_log_int(rng, case["shortest"], case["longest"]) for _ in range(case["requests"])]
    lens[-1] = case["longest"]
    return lens


def _tables(g, counts, page, width, spare):
    """Block tables whose first counts[r] entries are pages in random order,
    and the pages left over."""
    used = sum(counts)
    order = torch.randperm(used + spare, generator=g, device="cuda").to(torch.int32)
    have = torch.arange(width, device="cuda")[None, :] < torch.tensor(counts).cuda()[:, None]
    table = torch.zeros(len(counts), width, dtype=torch.int32, device="cuda")
    table[have] = order[:used]
    return table, order[used:].contiguous()


def prepare(case, seed):
    g = _gen(seed)
    state = dict(case)
    kind, dtype = case["kind"], _DTYPES.get(case.get("dtype"))
    if kind == "step":
        P = case["page"]
        cached, new = _step_counts(case)
        width = -(-(max(c + n for c, n in zip(cached, new)) + P) // P)
        need = sum(-(-(c + n) // P) - -(-c // P) for c, n in zip(cached, new))
        table, free = _tables(g, [-(-c // P) for c in cached], P, width, need + 64)
        state.update(lengths=_ints(cached), new=_ints(new), table=table, free=free,
                     pool=_ints([random.Random(seed).randrange(32), 0]), tokens=sum(new))
    elif kind == "append":
        T, D, P = case["tokens"], case["dim"], case["page"]
        pages = -(-T // P) + 16
        # the projections' outputs side by side, as one buffer
        qkv = _randn(g, (T, case["heads"] + 2 * case["kv_heads"], D), 1.0, dtype)
        first = random.Random(seed).randrange(2048)
        freq = 10000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"])
        angle = torch.arange(first + T, device="cuda", dtype=torch.float64)[:, None] * freq
        # consecutive tokens of one prompt: its pages in random order
        page_of = torch.randperm(pages, generator=g, device="cuda")
        t = torch.arange(T, device="cuda")
        state.update(q=qkv[:, :case["heads"]], k=qkv[:, case["heads"]:case["heads"] + case["kv_heads"]],
                     v=qkv[:, case["heads"] + case["kv_heads"]:],
                     k_cache=_randn(g, (pages, P, case["kv_heads"], D), 1.0, dtype),
                     v_cache=_randn(g, (pages, P, case["kv_heads"], D), 1.0, dtype),
                     slots=page_of[t // P] * P + t % P, positions=(first + t).to(torch.int32),
                     cos_sin=torch.cat([angle.cos(), angle.sin()], 1).float().contiguous())
    elif kind == "attend":
        P, D = case["page"], case["dim"]
        lens = _lengths(case)
        table, _ = _tables(g, [-(-n // P) for n in lens], P, case["context"] // P, 16)
        pages = sum(-(-n // P) for n in lens) + 16
        state.update(q=_randn(g, (len(lens), case["heads"], D), 2.0, dtype),
                     k_cache=_randn(g, (pages, P, case["kv_heads"], D), 1.0, dtype),
                     v_cache=_randn(g, (pages, P, case["kv_heads"], D), 1.0, dtype),
                     table=table, positions=_ints([n - 1 for n in lens]), scale=D ** -0.5)
    else:
        M, K, N, r = case["tokens"], case["K"], case["N"], case["rank"]
        ids = _adapters(case)
        names = torch.randperm(case["adapters"], generator=g, device="cuda").to(torch.int32)
        ids = _ints(ids)
        state.update(x=_randn(g, (M, K), 1.0, dtype), y=_randn(g, (M, N), 1.0, dtype),
                     a=_randn(g, (case["adapters"], r, K), K ** -0.5, dtype),
                     b=_randn(g, (case["adapters"], N, r), 0.5 * r ** -0.5, dtype),
                     adapters=torch.where(ids >= 0, names[ids.clamp(min=0).long()], ids),
                     scales=torch.rand(case["adapters"], generator=g, device="cuda") * 1.5 + 0.5)
    return state


def _adapters(case):
    """Each token's adapter before their names are shuffled, -1 for none: in
    runs as prompts come, else in turn as a decode batch's requests do."""
    M, n = case["tokens"], case["adapters"]
    ids = [m * min(n, M) // M if case["runs"] else m % n for m in range(M)]
    for i in range(min(case["bare"], M - 1)):
        ids[(i + 1) * M // (case["bare"] + 1)] = -1
    return ids


# ----------------------------------------------------------------- one pass

def run(state):
    if own:
        return _run_own(state)
    return {"step": _plain_step, "append": _plain_append, "attend": _plain_attend, "adapt": _plain_adapt}[state["kind"]](state)


def _run_own(s):
    from libortho_amd import _C_ops
    if s["kind"] == "step":
        lengths, pool, query_start, rows, positions, slots = _C_ops.page_step(
            s["lengths"], s["new"], s["table"], s["free"], s["pool"], s["page"], s["tokens"])
        return {"lengths": lengths, "pool": pool, "query_start": query_start, "rows": rows, "positions": positions,
                "slots": slots, "table": s["table"]}
    if s["kind"] == "append":
        q = _C_ops.cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], q=s["q"],
                                positions=s["positions"], cos_sin=s["cos_sin"], interleaved=s["interleaved"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if s["kind"] == "attend":
        return _C_ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["positions"],
                                      scale=s["scale"], window=s["window"])
    return _C_ops.adapter_add(s["y"], s["x"], s["a"], s["b"], s["adapters"], s["scales"])


def _plain_step(s):
    P, T = s["page"], s["tokens"]
    L, n, table, free = s["lengths"].long(), s["new"].long(), s["table"], s["free"].long()
    zero = torch.zeros(1, dtype=torch.int64, device=L.device)
    query_start = torch.cat([zero, n.cumsum(0)])
    old = (L + P - 1) // P
    need = (L + n + P - 1) // P - old
    first = s["pool"][0] + need.cumsum(0) - need
    t = torch.arange(T, device=L.device)
    rows = torch.searchsorted(query_start, t, right=True) - 1
    positions = L[rows] + t - query_start[rows]
    at = positions // P
    new = at - old[rows]  # which of the request's new pages, negative: one it had
    page = torch.where(new >= 0, free[(first[rows] + new).clamp(max=free.numel() - 1)], table[rows, at].long())
    table[rows, at] = page.int()
    pool = torch.stack([s["pool"][0] + need.sum(), zero[0]]).int()
    return {"lengths": (L + n).int(), "pool": pool, "query_start": query_start.int(), "rows": rows.int(),
            "positions": positions.int(), "slots": page * P + positions % P, "table": table}


def _rotate(x, cos, sin, rot, interleaved):
    x = x.float()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_append(s):
    rot, dtype = s["rot"], s["q"].dtype
    cs = s["cos_sin"][s["positions"].long()][:, None, :]
    cos, sin = cs[..., :rot // 2], cs[..., rot // 2:]
    q = _rotate(s["q"], cos, sin, rot, s["interleaved"]).to(dtype)
    k = _rotate(s["k"], cos, sin, rot, s["interleaved"]).to(dtype)
    s["k_cache"].flatten(0, 1).index_copy_(0, s["slots"], k)
    s["v_cache"].flatten(0, 1).index_copy_(0, s["slots"], s["v"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attend(s):
    q, table, positions = s["q"].float(), s["table"].long(), s["positions"].long()
    T, H, D = q.shape
    P, heads = s["page"], s["kv_heads"]
    width = -(-s["longest"] // P)  # pages of the longest request
    k = s["k_cache"][table[:, :width]].reshape(T, width * P, heads, D).float()
    scores = torch.matmul(k.permute(0, 2, 1, 3).contiguous(), q.reshape(T, heads, H // heads, D).transpose(2, 3).contiguous()) * s["scale"]
    del k
    j = torch.arange(width * P, device=q.device)
    seen = (j <= positions[:, None]) & ((j > positions[:, None] - s["window"]) if s["window"] else True)
    scores = scores.masked_fill(~seen[:, None, :, None], float("-inf"))
    p = (scores - scores.amax(2, keepdim=True)).exp()
    p = (p / p.sum(2, keepdim=True)).transpose(2, 3).contiguous()
    v = s["v_cache"][table[:, :width]].reshape(T, width * P, heads, D).float()
    return torch.matmul(p, v.permute(0, 2, 1, 3).contiguous()).reshape(T, H, D).to(s["q"].dtype)


def _plain_adapt(s):
    x, a, b, ids = s["x"].float(), s["a"].float(), s["b"].float(), s["adapters"].long()
    n, r, K = a.shape
    t = (x @ a.reshape(n * r, K).T).reshape(-1, n, r)  # every token through every adapter, its own one kept
    mine = torch.where(ids[:, None] == torch.arange(n, device=ids.device), s["scales"], torch.zeros_like(s["scales"]))
    t = (t * mine[:, :, None]).reshape(-1, n * r)
    return (s["y"].float() + t @ b.permute(0, 2, 1).reshape(n * r, -1)).to(s["y"].dtype)


# --------------------------------------------------------- work and 64 bits

def work(case):
    kind = case["kind"]
    if kind == "step":
        R, P = case["requests"], case["page"]
        cached, new = _step_counts(case)
        T = sum(new)
        pages = sum(-(-(c + n) // P) - -(-c // P) for c, n in zip(cached, new))
        # lengths and counts in, lengths, starts out, the last page of each
        # request; pages moved to the tables; rows, positions and slots out
        return {"bytes": 4 * 2 * R + 4 * (2 * R + 1) + 4 * R + 8 * pages + 16 * T + 16, "flops": 0}
    if kind == "append":
        T, D, H, G, rot = case["tokens"], case["dim"], case["heads"], case["kv_heads"], case["rot"]
        return {"bytes": T * (2 * D * (2 * H + 4 * G) + 4 * rot + 12), "flops": 3 * T * (H + G) * rot}
    if kind == "attend":
        H, G, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
        seen = [min(n, case["window"] or n) for n in _lengths(case)]
        return {"bytes": 4 * G * D * sum(seen) + len(seen) * (4 * H * D + 4) + 4 * sum(-(-n // P) for n in seen),
                "flops": 4 * H * D * sum(seen)}
    M, K, N, r = case["tokens"], case["K"], case["N"], case["rank"]
    ids = [i for i in _adapters(case) if i >= 0]
    return {"bytes": 2 * len(ids) * K + 4 * M * N + 4 * M + len(set(ids)) * (2 * r * (K + N) + 4),
            "flops": 2 * len(ids) * r * (K + N)}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "step":
        return None  # whole numbers only
    if kind == "append":
        rot = case["rot"]
        angle = s["cos_sin"].double()[s["positions"].long()].cpu()
        turn = torch.complex(angle[:, :rot // 2], angle[:, rot // 2:])[:, None, :]

        def rotated(x):
            x = x.double().cpu().clone()
            pair = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
            z = torch.complex(x[..., pair[0]], x[..., pair[1]]) * turn
            x[..., pair[0]], x[..., pair[1]] = z.real, z.imag
            return x

        caches = []
        for cache, rows in ((s["k_cache"], rotated(s["k"])), (s["v_cache"], s["v"].double().cpu())):
            full = cache.double().cpu()
            for i, slot in enumerate(s["slots"].tolist()):
                full[slot // case["page"], slot % case["page"]] = rows[i]
            caches.append(full)
        return {"q": rotated(s["q"]), "k_cache": caches[0], "v_cache": caches[1]}
    if kind == "attend":
        group = case["heads"] // case["kv_heads"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for t, last in enumerate(s["positions"].tolist()):
            first = max(0, last + 1 - case["window"]) if case["window"] else 0
            j = torch.arange(first, last + 1, device="cuda")
            page = s["table"][t].long()[j // case["page"]]
            k, v = (c[page, j % case["page"]].double() for c in (s["k_cache"], s["v_cache"]))
            for h in range(case["kv_heads"]):
                mine = slice(h * group, (h + 1) * group)
                w = torch.softmax(s["q"][t, mine].double() @ k[:, h].T.contiguous() * s["scale"], -1)
                out[t, mine] = w @ v[:, h].contiguous()
        return out
    out = s["y"].double()
    for i in range(case["adapters"]):
        m = (s["adapters"] == i).nonzero().flatten()
        if m.numel():
            low = s["x"][m].double() @ s["a"][i].double().T
            out[m] += s["scales"][i].double() * (low @ s["b"][i].double().T)
    return out
