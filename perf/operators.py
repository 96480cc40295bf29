"""Cases of the bounded-cache operators: attention with a sliding window and sinks (one new token per sequence,
and a prompt chunk), decode attention that accumulates each cached token's attention weight, and eviction from the
paged cache by that weight. `own` False: plain form in elementary torch operations; True: the framework's launchers.
"""
import math
import random

import numpy as np
import torch

own = False

D = 128            # head dimension of the cache
PAGE = 16          # tokens per page
SCALE = 1.0 / math.sqrt(D)
WHOLE = 1 << 30    # a window that no sequence outgrows


def listed():
    return [
        # One interactive request with a short window: the latency of a single launch.
        dict(name="window_decode_one", op="window_decode", seqs=1, lo=700, hi=700, idle=0, q_heads=12, kv_heads=2,
             window=512, sinks=4, pick=1),
        # A half-filled bucket of odd lengths, some shorter than the window, eight query heads to a KV head.
        dict(name="window_decode_ragged", op="window_decode", seqs=7, lo=3, hi=2500, idle=1, q_heads=32, kv_heads=4,
             window=1000, sinks=5, pick=2),
        # The largest decode bucket over long contexts of mixed lengths: what a window saves on a serving GPU.
        dict(name="window_decode_bucket", op="window_decode", seqs=64, lo=1024, hi=32768, idle=0, q_heads=12, kv_heads=2,
             window=4096, sinks=16, pick=3),
        # A short odd chunk in the middle of a prompt, no sinks.
        dict(name="window_prefill_short", op="window_prefill", start=1000, rows=257, q_heads=12, kv_heads=2, window=250,
             sinks=0),
        # A chunk deep inside a prompt: most of the context lies outside the window.
        dict(name="window_prefill_deep", op="window_prefill", start=6144, rows=2048, q_heads=12, kv_heads=2,
             window=1024, sinks=4),
        # A whole long prompt in one call with a wide window and a page-crossing number of sinks.
        dict(name="window_prefill_long", op="window_prefill", start=0, rows=8192, q_heads=12, kv_heads=2, window=4096,
             sinks=100),
        # One request, odd length: accumulation at the latency end.
        dict(name="weights_decode_one", op="weights_decode", seqs=1, lo=1031, hi=1031, idle=0, q_heads=12, kv_heads=2,
             pick=4),
        # The serving bucket the framework's attention benchmark uses.
        dict(name="weights_decode_bucket", op="weights_decode", seqs=64, lo=1024, hi=1280, idle=0, q_heads=12, kv_heads=2,
             pick=5),
        # A few long contexts whose keys are spread over the whole machine.
        dict(name="weights_decode_long", op="weights_decode", seqs=6, lo=8000, hi=32768, idle=0, q_heads=14, kv_heads=2,
             pick=6),
        # One request that has grown a little past its budget.
        dict(name="evict_one", op="evict", seqs=1, lo=1100, hi=1100, kv_heads=2, budget=1024, sinks=4, recent=128,
             pick=7),
        # A bucket of requests after their prompts; a few are still inside the budget and move whole.
        dict(name="evict_bucket", op="evict", seqs=64, lo=1500, hi=4500, kv_heads=2, budget=2048, sinks=4, recent=256,
             pick=8),
        # Long prompts cut down to an odd budget.
        dict(name="evict_long", op="evict", seqs=5, lo=16000, hi=32768, kv_heads=4, budget=4099, sinks=0, recent=1000,
             pick=9),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _odd(rng, lo, hi):
    v = _log(rng, lo, hi)
    return v if rng.random() < 0.4 else min(hi, v | 1)


def draw(rng):
    op = rng.choice(["window_decode", "window_prefill", "weights_decode", "evict"])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.randint(1, 8)
    pick = rng.randrange(1 << 30)
    if op == "window_prefill":
        start = rng.choice([0, _odd(rng, 1, 12000)])
        rows = _odd(rng, 1, 4096)
        case = dict(op=op, start=start, rows=rows, q_heads=heads, kv_heads=kv, window=_odd(rng, 1, 6000),
                    sinks=rng.choice([0, 4, _odd(rng, 1, 300)]))
        while case["rows"] > 1 and (work(case)["flops"] > 1.0e11 or case["rows"] * (start + case["rows"]) * heads > 8.0e8):
            case["rows"] = case["rows"] // 2 + 1 if case["rows"] > 2 else 1
        return case
    seqs = _log(rng, 1, 64)
    hi = _odd(rng, 2, 32768)
    lo = _odd(rng, 1, hi)
    if op == "evict":
        budget = _odd(rng, 1, max(2, hi))
        sinks = rng.choice([0, min(4, budget)])
        recent = rng.randint(0, max(0, (budget - sinks) // 2))
        case = dict(op=op, seqs=seqs, lo=lo, hi=hi, kv_heads=kv, budget=budget, sinks=sinks, recent=recent, pick=pick)
        largest = 3.0e8
    else:
        case = dict(op=op, seqs=seqs, lo=lo, hi=hi, idle=rng.choice([0, 0, rng.randint(0, seqs - 1)]), q_heads=heads,
                    kv_heads=kv, pick=pick)
        if op == "window_decode":
            case.update(window=_odd(rng, 1, 8192), sinks=rng.choice([0, 4, _odd(rng, 1, 300)]))
        largest = 2.5e8 if op == "window_decode" else 1.2e8
    while case["seqs"] > 1 and (work(case)["bytes"] > largest or sum(_lens(case)) * kv > 2500000):
        case["seqs"] = case["seqs"] // 2
        if "idle" in case:
            case["idle"] = min(case["idle"], case["seqs"] - 1)
    return case


def _lens(case):
    """Cached tokens of each sequence: spread over [lo, hi] by the case alone; `idle` rows of a padded bucket are 0."""
    r = random.Random(case["pick"])
    lens = [r.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    for i in r.sample(range(len(lens)), case.get("idle", 0)):
        lens[i] = 0
    return lens


def _visible(n, window, sinks):
    return n if n <= window else window + min(sinks, n - window)


def work(case):
    kv = case["kv_heads"]
    if case["op"] == "window_prefill":
        w, s, start, rows = case["window"], case["sinks"], case["start"], case["rows"]
        pos = np.arange(start, start + rows, dtype=np.int64) + 1
        pairs = int(np.where(pos <= w, pos, w + np.minimum(s, pos - w)).sum())
        keys = _visible(start + rows, w + rows - 1, s)
        return {"bytes": 2 * 2 * rows * case["q_heads"] * D + 2 * 2 * keys * kv * D, "flops": 4 * D * case["q_heads"] * pairs}
    lens = [n for n in _lens(case) if n > 0]
    row = 2 * 2 * kv * D                                     # K and V of one token, FP16, all heads
    if case["op"] == "evict":
        kept = [min(n, case["budget"]) for n in lens]
        moved = sum(kept) * (2 * row + 2 * 4 * kv + 4 * kv)  # rows and weights both ways, the list of kept positions
        ranked = sum((n - case["sinks"] - case["recent"]) * 4 * kv for n in lens if n > case["budget"])
        return {"bytes": moved + ranked, "flops": 0}
    seen = sum(_visible(n, case.get("window", WHOLE), case.get("sinks", 0)) for n in lens)
    more = 2 * 4 * kv * seen if case["op"] == "weights_decode" else 0
    return {"bytes": seen * row + more + 2 * 2 * len(lens) * case["q_heads"] * D + 4 * len(lens) + seen // PAGE * 4,
            "flops": 4 * D * case["q_heads"] * seen}


def _pages(n):
    return (n + PAGE - 1) // PAGE


def prepare(case, seed):
    """A serving program's state: the pool of one layer, block tables over a shuffled page order, lengths, queries."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 11)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float16)

    kv, op = case["kv_heads"], case["op"]
    lens = [case["start"] + case["rows"]] if op == "window_prefill" else _lens(case)
    need = [_pages(n) for n in lens]
    kept = [_pages(case["budget"]) if op == "evict" else 0 for _ in lens]
    mbps = max(1, max(need))
    blocks = 1 + sum(need) + sum(kept)                       # block 0 is the padding target
    order = (torch.randperm(blocks - 1, generator=g, device="cuda") + 1).to(torch.int32).cpu()
    tables = torch.zeros(len(lens), mbps, dtype=torch.int32)
    fresh = torch.zeros(len(lens), max(1, max(kept)), dtype=torch.int32)
    at = 0
    for i, (a, b) in enumerate(zip(need, kept)):
        tables[i, :a] = order[at:at + a]
        fresh[i, :b] = order[at + a:at + a + b]
        at += a + b
    state = dict(case=dict(case), tables=tables.cuda(), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                 mbps=mbps, workspace=None, pool=normal(blocks, 2, kv, PAGE, D))
    if op in ("weights_decode", "evict"):
        # attention weight gathers on few tokens; some have gathered none at all
        u = torch.rand(blocks, kv, PAGE, generator=g, device="cuda")
        state["weights"] = torch.where(u < 0.05, torch.zeros_like(u), u.pow(-0.7) - 0.99)
    if op == "evict":
        state.update(fresh=fresh.cuda(), new_lens=torch.zeros(len(lens), dtype=torch.int32, device="cuda"),
                     kept=torch.zeros(len(lens), kv, case["budget"], dtype=torch.int32, device="cuda"))
    else:
        rows = case["rows"] if op == "window_prefill" else len(lens)
        state["q"] = normal(rows, case["q_heads"] * D)
        state["out"] = torch.zeros(rows, case["q_heads"] * D, dtype=torch.float16, device="cuda")
    return state


# ---------------------------------------------------------------- plain form

def _token_rows(pool, tables, positions):
    """K and V rows [seqs, positions, kv_heads, D] in 32 bits, positions [seqs, n] looked up through the tables."""
    block = torch.gather(tables.long(), 1, positions // PAGE)
    rows = pool.permute(0, 3, 1, 2, 4)[block, positions % PAGE]          # [seqs, n, 2, kv_heads, D]
    return rows[:, :, 0].float(), rows[:, :, 1].float(), block


def _attend(q, k, v, seen, kv):
    """q [s, heads*D], k / v [s, n, kv, D], seen [s, n] -> out [s, heads*D], probabilities [s, kv, group, n]."""
    s = q.shape[0]
    qh = q.float().view(s, kv, -1, D)
    scores = torch.matmul(qh, k.permute(0, 2, 3, 1)) * SCALE
    scores = torch.where(seen[:, None, None, :], scores, torch.full_like(scores, -torch.inf))
    top = scores.amax(dim=-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = e.sum(dim=-1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    return torch.matmul(p, v.permute(0, 2, 1, 3)).reshape(s, -1), p


def _plain_window_decode(s):
    c, lens = s["case"], s["lens"].long()
    longest = s["mbps"] * PAGE
    window, sinks = min(c["window"], longest), min(c["sinks"], longest)
    first = torch.arange(sinks, device="cuda")[None, :].expand(len(lens), -1)
    last = lens[:, None] - window + torch.arange(window, device="cuda")[None, :]
    pos = torch.cat([first, last], dim=1)
    seen = torch.cat([(first < lens[:, None]) & (first < lens[:, None] - window), last >= 0], dim=1)
    seen = seen & (lens > 0)[:, None]
    k, v, _ = _token_rows(s["pool"], s["tables"], pos.clamp(0, longest - 1))
    out, _ = _attend(s["q"], k, v, seen, c["kv_heads"])
    s["out"].copy_(torch.where((lens > 0)[:, None], out, s["out"].float()))
    return {"out": s["out"]}


def _plain_window_prefill(s):
    c = s["case"]
    kv, n = c["kv_heads"], c["start"] + c["rows"]
    pos = torch.arange(n, device="cuda")
    k, v, _ = _token_rows(s["pool"], s["tables"], pos[None, :])
    row = torch.arange(c["start"], n, device="cuda")[:, None]
    seen = (pos <= row) & ((pos > row - c["window"]) | (pos < c["sinks"]))
    qh = s["q"].float().view(c["rows"], kv, -1, D).permute(1, 2, 0, 3)                     # [kv, group, rows, D]
    scores = torch.matmul(qh, k[0].permute(1, 2, 0)[:, None]) * SCALE
    scores = torch.where(seen, scores, torch.full_like(scores, -torch.inf))
    e = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    p = e / e.sum(dim=-1, keepdim=True)
    out = torch.matmul(p, v[0].permute(1, 0, 2)[:, None])                                  # [kv, group, rows, D]
    s["out"].copy_(out.permute(2, 0, 1, 3).reshape(c["rows"], -1))
    return {"out": s["out"]}


def _plain_weights_decode(s):
    c, lens = s["case"], s["lens"].long()
    pos = torch.arange(s["mbps"] * PAGE, device="cuda")[None, :].expand(len(lens), -1)
    seen = pos < lens[:, None]
    k, v, block = _token_rows(s["pool"], s["tables"], pos)
    out, p = _attend(s["q"], k, v, seen, c["kv_heads"])
    s["out"].copy_(torch.where((lens > 0)[:, None], out, s["out"].float()))
    got = p.sum(dim=2).permute(0, 2, 1)                                                    # [seqs, n, kv]
    old = s["weights"][block, :, pos % PAGE]
    new = torch.where((pos == lens[:, None] - 1)[..., None], got, old + got)
    s["weights"][block[seen], :, (pos % PAGE)[seen]] = new[seen]
    return {"out": s["out"], "weights": s["weights"]}


def _plain_evict(s):
    c, lens = s["case"], s["lens"].long()
    kv, budget = c["kv_heads"], c["budget"]
    n = max(s["mbps"] * PAGE, budget)
    pos = torch.arange(n, device="cuda")[None, :].expand(len(lens), -1)
    block = torch.gather(s["tables"].long(), 1, (pos // PAGE).clamp(max=s["mbps"] - 1))
    live = pos < lens[:, None]
    safe = (pos < c["sinks"]) | (pos >= lens[:, None] - c["recent"])
    w = s["weights"][block, :, pos % PAGE].permute(0, 2, 1)                                # [seqs, kv, n]
    key = torch.where(safe[:, None], torch.full_like(w, torch.inf), w)
    key = torch.where(live[:, None], key, torch.full_like(w, -torch.inf))
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :, :budget]
    new_lens = lens.clamp(max=budget)
    rank = torch.arange(budget, device="cuda")
    here = (rank < new_lens[:, None])[:, None].expand(-1, kv, -1)
    kept = torch.sort(torch.where(here, best, torch.full_like(best, n)), dim=-1).values    # cache order
    src = torch.gather(block[:, None].expand(-1, kv, -1), 2, kept.clamp(max=n - 1))
    dst = s["fresh"].long()[:, rank // PAGE][:, None].expand(-1, kv, -1)
    head = torch.arange(kv, device="cuda")[None, :, None].expand_as(dst)
    slot = (rank % PAGE).expand_as(dst)
    rows = s["pool"][src[here], :, head[here], (kept % PAGE)[here]]
    s["pool"][dst[here], :, head[here], slot[here]] = rows
    s["weights"][dst[here], head[here], slot[here]] = s["weights"][src[here], head[here], (kept % PAGE)[here]]
    s["kept"].copy_(torch.where(here, kept, torch.full_like(kept, -1)))
    s["new_lens"].copy_(new_lens)
    return {"pool": s["pool"], "weights": s["weights"], "kept": s["kept"], "new_lens": s["new_lens"]}


_PLAIN = {"window_decode": _plain_window_decode, "window_prefill": _plain_window_prefill,
          "weights_decode": _plain_weights_decode, "evict": _plain_evict}


# ---------------------------------------------------------------- the framework's launchers

def _own(s):
    from redline_llm_b200 import kernels as K
    c = s["case"]
    op, kv, heads = c["op"], c["kv_heads"], c.get("q_heads", 0)
    width = heads * D
    if op == "evict":
        K.launch_kv_evict(s["pool"], s["weights"], s["tables"], s["mbps"], s["fresh"], s["fresh"].shape[1], s["lens"],
                          s["new_lens"], s["kept"], c["seqs"], kv, D, c["budget"], c["sinks"], c["recent"])
        return {"pool": s["pool"], "weights": s["weights"], "kept": s["kept"], "new_lens": s["new_lens"]}
    if op == "window_prefill":
        if s["workspace"] is None:
            s["workspace"] = K.window_prefill_workspace(c["start"], c["rows"], heads, c["window"], c["sinks"])
        K.launch_paged_window_prefill_attention(s["out"], width, s["q"], width, s["pool"], s["tables"], s["mbps"],
                                                c["start"], c["rows"], heads, kv, D, SCALE, c["window"], c["sinks"],
                                                s["workspace"])
        return {"out": s["out"]}
    if s["workspace"] is None:
        s["workspace"] = K.window_attention_workspace(c["seqs"], s["mbps"], heads, kv, weights=op == "weights_decode")
    if op == "window_decode":
        K.launch_paged_window_attention_decode(s["out"], width, s["q"], width, s["pool"], s["tables"], s["lens"],
                                               c["seqs"], s["mbps"], heads, kv, D, SCALE, c["window"], c["sinks"],
                                               s["workspace"])
        return {"out": s["out"]}
    K.launch_paged_attention_decode_weights(s["out"], width, s["q"], width, s["pool"], s["tables"], s["lens"], c["seqs"],
                                            s["mbps"], heads, kv, D, SCALE, s["weights"], s["workspace"])
    return {"out": s["out"], "weights": s["weights"]}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------- 64 bits, straight from the definitions

def exact(case, seed):
    s = prepare(case, seed)
    lens, kv, op = s["lens"].tolist(), case["kv_heads"], case["op"]
    tables = s["tables"].long()

    def cached(i, n):
        """K and V of sequence i in 64 bits, [kv, n, D] each, and where token t lies: flat slot (page * 16 + slot)."""
        pages = tables[i, :_pages(n)]
        flat = (pages[:, None] * PAGE + torch.arange(PAGE, device="cuda")).reshape(-1)[:n]
        data = s["pool"][pages].double().permute(1, 2, 0, 3, 4).reshape(2, kv, -1, D)[:, :, :n]
        return data[0], data[1], flat

    if op == "window_prefill":
        n, rows, group = lens[0], case["rows"], case["q_heads"] // kv
        k, v, _ = cached(0, n)
        q = s["q"].double().view(rows, case["q_heads"], D)
        out = torch.empty(rows, case["q_heads"], D, dtype=torch.float64, device="cuda")
        t = torch.arange(n, device="cuda")
        for r0 in range(0, rows, 1024):
            p = case["start"] + torch.arange(r0, min(rows, r0 + 1024), device="cuda")[:, None]
            hidden = (t > p) | ((t <= p - case["window"]) & (t >= case["sinks"]))
            for h in range(case["q_heads"]):
                a = (q[r0:r0 + 1024, h] @ k[h // group].T) / math.sqrt(D)
                out[r0:r0 + 1024, h] = torch.softmax(a.masked_fill(hidden, -math.inf), dim=1) @ v[h // group]
        return {"out": out.reshape(rows, -1)}
    if op == "evict":
        pool, weights = s["pool"].double(), s["weights"].double()
        kept = torch.full((len(lens), kv, case["budget"]), -1, dtype=torch.int64, device="cuda")
        for i, n in enumerate(lens):
            m = min(n, case["budget"])
            for h in range(kv):
                flat = cached(i, n)[2]
                w = s["weights"][:, h].reshape(-1)[flat].cpu().numpy().astype(np.float64)
                held = np.ones(n, dtype=bool)
                if n > m:
                    rest = np.arange(case["sinks"], n - case["recent"])
                    ranked = rest[np.argsort(-w[rest], kind="stable")]
                    held[ranked[m - case["sinks"] - case["recent"]:]] = False
                keep = torch.from_numpy(np.flatnonzero(held)).cuda()
                kept[i, h, :m] = keep
                to = s["fresh"].long()[i, torch.arange(m, device="cuda") // PAGE]
                slot = torch.arange(m, device="cuda") % PAGE
                come, from_slot = flat[keep] // PAGE, flat[keep] % PAGE
                pool[to, :, h, slot] = s["pool"][come, :, h, from_slot].double()
                weights[to, h, slot] = s["weights"][come, h, from_slot].double()
        return {"pool": pool, "weights": weights, "kept": None, "new_lens": None}
    window, sinks = case.get("window", WHOLE), case.get("sinks", 0)
    out = torch.zeros(len(lens), case["q_heads"], D, dtype=torch.float64, device="cuda")
    weights = s["weights"].double() if op == "weights_decode" else None
    for i, n in enumerate(lens):
        if n == 0:
            continue
        k, v, flat = cached(i, n)
        q = s["q"][i].double().view(kv, -1, D)
        t = torch.arange(n, device="cuda")
        a = torch.einsum("hgd,hnd->hgn", q, k) / math.sqrt(D)
        a = a.masked_fill((t >= sinks) & (t < n - window), -math.inf)
        p = torch.softmax(a, dim=2)
        out[i] = torch.einsum("hgn,hnd->hgd", p, v).reshape(-1, D)
        if weights is not None:
            old = weights[flat // PAGE, :, flat % PAGE]                                    # [n, kv]
            old[n - 1] = 0.0
            weights[flat // PAGE, :, flat % PAGE] = old + p.sum(dim=1).T
    got = {"out": out.reshape(len(lens), -1)}
    if weights is not None:
        got["weights"] = weights
    return got
