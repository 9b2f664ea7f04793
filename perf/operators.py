"""Operators of a step that serves many continuations of one prompt: block tables and slot maps
made on the GPU, decode attention over a prefix that rows share, and the pick under top-k, top-p
and min-p. Every operator here in its plain form (elementary torch operations) and, where `own` is
true, as a user calls it.

`listed()` and `draw()` name cases, `prepare()` makes what a program holds before the call, `run()`
is one pass, `work()` what a pass cannot do without, `exact()` the result in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"


# ---------------------------------------------------------------------------------- cases
def listed():
    return [
        # one chat drawing its next token over the vocabulary of the 1.2B shape
        {"name": "pick_1_top_p", "op": "pick", "rows": 1, "vocab": 65536, "mode": "top_p"},
        # a small odd vocabulary (test models), every filter in use
        {"name": "pick_5_odd", "op": "pick", "rows": 5, "vocab": 1003, "mode": "mixed"},
        # a batch whose requests ask for the 50 or so likeliest, then a nucleus of those
        {"name": "pick_64_top_k", "op": "pick", "rows": 64, "vocab": 65536, "mode": "top_k"},
        # a full server, every request with filters of its own, over a large vocabulary of odd size
        {"name": "pick_256_mixed", "op": "pick", "rows": 256, "vocab": 130001, "mode": "mixed"},
        # four samples of one short question
        {"name": "attend_4_short", "op": "attend", "groups": 1, "rows": 4, "heads": 32, "kv_heads": 8, "dim": 64,
         "page": 64, "shared": 448, "own": 40},
        # eight chats behind one system prompt, heads of 128, small pages
        {"name": "attend_8_dim128", "op": "attend", "groups": 1, "rows": 8, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "shared": 4096, "own": 300},
        # four prompts with 16 continuations each, heads of 128
        {"name": "attend_4x16_dim128", "op": "attend", "groups": 4, "rows": 16, "heads": 24, "kv_heads": 8, "dim": 128,
         "page": 64, "shared": 8192, "own": 512},
        # 64 samples behind one document, the 1.2B shape
        {"name": "attend_64_document", "op": "attend", "groups": 1, "rows": 64, "heads": 32, "kv_heads": 8, "dim": 64,
         "page": 64, "shared": 32768, "own": 1024},
        # a full server behind one system prompt, contexts of their own behind it
        {"name": "attend_256_prompt", "op": "attend", "groups": 1, "rows": 256, "heads": 32, "kv_heads": 8, "dim": 64,
         "page": 64, "shared": 4096, "own": 2048},
        # the tables of a decode step of eight rows
        {"name": "tables_8", "op": "tables", "rows": 8, "page": 64, "context": 4096, "new": 1, "shared": 2048},
        # prompt portions beside decoded tokens, long contexts in small pages
        {"name": "tables_64_portions", "op": "tables", "rows": 64, "page": 16, "context": 32768, "new": 512,
         "shared": 8192},
        # a full server's tables
        {"name": "tables_256", "op": "tables", "rows": 256, "page": 16, "context": 65536, "new": 1, "shared": 0},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pick", "pick", "attend", "attend", "attend", "tables"])
    if op == "pick":
        return {"op": op, "rows": _spread(rng, 2, 256), "vocab": _spread(rng, 1000, 130001),
                "mode": rng.choice(["top_p", "top_k", "min_p", "mixed"])}
    if op == "attend":
        groups = rng.choice([1, 1, 2, 3, 4])
        kv_heads = rng.choice([1, 2, 4, 8])
        return {"op": op, "groups": groups, "rows": max(1, _spread(rng, 1, 128) // groups),
                "heads": kv_heads * rng.choice([1, 2, 3, 4, 8]), "kv_heads": kv_heads,
                "dim": rng.choice([32, 48, 64, 80, 96, 128]), "page": rng.choice([16, 32, 64, 128]),
                "shared": _spread(rng, 100, 16384), "own": _spread(rng, 1, 1024)}
    return {"op": op, "rows": _spread(rng, 1, 256), "page": rng.choice([16, 32, 64, 128]),
            "context": _spread(rng, 16, 32768), "new": rng.choice([1, 1, _spread(rng, 2, 512)]),
            "shared": rng.choice([0, _spread(rng, 16, 8192)])}


# ---------------------------------------------------------------------------------- the lengths a case stands for
def _attend_lengths(case):
    """Per group the shared keys (whole pages), per row the keys behind them (at least the new token's)."""
    page = case["page"]
    shared = [max(page, (case["shared"] - g * case["shared"] // 11) // page * page) for g in range(case["groups"])]
    n = case["groups"] * case["rows"]
    return shared, [1 + (7919 * i + 31 * case["own"]) % case["own"] for i in range(n)]


def _table_lengths(case):
    """Tokens in the cache, tokens that come, leading pages taken over from row 0, per row."""
    n, page = case["rows"], case["page"]
    shared = min(case["shared"], case["context"]) // page
    length = [shared * page + (7907 * i + 13) % max(1, case["context"] - shared * page) for i in range(n)]
    new = [1 if case["new"] == 1 or i % 4 else 1 + (4099 * i) % case["new"] for i in range(n)]
    return length, new, [0] + [shared] * (n - 1)


# ---------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return {"pick": _prepare_pick, "attend": _prepare_attend, "tables": _prepare_tables}[case["op"]](case, seed, gen)


def _pick_inputs(case, gen):
    n, vocab = case["rows"], case["vocab"]

    def uniform(lo, hi):
        return lo + (hi - lo) * torch.rand(n, generator=gen, device=DEV)

    # a body of normal logits and a tail of likely tokens above it, steeper in some rows than in others
    body = torch.randn(n, vocab, generator=gen, device=DEV)
    tail = torch.rand(n, vocab, generator=gen, device=DEV)
    logits = body * uniform(0.8, 2.5)[:, None] + torch.where(tail < 30.0 / vocab, -torch.log((tail * vocab / 30.0).clamp(min=1e-6)), 0.0) * 3.0
    temperature = uniform(0.6, 1.2)
    top_k = (1 + uniform(20, 80)).to(torch.int32)
    top_p = uniform(0.8, 0.98)
    min_p = uniform(0.02, 0.1)
    off_k, off_p, off_m = torch.zeros_like(top_k), torch.ones_like(top_p), torch.zeros_like(min_p)
    mode = case["mode"]
    if mode == "top_p":
        top_k, min_p = off_k, off_m
    elif mode == "top_k":
        min_p = off_m
    elif mode == "min_p":
        top_k, top_p = off_k, off_p
    else:                             # every row some of the filters, one of them at least
        which = torch.randint(1, 8, (n,), generator=gen, device=DEV)
        top_k = torch.where(which & 1 > 0, top_k, off_k)
        top_p = torch.where(which & 2 > 0, top_p, off_p)
        min_p = torch.where(which & 4 > 0, min_p, off_m)
    u = torch.randint(0, 1 << 24, (n,), generator=gen, device=DEV).to(torch.float32) / float(1 << 24)
    return logits, temperature, u, top_k.contiguous(), top_p.contiguous(), min_p.contiguous()


def _prepare_pick(case, seed, gen):
    logits, temperature, u, top_k, top_p, min_p = _pick_inputs(case, gen)
    return {"case": case, "logits": logits, "temperature": temperature, "u": u, "top_k": top_k, "top_p": top_p,
            "min_p": min_p, "out": torch.empty(case["rows"], dtype=torch.int32, device=DEV)}


def _attend_inputs(case, seed, gen):
    page, kv, d = case["page"], case["kv_heads"], case["dim"]
    shared, behind = _attend_lengths(case)
    n, per = len(behind), case["rows"]
    rng = np.random.default_rng(seed)
    own_pages = [-(-b // page) for b in behind]
    n_pages = sum(s // page for s in shared) + sum(own_pages) + 3
    free = iter(rng.permutation(n_pages).tolist())
    of_group = [[next(free) for _ in range(s // page)] for s in shared]
    width = max(len(of_group[r // per]) + own_pages[r] for r in range(n))
    table = np.full((n, width), -1, dtype=np.int32)
    for r in range(n):
        pages = of_group[r // per] + [next(free) for _ in range(own_pages[r])]
        table[r, :len(pages)] = pages
    positions = np.array([shared[r // per] + behind[r] - 1 for r in range(n)], dtype=np.int32)
    k = torch.randn(n_pages, kv, page, d, generator=gen, device=DEV, dtype=torch.bfloat16)
    v = torch.randn(n_pages, kv, d, page, generator=gen, device=DEV, dtype=torch.bfloat16)
    q = torch.randn(n, case["heads"], d, generator=gen, device=DEV, dtype=torch.bfloat16) * 1.5

    def ints(a):
        return torch.tensor(np.asarray(a, dtype=np.int32), device=DEV)

    return {"case": case, "q": q, "k": k, "v": v, "table": ints(table), "positions": ints(positions),
            "rows": ints(np.arange(n)), "seg_start": ints(np.arange(n)), "group_start": ints(per * np.arange(case["groups"] + 1)),
            "shared": ints(shared), "host_shared": shared, "host_behind": behind, "scale": d ** -0.5}


def _prepare_attend(case, seed, gen):
    s = _attend_inputs(case, seed, gen)
    n, heads, d = s["q"].shape
    s["out"] = torch.empty(n, heads * d, dtype=torch.bfloat16, device=DEV)
    s["max_shared"], s["max_own"] = max(s["host_shared"]), max(s["host_behind"])
    return s


def _prepare_tables(case, seed, gen):
    length, new, shared = _table_lengths(case)
    page = case["page"]
    rng = np.random.default_rng(seed)
    need = [-(-(a + b) // page) for a, b in zip(length, new)]
    n_pages = sum(m - s for m, s in zip(need, shared))
    pages = rng.permutation(2 * n_pages + 4096)[:n_pages]
    n, tokens = case["rows"], sum(new)

    def ints(a):
        return torch.tensor(np.asarray(a, dtype=np.int32), device=DEV)

    def empty(*shape, dtype=torch.int32):
        return torch.empty(*shape, dtype=dtype, device=DEV)

    return {"case": case, "lengths": ints(length), "new": ints(new), "pages": ints(pages), "leader": ints([0] * n),
            "shared": ints(shared), "width": max(need), "tokens": tokens,
            "table": empty(n, max(need)), "seg_start": empty(n), "positions": empty(tokens), "row_of_token": empty(tokens),
            "slots": empty(tokens, dtype=torch.int64), "lists": empty(n), "counts": empty(4)}


# ---------------------------------------------------------------------------------- one pass
def run(state):
    return {"pick": _run_pick, "attend": _run_attend, "tables": _run_tables}[state["case"]["op"]](state)


def _run_pick(s):
    if own:
        from imparo_amd.kernels import ops
        return ops.sample_rows(s["logits"], s["temperature"], s["u"], s["out"], top_k=s["top_k"], top_p=s["top_p"],
                               min_p=s["min_p"])
    # in 64 bits: a pick is a comparison of long sums
    x, k = s["logits"], s["top_k"].long()
    n, vocab = x.shape
    place = torch.arange(vocab, device=x.device)[None, :]
    ordered, index = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((ordered.double() - ordered[:, :1].double()) / s["temperature"].double()[:, None])
    w = torch.where(w >= 2.0 ** -44, w, 0.0)
    w = torch.where((k[:, None] <= 0) | (place < k[:, None]), w, 0.0)
    before = torch.cumsum(w, 1) - w
    p = s["top_p"].double()[:, None]
    w = torch.where((p >= 1.0) | (before < p * w.sum(1, keepdim=True)), w, 0.0)
    w = torch.where(w >= s["min_p"].double()[:, None], w, 0.0)
    by_index = torch.zeros_like(w).scatter_(1, index, w)
    running = torch.cumsum(by_index, 1)
    past = running > s["u"].double()[:, None] * running[:, -1:]
    first = torch.where(past, place, vocab).min(1).values
    last = torch.where(by_index > 0, place, 0).max(1).values
    return torch.where(first < vocab, first, last).to(torch.int32)


def _run_attend(s):
    case = s["case"]
    if own:
        from imparo_amd.kernels import ops
        n, heads, _ = s["q"].shape
        if "part_o" not in s:         # the workspace, allocated once for the plan
            parts = ops.attention_shared_parts(n, heads, case["kv_heads"], case["dim"], case["groups"], case["rows"],
                                               s["max_shared"], s["max_own"])
            s["part_o"] = torch.empty(n, heads, parts, case["dim"], dtype=torch.float32, device=DEV)
            s["part_ml"] = torch.empty(n, heads, parts, 2, dtype=torch.float32, device=DEV)
        return ops.attention_decode_shared(
            s["q"], s["k"], s["v"], s["out"], s["part_o"], s["part_ml"], s["rows"], n, s["group_start"],
            s["shared"], s["seg_start"], s["positions"], s["table"], s["scale"], None, max_shared=s["max_shared"],
            max_own=s["max_own"], max_group=case["rows"])
    kv, d, page, per = case["kv_heads"], case["dim"], case["page"], case["rows"]
    gq = case["heads"] // kv
    outs = []
    for g in range(case["groups"]):
        mine = slice(g * per, (g + 1) * per)
        q = s["q"][mine].float().view(per, kv, gq, d) * s["scale"]
        n_shared = s["host_shared"][g]
        pages = s["table"][g * per, :n_shared // page].long()
        k = s["k"][pages].float().transpose(0, 1).reshape(kv, n_shared, d)
        v = s["v"][pages].float().permute(1, 0, 3, 2).reshape(kv, n_shared, d)
        a = torch.matmul(q.transpose(0, 1).reshape(kv, per * gq, d), k.transpose(1, 2).contiguous())
        m_a = a.max(2, keepdim=True).values
        e_a = torch.exp(a - m_a)
        o_a = torch.matmul(e_a, v).view(kv, per, gq, d).transpose(0, 1)
        l_a = e_a.sum(2).view(kv, per, gq, 1).transpose(0, 1)
        m_a = m_a.view(kv, per, gq, 1).transpose(0, 1)
        # the rows' own keys, padded to the longest row of the group
        longest = -(-max(s["host_behind"][mine]) // page)
        tables = s["table"][mine, n_shared // page:n_shared // page + longest].long().clamp(min=0)
        k = s["k"][tables].float().transpose(1, 2).reshape(per, kv, tables.shape[1] * page, d)
        v = s["v"][tables].float().permute(0, 2, 1, 4, 3).reshape(per, kv, tables.shape[1] * page, d)
        b = torch.matmul(q, k.transpose(2, 3).contiguous())
        key = n_shared + torch.arange(b.shape[3], device=b.device)
        b = torch.where(key[None, None, None, :] <= s["positions"][mine, None, None, None], b, -math.inf)
        m = torch.maximum(m_a, b.max(3, keepdim=True).values)
        e_b = torch.exp(b - m)
        f = torch.exp(m_a - m)
        o = (f * o_a + torch.matmul(e_b, v)) / (f * l_a + e_b.sum(3, keepdim=True))
        outs.append(o.reshape(per, kv * gq * d))
    return torch.cat(outs).to(torch.bfloat16)


def _run_tables(s):
    page = s["case"]["page"]
    if own:
        from imparo_amd.kernels import ops
        return ops.step_tables(s["lengths"], s["new"], s["pages"], page, s["table"], s["seg_start"], s["positions"],
                               s["row_of_token"], s["slots"], s["lists"], s["counts"], leader=s["leader"], shared=s["shared"])
    length, new, shared = s["lengths"].long(), s["new"].long(), s["shared"].long()
    n = length.shape[0]
    need = (length + new + page - 1) // page
    mine = need - shared
    first = torch.cumsum(mine, 0) - mine
    j = torch.arange(s["width"], device=length.device)[None, :]
    at = (first[:, None] + j - shared[:, None]).clamp(0, s["pages"].shape[0] - 1)
    table = torch.where((j >= shared[:, None]) & (j < need[:, None]), s["pages"][at], -1)
    table = torch.where(j < shared[:, None], table[s["leader"].long()], table)
    start = torch.cumsum(new, 0) - new
    row = torch.repeat_interleave(torch.arange(n, device=length.device), new, output_size=s["tokens"])
    position = length[row] + torch.arange(s["tokens"], device=length.device) - start[row]
    slots = table[row, position // page].long() * page + position % page
    single = (new == 1).long()
    rank = torch.where(single > 0, torch.cumsum(single, 0) - 1, single.sum() + torch.cumsum(1 - single, 0) - 1)
    lists = torch.empty(n, dtype=torch.int32, device=length.device)
    lists[rank] = torch.arange(n, dtype=torch.int32, device=length.device)
    counts = torch.stack([new.sum(), mine.sum(), single.sum(), (1 - single).sum()]).to(torch.int32)
    return (table, start.to(torch.int32), position.to(torch.int32), row.to(torch.int32), slots, lists, counts)


# ---------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "pick":
        values = case["rows"] * case["vocab"]
        return {"bytes": 4 * values + 24 * case["rows"], "flops": 4 * values}
    if case["op"] == "attend":
        shared, behind = _attend_lengths(case)
        keys = sum(shared) + sum(behind)
        seen = sum(shared[r // case["rows"]] + b for r, b in enumerate(behind))
        return {"bytes": keys * case["kv_heads"] * case["dim"] * 4 + len(behind) * case["heads"] * case["dim"] * 4,
                "flops": 4 * case["heads"] * case["dim"] * seen}
    length, new, shared = _table_lengths(case)
    need = [-(-(a + b) // case["page"]) for a, b in zip(length, new)]
    own_pages = sum(m - s for m, s in zip(need, shared))
    return {"bytes": 4 * (own_pages + len(need) * max(need)) + 20 * sum(new) + 24 * len(need), "flops": 0}


# ---------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "pick":
        parts = [t.cpu().numpy() for t in _pick_inputs(case, gen)]
        return torch.tensor([_pick_row(*row) for row in zip(*parts)], dtype=torch.int32, device=DEV)
    if case["op"] == "attend":
        return _exact_attend(_attend_inputs(case, seed, gen))
    return _exact_tables(case, seed)


def _pick_row(x, temperature, u, top_k, top_p, min_p):
    """One row's pick: the kept tokens counted off one after the other in the order of their logits."""
    z = (x.astype(np.float64) - float(x.max())) / float(temperature)
    w = np.exp(z)
    likely = np.flatnonzero(w >= 2.0 ** -44)
    order = likely[np.lexsort((likely, -x[likely].astype(np.float64)))]
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1.0:
        sums = np.cumsum(w[order])
        enough = np.flatnonzero(sums >= float(top_p) * sums[-1])
        order = order[:enough[0] + 1] if len(enough) else order
    kept = np.sort(order[w[order] >= float(min_p)])
    sums = np.cumsum(w[kept])
    return int(kept[min(np.searchsorted(sums, float(u) * sums[-1], side="right"), len(kept) - 1)])


def _exact_attend(s):
    """Row by row over the whole context of each, without a shared part."""
    case = s["case"]
    kv, d, page = case["kv_heads"], case["dim"], case["page"]
    out = []
    for r, position in enumerate(s["positions"].tolist()):
        pages = s["table"][r, :position // page + 1].long()
        k = s["k"][pages].double().transpose(0, 1).reshape(kv, -1, d)[:, :position + 1]
        v = s["v"][pages].double().permute(1, 0, 3, 2).reshape(kv, -1, d)[:, :position + 1]
        q = s["q"][r].double().view(kv, -1, d)
        a = torch.softmax(torch.bmm(q, k.transpose(1, 2).contiguous()) * s["scale"], dim=2)
        out.append(torch.bmm(a, v).reshape(-1))
    return torch.stack(out)


def _exact_tables(case, seed):
    s = _prepare_tables(case, seed, None)
    page, n, width = case["page"], case["rows"], s["width"]
    length, new, shared = (s[k].tolist() for k in ("lengths", "new", "shared"))
    pages = iter(s["pages"].tolist())
    table = [[-1] * width for _ in range(n)]
    start, positions, rows, slots, used, tokens = [], [], [], [], 0, 0
    for r in range(n):
        table[r][:shared[r]] = table[0][:shared[r]]
        for j in range(shared[r], -(-(length[r] + new[r]) // page)):
            table[r][j] = next(pages)
            used += 1
        start.append(tokens)
        for p in range(length[r], length[r] + new[r]):
            positions.append(p)
            rows.append(r)
            slots.append(table[r][p // page] * page + p % page)
        tokens += new[r]
    single = [r for r in range(n) if new[r] == 1]
    other = [r for r in range(n) if new[r] != 1]

    def ints(a, dtype=torch.int32):
        return torch.tensor(a, dtype=dtype, device=DEV)

    return (ints(table), ints(start), ints(positions), ints(rows), ints(slots, torch.int64), ints(single + other),
            ints([tokens, used, len(single), len(other)]))
