"""The operators that generation needs around a paged key/value cache, as cases that can be timed, each in a plain form of elementary torch
operations too:

  plan     block tables and slot maps from request lengths, on the GPU (cache_plan)
  append   rows of new keys and values into their slots (cache_append)
  gather   the pages of every request as one contiguous tensor, which is what htree_forward takes (cache_gather)
  attend   attention of drafted tokens over the cache and over one another (draft_attention)

A cache is k [P, page, H_kv, K] and v [P, page, H_kv, V]; a request's block table row names its pages in order.  `op` says which operator
a case is of.  Sizes: B requests of up to L cached tokens (`spread`: how far the shortest is below the longest), N new tokens each, H query
heads over H_kv key/value heads, K- and V-wide rows."""
import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def _attend(dtype, B, N, H, H_kv, K, V, L, page, tree, spread=0.0, pad=False, name=None):
    c = dict(op="attend", dtype=dtype, B=B, N=N, H=H, H_kv=H_kv, K=K, V=V, L=L, page=page, tree=tree, spread=spread, pad=pad)
    return dict(c, name=name) if name else c


def _append(dtype, B, N, n, H_kv, K, V, L, page, name=None):
    c = dict(op="append", dtype=dtype, B=B, N=N, n=n, H_kv=H_kv, K=K, V=V, L=L, page=page, spread=0.5)
    return dict(c, name=name) if name else c


def _gather(dtype, B, H_kv, K, V, L, page, spread=0.0, name=None):
    c = dict(op="gather", dtype=dtype, B=B, H_kv=H_kv, K=K, V=V, L=L, page=page, spread=spread)
    return dict(c, name=name) if name else c


def _plan(B, L, n, page, spread=0.5, name=None):
    c = dict(op="plan", B=B, L=L, n=n, page=page, spread=spread)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a turn of a small batch's tables: admitted, extended by the accepted drafts, ended; latency is all there is
        _plan(16, 2048, 8, 16, name="plan_16_rows"),
        # a server's batch with long requests in small pages
        _plan(512, 16384, 16, 16, name="plan_512_rows"),
        # the accepted tokens of a batch's drafts go into the cache
        _append("bfloat16", 32, 16, 6, 4, 128, 128, 2048, 16, name="append_accepted"),
        # a prompt's keys and values go into the cache
        _append("bfloat16", 4, 16384, 16384, 2, 128, 128, 0, 64, name="append_prompt_16k"),
        # a short sequence handed to htree_forward, fp32, 64-wide heads
        _gather("float32", 1, 2, 64, 64, 2000, 16, name="gather_f32_2k"),
        # a long one
        _gather("bfloat16", 4, 4, 128, 128, 65536, 64, 0.3, name="gather_64k"),
        # one token of one request, fp32 (the smallest benchmark configuration's heads): latency
        _attend("float32", 1, 1, 8, 2, 64, 64, 2048, 16, False, name="one_token_f32_2k"),
        # generation: one new position per sequence against a cache of 16K, a batch of four
        _attend("bfloat16", 4, 1, 32, 2, 128, 128, 16384, 16, False, name="one_token_16k"),
        # drafts of many requests of all lengths, 64-wide heads, odd counts, small pages
        _attend("float16", 32, 13, 16, 2, 64, 64, 4001, 16, True, 0.95, True, name="tree_ragged_f16"),
        # a tree of drafted tokens in every request of a batch, 16 heads to a key/value head
        _attend("bfloat16", 8, 32, 64, 4, 128, 128, 16384, 32, True, 0.4, name="tree_16k"),
        # drafts against one very long cache
        _attend("bfloat16", 1, 8, 32, 4, 128, 128, 524288, 64, True, name="tree_512k"),
        # a chunk of a prompt against what is already cached
        _attend("bfloat16", 2, 512, 64, 4, 128, 128, 8192, 64, False, 0.5, name="chunk_8k"),
    ]


def draw(rng):
    """One more case of the same ranges: 1 to 64 requests (plans: 1024) of 0 to 512K tokens, chains and trees of 1 to 512 drafts, one to 16
    heads per key/value head, rows of 32 to 128, pages of 1 to 256 tokens, every storage type."""
    most = work(listed()[-1])["flops"]
    while True:
        op = rng.choice(["attend", "attend", "attend", "attend", "plan", "append", "gather"])
        dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        K, V = rng.choice([(128, 128), (128, 128), (64, 64), (64, 64), (32, 32), (80, 80), (128, 64), (96, 128)])
        page = rng.choice([1, 7, 16, 16, 32, 64, 64, 256])
        H_kv = rng.choice([1, 2, 4, 8])
        B = int(round(64 ** rng.random()))
        L = int(round(524288 ** rng.random())) - 1
        spread = rng.choice([0.0, 0.5, 1.0])
        if op == "plan":
            c = _plan(int(round(1024 ** rng.random())), min(L, 32768), int(round(32 ** rng.random())), page, spread)
            if c["B"] * (c["L"] + 64) <= 1 << 23:
                return c
        elif op == "append":
            N = int(round(16384 ** rng.random()))
            c = _append(dtype, B, N, rng.choice([N, max(1, N // 3)]), H_kv, K, V, min(L, 4096), page)
            if B * (N + c["L"]) * H_kv * (K + V) <= 1 << 27:
                return c
        elif op == "gather":
            c = _gather(dtype, B, H_kv, K, V, max(L, 1), page, spread)
            if B * L * H_kv * (K + V) <= 1 << 28:
                return c
        else:
            tree = rng.random() < 0.6
            N = int(round((64 if tree else 512) ** rng.random()))
            G = rng.choice([1, 2, 4, 5, 8, 8, 16])
            c = _attend(dtype, B, N, G * H_kv, H_kv, K, V, L, page, tree, spread, tree and rng.random() < 0.5)
            w = work(c)
            # fp32 does fewer operations a second
            if w["flops"] * (16 if dtype == "float32" else 2) <= most and w["bytes"] <= 2 << 30 and B * N * G * H_kv * (L + N) <= 1 << 29:
                return c


def _lengths(c):
    """Cached tokens of every request, longest first."""
    B, L = c["B"], c["L"]
    return [max(0, L - int(L * c["spread"] * b / max(1, B - 1)) - (b % 3 if c["spread"] else 0)) for b in range(B)]


def _drafts(c):
    """Drafted tokens of every request; the rows behind them are padding."""
    return [max(1, c["N"] - (b * 5) % c["N"]) if c["pad"] else c["N"] for b in range(c["B"])]


def _pages(tokens, page):
    return (tokens + page - 1) // page


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    lengths, page, B = _lengths(case), case["page"], case["B"]
    ints = dict(device=dev, dtype=torch.int32)

    if case["op"] == "plan":
        n = case["n"]
        most = max(lengths)
        M = _pages(most + 64, page) + 1
        P = sum(_pages(x + n, page) for x in lengths) + 1
        some = torch.randint(0, n + 1, (B,), generator=g, device=dev)
        return dict(case, width=max(1, most), M=M, lengths=torch.zeros(B, **ints), table=torch.full((B, M), -1, **ints),
                    pool=torch.randperm(P, generator=g, device=dev).to(torch.int32), top=torch.full((1,), P, **ints),
                    prompt=torch.tensor(lengths, **ints), accepted=some.to(torch.int32), ended=torch.full((B,), -1, **ints))

    dt = _DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=dt)

    H_kv, K, V = case["H_kv"], case["K"], case["V"]
    room = case.get("n", 0) if case["op"] == "append" else 0
    need = [_pages(x + room, page) for x in lengths]
    P, M = sum(need) + 3, max(max(need), 1)
    order = torch.randperm(P, generator=g, device=dev).to(torch.int32)
    table = torch.full((B, M), -1, **ints)
    at = 0
    for b, x in enumerate(need):
        table[b, :x] = order[at:at + x]
        at += x
    state = dict(case, k_cache=randn(P, page, H_kv, K), v_cache=randn(P, page, H_kv, V), table=table, lengths=torch.tensor(lengths, **ints))
    if case["op"] == "gather":
        return dict(state, T=max(case["L"], 1))
    N = case["N"]
    state.update(k=randn(B, N, H_kv, K), v=randn(B, N, H_kv, V))
    i = torch.arange(N, device=dev)
    if case["op"] == "append":
        n = case["n"]
        kept = torch.randint(1, n + 1, (B, 1), generator=g, device=dev) if n < N else torch.full((B, 1), n, device=dev)
        index = torch.rand(B, N, generator=g, device=dev).argsort(1)[:, :n].sort(1).values.to(torch.int32).contiguous() if n < N else None
        pos = state["lengths"].long()[:, None] + torch.arange(n, device=dev)
        slots = table.long().gather(1, (pos // page).clamp(max=M - 1)) * page + pos % page
        return dict(state, slots=torch.where(torch.arange(n, device=dev) < kept, slots, -1), index=index)
    parents = None
    if case["tree"]:
        # every drafted token grows out of an earlier one, or out of the cache's last
        parents = (torch.rand(B, N, generator=g, device=dev) * (i + 1)).floor().long() - 1
        drafts = torch.tensor(_drafts(case), device=dev)[:, None]
        parents = torch.where(i < drafts, torch.minimum(parents, i - 1), -2).to(torch.int32)
    return dict(state, q=randn(B, N, case["H"], K), parents=parents)


def _plan_plain(lengths, counts, table, pool, top, page, n):
    """Rows with a negative count give their pages back, in row order; then the others take theirs, in row order, from the pool's end."""
    B, M = table.shape
    P = pool.numel()
    dev = table.device
    j = torch.arange(M, device=dev)
    zero = torch.zeros_like(lengths)
    held = (lengths + page - 1) // page
    ends = counts < 0
    freed = torch.where(ends, held, zero)
    to = top + (freed.cumsum(0) - freed)[:, None] + j
    to = torch.where(j < freed[:, None], to, P).long()
    stack = torch.cat([pool, pool.new_zeros(1)]).scatter(0, to.reshape(-1), table.reshape(-1))
    free = top + freed.sum()
    table = torch.where(j < freed[:, None], -1, table)
    lengths = torch.where(ends, zero, lengths)
    held = torch.where(ends, zero, held)
    grows = (counts > 0) & (counts <= n) & ((lengths + counts + page - 1) // page <= M)
    need = torch.where(grows, (lengths + counts + page - 1) // page - held, zero)
    upto = need.cumsum(0)
    served = grows & ((upto <= free) | (need == 0))
    need_s = torch.where(served, need, zero)
    new = j - held[:, None]
    has = (new >= 0) & (new < need_s[:, None])
    from_ = free - 1 - ((upto - need)[:, None] + new)
    table = torch.where(has, stack[from_.clamp(0, P).long()], table)
    i = torch.arange(n, device=dev)
    pos = lengths[:, None] + i
    slots = table.gather(1, (pos // page).clamp(max=M - 1).long()).long() * page + pos % page
    taken = torch.where(served, counts, zero)
    slots = torch.where(i < taken[:, None], slots, -1)
    return slots, taken.to(torch.int32), (lengths + taken).to(torch.int32), table.to(torch.int32), stack[:P], (free - need_s.sum()).to(torch.int32)


def _plan_run(s):
    page, calls = s["page"], ((s["prompt"], s["width"]), (s["accepted"], s["n"]), (s["ended"], 1))
    out = {}
    for step, (counts, n) in zip(("admit", "extend", "end"), calls):
        if own:
            from htree_b200 import cache_plan
            slots, taken = cache_plan(s["lengths"], counts, s["table"], s["pool"], s["top"], page, n)
        else:
            slots, taken, lengths, table, pool, top = _plan_plain(s["lengths"], counts, s["table"], s["pool"], s["top"], page, n)
            s.update(lengths=lengths, table=table, pool=pool, top=top.view(1))
        out[step] = [slots, taken]
    return dict(out, lengths=s["lengths"], table=s["table"], pool=s["pool"], top=s["top"])


def _append_run(s):
    if own:
        from htree_b200 import cache_append
        cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], s["index"])
    else:
        B, n = s["slots"].shape
        rows = torch.arange(B, device=s["k"].device)[:, None]
        index = s["index"].long() if s["index"] is not None else torch.arange(n, device=s["k"].device)[None]
        for x, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
            flat = cache.view(-1, *cache.shape[2:])
            kept = s["slots"] >= 0
            new = x[rows, index]
            flat[s["slots"][kept]] = new[kept]
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _rows_of_cache(cache, table, T):
    """[B, T, H_kv, D]: the rows that a block table names (whatever, where it names none)."""
    page = cache.shape[1]
    pos = torch.arange(T, device=cache.device)
    at = table.long().clamp(min=0).gather(1, (pos // page).clamp(max=table.shape[1] - 1).expand(table.shape[0], T)) * page + pos % page
    return cache.reshape(-1, *cache.shape[2:])[at]


def _gather_run(s):
    if own:
        from htree_b200 import cache_gather
        return list(cache_gather(s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["T"]))
    there = (torch.arange(s["T"], device=s["table"].device) < s["lengths"][:, None])[:, :, None, None]
    return [torch.where(there, _rows_of_cache(c, s["table"], s["T"]), torch.zeros((), dtype=c.dtype, device=c.device)) for c in (s["k_cache"], s["v_cache"])]


def _ancestors(parents):
    """[B, N, N]: which drafts each draft sees, itself among them; nothing for padding.  Paths double in length from step to step."""
    B, N = parents.shape
    eye = torch.eye(N, dtype=torch.bool, device=parents.device)
    real = parents >= -1
    step = (parents.long()[:, :, None] == torch.arange(N, device=parents.device)) | eye
    seen, length = step.float(), 1
    while length < N:
        seen = (seen @ seen > 0).float()
        length *= 2
    return (seen > 0) & real[:, :, None]


def _attend_run(s):
    if own:
        from htree_b200 import draft_attention
        return list(draft_attention(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["parents"], return_lse=True))
    q, parents = s["q"], s["parents"]
    B, N, H, K = q.shape
    H_kv, V = s["H_kv"], s["V"]
    G, T = H // H_kv, s["L"]
    k = torch.cat([_rows_of_cache(s["k_cache"], s["table"], T).float(), s["k"].float()], 1)
    v = torch.cat([_rows_of_cache(s["v_cache"], s["table"], T).float(), s["v"].float()], 1)
    i = torch.arange(N, device=q.device)
    cached = (torch.arange(T, device=q.device) < s["lengths"][:, None])[:, None].expand(B, N, T)
    among = _ancestors(parents) if parents is not None else (i <= i[:, None]).expand(B, N, N)
    if parents is not None:
        cached = cached & (parents >= -1)[:, :, None]
    sees = torch.cat([cached, among], 2)[:, None, :, None]                                     # [B, 1, N, 1, T+N]
    qg = q.float().view(B, N, H_kv, G, K).permute(0, 2, 1, 3, 4).reshape(B, H_kv, N * G, K)
    score = (qg @ k.permute(0, 2, 3, 1)).mul_(K ** -0.5).view(B, H_kv, N, G, T + N).masked_fill_(~sees, -math.inf)
    most = score.amax(-1, keepdim=True)
    p = score.sub_(most.clamp(min=torch.finfo(torch.float32).min)).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(B, H_kv, N * G, T + N) @ v.permute(0, 2, 1, 3)).view(B, H_kv, N, G, V) / total.clamp(min=torch.finfo(torch.float32).tiny)
    lse = (most + total.log()).squeeze(-1)
    return [out.permute(0, 2, 1, 3, 4).reshape(B, N, H, V).to(q.dtype), lse.permute(0, 2, 1, 3).reshape(B, N, H)]


def run(state):
    return {"plan": _plan_run, "append": _append_run, "gather": _gather_run, "attend": _attend_run}[state["op"]](state)


def _bytes(dtype):
    return 4 if dtype == "float32" else 2


def work(case):
    B, page, lengths = case["B"], case["page"], _lengths(case)
    if case["op"] == "plan":
        # three calls: counts and lengths read, lengths and taken written, a table entry and a pool entry for each page given and for each
        # one taken back, and the slots
        pages = sum(_pages(x, page) for x in lengths)
        return {"bytes": 3 * 16 * B + 16 * pages + 8 * B * (max(1, max(lengths)) + case["n"] + 1), "flops": 0}
    row = _bytes(case["dtype"]) * case["H_kv"] * (case["K"] + case["V"])
    if case["op"] == "append":
        n = case["n"]
        kept = B * n if n == case["N"] else B * (n + 1) // 2
        return {"bytes": 2 * row * kept + 8 * B * n, "flops": 0}
    if case["op"] == "gather":
        return {"bytes": row * (sum(lengths) + B * max(case["L"], 1)) + 4 * sum(_pages(x, page) for x in lengths), "flops": 0}
    drafts = _drafts(case)
    seen = lambda n: sum(sum(1 / (j + 1) for j in range(i + 1)) for i in range(n)) if case["tree"] else n * (n + 1) // 2   # noqa: E731
    pairs = sum(n * x + seen(n) for n, x in zip(drafts, lengths))
    H, K, V = case["H"], case["K"], case["V"]
    rows = sum(x + n for n, x in zip(drafts, lengths))
    return {"bytes": int(row * rows + B * case["N"] * H * ((K + V) * _bytes(case["dtype"]) + 4)), "flops": int(2 * H * (K + V) * pairs)}


def exact(case, seed):
    """The attention from its definition, in 64 bits, request by request; the other operators move values and have none to compute."""
    if case["op"] != "attend":
        return None
    s = prepare(case, seed)
    q, page = s["q"].double(), s["page"]
    B, N, H, K = q.shape
    H_kv, V = s["H_kv"], s["V"]
    out = torch.zeros(B, N, H, V, dtype=torch.float64, device=q.device)
    lse = torch.full((B, N, H), -math.inf, dtype=torch.float64, device=q.device)
    for b, x in enumerate(_lengths(case)):
        parents = s["parents"][b].tolist() if s["parents"] is not None else list(range(-1, N - 1))
        sees = torch.zeros(N, N, dtype=torch.bool)
        for i, p in enumerate(parents):
            if p >= -1:
                if p >= 0:
                    sees[i] = sees[p]
                sees[i, i] = True
        real = [i for i, p in enumerate(parents) if p >= -1]
        sees = sees[real].to(q.device)
        pages = s["table"][b, :_pages(x, page)].long()
        for h in range(H_kv):
            k = torch.cat([s["k_cache"][pages, :, h].reshape(-1, K)[:x], s["k"][b, :, h]]).double()
            v = torch.cat([s["v_cache"][pages, :, h].reshape(-1, V)[:x], s["v"][b, :, h]]).double()
            for head in range(h * (H // H_kv), (h + 1) * (H // H_kv)):
                score = q[b, real, head] @ k.T / math.sqrt(K)
                score[:, x:][~sees] = -math.inf
                lse[b, real, head] = score.logsumexp(-1)
                out[b, real, head] = score.softmax(-1) @ v
    return [out, lse]
