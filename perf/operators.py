"""Pages of the cache copied, and attention of batches whose requests share prefixes, as a serving engine calls them.

A *copy* case moves pages of every layer of a cache inside its pools (requests are forked: each new one takes a copy of the page that its parent is still
writing to, and of the parent's recurrent state) or into pools of another size (the cache is resized, what is live lies at the front of the new pools).

An *attend* case is one step's attention in some layers: `prompts` prompts, each continued by `members` requests.  The pages of a prompt are held by all its
members; `root` tokens at the front of all prompts are shared by everybody.  Every request has up to `own` tokens of its own behind its prompt and brings up to
`tokens` new ones (1: a decoded token each).  How the requests share their pages is worked out once a step from their block tables, as a step does it,
and serves all its layers.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# -- cases ----------------------------------------------------------------------------------------------------------------------------
def _copy(name, layers, kv_heads, dim, vdim, page, pages, moves, ragged=True, to=0, state=0, dtype="bfloat16") -> dict:
    return {"name": name, "kind": "copy", "layers": layers, "kv_heads": kv_heads, "dim": dim, "vdim": vdim, "page": page, "pages": pages, "moves": moves,
            "ragged": ragged, "to": to, "state": state, "dtype": dtype}


def _attend(name, layers, heads, kv_heads, dim, vdim, page, prompts, members, prefix, root, own_tokens, tokens=1, rule="plain", dtype="bfloat16") -> dict:
    return {"name": name, "kind": "attend", "layers": layers, "heads": heads, "kv_heads": kv_heads, "dim": dim, "vdim": vdim, "page": page, "prompts": prompts,
            "members": members, "prefix": prefix, "root": root, "own": own_tokens, "tokens": tokens, "rule": rule, "dtype": dtype}


def listed() -> list:
    return [
        # one conversation is forked: the page that it is writing to, in all layers of Gemma-2B
        _copy("fork one", 18, 1, 256, 256, 64, 64, 1),
        # four samples of each of eight prompts: a page and the recurrent state of every new request, keys beside a model's delta-rule layers
        _copy("fork 24 and their states", 8, 4, 128, 128, 64, 160, 24, state=16 * 128 * 128),
        # 32-bit pages of odd heads, values of a size of their own, small pages
        _copy("fork 61 float32", 5, 2, 72, 40, 16, 300, 61, dtype="float32"),
        # the cache is made smaller after a burst: what is live moves to the front of smaller pools
        _copy("shrink to 320 pages", 18, 1, 256, 256, 64, 800, 300, ragged=False, to=320),
        # four samples of one prompt, every token waited for
        _attend("4 on 700", 4, 8, 1, 256, 256, 64, 1, 4, 700, 0, 40),
        # chats behind one system prompt, scores that lose by distance, small pages
        _attend("24 on 2000", 4, 16, 4, 128, 128, 16, 1, 24, 2000, 0, 500, rule="slopes"),
        # a busy server on one long instruction
        _attend("64 on 8192", 4, 8, 1, 256, 256, 64, 1, 64, 8192, 0, 300),
        # eight documents behind one instruction, eight samples each, every query head with a key head of its own
        _attend("8 x 8 on 4000", 2, 16, 16, 256, 256, 64, 8, 8, 4000, 1024, 200),
        # a book that many ask about
        _attend("96 on 32768", 2, 16, 4, 128, 128, 64, 1, 96, 32768, 0, 1000),
        # questions that arrive together behind a document: portions of prompts beside decoded tokens
        _attend("questions on 6000", 2, 8, 1, 256, 256, 64, 1, 24, 6000, 0, 100, tokens=64),
        # the 32-bit path, capped scores and sinks
        _attend("float32 16 on 1000", 2, 8, 1, 256, 256, 64, 1, 16, 1000, 0, 100, rule="capped", dtype="float32"),
        # the same with odd heads, values of a size of their own, several tokens a request
        _attend("float32 questions on 700", 2, 6, 2, 72, 40, 16, 3, 5, 700, 130, 60, tokens=9, dtype="float32"),
    ]


def _log_uniform(rng, lo, hi) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    page = rng.choice([16, 32, 64, 128])
    if rng.random() < 0.35:
        layers, kv_heads = _log_uniform(rng, 1, 18), rng.choice([1, 2, 4, 8])
        dim = rng.choice([64, 72, 128, 256])
        vdim = rng.choice([dim, dim, 40, 256])
        token = layers * kv_heads * (dim + vdim) * (2 if dtype == "bfloat16" else 4)
        most = max(1, min(400, 350_000_000 // (token * page)))
        moves = _log_uniform(rng, 1, most)
        shrink = rng.random() < 0.3
        case = _copy("", layers, kv_heads, dim, vdim, page, 2 * moves + rng.randint(2, 60), moves, not shrink, moves + rng.randint(0, 9) if shrink else 0,
                     rng.choice([0, 0, 2048, 40 * 64]), dtype)
    else:
        heads, kv_heads = rng.choice([(8, 1), (16, 4), (16, 16), (6, 2), (7, 1), (32, 8)])
        dim = rng.choice([64, 72, 96, 128, 192, 256])
        vdim = dim if rng.random() < 0.7 else rng.choice([40, 64, 128, 256])
        prompts = rng.choice([1, 1, 1, 2, 5])
        tokens = rng.choice([1, 1, 1, 5, 48])
        # (query rows, keys) of a case stay below a part of those of the largest listed one
        most = 2e8 if dtype == "bfloat16" else 2e7
        members = _log_uniform(rng, 2, max(2, 96 // prompts // (1 if tokens == 1 else 4)))
        prefix = _log_uniform(rng, 17, max(64, min(32768, int(most / (heads * prompts * members * tokens)))))
        case = _attend("", rng.choice([1, 2, 4]), heads, kv_heads, dim, vdim, page, prompts, members, prefix, rng.choice([0, 0, prefix // 3]),
                       _log_uniform(rng, 1, max(2, min(1000, prefix))), tokens, rng.choice(["plain", "plain", "slopes", "capped"]), dtype)
    del case["name"]
    return case


# -- what a program has in hand -----------------------------------------------------------------------------------------------------------
def prepare(case: dict, seed: int) -> dict:
    return _prepare_copy(case, seed) if case["kind"] == "copy" else _prepare_attend(case, seed)


def _prepare_copy(case: dict, seed: int) -> dict:
    gpu, cpu = torch.Generator(device="cuda").manual_seed(seed), torch.Generator().manual_seed(seed)
    dtype, L, H, ps = DTYPES[case["dtype"]], case["layers"], case["kv_heads"], case["page"]

    def pool(pages, *rest):
        return torch.randn(*rest[:-1], pages, H, ps, rest[-1], generator=gpu, device="cuda").to(dtype)
    n, pages, to = case["moves"], case["pages"], case["to"]
    shapes = [(L, 2, case["dim"])] if case["dim"] == case["vdim"] else [(L, case["dim"]), (L, case["vdim"])]
    pools = [pool(pages, *s) for s in shapes]
    news = [torch.zeros(*p.shape[:-4], to, *p.shape[-3:], dtype=dtype, device="cuda") for p in pools] if to else pools
    order = torch.randperm(pages, generator=cpu).tolist()
    src = order[:n]
    dst = list(range(n)) if to else order[n:2 * n]
    slots = (torch.randint(1, ps + 1, (n,), generator=cpu) if case["ragged"] else torch.full((n,), ps)).tolist()
    states, rows = None, ([], [])
    if case["state"]:
        states = torch.randn(L, 2 * n + 1, case["state"], generator=gpu, device="cuda")
        rows = (list(range(n)), list(range(n, 2 * n)))
    i64 = lambda x: torch.tensor(x, dtype=torch.int64, device="cuda")  # noqa: E731
    return {"kind": "copy", "pools": pools, "news": news, "src": src, "dst": dst, "slots": slots, "states": states, "rows": rows,
            "at": [i64(x) for x in (src, dst, slots, *rows)]}


def _lengths(case: dict, seed: int):
    """(tokens of every prompt, tokens of every request in front of its new ones, new tokens of every request)."""
    g = torch.Generator().manual_seed(seed + 3)
    G, M, ps = case["prompts"], case["members"], case["page"]
    prefix = [max(case["root"], case["prefix"] - (37 * i) % (1 + case["prefix"] // 4)) for i in range(G)]
    extra = torch.randint(0, case["own"], (G * M,), generator=g).tolist()
    # (the numbers of new tokens, which the outputs' sizes go by, are the case's own)
    new = torch.randint(1, case["tokens"] + 1, (G * M,), generator=torch.Generator().manual_seed(case["prefix"])).tolist()
    # what a prompt's last page holds beyond whole pages was copied when its members were forked: it is their own
    return [p // ps * ps for p in prefix], [prefix[r // M] + extra[r] for r in range(G * M)], new


def _prepare_attend(case: dict, seed: int) -> dict:
    gpu, cpu = torch.Generator(device="cuda").manual_seed(seed), torch.Generator().manual_seed(seed)
    dtype, L, M, ps = DTYPES[case["dtype"]], case["layers"], case["members"], case["page"]
    shared, before, new = _lengths(case, seed)
    R, root = len(before), case["root"] // ps
    ctx = [b + n for b, n in zip(before, new)]
    width = max(-(-c // ps) for c in ctx)
    total = root + sum(s // ps - min(root, s // ps) for s in shared) + sum(-(-c // ps) - shared[r // M] // ps for r, c in enumerate(ctx))
    ids = iter(torch.randperm(total, generator=cpu).tolist())
    table = torch.full((R, width), -1, dtype=torch.int32)
    front = [next(ids) for _ in range(root)]
    for p, s in enumerate(shared):
        pages = front[:s // ps] + [next(ids) for _ in range(s // ps - min(root, s // ps))]
        for r in range(p * M, (p + 1) * M):
            mine = pages + [next(ids) for _ in range(-(-ctx[r] // ps) - len(pages))]
            table[r, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
    nq, nkv, hd, vd, n = case["heads"], case["kv_heads"], case["dim"], case["vdim"], sum(new)

    def randn(*shape):
        return torch.randn(*shape, generator=gpu, device="cuda")
    state = {"kind": "attend", "case": case, "q": (2.0 * randn(L, n, nq * hd)).to(dtype), "k": randn(L, total, nkv, ps, hd).to(dtype),
             "v": randn(L, total, nkv, ps, vd).to(dtype), "table": table, "table_gpu": table.to("cuda"), "q_lens": new, "ctx_lens": ctx, "shared": shared,
             "out": torch.zeros(L, n, nq * vd, dtype=dtype, device="cuda")}
    rule = case["rule"]
    state["sinks"] = randn(nq) if rule == "capped" else None
    state["slopes"] = torch.tensor([2.0 ** (-2 - 6 * h / nq) for h in range(nq)], device="cuda") if rule == "slopes" else None
    state["cap"] = 20.0 if rule == "capped" else 0.0
    # the places of the new tokens in [requests, longest portion], the lengths, on the device
    T = max(new)
    state["places"] = torch.tensor([r * T + t for r in range(R) for t in range(new[r])], dtype=torch.int64, device="cuda")
    state["lens"] = [torch.tensor(x, dtype=torch.int64, device="cuda") for x in (shared, before)]
    return state


# -- one pass ------------------------------------------------------------------------------------------------------------------------------
@torch.inference_mode()
def run(state: dict):
    if state["kind"] == "copy":
        return _run_copy(state)
    if own:
        from wllm_b200.kernels import ops
        c, q, out, k, v = state["case"], state["q"], state["out"], state["k"], state["v"]
        nq, nkv, hd, vd, ps = c["heads"], c["kv_heads"], c["dim"], c["vdim"], c["page"]
        plan = ops.prefix_plan(state["table"], state["q_lens"], state["ctx_lens"], ps, nq, nkv, hd, vd, q.dtype)
        arrays = plan.to(q.device)
        scratch = torch.empty(plan.scratch_floats, dtype=torch.float32, device=q.device)
        for layer in range(c["layers"]):
            ops.prefix_attention(q[layer], out[layer], k[layer], v[layer], state["table_gpu"], plan, arrays, nq, nkv, hd, ps, hd ** -0.5, scratch, vd=vd,
                                 sinks=state["sinks"], cap=state["cap"], slopes=state["slopes"])
        return out
    return _attend_plain(state)


def _run_copy(state: dict):
    pools, news, states = state["pools"], state["news"], state["states"]
    if own:
        from wllm_b200.kernels import ops
        moves = [(p, q, state["src"], state["dst"], state["slots"]) for p, q in zip(pools, news)]
        if states is not None:
            rows = states.view(*states.shape[:2], 1, 1, states.shape[2])
            moves.append((rows, rows, *state["rows"], None))
        ops.copy_pages(moves)
    else:
        src, dst, slots, old, new = state["at"]
        for p, q in zip(pools, news):
            there = torch.arange(p.shape[-2], device="cuda")[None, :] < slots[:, None]                 # [moves, slots of a page]
            axis = p.dim() - 4
            moved = torch.where(there[:, None, :, None], p.index_select(axis, src), q.index_select(axis, dst))
            q.index_copy_(axis, dst, moved)
        if states is not None:
            states.index_copy_(1, new, states.index_select(1, old))
    return {"pools": news, "states": states}


def _attend_plain(state: dict):
    """Each prompt's scores for the rows of all its members at once, each request's own keys for its rows, one softmax over both."""
    c, ps, q, k, v = state["case"], state["case"]["page"], state["q"].float(), state["k"], state["v"]
    L, G, M, nq, nkv, hd, vd = c["layers"], c["prompts"], c["members"], c["heads"], c["kv_heads"], c["dim"], c["vdim"]
    R, rep, T, shared, before = G * M, nq // nkv, max(state["q_lens"]), *state["lens"]
    rows = q.new_zeros(L, R * T, nq * hd)
    rows[:, state["places"]] = q
    rows = rows.view(L, G, M, T, nkv, rep, hd).permute(0, 4, 1, 2, 3, 5, 6) * hd ** -0.5              # [L, kv heads, prompts, members, tokens, rep, hd]
    table = state["table_gpu"].long()
    front = int(max(state["shared"])) // ps                                                             # pages of the longest prompt
    at = before.view(G, M)[:, :, None] + torch.arange(T, device="cuda")                                  # positions of the new tokens [G, M, T]

    def pages(pool, which):                                                                              # [L, kv heads, ..., keys, head]
        x = pool[:, which.clamp(min=0)].float()                                                         # [L, ..., pages, kv heads, slots, head]
        return x.movedim(-3, 1).flatten(-3, -2)
    index = torch.arange(front * ps, device="cuda")
    first = table.view(G, M, -1)[:, 0, :front]
    s_front = rows.flatten(3, 5) @ pages(k, first).transpose(-1, -2)                                     # [L, kv, G, M T rep, keys]
    s_front = s_front.view(L, nkv, G, M, T, rep, -1)
    seen = (index[None, :] < shared[:, None])[:, None, None, :].expand(G, M, T, -1)
    scores, keys_at, visible = [s_front], [index.expand(G, M, T, -1)], [seen]
    # a request's own pages: its table from its prompt's end on
    widest = table.shape[1] - int(min(state["shared"])) // ps
    places = (shared // ps).repeat_interleave(M)[:, None] + torch.arange(widest, device="cuda")          # [R, pages]
    mine = table.gather(1, places.clamp(max=table.shape[1] - 1))
    key = (places * ps)[:, :, None] + torch.arange(ps, device="cuda")
    key = key.view(G, M, 1, -1).expand(G, M, T, -1)
    s_own = rows.flatten(4, 5) @ pages(k, mine).unflatten(2, (G, M)).transpose(-1, -2)
    scores.append(s_own.view(L, nkv, G, M, T, rep, -1))
    keys_at.append(key)
    visible.append(key <= at[..., None])
    s, key, visible = torch.cat(scores, -1), torch.cat(keys_at, -1), torch.cat(visible, -1)
    if state["cap"]:
        s = state["cap"] * torch.tanh(s / state["cap"])
    if state["slopes"] is not None:
        s = s - state["slopes"].view(nkv, 1, 1, 1, rep, 1) * (at[..., None] - key)[:, :, :, None, :]
    s = s.masked_fill(~visible[:, :, :, None, :], float("-inf"))
    top = s.amax(-1, keepdim=True)
    if state["sinks"] is not None:
        sink = state["sinks"].view(nkv, 1, 1, 1, rep, 1)
        top = torch.maximum(top, sink)
    e = torch.exp(s - top)
    z = e.sum(-1, keepdim=True)
    if state["sinks"] is not None:
        z = z + torch.exp(sink - top)
    cut = front * ps
    o = (e[..., :cut].flatten(3, 5) @ pages(v, first)).view(L, nkv, G, M, T, rep, vd)
    o = o + (e[..., cut:].flatten(4, 5) @ pages(v, mine).unflatten(2, (G, M))).view(L, nkv, G, M, T, rep, vd)
    o = (o / z).permute(0, 2, 3, 4, 1, 5, 6).reshape(L, R * T, nq * vd)
    return o[:, state["places"]].to(state["q"].dtype)


# -- what a pass cannot do without ------------------------------------------------------------------------------------------------------------
def work(case: dict) -> dict:
    item = 2 if case["dtype"] == "bfloat16" else 4
    if case["kind"] == "copy":
        slots = case["moves"] * case["page"] * (0.5 if case["ragged"] else 1.0)                       # (half a page on average)
        row = case["layers"] * case["kv_heads"] * (case["dim"] + case["vdim"]) * item
        return {"bytes": 2.0 * (slots * row + case["moves"] * case["layers"] * case["state"] * 4), "flops": 0.0}
    shared, before, new = _lengths(case, 0)
    M, root = case["members"], case["root"] // case["page"] * case["page"]
    keys = root + sum(s - min(root, s) for s in shared) + sum(b + n - shared[r // M] for r, (b, n) in enumerate(zip(before, new)))
    pairs = sum(n * b + n * (n + 1) / 2 for b, n in zip(before, new))
    width = case["dim"] + case["vdim"]
    return {"bytes": case["layers"] * item * float(keys * case["kv_heads"] * width + sum(new) * case["heads"] * width),
            "flops": case["layers"] * 2.0 * case["heads"] * width * pairs}


# -- the same in 64 bits, request by request ----------------------------------------------------------------------------------------------------
@torch.no_grad()
def exact(case: dict, seed: int):
    if case["kind"] == "copy":
        return None
    s = prepare(case, seed)
    nq, nkv, hd, vd, ps = case["heads"], case["kv_heads"], case["dim"], case["vdim"], case["page"]
    out = torch.empty(s["out"].shape, dtype=torch.float64, device="cuda")
    start = 0
    for r, (n, ctx) in enumerate(zip(s["q_lens"], s["ctx_lens"])):
        held = s["table"][r, :-(-ctx // ps)].tolist()
        for layer in range(case["layers"]):
            k = torch.cat([s["k"][layer, p] for p in held], dim=1)[:, :ctx].double()                   # [kv heads, ctx, hd]
            v = torch.cat([s["v"][layer, p] for p in held], dim=1)[:, :ctx].double()
            q = s["q"][layer, start:start + n].double().view(n, nq, hd)
            pos = torch.arange(ctx - n, ctx, device="cuda")
            away = pos[:, None] - torch.arange(ctx, device="cuda")[None, :]
            for h in range(nq):
                x = q[:, h] @ k[h // (nq // nkv)].T / math.sqrt(hd)
                if s["cap"]:
                    x = s["cap"] * torch.tanh(x / s["cap"])
                if s["slopes"] is not None:
                    x = x - s["slopes"][h].double() * away
                x = torch.where(away >= 0, x, float("-inf"))
                if s["sinks"] is not None:                                                               # one more term, without a value
                    x = torch.cat([x, s["sinks"][h].double().expand(n, 1)], dim=1)
                w = torch.softmax(x, dim=1)[:, :ctx]
                out[layer, start:start + n, h * vd:(h + 1) * vd] = w @ v[h // (nq // nkv)]
        start += n
    return out
