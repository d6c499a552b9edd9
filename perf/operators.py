"""Cases of the paged KV cache operators: append, attention of one new token (with accumulated attention weight), and
append under a budget with eviction by that weight.

State of a case (one layer): `kv [2, P, Hkv, page, Dh]` is a pool of pages, `table [S, M]` gives the page of every block of
`page` tokens of a session, `lens [S, Hkv]` the tokens each kv head holds, `next_pos` the position the next token gets,
`weights` / `positions` `[P, Hkv, page]` what each held token has been given by the softmax so far and where it stood.
"""
import math

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------------------------ cases
def _attn(name, S, Hq, Hkv, Dh, page, length, dtype, accumulate, ragged):
    return {"name": name, "op": "attn", "S": S, "Hq": Hq, "Hkv": Hkv, "Dh": Dh, "page": page, "length": length,
            "dtype": dtype, "accumulate": accumulate, "ragged": ragged}


def _append(name, S, Hkv, Dh, page, length, T, dtype, ragged):
    return {"name": name, "op": "append", "S": S, "Hkv": Hkv, "Dh": Dh, "page": page, "length": length, "T": T,
            "dtype": dtype, "ragged": ragged}


def _evict(name, S, Hkv, Dh, page, keep, T, sink, recent, dtype, new_weights):
    return {"name": name, "op": "evict", "S": S, "Hkv": Hkv, "Dh": Dh, "page": page, "keep": keep, "T": T, "sink": sink,
            "recent": recent, "dtype": dtype, "new_weights": new_weights}


def listed():
    return [
        # the first token of one session: nothing but latency
        _attn("attn first token", 1, 16, 16, 128, 16, 1, "bf16", False, "no"),
        # one session at the length of a 16-frame ring of 256 tokens, keeping count of what is attended to
        _attn("attn one session", 1, 16, 16, 128, 64, 4096, "bf16", True, "no"),
        # few small heads in threes, many short sessions of odd lengths, some of them empty
        _attn("attn short ragged", 33, 12, 4, 64, 32, 2000, "f16", False, "empty"),
        # a slab of 64 sessions at every length up to 17 frames of 256 tokens
        _attn("attn ragged slab", 64, 16, 16, 128, 16, 4352, "bf16", False, "yes"),
        # one long session, four query heads to a kv head, an odd length
        _attn("attn long", 1, 16, 4, 128, 128, 130001, "f16", True, "no"),
        # a slab with eight query heads to a kv head, keeping count; lengths differ between kv heads
        _attn("attn grouped slab", 64, 32, 4, 128, 64, 8192, "bf16", True, "heads"),
        # one decoding step of 64 sessions
        _append("append step", 64, 16, 128, 16, 500, 1, "bf16", "yes"),
        # prompts of different lengths, padded to the longest
        _append("append prompts", 8, 16, 128, 64, 500, 2048, "bf16", "yes"),
        # one decoding step of one session that is at its budget
        _evict("evict step", 1, 16, 128, 16, 4096, 1, 4, 64, "bf16", False),
        # 64 sessions at their budgets, a block of 16 tokens each
        _evict("evict slab", 64, 8, 128, 16, 2048, 16, 4, 128, "bf16", False),
        # prompts with the weights their own attention gave them, cut down to a budget of odd size
        _evict("evict prompts", 4, 4, 64, 32, 1001, 16000, 4, 100, "f16", True),
        # a long budget, a frame of 256 tokens
        _evict("evict long", 1, 4, 128, 64, 65536, 256, 16, 1024, "bf16", False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "append", "evict", "evict"])
    Dh, page, dtype = rng.choice([64, 128]), rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "f16"])
    S, Hkv = _log(rng, 1, 64), rng.choice([1, 2, 3, 4, 5, 8, 16])
    most = 1.0e9 / (S * Hkv * Dh * 4)          # tokens a session may have: no more than the largest listed case moves
    if op == "attn":
        Hq = Hkv * rng.choice([1, 1, 2, 3, 4, 6, 8, 16, 20])
        c = _attn("", S, Hq, Hkv, Dh, page, _log(rng, 1, int(min(131072, most))), dtype, rng.random() < 0.5,
                  rng.choice(["no", "yes", "empty", "heads"]))
    elif op == "append":
        T = _log(rng, 1, int(min(4096, most)))
        c = _append("", S, Hkv, Dh, page, _log(rng, 1, 8192), T, dtype, rng.choice(["no", "yes"]))
    else:
        keep = _log(rng, 32, int(min(65536, most)))
        T = _log(rng, 1, int(min(16384, most)))
        sink = rng.randint(0, keep // 8)
        c = _evict("", S, Hkv, Dh, page, keep, T, sink, rng.randint(0, keep // 2), dtype, rng.random() < 0.5)
    del c["name"]
    return c


def _counts(S, Hkv, most, ragged):
    """[S][Hkv] token counts up to `most`: the same for every seed, spread evenly by multiples of the golden ratio."""
    def part(i):
        return max(1, min(most, int(math.ceil(most * ((i * 0.6180339887498949) % 1.0)))))
    if ragged == "no":
        return [[most] * Hkv for _ in range(S)]
    if ragged == "heads":
        return [[most if s + h == 0 else part(s * Hkv + h) for h in range(Hkv)] for s in range(S)]
    rows = [most if s == 0 else part(s) for s in range(S)]
    if ragged == "empty":
        rows = [0 if s % 5 == 2 else n for s, n in enumerate(rows)]
    return [[n] * Hkv for n in rows]


def work(case):
    S, Hkv, Dh = case["S"], case["Hkv"], case["Dh"]
    row = 2 * Dh * 2                                                # a token's K and V of one kv head
    if case["op"] == "attn":
        tokens = sum(map(sum, _counts(S, Hkv, case["length"], case["ragged"])))
        pages = sum(-(-max(r) // case["page"]) for r in _counts(S, Hkv, case["length"], case["ragged"]))
        per = row + (8 if case["accumulate"] else 0)                # its weight is read and written
        return {"bytes": tokens * per + 2 * S * case["Hq"] * Dh * 2 + 4 * pages + 4 * S * Hkv,
                "flops": 4.0 * tokens * (case["Hq"] // Hkv) * Dh}
    if case["op"] == "append":
        new = sum(map(sum, _counts(S, Hkv, case["T"], case["ragged"])))
        return {"bytes": new * (2 * row + 8) + 16 * S * Hkv, "flops": 0}
    # every held token's weight and position is read; of the new ones those stay that are among the last `recent`, or of
    # those with weights their share of the budget, and each of them is read and written
    T, keep = case["T"], case["keep"]
    stay = T * keep // (T + keep) if case["new_weights"] else min(T, case["recent"])
    new = T * (4 if case["new_weights"] else 0)
    return {"bytes": S * Hkv * (case["keep"] * 8 + new + stay * (2 * row + 8) + 16), "flops": 0}


# ------------------------------------------------------------------------------------------------ inputs
def _held_positions(g, S, Hkv, keep, sink, recent, next_pos):
    """Positions of a cache at its budget: the first `sink`, the last `recent`, and others between, in any order."""
    i = torch.arange(keep, device="cuda")
    middle = keep - sink - recent
    gap = (next_pos - recent - sink) // max(1, middle)
    pos = torch.where(i < sink, i, torch.where(i < sink + middle, sink + (i - sink) * gap, next_pos - keep + i))
    order = torch.rand(S, Hkv, keep, generator=g, device="cuda").argsort(-1)
    return pos.int()[order]


def _spread(pool, table, values):
    """values [S, Hkv, n] into the first n slots of every session's pages."""
    S, Hkv, n = values.shape
    page = pool.shape[2]
    M = -(-n // page)
    full = torch.zeros(S, Hkv, M * page, dtype=pool.dtype, device="cuda")
    full[:, :, :n] = values
    pool[table[:, :M].reshape(-1).long()] = full.view(S, Hkv, M, page).transpose(1, 2).reshape(S * M, Hkv, page)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    S, Hkv, Dh, page, op = case["S"], case["Hkv"], case["Dh"], case["page"], case["op"]
    dtype = _DTYPE[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    room = {"attn": lambda: case["length"], "append": lambda: case["length"] + case["T"], "evict": lambda: case["keep"]}[op]()
    M = -(-room // page)
    P = S * M + 3
    table = torch.randperm(P, generator=g, device="cuda")[:S * M].view(S, M).int()
    st = {"case": case, "kv": normal(2, P, Hkv, page, Dh), "table": table,
          "weights": torch.zeros(P, Hkv, page, device="cuda"), "positions": torch.zeros(P, Hkv, page, device="cuda", dtype=torch.int32)}
    if op == "attn":
        st["q"] = normal(S, case["Hq"], 1, Dh)
        st["lens"] = torch.tensor(_counts(S, Hkv, case["length"], case["ragged"]), dtype=torch.int32, device="cuda")
        # what a token has been given in some hundred steps: most of them little
        st["weights"] = torch.rand(P, Hkv, page, generator=g, device="cuda").pow_(4)
        return st
    # new rows lie as the merged projection leaves them: [S, T, K and V of all heads]
    new = normal(S, case["T"], 2, Hkv, Dh)
    st["k_new"], st["v_new"] = new[:, :, 0].transpose(1, 2), new[:, :, 1].transpose(1, 2)
    if op == "append":
        held = torch.tensor(_counts(S, Hkv, case["length"], case["ragged"]), dtype=torch.int32, device="cuda")
        st["lens"], st["next_pos"] = held, held + 7
        st["n_new"] = torch.tensor([r[0] for r in _counts(S, Hkv, case["T"], case["ragged"])], dtype=torch.int32, device="cuda")
        st["lens_out"], st["next_pos_out"] = torch.empty_like(held), torch.empty_like(held)
        return st
    keep, sink, recent = case["keep"], case["sink"], case["recent"]
    next_pos = 4 * keep
    st["lens"] = torch.full((S, Hkv), keep, dtype=torch.int32, device="cuda")
    st["next_pos"] = torch.full((S, Hkv), next_pos, dtype=torch.int32, device="cuda")
    held = torch.rand(S, Hkv, keep, generator=g, device="cuda").pow_(4)
    held = torch.where(torch.rand(S, Hkv, keep, generator=g, device="cuda") < 0.02, 0.0, held)   # never attended to: equal
    _spread(st["weights"], table, held)
    _spread(st["positions"], table, _held_positions(g, S, Hkv, keep, sink, recent, next_pos))
    st["w_new"] = torch.rand(S, Hkv, case["T"], generator=g, device="cuda").pow_(4) if case["new_weights"] else None
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(st):
    case = st["case"]
    if case["op"] == "attn":
        weights = st["weights"] if case["accumulate"] else None
        if own:
            from world_engine_b200 import ops
            out = ops.paged_attn(st["q"], st["kv"], st["table"], st["lens"], weights=weights)
        else:
            out = _plain_attn(st["q"], st["kv"], st["table"], st["lens"], weights)
        return {"out": out, "weights": weights} if case["accumulate"] else {"out": out}
    if case["op"] == "append":
        a = (st["kv"], st["table"], st["lens"], st["next_pos"], st["k_new"], st["v_new"])
        b = {k: st[k] for k in ("n_new", "weights", "positions", "lens_out", "next_pos_out")}
        if own:
            from world_engine_b200 import ops
            ops.paged_append_(*a, **b)
        else:
            _plain_append(*a, **b)
        return {k: st[k] for k in ("kv", "weights", "positions", "lens_out", "next_pos_out")}
    a = (st["kv"], st["table"], st["lens"], st["next_pos"], st["k_new"], st["v_new"], st["weights"], st["positions"])
    b = {"keep": case["keep"], "sink": case["sink"], "recent": case["recent"], "w_new": st["w_new"]}
    if own:
        from world_engine_b200 import ops
        ops.paged_append_evict_(*a, **b)
    else:
        _plain_append_evict(*a, **b)
    return {k: st[k] for k in ("kv", "weights", "positions", "lens", "next_pos")}


# ------------------------------------------------------------------------------------------------ plain forms
def _gather(pool, table):
    """pool [P, H, page, ...] -> [S, H, M * page, ...] in the order of the tokens."""
    x = pool[table.long()].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, *x.shape[4:])


def _slots(table, index, page):
    """(page, row) of the token indexes [S, H, n]."""
    S = table.shape[0]
    block = (index // page).clamp(0, table.shape[1] - 1)
    return torch.gather(table.long()[:, None, :].expand(S, index.shape[1], -1), 2, block), index % page


def _plain_attn(q, kv, table, lens, weights):
    S, Hq, _, Dh = q.shape
    Hkv = kv.shape[2]
    held = torch.arange(table.shape[1] * kv.shape[3], device=q.device) < lens[..., None]             # [S, Hkv, N]
    k = torch.where(held[..., None], _gather(kv[0], table).float(), 0.0)
    v = torch.where(held[..., None], _gather(kv[1], table).float(), 0.0)
    x = torch.matmul(q.float().reshape(S, Hkv, Hq // Hkv, Dh), k.transpose(2, 3)) / math.sqrt(Dh)
    x = torch.where(held[:, :, None, :], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(lens[:, :, None, None] > 0, top, 0.0))
    p = e / torch.where(lens[:, :, None, None] > 0, e.sum(-1, keepdim=True), 1.0)
    if weights is not None:
        block = table.long().reshape(-1)
        add = p.sum(2).reshape(S, Hkv, table.shape[1], -1).transpose(1, 2).flatten(0, 1)
        weights[block] = weights[block] + add
    return torch.matmul(p, v).reshape(S, Hq, 1, Dh).to(q.dtype)


def _plain_append(kv, table, lens, next_pos, k_new, v_new, n_new, weights, positions, lens_out, next_pos_out):
    S, Hkv, T, Dh = k_new.shape
    t = torch.arange(T, device=kv.device)
    block, row = _slots(table, lens[..., None].long() + t, kv.shape[3])
    s, h, t = (t < n_new[:, None, None]).expand(S, Hkv, T).nonzero(as_tuple=True)
    block, row = block[s, h, t], row[s, h, t]
    kv[0, block, h, row] = k_new[s, h, t]
    kv[1, block, h, row] = v_new[s, h, t]
    weights[block, h, row] = 0.0
    positions[block, h, row] = next_pos[s, h] + t.int()
    torch.add(lens, n_new[:, None], out=lens_out)
    torch.add(next_pos, n_new[:, None], out=next_pos_out)


def _plain_append_evict(kv, table, lens, next_pos, k_new, v_new, weights, positions, keep, sink, recent, w_new):
    S, Hkv, T, Dh = k_new.shape
    page, dev = kv.shape[3], kv.device
    cap = table.shape[1] * page
    i = torch.arange(cap + T, device=dev)                     # candidates: the slots, then the new tokens
    w = torch.cat([_gather(weights, table), torch.zeros(S, Hkv, T, device=dev) if w_new is None else w_new], 2)
    pos = torch.cat([_gather(positions, table), next_pos[..., None] + torch.arange(T, device=dev, dtype=torch.int32)], 2)
    there = (i < lens[..., None]) | (i >= cap)
    end = next_pos[..., None] + T
    shielded = (pos < sink) | (pos >= end - recent)
    # best first: shielded ones, then by weight, then by index (both sorts keep the order of equals)
    order = w.sort(dim=2, descending=True, stable=True).indices
    rank = torch.where(there, torch.where(shielded, 2, 1), 0).gather(2, order).sort(dim=2, descending=True, stable=True).indices
    order = order.gather(2, rank)[:, :, :keep]
    kept = torch.zeros(S, Hkv, cap + T, dtype=torch.bool, device=dev).scatter_(2, order, True) & there
    # the index a candidate has in the order of tokens: a new one follows the held ones
    place = torch.where(i < cap, i, lens[..., None] + i - cap)
    stays = torch.zeros(S, Hkv, cap + 2 * T + 1, dtype=torch.bool, device=dev)
    stays.scatter_(2, torch.where(kept, place, cap + 2 * T), True)
    goes = kept & (place >= keep)
    hole = ~stays[:, :, :keep]
    m = min(keep, T + cap)
    src = goes.sort(dim=2, descending=True, stable=True).indices[:, :, :m]                  # j-th mover
    dst = hole.sort(dim=2, descending=True, stable=True).indices[:, :, :m]                  # j-th hole
    moving = torch.arange(m, device=dev) < goes.sum(2, keepdim=True)
    at = (kept & (i >= cap) & (place < keep)).nonzero(as_tuple=True)                        # new ones that lie below the budget
    s, h, j = moving[:, :, :src.shape[2]].nonzero(as_tuple=True)
    s, h, src, dst = (torch.cat(x) for x in ((s, at[0]), (h, at[1]), (src[s, h, j], at[2]), (dst[s, h, j], place[at])))
    new = src >= cap
    t = (src - cap).clamp(min=0)
    old = src.clamp(max=cap - 1)
    from_page, from_row = table.long()[s, old // page], old % page
    to_page, to_row = table.long()[s, dst // page], dst % page
    k = torch.where(new[:, None], k_new[s, h, t], kv[0, from_page, h, from_row])
    v = torch.where(new[:, None], v_new[s, h, t], kv[1, from_page, h, from_row])
    kv[0, to_page, h, to_row] = k
    kv[1, to_page, h, to_row] = v
    weights[to_page, h, to_row] = w[s, h, src]
    positions[to_page, h, to_row] = pos[s, h, src]
    lens.copy_((lens + T).clamp(max=keep))
    next_pos.add_(T)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_attn(case, st):
    S, Hq, Hkv, page, Dh = case["S"], case["Hq"], case["Hkv"], case["page"], case["Dh"]
    G = Hq // Hkv
    out = torch.zeros(S, Hq, 1, Dh, dtype=torch.float64, device="cuda")
    weights = st["weights"].double()
    lens, table = st["lens"].tolist(), st["table"].long()
    for s in range(S):
        for h in range(Hkv):
            n = lens[s][h]
            if n == 0:
                continue
            blocks = table[s, :-(-n // page)]
            k, v = (st["kv"][c, blocks, h].double().reshape(-1, Dh)[:n] for c in (0, 1))
            x = (k @ st["q"][s, h * G:(h + 1) * G, 0].double().T) * Dh ** -0.5                # [n, G]
            x = torch.exp(x - x.max(0).values)
            p = x / x.sum(0)
            out[s, h * G:(h + 1) * G, 0] = p.T @ v
            row = torch.zeros(len(blocks) * page, dtype=torch.float64, device="cuda")
            row[:n] = p.sum(1)
            weights[blocks, h] += row.view(-1, page)
    return {"out": out, "weights": weights} if case["accumulate"] else {"out": out}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "attn":
        return _exact_attn(case, st)
    # rows are copied and nothing is computed: what goes where is decided token by token, on the host
    S, Hkv, page, T = case["S"], case["Hkv"], case["page"], case["T"]
    if S * Hkv * (T + case.get("keep", 0)) > 3_000_000:
        return None
    kv, weights, positions = st["kv"].float().cpu(), st["weights"].double().cpu(), st["positions"].cpu()
    k_new, v_new = st["k_new"].float().cpu(), st["v_new"].float().cpu()
    table, lens, next_pos = st["table"].tolist(), st["lens"].tolist(), st["next_pos"].tolist()
    moves = []                                                                          # (s, h, from page, from row or new token, page, row)
    for s in range(S):
        for h in range(Hkv):
            n = lens[s][h]
            where = [(table[s][i // page], i % page) for i in range(min(n + T, len(table[s]) * page))]
            if case["op"] == "append":
                moves += [(s, h, None, t) + where[n + t] for t in range(int(st["n_new"][s]))]
                continue
            held = torch.tensor(where[:n]).long().reshape(-1, 2)
            w = weights[held[:, 0], h, held[:, 1]].tolist() + (st["w_new"][s, h].tolist() if st["w_new"] is not None else [0.0] * T)
            pos = positions[held[:, 0], h, held[:, 1]].tolist() + [next_pos[s][h] + t for t in range(T)]
            safe = [p < case["sink"] or p >= next_pos[s][h] + T - case["recent"] for p in pos]
            best = sorted(range(n + T), key=lambda i: (not safe[i], -w[i], i))[:case["keep"]]
            best_set = set(best)
            holes = [i for i in range(min(case["keep"], n + T)) if i not in best_set]
            movers = sorted(i for i in best if i >= case["keep"])
            for i, j in list(zip(movers, holes)) + [(i, i) for i in best if n <= i < case["keep"]]:
                moves.append((s, h, where[i][0] if i < n else None, where[i][1] if i < n else i - n) + where[j])
    if moves:
        s, h, block, row, to, at = (torch.tensor([-1 if x is None else x for x in c]) for c in zip(*moves))
        new, old, t = block < 0, block.clamp(min=0), torch.where(block < 0, row, 0)
        row = torch.where(new, 0, row)
        w_new = st["w_new"].cpu().double() if st.get("w_new") is not None else torch.zeros(S, Hkv, T, dtype=torch.float64)
        k = torch.where(new[:, None], k_new[s, h, t], kv[0, old, h, row])
        v = torch.where(new[:, None], v_new[s, h, t], kv[1, old, h, row])
        w = torch.where(new, w_new[s, h, t], weights[old, h, row])
        p = torch.where(new, st["next_pos"].cpu()[s, h] + t.int(), positions[old, h, row])
        kv[0, to, h, at], kv[1, to, h, at], weights[to, h, at], positions[to, h, at] = k, v, w, p
    if case["op"] == "append":
        n = st["n_new"].cpu()[:, None]
        return {"kv": kv, "weights": weights, "positions": positions, "lens_out": st["lens"].cpu() + n, "next_pos_out": st["next_pos"].cpu() + n}
    return {"kv": kv, "weights": weights, "positions": positions, "lens": (st["lens"].cpu() + T).clamp(max=case["keep"]),
            "next_pos": st["next_pos"].cpu() + T}
