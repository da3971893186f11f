"""Measured cases of what speculative decoding and cache eviction need around the paged KV cache.

One layer's cache holds bf16 keys and values [slots, hkv * 128], slot = page * 16 + offset; a page table names each
sequence's pages in order.

* decode: one query token for each sequence, which also adds what each key received: ``mass[sequence, KV head, key] +=``
  the softmax weights of the KV head's query heads, summed.
* evict: each KV head keeps ``keep`` of its sequence's keys: the first ``sink``, the last ``recent`` and, of the others,
  those with the largest mass (equal ones: the lowest place). Kept rows move, in order, to the front of the sequence's
  pages.
* tree: attention of drafted tokens. A sequence's last keys are its drafted nodes; a node sees all keys before them and
  the nodes that its mask names (its ancestors and itself).
* verify: what a step does around a tree: each node's mask from the nodes' parents, the walk from the root along nodes
  whose token is what the model chose at their parent, and the walk's rows moved, in every layer, to where the sequence
  goes on.

The shapes are those of the framework's presets (32 or 64 query heads over 8 KV heads of 128), and of their
tensor-parallel shards in the drawn cases.
"""

import math

import torch

own = False

D = 128
PAGE = 16


# ------------------------------------------------------------------ cases


def listed():
    return [
        # one user, one token
        {"name": "decode 1 x 100", "op": "decode", "hq": 32, "hkv": 8, "batch": 1, "len": 100, "ragged": False, "runs": True},
        # continuous batching: sequences of every age, pages from all over the pool
        {"name": "decode 61 ragged 12000", "op": "decode", "hq": 32, "hkv": 8, "batch": 61, "len": 12000, "ragged": True, "runs": False},
        # a large batch over long contexts, eight query heads to a KV head
        {"name": "decode 32 x 8192", "op": "decode", "hq": 64, "hkv": 8, "batch": 32, "len": 8192, "ragged": False, "runs": True},
        # one chat that reached its budget: half of a small cache goes
        {"name": "evict 1 x 1025 to 512", "op": "evict", "hkv": 8, "batch": 1, "len": 1025, "ragged": False, "keep": 512, "recent": 64, "sink": 4, "runs": True},
        # sequences of every age brought under one budget (some are below it already)
        {"name": "evict 12 ragged 9000 to 2048", "op": "evict", "hkv": 8, "batch": 12, "len": 9000, "ragged": True, "keep": 2048, "recent": 256, "sink": 4, "runs": False},
        # long documents after their prompt
        {"name": "evict 4 x 100001 to 8192", "op": "evict", "hkv": 8, "batch": 4, "len": 100001, "ragged": False, "keep": 8192, "recent": 1024, "sink": 16, "runs": True},
        # one user, a chain or a small tree of guesses after a short question
        {"name": "tree 1 x 8 over 500", "op": "tree", "hq": 32, "hkv": 8, "seqs": 1, "nodes": 8, "ctx": 500, "ragged": False, "runs": True},
        # continuous batching: trees and contexts of every size, scattered pages
        {"name": "tree 40 ragged 26 over 5000", "op": "tree", "hq": 32, "hkv": 8, "seqs": 40, "nodes": 26, "ctx": 5000, "ragged": True, "runs": False},
        # large trees over long contexts, eight query heads to a KV head
        {"name": "tree 16 x 64 over 8192", "op": "tree", "hq": 64, "hkv": 8, "seqs": 16, "nodes": 64, "ctx": 8192, "ragged": False, "runs": True},
        # one very long document
        {"name": "tree 1 x 61 over 100001", "op": "tree", "hq": 32, "hkv": 8, "seqs": 1, "nodes": 61, "ctx": 100001, "ragged": False, "runs": True},
        # one user, a small model
        {"name": "verify 1 x 8, 32 layers", "op": "verify", "hkv": 8, "layers": 32, "seqs": 1, "nodes": 8, "ctx": 500, "ragged": False, "runs": True},
        # a full batch of large trees, a deep model
        {"name": "verify 48 ragged 60, 80 layers", "op": "verify", "hkv": 8, "layers": 80, "seqs": 48, "nodes": 60, "ctx": 300, "ragged": True, "runs": False},
    ]


def _between(rng, lo, hi):
    """A whole number, even over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["decode", "evict", "tree", "verify"])
    hkv = rng.choice([1, 2, 4, 8])
    case = {"op": op, "hkv": hkv, "ragged": rng.random() < 0.5, "runs": rng.random() < 0.5}
    if op in ("decode", "tree"):
        case["hq"] = hkv * rng.choice([1, 2, 4, 8])
    if op == "decode":
        case["batch"] = _between(rng, 1, 128)
        case["len"] = _between(rng, 1, min(100000, 32 * 8192 // case["batch"]))
    elif op == "evict":
        case["batch"] = _between(rng, 1, 32)
        case["len"] = _between(rng, 2, min(100000, 300000 // case["batch"]))
        case["keep"] = _between(rng, 1, min(8192, case["len"]))
        case["sink"] = rng.choice([0, 4, 16]) if case["keep"] >= 32 else 0
        case["recent"] = rng.choice([0, 1, case["keep"] // 8, case["keep"] // 2])
    elif op == "tree":
        case["seqs"] = _between(rng, 1, 48)
        case["nodes"] = _between(rng, 1, 128)
        case["ctx"] = _between(rng, 1, min(100000, 16 * 8192 // case["seqs"]))
    else:
        case["layers"] = rng.choice([32, 64, 80])
        case["seqs"] = _between(rng, 1, 48)
        case["nodes"] = _between(rng, 1, 128)
        case["ctx"] = _between(rng, 1, 300)
    return case


def _shape(case):
    """(new tokens, keys) of every sequence: its drafted nodes or one token, and all of its keys with them. The case alone sets them."""
    g = torch.Generator().manual_seed(5)
    rnd = lambda n, lo, hi: torch.randint(lo, hi + 1, (n,), generator=g).tolist()  # noqa: E731
    if case["op"] in ("decode", "evict"):
        n = case["batch"]
        return [1] * n, rnd(n, 1, case["len"]) if case["ragged"] else [case["len"]] * n
    n = case["seqs"]
    rows = rnd(n, 1, case["nodes"]) if case["ragged"] else [case["nodes"]] * n
    ctx = rnd(n, 0, case["ctx"]) if case["ragged"] else [case["ctx"]] * n
    return rows, [c + r for c, r in zip(ctx, rows)]


def _trees(rows):
    """Parents of every sequence's nodes (-1: the root), and whether the model's choice at a node's parent is the node's token. The sizes alone set them."""
    g = torch.Generator().manual_seed(7)
    parents, hits = [], []
    for n in rows:
        # mostly the node before or one of the first few: some chains, some wide levels
        back = torch.where(torch.rand(n, generator=g) < 0.4, torch.ones(n), torch.rand(n, generator=g) * torch.arange(n) + 1).long()
        parents.append([-1] + [max(0, i - int(back[i])) for i in range(1, n)])
        hits.append((torch.rand(n, generator=g) < 0.6).tolist())
    return parents, hits


def _walk(parents, hits):
    """The nodes from the root on, each the first child whose token was chosen."""
    path = [0]
    while True:
        on = [i for i in range(path[-1] + 1, len(parents)) if parents[i] == path[-1] and hits[i]]
        if not on:
            return path
        path.append(on[0])


def work(case):
    rows, keys = _shape(case)
    hkv, T = case["hkv"], sum(rows)
    row = 2 * D  # bytes
    if case["op"] == "evict":
        kept = [min(n, case["keep"]) for n in keys]
        moved = sum(k - case["sink"] for n, k in zip(keys, kept) if n > k)
        return {"bytes": 4 * hkv * (sum(keys) + 2 * sum(kept)) + 4 * hkv * moved * row, "flops": hkv * sum(keys)}
    if case["op"] == "verify":
        parents, hits = _trees(rows)
        paths = [_walk(p, h) for p, h in zip(parents, hits)]
        moved = sum(i != n for p in paths for i, n in enumerate(p))
        words = -(-max(rows) // 32)
        return {"bytes": (12 + 4 * words) * T + 4 * sum(len(p) for p in paths) + 4 * case["layers"] * hkv * moved * row, "flops": T}
    hq = case["hq"]
    cache = sum(2 * hkv * n * row + 4 * -(-n // PAGE) for n in keys)
    if case["op"] == "decode":  # the accumulated weights are read and written
        return {"bytes": cache + 2 * T * hq * row + 8 * hkv * sum(keys), "flops": 4 * D * hq * sum(keys) + 2 * hq * sum(keys)}
    # a tree is dense in its context and sees a few of its own nodes
    pairs = sum(r * (n - r) + r * min(r, 6) for r, n in zip(rows, keys))
    return {"bytes": cache + 2 * T * hq * row + 4 * T * -(-max(rows) // 32), "flops": 4 * D * hq * pairs}


# ------------------------------------------------------------------ inputs


def _table(keys, g, runs):
    """Page table [sequences, most pages] over a pool with a few pages to spare, and the pool's size."""
    need = [-(-n // PAGE) for n in keys]
    pool = sum(need) + 7
    order = torch.arange(pool) if runs else torch.randperm(pool, generator=g)
    table = torch.zeros(len(keys), max(1, max(need)), dtype=torch.int32)
    at = 3
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n].to(torch.int32)
        at += n
    return table, pool


def _cache(shape, g, v):
    """Keys have a few large dimensions, as rotated keys do; values differ in size from token to token."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)
    if v:
        x *= torch.exp2(torch.randint(-2, 2, (*shape[:-1], 1), generator=g, device="cuda").float()).to(x.dtype)
    else:
        x.unflatten(-1, (-1, D))[..., 5:11] *= 4.0
    return x


def _masks(parents, words):
    """int32 [nodes of all sequences, words]: bit j of a row, node j of its sequence is the row's own or an ancestor."""
    out = []
    for p in parents:
        bits = []
        for i, up in enumerate(p):
            bits.append((1 << i) | (bits[up] if up >= 0 else 0))
        out += [[(b >> (32 * w)) & 0xFFFFFFFF for w in range(words)] for b in bits]
    t = torch.tensor(out, dtype=torch.int64)
    return torch.where(t >= 1 << 31, t - (1 << 32), t).to(torch.int32)


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed * 13 + 1)
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, hkv = case["op"], case["hkv"]
    rows, keys = _shape(case)
    n, T = len(rows), sum(rows)
    table, pool = _table(keys, host, case["runs"])
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    st = {"case": case, "hkv": hkv, "rows": rows, "keys": keys, "table": table.cuda(), "len": i32(keys), "scale": 1.0 / math.sqrt(D)}
    lead = (case["layers"],) if op == "verify" else ()
    st["k"], st["v"] = (_cache((*lead, pool * PAGE, hkv * D), g, v) for v in (False, True))
    if op in ("decode", "tree"):
        # the queries lie in front of the step's keys and values, as the projection left them
        st["qkv"] = torch.randn(T, (case["hq"] + 2 * hkv) * D, generator=g, device="cuda").to(torch.bfloat16)
    if op in ("decode", "evict"):
        # a few keys hold most of the weight, some never got any; nothing behind a sequence's last key
        mass = torch.exp(2.5 * torch.randn(n, hkv, table.shape[1] * PAGE, generator=g, device="cuda") - 3)
        mass[torch.rand(mass.shape, generator=g, device="cuda") < 0.1] = 0
        mass[(torch.arange(mass.shape[2], device="cuda") >= st["len"][:, None])[:, None].expand_as(mass)] = 0
        st["mass"] = mass
    if op in ("tree", "verify"):
        parents, hits = _trees(rows)
        start = [sum(rows[:i]) for i in range(n)]
        st["start"], st["n"], st["words"] = i32(start), i32(rows), -(-max(rows) // 32)
        st["past"] = i32([k - r for k, r in zip(keys, rows)])
        st["parents"] = i32([p for t in parents for p in t])
        # plan of the plain forms: which row of a padded [sequences, most rows] block each row is
        st["at"] = torch.cat([torch.arange(r) + i * max(rows) for i, r in enumerate(rows)]).cuda()
        if op == "tree":
            st["mask"] = _masks(parents, st["words"]).cuda()
            return st
        target = torch.randint(0, 128256, (T,), generator=host)
        other = torch.randint(0, 128256, (T,), generator=host)
        up = torch.tensor([s + max(p, 0) for s, t in zip(start, parents) for p in t])
        hit = torch.tensor([h for t in hits for h in t])
        st["tokens"] = torch.where(hit, target[up], torch.where(other == target[up], (other + 1) % 128256, other)).to(torch.int32).cuda()
        st["target"] = target.to(torch.int32).cuda()
        st["most"] = max(len(_walk(p, h)) for p, h in zip(parents, hits)) + 2
    return st


# ------------------------------------------------------------------ plain forms


def _gather(x, table):
    """fp32 rows [sequences, keys, heads, 128] of a page table's pages."""
    n, pages = table.shape
    return x.view(-1, PAGE, x.shape[-1])[table.long()].float().view(n, pages * PAGE, -1, D)


def _weights(q, st, seen):
    """Softmax weights [sequences, hkv, group, rows, keys] of q [sequences, rows, hq, 128] over the keys that `seen`
    [sequences, rows, keys] names, and the values. Rows that see none have weights of zero."""
    n, r, hq, _ = q.shape
    hkv = st["hkv"]
    k, v = _gather(st["k"], st["table"]), _gather(st["v"], st["table"])
    v = torch.where((torch.arange(k.shape[1], device=q.device) < st["len"][:, None])[..., None, None], v, 0.0)
    qg = q.view(n, r, hkv, hq // hkv, D).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, D)
    s = (qg @ k.permute(0, 2, 3, 1)).view(n, hkv, hq // hkv, r, -1) * st["scale"]
    s = torch.where(seen[:, None, None], s, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > float("-inf"), top, 0.0))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, 1.0), v


def _values(p, v):
    n, hkv, g, r, _ = p.shape
    o = p.reshape(n, hkv, g * r, -1) @ v.permute(0, 2, 1, 3)
    return o.view(n, hkv, g, r, D).permute(0, 3, 1, 2, 4).reshape(n, r, hkv * g * D)


def _plain_decode(st):
    hq = st["case"]["hq"]
    q = st["qkv"][:, :hq * D].float().view(-1, 1, hq, D)
    p, v = _weights(q, st, (torch.arange(st["table"].shape[1] * PAGE, device=q.device) < st["len"][:, None])[:, None])
    st["mass"] += p.sum((2, 3))
    return [_values(p, v)[:, 0].to(torch.bfloat16), st["mass"]]


def _slots(table, place):
    """Cache slots of places [sequences, ...] in the sequences' pages."""
    flat = place.reshape(place.shape[0], -1)
    return (table.long().gather(1, flat // PAGE) * PAGE + flat % PAGE).view(place.shape)


def _move(st, src, dst):
    """Rows of places `src` [sequences, hkv, m] to places `dst` of the same sequence and KV head, in every layer."""
    a, b = _slots(st["table"], src), _slots(st["table"], dst)
    head = torch.arange(st["hkv"], device=src.device)[None, :, None].expand_as(src)
    for x in (st["k"], st["v"]):
        x = x.view(-1, x.shape[-2], st["hkv"], D)
        x[:, b, head] = x[:, a, head]


def _plain_evict(st):
    c, mass = st["case"], st["mass"]
    n, hkv, cap = mass.shape
    place = torch.arange(cap, device=mass.device)
    size = st["len"].long()[:, None, None]
    must = ((place < c["sink"]) | (place >= size - c["recent"])) & (place < size)
    value = torch.where(must, float("inf"), torch.where(place < size, mass, float("-inf")))
    best = torch.sort(value, dim=-1, descending=True, stable=True).indices[..., :c["keep"]]
    # those of shorter sequences that do not exist go behind the others
    kept = torch.full((n, hkv, c["keep"]), cap, device=mass.device)
    kept[..., :best.shape[-1]] = torch.sort(torch.where(best < size, best, cap)).values
    have = kept < size
    kept_mass = torch.where(have, mass.gather(2, kept.clamp(max=cap - 1)), 0.0)
    # (a sequence with fewer keys than `keep` keeps its places: there, the first row is read and written)
    to = torch.arange(c["keep"], device=mass.device).expand_as(kept)
    _move(st, torch.where(have, kept, 0), torch.where(have, to, 0))
    count = st["len"].clamp(max=c["keep"])
    return [torch.where(have, kept, -1).to(torch.int32), kept_mass, count, st["k"], st["v"]]


def _bits(mask, n):
    j = torch.arange(n, device=mask.device)
    return (mask[:, j // 32] >> (j % 32)) & 1 > 0


def _plain_tree(st):
    hq, n, most = st["case"]["hq"], len(st["rows"]), max(st["rows"])
    q = torch.zeros(n * most, hq * D, device="cuda")
    q[st["at"]] = st["qkv"][:, :hq * D].float()
    nodes = torch.zeros(n * most, 32 * st["words"], dtype=torch.bool, device="cuda")
    nodes[st["at"]] = _bits(st["mask"], 32 * st["words"])
    place = torch.arange(st["table"].shape[1] * PAGE, device="cuda") - st["past"][:, None]
    mine = nodes.view(n, most, -1).gather(2, place.clamp(0, 32 * st["words"] - 1).long()[:, None].expand(-1, most, -1))
    seen = (place < 0)[:, None] | (mine & (place < st["n"][:, None])[:, None])
    p, v = _weights(q.view(n, most, hq, D), st, seen)
    return [_values(p, v).view(n * most, -1)[st["at"]].to(torch.bfloat16)]


def _plain_verify(st):
    n, most, words = len(st["rows"]), max(st["rows"]), st["words"]
    pad = lambda x, fill: torch.full((n * most,), fill, device="cuda").index_copy_(0, st["at"], x.long()).view(n, most)  # noqa: E731
    up, token, target = pad(st["parents"], -1), pad(st["tokens"], -1), pad(st["target"], -2)
    node = torch.arange(most, device="cuda")
    # (ancestors, own) by doubling: after step i the edges of up to 2^i generations
    over = ((up[..., None] == node) | (node[:, None] == node)).float()
    for _ in range(max(1, (most - 1).bit_length())):
        over = ((over @ over) > 0).float()
    bits = torch.zeros(n, most, words * 32, dtype=torch.int64, device="cuda")
    bits[..., :most] = over.long()
    mask = (bits.view(n, most, words, 32) << torch.arange(32, device="cuda")).sum(-1)
    mask = torch.where(mask >= 1 << 31, mask - (1 << 32), mask).to(torch.int32).view(n * most, words)[st["at"]]
    # a node is on the way if its token is its parent's choice and no earlier child's is
    hit = (up >= 0) & (token == target.gather(1, up.clamp(min=0)))
    rival = (up[:, :, None] == up[:, None, :]) & hit[:, None, :] & (node[None, :] < node[:, None])
    on = (hit & ~rival.any(-1)) | (node == 0)
    good = ((over > 0) & ~on[:, None, :]).sum(-1) == 0
    good &= over[..., 0] > 0
    depth = torch.where(good, over.sum(-1).long() - 1, most)
    path = torch.full((n, max(most, st["most"]) + 1), -1, dtype=torch.int64, device="cuda")
    path.scatter_(1, depth, torch.where(good, node, -1))
    path[:, most] = -1
    path = path[:, :st["most"]]
    count = (path >= 0).sum(1)
    last = path.gather(1, count[:, None] - 1)
    after = target.gather(1, last)[:, 0]
    step = torch.arange(st["most"], device="cuda").expand_as(path)
    there = path >= 0
    # (places that do not move read and write the sequence's first row)
    from_, to = (torch.where(there, x + st["past"].long()[:, None], 0)[:, None].expand(-1, st["hkv"], -1) for x in (path, step))
    _move(st, from_, to)
    return [mask, path.to(torch.int32), count.to(torch.int32), after.to(torch.int32), st["k"], st["v"]]


# ------------------------------------------------------------------ the framework's calls


def _own(st):
    from infera_b200.ops import evict, tree
    from infera_b200.ops import kernels as K

    c, op, hkv = st["case"], st["case"]["op"], st["hkv"]
    if op == "decode":
        splits, tps = evict.decode_plan(len(st["keys"]), hkv, max(st["keys"]))
        out = K.attn_decode(st["qkv"], st["k"], st["v"], st["table"], st["len"], c["hq"], hkv, st["scale"], splits=splits, tiles_per_split=tps, mass=st["mass"])
        return [out, st["mass"]]
    if op == "evict":
        kept, kept_mass, count = evict.select_keys(st["mass"], st["len"], c["keep"], recent=c["recent"], sink=c["sink"])
        K.kv_compact(st["k"], st["v"], st["table"], kept, count)
        return [kept, kept_mass, count, st["k"], st["v"]]
    if op == "tree":
        return [tree.attn_tree(st["qkv"], st["k"], st["v"], st["table"], st["start"], st["n"], st["len"], st["mask"], c["hq"], hkv, st["scale"],
                               host_meta=(st["rows"], st["keys"]))]
    mask = tree.tree_mask(st["parents"], st["start"], st["n"], st["words"])
    path, count, after = tree.tree_accept(st["tokens"], st["target"], st["parents"], st["start"], st["n"], st["most"])
    K.kv_compact(st["k"], st["v"], st["table"], path, count, start=st["past"])
    return [mask, path, count, after, st["k"], st["v"]]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "decode":
        return _plain_decode(state)
    if op == "evict":
        return _plain_evict(state)
    return _plain_tree(state) if op == "tree" else _plain_verify(state)


# ------------------------------------------------------------------ 64 bits


def _exact_attention(st, sees):
    """fp64 attention, sequence by sequence and head by head; `sees(i)` is the [rows, keys] mask of sequence i. Also every
    KV head's summed weights."""
    hq, hkv = st["case"]["hq"], st["hkv"]
    out = torch.zeros(st["qkv"].shape[0], hq * D, dtype=torch.float64, device="cuda")
    got = torch.zeros(len(st["keys"]), hkv, st["table"].shape[1] * PAGE, dtype=torch.float64, device="cuda")
    at = 0
    for i, (r, n) in enumerate(zip(st["rows"], st["keys"])):
        pages = st["table"][i, :-(-n // PAGE)].long()
        hidden = ~sees(i)
        for h in range(hq):
            kv = h // (hq // hkv)
            k, v = (x.view(-1, PAGE, hkv, D)[pages, :, kv].reshape(-1, D)[:n].double() for x in (st["k"], st["v"]))
            s = st["qkv"][at:at + r, h * D:(h + 1) * D].double() @ k.T / math.sqrt(D)
            p = torch.softmax(s.masked_fill(hidden, float("-inf")), -1)
            out[at:at + r, h * D:(h + 1) * D] = p @ v
            got[i, kv, :n] += p.sum(0)
        at += r
    return out, got


def _exact_moves(st, moves):
    """Both caches after moves[i][head] = [(from, to)] of places of sequence i."""
    table = st["table"].cpu()
    seq, head, src, dst = [], [], [], []
    for i, per in enumerate(moves):
        for h, pairs in enumerate(per):
            seq += [i] * len(pairs)
            head += [h] * len(pairs)
            src += [a for a, _ in pairs]
            dst += [b for _, b in pairs]
    seq, head, src, dst = (torch.tensor(x, dtype=torch.int64) for x in (seq, head, src, dst))
    a, b = (table[seq, x // PAGE].long() * PAGE + x % PAGE for x in (src, dst))
    a, b, head = a.cuda(), b.cuda(), head.cuda()
    res = []
    for x in (st["k"], st["v"]):
        y = x.view(-1, x.shape[-2], st["hkv"], D).double()
        y[:, b, head] = x.view(y.shape)[:, a, head].double()
        res.append(y.view(x.shape))
    return res


def _exact_evict(st):
    c, mass = st["case"], st["mass"].double().cpu().numpy()
    keep = c["keep"]
    kept = torch.full((len(st["keys"]), st["hkv"], keep), -1, dtype=torch.int64)
    value = torch.zeros(kept.shape, dtype=torch.float64)
    moves = []
    for i, n in enumerate(st["keys"]):
        moves.append([])
        for h in range(st["hkv"]):
            if n <= keep:
                on = list(range(n))
            else:
                mid = range(c["sink"], n - c["recent"])
                want = keep - c["sink"] - c["recent"]
                m = mass[i, h].tolist()
                best = sorted(mid, key=lambda j: -m[j])[:want]  # (stable: the lowest place first)
                on = list(range(c["sink"])) + sorted(best) + list(range(n - c["recent"], n))
            kept[i, h, :len(on)] = torch.tensor(on)
            value[i, h, :len(on)] = torch.from_numpy(mass[i, h])[on]
            moves[-1].append([(a, b) for b, a in enumerate(on) if a != b])
    count = torch.tensor([min(n, keep) for n in st["keys"]])
    return [kept, value, count, *_exact_moves(st, moves)]


def _exact_verify(st):
    parents, tokens, target = (st[x].tolist() for x in ("parents", "tokens", "target"))
    masks, paths, counts, after, moves, at = [], [], [], [], [], 0
    for r, n in zip(st["rows"], st["keys"]):
        up, tok, tgt = (x[at:at + r] for x in (parents, tokens, target))
        masks.append(up)
        path = _walk(up, [p >= 0 and tok[i] == tgt[p] for i, p in enumerate(up)])[:st["most"]]
        paths.append(path + [-1] * (st["most"] - len(path)))
        counts.append(len(path))
        after.append(tgt[path[-1]])
        moves.append([[(n - r + a, n - r + b) for b, a in enumerate(path) if a != b]] * st["hkv"])
        at += r
    return [_masks(masks, st["words"]), torch.tensor(paths), torch.tensor(counts), torch.tensor(after), *_exact_moves(st, moves)]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "evict":
        return _exact_evict(st)
    if case["op"] == "verify":
        return _exact_verify(st)
    if case["op"] == "decode":
        out, got = _exact_attention(st, lambda i: torch.ones(1, st["keys"][i], dtype=torch.bool, device="cuda"))
        return [out, st["mass"].double() + got]
    rows, keys, words = st["rows"], st["keys"], st["mask"].tolist()

    def sees(i):
        at, r, n = sum(rows[:i]), rows[i], keys[i]
        m = torch.ones(r, n, dtype=torch.bool)
        for t in range(r):
            for j in range(r):
                m[t, n - r + j] = bool(words[at + t][j // 32] >> (j % 32) & 1)
        return m.cuda()

    return [_exact_attention(st, sees)[0]]
