"""What checking a tree of drafted tokens over the paged cache is measured on, operator by operator.

A program that drafts several tokens a request and has the model check them in one step calls, in this order:

* ``step_maps``: from request lengths, page lists and the tokens each sequence brings, on the device: block tables, positions,
  page rows of the tokens and, for trees, every node's depth and the set of nodes above it (64 nodes a word);
* ``rotary``: queries and keys turned by those positions;
* ``tree_attention``: every node sees its request's cached positions (in the pages) and the nodes above it (in the step's rows);
* ``tree_accept``: from the token the model chose at every node, the path of drafted tokens that stands, where their keys and
  values go, the next token and the new lengths.

Lengths, tree shapes and page numbers follow from a case's own numbers and the seed; the work of a case does not depend on the seed.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
VOCAB = 50257
MOST_NODES = 256                 # of one request's tree


# -- the cases ----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # eight users of a small model answer token by token: one node each, the form without drafts
        dict(name="attention_single_tokens_bf16", op="attention", dtype="bfloat16", seqs=8, nodes=1, cached=1000, heads=12, kv_heads=12, dim=64, page=16, window=0),
        # one user of the same model, 26 drafted nodes: latency counts
        dict(name="attention_one_user_bf16", op="attention", dtype="bfloat16", seqs=1, nodes=26, cached=900, heads=12, kv_heads=12, dim=64, page=16, window=0),
        # a long text, one user, a wide tree: few heads and a long axis
        dict(name="attention_long_text_bf16", op="attention", dtype="bfloat16", seqs=1, nodes=64, cached=31000, heads=25, kv_heads=25, dim=64, page=16, window=0),
        # a full server: 32 requests of ragged lengths, four query heads to a key head
        dict(name="attention_shared_heads_bf16", op="attention", dtype="bfloat16", seqs=32, nodes=64, cached=8192, heads=32, kv_heads=8, dim=128, page=64, window=0),
        # odd sizes all over: pages of 24, heads of 80, a window whose border lies inside pages
        dict(name="attention_window_odd_bf16", op="attention", dtype="bfloat16", seqs=3, nodes=37, cached=4100, heads=10, kv_heads=5, dim=80, page=24, window=1000),
        # eight users on the true 32-bit path
        dict(name="attention_batch_f32", op="attention", dtype="float32", seqs=8, nodes=24, cached=768, heads=12, kv_heads=12, dim=64, page=16, window=0),
        # the step's arrays for eight trees; and for a full server of long texts, whose tables are most of the work
        dict(name="maps_few", op="maps", seqs=8, nodes=16, cached=900, page=16, tree=True),
        dict(name="maps_many_long", op="maps", seqs=256, nodes=128, cached=100000, page=16, tree=True),
        # eight trees' queries and keys with part of each head turned as neighbouring pairs; and a prompt at positions far beyond the
        # trained ones, halves turned, frequencies slowed
        dict(name="rotary_part_pairs_f32", op="rotary", dtype="float32", tokens=200, heads=18, dim=96, rot=32, pairs="neighbours", far=4000, factor=1.0),
        dict(name="rotary_long_halves_bf16", op="rotary", dtype="bfloat16", tokens=8192, heads=40, dim=128, rot=128, pairs="halves", far=1000000, factor=8.0),
        # one user's 26 nodes; and 512 requests' trees of up to 200 nodes
        dict(name="accept_one_user", op="accept", seqs=1, nodes=26, cached=900, page=16),
        dict(name="accept_many", op="accept", seqs=512, nodes=200, cached=8192, page=16),
    ]


def draw(rng):
    def spread(low, high):      # even over the logarithm
        return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))

    op = rng.choice(["attention"] * 3 + ["maps", "rotary", "accept"])
    if op == "attention":
        most = work(listed()[3])
        while True:
            kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 12, 25])
            case = dict(op=op, dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), seqs=spread(1, 48), nodes=spread(1, MOST_NODES), cached=spread(1, 40000),
                        heads=kv_heads * rng.choice([1, 1, 2, 4, 7]), kv_heads=kv_heads, dim=rng.choice([16, 32, 64, 64, 80, 96, 128, 128, 256]),
                        page=rng.choice([1, 8, 16, 16, 24, 32, 64, 256]), window=0)
            if rng.random() < 0.25:
                case["window"] = spread(8, 8192)
            w = work(case)
            # (no case costs more than the largest listed one; 32-bit products run at a sixteenth of the rate)
            if w["bytes"] <= most["bytes"] and w["flops"] * (16 if case["dtype"] == "float32" else 1) <= most["flops"]:
                return case
    if op == "maps":
        while True:
            case = dict(op=op, seqs=spread(1, 256), nodes=spread(1, 2000), cached=spread(1, 100000), page=rng.choice([1, 8, 16, 16, 24, 64, 128]), tree=False)
            if case["nodes"] <= MOST_NODES:
                case["tree"] = rng.random() < 0.7
            if work(case)["bytes"] <= work(listed()[7])["bytes"]:
                return case
    if op == "rotary":
        while True:
            dim = rng.choice([32, 64, 80, 96, 128, 256])
            case = dict(op=op, dtype=rng.choice(["bfloat16", "float32"]), tokens=spread(1, 20000), heads=spread(1, 64), dim=dim,
                        rot=2 * rng.randint(1, dim // 2) if rng.random() < 0.5 else dim, pairs=rng.choice(["halves", "neighbours"]), far=spread(10, 1000000),
                        factor=rng.choice([1.0, 2.0, 4.0, 8.0, 32.0]))
            if work(case)["bytes"] <= work(listed()[9])["bytes"]:
                return case
    return dict(op=op, seqs=spread(1, 512), nodes=spread(1, 200), cached=spread(1, 8192), page=rng.choice([1, 8, 16, 16, 24, 64]))


# -- shapes that follow from a case alone --------------------------------------------------------------------------------
def shape_rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def lengths_of(case):
    """Cached positions and nodes of every sequence: the first has the case's own numbers, the others down to half of them."""
    rng = shape_rng(case)
    cached = [case["cached"]] + [rng.randint(case["cached"] // 2, case["cached"]) for _ in range(case["seqs"] - 1)]
    nodes = [case["nodes"]] + [rng.randint((case["nodes"] + 1) // 2, case["nodes"]) for _ in range(case["seqs"] - 1)]
    return cached, nodes


def trees_of(case):
    """The parent of every node within its sequence (-1: the root), in front of its children. Chains and bushes, by sequence."""
    rng = random.Random(shape_rng(case).random())
    trees = []
    for n in lengths_of(case)[1]:
        reach = rng.choice([1, 4, 16, n])
        trees.append([-1] + [rng.randint(max(0, i - reach), i - 1) for i in range(1, n)])
    return trees


def seen_of(case):
    """Keys that all nodes see together (cached and above them, inside the window), and cached keys that any node of a sequence sees."""
    pairs = read = 0
    for cached, tree in zip(lengths_of(case)[0], trees_of(case)):
        depth, first = [], cached
        for i, p in enumerate(tree):
            depth.append(0 if p < 0 else depth[p] + 1)
            at = cached + depth[i]
            low = max(0, at - case["window"] + 1) if case["window"] else 0
            pairs += max(0, cached - low) + min(depth[i] + 1, case["window"] or depth[i] + 1)
            first = min(first, low)
        read += cached - first
    return pairs, read


def work(case):
    if case["op"] == "rotary":
        size = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * size * TYPES[case["dtype"]].itemsize + 4 * case["tokens"], "flops": 3 * case["tokens"] * case["heads"] * case["rot"]}
    cached, nodes = lengths_of(case)
    T = sum(nodes)
    if case["op"] == "attention":
        pairs, read = seen_of(case)
        rows = T * (2 * case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        return {"bytes": (rows + 2 * read * case["kv_heads"] * case["dim"]) * TYPES[case["dtype"]].itemsize + 4 * (read // case["page"]) + 12 * T,
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    if case["op"] == "maps":
        tables = sum(-(-(c + n) // case["page"]) for c, n in zip(cached, nodes)) + case["seqs"] * blocks_of(case)
        return {"bytes": 4 * tables + T * (16 + 8 * -(-case["nodes"] // 64) if case["tree"] else 12) + 24 * case["seqs"], "flops": T}
    return {"bytes": 16 * T + 4 * case["seqs"] * (5 + case["nodes"]), "flops": T}


def blocks_of(case):
    return -(-(case["cached"] + case["nodes"]) // case["page"])


# -- inputs --------------------------------------------------------------------------------------------------------------
def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(case)
    if case["op"] == "rotary":
        s["x"] = torch.randn(case["tokens"], case["heads"] * case["dim"], device=DEV, generator=g).to(TYPES[case["dtype"]])
        s["out"] = torch.empty_like(s["x"])
        # neighbouring tokens stand at neighbouring positions, as in a prompt, from somewhere up to the farthest
        start = int(torch.randint(0, max(1, case["far"] - case["tokens"]), (1,), device=DEV, generator=g))
        s["positions"] = torch.arange(start, start + case["tokens"], dtype=torch.int32, device=DEV)
        s["scaling"] = scaling_of(case)
        s["frequencies"] = frequencies(case)
        if own:
            from mini_llm_amd.kernels import ops
            s["plan"] = ops.rotary_freqs(case["rot"], 10000.0, s["scaling"], device=DEV)
        return s
    cached, nodes = lengths_of(case)
    B, T, blocks = case["seqs"], sum(nodes), blocks_of(case)
    starts = [sum(nodes[:b]) for b in range(B + 1)]
    # every request's pages, scattered over the pool; its unused places name page 0
    needed = [-(-(c + n) // case["page"]) for c, n in zip(cached, nodes)]
    n_pages = sum(needed) + 7
    order = torch.randperm(n_pages, device=DEV, generator=g).to(torch.int32)
    tables = torch.zeros(B, blocks, dtype=torch.int32, device=DEV)
    at = 0
    for b in range(B):
        tables[b, :needed[b]] = order[at:at + needed[b]]
        at += needed[b]
    parents = ints([p for tree in trees_of(case) for p in tree]) if case["op"] != "maps" or case["tree"] else None
    s.update(B=B, T=T, blocks=blocks, n_pages=n_pages, starts=starts, cached_host=cached, nodes_host=nodes, cu_q=ints(starts), cached_dev=ints(cached), tables=tables, parents=parents)
    if case["op"] == "maps":
        # the requests' own places in the program's tables are another order than the step's
        rows = torch.randperm(B, device=DEV, generator=g).to(torch.int32)
        s["rows"], s["n_new"] = rows, ints(nodes)
        s["lengths"], s["pages"] = torch.empty_like(s["cached_dev"]), torch.empty_like(tables)
        s["lengths"][rows.long()] = s["cached_dev"]
        s["pages"][rows.long()] = tables
        if own:
            from mini_llm_amd.kernels import ops
            s["maps"] = ops.StepMaps(B, T, blocks, case["nodes"], tree=case["tree"], device=DEV)
        return s
    if case["op"] == "accept":
        # drafted tokens, and at most nodes the model chooses the token of one of the node's children
        s["ids"] = torch.randint(0, VOCAB, (T,), device=DEV, generator=g, dtype=torch.int32)
        choices = torch.randint(0, VOCAB, (T,), device=DEV, generator=g, dtype=torch.int32)
        first = torch.repeat_interleave(s["cu_q"][:-1].long(), torch.tensor(nodes, device=DEV))
        child = torch.nonzero(parents >= 0).flatten()
        child = child[torch.randperm(child.numel(), device=DEV, generator=g)]
        child = child[torch.rand(child.numel(), device=DEV, generator=g) < 0.9]
        # (of a node's children the last in this order)
        last = torch.full((T,), -1, device=DEV).scatter_reduce(0, (first + parents)[child], torch.arange(child.numel(), device=DEV), "amax")
        node = torch.nonzero(last >= 0).flatten()
        choices[node] = s["ids"][child[last[node]]]
        s["choices"] = choices
        if own:
            s["kept"], s["next"], s["lengths"] = ints([0] * B), ints([0] * B), ints([0] * B)
            s["path"] = torch.empty(B, case["nodes"], dtype=torch.int32, device=DEV)
            s["slots"] = torch.empty(T, dtype=torch.int32, device=DEV)
        return s
    dtype, kv = TYPES[case["dtype"]], case["kv_heads"] * case["dim"]
    s["k_pages"], s["v_pages"] = (torch.randn(n_pages * case["page"], kv, device=DEV, generator=g).to(dtype) for _ in range(2))
    # queries, keys and values as the step's projection leaves them, side by side
    qkv = torch.randn(T, case["heads"] * case["dim"] + 2 * kv, device=DEV, generator=g).to(dtype)
    s["q"], s["k"], s["v"] = qkv[:, :-2 * kv], qkv[:, -2 * kv:-kv], qkv[:, -kv:]
    s["scale"] = case["dim"] ** -0.5
    maps = plain_maps(dict(s, rows=torch.arange(B, dtype=torch.int32, device=DEV), n_new=ints(nodes), lengths=s["cached_dev"], pages=tables, tree=True))
    s["positions"], s["ancestors"] = maps[4], maps[7]
    s["out"] = torch.empty(T, case["heads"] * case["dim"], dtype=dtype, device=DEV)
    return s


def scaling_of(case):
    """Far positions: pairs that turn more than 32 times over the 8,192 positions of training stay, those that turn less than once are
    slowed by the factor, those between by a share of it."""
    return None if case["factor"] == 1.0 else dict(kind="by_turns", factor=case["factor"], original=8192, fast=32.0, slow=1.0)


def amplitude_of(case):
    return 1.0 + 0.1 * math.log(case["factor"])


def frequencies(case):
    """Every pair's angle per position, in 64 bits."""
    f = 10000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device=DEV) / case["rot"])
    if case["factor"] != 1.0:
        share = ((8192 * f / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        f = f * (share + (1.0 - share) / case["factor"])
    return f


# -- one pass ------------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return OWN[state["op"]](state)
    return PLAIN[state["op"]](state)


def own_attention(s):
    from mini_llm_amd.kernels import ops
    return ops.tree_attention(s["q"], s["k"], s["v"], s["heads"], s["kv_heads"], s["dim"], s["k_pages"], s["v_pages"], s["page"], s["tables"], s["cached_dev"],
                              s["cu_q"], s["ancestors"], s["positions"], s["scale"], s["out"], max_new=s["nodes"], max_cached=s["cached"], window=s["window"])


def own_maps(s):
    from mini_llm_amd.kernels import ops
    m = ops.step_maps(s["maps"], s["rows"], s["n_new"], s["lengths"], s["pages"], s["page"], s["n_pages"], parents=s["parents"])
    return [m.cu_q, m.cached, m.ctx_len, m.token_seq, m.positions, m.slots, m.block_tables] + ([m.ancestors] if s["tree"] else [])


def own_rotary(s):
    from mini_llm_amd.kernels import ops
    return ops.rotary(s["x"], s["positions"], s["plan"], s["heads"], s["dim"], s["out"], interleaved=s["pairs"] == "neighbours", amplitude=amplitude_of(s))


def own_accept(s):
    from mini_llm_amd.kernels import ops
    ops.tree_accept(s["choices"], s["ids"], s["parents"], s["cu_q"], s["cached_dev"], s["tables"], s["page"], s["n_pages"], s["kept"], s["path"], s["next"],
                    s["slots"], lengths=s["lengths"])
    return [s["kept"], s["path"], s["next"], s["slots"], s["lengths"]]


OWN = {"attention": own_attention, "maps": own_maps, "rotary": own_rotary, "accept": own_accept}


# -- the plain forms -----------------------------------------------------------------------------------------------------
def plain_attention(s):
    H, G, D = s["heads"], s["heads"] // s["kv_heads"], s["dim"]
    out = torch.empty(s["T"], H * D, dtype=s["q"].dtype, device=DEV)
    for b in range(s["B"]):
        first, last, cached = s["starts"][b], s["starts"][b + 1], s["cached_host"][b]
        n, at = last - first, torch.arange(cached, device=DEV)
        rows = s["tables"][b].long()[at // s["page"]] * s["page"] + at % s["page"]
        k, v = (torch.cat([pages[rows], new[first:last]]).float().view(-1, s["kv_heads"], D).permute(1, 0, 2).contiguous()
                for pages, new in ((s["k_pages"], s["k"]), (s["v_pages"], s["v"])))
        q = s["q"][first:last].float().view(n, s["kv_heads"], G, D).permute(1, 2, 0, 3).reshape(s["kv_heads"], G * n, D)
        scores = torch.matmul(q, k.transpose(1, 2).contiguous()).view(s["kv_heads"], G, n, cached + n) * s["scale"]
        node = torch.arange(n, device=DEV)
        above = ((s["ancestors"][first:last, node // 64] >> (node % 64)) & 1) != 0
        p = s["positions"][first:last].long()
        visible = torch.cat([torch.ones(n, cached, dtype=torch.bool, device=DEV), above], 1)
        if s["window"]:
            visible = visible & (torch.cat([at, p])[None, :] > p[:, None] - s["window"])
        scores = scores.masked_fill(~visible, -math.inf)
        e = torch.exp(scores - scores.amax(-1, keepdim=True))
        o = torch.matmul(e.view(s["kv_heads"], G * n, cached + n), v) / e.sum(-1).view(s["kv_heads"], G * n, 1)
        out[first:last] = o.view(s["kv_heads"], G, n, D).permute(2, 0, 1, 3).reshape(n, H * D).to(out.dtype)
    return out


def plain_maps(s):
    rows, n_new = s["rows"].long(), s["n_new"].long()
    ends = torch.cumsum(n_new, 0)
    cu_q = torch.cat([torch.zeros_like(ends[:1]), ends])
    cached = s["lengths"][rows].long()
    ctx_len = cached + n_new
    token = torch.arange(s["T"], device=DEV)
    seq = torch.searchsorted(ends, token, right=True)
    first = cu_q[seq]
    place = torch.arange(s["blocks"], device=DEV)
    tables = torch.where(place[None, :] * s["page"] < ctx_len[:, None], s["pages"][rows], 0)
    if not s["tree"]:
        positions = cached[seq] + token - first
        slots = tables[seq, positions // s["page"]] * s["page"] + positions % s["page"]
        return [x.to(torch.int32) for x in (cu_q, cached, ctx_len, seq, positions, slots, tables)]
    # nodes above a node: its own bit and those above its parent, doubled round by round (the last row: above a root)
    local, words = token - first, -(-s["nodes"] // 64)
    above = torch.where(torch.arange(words, device=DEV)[None, :] == (local // 64)[:, None], torch.ones_like(local)[:, None] << (local % 64)[:, None], 0)
    above = torch.cat([above, torch.zeros_like(above[:1])])
    up = torch.cat([torch.where(s["parents"] >= 0, first + s["parents"], s["T"]), torch.full_like(first[:1], s["T"])])
    depth = (up < s["T"]).long()
    for _ in range(max(1, (s["nodes"] - 1).bit_length())):
        above, depth, up = above | above[up], depth + depth[up], up[up]
    positions = cached[seq] + depth[:-1]
    return [x.to(torch.int32) for x in (cu_q, cached, ctx_len, seq, positions, torch.full_like(positions, -1), tables)] + [above[:-1]]


def plain_rotary(s):
    angle = s["positions"].double()[:, None] * s["frequencies"][None, :]
    angle = angle - 2 * math.pi * torch.round(angle / (2 * math.pi))
    c, d = (torch.cos(angle) * amplitude_of(s)).float()[:, None, :], (torch.sin(angle) * amplitude_of(s)).float()[:, None, :]
    x = s["x"].float().view(s["tokens"], s["heads"], s["dim"])
    turned, rest = x[..., :s["rot"]], x[..., s["rot"]:]
    if s["pairs"] == "halves":
        a, b = turned[..., :s["rot"] // 2], turned[..., s["rot"] // 2:]
        turned = torch.cat([a * c - b * d, a * d + b * c], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * c - b * d, a * d + b * c], -1).flatten(-2)
    return torch.cat([turned, rest], -1).view(s["tokens"], -1).to(s["x"].dtype)


def plain_accept(s):
    # the child that every node's choice names (the first of equal ones), then the walk from all roots side by side
    token, T = torch.arange(s["T"], device=DEV), s["T"]
    seq = torch.searchsorted(s["cu_q"][1:].long(), token, right=True)
    up = torch.where(s["parents"] >= 0, s["cu_q"].long()[seq] + s["parents"], T)
    named = torch.where((up < T) & (s["ids"] == s["choices"][up.clamp(max=T - 1)]), up, T)
    child = torch.full((T + 1,), T, device=DEV).scatter_reduce(0, named, token, "amin")
    child[T] = T
    path, node = [], s["cu_q"][:-1].long()
    for _ in range(s["nodes"]):
        path.append(node)
        node = child[node]
    path = torch.stack(path, 1)
    kept = (path < T).sum(1)
    last = path.gather(1, kept[:, None] - 1)[:, 0]
    at = s["cached_dev"].long()[:, None] + torch.arange(s["nodes"], device=DEV)[None, :]
    row = s["tables"].long().gather(1, (at // s["page"]).clamp(max=s["blocks"] - 1)) * s["page"] + at % s["page"]
    slots = torch.full((T + 1,), -1, device=DEV).scatter(0, path.flatten(), torch.where(path < T, row, -1).flatten())[:T]
    return [x.to(torch.int32) for x in (kept, torch.where(path < T, path, -1), s["choices"][last], slots, s["cached_dev"] + kept)]


PLAIN = {"attention": plain_attention, "maps": plain_maps, "rotary": plain_rotary, "accept": plain_accept}


# -- the definitions, in 64 bits and on their own ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": exact_attention, "maps": exact_maps, "rotary": exact_rotary, "accept": exact_accept}[case["op"]](case, s)


def chains(tree):
    """Every node with the nodes above it, itself first."""
    out = []
    for i, p in enumerate(tree):
        out.append([i] + (out[p] if p >= 0 else []))
    return out


def exact_attention(case, s):
    cached, nodes = lengths_of(case)
    D, H = case["dim"], case["heads"]
    result, first = torch.zeros(sum(nodes), H * D, dtype=torch.float64, device=DEV), 0
    for b, tree in enumerate(trees_of(case)):
        n, L = nodes[b], cached[b]
        above = chains(tree)
        page_of = s["tables"][b].tolist()
        rows = torch.tensor([page_of[j // case["page"]] * case["page"] + j % case["page"] for j in range(L)], dtype=torch.long, device=DEV)
        # what is not seen, added to the scores
        bar = torch.full((n, L + n), -math.inf, dtype=torch.float64)
        for i, chain in enumerate(above):
            at = L + len(chain) - 1
            low = max(0, at - case["window"] + 1) if case["window"] else 0
            bar[i, low:L] = 0.0
            for up, j in enumerate(chain):
                if not case["window"] or up < case["window"]:
                    bar[i, L + j] = 0.0
        bar = bar.to(DEV)
        for h in range(H):
            cols = slice(h * D, (h + 1) * D)
            kc = slice(h // (H // case["kv_heads"]) * D, (h // (H // case["kv_heads"]) + 1) * D)
            keys = torch.cat([s["k_pages"][rows, kc], s["k"][first:first + n, kc]]).double()
            values = torch.cat([s["v_pages"][rows, kc], s["v"][first:first + n, kc]]).double()
            z = s["q"][first:first + n, cols].double() @ keys.t().contiguous() / math.sqrt(D) + bar
            z = (z - torch.logsumexp(z, 1, keepdim=True)).exp()
            result[first:first + n, cols] = z @ values
        first += n
    return result


def exact_maps(case, s):
    cached, nodes = lengths_of(case)
    pages, rows = s["pages"].cpu(), s["rows"].tolist()
    cu, seqs, positions, slots, bits = [0], [], [], [], []
    tables = torch.zeros(case["seqs"], blocks_of(case), dtype=torch.int32)
    trees = trees_of(case) if case["tree"] else [None] * case["seqs"]
    for b, (L, n, tree) in enumerate(zip(cached, nodes, trees)):
        have = -(-(L + n) // case["page"])
        tables[b, :have] = pages[rows[b], :have]
        table = tables[b].tolist()
        cu.append(cu[-1] + n)
        seqs += [b] * n
        if tree is None:
            positions += range(L, L + n)
            slots += [table[p // case["page"]] * case["page"] + p % case["page"] for p in range(L, L + n)]
            continue
        for chain in chains(tree):
            positions.append(L + len(chain) - 1)
            slots.append(-1)
            mask = sum(1 << j for j in chain)
            words = [(mask >> (64 * w)) & (2 ** 64 - 1) for w in range(-(-case["nodes"] // 64))]
            bits.append([w - 2 ** 64 if w >= 2 ** 63 else w for w in words])
    out = [ints(cu), ints(cached), ints([c + n for c, n in zip(cached, nodes)]), ints(seqs), ints(positions), ints(slots), tables.to(DEV)]
    return out + ([torch.tensor(bits, dtype=torch.int64, device=DEV)] if case["tree"] else [])


def exact_rotary(case, s):
    x = s["x"].double().view(case["tokens"], case["heads"], case["dim"])
    out, p = x.clone(), s["positions"].double()[:, None]
    for i in range(case["rot"] // 2):
        f = 10000.0 ** (-2.0 * i / case["rot"])
        if case["factor"] != 1.0:
            turns = 8192 * f / (2 * math.pi)
            keep = 0.0 if turns <= 1.0 else 1.0 if turns >= 32.0 else (turns - 1.0) / 31.0
            f = keep * f + (1.0 - keep) * f / case["factor"]
        first, second = (i, i + case["rot"] // 2) if case["pairs"] == "halves" else (2 * i, 2 * i + 1)
        a, b = x[..., first], x[..., second]
        c, d = amplitude_of(case) * torch.cos(p * f), amplitude_of(case) * torch.sin(p * f)
        out[..., first] = a * c - b * d
        out[..., second] = a * d + b * c
    return out.reshape(case["tokens"], -1)


def exact_accept(case, s):
    cached, nodes = lengths_of(case)
    choices, ids, tables = s["choices"].tolist(), s["ids"].tolist(), s["tables"].cpu()
    kept, paths, following, slots, lengths, first = [], [], [], [-1] * sum(nodes), [], 0
    for b, tree in enumerate(trees_of(case)):
        children = {}
        for i, p in enumerate(tree):
            children.setdefault(p, []).append(i)
        path = [0]
        while True:
            named = [c for c in children.get(path[-1], []) if ids[first + c] == choices[first + path[-1]]]
            if not named:
                break
            path.append(named[0])
        table = tables[b].tolist()
        for k, i in enumerate(path):
            at = cached[b] + k
            slots[first + i] = table[at // case["page"]] * case["page"] + at % case["page"]
        kept.append(len(path))
        paths.append([first + i for i in path] + [-1] * (case["nodes"] - len(path)))
        following.append(choices[first + path[-1]])
        lengths.append(cached[b] + len(path))
        first += nodes[b]
    return [ints(kept), ints(paths), ints(following), ints(slots), ints(lengths)]
