"""Plain implementations of a step over trees of drafted tokens (mini_llm_amd.kernels.ops: step_maps, rotary, tree_attention,
tree_accept): whole loops on the CPU in 64 bits, from the definitions."""
import math

import torch


def step_maps(rows, n_new, lengths, pages, page_size, n_pages, tokens, max_blocks, max_new, parents=None):
    """Lists and tensors as ops.StepMaps names them."""
    words = (max_new + 63) // 64
    out = dict(cu_q=[], cached=[], ctx_len=[], token_seq=[0] * tokens, positions=[0] * tokens, slots=[-1] * tokens, block_tables=[], ancestors=[[0] * words for _ in range(tokens)])
    at = 0
    for b in range(len(n_new)):
        r = b if rows is None else rows[b]
        there = 0 <= r < len(lengths)
        n = min(max(n_new[b], 0), max_new, tokens - at) if there else 0
        cached = max(lengths[r], 0) if there else 0
        out["cu_q"].append(at)
        out["cached"].append(cached)
        out["ctx_len"].append(cached + n)
        have = min(-(-(cached + n) // page_size), max_blocks)
        out["block_tables"].append((pages[r][:have] if there else []) + [0] * (max_blocks - have))
        chains = []
        for i in range(n):
            out["token_seq"][at + i] = b
            if parents is None:
                out["positions"][at + i] = cached + i
                out["slots"][at + i] = slot(pages[r], max_blocks, page_size, n_pages, cached + i)
                continue
            p = parents[at + i]
            chains.append([i] + (chains[p] if 0 <= p < i else []))
            out["positions"][at + i] = cached + len(chains[i]) - 1
            for j in chains[i]:
                out["ancestors"][at + i][j // 64] |= 1 << (j % 64)
        at += n
    out["cu_q"].append(at)
    out["ancestors"] = [[w - 2 ** 64 if w >= 2 ** 63 else w for w in node] for node in out["ancestors"]]
    return out


def slot(pages, max_blocks, page_size, n_pages, position):
    block = position // page_size
    if position < 0 or block >= max_blocks or not 0 <= pages[block] < n_pages:
        return -1
    return pages[block] * page_size + position % page_size


def frequencies(rot_dims, base=10000.0, scaling=None):
    """Radians a position, as ops.rotary_freqs defines them."""
    out = []
    for i in range(rot_dims // 2):
        f = base ** (-2.0 * i / rot_dims)
        if scaling is not None:
            s = scaling["factor"]
            if scaling["kind"] == "linear":
                f = f / s
            elif scaling["kind"] == "base":
                f = (base * s ** (rot_dims / (rot_dims - 2.0))) ** (-2.0 * i / rot_dims)
            else:
                turns = scaling["original"] * f / (2 * math.pi)
                if scaling["kind"] == "by_turns":
                    keep = (turns - scaling["slow"]) / (scaling["fast"] - scaling["slow"])
                else:       # (a pair's number is linear in the logarithm of its turns)
                    keep = math.log(turns / scaling["slow"]) / math.log(scaling["fast"] / scaling["slow"])
                keep = min(1.0, max(0.0, keep))
                f = keep * f + (1.0 - keep) * f / s
        out.append(f)
    return torch.tensor(out, dtype=torch.float64)


def rotary(x, positions, freqs, n_heads, head_dim, interleaved, amplitude):
    T, pairs = x.shape[0], freqs.numel()
    y = x.double().view(T, n_heads, head_dim).clone()
    first = torch.arange(pairs) * 2 if interleaved else torch.arange(pairs)
    second = first + 1 if interleaved else first + pairs
    angle = positions.double()[:, None] * freqs[None, :]
    c, s = (amplitude * torch.cos(angle))[:, None, :], (amplitude * torch.sin(angle))[:, None, :]
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first] = a * c - b * s
    y[..., second] = a * s + b * c
    return y.reshape(T, -1), (abs(a) + abs(b)) * amplitude, first, second


def attention(q, k, v, n_heads, n_kv_heads, head_dim, k_pages, v_pages, page_size, tables, cached, cu_q, ancestors, positions, scale, window):
    """The result, and three arrays that bounds of its error are made of: sum_j w_j |v_j|, the largest |v_j| seen and the largest
    sum_e |q_e k_e| * scale of a seen key. Rows of no sequence: NaN. Nothing that is not seen is read."""
    T, n_pages = q.shape[0], k_pages.shape[0] // page_size
    out, spread, top, mass = (torch.full((T, n_heads, head_dim), math.nan, dtype=torch.float64) for _ in range(4))
    q, k, v = (t.double().view(T, -1, head_dim) for t in (q, k, v))
    for b in range(len(cached)):
        first, last = cu_q[b], cu_q[b + 1]
        for t in range(first, last):
            low = positions[t] - window + 1 if window else -2 ** 31
            rows = [tables[b][j // page_size] * page_size + j % page_size for j in range(max(0, low), cached[b])
                    if j // page_size < len(tables[b]) and 0 <= tables[b][j // page_size] < n_pages]
            nodes = [first + j for j in range(last - first) if ancestors[t][j // 64] >> (j % 64) & 1 and (not window or positions[first + j] >= low)]
            keys = torch.cat([k_pages[rows].double().view(-1, n_kv_heads, head_dim), k[nodes]])
            values = torch.cat([v_pages[rows].double().view(-1, n_kv_heads, head_dim), v[nodes]])
            if keys.shape[0] == 0:
                out[t], spread[t], top[t], mass[t] = 0.0, 0.0, 0.0, 0.0
                continue
            for h in range(n_heads):
                kh, vh = keys[:, h // (n_heads // n_kv_heads)], values[:, h // (n_heads // n_kv_heads)]
                w = torch.softmax((kh * q[t, h]).sum(1) * scale, 0)
                out[t, h], spread[t, h], top[t, h] = w @ vh, w @ vh.abs(), vh.abs().amax(0)
                mass[t, h] = ((kh * q[t, h]).abs().sum(1) * abs(scale)).max()
    return [x.view(T, -1) for x in (out, spread, top, mass)]


def accept(choices, ids, parents, cu_q, cached, tables, page_size, n_pages, max_new):
    T = len(choices)
    kept, paths, following, slots = [], [], [], [-1] * T
    for b in range(len(cached)):
        first, n = cu_q[b], min(cu_q[b + 1] - cu_q[b], max_new)
        path = [0] if n > 0 else []
        while path:
            named = [i for i in range(path[-1] + 1, n) if parents[first + i] == path[-1] and ids[first + i] == choices[first + path[-1]]]
            if not named:
                break
            path.append(named[0])
        for place, i in enumerate(path):
            slots[first + i] = slot(tables[b], len(tables[b]), page_size, n_pages, cached[b] + place)
        kept.append(len(path))
        paths.append([first + i for i in path] + [-1] * (max_new - len(path)))
        following.append(choices[first + path[-1]] if path else -1)
    return kept, paths, following, slots
