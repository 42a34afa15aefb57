"""Measured cases of the operators that verify drafted tokens: what a program that decodes speculatively calls per step.

A request's draft is a tree of tokens behind its cached ones: node 0 is the last token that was answered, every other
node hangs on one before it.  One step runs all nodes of all requests; a node sees the request's cached tokens and its own
ancestors.  Four operators: the attention of such a step over the paged cache, the penalties, biases and grammar masks of
every node's logits, the walk that keeps the longest drafted path that the model agrees with, and the move of the kept nodes'
keys and values to where the cache goes on.  Head layouts, vocabularies, pages and layer counts are those of the benchmark's
and the tests' models.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
LOWEST = -math.inf
#: heads, key/value heads, head size, layers
MODELS = {
    "0.5b": dict(heads=14, kv_heads=2, size=64, layers=24, vocab=151936),
    "1.5b": dict(heads=12, kv_heads=2, size=128, layers=28, vocab=151936),
    "7b": dict(heads=28, kv_heads=4, size=128, layers=28, vocab=151936),
    "c": dict(heads=6, kv_heads=2, size=48, layers=4, vocab=331),
}
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# --------------------------------------------------------------------------- the cases
def attention(model, requests, nodes, cached, dtype="bfloat16", page=16, window=0, softcap=0.0, name=None):
    case = dict(kind="attention", model=model, requests=requests, nodes=nodes, cached=cached, dtype=dtype, page=page, window=window,
                softcap=softcap)
    return dict(case, name=name) if name else case


def logits(requests, nodes, vocab, history, biases, masks, name=None):
    case = dict(kind="logits", requests=requests, nodes=nodes, vocab=vocab, history=history, biases=biases, masks=masks)
    return dict(case, name=name) if name else case


def accept(requests, nodes, vocab, name=None):
    case = dict(kind="accept", requests=requests, nodes=nodes, vocab=vocab)
    return dict(case, name=name) if name else case


def move(model, requests, nodes, kept, cached, dtype="bfloat16", page=16, name=None):
    case = dict(kind="move", model=model, requests=requests, nodes=nodes, kept=kept, cached=cached, dtype=dtype, page=page)
    return dict(case, name=name) if name else case


def listed():
    return [
        # one user of the small model with a small tree: latency is all there is
        attention("0.5b", 1, 8, 1024, name="tree-1"),
        # the benchmark's eight users at contexts of up to 4,096, trees of up to 16 nodes
        attention("1.5b", 8, 16, 4096, name="tree-8"),
        # one long document, a wider tree: the work has to be split over the keys
        attention("7b", 1, 32, 32768, name="tree-long"),
        # a full server with the widest trees
        attention("7b", 32, 64, 8192, name="tree-32"),
        # the 32-bit path, by which users check a model
        attention("0.5b", 2, 13, 700, dtype="float32", name="tree-32bit"),
        # one user: one row after a short answer
        logits(1, 1, 151936, 300, 8, False, name="logits-1"),
        # 64 users who each take one token, long histories, no grammar
        logits(64, 1, 151936, 4096, 0, False, name="logits-64"),
        # every node of eight users' trees under a grammar, with biases
        logits(8, 24, 151936, 2048, 300, True, name="logits-nodes"),
        # the walk through one small tree
        accept(1, 8, 151936, name="accept-1"),
        # the walk through a full server's trees
        accept(64, 64, 151936, name="accept-64"),
        # kept keys and values of one user in all layers of the small model
        move("0.5b", 1, 8, 3, 1024, name="move-1"),
        # the same for a full server
        move("1.5b", 32, 64, 6, 1000, name="move-32"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "logits", "logits", "accept", "move"])
    if kind == "attention":
        model = rng.choice(["0.5b", "0.5b", "1.5b", "1.5b", "7b", "7b", "c"])
        dtype = "float32" if rng.random() < 0.2 else "bfloat16"
        nodes, requests = _log(rng, 1, 64), _log(rng, 1, 32)
        # at most a quarter of the largest listed case's products, far less where they are 32-bit ones
        most = 28 * 128 * 64 * 32 * 8192 // (200 if dtype == "float32" or model == "c" else 4)
        sizes = MODELS[model]
        cached = _log(rng, 1, max(1, min(32768, most // (sizes["heads"] * sizes["size"] * nodes * requests))))
        return attention(model, requests, nodes, cached, dtype=dtype, page=rng.choice([16, 16, 16, 32, 64, 8, 5]),
                         window=rng.choice([0, 0, 0, _log(rng, 1, 4096)]), softcap=rng.choice([0.0, 0.0, 0.0, 30.0]))
    if kind == "logits":
        vocab = rng.choice([151936, 151936, 32003, 3001, 331])
        nodes, requests = _log(rng, 1, 32), _log(rng, 1, 64)
        requests = max(1, min(requests, 192 // nodes))
        return logits(requests, nodes, vocab, _log(rng, 1, 16384), rng.choice([0, 0, 1, _log(rng, 1, 300)]), rng.random() < 0.5)
    if kind == "accept":
        return accept(_log(rng, 1, 256), _log(rng, 1, 64), rng.choice([151936, 3001, 331]))
    nodes = _log(rng, 2, 64)
    return move(rng.choice(["0.5b", "1.5b", "7b", "c"]), _log(rng, 1, 32), nodes, rng.randint(1, max(1, nodes // 2)), _log(rng, 1, 2048),
                dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), page=rng.choice([16, 16, 32, 5]))


def _nodes(case):
    """Nodes of every request: ragged, the first has the most."""
    n = case["nodes"]
    return [max(1, n - (5 * r) % (n // 2 + 1)) for r in range(case["requests"])]


def _cached(case):
    c = case["cached"]
    return [c - (977 * r) % (c // 2 + 1) for r in range(case["requests"])]


def _kept(case):
    """Nodes that a request keeps, the root among them; the others stand behind the places they move to."""
    return [min(max(1, case["kept"] - r % 3), 1 + max(0, n - case["kept"])) for r, n in enumerate(_nodes(case))]


def work(case):
    kind = case["kind"]
    nodes = _nodes(case)
    rows = sum(nodes)
    if kind == "logits":
        bytes_ = rows * case["vocab"] * 8 + 4 * sum(_history(case)) + 8 * case["requests"] * case["biases"]
        return {"bytes": bytes_ + (rows * 4 * -(-case["vocab"] // 32) if case["masks"] else 0), "flops": 4 * rows * case["vocab"]}
    if kind == "accept":
        return {"bytes": 12 * rows + 8 * case["requests"] * (case["nodes"] + 2), "flops": 2 * rows}
    sizes, item = MODELS[case["model"]], 4 if case["dtype"] == "float32" else 2
    row = sizes["kv_heads"] * sizes["size"] * item
    if kind == "move":
        moved = sum(k - 1 for k in _kept(case))
        return {"bytes": sizes["layers"] * 2 * 2 * moved * row, "flops": 0}
    window = case["window"] or case["cached"] + case["nodes"]
    cached = [min(c, window) for c in _cached(case)]
    return {"bytes": 2 * rows * sizes["heads"] * sizes["size"] * item + 2 * (sum(cached) + rows) * row,
            "flops": 4 * sizes["heads"] * sizes["size"] * sum(n * (c + 1) for n, c in zip(nodes, cached))}


def _history(case):
    h = case["history"]
    return [h - (613 * r) % (h // 2 + 1) for r in range(case["requests"])]


# --------------------------------------------------------------------------- what a program has in hand
def _tree(rng, nodes):
    """Parents of one tree, mostly short branches off a main line, and every node's ancestors as bits."""
    parents, bits = [-1], [1]
    for k in range(1, nodes):
        parents.append(k - 1 - int(rng.random() ** 2 * min(k, 6)))
        bits.append(bits[parents[k]] | 1 << k)
    return parents, bits


def _signed(bits, words):
    out = []
    for w in range(words):
        v = bits >> (64 * w) & (1 << 64) - 1
        out.append(v - (1 << 64) if v >> 63 else v)
    return out


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).to(DEVICE)


def _starts(lengths):
    return [sum(lengths[:r]) for r in range(len(lengths) + 1)]


def _trees(case, rng):
    nodes = _nodes(case)
    parents, mask, depth = [], [], []
    words = -(-case["nodes"] // 64)
    for n in nodes:
        up, bits = _tree(rng, n)
        parents += up
        mask += [_signed(b, words) for b in bits]
        depth += [bin(b).count("1") - 1 for b in bits]
    return nodes, parents, mask, depth


def _pages(case, lengths, generator):
    """A block table over pages in no order, as a long-running server has them, and how many pages there are."""
    each = [-(-n // case["page"]) for n in lengths]
    order = torch.randperm(sum(each), generator=generator).tolist()
    width, table, at = max(each), [], 0
    for n in each:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return _ints(table), sum(each)


def prepare(case, seed):
    rng = random.Random(seed)
    host = torch.Generator().manual_seed(seed)
    device = torch.Generator(DEVICE).manual_seed(seed)
    state = {"case": case, "status": torch.zeros(1, dtype=torch.int32, device=DEVICE)}
    return {"attention": _prepare_attention, "logits": _prepare_logits, "accept": _prepare_accept,
            "move": _prepare_move}[case["kind"]](case, state, rng, host, device)


def _prepare_attention(case, state, rng, host, device):
    sizes, dtype = MODELS[case["model"]], TYPES[case["dtype"]]
    nodes, _, mask, depth = _trees(case, rng)
    cached, rows = _cached(case), sum(nodes)
    table, pages = _pages(case, [c + n for c, n in zip(cached, nodes)], host)
    shape = (pages, sizes["kv_heads"], case["page"], sizes["size"])
    state["k"] = torch.randn(shape, generator=device, device=DEVICE, dtype=dtype)
    state["v"] = torch.randn(shape, generator=device, device=DEVICE, dtype=dtype)
    state["q"] = torch.randn((rows, sizes["heads"], sizes["size"]), generator=device, device=DEVICE, dtype=dtype) * 1.5
    state["out"] = torch.empty_like(state["q"])
    state["table"], state["q_start"], state["cached"] = table, _ints(_starts(nodes)), _ints(cached)
    state["mask"] = _ints(mask, torch.int64)
    first = [c for c, n in zip(cached, nodes) for _ in range(n)]
    state["positions"] = _ints([c + d for c, d in zip(first, depth)])
    state["scale"] = sizes["size"] ** -0.5
    return state


def _prepare_logits(case, state, rng, host, device):
    nodes, _, mask, _ = _trees(case, rng)
    rows, vocab, requests = sum(nodes), case["vocab"], case["requests"]
    lengths = _history(case)

    def tokens(shape):      # few tokens often, most of them never
        return (torch.rand(shape, generator=device, device=DEVICE) ** 4 * vocab).to(torch.int32).clamp_(max=vocab - 1)

    state["logits"] = torch.randn((rows, vocab), generator=device, device=DEVICE) * 4
    state["out"] = torch.empty_like(state["logits"])
    state["row_start"] = _ints(_starts(nodes))
    state["history"] = tokens((requests, case["history"]))
    state["history_lens"] = _ints(lengths)
    state["prompt_lens"] = _ints([int(rng.random() * n) for n in lengths])
    state["repetition"] = _ints([rng.choice([1.0, 1.1, 1.3]) for _ in nodes], torch.float32)
    state["presence"] = _ints([rng.choice([0.0, 0.5]) for _ in nodes], torch.float32)
    state["frequency"] = _ints([rng.choice([0.0, 0.2, -0.1]) for _ in nodes], torch.float32)
    state["tokens"] = state["mask"] = state["bias_ids"] = state["bias"] = state["allowed"] = None
    if case["nodes"] > 1:
        state["tokens"], state["mask"] = tokens((rows,)), _ints(mask, torch.int64)
    if case["biases"]:
        count = min(case["biases"], vocab)
        ids = [rng.sample(range(vocab), count - r % (count // 2 + 1)) for r in range(requests)]
        state["bias_ids"] = _ints([i + [-1] * (count - len(i)) for i in ids])
        state["bias"] = torch.randn((requests, count), generator=device, device=DEVICE) * 3
    if case["masks"]:
        state["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), generator=device, device=DEVICE).to(torch.int32)
    return state


def _prepare_accept(case, state, rng, host, device):
    nodes, parents, mask, _ = _trees(case, rng)
    starts, rows = _starts(nodes), sum(nodes)
    tokens = [rng.randrange(case["vocab"]) for _ in range(rows)]
    targets = [rng.randrange(case["vocab"]) for _ in range(rows)]
    for first, n in zip(starts, nodes):     # three of four nodes with a child agree with one of their children
        for k in range(1, n):
            if rng.random() < 0.75:
                targets[first + parents[first + k]] = tokens[first + k]
    state["q_start"], state["parents"], state["mask"] = _ints(starts), _ints(parents), _ints(mask, torch.int64)
    state["tokens"], state["targets"] = _ints(tokens), _ints(targets)
    shape = (len(nodes), case["nodes"])
    state["path"] = torch.empty(shape, dtype=torch.int32, device=DEVICE)
    state["answer"] = torch.empty(shape, dtype=torch.int32, device=DEVICE)
    state["counts"] = torch.empty(len(nodes), dtype=torch.int32, device=DEVICE)
    return state


def _prepare_move(case, state, rng, host, device):
    sizes = MODELS[case["model"]]
    nodes, cached, kept = _nodes(case), _cached(case), _kept(case)
    table, pages = _pages(case, [c + n for c, n in zip(cached, nodes)], host)
    shape = (sizes["layers"], 2, pages, sizes["kv_heads"], case["page"], sizes["size"])
    state["cache"] = torch.randn(shape, generator=device, device=DEVICE, dtype=TYPES[case["dtype"]])
    state["layers"] = list(state["cache"].flatten(0, 1).unbind(0))
    state["plan"] = None
    paths = [[0] + sorted(rng.sample(range(case["kept"], n), k - 1)) for n, k in zip(nodes, kept)]
    state["path"] = _ints([p + [-1] * (case["kept"] - len(p)) for p in paths])
    state["counts"], state["cached"], state["table"] = _ints(kept), _ints(cached), table
    return state


# --------------------------------------------------------------------------- the operators
def run(state):
    return {"attention": _attention, "logits": _logits, "accept": _accept, "move": _move}[state["case"]["kind"]](state)


def _rows(starts, most):
    """``[requests, most]``: every request's rows, and which of them it has."""
    place = torch.arange(most, device=DEVICE)
    rows, live = starts[:-1, None] + place, place < (starts[1:] - starts[:-1])[:, None]
    return torch.where(live, rows, 0), live


def _bits(mask, count):
    """``[rows, count]``: the bits of words as truth values."""
    place = torch.arange(count, device=DEVICE)
    return (mask[:, place // 64] >> place % 64 & 1).bool()


def _attention(state):
    case = state["case"]
    if own:
        from einf_b200 import ops

        ops.tree_attention(state["q"], state["k"], state["v"], state["table"], state["q_start"], state["cached"], state["mask"],
                           state["out"], state["scale"], state["status"], positions=state["positions"], window=case["window"] or None,
                           softcap=case["softcap"] or None, max_nodes=case["nodes"], max_cached=case["cached"])
        return state["out"]
    q, page = state["q"].float(), case["page"]
    heads, kv_heads, size = q.shape[1], state["k"].shape[1], q.shape[2]
    most, length = case["nodes"], case["cached"] + case["nodes"]
    rows, live = _rows(state["q_start"].long(), most)
    cached = state["cached"].long()
    key = torch.arange(min(length, state["table"].shape[1] * page), device=DEVICE)
    pages = state["table"].long()[:, key // page].clamp(min=0)
    k = state["k"][pages, :, key % page].float()                            # [requests, keys, kv heads, size]
    v = state["v"][pages, :, key % page].float()
    node = key - cached[:, None]                                            # which of the request's nodes a key is
    seen = _bits(state["mask"], most)[rows]                                 # [requests, nodes, nodes]
    inside = (node >= 0) & (node < (state["q_start"][1:] - state["q_start"][:-1])[:, None])
    node = node.clamp(0, most - 1)
    visible = (key < cached[:, None])[:, None] | (seen.gather(2, node[:, None].expand(-1, most, -1)) & inside[:, None])
    if case["window"]:
        positions = state["positions"].long()[rows]
        place = torch.where(key < cached[:, None], key, positions.gather(1, node))
        visible &= positions[:, :, None] - place[:, None] < case["window"]
    groups = heads // kv_heads
    grouped = q[rows].view(-1, most, kv_heads, groups, size).permute(0, 2, 1, 3, 4).reshape(-1, kv_heads, most * groups, size)
    scores = grouped @ k.permute(0, 2, 3, 1) * state["scale"]
    if case["softcap"]:
        scores = case["softcap"] * torch.tanh(scores / case["softcap"])
    scores = scores.view(-1, kv_heads, most, groups, key.shape[0]).masked_fill(~visible[:, None, :, None], LOWEST)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == LOWEST, 0.0, top))
    mixed = e.flatten(2, 3) @ v.transpose(1, 2) / e.sum(-1, keepdim=True).flatten(2, 3).clamp(min=1e-30)
    mixed = mixed.view(-1, kv_heads, most, groups, size).permute(0, 2, 1, 3, 4).reshape(-1, most, heads, size)
    return mixed[live].to(state["q"].dtype)


def _logits(state):
    case = state["case"]
    if own:
        from einf_b200 import ops

        ops.shape_logits(state["logits"], state["out"], state["row_start"], state["status"], history=state["history"],
                         history_lens=state["history_lens"], prompt_lens=state["prompt_lens"], repetition=state["repetition"],
                         presence=state["presence"], frequency=state["frequency"], node_tokens=state["tokens"],
                         tree_mask=state["mask"], bias_ids=state["bias_ids"], bias=state["bias"], allowed=state["allowed"])
        return state["out"]
    values, vocab, starts = state["logits"], case["vocab"], state["row_start"].long()
    request = torch.searchsorted(starts, torch.arange(values.shape[0], device=DEVICE), right=True) - 1
    place = torch.arange(state["history"].shape[1], device=DEVICE)
    there, tokens = place < state["history_lens"][:, None], state["history"].long()
    answered = there & (place >= state["prompt_lens"][:, None])
    empty = torch.zeros((case["requests"], vocab), device=DEVICE)
    prompt = empty.scatter_add(1, tokens, (there & ~answered).float())[request] > 0
    count = empty.scatter_add(1, tokens, answered.float())[request]
    if state["tokens"] is not None:
        rows, live = _rows(starts, case["nodes"])
        on_path = _bits(state["mask"], case["nodes"]) & live[request]
        count = count.scatter_add(1, state["tokens"].long()[rows][request], on_path.float())
    factor = state["repetition"][request, None]
    values = torch.where(prompt | (count > 0), torch.where(values > 0, values / factor, values * factor), values)
    values = values - (state["frequency"][request, None] * count + state["presence"][request, None] * (count > 0))
    if state["bias"] is not None:
        ids, known = state["bias_ids"].long().clamp(min=0), state["bias_ids"] >= 0
        values = values + empty.scatter_add(1, ids, torch.where(known, state["bias"], 0.0))[request]
    if state["allowed"] is not None:
        token = torch.arange(vocab, device=DEVICE)
        values = torch.where((state["allowed"][:, token // 32] >> token % 32 & 1).bool(), values, LOWEST)
    return values


def _accept(state):
    case = state["case"]
    if own:
        from einf_b200 import ops

        ops.accept_drafts(state["tokens"], state["targets"], state["parents"], state["q_start"], state["path"], state["answer"],
                          state["counts"])
        return state["path"], state["answer"], state["counts"]
    most = case["nodes"]
    rows, live = _rows(state["q_start"].long(), most)
    up = state["parents"].long()[rows]
    agreed = live & (state["tokens"][rows] == state["targets"][rows].gather(1, up.clamp(min=0))) & (up >= 0)
    place = torch.arange(most, device=DEVICE)
    # of siblings that agree the first is kept
    beaten = (agreed[:, None] & (up[:, None] == up[:, :, None]) & (place[None, :] < place[:, None])).any(2)
    kept = (agreed & ~beaten) | (live & (place == 0))
    ancestors = _bits(state["mask"], most)[rows]
    on_path = live & (~ancestors | kept[:, None]).all(2)
    order = torch.where(on_path, on_path.cumsum(1) - 1, most)
    empty = torch.full((rows.shape[0], most + 1), -1, dtype=torch.int32, device=DEVICE)
    path = empty.scatter(1, order, place.int().expand_as(order))[:, :most]
    answer = empty.scatter(1, order, state["targets"][rows])[:, :most]
    return path, answer, on_path.sum(1, dtype=torch.int32)


def _move(state):
    case = state["case"]
    if own:
        from einf_b200 import ops

        if state["plan"] is None:       # what a program makes once of its cache
            state["plan"] = ops.CacheRows(state["layers"])
        ops.move_accepted(state["plan"], state["table"], state["cached"], state["path"], state["counts"], state["status"])
        return state["cache"]
    page, cache = case["page"], state["cache"]
    step = torch.arange(state["path"].shape[1], device=DEVICE)
    live = step < state["counts"][:, None]
    cached = state["cached"].long()[:, None]
    to, start = torch.where(live, cached + step, cached), torch.where(live, cached + state["path"], cached)
    table = state["table"].long()
    rows = cache[:, :, table.gather(1, start // page), :, start % page]
    cache[:, :, table.gather(1, to // page), :, to % page] = rows
    return cache


# --------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    return {"attention": _exact_attention, "logits": _exact_logits, "accept": _exact_accept,
            "move": _exact_move}[case["kind"]](prepare(case, seed))


def _exact_attention(state):
    """Request by request, key/value head by key/value head, over the keys in their order."""
    case, page = state["case"], state["case"]["page"]
    q = state["q"].double()
    heads, kv_heads = q.shape[1], state["k"].shape[1]
    starts, cached, out = state["q_start"].tolist(), state["cached"].tolist(), torch.zeros_like(q)
    bits = np.array(state["mask"].cpu().numpy()).view(np.uint64)
    positions = state["positions"].cpu().numpy()
    for r, c in enumerate(cached):
        a, b = starts[r], starts[r + 1]
        n = b - a
        slots = torch.cat([torch.arange(int(p) * page, int(p) * page + page) for p in state["table"][r].tolist() if p >= 0])[:c + n].to(DEVICE)
        see = np.ones((n, c + n), dtype=bool)
        for k in range(n):
            see[:, c + k] = (bits[a:b, k // 64] >> np.uint64(k % 64)) & np.uint64(1) == 1
        if case["window"]:
            at = np.concatenate([np.arange(c), positions[a:b]])
            see &= positions[a:b, None] - at[None] < case["window"]
        see = torch.from_numpy(see).to(DEVICE)
        for g in range(kv_heads):
            k = state["k"][:, g].reshape(-1, q.shape[2])[slots].double()
            v = state["v"][:, g].reshape(-1, q.shape[2])[slots].double()
            for h in range(g * heads // kv_heads, (g + 1) * heads // kv_heads):
                s = torch.einsum("nd,ld->nl", q[a:b, h], k) * state["scale"]
                if case["softcap"]:
                    s = torch.tanh(s / case["softcap"]) * case["softcap"]
                p = torch.softmax(torch.where(see, s, torch.tensor(LOWEST, dtype=s.dtype, device=DEVICE)), 1)
                out[a:b, h] = torch.einsum("nl,ld->nd", torch.nan_to_num(p), v)
    return out


def _exact_logits(state):
    """Row by row, with the counts of every row's tokens kept by the host."""
    case, vocab = state["case"], state["case"]["vocab"]
    starts, lens, prompts = state["row_start"].tolist(), state["history_lens"].tolist(), state["prompt_lens"].tolist()
    out = torch.empty(state["logits"].shape, dtype=torch.float64, device=DEVICE)
    for r in range(case["requests"]):
        history = state["history"][r].cpu().numpy()
        seen = np.bincount(history[:lens[r]], minlength=vocab) > 0
        base = np.bincount(history[prompts[r]:lens[r]], minlength=vocab).astype(np.float64)
        rep, pres, freq = (float(state[name][r]) for name in ("repetition", "presence", "frequency"))
        for row in range(starts[r], starts[r + 1]):
            count = base.copy()
            if state["tokens"] is not None:
                words = [w % (1 << 64) for w in state["mask"][row].tolist()]
                for k in range(starts[r + 1] - starts[r]):
                    if words[k // 64] >> k % 64 & 1:
                        count[int(state["tokens"][starts[r] + k])] += 1
            x = state["logits"][row].double().cpu().numpy().copy()
            hit = seen | (count > 0)
            x[hit] = np.where(x[hit] > 0, x[hit] / rep, x[hit] * rep)
            x -= freq * count + pres * (count > 0)
            if state["bias"] is not None:
                for i, b in zip(state["bias_ids"][r].tolist(), state["bias"][r].tolist()):
                    if i >= 0:
                        x[i] += b
            if state["allowed"] is not None:
                packed = state["allowed"][row].cpu().numpy().astype("<i4").view(np.uint8)
                x[np.unpackbits(packed, bitorder="little")[:vocab] == 0] = LOWEST
            out[row] = torch.from_numpy(x)
    return out


def _exact_accept(state):
    """The walk from the root, node by node."""
    starts, tokens = state["q_start"].tolist(), state["tokens"].tolist()
    targets, parents, most = state["targets"].tolist(), state["parents"].tolist(), state["case"]["nodes"]
    path, answer, counts = [], [], []
    for a, b in zip(starts, starts[1:]):
        walk = [0]
        while len(walk) < most:
            here = walk[-1]
            after = [k for k in range(here + 1, b - a) if parents[a + k] == here and tokens[a + k] == targets[a + here]]
            if not after:
                break
            walk.append(after[0])
        path.append(walk + [-1] * (most - len(walk)))
        answer.append([targets[a + k] for k in walk] + [-1] * (most - len(walk)))
        counts.append(len(walk))
    return _ints(path), _ints(answer), _ints(counts)


def _exact_move(state):
    """Row by row: what stood there before any row was moved."""
    page, before = state["case"]["page"], state["cache"]
    after = before.double()
    for r, (c, count) in enumerate(zip(state["cached"].tolist(), state["counts"].tolist())):
        table, path = state["table"][r].tolist(), state["path"][r].tolist()
        for i in range(count):
            a, b = c + path[i], c + i
            after[:, :, table[b // page], :, b % page] = before[:, :, table[a // page], :, a % page].double()
    return after
