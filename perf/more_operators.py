"""A step on drafted tokens, as cases for timing: several tokens per sequence, proposed by a cheaper model, go through the
model at once, the target's probabilities decide which of them stand, and the cache keeps those.

``op`` of a case is one public entry point:

* ``tree``: attention of a tree of drafted tokens (node 0 is the last token that stands, every other node has an earlier
  one as its parent) over a cache that holds the sequence's rows and, behind them, the nodes' own: a node sees the
  sequence, its ancestors and itself. On contiguous buffers or on pages, with a mask over a padded batch or without one;
* ``verify``: which drafted tokens the target's probabilities accept, from given random numbers, and the token that
  follows them. A chain of tokens drawn from the draft's probabilities, or a tree of candidates without any;
* ``commit``: the accepted nodes' rows of every layer's cache moved to their places behind the sequence, and the lengths
  after it.

Heads, head dims and the vocabulary are those of the Qwen2-0.5B shape that the model builders and the benchmark use (14
query heads, 2 KV heads of 64, 24 layers, vocabulary 151936) and of the tests, or generic ones.

Plain forms compare and sum probabilities in 64 bits: a random number next to a border is lost in 32.
"""

import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
VOCAB, LAYERS = 151936, 24


def listed():
    return [
        # One conversation, a small tree: the latency of a call.
        {"name": "tree, one sequence", "op": "tree", "batch": 1, "tokens": 8, "q_heads": 14, "kv_heads": 2,
         "head_dim": 64, "low": 600, "high": 600, "page": 0, "mask": "none", "dtype": "bf16"},
        # An ordinary serving batch.
        {"name": "tree, batch of 8", "op": "tree", "batch": 8, "tokens": 16, "q_heads": 14, "kv_heads": 2,
         "head_dim": 64, "low": 900, "high": 2000, "page": 0, "mask": "none", "dtype": "bf16"},
        # The benchmark's decode batch and lengths: bound by the cache's bytes.
        {"name": "tree, long caches", "op": "tree", "batch": 32, "tokens": 16, "q_heads": 14, "kv_heads": 2,
         "head_dim": 64, "low": 4096, "high": 8192, "page": 0, "mask": "none", "dtype": "bf16"},
        # The widest trees: bound by the products and the exponentials.
        {"name": "tree, 64 nodes", "op": "tree", "batch": 16, "tokens": 64, "q_heads": 14, "kv_heads": 2,
         "head_dim": 64, "low": 2000, "high": 4096, "page": 0, "mask": "none", "dtype": "bf16"},
        # Sequences of all lengths, one of them empty, in a shared pool of pages.
        {"name": "tree, pages", "op": "tree", "batch": 16, "tokens": 7, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "low": 0, "high": 4000, "page": 64, "mask": "none", "dtype": "fp16"},
        # A padded batch in fp32.
        {"name": "tree, padded fp32", "op": "tree", "batch": 4, "tokens": 13, "q_heads": 4, "kv_heads": 2,
         "head_dim": 64, "low": 301, "high": 1001, "page": 0, "mask": "lowest", "dtype": "fp32"},
        # Four drafted tokens of one conversation.
        {"name": "verify, one chain", "op": "verify", "batch": 1, "tokens": 5, "vocab": VOCAB, "draft": True,
         "dtype": "fp32"},
        # Eight drafted tokens in each sequence of a large batch.
        {"name": "verify, 32 chains", "op": "verify", "batch": 32, "tokens": 9, "vocab": VOCAB, "draft": True,
         "dtype": "fp32"},
        # Trees of candidates that come without probabilities.
        {"name": "verify, 8 trees", "op": "verify", "batch": 8, "tokens": 64, "vocab": VOCAB, "draft": False,
         "dtype": "fp32"},
        # The cache of one conversation, every layer.
        {"name": "commit, one sequence", "op": "commit", "batch": 1, "tokens": 8, "kept": 4, "kv_heads": 2,
         "head_dim": 64, "capacity": 2048, "page": 0, "dtype": "bf16"},
        # The pages of a large batch, every layer.
        {"name": "commit, pages", "op": "commit", "batch": 32, "tokens": 64, "kept": 12, "kv_heads": 2, "head_dim": 64,
         "capacity": 1024, "page": 64, "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""

    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "verify", "verify", "commit"])
    if op == "verify":
        tokens, vocab = _spread(rng, 1, 64), rng.choice([VOCAB, VOCAB, _spread(rng, 32, 200000)])
        # At most the largest listed tensors of probabilities.
        batch = _spread(rng, 1, min(32, max(1, 512 * VOCAB // (tokens * vocab))))
        return {"op": op, "batch": batch, "tokens": tokens, "vocab": vocab, "draft": rng.random() < 0.5,
                "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"])}
    if op == "commit":
        tokens = _spread(rng, 2, 64)
        page = rng.choice([0, 0, 16, 64])
        return {"op": op, "batch": _spread(rng, 1, 32), "tokens": tokens, "kept": rng.randint(1, min(12, tokens)),
                "kv_heads": rng.choice([1, 2, 2, 4]), "head_dim": rng.choice([64, 64, 80]),
                "capacity": 64 * rng.randint(2, 8), "page": page, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    q_heads, kv_heads, head_dim = rng.choice([(14, 2, 64), (14, 2, 64), (4, 2, 64), (4, 2, 128), (32, 8, 128),
                                              (8, 8, 64), (6, 2, 80), (5, 1, 72), (12, 1, 256), (9, 3, 33)])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    batch, tokens = _spread(rng, 1, 32), _spread(rng, 1, 64)
    # At most the largest listed scores, and caches half as large.
    most = min(8192, 16 * 14 * 64 * 4096 // (batch * q_heads * tokens),
               32 * 8192 * 64 // (batch * kv_heads * head_dim))
    high = _spread(rng, 1, max(1, most))
    return {"op": "tree", "batch": batch, "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "low": rng.randint(0, high), "high": high, "page": rng.choice([0, 0, 16, 64, 128]),
            "mask": rng.choice(["none", "none", "-inf", "lowest"]), "dtype": dtype}


def _lengths(case):
    """The sequences' lengths, evenly from low to high."""

    batch, low, high = case["batch"], case["low"], case["high"]
    return [low + (high - low) * b // max(1, batch - 1) for b in range(batch)]


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _trees(batch, tokens, g):
    """Parents [batch, tokens] (the root's is -1) of trees whose nodes follow near their parents, and the masks of
    ancestors and selves [batch, tokens, tokens]."""

    index = torch.arange(tokens, device=DEVICE)
    back = torch.rand(batch, tokens, device=DEVICE, generator=g).square().mul(min(8, tokens)).long()
    parents = (index - 1 - back).clamp_min(0)
    parents[:, 0] = -1
    return parents, _ancestors(parents)


def _ancestors(parents):
    batch, tokens = parents.shape
    eye = torch.eye(tokens, device=DEVICE).expand(batch, -1, -1)
    up = (parents.unsqueeze(-1) == torch.arange(tokens, device=DEVICE)).float()
    seen, steps = eye + up, 1
    while steps < tokens:  # paths of twice the length in each product
        seen, steps = ((seen @ seen) > 0).float(), 2 * steps
    return seen > 0


def _page_table(batch, pages, g):
    """Every sequence's pages, scattered over the pool."""

    return torch.randperm(batch * pages, device=DEVICE, generator=g).to(torch.int32).view(batch, pages)


def prepare(case, seed):
    g = _generator(seed)
    op, batch, tokens = case["op"], case["batch"], case["tokens"]
    dtype = DTYPES[case["dtype"]]
    state = {"op": op}

    def normal(*shape):
        return torch.randn(*shape, device=DEVICE, generator=g)

    if op == "tree":
        heads, dim, page = case["kv_heads"], case["head_dim"], case["page"]
        state["query"] = normal(batch, tokens, case["q_heads"], dim).to(dtype).transpose(1, 2)
        state["scale"] = dim ** -0.5
        order = torch.randperm(batch, device=DEVICE, generator=g)
        state["lengths"] = torch.tensor(_lengths(case), device=DEVICE, dtype=torch.int64)[order]
        capacity = case["high"] + tokens
        state["table"] = None
        shape = (batch, capacity, heads, dim)
        if page:
            capacity = -(-capacity // page) * page
            state["table"] = _page_table(batch, capacity // page, g)
            shape = (batch * capacity // page, page, heads, dim)
        state["key"], state["value"] = normal(*shape).to(dtype), normal(*shape).to(dtype)
        state["tree"] = _trees(batch, tokens, g)[1]
        state["mask"] = None
        if case["mask"] != "none":  # left padding of up to a quarter of a sequence
            padding = (torch.rand(batch, device=DEVICE, generator=g) * 0.25 * state["lengths"]).long()
            low = -math.inf if case["mask"] == "-inf" else torch.finfo(dtype).min
            behind = torch.arange(capacity, device=DEVICE) < padding.unsqueeze(-1)
            state["mask"] = torch.zeros(batch, 1, 1, capacity, device=DEVICE, dtype=dtype).masked_fill_(
                behind.view(batch, 1, 1, capacity), low)
    elif op == "verify":
        vocab = case["vocab"]
        state["parents"], state["tree"] = None, None
        if case["draft"]:
            state["tree"] = torch.ones(tokens, tokens, device=DEVICE).tril_().bool().expand(batch, -1, -1)
        else:
            state["parents"], state["tree"] = _trees(batch, tokens, g)
        logits = normal(batch, tokens, vocab).mul_(4)
        drafted = (logits + normal(batch, tokens, vocab))[:, : tokens - 1]
        state["target"] = torch.softmax(logits, -1).to(dtype)
        state["tokens"] = torch.randint(vocab, (batch, tokens), device=DEVICE, generator=g)
        state["draft"] = None
        if tokens > 1 and case["draft"]:
            state["draft"] = torch.softmax(drafted, -1).to(dtype)
            state["tokens"][:, 1:] = torch.multinomial(state["draft"].float().view(-1, vocab), 1,
                                                       generator=g).view(batch, tokens - 1)
        elif tokens > 1:  # the best candidates of the draft behind each node, the first child the best
            parents = state["parents"][:, 1:]
            rank = torch.tril(parents.unsqueeze(-1) == parents.unsqueeze(-2), -1).sum(-1)
            most = min(vocab, tokens)
            best = drafted.topk(most).indices
            state["tokens"][:, 1:] = best[torch.arange(batch, device=DEVICE).unsqueeze(-1), parents, rank % most]
        elif case["draft"]:
            state["draft"] = state["target"][:, :0]
        state["uniforms"] = torch.rand(batch, tokens, device=DEVICE, generator=g)
    else:
        heads, dim, page, capacity = case["kv_heads"], case["head_dim"], case["page"], case["capacity"]
        shape = (batch, capacity, heads, dim)
        state["table"] = None
        if page:
            state["table"] = _page_table(batch, capacity // page, g)
            shape = (batch * capacity // page, page, heads, dim)
        # Every layer's keys, then every layer's values, in one allocation.
        state["cache"] = normal(2 * LAYERS, *shape).to(dtype)
        state["keys"], state["values"] = (state["cache"][:LAYERS].unbind(0), state["cache"][LAYERS:].unbind(0))
        lengths = torch.randint(0, capacity - tokens + 1, (batch,), device=DEVICE, generator=g)
        state["lengths"] = lengths.repeat(LAYERS, 1)
        # The tree's first branch lies in front of the others: an accepted path follows it for some nodes, then
        # goes on in a branch that lies behind.
        kept = case["kept"]
        same = torch.randint(1, kept + 1, (batch, 1), device=DEVICE, generator=g)
        behind = torch.rand(batch, tokens, device=DEVICE, generator=g)
        behind[:, :kept] = 2.0
        behind = behind.argsort(-1)[:, :kept].sort(-1).values
        place = torch.arange(tokens, device=DEVICE).expand(batch, -1)
        path = place.clone()
        path[:, :kept] = torch.where((place[:, :kept] < same) | (tokens < 2 * kept), place[:, :kept], behind)
        state["path"] = torch.where(place < kept, path, -1)
        state["counts"] = torch.full((batch,), kept, device=DEVICE, dtype=torch.int64)
    return state


def _tree(state):
    query, lengths, tree = state["query"], state["lengths"], state["tree"]
    batch, q_heads, tokens, dim = query.shape
    key, value, table = state["key"], state["value"], state["table"]
    if table is not None:
        key, value = (t[table.long()].flatten(1, 2) for t in (key, value))
    heads, rows = key.shape[2], key.shape[1]
    key, value = (t.float().transpose(1, 2).contiguous() for t in (key, value))
    q = query.float().reshape(batch, heads, q_heads // heads * tokens, dim)
    scores = q @ key.transpose(-1, -2) * state["scale"]
    if state["mask"] is not None:
        scores = scores + state["mask"].float()
    node = torch.arange(rows, device=query.device) - lengths.unsqueeze(-1)  # [batch, rows]: < 0 in the sequence
    in_tree = ((node >= 0) & (node < tokens)).unsqueeze(1)
    nodes = node.clamp(0, tokens - 1).unsqueeze(1).expand(-1, tokens, -1)
    seen = (node < 0).unsqueeze(1) | (in_tree & tree.gather(2, nodes))  # [batch, tokens, rows]
    scores = scores.view(batch, heads, -1, tokens, rows).masked_fill_(~seen[:, None, None], -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    weights = (weights / weights.sum(-1, keepdim=True)).view(batch, heads, -1, rows)
    return (weights @ value).view(batch, q_heads, tokens, dim).to(query.dtype)


def _verify(state):
    target, draft, tokens, uniforms = state["target"], state["draft"], state["tokens"], state["uniforms"]
    batch, count, vocab = target.shape
    device = target.device
    each = torch.arange(batch, device=device)
    node = torch.arange(count, device=device)
    parents = (node - 1).expand(batch, -1) if state["parents"] is None else state["parents"]
    above = parents.clamp_min(0)
    p = target[each.unsqueeze(-1), above, tokens].double()
    u = uniforms.double()
    elder = torch.tril(parents.unsqueeze(-1) == parents.unsqueeze(-2), -1)  # [batch, node, elder sibling]
    if draft is not None:  # a chain: no node has a sibling
        q = draft[each.unsqueeze(-1), above.clamp_max(count - 2), tokens].double() if count > 1 else p
        accepted = u * q < p
    else:
        twice = (elder & (tokens.unsqueeze(-1) == tokens.unsqueeze(-2))).any(-1)
        p = torch.where(twice, 0.0, p)
        left = 1 - (elder * p.unsqueeze(-2)).sum(-1)
        accepted = u * left < p
    accepted &= node > 0
    chosen = accepted & ~(elder & accepted.unsqueeze(-2)).any(-1)
    chosen |= node == 0
    reached = ~(state["tree"] & ~chosen.unsqueeze(-2)).any(-1)
    counts = reached.sum(-1)
    path = torch.where(reached, node, count).sort(-1).values
    last = path.gather(-1, counts.unsqueeze(-1) - 1).squeeze(-1)
    weights = target[each, last].double()
    child = parents == last.unsqueeze(-1)
    if draft is not None:
        if count > 1:
            rest = (weights - draft[each, last.clamp_max(count - 2)].double()).clamp_min(0)
            weights = torch.where((child.any(-1, keepdim=True)) & (rest.sum(-1, keepdim=True) > 0), rest, weights)
    else:
        out = torch.zeros(batch, vocab, device=device, dtype=torch.float64)
        out.scatter_add_(1, tokens, child.double())
        rest = torch.where(out > 0, 0.0, weights)
        weights = torch.where(rest.sum(-1, keepdim=True) > 0, rest, weights)
    sums = weights.cumsum(-1)
    drawn = (sums <= u[:, :1] * sums[:, -1:]).sum(-1)
    ahead = path[:, 1:].clamp_max(count - 1)
    follow = torch.cat([tokens.gather(-1, ahead), tokens[:, :1]], -1)
    emitted = torch.where(node < counts.unsqueeze(-1) - 1, follow, -1)
    emitted = torch.where(node == counts.unsqueeze(-1) - 1, drawn.unsqueeze(-1), emitted)
    return torch.where(path < count, path, -1), emitted, counts


def _commit(state):
    cache, lengths, path, counts, table = (state[k] for k in ("cache", "lengths", "path", "counts", "table"))
    batch, tokens = path.shape
    each = torch.arange(batch, device=cache.device).view(1, batch, 1)
    layer = torch.arange(2 * LAYERS, device=cache.device).view(-1, 1, 1)
    place = torch.arange(tokens, device=cache.device)
    valid = place < counts.unsqueeze(-1)
    start = torch.cat([lengths, lengths]).unsqueeze(-1)
    source, target = start + torch.where(valid, path, place), start + place
    if table is None:
        cache[layer, each, target] = cache[layer, each, source]
    else:
        page = state["cache"].shape[2]
        cache[layer, table[each, target // page].long(), target % page] = cache[
            layer, table[each, source // page].long(), source % page]
    return cache, lengths + counts


def _import_backends():
    """The framework's kernels, imported once as a program does, not in every pass."""

    package = str(Path("llm-compiler_amd").resolve())
    if package not in sys.path:
        sys.path.insert(0, package)
    from stateful_llm_compiler_hip import backends

    _run_own.backends = backends
    return backends


def _run_own(state):
    backends = getattr(_run_own, "backends", None) or _import_backends()
    op = state["op"]
    if op == "verify":
        return backends.hip_verify_tokens(state["tokens"], state["target"], state["uniforms"],
                                          parents=state["parents"], draft_probs=state["draft"])
    if op == "commit":
        if "layers" not in state:  # made once, with the cache, and kept as long
            state["layers"] = backends.KVLayers(state["keys"], state["values"], block_table=state["table"])
        return state["cache"], backends.hip_kv_commit(state["layers"], state["lengths"], state["path"], state["counts"])
    if state["table"] is None:
        return backends.hip_tree_attention(state["query"], state["key"], state["value"], state["lengths"],
                                           state["tree"], state["mask"], scale=state["scale"])
    return backends.hip_paged_tree_attention(state["query"], state["key"], state["value"], state["table"],
                                             state["lengths"], state["tree"], state["mask"], scale=state["scale"])


def run(state):
    if own:
        return _run_own(state)
    return {"tree": _tree, "verify": _verify, "commit": _commit}[state["op"]](state)


def work(case):
    op, batch, tokens, size = case["op"], case["batch"], case["tokens"], BYTES[case["dtype"]]
    if op == "verify":
        # The chosen row of the target, the draft's too behind a refused token, and each node's own probabilities.
        rows = 2 if case["draft"] else 1
        return {"bytes": batch * (rows * case["vocab"] * size + tokens * (rows * size + 8 * 4 + 4)),
                "flops": 3 * batch * case["vocab"]}
    row = case["kv_heads"] * case["head_dim"] * size
    if op == "commit":
        # Half of the kept nodes lie behind their places; a kept row is read and written in every layer, K and V.
        return {"bytes": batch * (LAYERS * (2 * case["kept"] * row + 16) + 8 * tokens + 8),
                "flops": batch * LAYERS}
    lengths = _lengths(case)
    rows = sum(lengths) + batch * tokens
    queries = batch * case["q_heads"] * tokens * case["head_dim"] * size
    mask = batch * (case["high"] + tokens) * size if case["mask"] != "none" else 0
    pairs = sum(length * tokens + tokens * (tokens + 1) // 2 for length in lengths)
    return {"bytes": 2 * rows * row + 2 * queries + batch * (tokens * tokens + 8) + mask,
            "flops": 4 * pairs * case["q_heads"] * case["head_dim"]}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "commit":
        return None  # copies
    if case["op"] == "verify":
        return _exact_verify(state)
    query, table = state["query"], state["table"]
    batch, q_heads, tokens, dim = query.shape
    group = q_heads // case["kv_heads"]
    out = torch.empty(batch, q_heads, tokens, dim, device=DEVICE, dtype=torch.float64)
    for b in range(batch):
        length = int(state["lengths"][b])
        if table is None:
            k, v = state["key"][b], state["value"][b]
        else:
            pages = table[b].long()
            k, v = (t.index_select(0, pages).reshape(-1, case["kv_heads"], dim) for t in (state["key"], state["value"]))
        rows = length + tokens
        k, v = (t[:rows].double().repeat_interleave(group, 1).permute(1, 0, 2).contiguous() for t in (k, v))
        logits = torch.bmm(query[b].double(), k.transpose(1, 2).contiguous()) * state["scale"]
        if state["mask"] is not None:
            logits += state["mask"][b, 0, 0, :rows].double()
        logits[:, :, length:] = torch.where(state["tree"][b], logits[:, :, length:], -math.inf)
        out[b] = torch.bmm(torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True)), v)
    return out


def _exact_verify(state):
    """One sequence at a time, node by node."""

    target, draft = state["target"], state["draft"]
    batch, count, vocab = target.shape
    paths, emitted, counts = [], [], []
    for b in range(batch):
        tokens, u = state["tokens"][b].tolist(), state["uniforms"][b].tolist()
        parents = list(range(-1, count - 1)) if state["parents"] is None else state["parents"][b].tolist()
        path = [0]
        while True:
            row = target[b, path[-1]].double()
            children = [c for c in range(path[-1] + 1, count) if parents[c] == path[-1]]
            rest, left, follows = row.clone(), 1.0, None
            for c in children:
                token = tokens[c]
                chance = float(rest[token])
                if u[c] * left * (1.0 if draft is None else float(draft[b, path[-1], token])) < chance:
                    follows = c
                    break
                if draft is None:
                    rest[token] = 0.0
                    left -= chance
                else:
                    rest = torch.clamp(rest - left * draft[b, path[-1]].double(), min=0.0)
                    left = float(rest.sum())
            if follows is None:
                break
            path.append(follows)
        rest = rest if float(rest.sum()) > 0 else row
        sums = torch.cumsum(rest, 0)
        drawn = int(torch.searchsorted(sums, u[0] * sums[-1], right=True))
        fill = [-1] * (count - len(path))
        paths.append(path + fill)
        emitted.append([tokens[c] for c in path[1:]] + [drawn] + fill)
        counts.append(len(path))
    return tuple(torch.tensor(v, device=DEVICE) for v in (paths, emitted, counts))
