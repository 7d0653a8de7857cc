"""GPU tests of the operators on drafted tokens against plain 64-bit implementations."""

from __future__ import annotations

import math

import pytest
import torch

from helpers import announce, assert_bitwise_equal, generator
from stateful_llm_compiler_hip import _native, backends

pytestmark = pytest.mark.gpu

INF = float("inf")
NAN = float("nan")


# ---- tree attention -----------------------------------------------------------------


def random_tree(nodes, g, batch=None):
    """Masks of ancestors and selves of random trees."""

    masks = []
    for _ in range(batch or 1):
        mask = torch.eye(nodes, dtype=torch.bool)
        for c in range(1, nodes):
            mask[c] |= mask[int(torch.randint(max(0, c - 5), c, (1,), generator=g))]
        masks.append(mask)
    return torch.stack(masks) if batch else masks[0]


def tree_reference(query, key, value, lengths, tree, mask, scale):
    """fp64 output of tree attention over [B, Cap, KVH, D] buffers, and bounds of its
    parts per output: the weighted magnitudes of V, the largest score and the largest
    sum of a score's products' magnitudes of the row."""

    batch, q_heads, nodes, head_dim = query.shape
    capacity, kv_heads = key.shape[1:3]
    groups = q_heads // kv_heads
    out = torch.full(query.shape, NAN, dtype=torch.float64)
    weighted, top, products = (torch.zeros(query.shape, dtype=torch.float64) for _ in range(3))
    rows = capacity if mask is None else mask.shape[-1]
    if tree is None:
        tree = torch.ones(nodes, nodes, dtype=torch.bool).tril_()
    tree = tree.expand(batch, nodes, nodes)
    for b in range(batch):
        length = min(max(int(lengths[b]), 0), capacity)
        end = min(length + nodes, rows)
        for i in range(nodes):
            seen = torch.arange(end) < length
            behind = torch.arange(length, max(end, length))
            seen[length:end] = tree[b, i, behind - length]
            if mask is not None:
                seen &= mask[b, 0, 0, :end] != -INF
            at = seen.nonzero().view(-1)
            if not len(at):
                continue
            for h in range(q_heads):
                q = query[b, h, i].double()
                k, v = key[b, at, h // groups].double(), value[b, at, h // groups].double()
                t = k @ q * scale
                size = (k.abs() @ q.abs() * scale).max()
                if mask is not None:
                    t = t + mask[b, 0, 0, at].double()
                w = torch.softmax(t, 0)
                out[b, h, i] = w @ v
                weighted[b, h, i] = w @ v.abs()
                top[b, h, i], products[b, h, i] = (t - t.max()).abs().clamp_max(200).max(), size
    return out, weighted, top, products


def assert_tree_close(actual, reference, keys):
    """|actual - exact| within what the formula's steps may be off.

    With h half the type's spacing (bf16 2^-8, fp16 2^-11 relative) the 16-bit forms
    round each weight (h of the weighted |V|, and h again through their sum) and the
    output (h of it); fp16 weights under 2^-14 of the row's largest are off by up to
    2^-25 each, of at most `keys` values of size |V|.  In fp32 (u = 2^-24): a score's
    products and their sum are off by (D + 2) u of the products' magnitudes, the score
    times log2 e by 3 u of its distance from the maximum, exp2 by 2 u (a unit in the
    last place): each moves a weight by as much, and again through the sum; the sums
    of `keys` weights and weighted values, in any order, by keys u each, and the
    division by 2 u."""

    exact, weighted, top, products = reference
    actual = actual.cpu()
    dtype = actual.dtype
    actual = actual.double()
    empty = torch.isnan(exact)
    assert torch.equal(torch.isnan(actual), empty)
    u = 2.0**-24
    weights = 2 * ((exact.shape[-1] + 2) * u * products + 3 * u * top + 2 * u) + 2 * keys * u + 2 * u
    bound = weighted * weights
    if dtype == torch.float32:
        bound = bound + u * exact.abs()
    else:
        h = torch.finfo(dtype).eps / 2
        bound = bound + 2 * h * weighted + h * exact.abs() + h * bound
        if dtype == torch.float16:
            bound = bound + keys * 2.0**-25 * 2 * weighted.abs().amax() + 2.0**-25
    bound, error = bound[~empty], (actual - exact)[~empty].abs()
    assert (error <= bound).all(), float((error / bound).max())


def paged(buffer, page_tokens, g, extra=3):
    """Pool and table whose gather is ``buffer`` (capacity padded to whole pages with
    NaN); the pages that no sequence owns hold NaN."""

    batch, capacity = buffer[0].shape[:2]
    pages = -(-capacity // page_tokens)
    order = torch.randperm(batch * pages + extra, generator=g)[: batch * pages].view(batch, pages)
    pools = []
    for side in buffer:
        pool = torch.full((batch * pages + extra, page_tokens, *side.shape[2:]), NAN, dtype=side.dtype)
        whole = torch.full((batch, pages * page_tokens, *side.shape[2:]), NAN, dtype=side.dtype)
        whole[:, :capacity] = side
        pool[order.view(-1)] = whole.view(batch * pages, page_tokens, *side.shape[2:])
        pools.append(pool)
    return *pools, order.to(torch.int32)


def tree_inputs(g, batch, q_heads, kv_heads, head_dim, nodes, capacity, dtype, lengths):
    """Queries and caches; NaN and infinities in the rows behind the nodes."""

    query = torch.randn(batch, q_heads, nodes, head_dim, generator=g).to(dtype)
    key, value = (torch.randn(batch, capacity, kv_heads, head_dim, generator=g).to(dtype) for _ in range(2))
    for b, length in enumerate(lengths):
        end = max(0, length) + nodes
        key[b, end:], value[b, end:] = NAN, INF
        value[b, end + 1 :: 2] = NAN
    return query, key, value, torch.tensor(lengths)


TREE_CASES = [
    # q_heads, kv_heads, head_dim, nodes, capacity, lengths
    (14, 2, 64, 8, 700, [600, 13]),
    (14, 2, 64, 16, 1100, [0, 1, 63, 1000]),
    (14, 2, 64, 1, 300, [299, 0]),
    (14, 2, 64, 33, 200, [130, 64]),
    (14, 2, 64, 64, 420, [350, 17]),
    (4, 2, 128, 5, 300, [255, 100, 40]),
    (32, 8, 128, 7, 200, [129, 0]),
    (8, 8, 64, 16, 128, [112]),
    (2, 1, 64, 130, 400, [200, 64]),
    (20, 1, 64, 3, 200, [100]),
    (40, 1, 128, 9, 150, [100]),
    (6, 2, 80, 11, 150, [90, 20]),
    (5, 1, 72, 4, 150, [65]),
    (12, 1, 256, 6, 150, [77]),
    (6, 3, 256, 40, 150, [77]),
    (9, 3, 33, 10, 150, [70, 3]),
    (3, 1, 1, 4, 50, [20]),
    (4, 4, 200, 17, 90, [64]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", TREE_CASES)
def test_tree_attention(gpu, case, dtype):
    q_heads, kv_heads, head_dim, nodes, capacity, lengths = case
    announce(f"tree attention {case} {dtype}")
    g = generator(1000 * q_heads + 10 * nodes + head_dim)
    query, key, value, lengths = tree_inputs(g, len(lengths), q_heads, kv_heads, head_dim, nodes, capacity, dtype,
                                             lengths)
    tree = random_tree(nodes, g, len(lengths))
    scale = head_dim**-0.5
    reference = tree_reference(query, key, value, lengths, tree, None, scale)
    out = backends.hip_tree_attention(query.to(gpu), key.to(gpu), value.to(gpu), lengths.to(gpu), tree.to(gpu),
                                      scale=scale)
    assert out.shape == query.shape and out.dtype == dtype
    assert_tree_close(out, reference, int(lengths.max()) + nodes)
    for page_tokens in (16, 64):
        key_pool, value_pool, table = paged((key, value), page_tokens, g)
        again = backends.hip_paged_tree_attention(query.to(gpu), key_pool.to(gpu), value_pool.to(gpu), table.to(gpu),
                                                  lengths.int().to(gpu), tree.to(gpu), scale=scale)
        assert_tree_close(again, reference, int(lengths.max()) + nodes)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kind", ["-inf", "lowest", "random", "all -inf", "all lowest", "short"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (4, 1, 80)])
def test_tree_attention_with_a_mask(gpu, kind, dtype, heads):
    q_heads, kv_heads, head_dim = heads
    announce(f"tree attention mask {kind} {dtype} {heads}")
    g = generator(5)
    nodes, capacity = 9, 330
    query, key, value, lengths = tree_inputs(g, 3, q_heads, kv_heads, head_dim, nodes, capacity, dtype, [310, 64, 0])
    low = -INF if "-inf" in kind else torch.finfo(dtype).min
    rows = 200 if kind == "short" else capacity
    mask = torch.zeros(3, 1, 1, rows, dtype=dtype)
    if kind == "random":
        mask = (torch.randn(3, 1, 1, rows, generator=g) * 3).to(dtype)
        mask[:, :, :, ::7] = -INF
    elif kind.startswith("all"):
        mask[0] = low
        mask[1, :, :, :60] = low
    elif kind == "short":
        mask[0, :, :, 70:90] = low
    else:
        mask[0, :, :, :133] = low
        mask[1, :, :, :64] = low  # nothing of the sequence is left
    hidden = mask == -INF
    for b in range(3):  # what a masked row holds is not seen
        key[b, :rows][hidden[b, 0, 0]] = NAN
        value[b, :rows][hidden[b, 0, 0]] = INF
    tree = random_tree(nodes, g)
    scale = head_dim**-0.5
    reference = tree_reference(query, key, value, lengths, tree, mask, scale)
    args = [t.to(gpu) for t in (query, key, value, lengths, tree, mask)]
    assert_tree_close(backends.hip_tree_attention(*args, scale=scale), reference, capacity)
    # The same from an fp32 mask that is a strided view.
    wide = torch.zeros(3, 1, 1, 2 * rows)
    wide[..., ::2] = mask.float()
    args[5] = wide.to(gpu)[..., ::2]
    assert_tree_close(backends.hip_tree_attention(*args, scale=scale), reference, capacity)
    key_pool, value_pool, table = paged((key, value), 32, g)
    out = backends.hip_paged_tree_attention(args[0], key_pool.to(gpu), value_pool.to(gpu), table.to(gpu), args[3],
                                            args[4], mask.to(gpu), scale=scale)
    assert_tree_close(out, reference, capacity)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kind", ["blocks", "padding", "lowest", "NaN", "short"])
@pytest.mark.parametrize("q_heads,kv_heads,head_dim,nodes", [(14, 2, 64, 20), (14, 2, 64, 16), (6, 1, 64, 9), (2, 1, 64, 3),
                                                             (4, 2, 128, 7), (2, 1, 256, 5)])
def test_tree_attention_of_long_masked_caches(gpu, q_heads, kv_heads, head_dim, nodes, kind, dtype):
    """Masks over thousands of rows: tiles of which all, some and no keys are masked out."""

    announce(f"tree attention long mask {q_heads} {head_dim} {nodes} {kind} {dtype}")
    g = generator(nodes)
    lengths, capacity = [1900, 611], 1950
    query, key, value, lengths = tree_inputs(g, 2, q_heads, kv_heads, head_dim, nodes, capacity, dtype, lengths)
    rows = 1500 if kind == "short" else capacity
    mask = (torch.randn(2, 1, 1, rows, generator=g) * 2).to(dtype)
    if kind == "blocks":
        for first in range(0, rows, 50):
            if torch.rand(1, generator=g) < 0.6:
                mask[0, ..., first : first + int(torch.randint(20, 140, (1,), generator=g))] = -INF
        mask[1, ..., 200:456] = -INF
    elif kind in ("padding", "short"):
        mask[0, ..., :1111] = -INF
        mask[1, ..., :512] = -INF
    elif kind == "lowest":
        mask[0, ..., :1111] = torch.finfo(dtype).min
        mask[1, ..., :620] = torch.finfo(dtype).min  # and of some nodes
    else:
        mask[0, ..., 1203] = NAN
        mask[1, ..., 700:] = NAN  # behind the nodes
    hidden = mask == -INF
    for b in range(2):
        key[b, :rows][hidden[b, 0, 0]] = INF
        value[b, :rows][hidden[b, 0, 0]] = NAN
    tree = random_tree(nodes, g)
    scale = head_dim**-0.5
    reference = tree_reference(query, key, value, lengths, tree, mask, scale)
    args = [t.to(gpu) for t in (query, key, value, lengths, tree, mask)]

    def check(out):
        for b in range(2):  # by itself: a sequence of NaN has no bounds for the other
            assert_tree_close(out[b], [part[b] for part in reference], capacity)

    check(backends.hip_tree_attention(*args, scale=scale))
    key_pool, value_pool, table = paged((key, value), 16, g)
    out = backends.hip_paged_tree_attention(args[0], key_pool.to(gpu), value_pool.to(gpu), table.to(gpu), *args[3:],
                                            scale=scale)
    check(out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("head_dim", [64, 128, 40])
@pytest.mark.parametrize("nodes,length", [(12, 61), (70, 100), (3, 0)])
def test_tree_attention_keeps_what_a_node_does_not_see_from_it(gpu, nodes, length, head_dim, dtype):
    announce(f"tree attention unseen NaN {nodes} {length} {head_dim} {dtype}")
    g = generator(17)
    query, key, value, lengths = tree_inputs(g, 1, 6, 2, head_dim, nodes, length + nodes + 5, dtype, [length])
    tree = random_tree(nodes, g)
    tree[0, 0] = False  # node 0 sees the sequence only: nothing where that is empty
    bad = nodes // 2
    args = [query.to(gpu), key.to(gpu), value.to(gpu), lengths.to(gpu), tree.to(gpu)]
    clean = backends.hip_tree_attention(*args, scale=0.1).cpu()
    for fill in (NAN, INF, -INF):
        for side in (1, 2):
            dirty = list(args)
            dirty[side] = args[side].clone()
            dirty[side][0, length + bad, 0] = fill
            out = backends.hip_tree_attention(*dirty, scale=0.1).cpu()
            sees = tree[:, bad].clone()
            assert torch.isfinite(out[:, 3:][:, :, 1:]).all()  # the other KV head's queries
            assert torch.equal(out[:, 3:, 1:], clean[:, 3:, 1:])
            assert torch.equal(out[:, :3, ~sees].nan_to_num(7.0), clean[:, :3, ~sees].nan_to_num(7.0))
            if side == 2:
                expected = torch.full_like(out[:, :3, sees], fill)
                assert torch.equal(torch.isnan(out[:, :3, sees]), torch.isnan(expected))
                if fill == fill:
                    assert torch.equal(out[:, :3, sees], expected)


def test_tree_attention_layouts(gpu):
    announce("tree attention layouts")
    g = generator(3)
    batch, q_heads, kv_heads, head_dim, nodes, capacity = 3, 14, 2, 64, 10, 200
    for dtype in (torch.bfloat16, torch.float32):
        query, key, value, lengths = tree_inputs(g, batch, q_heads, kv_heads, head_dim, nodes, capacity, dtype,
                                                 [100, 7, 150])
        tree = random_tree(nodes, g, batch)
        reference = tree_reference(query, key, value, lengths, tree, None, 0.125)
        base = [t.to(gpu) for t in (query, key, value, lengths, tree)]
        want = backends.hip_tree_attention(*base, scale=0.125)
        assert_tree_close(want, reference, 200)

        def same(query=base[0], key=base[1], value=base[2], lengths=base[3], tree=base[4]):
            out = backends.hip_tree_attention(query, key, value, lengths, tree, scale=0.125)
            assert out.shape == want.shape
            assert_bitwise_equal(out, want)

        def unaligned(query=base[0], key=base[1], value=base[2]):
            out = backends.hip_tree_attention(query, key, value, base[3], base[4], scale=0.125)
            assert_tree_close(out, reference, 200)

        same(query=base[0].transpose(1, 2).contiguous().transpose(1, 2))  # [B, T, H, D]
        same(lengths=base[3].int())
        same(tree=base[4].transpose(1, 2).contiguous().transpose(1, 2))
        # [B, KVH, Cap, D] caches, and rows with room between them.
        same(key=base[1].permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3),
             value=base[2].permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3))
        roomy = [torch.full((batch, capacity + 3, kv_heads, 2 * head_dim), NAN, dtype=dtype, device=gpu)
                 for _ in range(2)]
        for room, side in zip(roomy, base[1:3]):
            room[:, :capacity, :, :head_dim] = side
        same(key=roomy[0][:, :capacity, :, :head_dim], value=roomy[1][:, :capacity, :, :head_dim])
        # Rows that start on any element.
        odd = [torch.full((batch, capacity, kv_heads, head_dim + 3), NAN, dtype=dtype, device=gpu) for _ in range(2)]
        for room, side in zip(odd, base[1:3]):
            room[..., 1 : head_dim + 1] = side
        unaligned(key=odd[0][..., 1 : head_dim + 1], value=odd[1][..., 1 : head_dim + 1])
        odd_query = torch.full((batch, q_heads, nodes, head_dim + 1), NAN, dtype=dtype, device=gpu)
        odd_query[..., 1:] = base[0]
        unaligned(query=odd_query[..., 1:])
        # One query for all sequences, as an expanded view.
        one = base[0][:1].expand(batch, -1, -1, -1)
        out = backends.hip_tree_attention(one, *base[1:], scale=0.125)
        assert_tree_close(out, tree_reference(query[:1].expand(batch, -1, -1, -1), key, value, lengths, tree, None, 0.125),
                          200)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tree_attention_lengths_at_and_past_the_ends(gpu, dtype):
    # Nodes past the capacity were not stored; a negative length is none.
    announce(f"tree attention lengths {dtype}")
    g = generator(8)
    capacity, nodes, lengths = 100, 6, [97, 100, 105, -4, 94, 2**31 + 5]
    query, key, value, _ = tree_inputs(g, len(lengths), 4, 2, 64, nodes, capacity, dtype, [capacity] * len(lengths))
    tree = random_tree(nodes, g)
    lengths = torch.tensor(lengths)
    reference = tree_reference(query, key, value, lengths, tree, None, 0.125)
    args = [t.to(gpu) for t in (query, key, value, lengths, tree)]
    assert_tree_close(backends.hip_tree_attention(*args, scale=0.125), reference, capacity)


def test_tree_attention_chain_and_single_tokens(gpu):
    announce("tree attention chain")
    g = generator(9)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        query, key, value, lengths = tree_inputs(g, 5, 14, 2, 64, 21, 400, dtype, [300, 5, 0, 64, 377])
        args = [t.to(gpu) for t in (query, key, value, lengths)]
        out = backends.hip_tree_attention(*args, None, scale=0.125)
        assert_tree_close(out, tree_reference(query, key, value, lengths, None, None, 0.125), 400)
        # One node is decode attention over a length that counts it.
        one = backends.hip_tree_attention(args[0][:, :, :1], *args[1:], None, scale=0.125)
        assert_tree_close(one, tree_reference(query[:, :, :1], key, value, lengths, None, None, 0.125), 400)
        decode = backends.hip_decode_attention(args[0][:, :, :1], args[1], args[2], args[3] + 1, None, scale=0.125)
        assert (one.float() - decode.float()).abs().max() <= 2e-2


def test_tree_attention_of_many_sequences(gpu):
    announce("tree attention 150 sequences")
    g = generator(10)
    lengths = torch.randint(0, 40, (150,), generator=g).tolist()
    lengths[77] = 300
    for dtype in (torch.bfloat16, torch.float32):
        query, key, value, lengths_t = tree_inputs(g, 150, 4, 2, 64, 3, 310, dtype, lengths)
        tree = random_tree(3, g, 150)
        args = [t.to(gpu) for t in (query, key, value, lengths_t, tree)]
        out = backends.hip_tree_attention(*args, scale=0.125)
        assert_tree_close(out, tree_reference(query, key, value, lengths_t, tree, None, 0.125), 303)


def test_tree_attention_of_large_and_far_scores(gpu):
    # The running maximum moves over many tiles, by more than exp's range.
    announce("tree attention large scores")
    g = generator(11)
    for dtype in (torch.bfloat16, torch.float32):
        query, key, value, lengths = tree_inputs(g, 2, 4, 2, 64, 8, 900, dtype, [880, 880])
        ramp = torch.linspace(0, 1, 900).view(1, -1, 1, 1)
        key[0] = (query[0, 0, 0].float() * ramp[0] * 2).to(dtype)
        key[1] = (query[1, 0, 0].float() * (1 - ramp[0]) * 2).to(dtype)
        tree = random_tree(8, g)
        args = [t.to(gpu) for t in (query, key, value, lengths, tree)]
        out = backends.hip_tree_attention(*args, scale=1.0)
        assert_tree_close(out, tree_reference(query, key, value, lengths, tree, None, 1.0), 900)


def test_tree_attention_repeats_bit_for_bit_on_streams_and_in_graphs(gpu):
    announce("tree attention streams and graphs")
    g = generator(12)
    query, key, value, lengths = tree_inputs(g, 4, 14, 2, 64, 16, 2100, torch.bfloat16, [2000, 1500, 3, 700])
    tree = random_tree(16, g, 4).to(gpu)
    args = [t.to(gpu) for t in (query, key, value, lengths)]
    want = backends.hip_tree_attention(*args, tree, scale=0.125)
    for _ in range(3):
        assert_bitwise_equal(backends.hip_tree_attention(*args, tree, scale=0.125), want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for stream in streams * 2:
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            outs.append(backends.hip_tree_attention(*args, tree, scale=0.125))
    torch.cuda.synchronize()
    for out in outs:
        assert_bitwise_equal(out, want)
    static = [t.clone() for t in args]
    workspace = _native.DeviceWorkspace(gpu)
    backends.hip_tree_attention(*static, tree, scale=0.125, workspace=workspace)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = backends.hip_tree_attention(*static, tree, scale=0.125, workspace=workspace)
    for turn in range(4):
        static[0].copy_(args[0].roll(turn, 1))
        static[3].copy_((args[3] + 5 * turn).clamp_max(2000))
        graph.replay()
        torch.cuda.synchronize()
        assert_bitwise_equal(out, backends.hip_tree_attention(static[0], *args[1:3], static[3], tree, scale=0.125))


def dense_reference(query, key, value, lengths, tree, scale):
    """``tree_reference`` without a mask, on the inputs' device a head at a time, for
    lengths of at least one."""

    batch, q_heads, nodes, head_dim = query.shape
    capacity, kv_heads = key.shape[1:3]
    parts = [torch.empty(query.shape, dtype=torch.float64) for _ in range(4)]
    if tree is None:
        tree = torch.ones(nodes, nodes, dtype=torch.bool, device=query.device).tril_()
    for b in range(batch):
        length = int(lengths[b])
        end = length + nodes
        seen = torch.cat([torch.ones(nodes, length, dtype=torch.bool, device=query.device), tree], 1)
        for h in range(q_heads):
            q = query[b, h].double()
            k, v = (side[b, :end, h * kv_heads // q_heads].double() for side in (key, value))
            t = (q @ k.T * scale).masked_fill(~seen, -INF)
            w = torch.softmax(t, -1)
            away = (t.amax(-1, keepdim=True) - t).clamp_max(200).masked_fill(~seen, 0).amax(-1, keepdim=True)
            size = (q.abs() @ k.abs().T * scale).masked_fill(~seen, 0).amax(-1, keepdim=True)
            for part, x in zip(parts, (w @ v, w @ v.abs(), away.expand(nodes, head_dim), size.expand(nodes, head_dim))):
                part[b, h] = x.cpu()
    return parts


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", [
    # q_heads, kv_heads, head_dim, nodes, lengths, whether a tree
    (2, 1, 64, 1024, [900], True),
    (2, 1, 64, 4096, [301], False),
    (14, 2, 64, 8, [69001], True),
    (4, 2, 128, 5, [39990, 3], True),
    (16, 1, 64, 100, [9000, 1], True),
    (3, 1, 40, 30, [20000], True),
    (6, 2, 256, 9, [5001, 700], True),
    (8, 2, 200, 30, [3000], True),
])
def test_tree_attention_of_wide_trees_and_long_caches(gpu, case, dtype):
    q_heads, kv_heads, head_dim, nodes, lengths, is_tree = case
    announce(f"tree attention {case} {dtype}")
    g = generator(nodes)
    capacity = max(lengths) + nodes + 7
    tensors = tree_inputs(g, len(lengths), q_heads, kv_heads, head_dim, nodes, capacity, dtype, lengths)
    query, key, value, lengths = (t.to(gpu) for t in tensors)
    tree = random_tree(nodes, g).to(gpu) if is_tree else None
    out = backends.hip_tree_attention(query, key, value, lengths, tree, scale=head_dim**-0.5)
    reference = dense_reference(query, key, value, lengths, tree, head_dim**-0.5)
    assert_tree_close(out, reference, capacity)
    key_pool, value_pool, table = paged(tensors[1:3], 16, g)
    out = backends.hip_paged_tree_attention(query, key_pool.to(gpu), value_pool.to(gpu), table.to(gpu), lengths, tree,
                                            scale=head_dim**-0.5)
    assert_tree_close(out, reference, capacity)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", [
    # batch, q_heads, kv_heads, head_dim, nodes, low, high
    (17, 14, 2, 64, 16, 211, 221),
    (17, 14, 2, 64, 32, 211, 240),
    (17, 14, 2, 64, 49, 211, 221),
    (20, 32, 8, 128, 15, 91, 145),
    (29, 12, 1, 256, 11, 50, 286),
    (9, 14, 2, 64, 8, 1, 700),
    (3, 4, 2, 64, 5, 100, 270),
])
def test_tree_attention_of_batches_of_short_caches(gpu, case, dtype):
    """Around the fewest rows that a piece has, where one, two and more are cut."""

    batch, q_heads, kv_heads, head_dim, nodes, low, high = case
    announce(f"tree attention short {case} {dtype}")
    g = generator(nodes + batch)
    lengths = torch.randint(low, high + 1, (batch,), generator=g).tolist()
    tensors = tree_inputs(g, batch, q_heads, kv_heads, head_dim, nodes, high + nodes, dtype, lengths)
    query, key, value, lengths = (t.to(gpu) for t in tensors)
    tree = random_tree(nodes, g).to(gpu)
    reference = dense_reference(query, key, value, lengths, tree, head_dim**-0.5)
    for _ in range(2):
        out = backends.hip_tree_attention(query, key, value, lengths, tree, scale=head_dim**-0.5)
        assert_tree_close(out, reference, high + nodes)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("batch,q_heads,kv_heads,head_dim,nodes", [(140, 4, 2, 64, 3), (70, 32, 4, 64, 2), (301, 2, 1, 128, 1)])
def test_tree_attention_of_large_batches_of_uneven_lengths(gpu, batch, q_heads, kv_heads, head_dim, nodes, dtype):
    """Whole sequences for all CUs, but for a few that are far longer."""

    announce(f"tree attention uneven {batch} {dtype}")
    g = generator(batch)
    capacity = 1800
    lengths = torch.randint(1, 60, (batch,), generator=g).tolist()
    for at, length in ((0, 1500), (batch // 2, 900), (batch // 2 + 1, 1790), (batch - 1, 1200)):
        lengths[at] = length
    query = torch.randn(batch, q_heads, nodes, head_dim, generator=g).to(dtype).to(gpu)
    key, value = (torch.randn(batch, capacity, kv_heads, head_dim, device=gpu, generator=torch.Generator(gpu).manual_seed(n))
                  .to(dtype) for n in (1, 2))
    lengths = torch.tensor(lengths, device=gpu)
    tree = random_tree(nodes, g).to(gpu)
    reference = dense_reference(query, key, value, lengths, tree, head_dim**-0.5)
    for _ in range(2):
        out = backends.hip_tree_attention(query, key, value, lengths, tree, scale=head_dim**-0.5)
        assert_tree_close(out, reference, capacity)


def large_reference(query, key, value, lengths, tree, mask, scale):
    """``tree_reference`` on the inputs' device, a KV head at a time; rows that the mask
    hides take no part, whatever they hold."""

    batch, q_heads, nodes, head_dim = query.shape
    capacity, kv_heads = key.shape[1:3]
    group = q_heads // kv_heads
    if tree is None:
        tree = torch.ones(nodes, nodes, dtype=torch.bool, device=query.device).tril_()
    parts = [torch.empty(query.shape, dtype=torch.float64, device=query.device) for _ in range(4)]
    for b, length in enumerate(lengths.tolist()):
        end = min(length + nodes, capacity)
        seen = torch.cat([torch.ones(nodes, length, dtype=torch.bool, device=query.device), tree], 1)[:, :end]
        add = torch.zeros(end, dtype=torch.float64, device=query.device)
        if mask is not None:
            hidden = mask[b, 0, 0, :end] == -INF
            add, seen = mask[b, 0, 0, :end].double().masked_fill(hidden, 0), seen & ~hidden
        for h in range(kv_heads):
            q = query[b, h * group : (h + 1) * group].double()
            k, v = (side[b, :end, h].double() for side in (key, value))
            if mask is not None:
                k, v = (side.masked_fill(hidden.unsqueeze(1), 0) for side in (k, v))
            products = (q.view(-1, head_dim) @ k.T).view(group, nodes, end) * scale + add
            t = products.masked_fill(~seen, -INF)
            w = torch.softmax(t, -1)
            away = (t.amax(-1, keepdim=True) - t).clamp_max(200).masked_fill(~seen, 0).amax(-1, keepdim=True)
            size = (q.abs().view(-1, head_dim) @ k.abs().T).view(group, nodes, end) * scale
            size = size.masked_fill(~seen, 0).amax(-1, keepdim=True)
            rows = w.view(-1, end)
            bounds = (rows @ v.abs(), away.expand(-1, -1, head_dim), size.expand(-1, -1, head_dim))
            for part, x in zip(parts, (rows @ v, *(bound.nan_to_num(0.0) for bound in bounds))):
                part[b, h * group : (h + 1) * group] = x.reshape(group, nodes, head_dim)
    return [part.cpu() for part in parts]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("batch,q_heads,kv_heads,head_dim,nodes", [
    (140, 4, 2, 64, 3), (70, 32, 4, 64, 2), (301, 2, 1, 128, 1), (130, 14, 2, 40, 9), (9, 60, 30, 256, 2),
    # Fewer than four sequences: none is cut.
    (3, 180, 90, 64, 2), (1, 256, 256, 64, 1), (2, 8, 2, 64, 4096)])
def test_tree_attention_of_large_batches_on_pages_with_masks_in_graphs(gpu, batch, q_heads, kv_heads, head_dim, nodes,
                                                                       masked, dtype):
    """Whole sequences for all CUs, of which the far longer ones are cut: others at every
    replay of one graph, and none; masks that hide whole tiles within the cut pieces."""

    announce(f"tree attention large {batch} {kv_heads} {nodes} {masked} {dtype}")
    g = generator(batch + nodes)
    chain = nodes > 1024
    capacity = 1808 if not chain else 4608
    query = torch.randn(batch, q_heads, nodes, head_dim, generator=g).to(dtype).to(gpu)
    key, value = (torch.randn(batch, capacity, kv_heads, head_dim, device=gpu, generator=torch.Generator(gpu).manual_seed(n))
                  .to(dtype) for n in (1, 2))
    high = capacity - nodes
    turns = []
    for long in ((0, batch // 2, batch - 1), (batch // 3, batch // 3 + 1), ()):
        lengths = torch.randint(0, 60, (batch,), generator=g)
        for at, length in zip(long, (high, high * 2 // 3, high - 65)):
            lengths[at % batch] = length
        turns.append(lengths)
    tree = None if chain else random_tree(nodes, g).to(gpu)
    mask = None
    if masked:
        mask = torch.randn(batch, 1, 1, capacity, generator=g)
        mask[0, ..., :700] = mask[1::3, ..., 200:900] = mask[::5, ..., 1000:1300] = -INF
        mask[1::4, ..., :21] = -INF  # and some whole sequences
        mask[torch.rand(mask.shape, generator=g) < 0.02] = -INF
        mask = mask.to(gpu, dtype)
        hidden = (mask[:, 0, 0] == -INF)[..., None, None]
        key, value = key.masked_fill(hidden, INF), value.masked_fill(hidden, NAN)
    pages = capacity // 16
    order = torch.randperm(batch * pages + 2, generator=g)[: batch * pages].view(batch, pages).to(gpu)
    pools = []
    for side in (key, value):
        pool = torch.full((batch * pages + 2, 16, kv_heads, head_dim), NAN, dtype=dtype, device=gpu)
        pool[order.view(-1)] = side.view(batch * pages, 16, kv_heads, head_dim)
        pools.append(pool)
    table = order.to(torch.int32)
    references = [large_reference(query, key, value, lengths.to(gpu), tree, mask, head_dim**-0.5) for lengths in turns]
    for paged_form in (False, True):
        workspace = _native.DeviceWorkspace(gpu)
        lengths = turns[0].to(gpu)

        def run(lengths, workspace=None):
            if paged_form:
                return backends.hip_paged_tree_attention(query, *pools, table, lengths, tree, mask, scale=head_dim**-0.5,
                                                         workspace=workspace)
            return backends.hip_tree_attention(query, key, value, lengths, tree, mask, scale=head_dim**-0.5,
                                               workspace=workspace)

        run(lengths, workspace)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(lengths, workspace)
        for turn in (1, 0, 2, 1):
            lengths.copy_(turns[turn])
            out.fill_(7.0)
            graph.replay()
            torch.cuda.synchronize()
            assert_tree_close(out, references[turn], capacity)
            assert_bitwise_equal(out, run(lengths))


def test_tree_attention_with_a_mask_of_no_rows(gpu):
    announce("tree attention empty mask")
    for dtype in (torch.bfloat16, torch.float32):
        query, cache = torch.ones(2, 4, 3, 64, device=gpu, dtype=dtype), torch.ones(2, 32, 2, 64, device=gpu, dtype=dtype)
        lengths = torch.tensor([0, 20], device=gpu)
        mask = torch.zeros(2, 1, 1, 0, device=gpu)
        assert backends.hip_tree_attention(query, cache, cache, lengths, None, mask, scale=1.0).isnan().all()


def test_offsets_past_32_bits(gpu):
    """Caches and pools of more than 2^31 elements: attention and commit at their ends."""

    g = generator(31)
    dtype, nodes, length = torch.bfloat16, 6, 300
    query, key, value, lengths = tree_inputs(g, 1, 4, 1, 64, nodes, 320, dtype, [length])
    tree = random_tree(nodes, g)
    reference = tree_reference(query, key, value, lengths, tree, None, 0.125)
    path, counts = torch.tensor([[0, 2, 5, -1, -1, -1]], device=gpu), torch.tensor([3], device=gpu)
    moved = commit_reference([key, value], lengths, path.cpu(), counts.cpu())
    query, lengths, tree = query.to(gpu), lengths.to(gpu), tree.to(gpu)

    announce("offsets past 32 bits: a sequence")
    caches = [torch.zeros(2, 2**25 + 16, 1, 64, dtype=dtype, device=gpu) for _ in range(2)]
    for cache, side in zip(caches, (key, value)):
        cache[1, :320] = side[0].to(gpu)
    both = torch.cat([lengths * 0, lengths])
    out = backends.hip_tree_attention(query.expand(2, -1, -1, -1), *caches, both, tree, scale=0.125)
    assert_tree_close(out[1:], reference, 320)
    backends.hip_kv_commit(backends.KVLayers(caches[:1], caches[1:]), both, path.expand(2, -1).contiguous(),
                           torch.cat([counts * 0, counts]))
    for cache, side in zip(caches, moved):
        assert torch.equal(bits(cache[1:, :320].cpu()), bits(side))
        assert not cache[0].any()
    del caches, cache

    announce("offsets past 32 bits: pages")
    pools = [torch.zeros(2**21 + 40, 16, 1, 64, dtype=dtype, device=gpu) for _ in range(2)]
    table = (2**21 + 39 - torch.arange(20, dtype=torch.int32, device=gpu)).unsqueeze(0)
    for pool, side in zip(pools, (key, value)):
        pool[table[0].long()] = side.view(20, 16, 1, 64).to(gpu)
    out = backends.hip_paged_tree_attention(query, *pools, table, lengths, tree, scale=0.125)
    assert_tree_close(out, reference, 320)
    backends.hip_kv_commit(backends.KVLayers(pools[:1], pools[1:], block_table=table), lengths, path, counts)
    for pool, side in zip(pools, moved):
        assert torch.equal(bits(pool[table[0].long()].cpu().view(1, 320, 1, 64)), bits(side))
        assert not pool[: 2**21].any()
    del pools, pool

    # Rows 4 MB apart, and a little more, which are no longer on 16 bytes.
    query, key, value, lengths = tree_inputs(g, 1, 4, 1, 64, nodes, 1060, dtype, [1050])
    reference = tree_reference(query, key, value, lengths, tree.cpu(), None, 0.125)
    rooms = [torch.empty(1060 * (2**21 + 1), dtype=dtype, device=gpu) for _ in range(2)]
    for step in (2**21, 2**21 + 1):
        announce(f"offsets past 32 bits: rows {step} elements apart")
        caches = [room.as_strided((1, 1060, 1, 64), (2**21, step, 64, 1)) for room in rooms]
        for cache, side in zip(caches, (key, value)):
            cache.copy_(side)
        out = backends.hip_tree_attention(query.to(gpu), *caches, lengths.to(gpu), tree, scale=0.125)
        assert_tree_close(out, reference, 1060)


def test_tree_attention_refuses(gpu):
    q = torch.zeros(2, 4, 3, 64, device=gpu, dtype=torch.bfloat16)
    kv = torch.zeros(2, 32, 2, 64, device=gpu, dtype=torch.bfloat16)
    n = torch.zeros(2, device=gpu, dtype=torch.int64)
    tree = torch.ones(3, 3, device=gpu, dtype=torch.bool)
    mask = torch.zeros(2, 1, 1, 32, device=gpu)
    run = backends.hip_tree_attention
    for bad in (
        lambda: run(q[0], kv, kv, n, tree, scale=1.0),
        lambda: run(q, kv[0], kv[0], n, tree, scale=1.0),
        lambda: run(q, kv, kv[:, :16], n, tree, scale=1.0),
        lambda: run(q, kv[:1], kv[:1], n, tree, scale=1.0),
        lambda: run(q[:, :3], kv, kv, n, tree, scale=1.0),
        lambda: run(q[..., :32], kv, kv, n, tree, scale=1.0),
        lambda: run(q.half(), kv, kv, n, tree, scale=1.0),
        lambda: run(q.double(), kv.double(), kv.double(), n, tree, scale=1.0),
        lambda: run(q, kv, kv, n.float(), tree, scale=1.0),
        lambda: run(q, kv, kv, n[:1], tree, scale=1.0),
        lambda: run(q, kv, kv, n, tree.float(), scale=1.0),
        lambda: run(q, kv, kv, n, tree[:2], scale=1.0),
        lambda: run(q, kv, kv, n, tree.expand(3, 3, 3), scale=1.0),
        lambda: run(q, kv, kv, n, tree.cpu(), scale=1.0),
        lambda: run(q, kv, kv, n, tree, mask.long(), scale=1.0),
        lambda: run(q, kv, kv, n, tree, mask[:1], scale=1.0),
        lambda: run(q, kv, kv, n, tree, torch.zeros(2, 1, 1, 33, device=gpu), scale=1.0),
        lambda: run(q, kv, kv, n, tree, scale=0.0),
        lambda: run(q, kv, kv, n, tree, scale=NAN),
        lambda: run(q.transpose(2, 3), kv[..., :3], kv[..., :3], n, None, scale=1.0),
        lambda: run(q, kv, kv.transpose(1, 2).contiguous().transpose(1, 2), n, tree, scale=1.0),
        lambda: backends.hip_paged_tree_attention(q, kv, kv, torch.zeros(2, 2, device=gpu), n, tree, scale=1.0),
        lambda: backends.hip_paged_tree_attention(q, kv, kv, torch.zeros(2, 0, device=gpu, dtype=torch.int32), n, tree,
                                                  scale=1.0),
    ):
        with pytest.raises(ValueError):
            bad()
    assert run(q[:0], kv[:0], kv[:0], n[:0], tree, scale=1.0).shape == (0, 4, 3, 64)
    assert run(q[:, :, :0], kv, kv, n, None, scale=1.0).shape == (2, 4, 0, 64)


# ---- verification -------------------------------------------------------------------


def verify_reference(tokens, target, uniforms, parents=None, draft=None):
    """The documented walk, a node at a time in 64 bits; also how near the closest
    comparison came to its border, relative to its sides."""

    batch, nodes, vocab = target.shape
    paths, emitted, counts = [], [], []
    for b in range(batch):
        up = list(range(-1, nodes - 1)) if parents is None else parents[b].tolist()
        path = [0]
        while True:
            node = path[-1]
            p = target[b, node].double().nan_to_num(0.0).clamp_min(0)
            w, m, mass, follows = p.clone(), 1.0, 0.0, None
            for c in (c for c in range(node + 1, nodes) if up[c] == node):
                x, u = int(tokens[b, c]), float(uniforms[b, c])
                chance = float(w[x]) if 0 <= x < vocab else 0.0
                if draft is None:
                    accepted = u * m < chance and chance > 0
                else:
                    accepted = u * m * (float(draft[b, node, x]) if 0 <= x < vocab else 0.0) < chance
                if accepted:
                    follows = c
                    break
                if draft is None:
                    m -= chance
                    if 0 <= x < vocab:
                        w[x] = 0.0
                else:
                    mass += m
                    w = (p - mass * draft[b, node].double()).clamp_min(0)
                    m = float(w.sum())
            if follows is None:
                break
            path.append(follows)
        if not float(w.sum()) > 0:
            w = p
        sums = w.cumsum(0)
        drawn = int((sums <= float(uniforms[b, 0]) * sums[-1]).sum()) if float(sums[-1]) > 0 else -1
        fill = [-1] * (nodes - len(path))
        paths.append(path + fill)
        emitted.append([int(tokens[b, c]) for c in path[1:]] + [drawn] + fill)
        counts.append(len(path))
    return tuple(torch.tensor(v) for v in (paths, emitted, counts))


def check_verify(gpu, tokens, target, uniforms, parents=None, draft=None):
    want = verify_reference(tokens, target, uniforms, parents, draft)
    got = backends.hip_verify_tokens(tokens.to(gpu), target.to(gpu), uniforms.to(gpu),
                                     parents=None if parents is None else parents.to(gpu),
                                     draft_probs=None if draft is None else draft.to(gpu))
    for a, b in zip(got, want):
        assert a.dtype == torch.int64
        assert torch.equal(a.cpu(), b)
    return want


def random_parents(batch, nodes, g, back=4):
    parents = torch.full((batch, nodes), -1)
    for c in range(1, nodes):
        parents[:, c] = torch.randint(max(0, c - back), c, (batch,), generator=g)
    return parents


def probabilities(g, *shape, dtype=torch.float32, sharp=3.0):
    return torch.softmax(torch.randn(*shape, generator=g) * sharp, -1).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("batch,nodes,vocab", [(1, 5, 151936), (3, 1, 1000), (2, 9, 1024), (7, 4, 1025), (4, 17, 33),
                                               (2, 3, 1), (5, 2, 4099), (40, 6, 2048), (2, 70, 300)])
def test_verify_chains(gpu, batch, nodes, vocab, dtype):
    announce(f"verify chains {batch} {nodes} {vocab} {dtype}")
    g = generator(vocab + nodes)
    for turn in range(3):
        logits = torch.randn(batch, nodes, vocab, generator=g) * 3
        target = torch.softmax(logits, -1).to(dtype)
        draft = torch.softmax(logits + 0.7 * torch.randn(batch, nodes, vocab, generator=g), -1).to(dtype)[:, : nodes - 1]
        tokens = torch.zeros(batch, nodes, dtype=torch.int64)
        if nodes > 1:
            tokens[:, 1:] = torch.multinomial(draft.float().reshape(-1, vocab), 1, generator=g).view(batch, -1)
        check_verify(gpu, tokens, target, torch.rand(batch, nodes, generator=g), draft=draft)
        check_verify(gpu, tokens, target, torch.rand(batch, nodes, generator=g))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("batch,nodes,vocab", [(4, 12, 50), (3, 64, 2000), (2, 65, 1100), (2, 200, 40), (1, 30, 151936)])
def test_verify_trees(gpu, batch, nodes, vocab, with_draft, dtype):
    announce(f"verify trees {batch} {nodes} {vocab} {with_draft} {dtype}")
    g = generator(nodes)
    for back in (2, 8, nodes):
        parents = random_parents(batch, nodes, g, back)
        target, draft = (probabilities(g, batch, nodes, vocab, dtype=dtype) for _ in range(2))
        draft = ((draft.float() + target.float()) / 2).to(dtype)[:, : nodes - 1]
        at = parents.clamp_min(0).clamp_max(nodes - 2)
        rows = draft.float()[torch.arange(batch).unsqueeze(1), at]
        tokens = torch.multinomial(rows.view(-1, vocab), 1, generator=g).view(batch, nodes)
        check_verify(gpu, tokens, target, torch.rand(batch, nodes, generator=g), parents, draft if with_draft else None)


def test_verify_at_borders(gpu):
    announce("verify borders")
    # Whole multiples of powers of two: every sum and product is exact, ties are real.
    vocab, nodes = 4096, 3
    target = torch.full((6, nodes, vocab), 1 / vocab)
    draft = torch.full((6, nodes - 1, vocab), 1 / vocab)
    draft[:, :, :2] = torch.tensor([2 / vocab, 0.0])
    tokens = torch.tensor([[9, 0, 5]] * 6)
    uniforms = torch.tensor([[0.0, 0.5, 0.0], [0.5, 0.499, 0.99], [0.25, 0.0, 0.0], [0.999, 0.5, 0.5],
                             [1 - 2**-24, 0.0, 0.5], [0.75, 0.75, 0.75]])
    want = check_verify(gpu, tokens, target, uniforms, draft=draft)
    assert want[2].tolist() == [1, 3, 3, 1, 3, 1]  # u q < p, not <=
    assert want[1][0, 0] == 1  # only token 1 is left
    assert want[1][1].tolist() == [0, 5, vocab // 2]  # the first sum past one half
    # Without a draft: u < p.
    want = check_verify(gpu, tokens, target, torch.tensor([[0.5, 1 / vocab, 0.0], [0.0, 0.0, 1 / vocab]] * 3))
    assert want[2].tolist() == [1, 2] * 3
    assert want[1][0, 0] == vocab // 2  # of the 4095 that are left


def test_verify_odd_probabilities(gpu):
    announce("verify odd probabilities")
    g = generator(2)
    batch, nodes, vocab = 8, 4, 1500
    target = probabilities(g, batch, nodes, vocab)
    draft = probabilities(g, batch, nodes - 1, vocab)
    tokens = torch.randint(0, vocab, (batch, nodes), generator=g)
    uniforms = torch.rand(batch, nodes, generator=g)
    # Tokens outside the vocabulary are refused, NaN has no weight, a draft that is the target leaves none.
    tokens[0, 1], tokens[1, 1], tokens[2, 2], tokens[3, 1] = -1, vocab, 2**40, -(2**40)
    target[4, 0, 3:7] = NAN
    tokens[4, 1] = 4
    draft[5] = target[5, : nodes - 1]
    draft[5, :, 17] = target[5, : nodes - 1, 17] = 0.0
    tokens[5, 1:] = 17  # never accepted, and then nothing is left: the target is drawn from
    target[6] = 0.0  # no probability at all: -1
    target[7, :, : vocab - 1] = 0.0
    target[7, :, vocab - 1] = 1.0
    for d in (None, draft):
        want = check_verify(gpu, tokens, target, uniforms, draft=d)
        assert want[1][6, 0] == -1
        assert want[2][:4].tolist()[:2] == [1, 1]


def test_verify_padding_and_duplicates(gpu):
    announce("verify padding and duplicates")
    g = generator(4)
    batch, nodes, vocab = 6, 7, 20
    target = probabilities(g, batch, nodes, vocab, sharp=1.0)
    # A node that is no earlier one's child is never reached: -1, itself, a later one, far ones.
    parents = torch.tensor([[-1, 0, 0, 0, 0, 0, 0], [5, -1, 0, 2, -1, 2, 2], [0, 1, 2, 3, 4, 5, 6],
                            [0, 0, 1, 2, 6, 6, 5], [-1, -1, -1, -1, -1, -1, -1], [-1, 2**40, 0, -(2**40), 2, 4, 7]])
    tokens = torch.randint(0, vocab, (batch, nodes), generator=g)
    tokens[0] = torch.tensor([1, 3, 3, 3, 5, 5, 3])  # one token three times among the children
    target[0, 0] = 0.0
    target[0, 0, 3], target[0, 0, 5], target[0, 0, 11] = 0.25, 0.25, 0.5
    draft = probabilities(g, batch, nodes - 1, vocab, sharp=1.0)
    for turn in range(8):
        uniforms = torch.rand(batch, nodes, generator=g)
        check_verify(gpu, tokens, target, uniforms, parents)
        check_verify(gpu, tokens, target, uniforms, parents, draft)


def test_verify_widest_trees(gpu):
    announce("verify 1024 nodes")
    g = generator(6)
    target = probabilities(g, 1, 1024, 700, sharp=1.0)
    uniforms = torch.rand(1, 1024, generator=g)
    star = torch.zeros(1, 1024, dtype=torch.int64)
    star[0, 0] = -1
    tokens = torch.randint(0, 700, (1, 1024), generator=g)
    check_verify(gpu, tokens, target, uniforms, star)
    # A chain of all of them, accepted throughout.
    sure = torch.zeros(1, 1024, 700)
    sure[0, torch.arange(1023), tokens[0, 1:]] = 1.0
    sure[0, 1023, 699] = 1.0
    want = check_verify(gpu, tokens, sure, uniforms)
    assert want[2].item() == 1024 and want[1][0, -1] == 699


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("drafted", [False, True])
def test_verify_draws_a_token_with_weight_at_a_border_between_sums(gpu, drafted, dtype):
    """A goal of half the sum, next to which the order of additions decides on which side
    of it a block's sum lies, with blocks of no weight behind: what is drawn has weight."""

    announce(f"verify border between sums {drafted} {dtype}")
    # Vocabularies of up to 256 blocks of 1024, and more than 256.
    for blocks, small, last in ((13, (4, 5), 12), (64, (12, 13, 14), 63), (300, (255, 256, 257), 299), (300, (4, 5), 299)):
        for few in range(1, len(small) + 1):
            for power in (-53, -54, -55, -56):
                target = torch.zeros(1, 2, blocks * 1024, dtype=torch.float64)
                target[:, :, 7] = target[:, :, last * 1024 + 9] = 0.5
                for block in small[:few]:
                    target[:, :, block * 1024 + 3] = 2.0**power
                target = target.to(dtype)
                draft = torch.zeros(1, 1, blocks * 1024, dtype=dtype)
                draft[:, :, 5] = 1.0  # a token that the target does not give: what it leaves is the target
                tokens = torch.tensor([[0, 5]], device=gpu)
                _, emitted, counts = backends.hip_verify_tokens(
                    tokens, target.to(gpu), torch.tensor([[0.5, 0.5]], device=gpu),
                    draft_probs=draft.to(gpu) if drafted else None)
                assert counts.tolist() == [1]
                token = int(emitted[0, 0])
                assert token >= 0 and float(target[0, 0, token]) > 0, (blocks, few, power, token)


@pytest.mark.parametrize("nodes", [5, 64, 65, 130])
def test_verify_siblings_without_a_probability(gpu, nodes):
    """A refused sibling's NaN or negative probability takes nothing from the mass that
    the younger ones are tried with."""

    announce(f"verify siblings without a probability {nodes}")
    g = generator(nodes)
    vocab = 1100
    rows = []
    for odd in (NAN, -0.25, -INF, 0.0):
        target = probabilities(g, 1, nodes, vocab, sharp=1.0)
        target[0, 0] = 0.0
        target[0, 0, 3], target[0, 0, 5], target[0, 0, 7], target[0, 0, 11] = odd, 0.25, 0.5, 0.25
        rows.append(target)
    target = torch.cat(rows)
    parents = torch.zeros(4, nodes, dtype=torch.int64)
    parents[:, 0] = -1
    tokens = torch.full((4, nodes), 3)  # the first, and all between the tried ones and behind them
    tokens[:, nodes // 2], tokens[:, nodes - 1] = 5, 7
    # 0.5 of the 0.75 that the refusal of token 5 leaves is 2 / 3, of 1 one half.
    for first, second, count in ((0.5, 0.66, 2), (0.5, 0.67, 1), (0.2, 0.9, 2), (0.25, 0.5, 2), (0.26, 0.999, 1)):
        uniforms = torch.full((4, nodes), 0.5)
        uniforms[:, nodes // 2], uniforms[:, nodes - 1] = first, second
        want = check_verify(gpu, tokens, target, uniforms, parents)
        assert want[2].tolist() == [count] * 4


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("nodes", [6, 70])
def test_verify_draft_probabilities_that_are_none(gpu, nodes, dtype):
    """NaN and negative draft probabilities count as zero: a token without weight is not
    accepted by them, and they take nothing from the target's and add nothing to it."""

    announce(f"verify draft probabilities that are none {nodes} {dtype}")
    g = generator(nodes)
    vocab, batch = 1500, 6
    target = probabilities(g, batch, nodes, vocab).to(dtype)
    draft = probabilities(g, batch, nodes - 1, vocab).to(dtype)
    odd = torch.rand(draft.shape, generator=g)
    draft[odd < 0.2] = NAN
    draft[(odd >= 0.2) & (odd < 0.4)] = -0.5
    tokens = torch.randint(0, vocab, (batch, nodes), generator=g)
    # Tokens without weight whose draft probability is negative or NaN, first among the children.
    target[:3, 0, 17], draft[:2, 0, 17], draft[2, 0, 17] = 0.0, -0.25, NAN
    tokens[:3, 1] = 17
    clean = draft.float().nan_to_num(0.0).clamp_min(0.0).to(dtype)
    for parents in (None, random_parents(batch, nodes, g)):
        for turn in range(4):
            uniforms = torch.rand(batch, nodes, generator=g).clamp_min(2.0**-20)
            want = verify_reference(tokens, target, uniforms, parents, clean)
            got = backends.hip_verify_tokens(tokens.to(gpu), target.to(gpu), uniforms.to(gpu),
                                             parents=None if parents is None else parents.to(gpu),
                                             draft_probs=draft.to(gpu))
            for a, b in zip(got, want):
                assert torch.equal(a.cpu(), b)
            if parents is None:
                assert want[2][:3].tolist() == [1] * 3


def test_verify_layouts_streams_and_graphs(gpu):
    announce("verify layouts")
    g = generator(7)
    batch, nodes, vocab = 5, 6, 5003
    target, draft = probabilities(g, batch, nodes, vocab), probabilities(g, batch, nodes - 1, vocab)
    tokens = torch.randint(0, vocab, (batch, nodes), generator=g)
    uniforms = torch.rand(batch, nodes, generator=g)
    want = check_verify(gpu, tokens, target, uniforms, draft=draft)
    wide = torch.full((batch, nodes + 1, vocab + 9), NAN, device=gpu)
    wide[:, :nodes, 3 : vocab + 3] = target.to(gpu)
    views = (tokens.to(gpu).t().contiguous().t(), wide[:, :nodes, 3 : vocab + 3], uniforms.to(gpu).t().contiguous().t())
    workspace = _native.DeviceWorkspace(gpu)
    for _ in range(3):
        got = backends.hip_verify_tokens(*views, draft_probs=draft.to(gpu), workspace=workspace)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))
    streams = [torch.cuda.Stream() for _ in range(2)]
    draft_gpu, results = draft.to(gpu), []
    for stream in streams * 2:
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            results.append(backends.hip_verify_tokens(*views, draft_probs=draft_gpu))
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))
    static = [tokens.to(gpu), target.to(gpu), uniforms.to(gpu)]
    backends.hip_verify_tokens(*static, draft_probs=draft_gpu, workspace=workspace)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = backends.hip_verify_tokens(*static, draft_probs=draft_gpu, workspace=workspace)
    for turn in range(4):
        static[2].copy_(torch.rand(batch, nodes, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        expected = verify_reference(tokens, target, static[2].cpu(), None, draft)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, expected))


def test_verify_gives_the_targets_distribution(gpu):
    """The first emitted token of 2^18 independent steps, with children drawn from the draft.

    For a token of probability p the count is binomial; 6 standard deviations, plus 2^-12 of
    the steps for fp32 probabilities that do not sum to 1 exactly, are passed by chance about
    once in 10^8 tokens."""

    announce("verify distribution")
    g = generator(21)
    steps, vocab, children = 2**18, 12, 3
    p, q = (torch.softmax(torch.randn(vocab, generator=g), -1) for _ in range(2))
    nodes = 1 + children
    tokens = torch.zeros(steps, nodes, dtype=torch.int64)
    tokens[:, 1:] = torch.multinomial(q, steps * children, replacement=True, generator=g).view(steps, children)
    parents = torch.tensor([-1] + [0] * children).expand(steps, -1)
    uniforms = torch.rand(steps, nodes, generator=g)
    target = p.expand(steps, nodes, vocab).to(gpu)
    draft = q.expand(steps, nodes - 1, vocab).to(gpu)
    for d in (None, draft):
        counts = torch.zeros(vocab, dtype=torch.int64)
        for first in range(0, steps, 2**15):
            part = slice(first, first + 2**15)
            emitted = backends.hip_verify_tokens(tokens[part].to(gpu), target[part], uniforms[part].to(gpu),
                                                 parents=parents[part].to(gpu),
                                                 draft_probs=None if d is None else d[part])[1]
            counts += torch.bincount(emitted[:, 0].cpu(), minlength=vocab)
        deviation = (steps * p.double() * (1 - p.double())).sqrt()
        assert ((counts - steps * p.double()).abs() <= 6 * deviation + steps * 2.0**-12).all()


def test_verify_offsets_past_32_bits(gpu):
    """A vocabulary of 2^24 + 8 and 2^31 probabilities and more."""

    announce("verify offsets past 32 bits")
    nodes, vocab = 64, 2**24 + 8
    target = torch.zeros(2, nodes, vocab, dtype=torch.float16, device=gpu)
    tokens = torch.randint(0, vocab, (2, nodes), generator=generator(3))
    target[0, 0, 7] = 1.0
    target[1, torch.arange(nodes - 1), tokens[1, 1:]] = 1.0
    target[1, -1, 5], target[1, -1, 2**24] = 0.25, 0.75
    uniforms = torch.full((2, nodes), 0.5, device=gpu)
    path, emitted, counts = backends.hip_verify_tokens(tokens.to(gpu), target, uniforms)
    assert counts.tolist() == [1, nodes] and emitted[0, 0].item() == 7
    assert emitted[1].tolist() == tokens[1, 1:].tolist() + [2**24]
    # And with draft rows, those of another token: the leftover is the target's.
    draft = torch.zeros_like(target[:, : nodes - 1])
    draft[..., vocab - 1] = 1.0
    tokens[:] = vocab - 1
    path, emitted, counts = backends.hip_verify_tokens(tokens.to(gpu), target.flip(0), uniforms, draft_probs=draft)
    assert counts.tolist() == [1, 1] and emitted[1, 0].item() == 7
    assert path.tolist() == [[0] + [-1] * (nodes - 1)] * 2


def test_verify_refuses(gpu):
    tokens = torch.zeros(2, 3, device=gpu, dtype=torch.int64)
    target, uniforms = torch.ones(2, 3, 5, device=gpu), torch.zeros(2, 3, device=gpu)
    run = backends.hip_verify_tokens
    for bad in (
        lambda: run(tokens.int(), target, uniforms),
        lambda: run(tokens[0], target, uniforms),
        lambda: run(tokens[:, :0], target[:, :0], uniforms[:, :0]),
        lambda: run(tokens, target[:, :2], uniforms),
        lambda: run(tokens, target[..., :0], uniforms),
        lambda: run(tokens, target.double(), uniforms),
        lambda: run(tokens, target, uniforms.double()),
        lambda: run(tokens, target, uniforms[:1]),
        lambda: run(tokens, target, uniforms, parents=tokens.int()),
        lambda: run(tokens, target, uniforms, parents=tokens[:, :2]),
        lambda: run(tokens, target, uniforms, draft_probs=target),
        lambda: run(tokens, target, uniforms, draft_probs=target[:, :2].half()),
        lambda: run(tokens, target, uniforms.cpu()),
        lambda: run(torch.zeros(1, 1025, device=gpu, dtype=torch.int64), torch.ones(1, 1025, 1, device=gpu),
                    torch.zeros(1, 1025, device=gpu)),
    ):
        with pytest.raises(ValueError):
            bad()
    assert [t.shape for t in run(tokens[:0], target[:0], uniforms[:0])] == [(0, 3), (0, 3), (0,)]


# ---- commit -------------------------------------------------------------------------


def commit_reference(buffers, lengths, path, counts):
    """Buffers [B, Cap, H, D] of one layer after the moves."""

    moved = [buffer.clone() for buffer in buffers]
    capacity = buffers[0].shape[1]
    for b in range(path.shape[0]):
        n = int(lengths[b])
        for j in range(int(counts[b])):
            if j < int(path[b, j]) and n + int(path[b, j]) < capacity:
                for old, new in zip(buffers, moved):
                    new[b, n + j] = old[b, n + int(path[b, j])]
    return moved


def random_paths(g, batch, nodes):
    path, counts = torch.full((batch, nodes), -1), torch.randint(1, nodes + 1, (batch,), generator=g)
    for b in range(batch):
        rest = torch.randperm(nodes - 1, generator=g)[: int(counts[b]) - 1] + 1
        path[b, : int(counts[b])] = torch.cat([torch.zeros(1, dtype=torch.int64), rest.sort().values])
    return path, counts


def bits(tensor):
    return tensor.view({2: torch.int16, 4: torch.int32}[tensor.element_size()])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layers,batch,nodes,heads,head_dim,capacity,page_tokens", [
    (24, 3, 8, 2, 64, 100, 0), (2, 5, 64, 2, 64, 256, 64), (3, 2, 5, 3, 33, 64, 16), (1, 1, 1, 1, 1, 4, 0),
    (100, 2, 6, 1, 8, 40, 0), (2, 2, 200, 16, 128, 512, 32), (1, 70, 3, 2, 80, 32, 16), (2, 1, 1024, 2, 6, 1100, 0)])
def test_commit(gpu, layers, batch, nodes, heads, head_dim, capacity, page_tokens, dtype):
    announce(f"commit {layers} {batch} {nodes} {heads} {head_dim} {page_tokens} {dtype}")
    g = generator(layers + nodes)
    whole = -(-capacity // max(1, page_tokens)) * max(1, page_tokens)
    keys, values = ([torch.randn(batch, whole, heads, head_dim, generator=g).to(dtype) for _ in range(layers)]
                    for _ in range(2))
    lengths = torch.randint(0, capacity - nodes + 1, (layers, batch), generator=g)
    path, counts = random_paths(g, batch, nodes)
    table = None
    if page_tokens:
        order = torch.randperm(batch * whole // page_tokens, generator=g).view(batch, -1)
        table = order.to(torch.int32).to(gpu)

        def place(buffer):
            pool = torch.empty(order.numel(), page_tokens, heads, head_dim, dtype=dtype)
            pool[order.view(-1)] = buffer.view(order.numel(), page_tokens, heads, head_dim)
            return pool.to(gpu)

        def back(pool):
            return pool.cpu()[order].reshape(batch, whole, heads, head_dim)
    else:
        def place(buffer):
            return buffer.to(gpu)

        def back(buffer):
            return buffer.cpu()

    on_gpu = [place(buffer) for buffer in keys + values]
    handle = backends.KVLayers(on_gpu[:layers], on_gpu[layers:], block_table=table)
    out = backends.hip_kv_commit(handle, lengths.to(gpu), path.to(gpu), counts.to(gpu))
    assert torch.equal(out.cpu(), lengths + counts)
    for layer in range(layers):
        want = commit_reference([keys[layer], values[layer]], lengths[layer], path, counts)
        for got, expected in zip((on_gpu[layer], on_gpu[layers + layer]), want):
            assert torch.equal(bits(back(got)), bits(expected))


def test_commit_forms_of_lengths(gpu):
    announce("commit lengths")
    g = generator(1)
    buffers = [torch.randn(2, 20, 2, 8, generator=g).to(gpu) for _ in range(6)]
    handle = backends.KVLayers(buffers[:3], buffers[3:])
    path, counts = torch.tensor([[0, 1, 2], [0, 1, -1]], device=gpu), torch.tensor([3, 2], device=gpu)
    one = torch.tensor([4, 17], device=gpu)
    run = backends.hip_kv_commit
    assert run(handle, one, path, counts).tolist() == [7, 19] and one.tolist() == [4, 17]
    each = [one.clone() for _ in range(3)]
    assert [t.tolist() for t in run(handle, each, path, counts)] == [[7, 19]] * 3
    assert run(handle, [one] * 3, path, counts, out=each) is each
    assert [t.tolist() for t in each] == [[7, 19]] * 3
    flag = torch.zeros(1, dtype=torch.int32, device=gpu)
    assert run(handle, each, path, counts, out=each, overflow=flag) is each
    assert [t.tolist() for t in each] == [[10, 21]] * 3 and flag.item() == 1  # past the capacity of 20
    stacked = one.repeat(3, 1)
    flag.zero_()
    run(handle, stacked, path, counts, out=stacked, overflow=flag)
    assert stacked.tolist() == [[7, 19]] * 3 and flag.item() == 0
    # Counts outside the path, and none at all.
    assert run(handle, one, path, torch.tensor([-3, 99], device=gpu)).tolist() == [4, 20]
    before = [t.clone() for t in buffers]
    assert run(handle, one, path, torch.zeros_like(counts)).tolist() == [4, 17]
    assert all(torch.equal(a, b) for a, b in zip(before, buffers))
    for bad in (
        lambda: run(handle, one, path, counts, out=one),  # three layers read it
        lambda: run(handle, [one] * 3, path, counts, out=[one, each[1], each[2]]),
        lambda: run(handle, each, path, counts, out=[each[1], each[0], each[2]]),
        lambda: run(handle, each, path, counts, out=[each[0], each[0], each[2]]),
        lambda: run(handle, each[:2], path, counts),
        lambda: run(handle, one.int(), path, counts),
        lambda: run(handle, one[:1], path, counts),
        lambda: run(handle, one, path.int(), counts),
        lambda: run(handle, one, path[:1], counts),
        lambda: run(handle, one, path[:, :0], counts),
        lambda: run(handle, one, path, counts.int()),
        lambda: run(handle, one, path, counts.cpu()),
        lambda: run(handle, one, path, counts, overflow=torch.zeros(1, device=gpu)),
        lambda: run(handle, one, path, counts, out=torch.zeros(5, dtype=torch.int64, device=gpu)[1:3:1].int()),
        lambda: backends.KVLayers(buffers[:3], buffers[:3]),
        lambda: backends.KVLayers(buffers[:3], buffers[3:5]),
        lambda: backends.KVLayers([], []),
        lambda: backends.KVLayers(buffers[:1], [buffers[1].half()]),
        lambda: backends.KVLayers(buffers[:1], [buffers[1][:, :10]]),
        lambda: backends.KVLayers([buffers[0].cpu()], [buffers[1].cpu()]),
        lambda: backends.KVLayers(buffers[:1], buffers[1:2], block_table=torch.zeros(1, 1, device=gpu)),
    ):
        with pytest.raises(ValueError):
            bad()
    lap = torch.zeros(7, dtype=torch.int64, device=gpu)
    with pytest.raises(ValueError):  # views that overlap in part
        run(handle, each, path, counts, out=[lap[0:2], lap[1:3], lap[4:6]])


def test_commit_refuses_outputs_over_its_inputs(gpu):
    announce("commit over its inputs")
    buffers = [torch.zeros(2, 20, 2, 8, device=gpu) for _ in range(4)]
    handle = backends.KVLayers(buffers[:2], buffers[2:])
    path = torch.zeros(2, 3, dtype=torch.int64, device=gpu)
    room = torch.zeros(5, dtype=torch.int64, device=gpu)
    lengths, counts = torch.zeros(2, dtype=torch.int64, device=gpu), room[1:3]
    for out in (counts, room[0:2], room[2:4], path[0, :2], path[1, 1:]):
        with pytest.raises(ValueError):
            backends.hip_kv_commit(handle, lengths, path, counts, out=out)
    assert backends.hip_kv_commit(handle, lengths, path, counts, out=room[3:5]).tolist() == [0, 0]
    with pytest.raises(ValueError):  # one sequence's rows for all
        backends.KVLayers([buffers[0][:1].expand(2, -1, -1, -1)], [buffers[1][:1].expand(2, -1, -1, -1)])


def test_commit_does_not_leave_the_cache(gpu):
    announce("commit bounds")
    # Entries that are no node, sources past the capacity, pages that are none of the pool's.
    buffers = [torch.arange(2 * 16.0, device=gpu).view(2, 16, 1, 1).clone() for _ in range(2)]
    handle = backends.KVLayers(buffers[:1], buffers[1:])
    path = torch.tensor([[0, 3, 2**40, -(2**40)], [1, 2, 3, 3]], device=gpu)
    lengths = torch.tensor([13, 2], device=gpu)
    out = backends.hip_kv_commit(handle, lengths, path, torch.tensor([4, 3], device=gpu))
    assert out.tolist() == [17, 5]
    want = torch.arange(2 * 16.0).view(2, 16)
    want[1, 2:5] = torch.tensor([19.0, 20.0, 21.0])
    assert all(torch.equal(b.cpu().view(2, 16), want) for b in buffers)
    for start in (-1, -(2**40), 16, 2**40):
        backends.hip_kv_commit(handle, torch.tensor([start, start], device=gpu), path,
                               torch.tensor([4, 3], device=gpu))
        assert all(torch.equal(b.cpu().view(2, 16), want) for b in buffers)
    pools = [torch.arange(3 * 16.0, device=gpu).view(3, 16, 1, 1).clone() for _ in range(2)]
    table = torch.tensor([[1, 7], [-1, 2]], dtype=torch.int32, device=gpu)
    handle = backends.KVLayers(pools[:1], pools[1:], block_table=table)
    path = torch.tensor([[0, 2, 3, -1], [0, 2, 3, -1]], device=gpu)
    backends.hip_kv_commit(handle, torch.tensor([13, 14], device=gpu), path, torch.tensor([3, 3], device=gpu))
    want = torch.arange(3 * 16.0).view(3, 16)
    want[1, 14] = want[1, 15]  # row 15 to 14 of the first sequence; its row 16 has no page
    want[2, 0] = want[2, 1]  # row 17 to 16 of the second; row 15 has no page
    assert all(torch.equal(p.cpu().view(3, 16), want) for p in pools)
    out = backends.hip_paged_tree_attention(
        torch.ones(2, 1, 4, 1, device=gpu), *pools, table, torch.tensor([10, 20], device=gpu), None, scale=1.0)
    assert out.shape == (2, 1, 4, 1)


@pytest.mark.parametrize("page_tokens", [0, 16])
def test_commit_of_lengths_next_to_the_largest_integer(gpu, page_tokens):
    """A length whose sum with a node passes 64 bits moves nothing."""

    announce(f"commit far lengths {page_tokens}")
    shape = (2, 16, 1, 4) if page_tokens else (1, 32, 1, 4)
    buffers = [torch.randn(shape, device=gpu) for _ in range(2)]
    before = [buffer.clone() for buffer in buffers]
    table = torch.tensor([[0, 1]], dtype=torch.int32, device=gpu) if page_tokens else None
    handle = backends.KVLayers(buffers[:1], buffers[1:], block_table=table)
    path, counts = torch.tensor([[0, 2, 3]], device=gpu), torch.tensor([3], device=gpu)
    flag = torch.zeros(1, dtype=torch.int32, device=gpu)
    for length in (2**63 - 1, 2**63 - 2, 2**63 - 3, 2**63 - 4, 2**62, -(2**63)):
        flag.zero_()
        backends.hip_kv_commit(handle, torch.tensor([length], device=gpu), path, counts, overflow=flag)
        assert flag.item() == 1
        assert all(torch.equal(a, b) for a, b in zip(buffers, before))


def test_commit_flags_rows_that_are_not_moved(gpu):
    """Accepted nodes whose rows were not stored, or whose places are none of the pool's,
    and counts that no path has set the flag; all else leaves it."""

    announce("commit flag")
    flag = torch.zeros(1, dtype=torch.int32, device=gpu)

    def flagged(handle, length, path, count):
        flag.zero_()
        batch = handle.batch
        lengths = torch.full((batch,), 2, device=gpu)
        lengths[-1] = length
        paths = torch.tensor([[0] + [-1] * (len(path) - 1)] * (batch - 1) + [path], device=gpu)
        counts = torch.ones(batch, dtype=torch.int64, device=gpu)
        counts[-1] = count
        out = backends.hip_kv_commit(handle, lengths, paths, counts, overflow=flag)
        assert int(out[-1]) == length + max(0, min(count, len(path)))
        return flag.item()

    for batch, layers in ((1, 1), (3, 2)):
        buffers = [torch.arange(batch * 100.0, device=gpu).view(batch, 100, 1, 1).clone() for _ in range(2 * layers)]
        handle = backends.KVLayers(buffers[:layers], buffers[layers:])
        before = buffers[0].clone()
        # Row 97 + 5 was not stored: row 98 keeps what it held, the new length 99 counts it.
        assert flagged(handle, 97, [0, 5, -1, -1, -1, -1], 2) == 1
        assert torch.equal(buffers[0], before)
        assert flagged(handle, 97, [0, 2, -1, -1, -1, -1], 2) == 0  # row 99, the last
        assert flagged(handle, 97, [0, 1, 2, -1, -1, -1], 3) == 0  # as far as the capacity
        assert flagged(handle, 97, [0, 5, 5, 5, 5, 5], 1) == 0  # what is not accepted does not count
        assert flagged(handle, 97, [0, 1, 2, 3, -1, -1], 4) == 1
        assert flagged(handle, 4, [0, 2, 4, -1, -1, -1], 3) == 0
        assert flagged(handle, 4, [0, 2, 4, -1, -1, -1], 0) == 0
        assert flagged(handle, 4, [0, 1, 2, 3, 4, 5], 6) == 0
        assert flagged(handle, 4, [0, 1, 2, 3, 4, 5], 7) == 1  # cut to the path's six
        assert flagged(handle, 4, [0, 1, 2, 3, 4, 5], -1) == 1
        assert flagged(handle, 4, [0, 2, -1, -1, -1, -1], 3) == 1  # the third is no node
        assert flagged(handle, 4, [0, 2, 6, -1, -1, -1], 3) == 1
        assert flagged(handle, 4, [0, 2, 6, -1, -1, -1], 2) == 0
    wide = [-1] * 200
    buffers = [torch.zeros(1, 300, 1, 1, device=gpu) for _ in range(2)]
    handle = backends.KVLayers(buffers[:1], buffers[1:])
    wide[:151] = range(49, 200)
    assert flagged(handle, 101, wide, 150) == 0  # past a wave's 64, to row 101 + 198
    assert flagged(handle, 101, wide, 151) == 1
    pools = [torch.arange(3 * 16.0, device=gpu).view(3, 16, 1, 1).clone() for _ in range(2)]
    table = torch.tensor([[1, 7]], dtype=torch.int32, device=gpu)
    handle = backends.KVLayers(pools[:1], pools[1:], block_table=table)
    assert flagged(handle, 12, [0, 2, 3, -1, -1, -1], 3) == 0
    assert flagged(handle, 12, [0, 2, 4, -1, -1, -1], 3) == 1  # row 16 has no page
    table[0, 1] = -1
    assert flagged(handle, 12, [0, 2, 4, -1, -1, -1], 3) == 1
    table[0, 1] = 0
    assert flagged(handle, 12, [0, 2, 4, -1, -1, -1], 3) == 0


# ---- together -----------------------------------------------------------------------


def model_step(config, weights, state, tokens, depths, tree):
    """Logits behind every node: the decoder's operators over ``state``, nodes stored
    behind the sequences."""

    from stateful_llm_compiler_hip.qwen2 import inverse_frequency

    b = backends
    batch, nodes = tokens.shape
    h = b.hip_embedding(tokens, weights["embed_tokens.weight"])
    start = state.positions(0)
    cosine, sine = b.hip_rope_table(start.unsqueeze(1) + depths, inverse_frequency(config, tokens.device), h.dtype)

    def heads(x, count):
        return x.view(batch, nodes, count, config.head_dim).transpose(1, 2)

    for layer in range(config.num_layers):
        p = f"layers.{layer}."
        x = b.hip_rms_norm(h, weights[p + "input_layernorm.weight"], epsilon=config.rms_norm_eps)
        q, k, v = (b.hip_linear(x, weights[f"{p}self_attn.{n}_proj.weight"], weights[f"{p}self_attn.{n}_proj.bias"])
                   for n in "qkv")
        q, state = state.rope_store(layer, heads(q, config.num_heads), heads(k, config.num_kv_heads),
                                    heads(v, config.num_kv_heads), cosine, sine, state.positions(layer))
        a = state.tree_attention(layer, q, tree, groups=config.groups, scale=config.head_dim**-0.5)
        a = a.transpose(1, 2).reshape(batch, nodes, config.hidden_size)
        h = b.hip_add(h, b.hip_linear(a, weights[p + "self_attn.o_proj.weight"], None))
        x = b.hip_rms_norm(h, weights[p + "post_attention_layernorm.weight"], epsilon=config.rms_norm_eps)
        m = b.hip_swiglu(b.hip_linear(x, weights[p + "mlp.gate_proj.weight"], None),
                         b.hip_linear(x, weights[p + "mlp.up_proj.weight"], None))
        h = b.hip_add(h, b.hip_linear(m, weights[p + "mlp.down_proj.weight"], None))
    h = b.hip_rms_norm(h, weights["norm.weight"], epsilon=config.rms_norm_eps)
    return b.hip_linear(h, weights["embed_tokens.weight"], None)


@pytest.mark.parametrize("page_tokens", [None, 16])
@pytest.mark.parametrize("in_place", [False, True])
def test_drafted_steps_give_the_tokens_of_single_steps(gpu, page_tokens, in_place):
    """Greedy decoding in steps on trees, some of whose nodes are right, gives what the
    runtime gives one token at a time, in fp32."""

    from dataclasses import replace

    from stateful_llm_compiler_hip.qwen2 import Qwen2Config, causal_prefill_mask, init_weights
    from stateful_llm_compiler_hip.runtime import Qwen2Runtime

    announce(f"drafted steps {page_tokens} {in_place}")
    config = Qwen2Config(hidden_size=128, intermediate_size=256, num_layers=3, num_heads=4, num_kv_heads=2,
                         vocab_size=503)
    weights = init_weights(config, seed=3, dtype=torch.float32, device=str(gpu), std=0.3)
    batch, prompt, steps, capacity = 3, 11, 24, 64
    rt = Qwen2Runtime(config, weights, capacity=capacity, dtype=torch.float32, device=str(gpu))
    g = generator(5)
    ids = torch.randint(0, config.vocab_size, (batch, prompt), generator=g).to(gpu)
    mask = causal_prefill_mask(batch, prompt, device=gpu)
    positions = torch.arange(prompt, device=gpu).expand(batch, -1).contiguous()
    logits, state = rt.prefill(ids, mask, positions)
    token = logits[:, -1].argmax(-1, keepdim=True)
    single = [token]
    for step in range(steps + 8):
        zero = torch.zeros(batch, 1, 1, prompt + step + 1, device=gpu)
        logits, state = rt.decode(token, zero, state)
        token = logits[:, -1].argmax(-1, keepdim=True)
        single.append(token)
    single = torch.cat(single, 1).cpu()

    if page_tokens:
        rt = Qwen2Runtime(config, weights, capacity=capacity, dtype=torch.float32, device=str(gpu),
                          page_tokens=page_tokens)
    logits, state = rt.prefill(ids, mask, positions)
    state = replace(state, in_place_lengths=in_place)
    done = [[int(t)] for t in logits[:, -1].argmax(-1)]
    parents = torch.tensor([-1, 0, 0, 1, 2, 2, 5, 6])
    nodes = len(parents)
    tree = torch.eye(nodes, dtype=torch.bool)
    for c in range(1, nodes):
        tree[c] |= tree[parents[c]]
    depths = tree.sum(-1) - 1
    taken = []
    while min(len(d) for d in done) < steps:
        # The branch 0, 2, 5, 6, 7 gets the right tokens up to each depth in turn, the rest wrong ones.
        tokens = torch.randint(0, config.vocab_size, (batch, nodes), generator=g)
        for b in range(batch):
            right = (len(taken) + b) % 5
            tokens[b, 0] = done[b][-1]
            for depth, c in enumerate((2, 5, 6, 7), 1):
                if depth <= right:
                    tokens[b, c] = single[b, min(len(done[b]) - 1 + depth, single.shape[1] - 1)]
        logits = model_step(config, weights, state, tokens.to(gpu), depths.to(gpu), tree.to(gpu))
        sure = torch.nn.functional.one_hot(logits.argmax(-1), config.vocab_size).float()
        path, emitted, counts = backends.hip_verify_tokens(
            tokens.to(gpu), sure, torch.full((batch, nodes), 0.5, device=gpu),
            parents=parents.expand(batch, -1).contiguous().to(gpu))
        state = state.commit(path, counts)
        for b in range(batch):
            done[b] += emitted[b, : counts[b]].tolist()
        taken += counts.tolist()
    state.check_capacity()
    for b in range(batch):
        assert done[b][:steps] == single[b, :steps].tolist()
        assert int(state.lengths[2][b]) == prompt + len(done[b]) - 1
    assert max(taken) == 5 and min(taken) == 1  # paths of all lengths were taken


def test_commit_follows_the_states_block_table(gpu):
    from dataclasses import replace

    from stateful_llm_compiler_hip.execution import PagedKVCacheState

    announce("commit block table")
    template = torch.zeros(1, 1, 1, 8, device=gpu, dtype=torch.bfloat16)
    state = PagedKVCacheState.empty_from_key_template(template, num_layers=2, capacity=32, page_tokens=16)
    path, counts = torch.tensor([[0, 2, -1]], device=gpu), torch.tensor([2], device=gpu)
    state = state.commit(path, counts)
    state = replace(state, block_table=state.block_table.flip(1).contiguous())
    for buffer in state.keys + state.values:
        buffer.copy_(torch.arange(32.0, device=gpu).view(2, 16, 1, 1).expand(2, 16, 1, 8))
    state = state.commit(path, counts)
    page = int(state.block_table[0, 0])
    for buffer in state.keys + state.values:
        want = torch.arange(32.0).view(2, 16)
        want[page, 3] = want[page, 4]  # row 2 + 2 to row 2 + 1
        assert torch.equal(buffer[:, :, 0, 0].float().cpu(), want)
    assert state.lengths[1].item() == 4


def test_a_captured_step_goes_on_at_every_replay(gpu):
    """Attention, verification and the commit in place, captured on a workspace that is
    new, and with another graph on the same one, replayed among eager steps."""

    from dataclasses import replace

    from stateful_llm_compiler_hip.execution import PreallocatedKVCacheState

    announce("captured step")
    g = generator(41)
    batch, nodes, vocab, capacity, layers = 3, 7, 900, 400, 2
    tree = random_tree(nodes, g)
    parents = torch.tensor([-1] + [int(tree[c, :c].nonzero().max()) for c in range(1, nodes)])
    tree, parents = tree.to(gpu), parents.expand(batch, -1).contiguous().to(gpu)
    query = torch.randn(batch, 8, nodes, 64, generator=g).to(gpu, torch.bfloat16)
    template = torch.zeros(batch, 2, 1, 64, device=gpu, dtype=torch.bfloat16)
    tokens = torch.randint(0, vocab, (batch, nodes), generator=g).to(gpu)
    target = probabilities(g, batch, nodes, vocab).to(gpu)
    target[torch.arange(batch).unsqueeze(1), parents.clamp_min(0), tokens] += 0.5
    uniforms = torch.rand(batch, nodes, generator=g).to(gpu)

    def state_of(workspace):
        state = PreallocatedKVCacheState.empty_from_key_template(template, num_layers=layers, capacity=capacity)
        start = torch.tensor([300, 0, 17], device=gpu)
        state = replace(state, in_place_lengths=True, workspace=workspace, lengths=tuple(start.clone() for _ in range(layers)),
                        zero_slots=frozenset())
        for buffer, seed in zip(state.keys + state.values, range(2 * layers)):
            buffer.copy_(torch.randn(buffer.shape, generator=generator(seed)))
        return state

    def step(state, workspace):
        outs = [state.tree_attention(slot, query, tree, groups=4, scale=0.125) for slot in range(layers)]
        path, emitted, counts = backends.hip_verify_tokens(tokens, target, uniforms, parents=parents, workspace=workspace)
        state.commit(path, counts)
        return outs + [path, emitted, counts]

    eager_workspace, workspace = _native.DeviceWorkspace(gpu), _native.DeviceWorkspace(gpu)
    eager, captured, other = state_of(eager_workspace), state_of(workspace), state_of(workspace)
    graphs = []
    for state in (captured, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(state, workspace)
        graphs.append((graph, outs, state))
    for turn in range(5):
        uniforms.copy_(torch.rand(batch, nodes, generator=g))
        want = step(eager, eager_workspace)
        for graph, outs, state in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, outs, state in graphs:
            for got, expected in zip(outs, want):
                assert torch.equal(got, expected)
            for got, expected in zip(state.lengths + state.keys + state.values, eager.lengths + eager.keys + eager.values):
                assert torch.equal(got, expected)
    assert eager.lengths[0].tolist() != [300, 0, 17]


@pytest.mark.parametrize("shared", [False, True])
def test_graphs_captured_without_a_call_before_run_in_any_order(gpu, shared):
    """On the capture stream's workspace and on one of their own: each graph, and eager
    calls between, has counters that are zero, whatever the memory held."""

    announce(f"graphs without a call before {shared}")
    g = generator(77)
    batch, nodes, vocab = 4, 5, 9000
    target, draft = probabilities(g, batch, nodes, vocab).to(gpu), probabilities(g, batch, nodes - 1, vocab).to(gpu)
    tokens = torch.randint(0, vocab, (batch, nodes), generator=g).to(gpu)
    uniforms = torch.rand(batch, nodes, generator=g).to(gpu)
    query, key, value, lengths = (t.to(gpu) for t in tree_inputs(g, 2, 4, 2, 64, 6, 700, torch.bfloat16, [600, 3]))

    def step(workspace):
        return (*backends.hip_verify_tokens(tokens, target, uniforms, draft_probs=draft, workspace=workspace),
                backends.hip_tree_attention(query, key, value, lengths, None, scale=0.125, workspace=workspace))

    want = step(None)
    workspace = _native.DeviceWorkspace(gpu) if shared else None
    # Graphs of one pool; the first leaves ones in memory that the next ones' temporaries take.
    filler = torch.cuda.CUDAGraph()
    with torch.cuda.graph(filler):
        rooms = [torch.full((size,), -1, dtype=torch.int32, device=gpu) for size in (64, 80, 128, 512, 1024) for _ in range(8)]
        del rooms
    filler.replay()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(3):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=filler.pool()):
            out = step(workspace)
        graphs.append((graph, out))

    def check(out):
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)

    check(step(workspace))
    for at in (2, 0, 1, 0, 2):
        for tensor in graphs[at][1]:
            tensor.fill_(3)
        graphs[at][0].replay()
        check(graphs[at][1])
        check(step(workspace))


def test_each_capture_has_a_number(gpu):
    announce("capture numbers")
    stream, seen = torch.cuda.Stream(), []
    assert _native.library().slc_hip_capture_id(stream.cuda_stream) == 0
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            x = torch.zeros(4, device=gpu)
            seen += [_native._capture_id(gpu), _native.library().slc_hip_capture_id(stream.cuda_stream)]
        assert _native._capture_id(gpu) == 0 and _native.library().slc_hip_capture_id(stream.cuda_stream) == 0
    assert seen[0] == seen[1] != 0 and seen[2] == seen[3] != 0 and seen[0] != seen[2]
    assert _native.library().slc_hip_capture_id(None) == 0 and x.numel() == 4
