"""A step on drafted tokens: attention of a tree of them over a KV cache, their
verification, and the commit of the accepted ones' rows.

A cheaper model proposes several tokens per sequence; they go through the model at
once.  A sequence's nodes form a tree: node 0, the last token that stands, is its
root, every other node has an earlier one as its parent.  A layer stores the nodes' K
and V behind the sequence, node j at row ``lengths[b] + j`` (``hip_kv_store`` or
``hip_rope_kv_store`` at the lengths, with the cosines and sines of each node's own
position, ``lengths[b]`` + its depth) and attends with ``hip_tree_attention``.  From
the target's probabilities ``hip_verify_tokens`` finds the accepted nodes and the token
that follows them, and ``hip_kv_commit`` moves the accepted rows of all layers to their
places and advances the lengths.  The reference has no such step.

``hip_tree_attention`` stands beside ``hip_decode_attention`` (one token per sequence)
and ``hip_prefill_attention`` (as many queries as keys), ``hip_verify_tokens`` beside
``hip_argmax`` and ``hip_kv_commit`` beside ``hip_kv_store`` and ``hip_kv_advance``.
The operators are for inference: their outputs carry no gradient.
"""

from __future__ import annotations

import functools
from array import array
from typing import Sequence

import torch

from .. import _native
from .hip_ops import _FLOATS, check_flag
from .hip_paged import _check_pools
from .hip_q8 import _CONTIGUOUS, _call

_LENGTHS = (torch.int64, torch.int32)
_MOST = torch.finfo(torch.float32).max

MAX_NODES = 1024  # SLC_TREE_MAX_NODES, SLC_VERIFY_MAX_NODES
MAX_CHAIN = 4096  # SLC_CHAIN_MAX_NODES: nodes of tree attention without a tree mask


def _tree_operands(what, query, key, value, lengths, tree_mask, attention_mask, rows, kv_heads, scale):
    """Device index and the tree's, mask's and lengths' arguments, after the checks
    that both layouts share."""

    index, dtype = query.get_device(), query.dtype
    if index < 0 or key.get_device() != index or value.get_device() != index or lengths.get_device() != index or (
        (tree_mask is not None and tree_mask.get_device() != index)
        or (attention_mask is not None and attention_mask.get_device() != index)
    ):
        raise ValueError(f"{what}: all tensors must be on the GPU, and on one")
    batch, q_heads, nodes, head_dim = query.shape
    if query.stride(3) != 1 and head_dim > 1:
        raise ValueError(f"{what}: query head dim must be contiguous")
    if dtype not in _FLOATS:
        raise ValueError(f"{what}: unsupported dtype {dtype}")
    if key.dtype != dtype or value.dtype != dtype:
        raise ValueError(f"{what}: Q/K/V dtypes must match")
    if key.shape[3] != head_dim or kv_heads < 1 or q_heads < 1 or q_heads % kv_heads:
        raise ValueError(f"{what}: GQA or head shapes do not match")
    if not 1 <= head_dim <= 256:
        raise ValueError(f"{what}: head_dim must be 1 to 256")
    if nodes > (MAX_CHAIN if tree_mask is None else MAX_NODES):
        raise ValueError(f"{what}: a tree has at most {MAX_NODES} nodes, a chain {MAX_CHAIN}")
    if lengths.shape != (batch,) or lengths.dtype not in _LENGTHS or not lengths.is_contiguous():
        raise ValueError(f"{what}: lengths must be a contiguous int64 (or int32) [batch] tensor")
    if not 0.0 < scale <= _MOST:
        raise ValueError(f"{what}: scale must be positive and finite")
    tree, tree_strides = None, (0, 0, 0)
    if tree_mask is not None:
        tree_strides = tree_mask.stride()
        if len(tree_strides) == 2:
            tree_strides = (0, *tree_strides)
        if tree_mask.dtype != torch.bool or tree_mask.shape not in ((nodes, nodes), (batch, nodes, nodes)):
            raise ValueError(f"{what}: tree_mask must be a bool [T, T] or [batch, T, T] tensor")
        tree = tree_mask.data_ptr()
    mask, mask_dtype, mask_strides, mask_len = None, 0, (0, 0), rows
    if attention_mask is not None:
        if (attention_mask.ndim != 4 or attention_mask.shape[:3] != (batch, 1, 1)
                or attention_mask.dtype not in _FLOATS):
            raise ValueError(f"{what}: mask must be a floating B x 1 x 1 x S tensor")
        mask_len = attention_mask.shape[3]
        if mask_len > rows:
            raise ValueError(f"{what}: mask is longer than the cache's capacity")
        # (A mask of no rows hides all; its null pointer would stand for no mask.)
        mask = attention_mask.data_ptr() if mask_len else lengths.data_ptr()
        mask_dtype = _native.dtype_tag(attention_mask.dtype)
        mask_strides = (attention_mask.stride(0), attention_mask.stride(3))
    return index, (lengths.data_ptr(), _native.dtype_tag(lengths.dtype), tree, mask, mask_dtype), mask_len, (
        *tree_strides, *mask_strides)


@functools.lru_cache(maxsize=1024)
def _tree_scratch(index, batch, q_heads, kv_heads, nodes, head_dim, dtype):
    """Workspace bytes and counters of a call, by its sizes."""

    lib = _native.library()
    sizes = (batch, q_heads, kv_heads, nodes, head_dim, dtype)
    with torch.cuda.device(index):
        return (lib.slc_hip_tree_attention_workspace_size(*sizes), lib.slc_hip_tree_attention_counter_count(*sizes))


def _tree_workspace(device, index, workspace, *sizes):
    nbytes, count = _tree_scratch(index, *sizes)
    owner = workspace if workspace is not None else _native.stream_workspace(device)
    counters = owner.counters(count)
    return owner.scratch("tree_attention", nbytes).data_ptr(), nbytes, counters.data_ptr(), counters.numel()


def hip_tree_attention(
    query: torch.Tensor,
    key_buffer: torch.Tensor,
    value_buffer: torch.Tensor,
    lengths: torch.Tensor,
    tree_mask: torch.Tensor | None,
    attention_mask: torch.Tensor | None = None,
    *,
    scale: float,
    workspace: _native.DeviceWorkspace | None = None,
) -> torch.Tensor:
    """B x H x T x D GQA attention of T nodes per sequence over B x Cap x KVH x D buffers.

    Node i of sequence b sees the rows ``s < lengths[b]`` and those of its nodes j,
    ``lengths[b] + j``, with ``tree_mask[b, i, j]`` (bool, [T, T] or [B, T, T]; None: a
    chain, j <= i); ``lengths`` are those before the nodes.  A tree has at most 1024
    nodes, a chain 4096.  ``attention_mask`` is as in
    ``hip_decode_attention``: additive [B, 1, 1, S] over the buffers' rows, the nodes'
    own included; rows from S on, and those whose mask is -inf, are not seen.  Rows
    past the capacity were not stored and are not seen either.  Nothing that a row
    holds reaches a node that does not see it; a node that sees none has NaN.

    ``key_buffer``/``value_buffer`` may be views with a contiguous head dim and equal
    strides.  The softmax is fp32; 16-bit types round its unnormalised weights for the
    product with V, as ``hip_decode_attention``'s online order does (there is no exact
    order here).  ``workspace``: the caller's ``DeviceWorkspace`` (else the current
    stream's); calls that may run concurrently need separate ones.
    """

    what = "HIP tree attention"
    shape, buffer_shape = query.shape, key_buffer.shape
    if len(shape) != 4 or len(buffer_shape) != 4 or buffer_shape != value_buffer.shape:
        raise ValueError(f"{what}: illegal shapes")
    strides = key_buffer.stride()
    if strides != value_buffer.stride() or (strides[3] != 1 and buffer_shape[3] > 1):
        raise ValueError(f"{what}: K/V buffers need equal strides and a contiguous head dim")
    batch, capacity, kv_heads, _ = buffer_shape
    if shape[0] != batch or capacity < 1:
        raise ValueError(f"{what}: query and buffers need one batch, and the buffers rows")
    index, operands, mask_len, mask_strides = _tree_operands(
        what, query, key_buffer, value_buffer, lengths, tree_mask, attention_mask, capacity, kv_heads, scale)
    output = torch.empty_like(query)
    _, q_heads, nodes, head_dim = shape
    if batch == 0 or nodes == 0:
        return output
    dtype = _native.dtype_tag(query.dtype)
    scratch = _tree_workspace(query.device, index, workspace, batch, q_heads, kv_heads, nodes, head_dim, dtype)
    _call("slc_hip_tree_attention", index, query.data_ptr(), key_buffer.data_ptr(), value_buffer.data_ptr(), *operands,
          output.data_ptr(), *scratch, dtype, batch, q_heads, kv_heads, nodes, head_dim, capacity, mask_len,
          *query.stride()[:3], *strides[:3], *mask_strides, *output.stride()[:3], scale)
    return output


def hip_paged_tree_attention(
    query: torch.Tensor,
    key_pool: torch.Tensor,
    value_pool: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    tree_mask: torch.Tensor | None,
    attention_mask: torch.Tensor | None = None,
    *,
    scale: float,
    workspace: _native.DeviceWorkspace | None = None,
) -> torch.Tensor:
    """``hip_tree_attention`` over paged K/V: the pools and the block table as in
    ``hip_paged_decode_attention``, every dtype and head layout of the contiguous form.
    Table entries that name no page of the pool are not followed; what a node that
    sees rows of such a page gets has no meaning."""

    what = "HIP paged tree attention"
    if query.ndim != 4:
        raise ValueError(f"{what}: illegal shapes")
    batch, q_heads, nodes, head_dim = query.shape
    pages, page_tokens = _check_pools(key_pool, value_pool, block_table, batch, what)
    if pages < 1:
        raise ValueError(f"{what}: the block table has no pages")
    index, operands, mask_len, strides = _tree_operands(
        what, query, key_pool, value_pool, lengths, tree_mask, attention_mask, pages * page_tokens, key_pool.shape[2],
        scale)
    if block_table.get_device() != index:
        raise ValueError(f"{what}: all tensors must be on the GPU, and on one")
    output = torch.empty_like(query)
    if query.numel() == 0:
        return output
    dtype = _native.dtype_tag(query.dtype)
    kv_heads = key_pool.shape[2]
    scratch = _tree_workspace(query.device, index, workspace, batch, q_heads, kv_heads, nodes, head_dim, dtype)
    _call("slc_hip_paged_tree_attention", index, query.data_ptr(), key_pool.data_ptr(), value_pool.data_ptr(),
          block_table.data_ptr(), block_table.stride(0), pages, page_tokens, key_pool.shape[0], key_pool.stride(0),
          *operands, output.data_ptr(), *scratch, dtype, batch, q_heads, kv_heads, nodes, head_dim, mask_len,
          *query.stride()[:3], *key_pool.stride()[1:3], *strides, *output.stride()[:3], scale)
    return output


def _rows(tensor):
    """``tensor``, or a copy of it where its last axis is not contiguous."""

    return tensor if tensor.stride(-1) == 1 or tensor.shape[-1] == 1 else tensor.contiguous()


@functools.lru_cache(maxsize=1024)
def _verify_counters(batch, vocab):
    return _native.library().slc_hip_verify_tokens_counter_count(batch, vocab)


def hip_verify_tokens(
    tokens: torch.Tensor,
    target_probs: torch.Tensor,
    uniforms: torch.Tensor,
    *,
    parents: torch.Tensor | None = None,
    draft_probs: torch.Tensor | None = None,
    workspace: _native.DeviceWorkspace | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(path, emitted, counts)``: the nodes that the target accepts, and the tokens
    that the step gives, with the target's distribution.

    ``tokens`` [B, T] int64 holds the nodes' tokens (node 0's is not looked at),
    ``parents`` [B, T] int64 their parents (None: a chain; a node whose parent is not
    an earlier node, -1 say, is padding), ``target_probs`` [B, T, V] the target's
    distribution of the token behind each node, ``uniforms`` [B, T] fp32 random numbers
    in [0, 1): one for each node's test, the root's for the token that follows.
    ``draft_probs`` [B, T - 1, V], of the target's dtype: the distributions that the
    children of each node were drawn from, independently of each other; None: the
    children are candidates, the best first, without probabilities.

    From node 0 down the children of a node are tried in ascending order.  With p and q
    the target's and the draft's row at the node, w = max(p - M q, 0), m = sum w (M = 0
    and m = 1 at first), a child of token x is accepted where u m q(x) < w(x), and a
    refusal adds m to M.  Without draft rows w = p, a child is accepted where
    u m < w(x), and a refusal takes w(x) from m and sets it to 0.  Where no child is
    accepted the token that follows is the first i with w(0) + .. + w(i) > u_0 sum w
    (p where no w is positive; -1 where no p is).  All in fp64; a probability that is NaN
    or negative counts as 0.

    ``path`` [B, T]: the accepted nodes in ascending order, then -1; ``emitted`` [B, T]:
    their tokens without node 0's, the token that follows, then -1; ``counts`` [B]: how
    many of each.  All int64, as ``hip_kv_commit`` takes them.
    """

    what = "HIP verify tokens"
    index = tokens.get_device()
    if index < 0 or target_probs.get_device() != index or uniforms.get_device() != index or (
        (parents is not None and parents.get_device() != index)
        or (draft_probs is not None and draft_probs.get_device() != index)
    ):
        raise ValueError(f"{what}: all tensors must be on the GPU, and on one")
    shape, target_shape = tokens.shape, target_probs.shape
    if tokens.dtype != torch.int64 or len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"{what}: tokens must be an int64 [batch, nodes] tensor")
    batch, nodes = shape
    if nodes > MAX_NODES:
        raise ValueError(f"{what}: at most {MAX_NODES} nodes")
    if parents is not None and (parents.dtype != torch.int64 or parents.shape != shape):
        raise ValueError(f"{what}: parents must be int64 and shaped like the tokens")
    if uniforms.dtype != torch.float32 or uniforms.shape != shape:
        raise ValueError(f"{what}: uniforms must be fp32 and shaped like the tokens")
    if len(target_shape) != 3 or target_shape[:2] != shape or target_shape[2] < 1:
        raise ValueError(f"{what}: target_probs must be [batch, nodes, vocabulary]")
    dtype, vocab = target_probs.dtype, target_shape[2]
    if dtype not in _FLOATS:
        raise ValueError(f"{what}: unsupported dtype {dtype}")
    if draft_probs is not None and (draft_probs.shape != (batch, nodes - 1, vocab) or draft_probs.dtype != dtype):
        raise ValueError(f"{what}: draft_probs must be [batch, nodes - 1, vocabulary] of the target's dtype")
    path = torch.empty_like(tokens, memory_format=_CONTIGUOUS)
    emitted = torch.empty_like(path)
    counts = path.new_empty(batch)
    if batch == 0:
        return path, emitted, counts
    tokens, uniforms, target_probs = _rows(tokens), _rows(uniforms), _rows(target_probs)
    up, up_stride, draft, draft_strides = None, 0, None, (0, 0)
    if parents is not None:
        parents = _rows(parents)
        up, up_stride = parents.data_ptr(), parents.stride(0)
    if draft_probs is not None:
        draft_probs = _rows(draft_probs)
        draft, draft_strides = draft_probs.data_ptr(), draft_probs.stride()[:2]
    owner = workspace if workspace is not None else _native.stream_workspace(tokens.device)
    counters = owner.counters(_verify_counters(batch, vocab))
    _call("slc_hip_verify_tokens", index, tokens.data_ptr(), up, target_probs.data_ptr(), draft, uniforms.data_ptr(),
          path.data_ptr(), emitted.data_ptr(), counts.data_ptr(), counters.data_ptr(), counters.numel(),
          _native.dtype_tag(dtype), batch, nodes, vocab, tokens.stride(0), up_stride, uniforms.stride(0),
          *target_probs.stride()[:2], *draft_strides)
    return path, emitted, counts


class KVLayers:
    """The KV caches of a model's layers, checked once, for ``hip_kv_commit``: a program
    makes it with its caches and keeps it as long as them (it holds their addresses: for
    tensors that get other memory, by ``set_`` or ``.data``, it is made anew).  A copy and
    an unpickled one are made and checked anew, of the copied buffers.

    ``keys`` and ``values``: one buffer per layer, B x Cap x KVH x D, or with
    ``block_table`` (int32 [B, pages]) one page pool per layer.
    """

    def __init__(self, keys: Sequence[torch.Tensor], values: Sequence[torch.Tensor], *,
                 block_table: torch.Tensor | None = None) -> None:
        what = "HIP KV layers"
        self.keys, self.values, self.block_table = tuple(keys), tuple(values), block_table
        buffers = self.keys + self.values
        if not self.keys or len(self.keys) != len(self.values):
            raise ValueError(f"{what}: one key and one value buffer per layer are needed")
        first = buffers[0]
        self.device, self.index = first.device, first.get_device()
        if self.index < 0 or any(buffer.get_device() != self.index for buffer in buffers):
            raise ValueError(f"{what}: all tensors must be on the GPU, and on one")
        if first.ndim != 4 or first.dtype not in _FLOATS:
            raise ValueError(f"{what}: buffers must be four-dimensional and floating")
        if any(buffer.shape != first.shape or buffer.dtype != first.dtype or buffer.stride() != first.stride()
               for buffer in buffers):
            raise ValueError(f"{what}: buffers need one shape, dtype and set of strides")
        if first.stride(3) != 1 and first.shape[3] > 1:
            raise ValueError(f"{what}: the head dim must be contiguous")
        if any(stride == 0 and size > 1 for stride, size in zip(first.stride(), first.shape)):
            raise ValueError(f"{what}: expanded buffers cannot be written")
        if block_table is None:
            self.batch, self.capacity, self.heads, self.head_dim = first.shape
            self._pages = (None, 0, 0, 0, 0)
        else:
            if block_table.ndim != 2 or block_table.get_device() != self.index:
                raise ValueError(f"{what}: block_table must be a [batch, pages] tensor on the buffers' GPU")
            self.batch = block_table.shape[0]
            pages, page_tokens = _check_pools(first, self.values[0], block_table, self.batch, what)
            self.capacity, self.heads, self.head_dim = pages * page_tokens, first.shape[2], first.shape[3]
            self._pages = (block_table.data_ptr(), block_table.stride(0), pages, page_tokens, first.shape[0])
        if self.capacity < 1 or self.heads < 1 or self.head_dim < 1:
            raise ValueError(f"{what}: the buffers are empty")
        self._pointers = array("Q", [buffer.data_ptr() for buffer in buffers])
        if len(set(self._pointers)) != len(buffers):
            raise ValueError(f"{what}: a buffer is there twice")
        self._dtype, self._strides = _native.dtype_tag(first.dtype), first.stride()[:3]

    def __reduce__(self):
        return _kv_layers, (type(self), self.keys, self.values, self.block_table)


def _kv_layers(kind, keys, values, block_table):
    return kind(keys, values, block_table=block_table)


def _layer_pointers(layers: KVLayers, lengths, what: str, name: str) -> array:
    """Device pointers of each layer's lengths: a tensor [B] (all layers'), [L, B], or
    a sequence of L tensors [B]."""

    count, batch, index = len(layers.keys), layers.batch, layers.index
    if isinstance(lengths, torch.Tensor):
        shape = lengths.shape
        if (lengths.dtype != torch.int64 or shape not in ((batch,), (count, batch)) or not lengths.is_contiguous()
                or lengths.get_device() != index):
            raise ValueError(f"{what}: {name} must be a contiguous int64 [B] or [layers, B] tensor on the caches' GPU")
        start, step = lengths.data_ptr(), 8 * batch
        if len(shape) == 1 or batch == 0:
            return array("Q", [start]) * count
        return array("Q", range(start, start + step * count, step))
    if len(lengths) != count or any(
        length.dtype != torch.int64 or length.shape != (batch,) or not length.is_contiguous()
        or length.get_device() != index for length in lengths
    ):
        raise ValueError(f"{what}: {name} must be one contiguous int64 [B] tensor per layer, on the caches' GPU")
    return array("Q", [length.data_ptr() for length in lengths])


def hip_kv_commit(
    layers: KVLayers,
    lengths: torch.Tensor | Sequence[torch.Tensor],
    path: torch.Tensor,
    counts: torch.Tensor,
    *,
    out: torch.Tensor | Sequence[torch.Tensor] | None = None,
    overflow: torch.Tensor | None = None,
):
    """Moves K and V row ``lengths[b] + path[b, j]`` to row ``lengths[b] + j``, for
    ``j < counts[b]``, in every layer, and returns ``lengths + counts``.

    ``path`` [B, T] and ``counts`` [B], int64, as ``hip_verify_tokens`` gives them:
    a row's path ascends within its count (entries that are no node are not moved).
    Pages that rows move in belong to one sequence.
    ``lengths``: int64 [B], the same for all layers, or [layers, B], or one [B] tensor
    per layer.  ``out`` receives the new ones, in any of these forms, and may be
    ``lengths`` itself where these are a tensor for each layer.  Rows behind the new
    lengths keep what they held.  The optional int32 ``overflow`` flag is set where a new
    length lies past the capacity, and where it counts a row that is not there: an accepted
    node whose row lies past the capacity (so that it was not stored) or in a page that is none of the
    pool's, an entry that is no node, a count outside [0, T] (taken as the nearest within).
    """

    what = "HIP KV commit"
    count, batch, index = len(layers.keys), layers.batch, layers.index
    check_flag(overflow, what)
    if path.get_device() != index or counts.get_device() != index or (
        overflow is not None and overflow.get_device() != index
    ):
        raise ValueError(f"{what}: all tensors must be on the GPU, and on one")
    shape = path.shape
    if path.dtype != torch.int64 or len(shape) != 2 or shape[0] != batch or not path.is_contiguous():
        raise ValueError(f"{what}: path must be a contiguous int64 [B, nodes] tensor")
    if not 1 <= shape[1] <= MAX_NODES:
        raise ValueError(f"{what}: 1 to {MAX_NODES} nodes")
    if counts.dtype != torch.int64 or counts.shape != (batch,) or not counts.is_contiguous():
        raise ValueError(f"{what}: counts must be a contiguous int64 [B] tensor")
    sources = _layer_pointers(layers, lengths, what, "lengths")
    if out is None:
        out = torch.empty_like(lengths) if isinstance(lengths, torch.Tensor) else tuple(
            torch.empty_like(length) for length in lengths)
        targets = _layer_pointers(layers, out, what, "out")
    else:
        targets = _layer_pointers(layers, out, what, "out")
        # A layer reads its length while another layer's is written.
        places = sorted({*sources, *targets})
        if batch and (any(high - low < 8 * batch for low, high in zip(places, places[1:])) or any(
            target in sources and (source != target or sources.count(target) > 1)
            for source, target in zip(sources, targets)
        )):
            raise ValueError(f"{what}: out may be a layer's own lengths, but overlap no other layer's")
        if len(set(targets)) not in (1, count):
            raise ValueError(f"{what}: every layer needs an output of its own")
        for tensor in (path, counts):
            start, end = tensor.data_ptr(), tensor.data_ptr() + 8 * tensor.numel()
            if any(start - 8 * batch < target < end for target in targets):
                raise ValueError(f"{what}: out overlaps the path or the counts")
    if batch == 0:
        return out
    if targets[0] == targets[-1]:  # one tensor for all layers: the first one's workgroups write it
        targets = targets[:1] + array("Q", [0]) * (count - 1)
    keys = layers._pointers.buffer_info()[0]
    _call("slc_hip_kv_commit", index, keys, keys + 8 * count, sources.buffer_info()[0], targets.buffer_info()[0],
          *layers._pages, path.data_ptr(), counts.data_ptr(), None if overflow is None else overflow.data_ptr(),
          layers._dtype, count, batch, shape[1], layers.heads, layers.head_dim, layers.capacity, *layers._strides)
    return out
