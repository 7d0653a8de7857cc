"""Refusals of the operators on drafted tokens: by the wrappers on host tensors and by the C
entry points on arguments that are checked before any device call."""

from __future__ import annotations

import copy
import ctypes
import pickle
from dataclasses import replace

import pytest
import torch

from stateful_llm_compiler_hip import _native, backends
from stateful_llm_compiler_hip.execution import ExecutionError, PagedKVCacheState, PreallocatedKVCacheState

P = 0x1000  # 4 KiB-aligned, never dereferenced on these paths
F32, F16, BF16, I32, I64 = 0, 1, 2, 3, 4


def test_wrappers_refuse_host_tensors():
    q, kv = torch.zeros(1, 2, 3, 64), torch.zeros(1, 16, 2, 64)
    lengths, table = torch.zeros(1, dtype=torch.int64), torch.zeros(1, 1, dtype=torch.int32)
    tokens, probs = torch.zeros(1, 3, dtype=torch.int64), torch.zeros(1, 3, 5)
    for call in (
        lambda: backends.hip_tree_attention(q, kv, kv, lengths, None, scale=1.0),
        lambda: backends.hip_paged_tree_attention(q, kv, kv, table, lengths, None, scale=1.0),
        lambda: backends.hip_verify_tokens(tokens, probs, torch.zeros(1, 3)),
        lambda: backends.KVLayers([kv], [kv.clone()]),
    ):
        with pytest.raises(ValueError, match="on the GPU"):
            call()


def tree(paged=False, query=P, key=P, value=P, lengths=P, lengths_dtype=I64, mask=None, mask_dtype=F32, out=P,
         workspace=P, nbytes=1 << 40, counters=P, num_counters=1 << 20, dtype=BF16, batch=2, q_heads=4, kv_heads=2, nodes=3, head_dim=64, rows=64,
         mask_len=64, scale=0.125, tree_mask=None, table=P, page_tokens=16, num_pages=9, kv_ss=128):
    lib = _native.library()
    tail = (scale, None)
    strides = (q_heads * nodes * head_dim, nodes * head_dim, head_dim)
    if paged:
        return lib.slc_hip_paged_tree_attention(
            query, key, value, table, rows // 16, rows // 16, page_tokens, num_pages, 16 * kv_ss, lengths,
            lengths_dtype, tree_mask, mask, mask_dtype, out, workspace, nbytes, counters, num_counters, dtype, batch, q_heads, kv_heads, nodes,
            head_dim, mask_len, *strides, kv_ss, head_dim, 0, 0, 0, 0, 0, *strides, *tail)
    return lib.slc_hip_tree_attention(
        query, key, value, lengths, lengths_dtype, tree_mask, mask, mask_dtype, out, workspace, nbytes, counters, num_counters, dtype, batch,
        q_heads, kv_heads, nodes, head_dim, rows, mask_len, *strides, rows * kv_ss, kv_ss, head_dim, 0, 0, 0, 0, 0,
        *strides, *tail)


@pytest.mark.parametrize("paged", [False, True])
def test_tree_attention_entry_points_refuse(paged):
    for bad in ({"dtype": I32}, {"dtype": 99}, {"lengths_dtype": F32}, {"batch": -1}, {"batch": 32769},
                {"nodes": -1}, {"nodes": 4097}, {"nodes": 1025, "tree_mask": P}, {"rows": 2**30, "batch": 17}, {"q_heads": 3}, {"q_heads": 0}, {"kv_heads": 0}, {"head_dim": 0},
                {"head_dim": 257}, {"query": None}, {"key": None}, {"value": None}, {"lengths": None}, {"out": None},
                {"workspace": None}, {"workspace": P + 8}, {"nbytes": 1000}, {"counters": None}, {"num_counters": 3},
                {"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")}, {"scale": float("inf")},
                {"mask": P, "mask_dtype": I32}, {"mask": P, "mask_len": 65}, {"mask": P, "mask_len": -1}):
        assert tree(paged, **bad) == -1, bad
    assert tree(paged, batch=0) == 0 and tree(paged, nodes=0) == 0  # nothing to do, nothing launched
    assert tree(paged, batch=0, query=None) == 0


def test_tree_attention_entry_points_refuse_their_own_operands():
    assert tree(rows=0) == -1 and tree(rows=2**30 + 1) == -1
    for bad in ({"page_tokens": 8}, {"page_tokens": 48}, {"page_tokens": 0}, {"num_pages": -1}, {"rows": 0},
                {"table": None}):
        assert tree(True, **bad) == -1, bad


def verify(tokens=P, parents=None, target=P, draft=None, uniforms=P, path=P, emitted=P, counts=P, counters=P,
           num_counters=64, dtype=F32, batch=2, nodes=3, vocab=100):
    return _native.library().slc_hip_verify_tokens(
        tokens, parents, target, draft, uniforms, path, emitted, counts, counters, num_counters, dtype,
        batch, nodes, vocab, nodes, nodes, nodes, nodes * vocab, vocab, nodes * vocab, vocab, None)


def test_verify_entry_point_refuses():
    for bad in ({"dtype": I64}, {"dtype": 99}, {"batch": -1}, {"batch": 65536}, {"nodes": 0}, {"nodes": 1025},
                {"vocab": 0}, {"vocab": 2**31}, {"num_counters": 5}, {"counters": P + 4},
                {"tokens": None}, {"target": None}, {"uniforms": None}, {"path": None}, {"emitted": None},
                {"counts": None}, {"counters": None}):
        assert verify(**bad) == -1, bad
    assert verify(batch=0) == 0 and verify(batch=0, tokens=None) == 0
    count = _native.library().slc_hip_verify_tokens_counter_count
    assert count(2, 1024) == 6 and count(3, 1025) == 16 and count(0, 5) == 0


def commit(key=(P, 2 * P), value=(3 * P, 4 * P), lengths=(5 * P, 6 * P), out=(7 * P, 8 * P), table=None, page_tokens=0,
           pages=0, num_pages=0, path=P, counts=P, dtype=BF16, layers=2, batch=2, nodes=3, heads=2, head_dim=64,
           capacity=64):
    def pointers(values):
        return None if values is None else (ctypes.c_void_p * len(values))(*values)

    return _native.library().slc_hip_kv_commit(
        pointers(key), pointers(value), pointers(lengths), pointers(out), table, pages, pages, page_tokens, num_pages,
        path, counts, None, dtype, layers, batch, nodes, heads, head_dim, capacity, capacity * heads * head_dim,
        heads * head_dim, head_dim, None)


def test_commit_entry_point_refuses():
    for bad in ({"dtype": I64}, {"layers": -1}, {"batch": -1}, {"batch": 65536}, {"nodes": 0}, {"nodes": 1025},
                {"heads": 0}, {"head_dim": 0}, {"capacity": 0}, {"key": None}, {"value": None}, {"lengths": None},
                {"out": None}, {"path": None}, {"counts": None}, {"key": (P, None)}, {"lengths": (None, P)},
                {"key": (P, P + 1)}, {"table": P, "page_tokens": 8, "pages": 8, "num_pages": 16},
                {"table": P, "page_tokens": 16, "pages": 3, "num_pages": 16},
                {"table": P, "page_tokens": 16, "pages": 4, "num_pages": -1}):
        assert commit(**bad) == -1, bad
    assert commit(layers=0) == 0 and commit(batch=0) == 0 and commit(batch=0, key=None) == 0


def test_state_refuses_what_does_not_fit_its_buffers():
    state = PreallocatedKVCacheState.empty_from_key_template(torch.zeros(2, 2, 1, 64), num_layers=2, capacity=32)
    query = torch.zeros(2, 4, 3, 64)
    for bad in (
        lambda: state.tree_attention(5, query, None, groups=2, scale=1.0),
        lambda: state.tree_attention(0, query[:1], None, groups=2, scale=1.0),
        lambda: state.tree_attention(0, query[..., :32], None, groups=2, scale=1.0),
        lambda: state.tree_attention(0, query[0], None, groups=2, scale=1.0),
        lambda: state.tree_attention(0, query, None, groups=4, scale=1.0),
        lambda: state.tree_attention(0, query, None, torch.zeros(2, 1, 1, 33), groups=2, scale=1.0),
        lambda: state.commit(torch.zeros(1, 3, dtype=torch.int64), torch.zeros(2, dtype=torch.int64)),
        lambda: state.commit(torch.zeros(2, 3, dtype=torch.int64), torch.zeros(3, dtype=torch.int64)),
    ):
        with pytest.raises(ExecutionError):
            bad()


def committing(monkeypatch):
    """States on host memory commit, the entry point left out: what it would get, the
    device pointers of keys and values, is noted."""

    from stateful_llm_compiler_hip.backends import hip_draft

    calls = []

    def entry_point(name, index, keys, values, lengths, out, *rest):
        layers = rest[-9]
        read = ctypes.c_uint64 * layers
        calls.append([list(read.from_address(at)) for at in (keys, values)])

    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    monkeypatch.setattr(hip_draft, "_call", entry_point)
    return calls


def pointers(state):
    return [[t.data_ptr() for t in side] for side in (state.keys, state.values)]


def state_to_commit(paged):
    template = torch.zeros(2, 2, 1, 8)
    make = PagedKVCacheState if paged else PreallocatedKVCacheState
    state = make.empty_from_key_template(template, num_layers=3, capacity=32, **({"page_tokens": 16} if paged else {}))
    return replace(state, overflow=None)


@pytest.mark.parametrize("paged", [False, True])
def test_copies_of_a_state_commit_their_own_buffers(monkeypatch, paged):
    calls = committing(monkeypatch)
    path, counts = torch.zeros(2, 3, dtype=torch.int64), torch.ones(2, dtype=torch.int64)
    state = state_to_commit(paged).commit(path, counts)
    assert calls[-1] == pointers(state)
    for other in (copy.deepcopy(state), pickle.loads(pickle.dumps(state)), copy.deepcopy(copy.copy(state))):
        assert other.keys[0].data_ptr() != state.keys[0].data_ptr()
        for _ in range(2):
            other = other.commit(path, counts)
            assert calls[-1] == pointers(other)
    copy.copy(state).commit(path, counts)
    assert calls[-1] == pointers(state)
    gone = copy.deepcopy(state)
    kept = pointers(state)
    del state
    gone.commit(path, counts)
    assert calls[-1] == pointers(gone) != kept


@pytest.mark.parametrize("paged", [False, True])
def test_copies_of_checked_layers_hold_their_own_buffers(monkeypatch, paged):
    calls = committing(monkeypatch)
    state = state_to_commit(paged)
    layers = backends.KVLayers(state.keys, state.values, block_table=state.block_table if paged else None)
    path, counts = torch.zeros(2, 3, dtype=torch.int64), torch.ones(2, dtype=torch.int64)
    for other in (copy.deepcopy(layers), pickle.loads(pickle.dumps(layers)), copy.copy(layers)):
        backends.hip_kv_commit(other, state.lengths, path, counts)
        assert calls[-1] == [[t.data_ptr() for t in side] for side in (other.keys, other.values)]
        assert (other.keys[0] is layers.keys[0]) == (calls[-1] == pointers(state))
        assert paged == (other.block_table is not None)
        if paged:
            assert other._pages[0] == other.block_table.data_ptr()


def test_committed_states_load_where_there_is_no_gpu(monkeypatch):
    with monkeypatch.context() as context:
        committing(context)
        state = state_to_commit(False).commit(torch.zeros(2, 3, dtype=torch.int64), torch.ones(2, dtype=torch.int64))
        saved = pickle.dumps(state)
    loaded = pickle.loads(saved)
    assert torch.equal(loaded.keys[0], state.keys[0]) and loaded.generation == state.generation
    assert torch.equal(copy.deepcopy(state).lengths[1], state.lengths[1])


def test_paged_states_take_their_table_as_the_tenth_argument():
    """The fields keep their order in the constructor, where ``layers`` is by name only."""

    state = PagedKVCacheState.empty_from_key_template(torch.zeros(2, 2, 1, 8), num_layers=2, capacity=32, page_tokens=16)
    other = PagedKVCacheState(state.keys, state.values, state.lengths, 32, 4, None, True, None, None, state.block_table, 16)
    assert other.block_table is state.block_table and other.page_tokens == 16 and other.generation == 4
    assert other.layers is None and other.zero_slots is None and other.in_place_lengths
    with pytest.raises(TypeError):
        PreallocatedKVCacheState(state.keys, state.values, state.lengths, 16, 0, None, False, None, None, None)
    assert replace(other, layers=None, generation=5).generation == 5


@pytest.mark.parametrize("paged", [False, True])
def test_what_a_commit_leaves_at_length_zero_takes_a_prefill(monkeypatch, paged):
    """Which slots are at zero is unknown to the host after a commit, whose counts the
    device has; slots that were past zero stay refused without a look."""

    committing(monkeypatch)
    stored = []
    for kind in (PreallocatedKVCacheState, PagedKVCacheState):
        monkeypatch.setattr(kind, "store", lambda self, slot, *args, **kwargs: stored.append(slot))
        monkeypatch.setattr(kind, "advance", lambda self, slot, *, delta: self)
    state = state_to_commit(paged)
    path, counts = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, dtype=torch.int64)
    rows = torch.zeros(2, 2, 4, 8)
    after = replace(state.commit(path, counts), lengths=state.lengths)  # as counts of zero leave them
    after.prefill_store(1, rows, rows)
    assert stored == [1]
    full = replace(state, lengths=tuple(torch.full((2,), 4) for _ in range(3)), zero_slots=frozenset())
    for later in (replace(state.commit(path, counts), lengths=full.lengths), full.commit(path, counts)):
        with pytest.raises(ExecutionError, match="length to be 0"):
            later.prefill_store(1, rows, rows)
    assert full.commit(path, counts).zero_slots == frozenset() and stored == [1]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_tree_workspace_of_large_batches_holds_what_is_cut_only(dtype):
    """Where whole sequences are enough for all CUs, a quarter as many further pieces and
    their sequences' first ones have partial results."""

    size = _native.library().slc_hip_tree_attention_workspace_size
    for batch, q_heads, kv_heads, nodes, head_dim in ((1024, 32, 8, 64, 128), (32, 32, 32, 1024, 128), (2048, 2, 1, 1, 64),
                                                      (3, 512, 512, 1, 64), (1027, 14, 2, 5, 256)):
        rows = q_heads // kv_heads * nodes
        padded = max(16, min(256, 1 << (rows - 1).bit_length()))  # of a row block at most
        places = 2 * (batch // 4) * kv_heads * (rows + padded - 1)
        assert size(batch, q_heads, kv_heads, nodes, head_dim, dtype) <= places * (4 * head_dim + 8) + 8 * batch


def test_counters_made_in_a_capture_serve_that_capture_only(monkeypatch):
    """They are zeroed where the graph is replayed, not where it is captured: an eager
    call and another graph that came first would find what the memory held."""

    now = [0]
    monkeypatch.setattr(_native, "_capture_id", lambda device: now[0], raising=False)
    workspace = _native.DeviceWorkspace("cpu")

    def counters(capture, count):
        now[0] = capture
        return workspace.counters(count)

    first = counters(7, 100)
    assert counters(7, 30) is first and first.numel() == 100  # within the capture: one
    second, eager = counters(8, 30), counters(0, 30)
    assert len({t.data_ptr() for t in (first, second, eager)}) == 3 and second.numel() == eager.numel() == 100
    # Those of an eager call were zeroed at once: all take them, while they are enough.
    assert counters(9, 100) is eager and counters(0, 1) is eager and counters(10, 64) is eager
    more = counters(11, 101)
    assert more is not eager and more.numel() == 200 and counters(11, 150) is more
    assert any(t is eager for t in workspace._retired)  # graph 9 holds them
    other = counters(0, 5)
    assert other is not more and other.numel() == 200 and counters(12, 200) is other
    assert not any(t is more or t is first or t is second for t in workspace._retired)
    assert all(int(t.abs().sum()) == 0 for t in (first, second, eager, more, other))
