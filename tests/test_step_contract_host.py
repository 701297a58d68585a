"""Host-side halves of what the operators round the selection path owe one another, with host tensors in the place of the device's: what
`release` returns, positions of trees, the selector's state between forwards."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import step_reference as reference
from kvip_b200 import BlockTables, IndexSelector, RequestPlan


def tables_on_the_host(lengths, held, table, free, *, block, tokens, head=0):
    """A BlockTables whose buffers are host tensors; `plan` is the restatement. The free list has a place for every block."""
    t = BlockTables.__new__(BlockTables)
    i32 = dict(dtype=torch.int32)
    t.torch, t.device, t.batch, t.pages, t.blocks, t.block, t.tokens = torch, torch.device("cpu"), len(lengths), len(table[0]), len(free), block, tokens
    t.lengths, t.held, t.table, t.free = (torch.tensor(x, **i32) for x in (lengths, held, table, free))
    t.ends, t.held_after, t.starts = t.lengths.clone(), t.held.clone(), torch.zeros(t.batch + 1, **i32)
    t.head, (t.taken, t.status) = torch.tensor([head], **i32), torch.zeros((2, 1), **i32)
    t._planned = ((t.ends, t.lengths), (t.held_after, t.held), (t.taken, torch.zeros(1, **i32)))

    def plan(counts):
        out = reference.slot_maps(t.lengths.numpy(), counts, t.held.numpy(), t.table.numpy(), t.free.numpy(), int(t.head), block=block, tokens=tokens)
        for name in ("table", "starts", "ends", "held_after", "taken"):
            getattr(t, name).copy_(torch.from_numpy(out[name]))
        t.positions, t.requests = torch.from_numpy(out["positions"]), torch.from_numpy(out["requests"])
        t.status |= torch.from_numpy(out["status"])
        return out

    t.plan = plan
    return t


def test_release_passes_over_entries_that_are_no_block():
    t = tables_on_the_host([9, 2], [3, 1], [[5, -1, 7], [8, -1, -1]], [0, 1, 2, 3], block=4, tokens=4, head=4)
    t.release([0])
    assert int(t.status) == 4 and int(t.head) == 2 and t.free.tolist() == [0, 1, 5, 7]
    t.status.zero_()
    t.release([1])
    assert int(t.status) == 0 and int(t.head) == 1 and t.free.tolist() == [0, 8, 5, 7]
    assert np.array_equal(t.held.numpy(), [0, 0]) and int(t.table.max()) == -1


def test_positions_of_trees_go_by_depth():
    t = tables_on_the_host([5, 0, 9], [1, 0, 1], [[0, -1], [-1, -1], [1, -1]], [2, 3, 3, 3], block=16, tokens=9)
    t.plan([4, 0, 3])
    assert t.positions.tolist() == [5, 6, 7, 8, 9, 10, 11, -1, -1]
    depths = torch.tensor([0, 1, 1, 2, 0, 1, 1, 5, -7], dtype=torch.int32)
    assert t.tree_positions(depths).tolist() == [5, 6, 6, 7, 9, 10, 10, -1, -1] and int(t.status) == 0
    depths[1:3] = torch.tensor([-1, 3])
    assert t.tree_positions(depths).tolist() == [5, 5, 7, 7, 9, 10, 10, -1, -1] and int(t.status) == 1
    with pytest.raises(ValueError, match="depths"):
        t.tree_positions(depths[:8])
    with pytest.raises(ValueError, match="depths"):
        t.tree_positions(depths.long())


class Inputs:
    """What the selector asks of QueryInputs, on the host."""

    batch, queries, index_heads = 2, 4, 64

    def __init__(self):
        self.query, self.weights, self.scale = torch.zeros(8, 64, 128), torch.zeros(8, 64), torch.zeros(8, 64)
        self.row_owners = torch.zeros(2, dtype=torch.int32)
        self.token_count, self.calls = 0, []

    def prepare(self, counts, *, query_starts, query_owners):
        self.row_owners[:len(query_owners)] = torch.tensor(query_owners, dtype=torch.int32)
        self.token_count = sum(counts)

    def prepare_device(self, layout, owners):
        self.row_owners.copy_(owners)
        self.token_count = 8

    def bind_positions(self, positions):
        self.positions = positions

    def pack(self, *_):
        self.calls.append("pack")


@pytest.mark.parametrize("plans", [[RequestPlan("a", 1, 0, 3, decode=False, key_end=3)],
                                   [RequestPlan("a", 1, 0, 3, decode=True, key_end=9), RequestPlan("b", 2, 3, 5, decode=False, key_end=2)]])
def test_a_step_prepared_on_the_device_forgets_the_plans_before_it(plans):
    """A prefill or mixed forward, then a decode step whose layout the device has made: the step is packed and selected whole, its owners
    reach a tensor of the selector's own, and slots of the step before are no longer there."""
    inputs = Inputs()
    storage = SimpleNamespace(prepare=lambda plans: None, ingest_prefill=lambda *_: inputs.calls.append("prefill"),
                              ingest_decode=lambda cache, metadata, inputs, owners: inputs.calls.append(("decode", owners.tolist())))
    rotating = SimpleNamespace(arguments=[inputs.query, None, inputs.weights, inputs.scale, None, None, torch.full((2,), 99, dtype=torch.int32)])
    update = SimpleNamespace(logical_output=torch.arange(8 * 2048, dtype=torch.int32).view(8, 1, 2048), slot_output=torch.zeros(8, 1, 2048, dtype=torch.int32))
    selector = IndexSelector(torch, inputs=inputs, rotating=rotating, update=update, logical_ids=torch.zeros(4, 8, dtype=torch.int64),
                             row_owners=torch.zeros(2, dtype=torch.int32), storage=storage, forward=lambda: inputs.calls.append("forward"))
    indexer = SimpleNamespace(k_cache=SimpleNamespace(kv_cache=None),
                              select_topk_native=lambda query, *_: torch.zeros(query.shape[0], 1, 2048, dtype=torch.int32))
    metadata = SimpleNamespace(block_table=torch.zeros(2, 4, dtype=torch.int32))

    def step(tokens):
        inputs.calls.clear()
        return selector(torch.zeros(tokens, 64, 128), torch.zeros(tokens, 64), indexer, metadata, torch.ones(tokens, 64))

    selector.prepare(plans)
    step(plans[-1].stop)
    assert "prefill" in inputs.calls
    tables = SimpleNamespace(layout=torch.zeros(4, 8, dtype=torch.int64), positions=torch.tensor([5, 6, 7, 8, 2, 3]),
                             lengths=torch.tensor([5, 2], dtype=torch.int32))
    selector.prepare_device(tables, torch.tensor([3, 2], dtype=torch.int32))
    with pytest.raises(RuntimeError, match="execute"):
        selector.slots(1)
    assert inputs.positions is tables.positions and selector.positions is tables.positions and rotating.arguments[6].tolist() == [5, 2]
    logical = step(6)
    assert inputs.calls == [("decode", [3, 2]), "pack", "forward"]
    assert torch.equal(logical, update.logical_output[:6]) and selector.slots(6).shape[0] == 6
    with pytest.raises(ValueError, match="query slots"):
        selector.prepare_device(SimpleNamespace(layout=None), torch.zeros(2, dtype=torch.int32))


def test_numbers_that_a_record_does_not_hold_are_value_errors():
    from kvip_b200 import _launch, _lib
    from kvip_b200.build import build_library
    build_library()
    launch = _launch.Launcher("kvip_b200_slot_attention")
    good = [0] * len(_lib.AttentionArgs._fields_)
    names = [name for name, _ in _lib.AttentionArgs._fields_]
    for name, value in (("splits", -1), ("wait_kilocycles", 1 << 32), ("output_stride", -5), ("scale", "x")):
        values = list(good)
        values[names.index(name)] = value
        with pytest.raises(ValueError, match="slot_attention"):
            launch(0, *values)
