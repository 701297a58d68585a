"""What the operators round the selection path refuse, and their host-side arithmetic: no device needed."""
import ctypes
import math

import numpy as np
import pytest
import torch

import step_reference as reference
from kvip_b200 import _lib, rotary


@pytest.fixture(scope="module")
def library():
    from kvip_b200.build import build_library
    build_library()
    return _lib.load_library()


def refused(library, name, args, word):
    assert getattr(library, name)(ctypes.byref(args), None) == _lib.BAD_ARGUMENT
    assert word.encode() in library.kvip_b200_last_error(), library.kvip_b200_last_error()


def filled(struct, **values):
    """An argument record whose every pointer is set (to an address that is never read: the checks come first)."""
    args = struct()
    for field, kind in struct._fields_:
        if kind is ctypes.c_void_p:
            setattr(args, field, 4096)
    for field, value in values.items():
        setattr(args, field, value)
    return args


MAPS = dict(batch=2, pages=8, blocks=4, tokens=16, block=16, queries=4)


@pytest.mark.parametrize("bad,word", [
    (dict(lengths=None), "null"), (dict(status=None), "null"), (dict(batch=0), "batch"), (dict(batch=1025), "batch"), (dict(pages=0), "pages"),
    (dict(block=0), "pages"), (dict(pages=1 << 20, block=1 << 12), "pages"), (dict(batch=1024, pages=1 << 20, block=1 << 10), "32 bits"),
    (dict(tokens=0), "tokens"), (dict(queries=5), "query slots"), (dict(queries=0), "query slots")])
def test_slot_maps_refusals(library, bad, word):
    refused(library, "kvip_b200_slot_maps", filled(_lib.SlotMapsArgs, **{**MAPS, **bad}), word)


ROTARY = dict(codes=None, heads0=4, heads1=1, tokens=3, width=64, dim=64, layout=0, dtype=0, factor=1.0, x_token0=256, x_head0=64, y_token0=256,
              y_head0=64, x_token1=64, y_token1=64)


@pytest.mark.parametrize("bad,word", [
    (dict(positions=None), "null"), (dict(y0=None), "null output"), (dict(y1=None), "null output"), (dict(x1=None), "second set"),
    (dict(heads1=0), "second set"), (dict(tokens=0), "token"), (dict(heads0=0), "head"), (dict(width=63), "even"), (dict(width=0), "even"),
    (dict(width=1026), "even"), (dict(layout=2), "layout"), (dict(dtype=3), "type"), (dict(codes=4096, scales=None), "null output"),
    (dict(codes=4096, dim=32, heads1=0), "quantised"), (dict(codes=4096, dim=5000, heads1=0), "quantised"), (dict(codes=4096, dim=128), "quantised"),
    (dict(heads0=65537), "65536"), (dict(y_head0=0), "overlap"), (dict(y_token0=0), "overlap"), (dict(y_head0=63), "overlap"),
    (dict(y_token0=255), "overlap"), (dict(y_token1=32), "overlap"), (dict(y_token0=64, y_head0=128), "overlap")])
def test_rotary_refusals(library, bad, word):
    refused(library, "kvip_b200_rotary", filled(_lib.RotaryArgs, **{**ROTARY, **bad}), word)


ATTENTION = dict(query_token=128 * 576, query_head=576, draft_token=576, pool_rows=8192, tokens=4, heads=128, entries=2048, batch=2, queries=2,
                 output_stride=4096, dtype=0, splits=0, scale=0.1)


@pytest.mark.parametrize("bad,word", [
    (dict(query=None), "null"), (dict(lse=None), "null"), (dict(tokens=0), "tokens"), (dict(heads=129), "heads"), (dict(heads=0), "heads"),
    (dict(entries=0), "entries"), (dict(batch=0), "requests"), (dict(requests=None, batch=1), "requests"), (dict(output_stride=0), "pool"),
    (dict(output_stride=8193), "pool"), (dict(starts=None), "starts"), (dict(dtype=2), "bf16"), (dict(query=4104), "aligned"),
    (dict(query_token=4), "aligned"), (dict(draft=4104), "aligned"), (dict(draft_token=578), "aligned"),
    (dict(splits=3), "shares"), (dict(splits=16), "shares"), (dict(pool_rows=1 << 31), "pool"), (dict(entries=(1 << 20) + 1), "entries")])
def test_attention_refusals(library, bad, word):
    refused(library, "kvip_b200_slot_attention", filled(_lib.AttentionArgs, **{**ATTENTION, **bad}), word)


VERIFY = dict(target_row=100, draft_row=100, rows=4, vocabulary=100, batch=2, depth=3, dtype=2)


@pytest.mark.parametrize("bad,word", [
    (dict(target=None), "null"), (dict(out_counts=None), "null"), (dict(rows=0), "row"), (dict(vocabulary=0), "vocabulary"),
    (dict(vocabulary=(1 << 24) + 1), "vocabulary"), (dict(batch=0), "requests"), (dict(batch=65537), "requests"), (dict(depth=0), "depth"),
    (dict(depth=64), "depth"), (dict(dtype=3), "type")])
def test_verify_refusals(library, bad, word):
    refused(library, "kvip_b200_verify_drafts", filled(_lib.VerifyArgs, **{**VERIFY, **bad}), word)


def test_objects_refuse_the_cpu_and_bad_geometry():
    import kvip_b200 as kvip
    cpu = torch.device("cpu")
    for make in (lambda d, **k: kvip.Rotary(torch, 64, d, **k), lambda d: kvip.BlockTables(torch, d, batch=1, pages=1, blocks=1, tokens=1),
                 lambda d: kvip.SlotAttention(torch, d, tokens=1, heads=1), lambda d: kvip.DraftVerifier(torch, d, batch=1)):
        with pytest.raises(ValueError, match="CUDA"):
            make(cpu)
    cuda = torch.device("cuda", 0)      # refused before anything touches the device
    for make in (lambda: kvip.Rotary(torch, 63, cuda), lambda: kvip.Rotary(torch, 1026, cuda), lambda: kvip.Rotary(torch, 64, cuda, layout="x"),
                 lambda: kvip.Rotary(torch, 64, cuda, scaling={"kind": "other"}), lambda: kvip.Rotary(torch, 64, cuda, scaling={"kind": "linear", "factor": 0.5}),
                 lambda: kvip.Rotary(torch, 64, cuda, scaling={"kind": "yarn", "factor": 4.0}),
                 lambda: kvip.Rotary(torch, 64, cuda, scaling={"kind": "yarn", "factor": 4.0, "original": 4096, "beta_fast": 1.0, "beta_slow": 2.0}),
                 lambda: kvip.BlockTables(torch, cuda, batch=1025, pages=1, blocks=1, tokens=1),
                 lambda: kvip.BlockTables(torch, cuda, batch=1, pages=0, blocks=1, tokens=1),
                 lambda: kvip.BlockTables(torch, cuda, batch=1, pages=1 << 20, blocks=1, tokens=1, block=1 << 12),
                 lambda: kvip.BlockTables(torch, cuda, batch=1, pages=1, blocks=1, tokens=1, queries=5),
                 lambda: kvip.SlotAttention(torch, cuda, tokens=1, heads=129), lambda: kvip.SlotAttention(torch, cuda, tokens=0, heads=1),
                 lambda: kvip.SlotAttention(torch, cuda, tokens=1, heads=1, entries=0),
                 lambda: kvip.SlotAttention(torch, cuda, tokens=1, heads=1, dtype=torch.float32),
                 lambda: kvip.DraftVerifier(torch, cuda, batch=0), lambda: kvip.DraftVerifier(torch, cuda, batch=1, depth=64)):
        with pytest.raises(ValueError):
            make()


@pytest.mark.parametrize("head,status", [(3, 0), (2, 4), (0, 4), (9, 4)])
def test_released_blocks_find_a_place_in_the_list_or_are_reported(head, status):
    """`release` with host tensors: a list that has handed out three blocks takes three back; one that has handed out fewer (rows loaded
    with blocks from elsewhere), or whose head lies behind its end, drops what has no place and says so."""
    from kvip_b200 import BlockTables
    tables = BlockTables.__new__(BlockTables)
    tables.torch, tables.device, tables.batch, tables.blocks, tables.pages = torch, torch.device("cpu"), 2, 6, 4
    tables.table = torch.tensor([[7, 8, -1, -1], [9, -1, -1, -1]], dtype=torch.int32)
    tables.held, tables.lengths = torch.tensor([2, 1], dtype=torch.int32), torch.tensor([20, 3], dtype=torch.int32)
    tables.free, tables.head = torch.arange(100, 106, dtype=torch.int32), torch.tensor([head], dtype=torch.int32)
    tables.status = torch.zeros(1, dtype=torch.int32)
    tables.release([0, 1])
    assert int(tables.status) == status
    assert int(tables.head) == max(0, head - 3) and int(tables.held.sum()) == 0 and int(tables.table.max()) == -1
    free = tables.free.tolist()
    if head == 3:
        assert free == [7, 8, 9, 103, 104, 105]
    elif head == 2:
        assert free == [8, 9, 102, 103, 104, 105]
    else:
        assert free == list(range(100, 106))


def test_rotary_frequencies():
    for width in (2, 64, 128):
        for scaling in (None, {"kind": "linear", "factor": 8.0}, {"kind": "yarn", "factor": 40.0, "original": 4096},
                        {"kind": "yarn", "factor": 4.0, "original": 32768, "beta_fast": 16, "beta_slow": 2, "attention_factor": 1.0}):
            pairs, factor = rotary.frequencies(width, 10000.0, scaling)
            expected, other = reference.rotary_frequencies(width, 10000.0, scaling)
            assert np.allclose(pairs, expected, rtol=1e-14, atol=0) and factor == other
    pairs, factor = rotary.frequencies(128, 10000.0, {"kind": "yarn", "factor": 40.0, "original": 4096})
    plain, _ = rotary.frequencies(128)
    assert pairs[0] == plain[0] and math.isclose(pairs[-1], plain[-1] / 40) and math.isclose(factor, 0.1 * math.log(40) + 1)


def test_reference_walk_keeps_the_targets_distribution():
    """The rule itself, by sums: one drafted child, then two, over every outcome of a small vocabulary."""
    rng = np.random.default_rng(0)
    p, q = rng.dirichlet(np.ones(5)), rng.dirichlet(np.ones(5))
    for children in (1, 2):
        out = np.zeros(5)

        def walk(r, z, left, weight):
            if left == 0:
                out[:] += weight * r / r.sum()
                return
            rest = np.maximum(r - z * q, 0)
            for token in range(5):
                good = min(1.0, r[token] / (q[token] * z))
                out[token] += weight * q[token] * good
                if good < 1:
                    walk(rest, rest.sum(), left - 1, weight * q[token] * (1 - good))

        walk(p, 1.0, children, 1.0)
        assert np.allclose(out, p, atol=1e-12)
