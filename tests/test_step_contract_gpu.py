"""What the operators round the selection path owe one another and their callers on the GPU: one rule of quantisation, indices of the
layout that are checked wherever they are used, block tables that carry the errors of a plan through, selection and drafted rows that show
every key once, and attention at the ends of its types."""
import numpy as np
import pytest
import torch

import step_reference as reference
from test_step_operators_gpu import HALF_STEP, attention_case, check_attention, host, visible_rows

pytestmark = pytest.mark.gpu


# ---- quantisation ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [128, 70])           # whole units of 16, and element by element
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, torch.float32])
def test_quantised_rows_are_the_rounded_quotients(device, kind, dim):
    """codes = x / scale, rounded to fp32 and to e4m3, bit for bit (position 0: nothing turns, so x is the row itself); NumPy's division is
    the correctly rounded one."""
    import kvip_b200 as kvip
    g = torch.Generator().manual_seed(dim)
    rows = (torch.randn((3000, 5, dim), generator=g) * torch.exp(torch.randn((3000, 5, 1), generator=g) * 2).clamp(1e-3, 50)).to(kind)
    codes, scales = kvip.Rotary(torch, 2, device).quantise(torch.zeros(3000, dtype=torch.int64, device=device), rows.to(device))
    x = rows.float().numpy()
    scale = (np.abs(x).max(-1) / np.float32(448)).astype(np.float32)
    assert np.array_equal(scales.cpu().numpy(), scale)
    quotient = torch.from_numpy(np.clip((x / scale[..., None]).astype(np.float32), -448, 448))
    assert torch.equal(codes.view(torch.uint8).cpu(), quotient.to(torch.float8_e4m3fn).view(torch.uint8))


@pytest.mark.parametrize("dim", [128, 70])
def test_quantised_rows_with_infinities_and_nan(device, dim):
    """An infinity makes its row's scale infinite: finite elements are 0 beside it, it is NaN itself. NaN stays NaN and does not scale."""
    import kvip_b200 as kvip
    rows = torch.ones((2, 2, dim), device=device)
    rows[0, 0, 9] = float("-inf")
    rows[1, 1, 11] = float("nan")
    codes, scales = kvip.Rotary(torch, 2, device).quantise(torch.zeros(2, dtype=torch.int64, device=device), rows)
    back = codes.float()
    expected = torch.full_like(rows, 448.0)
    expected[0, 0] = 0
    odd = torch.zeros_like(rows, dtype=torch.bool)
    odd[0, 0, 9] = odd[1, 1, 11] = True
    assert torch.equal(back.isnan(), odd) and torch.equal(back[~odd], expected[~odd])
    assert bool(scales[0, 0].isinf()) and torch.equal(scales.flatten()[1:], torch.full((3,), 1 / 448, device=device))


@pytest.mark.parametrize("smallest", [False, True])
def test_ingested_keys_are_the_quantised_rows(device, smallest):
    """`ingest_decode` of bf16 keys and `Rotary.quantise` of the same rows: the same codes and scales, down to the smallest rows. Codes are
    compared as values: -0 + 0 is +0, so a turned element of -0 (v cos 0 + u sin 0) has the other zero's code."""
    from types import SimpleNamespace

    import kvip_b200 as kvip
    tokens, history = 512, 1024
    inputs = kvip.QueryInputs(torch, tokens, device, history=history, queries=1)
    inputs.prepare((1,) * tokens, query_owners=tuple(range(1, tokens + 1)))
    positions = torch.arange(tokens, device=device)
    inputs.bind_positions(positions)
    g = torch.Generator(device=device)
    g.manual_seed(5)
    rows = torch.randn((tokens, 128), generator=g, device=device)
    if smallest:
        rows = rows.double() * torch.exp2(torch.linspace(-136, -100, tokens, dtype=torch.float64, device=device))[:, None]
        rows[:, ::7] = 0
    rows = rows.to(torch.bfloat16)
    storage = kvip.IndexCacheStorage(torch, tokens + 1, history, 256, device)
    storage.ingest_decode((rows, None), SimpleNamespace(slot_mapping=positions), inputs, inputs.row_owners)
    codes, scales = kvip.Rotary(torch, 2, device).quantise(torch.zeros_like(positions), rows[:, None])
    at = (positions + 1, positions)
    assert torch.equal(storage.scales[at], scales[:, 0])
    assert torch.equal(storage.keys[at].view(torch.float8_e4m3fn).float(), codes[:, 0].float())


# ---- slot maps and the layout of the query slots -----------------------------------------------------------------------
@pytest.mark.parametrize("counts,tokens", [([4] * 8, 16), ([4, 0, 3, 4, 1], 9), ([3, 3, 3], 8), ([4, 4], 1), ([2, 1], 3), ([2, 1], 11)])
def test_layout_ends_where_the_packed_tokens_end(device, counts, tokens):
    """Fewer output rows than packed tokens: what is dropped from positions, slots and starts is dropped from the layout as well."""
    import kvip_b200 as kvip
    batch, queries = len(counts), 4
    tables = kvip.BlockTables(torch, device, batch=batch, pages=2, blocks=2 * batch, tokens=tokens, block=16, queries=queries)
    tables.plan(torch.tensor(counts, dtype=torch.int32, device=device))
    owner = [(b, q) for b in range(batch) for q in range(counts[b])][:tokens]
    expected = np.zeros((4, batch * queries), np.int64)
    for t, (b, q) in enumerate(owner):
        expected[0, b * queries + q], expected[1, b * queries + q] = t, 1
        expected[2, t], expected[3, t] = b * queries + q, 1
    assert np.array_equal(tables.layout.cpu().numpy(), expected)
    assert int(tables.starts[-1]) == len(owner) and int(tables.status) == (1 if sum(counts) > tokens else 0)
    assert tables.requests.tolist() == [b for b, _ in owner] + [-1] * (tokens - len(owner))


@pytest.mark.parametrize("bf16", [False, True])
def test_ingest_skips_and_counts_what_is_out_of_range(device, bf16):
    """Slots, tokens, owners and positions out of range, one at a time among good rows: the good ones land, the storage keeps the rest."""
    from kvip_b200 import ops
    g = torch.Generator(device=device)
    g.manual_seed(0)
    owners, history, queries, batch, rows = 3, 256, 4, 5, 40
    source = (torch.randn((rows, 128), generator=g, device=device).to(torch.bfloat16) if bf16 else
              torch.randint(0, 120, (rows, 128), generator=g, device=device, dtype=torch.uint8))
    source_scales = None if bf16 else torch.rand(rows, generator=g, device=device)
    slots = torch.tensor([7, -1, 40, 3, 39, 1 << 40, 0], device=device)
    gather = torch.tensor([0, 1, 2, 3, 4, 5, 6, 7, -1, 0, 3, 1 << 35, 0, 3, 4, 6, 0, 3, 4, 6], device=device)
    ends = torch.tensor([10, 11, 12, 13, 256, 1, 257, 9, 9, 2, 3, 4, 20, 21, 0, 22, 30, 31, 32, 0], dtype=torch.int32, device=device)
    row_owners = torch.tensor([1, 2, 1, 3, -1], dtype=torch.int32, device=device)
    good = {0: 7, 3: 3, 4: 39, 9: 7, 10: 3}
    padding = [14, 19]
    keys = torch.randint(0, 120, (owners, history, 128), generator=g, device=device, dtype=torch.uint8)
    scales, errors = torch.rand((owners, history), generator=g, device=device), torch.zeros(1, dtype=torch.int32, device=device)
    want_keys, want_scales = keys.clone(), scales.clone()
    one = torch.zeros(1, dtype=torch.int64, device=device)
    for row, slot in [*good.items(), *((row, 0) for row in padding)]:
        if bf16:
            import kvip_b200 as kvip
            code, scale = kvip.Rotary(torch, 2, device).quantise(one, source[slot].view(1, 1, 128))
        else:
            code, scale = source[slot], source_scales[slot]
        at = (0, row) if row in padding else (int(row_owners[row // queries]), int(ends[row]) - 1)
        want_keys[at], want_scales[at] = code.view(torch.uint8).view(128), scale.view(())
    ops.ingest(keys, scales, source, source_scales, slots, gather, ends, row_owners, queries=queries, history=history, errors=errors)
    assert torch.equal(keys, want_keys) and torch.equal(scales, want_scales)
    assert int(errors) == 20 - len(good) - len(padding)
    with pytest.raises(ValueError, match="query slot"):
        ops.ingest(keys, scales, source, source_scales, slots, gather[:19], ends, row_owners, queries=queries, history=history)
    with pytest.raises(ValueError, match="history"):
        ops.ingest(keys, scales[:2], source, source_scales, slots, gather, ends, row_owners, queries=queries, history=history)


def test_ingest_padding_rows_stay_in_the_first_owner(device):
    """More query slots than owner 0 has positions: padding behind its last position is not written over the next owner's rows."""
    from kvip_b200 import ops
    keys = torch.full((2, 4, 128), 9, dtype=torch.uint8, device=device)
    scales = torch.full((2, 4), 5.0, device=device)
    source = torch.ones((1, 128), dtype=torch.uint8, device=device)
    zeros = torch.zeros(6, dtype=torch.int64, device=device)
    ops.ingest(keys, scales, source, torch.ones(1, device=device), zeros[:1], zeros, zeros.int(), zeros.int(), queries=1, history=4)
    assert bool((keys[0] == 1).all()) and bool((keys[1] == 9).all()) and bool((scales[1] == 5).all())


def test_packed_slots_of_no_token_are_not_live(device):
    """A layout whose indices leave the packed tensors: those slots have query end 0, whatever their valid word says."""
    import kvip_b200 as kvip
    inputs = kvip.QueryInputs(torch, 3, device, history=256, queries=2)
    layout = torch.tensor([[0, 2, 5, -1, 1, 1 << 40], [1] * 6, [0, 1, 2, 3, 4, 5], [1] * 6], device=device)
    inputs.prepare_device(layout, torch.tensor([1, 2, 3], dtype=torch.int32, device=device))
    assert inputs.bind_positions(torch.tensor([7, 8, 9], device=device)).tolist() == [[8, 10], [0, 0], [9, 0]]


def test_tokens_without_a_block_leave_the_index_rows_alone(device):
    """Tables with holes: the step's tokens have positions and slots of -1; their Index rows are not ingested, the others are."""
    from types import SimpleNamespace

    import kvip_b200 as kvip
    tables = kvip.BlockTables(torch, device, batch=2, pages=4, blocks=4, tokens=8, block=4, queries=4)
    tables.load(lengths=torch.tensor([3, 0]), held=torch.tensor([2, 0]), table=torch.tensor([[5, -1, -1, -1], [-1] * 4]), free=torch.tensor([6, -1, 8]))
    tables.plan(torch.tensor([3, 4], dtype=torch.int32, device=device))
    inputs = kvip.QueryInputs(torch, 2, device, history=128, queries=4)
    inputs.prepare_device(tables.layout, torch.tensor([1, 2], dtype=torch.int32, device=device))
    inputs.bind_positions(tables.positions)
    storage = kvip.IndexCacheStorage(torch, 3, 128, 128, device)
    cache = torch.arange(1, 9 * 4 + 1, device=device).to(torch.bfloat16)[:, None].expand(-1, 128).contiguous()
    storage.ingest_decode((cache, None), SimpleNamespace(slot_mapping=tables.slot_mapping), inputs, inputs.row_owners)
    assert tables.slot_mapping.tolist() == [23, -1, -1, 24, 25, 26, 27, -1]
    assert int(storage.ingest_errors) == 2
    expected = torch.tensor([[448.0, 448, 448, 24, 448], [25, 26, 27, 28, 448]]) / 448
    assert torch.equal(storage.scales[1:, :5].cpu(), expected)


def owned(t):
    """Blocks of all rows, then of the free list: each of them once, whatever happened."""
    rows = [int(x) for b in range(t.batch) for x in t.table[b, :int(t.held[b])]]
    return sorted(rows + t.free[int(t.head):].tolist())


def counts_of(device, *counts):
    return torch.tensor(counts, dtype=torch.int32, device=device)


def tables_of(device, lengths, held, table, free, *, block, tokens, head=0):
    """Tables in a given state; the free list has a place for every block."""
    import kvip_b200 as kvip
    tables = kvip.BlockTables(torch, device, batch=len(lengths), pages=len(table[0]), blocks=len(free), tokens=tokens, block=block)
    tables.load(lengths=torch.tensor(lengths), held=torch.tensor(held), table=torch.tensor(table), free=torch.tensor(free), head=head)
    return tables


def test_commit_keeps_nothing_of_a_request_without_blocks(device):
    """Three requests, blocks for one: the verifier returns a count for each of them all the same."""
    t = tables_of(device, [4, 4, 4], [1, 1, 1], [[0, -1, -1], [1, -1, -1], [2, -1, -1]], [9, 9, 9, 3], block=4, tokens=12, head=3)
    t.plan(counts_of(device, 2, 2, 2))
    assert int(t.status) == 4
    t.commit(counts_of(device, 2, 1, 2))
    assert t.lengths.tolist() == [6, 4, 4] and t.held.tolist() == [2, 1, 1] and owned(t) == [0, 1, 2, 3]
    assert int(t.status) == 4 | 1
    t.status.zero_()
    t.release([0])
    t.plan(counts_of(device, 0, 2, 2))
    assert int(t.status) == 0
    t.commit(counts_of(device, 0, 2, 2))
    assert t.lengths.tolist() == [0, 6, 6] and owned(t) == [0, 1, 2, 3] and int(t.status) == 0


def test_commit_keeps_no_token_that_was_dropped(device):
    t = tables_of(device, [0, 0], [0, 0], [[-1, -1], [-1, -1]], [0, 1, 2, 3], block=4, tokens=5)
    t.plan(counts_of(device, 4, 4))
    assert int(t.status) == 1
    t.commit(counts_of(device, 4, 4))
    assert t.lengths.tolist() == [4, 1]
    assert owned(t) == [0, 1, 2, 3]


def test_a_plan_is_committed_once(device):
    t = tables_of(device, [3], [1], [[0, -1, -1]], [9, 1, 2], block=4, tokens=4, head=1)
    t.plan(counts_of(device, 4))
    t.commit(counts_of(device, 1))
    assert t.lengths.tolist() == [4] and t.held.tolist() == [2] and int(t.status) == 0
    t.commit(counts_of(device, 0))
    assert int(t.status) == 0
    t.commit(counts_of(device, 3))
    assert t.lengths.tolist() == [4] and t.held.tolist() == [2] and int(t.head) == 2 and owned(t) == [0, 1, 2]
    assert int(t.status) == 1
    t.plan(counts_of(device, 2))
    assert int(t.taken) == 0                        # the block of the rejected tokens is still the request's
    t.commit(counts_of(device, -1))
    assert t.lengths.tolist() == [4]
    t.plan(counts_of(device, 2))
    t.commit(torch.tensor([2], device=device))      # int64 counts are taken as well
    assert t.lengths.tolist() == [6] and int(t.status) == 1
    for bad in (counts_of(device, 1, 2), torch.ones(1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="batch"):
            t.commit(bad)


@pytest.mark.parametrize("between", [False, True])
def test_release_between_a_plan_and_its_commit_puts_no_block_into_two_rows(device, between):
    """`release` ends the open plan; committed or not, every block stays in one place, and what was to be kept is reported."""
    t = tables_of(device, [4, 4], [1, 1], [[0, -1, -1], [1, -1, -1]], [9, 9, 2, 3, 4], block=4, tokens=8, head=2)
    t.plan(counts_of(device, 2, 2))
    if between:
        t.release([1])
        t.commit(counts_of(device, 2, 2))
        assert t.lengths.tolist() == [4, 0] and int(t.status) == 1
    else:
        t.commit(counts_of(device, 2, 2))
        t.release([1])
        assert t.lengths.tolist() == [6, 0] and int(t.status) == 0
    assert owned(t) == [0, 1, 2, 3, 4]
    t.plan(counts_of(device, 4, 8))
    t.commit(counts_of(device, 4, 8))
    assert owned(t) == [0, 1, 2, 3, 4] and t.held.tolist() == [3 if not between else 2, 2]


def test_block_tables_run_out_and_recover(device):
    """More requests than blocks: those without keep their lengths whatever is committed, from a captured graph too, and go on when blocks
    come back. Every block is in one place all the while."""
    import kvip_b200 as kvip
    batch, blocks = 4, 6
    tables = kvip.BlockTables(torch, device, batch=batch, pages=4, blocks=blocks, tokens=32, block=4, queries=4)
    counts, kept = (torch.full((batch,), n, dtype=torch.int32, device=device) for n in (4, 3))
    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        tables.plan(torch.zeros_like(counts)).commit(torch.zeros_like(counts))
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            tables.plan(counts).commit(kept)

        def whole():
            table, held = tables.table.cpu().numpy(), tables.held.cpu().numpy()
            rows = [int(x) for b in range(batch) for x in table[b, :held[b]]]
            return sorted(rows + tables.free[int(tables.head):].tolist()) == list(range(blocks))

        graph.replay()
        assert tables.lengths.tolist() == [3] * 4 and int(tables.status) == 0 and whole()
        graph.replay()                           # two blocks for four requests
        assert tables.lengths.tolist() == [6, 6, 3, 3] and int(tables.status) == 4 | 1 and whole()
        tables.status.zero_()
        tables.release([1])
        graph.replay()
        assert tables.lengths.tolist() == [9, 3, 3, 3] and tables.held.tolist() == [3, 1, 1, 1] and whole()


# ---- attention at the ends of its types ----------------------------------------------------------------------------------
@pytest.mark.parametrize("splits", [1, 2, 8])
@pytest.mark.parametrize("where", ["first tile", "middle", "all but one", "all"])
def test_attention_scores_of_minus_infinity_weigh_nothing(device, where, splits):
    """Finite queries and rows whose products leave fp32: scores of -inf in a head's first tile, in the middle of its list, in all of it. The
    rows that are left make the head's answer; the other heads do not notice."""
    import kvip_b200 as kvip
    entries, hot = 640, [0, 9, 17]
    case = attention_case(device, 51, counts=[1, 2], heads=24, entries=entries, stride=entries, context=[entries, entries], draft=False)
    case["slots"][:] = torch.arange(entries, dtype=torch.int32, device=device)
    low = torch.zeros(entries, dtype=torch.bool, device=device)
    low[{"first tile": slice(0, 64), "middle": slice(100, 400), "all but one": slice(0, entries), "all": slice(0, entries)}[where]] = True
    low[333] &= where != "all but one"
    pool = case["pool"].view(-1, entries, 576)
    pool[..., 0] = torch.where(low, -16.0, 0.0).to(torch.bfloat16)
    case["query"][:, hot, 0] = 2.0 ** 126
    attend = kvip.SlotAttention(torch, device, tokens=3, heads=24, entries=entries)
    out, lse = attend(**case, splits=splits)
    check_attention(dict(case, query=case["query"][:, [h for h in range(24) if h not in hot]]), out[:, [h for h in range(24) if h not in hot]],
                    lse[:, [h for h in range(24) if h not in hot]])
    for t in range(3):
        rows = host(visible_rows(case, t))[~low.cpu().numpy()]
        expected, log_sum, weight, size = reference.attention(host(case["query"][t, hot]), rows, case["scale"])
        if where == "all":
            assert bool((out[t, hot] == 0).all()) and bool((lse[t, hot] == float("-inf")).all())
            continue
        step, logit = HALF_STEP[torch.bfloat16], 577 * 2.0 ** -24 * size     # as in check_attention
        assert (np.abs(host(out[t, hot]) - expected) <= weight * (2 * step + 2 * logit + 2.0 ** -18) + np.abs(expected) * step + 1e-7).all()
        assert (np.abs(host(lse[t, hot]) - log_sum) <= logit + 2.0 ** -20 * (1 + np.abs(log_sum))).all()
    assert int(attend.status) == 0


@pytest.mark.parametrize("at", [0, 12345, -1])
@pytest.mark.parametrize("kind,entries,below", [(torch.float16, 1 << 18, 25.4), (torch.float16, 1 << 20, 25.4), (torch.float16, 1 << 20, 31.0),
                                                (torch.bfloat16, 1 << 18, 25.4), (torch.float16, 40000, 17.0)])
def test_attention_of_one_large_row_among_very_many_small_ones(device, kind, entries, below, at):
    """One row 2^below times as heavy as each of the others, whose values are 100 times its own: together they count. Closed form, with a
    list that names two pool rows over and over."""
    import kvip_b200 as kvip
    attend = kvip.SlotAttention(torch, device, tokens=1, heads=16, entries=entries, dtype=kind)
    pool = torch.zeros((128, 576), dtype=kind, device=device)
    pool[1, 0] = 4.0                               # the heavy row, by the first element, which the value of the others lacks too
    pool[0, 1:512], pool[1, 1:512] = 100.0, 1.0
    query = torch.zeros((1, 16, 576), dtype=kind, device=device)
    query[..., 0] = torch.linspace(0.5, 1, 16, device=device).to(kind)
    slots = torch.zeros((1, entries), dtype=torch.int32, device=device)
    slots[0, at] = 1
    scale = below * np.log(2.0) / 4
    logit = query[0, :, 0].double() * 4 * np.float64(np.float32(scale))
    rest = (entries - 1) * torch.exp(-logit)
    out, lse = attend(query, pool, slots, scale=scale, output_stride=128, requests=torch.zeros(1, dtype=torch.int32, device=device))
    expected = (1 + 100 * rest) / (1 + rest)
    # every weight half a step, the logit (two roundings in fp32, in the product and in units of log2) and exp2; sums in fp32: a thread adds an
    # entry in 32, the accumulators take four products a tile, whose sums may be cut (a whole step); one rounding of the output
    adds = entries / 32 * 2.0 ** -24 + entries / 16 * 2.0 ** -23
    tolerance = 2 * HALF_STEP[kind] + 3 * 2.0 ** -24 * below + 2.0 ** -21 + adds + HALF_STEP[kind]
    assert bool(((out[0, :, 1:].double() - expected[:, None]).abs() <= expected[:, None] * tolerance).all())
    log_sum = logit + torch.log1p(rest)
    assert bool(((lse[0].double() - log_sum).abs() <= 3 * 2.0 ** -24 * below + 2.0 ** -20 * (1 + log_sum) + adds).all())


@pytest.mark.parametrize("heads", [16, 64])
def test_attention_waits_give_up(device, heads):
    """Limits of one to a few kilocycles, which no tile's rows can meet everywhere: some call reports KVIP_ERR_PIPELINE, in one piece and in
    shares, over full lists and over tiles without rows; each call ends by itself, and the next one without a limit is right."""
    import kvip_b200 as kvip
    case = attention_case(device, 60, counts=[40, 24], heads=heads, entries=2048, stride=4096, context=[2048, 2048], draft=False)
    holes = dict(case, slots=case["slots"].clone())
    for tile in (0, 5, 31):
        holes["slots"][:, 64 * tile:64 * tile + 64] = -1
    holes["slots"][::2, 1024:] = -1
    attend = kvip.SlotAttention(torch, device, tokens=64, heads=heads)
    for now in (case, holes):
        for splits in (1, 4):
            seen = set()
            for limit in (1, 1, 2, 3):
                attend(**now, splits=splits, wait_kilocycles=limit)
                torch.cuda.synchronize()
                seen.add(int(attend.status))
                attend.status.zero_()
            assert seen <= {0, 32} and 32 in seen, (splits, seen)
            out, lse = attend(**now, splits=splits)
            check_attention(now, out, lse, tokens=range(0, 64, 7))
            assert int(attend.status) == 0
