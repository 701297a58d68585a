"""The operators round the selection path on the GPU, against their restatements in 64 bits (tests/step_reference.py):
slot maps, rotary positions, attention over selected slots with drafted tokens, verification of drafted tokens."""
import numpy as np
import pytest
import torch

import step_reference as reference

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def host(t):
    return t.detach().float().cpu().numpy().astype(np.float64) if t.is_floating_point() and t.dtype != torch.float64 else t.cpu().numpy()


# ---- slot maps ------------------------------------------------------------------------------------------------------
def make_tables(device, rng, *, batch, pages, block, tokens, counts, lengths=None, held=None, spare=3, queries=0):
    import kvip_b200 as kvip
    counts = np.asarray(counts, np.int32)
    lengths = rng.integers(0, pages * block - np.maximum(counts, 0) + 1).astype(np.int32) if lengths is None else np.asarray(lengths, np.int32)
    held = (-(-lengths // block)).astype(np.int32) if held is None else np.asarray(held, np.int32)
    need = np.maximum(0, -(-(lengths.astype(np.int64) + np.maximum(counts, 0)) // block) - held)
    own = int(np.clip(held, 0, pages).sum())
    free_count = max(0, int(need.sum()) + spare)
    order = rng.permutation(own + free_count + 7).astype(np.int32)
    table = np.full((batch, pages), -1, np.int32)
    at = 0
    for b in range(batch):
        n = int(np.clip(held[b], 0, pages))
        table[b, :n] = order[at:at + n]
        at += n
    free = order[at:at + free_count]
    tables = kvip.BlockTables(torch, device, batch=batch, pages=pages, blocks=max(1, free_count), tokens=tokens, block=block, queries=queries)
    tables.load(lengths=torch.from_numpy(lengths), held=torch.from_numpy(held), table=torch.from_numpy(table), free=torch.from_numpy(free))
    expected = reference.slot_maps(lengths, counts, held, table, tables.free.cpu().numpy()[:max(1, free_count)] if free_count else
                                   np.zeros(0, np.int32), int(tables.head.item()) if free_count else 0, block=block, tokens=tokens, queries=queries)
    return tables, torch.from_numpy(counts).to(device), expected


def check_maps(tables, expected):
    torch.cuda.synchronize()
    for name, value in expected.items():
        got = getattr(tables, name).cpu().numpy()
        assert np.array_equal(got, value), (name, got, value)


@pytest.mark.parametrize("batch,pages,block,tokens,most", [
    (1, 1, 1, 1, 1), (1, 1024, 128, 1, 1), (3, 7, 16, 40, 9), (64, 1024, 128, 256, 4), (257, 33, 64, 3000, 17), (1000, 200, 16, 20011, 40),
    (1024, 64, 128, 4096, 4), (5, 2048, 128, 131072, 20000)])
def test_slot_maps_match_the_restatement(device, batch, pages, block, tokens, most):
    rng = np.random.default_rng(batch + pages)
    most = min(most, pages * block, max(1, tokens // batch))
    counts = rng.integers(0, most + 1, batch)
    tables, counts, expected = make_tables(device, rng, batch=batch, pages=pages, block=block, tokens=tokens, counts=counts)
    assert tables.plan(counts) is tables
    check_maps(tables, expected)
    tables.plan(counts)            # a step planned again plans the same
    check_maps(tables, expected)


def test_slot_maps_blocks_held_from_a_rejected_step_are_used_first(device):
    rng = np.random.default_rng(3)
    tables, counts, expected = make_tables(device, rng, batch=4, pages=9, block=16, tokens=32, counts=[4, 0, 16, 2],
                                           lengths=[15, 16, 0, 31], held=[3, 1, 0, 2])
    tables.plan(counts)
    check_maps(tables, expected)
    assert expected["taken"][0] == 2 and expected["held_after"].tolist() == [3, 1, 1, 3]


@pytest.mark.parametrize("counts,lengths,held,spare,tokens,status", [
    ([3, 200, 2], [5, 0, 9], [1, 0, 1], 0, 64, 1),        # longer than its row
    ([3, -1, 2], [5, 4, 9], [1, 1, 1], 0, 64, 1),         # negative count
    ([3, 1, 2], [5, -4, 9], [1, 1, 1], 0, 64, 1),         # negative length
    ([30, 20, 2], [5, 4, 9], [1, 1, 1], -3, 64, 4),       # the free list is short
    ([30, 20, 2], [5, 4, 9], [1, 1, 1], 0, 20, 1),        # more tokens than the outputs hold
    ([2147483647, 1, 1], [2147483647, 1, 1], [0, 1, 1], 0, 8, 1)])
def test_slot_maps_report_what_does_not_fit(device, counts, lengths, held, spare, tokens, status):
    rng = np.random.default_rng(5)
    if counts[0] == 2147483647:
        import kvip_b200 as kvip
        tables = kvip.BlockTables(torch, device, batch=3, pages=8, blocks=4, tokens=tokens, block=16)
        tables.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        tables.held.copy_(torch.tensor(held, dtype=torch.int32))
        tables.table[1:, 0] = torch.tensor([7, 9], dtype=torch.int32)
        expected = reference.slot_maps(lengths, counts, held, tables.table.cpu().numpy(), np.arange(4, dtype=np.int32), 0, block=16, tokens=tokens)
        counts = torch.tensor(counts, dtype=torch.int32, device=device)
    else:
        tables, counts, expected = make_tables(device, rng, batch=3, pages=8, block=16, tokens=tokens, counts=counts, lengths=lengths,
                                               held=held, spare=spare)
    tables.plan(counts)
    assert expected["status"][0] == status
    check_maps(tables, expected)


def test_slot_maps_report_rows_and_lists_with_holes(device):
    """A row that lacks a block it is said to hold, and a free list with no block in a place: slot -1, position as ever, and the status."""
    import kvip_b200 as kvip
    tables = kvip.BlockTables(torch, device, batch=2, pages=4, blocks=4, tokens=8, block=4)
    tables.load(lengths=torch.tensor([3, 0]), held=torch.tensor([2, 0]), table=torch.tensor([[5, -1, -1, -1], [-1] * 4]), free=torch.tensor([6, -1, 8]))
    tables.plan(torch.tensor([3, 5], dtype=torch.int32, device=device))
    assert tables.positions.tolist() == [3, 4, 5, 0, 1, 2, 3, 4]
    assert tables.slot_mapping.tolist() == [23, -1, -1, 24, 25, 26, 27, -1]
    assert int(tables.status) == 4 and int(tables.taken) == 2


def test_slot_maps_layout_is_the_query_inputs_layout(device):
    from kvip_b200.inputs import slot_layout
    rng = np.random.default_rng(9)
    counts = rng.integers(0, 5, 33)
    tables, device_counts, expected = make_tables(device, rng, batch=33, pages=16, block=128, tokens=132, counts=counts, queries=4)
    tables.plan(device_counts)
    check_maps(tables, expected)
    layout, total = slot_layout(tuple(int(n) for n in counts), batch=33, queries=4)
    assert np.array_equal(tables.layout.cpu().numpy(), layout[:4]) and int(tables.starts[-1]) == total


def test_block_tables_live_through_steps_releases_and_a_graph(device):
    """Plan, keep some of the tokens, plan again, release requests and reuse their blocks: no block is ever in two rows,
    every token of the cache keeps its slot. The plan runs from a captured graph, on a stream of its own."""
    import kvip_b200 as kvip
    batch, pages, block = 6, 12, 4
    tables = kvip.BlockTables(torch, device, batch=batch, pages=pages, blocks=40, tokens=24, block=block)
    counts = torch.zeros(batch, dtype=torch.int32, device=device)
    stream = torch.cuda.Stream(device)
    with torch.cuda.stream(stream):
        tables.plan(counts)
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            tables.plan(counts)
    rng = np.random.default_rng(1)
    where = {}
    with torch.cuda.stream(stream):
        for step in range(14):
            n = rng.integers(0, 5, batch)
            n = np.minimum(n, pages * block - tables.lengths.cpu().numpy())
            counts.copy_(torch.from_numpy(n.astype(np.int32)))
            before = tables.lengths.cpu().numpy()
            graph.replay()
            slots, starts = tables.slot_mapping.cpu().numpy(), tables.starts.cpu().numpy()
            kept = np.minimum(n, rng.integers(0, 5, batch))
            for b in range(batch):
                for i in range(int(kept[b])):
                    where[(b, int(before[b]) + i)] = int(slots[starts[b] + i])
            tables.commit(torch.from_numpy(kept.astype(np.int32)).to(device))
            if step in (5, 9):
                gone = [1, 4]
                tables.release(gone)
                where = {k: v for k, v in where.items() if k[0] not in gone}
            table, held = tables.table.cpu().numpy(), tables.held.cpu().numpy()
            owned = [int(x) for b in range(batch) for x in table[b, :held[b]]]
            listed = tables.free.cpu().numpy()[int(tables.head.item()):40].tolist()
            assert sorted(owned + listed) == list(range(40))
            for (b, p), slot in where.items():
                assert int(table[b, p // block]) * block + p % block == slot
    assert int(tables.status.item()) == 0


# ---- rotary ---------------------------------------------------------------------------------------------------------
YARN = {"kind": "yarn", "factor": 16.0, "original": 4096}


def rotary_tolerance(y, size, kind, longest):
    # cos and sin carry an error of 2^-22 (angle reduced in fp64, 2 ulp), two products and a sum in fp32; one rounding at the end.
    # The angle itself, up to `longest` radians, is a product in fp64 here and there: the frequency (a power, 2 half ulp), the
    # product (1), and on the GPU 2 pi (1), the quotient (1) and the product (1) are 8 relative errors of 2^-53 with the pair's
    # other one. At 2^21 that is 2^-29 and does not count, at 2^34 it is 2^-16.
    return size * (2.0 ** -20 + 8 * longest * 2.0 ** -53) + np.abs(y) * HALF_STEP[kind] + 1e-30


@pytest.mark.parametrize("tokens,heads,width,pad,layout,kind,scaling,longest", [
    (1, 1, 2, 0, "half", torch.float32, None, 10), (1, 128, 64, 512, "interleaved", torch.bfloat16, YARN, 1 << 17),
    (64, 64, 64, 64, "half", torch.bfloat16, None, 1 << 21), (37, 5, 96, 3, "interleaved", torch.float16, YARN, 1 << 20),
    (33, 3, 6, 1, "half", torch.bfloat16, {"kind": "linear", "factor": 4.0}, 5000), (130, 16, 128, 0, "half", torch.float32, YARN, 1 << 34),
    (9, 7, 128, 0, "interleaved", torch.bfloat16, None, 1 << 21), (700, 33, 64, 0, "interleaved", torch.float16, None, 1 << 16),
    (5, 2, 1024, 0, "half", torch.bfloat16, None, 1 << 16), (257, 9, 32, 32, "half", torch.float32, None, 1 << 21)])
def test_rotary_matches_the_definition(device, tokens, heads, width, pad, layout, kind, scaling, longest):
    """Rotated rows inside longer rows (odd strides among them), in place and into other tensors, with one key head."""
    import kvip_b200 as kvip
    g = torch.Generator(device=device)
    g.manual_seed(tokens)
    positions = torch.randint(0, longest, (tokens,), generator=g, device=device)
    positions[0] = longest - 1
    query = torch.randn((tokens, heads, width + pad), generator=g, device=device).to(kind)
    key = torch.randn((tokens, width + pad), generator=g, device=device).to(kind)
    rope = kvip.Rotary(torch, width, device, layout=layout, scaling=scaling)
    views = query[..., pad:], key[..., pad:]
    out = torch.full((tokens, heads, width), 7.0, dtype=kind, device=device), torch.full((tokens, width), 7.0, dtype=kind, device=device)
    saved = query.clone(), key.clone()
    got = rope(positions, *views, query_out=out[0], key_out=out[1])
    assert got[0] is out[0] and got[1] is out[1]
    assert torch.equal(query, saved[0]) and torch.equal(key, saved[1])
    p = positions.cpu().numpy()
    for x, y in zip((views[0], views[1][:, None]), (out[0], out[1][:, None])):
        expected, size = reference.rotary(host(x), p, width, layout, scaling=scaling)
        assert (np.abs(host(y) - expected) <= rotary_tolerance(expected, size, kind, longest)).all()
    rope(positions, *views)        # in place: the same numbers, and nothing beside them moves
    assert torch.equal(views[0], out[0]) and torch.equal(views[1], out[1])
    assert torch.equal(query[..., :pad], saved[0][..., :pad]) and torch.equal(key[..., :pad], saved[1][..., :pad])


def test_rotary_leaves_padding_rows_alone(device):
    import kvip_b200 as kvip
    g = torch.Generator(device=device)
    g.manual_seed(0)
    positions = torch.tensor([4, -1, 0, 9, -1], device=device)
    rows = torch.randn((5, 8, 64), generator=g, device=device).to(torch.bfloat16)
    before = rows.clone()
    rope = kvip.Rotary(torch, 64, device)
    rope(positions, rows)
    assert torch.equal(rows[1], before[1]) and torch.equal(rows[4], before[4]) and not torch.equal(rows[0], before[0])
    assert torch.equal(rows[2], before[2])          # position zero turns nothing
    codes = torch.full((5, 8, 64), 5, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    scales = torch.full((5, 8), 3.0, device=device)
    rope.quantise(positions, before, codes, scales)
    assert (scales[[1, 4]] == 3.0).all() and (codes.view(torch.uint8)[[1, 4]] == 5).all() and (scales[[0, 2, 3]] != 3.0).all()


def test_rotary_head_major_and_broadcast_rows(device):
    """Rows whose heads lie further apart than their tokens; an input that is one row for all heads; an output that would be."""
    import kvip_b200 as kvip
    g = torch.Generator(device=device)
    g.manual_seed(6)
    rope = kvip.Rotary(torch, 64, device, layout="interleaved")
    positions = torch.randint(0, 1 << 20, (10,), generator=g, device=device)
    rows = torch.randn((6, 10, 64), generator=g, device=device).to(torch.bfloat16).transpose(0, 1)
    out = torch.empty((6, 10, 64), dtype=torch.bfloat16, device=device).transpose(0, 1)
    rope(positions, rows, query_out=out)
    expected, size = reference.rotary(host(rows), positions.cpu().numpy(), 64, "interleaved")
    assert (np.abs(host(out) - expected) <= rotary_tolerance(expected, size, torch.bfloat16, 1 << 20)).all()
    one = rows[:, :1].expand(10, 6, 64)
    rope(positions, one, query_out=out)
    assert torch.equal(out[:, 0], out[:, 5])
    with pytest.raises(ValueError, match="overlap"):
        rope(positions, one)


@pytest.mark.parametrize("tokens,heads,dim,width,layout,kind,stride", [
    (1, 64, 128, 64, "half", torch.bfloat16, 0), (64, 64, 128, 64, "half", torch.bfloat16, 0), (33, 32, 128, 128, "interleaved", torch.float16, 0),
    (7, 3, 130, 64, "half", torch.bfloat16, 0), (65, 1, 128, 32, "half", torch.float32, 8), (5, 64, 128, 64, "interleaved", torch.bfloat16, 1),
    (900, 32, 128, 64, "half", torch.bfloat16, 64), (3, 2, 64, 64, "half", torch.bfloat16, 0), (4, 5, 256, 64, "interleaved", torch.float32, 0),
    (2, 3, 40, 6, "half", torch.float32, 0), (3, 4, 512, 64, "half", torch.float16, 0)])
def test_rotary_quantised_rows(device, tokens, heads, dim, width, layout, kind, stride):
    import kvip_b200 as kvip
    g = torch.Generator(device=device)
    g.manual_seed(dim)
    positions = torch.randint(0, 1 << 20, (tokens,), generator=g, device=device)
    whole = (torch.randn((tokens, heads, dim + stride), generator=g, device=device)
             * torch.exp(torch.randn((tokens, heads, 1), generator=g, device=device) * 3).clamp(1e-3, 50)).to(kind)
    rows = whole[..., stride:]
    rows[-1, -1] = 0
    rope = kvip.Rotary(torch, width, device, layout=layout)
    codes, scales = rope.quantise(positions, rows)
    expected, size = reference.rotary(host(rows), positions.cpu().numpy(), width, layout)
    error = size * 2.0 ** -20
    amax = np.abs(expected).max(-1)
    scale = np.where(amax > 0, amax / 448, 1.0)
    got_scale, got = host(scales), host(codes.float())
    # scale: the error of the largest value, and two fp32 roundings; codes: half a step (2^-4 relative, 2^-10 below the normal range)
    assert (np.abs(got_scale - scale) <= scale * 2.0 ** -19).all()
    value = got * got_scale[..., None]
    assert (np.abs(value - expected) <= np.abs(expected) * (2.0 ** -4 + 2.0 ** -18) + scale[..., None] * 2.0 ** -10 + error).all()
    assert (np.abs(got).max(-1)[amax > 0] == 448).all() and (got[-1, -1] == 0).all() and got_scale[-1, -1] == 1


@pytest.mark.parametrize("dim", [128, 70])
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
def test_rotary_quantised_rows_near_the_smallest_numbers(device, kind, dim):
    """Rows whose largest element is anything from 2^-133 to 2^-110, among zeros, at position 0 (nothing turns: cos 1, sin 0). Zeros stay
    zeros; every element comes back within its e4m3 rounding, 2^-4 relative or half of the smallest step 2^-9 in units of the scale, and
    two fp32 roundings (the reciprocal and the product, 2^-23 together)."""
    import kvip_b200 as kvip
    exponents = torch.arange(-133, -109, dtype=torch.float64)
    rows = torch.zeros((exponents.numel(), 2, dim), dtype=torch.float64)
    rows[:, 0, ::3] = torch.linspace(-1, 1, len(range(0, dim, 3)), dtype=torch.float64)
    rows[:, 1, 5] = 1.0
    rows = (rows * torch.exp2(exponents)[:, None, None]).to(kind).to(device)
    turn = kvip.Rotary(torch, 64 if dim == 128 else 6, device)
    codes, scales = turn.quantise(torch.zeros(exponents.numel(), dtype=torch.int64, device=device), rows)
    exact, most = rows.double(), rows.float().abs().amax(-1)
    assert torch.equal(scales, torch.where(most > 0, (most / 448).clamp(min=2.0 ** -126), 1.0))
    back = codes.float().double() * scales.double()[..., None]
    assert bool(((back - exact).abs() <= exact.abs() * (2.0 ** -4 + 2.0 ** -22) + scales.double()[..., None] * 2.0 ** -10 * (1 + 2.0 ** -22)).all())
    assert bool((codes.float()[exact == 0] == 0).all())


def test_rotary_feeds_the_ingested_index_keys(device):
    """Keys rotated in place and ingested equal the rows that `quantise` makes (one rule of quantisation)."""
    from types import SimpleNamespace

    import kvip_b200 as kvip
    g = torch.Generator(device=device)
    g.manual_seed(4)
    tokens = 8
    inputs = kvip.QueryInputs(torch, tokens, device, history=256, queries=1)
    inputs.prepare((1,) * tokens, query_owners=tuple(range(tokens)))
    positions = torch.arange(tokens, device=device) * 5
    inputs.bind_positions(positions)
    keys = torch.randn((tokens, 128), generator=g, device=device)
    rope = kvip.Rotary(torch, 64, device)
    storage = kvip.IndexCacheStorage(torch, tokens, 256, 128, device)
    rotated = keys.to(torch.bfloat16)
    rope(positions, rotated[:, :64])
    storage.ingest_decode((rotated, None), SimpleNamespace(slot_mapping=torch.arange(tokens, device=device)), inputs, inputs.row_owners)
    still = kvip.Rotary(torch, 2, device)
    codes, scales = still.quantise(torch.zeros_like(positions), rotated[:, None])     # position 0: quantise alone
    at = (torch.arange(tokens, device=device), positions)
    assert torch.equal(storage.scales[at], scales[:, 0])
    got, want = storage.keys[at].view(torch.float8_e4m3fn).float(), codes[:, 0].float()
    # one rule, but x / scale there and x * (1 / scale) here: a value next to a border may fall on its other side
    assert ((got - want).abs() <= want.abs() * 2.0 ** -3 + 2.0 ** -9).all() and (got != want).float().mean() < 0.01


# ---- attention --------------------------------------------------------------------------------------------------------
def attention_case(device, seed, *, counts, heads, entries, stride, context, kind=torch.bfloat16, draft=True, tree=True, spread=1.0,
                   owners=None, holes=0.0, pool_rows=None):
    rng = np.random.default_rng(seed)
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    batch, tokens = len(counts), int(sum(counts))
    owners = rng.permutation(batch).astype(np.int32) if owners is None else np.asarray(owners, np.int32)
    starts = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    requests = np.repeat(np.arange(batch), counts).astype(np.int32)
    pool = torch.randn((pool_rows or (int(owners.max()) + 1) * stride, 576), generator=g, device=device).to(kind)
    context = np.broadcast_to(np.asarray(context), (batch,))
    slots = np.full((tokens, entries), -1, np.int32)
    for t in range(tokens):
        n = min(int(context[requests[t]]), entries)
        slots[t, :n] = rng.permutation(stride)[:n] if n <= stride else rng.integers(0, stride, n)
        slots[t, rng.random(entries) < holes] = -1
    ancestors = np.zeros(tokens, np.int64)
    for t in range(tokens):
        j = t - starts[requests[t]]
        parent = (j - 1 if not tree else int(rng.integers(0, j))) if j else -1
        own = 0 if j > 63 else (1 << int(j)) - (1 << 64 if j == 63 else 0)
        ancestors[t] = own | (int(ancestors[starts[requests[t]] + parent]) if j else 0)
    case = dict(
        query=(torch.randn((tokens, heads, 576), generator=g, device=device) * spread).to(kind), pool=pool,
        slots=torch.from_numpy(slots).to(device), requests=torch.from_numpy(requests).to(device),
        row_owners=torch.from_numpy(owners).to(device), output_stride=stride, scale=0.07)
    if draft:
        case.update(starts=torch.from_numpy(starts).to(device), draft=torch.randn((tokens, 576), generator=g, device=device).to(kind),
                    ancestors=torch.from_numpy(ancestors).to(device))
    return case


def visible_rows(case, t):
    """Pool rows, then drafted rows, that token t sees (as a torch tensor)."""
    request = int(case["requests"][t])
    owner = int(case["row_owners"][request])
    slots = case["slots"][t].reshape(-1)
    slots = slots[(slots >= 0) & (slots < case["output_stride"])].long()
    rows = case["pool"][owner * case["output_stride"] + slots]
    if case.get("draft") is not None:
        first, behind = int(case["starts"][request]), int(case["starts"][request + 1])
        mask = int(case["ancestors"][t]) if case.get("ancestors") is not None else (2 << (t - first)) - 1
        chosen = [first + j for j in range(min(64, behind - first)) if mask >> j & 1]
        rows = torch.cat((rows, case["draft"][chosen]))
    return rows


def check_attention(case, out, lse, tokens=None):
    torch.cuda.synchronize()
    kind = case["query"].dtype
    step = HALF_STEP[kind]
    for t in range(case["query"].shape[0]) if tokens is None else tokens:
        expected, log_sum, weight, size = reference.attention(host(case["query"][t]), host(visible_rows(case, t)), case["scale"])
        # logits: 576 products summed in fp32; the weights are rounded to the rows' type once, the output once; the sum of
        # the weights is that of the rounded ones or of exact ones (one more half step); exp2 and the rest in fp32
        logit = 577 * 2.0 ** -24 * size
        tolerance = weight * (2 * step + 2 * logit + 2.0 ** -18) + np.abs(expected) * step + 1e-7
        assert (np.abs(host(out[t]) - expected) <= tolerance).all(), (t, np.abs(host(out[t]) - expected).max())
        got = host(lse[t])
        assert np.array_equal(np.isinf(got), np.isinf(log_sum))
        fine = np.isfinite(log_sum)
        assert (np.abs(got[fine] - log_sum[fine]) <= logit + 2.0 ** -20 * (1 + np.abs(log_sum[fine]))).all()


def run_attention(case, device, **more):
    import kvip_b200 as kvip
    attend = kvip.SlotAttention(torch, device, tokens=case["query"].shape[0], heads=case["query"].shape[1],
                                entries=case["slots"].shape[-1], dtype=case["query"].dtype)
    out, lse = attend(**case, **more)
    return attend, out, lse


@pytest.mark.parametrize("heads", [1, 3, 8, 16, 17, 32, 40, 64, 65, 96, 100, 128])
def test_attention_heads(device, heads):
    case = attention_case(device, heads, counts=[2, 1, 3], heads=heads, entries=300, stride=512, context=[300, 77, 512])
    attend, out, lse = run_attention(case, device)
    check_attention(case, out, lse)
    assert int(attend.status.item()) == 0


@pytest.mark.parametrize("entries,context", [(1, 1), (1, 0), (2, 2), (63, 63), (64, 64), (65, 65), (128, 127), (129, 129), (1000, 999),
                                             (2048, 2048), (2048, 1), (2048, 1000), (5000, 5000)])
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
def test_attention_lengths(device, entries, context, kind):
    case = attention_case(device, entries + context, counts=[1, 2], heads=64, entries=entries, stride=2048, context=[context, max(0, context - 1)],
                          kind=kind)
    attend, out, lse = run_attention(case, device)
    check_attention(case, out, lse)
    assert int(attend.status.item()) == 0


@pytest.mark.parametrize("splits", [0, 1, 2, 4, 8])
@pytest.mark.parametrize("tokens", [1, 3])
def test_attention_shares_are_joined(device, splits, tokens):
    case = attention_case(device, 11, counts=[tokens], heads=128, entries=2048, stride=4096, context=[1800], holes=0.3)
    _, out, lse = run_attention(case, device, splits=splits)
    check_attention(case, out, lse)


def test_attention_empty_rows_holes_and_whole_empty_tiles(device):
    """Tokens that see nothing, lists that begin with long runs of -1, lists whose entries stand alone in their tiles."""
    case = attention_case(device, 5, counts=[1] * 8, heads=32, entries=1024, stride=1024, context=[1024] * 8, draft=False)
    slots = case["slots"]
    slots[0] = -1
    slots[1, :900] = -1
    slots[2, 1:] = -1
    slots[3, ::2] = -1
    keep = torch.zeros(1024, dtype=torch.bool, device=device)
    keep[[100, 500, 1023]] = True
    slots[4, ~keep] = -1
    slots[5, :] = slots[5, 0]                         # one row, over and over
    for splits in (0, 1, 4):
        attend, out, lse = run_attention(case, device, splits=splits)
        check_attention(case, out, lse)
        assert (out[0] == 0).all() and torch.isinf(lse[0]).all() and int(attend.status.item()) == 0


def test_attention_rows_that_nobody_selects_may_hold_anything(device):
    case = attention_case(device, 6, counts=[3, 2], heads=16, entries=200, stride=256, context=[120, 64])
    pool, slots = case["pool"], case["slots"]
    used = torch.zeros(pool.shape[0], dtype=torch.bool, device=device)
    for t in range(5):
        owner = int(case["row_owners"][int(case["requests"][t])])
        used[owner * 256 + slots[t][slots[t] >= 0].long()] = True
    pool[~used] = float("nan")
    pool[torch.nonzero(~used)[0]] = float("inf")
    case["ancestors"][1] = 0b010                      # sees itself, not the first node
    case["ancestors"][2] = 0b101
    _, out, lse = run_attention(case, device)
    check_attention(case, out, lse)
    case["draft"][1] = float("inf")                   # node 1 of the first request: tokens 0 and 2 do not see it
    _, out, lse = run_attention(case, device)
    check_attention(case, out, lse, tokens=[0, 2, 3, 4])


@pytest.mark.parametrize("order", ["ascending", "descending", "one"])
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
def test_attention_scores_far_apart(device, order, kind):
    """Logits that grow along the list by hundreds, so that the running maximum moves in every tile, and one that
    outweighs everything before it."""
    case = attention_case(device, 8, counts=[2], heads=64, entries=640, stride=640, context=[640], kind=kind, draft=False)
    pool, slots = case["pool"], case["slots"]
    slots[:] = torch.arange(640, dtype=torch.int32, device=device)
    direction = case["query"][0, 0].float() / case["query"][0, 0].float().norm()
    size = torch.linspace(-40, 40, 640, device=device)
    if order == "descending":
        size = -size
    elif order == "one":
        size = torch.zeros(640, device=device)
        size[500] = 60
    pool[:640] = (pool[:640].float() * 0.3 + size[:, None] * direction).to(kind)
    for splits in (1, 4):
        _, out, lse = run_attention(case, device, splits=splits)
        check_attention(case, out, lse)


def test_attention_trees_and_chains(device):
    case = attention_case(device, 21, counts=[64, 1, 13, 5], heads=16, entries=96, stride=128, context=[96, 0, 3, 50])
    attend, out, lse = run_attention(case, device)
    check_attention(case, out, lse)
    chain = dict(case, ancestors=None)
    attend, out, lse = run_attention(chain, device)
    check_attention(chain, out, lse)
    assert int(attend.status.item()) == 0


def test_attention_padding_rows_and_strided_queries(device):
    import kvip_b200 as kvip
    case = attention_case(device, 31, counts=[2, 2], heads=24, entries=70, stride=128, context=[70, 9])
    wide = torch.full((4, 24, 640), float("nan"), dtype=torch.bfloat16, device=device)
    wide[..., 64:] = case["query"]
    case["query"] = wide[..., 64:]
    rows = torch.zeros((4, 1152), dtype=torch.bfloat16, device=device)
    rows[:, 576:] = case["draft"]
    case["draft"] = rows[:, 576:]
    case["slots"] = case["slots"].view(4, 1, 70)      # the shape of slot_output
    case["pool"] = case["pool"].view(torch.uint8)     # the pool as the binding holds it
    attend = kvip.SlotAttention(torch, device, tokens=9, heads=24, entries=70)
    case["requests"][2] = -1
    out = torch.full((4, 24, 512), 3.0, dtype=torch.bfloat16, device=device)
    lse = torch.full((4, 24), 5.0, device=device)
    got = attend(**case, out=out, lse=lse)
    assert got[0] is out and (out[2] == 3.0).all() and (lse[2] == 5.0).all() and int(attend.status.item()) == 0
    check_attention(dict(case, pool=case["pool"].view(torch.bfloat16)), out, lse, tokens=[0, 1, 3])


def test_attention_reports_and_skips_what_is_out_of_range(device):
    case = attention_case(device, 32, counts=[1, 1, 1], heads=16, entries=64, stride=128, context=[64, 64, 64])
    case["slots"][0, 3] = 128                          # behind the owner's slots
    case["slots"][0, 60] = 2 ** 31 - 1
    attend, out, lse = run_attention(case, device)
    check_attention(case, out, lse)
    assert int(attend.status.item()) == 64
    case["row_owners"][1] = 3                          # the pool holds owners 0..2
    attend, out, lse = run_attention(dict(case, draft=None, starts=None, ancestors=None), device)
    assert int(attend.status.item()) == 64 and (out[1] == 0).all() and torch.isinf(lse[1]).all()
    case["requests"][2] = 3
    attend, out, lse = run_attention(dict(case, draft=None, starts=None, ancestors=None), device)
    assert int(attend.status.item()) & 1 and (out[2] == 0).all()


def test_attention_more_drafted_rows_than_a_mask_holds(device):
    case = attention_case(device, 37, counts=[70, 2], heads=16, entries=64, stride=64, context=[10, 64], draft=False)
    g = torch.Generator(device=device)
    g.manual_seed(1)
    case.update(starts=torch.tensor([0, 70, 72], dtype=torch.int32, device=device),
                draft=torch.randn((72, 576), generator=g, device=device).to(torch.bfloat16), ancestors=None)
    attend, out, lse = run_attention(case, device)
    assert int(attend.status.item()) == 1
    check_attention(case, out, lse)


def test_attention_bounded_waits_give_up_and_report(device):
    """A wait limit far below a tile's loading time: the call ends by itself, says so (unless everything came at once), and the next
    call is right again. In one piece and in shares."""
    import kvip_b200 as kvip
    case = attention_case(device, 38, counts=[2], heads=64, entries=2048, stride=4096, context=[2048])
    for splits in (1, 4):
        attend = kvip.SlotAttention(torch, device, tokens=2, heads=64)
        attend(**case, splits=splits, wait_kilocycles=1)
        torch.cuda.synchronize()
        assert int(attend.status.item()) in (0, 32)
        attend.status.zero_()
        out, lse = attend(**case, splits=splits)
        check_attention(case, out, lse)
        assert int(attend.status.item()) == 0


@pytest.mark.parametrize("heads", [16, 64])
def test_attention_bounded_waits_over_tiles_without_rows(device, heads):
    """Whole tiles of slots that name no row, the last one too, under wait limits from nothing to enough: warps whose wait ran out and warps
    that found the tile empty end the call together."""
    import kvip_b200 as kvip
    case = attention_case(device, 40, counts=[2, 1], heads=heads, entries=1024, stride=1024, context=[1024, 1024], draft=False)
    for tile in (0, 3, 4, 9, 15):
        case["slots"][:, 64 * tile:64 * tile + 64] = 1024 + 7            # behind the request's slots
    attend = kvip.SlotAttention(torch, device, tokens=3, heads=heads)
    for splits in (1, 4):
        for limit in (1, 2, 3, 5, 8, 13, 21):
            attend(**case, splits=splits, wait_kilocycles=limit)
            torch.cuda.synchronize()
            attend.status.zero_()
        out, lse = attend(**case, splits=splits)
        check_attention(case, out, lse)
        assert int(attend.status.item()) == 64        # KVIP_ERR_SOURCE: a slot outside the request


@pytest.mark.parametrize("splits", [1, 2, 8])
@pytest.mark.parametrize("heads", [16, 64])
def test_attention_a_query_of_nan_stays_one(device, heads, splits):
    """NaN in one head's query makes that head's row and lse NaN, however its rows are shared out; the other heads do not notice."""
    import kvip_b200 as kvip
    case = attention_case(device, 41, counts=[2, 1], heads=heads, entries=640, stride=1024, context=[640, 500])
    clean = dict(case, query=case["query"].clone())
    case["query"][1, 5, 17] = float("nan")
    case["query"][2, 0] = float("nan")
    attend = kvip.SlotAttention(torch, device, tokens=3, heads=heads)
    out, lse = attend(**case, splits=splits)
    hit = torch.zeros((3, heads), dtype=torch.bool, device=device)
    hit[1, 5] = hit[2, 0] = True
    assert torch.equal(out.isnan().all(-1), hit) and torch.equal(out.isnan().any(-1), hit) and torch.equal(lse.isnan(), hit)
    out, lse = out.clone(), lse.clone()
    fine_out, fine_lse = attend(**clean, splits=splits)
    check_attention(clean, fine_out, fine_lse)
    out[hit], lse[hit] = fine_out[hit], fine_lse[hit]
    check_attention(clean, out, lse)


@pytest.mark.parametrize("requests,heads,entries", [(78, 128, 700), (151, 64, 512), (170, 16, 1100)])
def test_attention_of_a_wave_and_a_few_tokens(device, requests, heads, entries):
    """A little more than one CTA per SM: the tokens behind the first wave may be cut on their own. All of them are compared, drafted
    rows and padding among them, and what is padding stays as it was."""
    import kvip_b200 as kvip
    rng = np.random.default_rng(requests)
    case = attention_case(device, 44, counts=[1] * (requests - 2) + [3, 1], heads=heads, entries=entries, stride=1200,
                          context=rng.integers(1, entries + 1, requests))
    tokens = requests + 2
    padding = torch.tensor([3, tokens - 1], device=device)
    case["requests"][padding] = -1
    attend = kvip.SlotAttention(torch, device, tokens=tokens, heads=heads, entries=entries)
    attend.out.fill_(7.0)
    attend.lse.fill_(7.0)
    out, lse = attend(**case)
    assert bool((out[padding] == 7).all()) and bool((lse[padding] == 7).all())
    check_attention(case, out, lse, [t for t in range(tokens) if t not in padding.tolist()])
    assert int(attend.status.item()) == 0


def test_attention_of_more_tokens_than_one_grid_dimension(device):
    """40001 tokens of two heads over six slots each: the tokens fill two planes of the grid, the second in part."""
    import kvip_b200 as kvip
    tokens = 40001
    g = torch.Generator(device=device)
    g.manual_seed(43)
    query = torch.randn((tokens, 2, 576), generator=g, device=device).to(torch.bfloat16)
    pool = torch.randn((256, 576), generator=g, device=device).to(torch.bfloat16)
    slots = torch.randint(-1, 64, (tokens, 6), generator=g, device=device, dtype=torch.int32)
    requests = torch.arange(tokens, device=device, dtype=torch.int32) % 4
    case = dict(query=query, pool=pool, slots=slots, requests=requests, row_owners=torch.tensor([2, 0, 3, 1], dtype=torch.int32, device=device),
                output_stride=64, scale=0.05)
    attend = kvip.SlotAttention(torch, device, tokens=tokens, heads=2, entries=6)
    out, lse = attend(**case)
    rows = torch.cat([torch.arange(0, tokens, 997), torch.tensor([32766, 32767, 32768, 32769, 40000])]).to(device)
    few = dict(case, query=query[rows], slots=slots[rows], requests=requests[rows])
    check_attention(few, out[rows], lse[rows])
    assert int(attend.status.item()) == 0 and not bool(out.isnan().any())


def test_attention_on_two_streams_with_outputs_of_their_own(device):
    """One object, two streams, outputs given by the caller: nothing is shared."""
    import kvip_b200 as kvip
    case = attention_case(device, 39, counts=[1, 2, 1], heads=128, entries=700, stride=1024, context=[700, 3, 650])
    attend = kvip.SlotAttention(torch, device, tokens=4, heads=128, entries=700)
    streams = [torch.cuda.Stream(device) for _ in range(2)]
    outs = [(torch.empty((4, 128, 512), dtype=torch.bfloat16, device=device), torch.empty((4, 128), device=device)) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for stream, (out, lse) in zip(streams, outs):
            with torch.cuda.stream(stream):
                attend(**case, out=out, lse=lse)
    torch.cuda.synchronize()
    check_attention(case, *outs[0])
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def test_attention_offsets_beyond_32_bits(device):
    """A pool of more than 2^32 bytes, and more than 2^31 elements: the last owner's rows."""
    stride = 131072
    case = attention_case(device, 33, counts=[1, 1], heads=16, entries=128, stride=stride, context=[128, 128], owners=[30, 0], draft=False,
                          pool_rows=1)
    pool = torch.zeros((31 * stride, 576), dtype=torch.bfloat16, device=device)
    assert pool.numel() > 1 << 31
    g = torch.Generator(device=device)
    g.manual_seed(3)
    for owner in (0, 30):
        pool[owner * stride:(owner + 1) * stride] = torch.randn((stride, 576), generator=g, device=device).to(torch.bfloat16)
    case["slots"][:, 0] = stride - 1
    case["pool"] = pool
    _, out, lse = run_attention(case, device)
    check_attention(case, out, lse)


def test_attention_many_tokens(device):
    """A prefill chunk's worth of tokens: more work than one wave of the GPU."""
    case = attention_case(device, 34, counts=[1] * 300, heads=128, entries=130, stride=256, context=130, owners=[0] * 300, draft=False)
    _, out, lse = run_attention(case, device)
    check_attention(case, out, lse, tokens=range(0, 300, 23))


def test_attention_graph_and_side_stream(device):
    import kvip_b200 as kvip
    case = attention_case(device, 35, counts=[2, 3], heads=64, entries=500, stride=512, context=[500, 200])
    attend = kvip.SlotAttention(torch, device, tokens=5, heads=64, entries=500)
    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        attend(**case)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out, lse = attend(**case)
        for _ in range(2):
            case["query"].copy_(torch.randn(case["query"].shape, device=device))
            out.zero_()
            graph.replay()
            check_attention(case, out, lse)
            first = out.clone()
            graph.replay()
            assert torch.equal(first, out)           # the same bits every time


# ---- verification -------------------------------------------------------------------------------------------------------
def verify_case(device, seed, *, counts, vocabulary, kind=torch.float32, draft=True, tree=True, near=0.7, sharp=2.5, pad=0):
    rng = np.random.default_rng(seed)
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    starts = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    rows = int(starts[-1])
    parents = np.concatenate([[-1] + [j - 1 if not tree else int(rng.integers(max(0, j - 4), j)) for j in range(1, n)] for n in counts if n]
                             or [[]]).astype(np.int32)
    logits = torch.randn((rows, vocabulary), generator=g, device=device) * sharp
    other = logits + near * torch.randn((rows, vocabulary), generator=g, device=device)
    buffers = torch.zeros((2, rows, vocabulary + pad), dtype=kind, device=device)
    target, guess = buffers[0, :, pad:], buffers[1, :, pad:]
    target.copy_(torch.softmax(logits, 1))
    guess.copy_(torch.softmax(other, 1))
    above = np.concatenate([starts[b] + np.maximum(parents[starts[b]:starts[b + 1]], 0) for b in range(len(counts))]).astype(np.int64)
    tokens = torch.multinomial(guess[torch.from_numpy(above).to(device)].float(), 1, generator=g)[:, 0]
    if not draft:
        tokens = logits[torch.from_numpy(above).to(device)].topk(2, dim=1).indices[torch.arange(rows, device=device), torch.arange(rows, device=device) % 2]
    return dict(target=target, draft=guess if draft else None, tokens=tokens, parents=torch.from_numpy(parents).to(device),
                starts=torch.from_numpy(starts).to(device), accept=torch.rand(rows, generator=g, device=device),
                sample=torch.rand(len(counts), generator=g, device=device))


def check_verify(case, device, depth):
    import kvip_b200 as kvip
    verifier = kvip.DraftVerifier(torch, device, batch=case["starts"].numel() - 1, depth=depth)
    tokens, nodes, counts = verifier(**case)
    torch.cuda.synchronize()
    expected = reference.verify(*(None if case[k] is None else host(case[k]) for k in ("target", "draft")),
                                *(case[k].cpu().numpy() for k in ("tokens", "parents", "starts", "accept", "sample")), depth)
    assert np.array_equal(counts.cpu().numpy(), expected[2])
    assert np.array_equal(nodes.cpu().numpy(), expected[1])
    assert np.array_equal(tokens.cpu().numpy(), expected[0])
    assert int(verifier.status.item()) == expected[3]
    return expected


@pytest.mark.parametrize("counts,vocabulary,kind,draft,tree,depth,pad", [
    ([4], 131072, torch.float32, True, False, 3, 0), ([4] * 16, 32768, torch.float32, True, False, 3, 0), ([1], 1, torch.float32, True, False, 1, 0),
    ([2, 1, 0, 5], 7, torch.float32, True, True, 4, 0), ([16, 3, 9, 0, 12], 10007, torch.bfloat16, True, True, 15, 0),
    ([64, 40, 7], 513, torch.float16, True, True, 63, 0), ([4] * 9, 50001, torch.bfloat16, False, False, 3, 0),
    ([12] * 6, 3001, torch.float32, False, True, 11, 0), ([6] * 5, 4096, torch.float32, True, True, 2, 0),
    ([5] * 4, 1000, torch.float32, True, True, 4, 3), ([5] * 4, 1024, torch.bfloat16, True, True, 4, 8), ([3] * 130, 257, torch.float32, True, False, 2, 0),
    ([4] * 3, 200000, torch.bfloat16, True, False, 3, 0)])
def test_verify_matches_the_walk(device, counts, vocabulary, kind, draft, tree, depth, pad):
    for seed in range(3):
        check_verify(verify_case(device, seed, counts=counts, vocabulary=vocabulary, kind=kind, draft=draft and vocabulary > 1 or draft, tree=tree,
                                 near=(0.1, 0.7, 3.0)[seed], pad=pad), device, depth)


@pytest.mark.parametrize("lift,most,deepest", [(2.5, 1.0, 2), (6.0, 0.4, 4)])
def test_verify_without_draft_rows_repeated_tokens(device, lift, most, deepest):
    """Deep trees over three tokens with certain drafts: every request accepts and rejects in turn, siblings and levels repeat tokens, so the
    rejected tokens of a node decide the next test. Passes over 24 tokens are short, so warps run close behind one another."""
    rng = np.random.default_rng(77)
    g = torch.Generator(device=device)
    g.manual_seed(77)
    counts = [64] * 48
    case = verify_case(device, 77, counts=counts, vocabulary=24, draft=False)
    logits = torch.randn((64 * 48, 24), generator=g, device=device)
    logits[:, :3] += lift
    case["target"].copy_(torch.softmax(logits, 1))
    case["tokens"] = torch.from_numpy(rng.integers(0, 3, 64 * 48)).to(device)
    accepted = 0
    for _ in range(20):
        case["accept"] = torch.rand(64 * 48, generator=g, device=device) * most
        accepted = max(accepted, int(check_verify(case, device, 63)[2].max()) - 1)
    assert accepted >= deepest             # walks that go on behind rejections


def test_verify_borders(device):
    """Numbers at the ends of [0, 1), distributions with one token, a draft equal to its target, rows of nothing."""
    counts, vocabulary = [3] * 8, 300
    case = verify_case(device, 1, counts=counts, vocabulary=vocabulary, tree=False)
    target, guess = case["target"], case["draft"]
    case["accept"][:] = torch.tensor([0.0, 0.0, 1 - 2.0 ** -24], device=device).repeat(8)
    case["sample"][:] = torch.tensor([0.0, 1 - 2.0 ** -24] * 4, device=device)
    target[3:6] = 0
    target[3:6, 17] = 1.0                               # request 1: certain target
    guess[6:9] = target[6:9]                            # request 2: nothing is left after a rejection
    case["accept"][6:9] = 1 - 2.0 ** -24
    target[9:12] = 0                                    # request 3: no probability at all
    target[12, :100] = float("nan")                     # request 4: what is no probability counts as nothing
    target[12, 100:200] = -1.0
    guess[15] = 0                                       # request 5: a draft without probability
    target[18:21] = 1.0 / 256                           # request 6: exact sums, and a border met exactly
    target[18:21, 256:] = 0
    case["sample"][6] = 0.5
    case["accept"][19] = 0.999
    check_verify(case, device, 2)
    case["draft"] = None
    check_verify(case, device, 2)


def test_verify_skips_bad_nodes(device):
    case = verify_case(device, 2, counts=[4, 4, 4], vocabulary=100, tree=False, near=0.1)
    case["accept"][:] = 0
    case["tokens"][1] = 100
    case["tokens"][6] = -1
    case["parents"][9] = 5
    expected = check_verify(case, device, 3)
    assert expected[3] == 1 and expected[2].tolist()[0] == 1 and expected[2].tolist()[1] == 2
    case["starts"][1:3] = torch.tensor([20, 3], dtype=torch.int32, device=device)
    check_verify(case, device, 3)


def test_verify_too_many_nodes(device):
    case = verify_case(device, 3, counts=[70, 2], vocabulary=64, tree=True, near=0.05)
    assert check_verify(case, device, 63)[3] == 1


def test_verify_draws_the_targets_distribution(device):
    """The first emitted token of many requests with one target is distributed as the target, whatever the draft."""
    batch, vocabulary = 4096, 8
    g = torch.Generator(device=device)
    g.manual_seed(0)
    p = torch.tensor([0.3, 0.25, 0.2, 0.1, 0.08, 0.04, 0.02, 0.01], device=device)
    q = torch.tensor([0.05, 0.05, 0.1, 0.3, 0.1, 0.2, 0.1, 0.1], device=device)
    rows = batch * 3                                    # a root with two drafted children
    import kvip_b200 as kvip
    tokens = torch.multinomial(q, rows, replacement=True, generator=g)
    verifier = kvip.DraftVerifier(torch, device, batch=batch, depth=2)
    out, _, _ = verifier(p.expand(rows, vocabulary).contiguous(), q.expand(rows, vocabulary).contiguous(), tokens,
                         torch.tensor([-1, 0, 0], dtype=torch.int32, device=device).repeat(batch),
                         torch.arange(0, rows + 1, 3, dtype=torch.int32, device=device), torch.rand(rows, generator=g, device=device),
                         torch.rand(batch, generator=g, device=device))
    seen = torch.bincount(out[:, 0], minlength=vocabulary).double().cpu() / batch
    # a binomial share of 4096 draws: six standard deviations
    assert ((seen - p.double().cpu()).abs() <= 6 * (p * (1 - p) / batch).sqrt().double().cpu()).all()
