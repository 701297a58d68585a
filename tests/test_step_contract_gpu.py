"""What the operators round the selection path owe one another and their callers on the GPU: one rule of quantisation, indices of the
layout that are checked wherever they are used, block tables that carry the errors of a plan through, selection and drafted rows that show
every key once, and attention at the ends of its types."""
import numpy as np
import pytest
import torch

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
