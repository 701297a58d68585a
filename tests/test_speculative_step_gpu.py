"""A speculative decode step as a whole: slot maps from lengths on the GPU, rotated and quantised Index queries and keys, the
selection path, attention of the drafted tokens over the selected slots, their verification, and the next step from what
was accepted - without a copy to the host in between, eager and from one CUDA graph."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import step_reference as reference
from test_step_operators_gpu import check_attention, host

pytestmark = pytest.mark.gpu

BATCH, QUERIES, HEADS, HISTORY, RESIDENT, VOCABULARY = 3, 4, 16, 8192, 4096, 997


class Step:
    def __init__(self, device, seed=0):
        import kvip_b200 as kvip
        from decode_harness import DecodePipeline
        tokens = BATCH * QUERIES
        self.p = p = DecodePipeline(device, batch=BATCH, queries=QUERIES, heads=64, history=HISTORY, resident=RESIDENT, len_lo=2500, len_hi=3000,
                                    seed=seed, host_pool=False, gather=False)
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        p.source.view(torch.bfloat16).copy_(torch.randn((p.owners * HISTORY, 576), generator=g, device=device))
        pages = HISTORY // 128
        self.tables = kvip.BlockTables(torch, device, batch=BATCH, pages=pages, blocks=BATCH * pages, tokens=tokens, queries=QUERIES)
        held = -(-p.lengths // 128)
        order = np.random.default_rng(seed).permutation(BATCH * pages).astype(np.int32)
        table = np.full((BATCH, pages), -1, np.int32)
        used = 0
        for b in range(BATCH):
            table[b, :held[b]] = order[used:used + held[b]]
            used += int(held[b])
        self.tables.load(lengths=torch.from_numpy(p.lengths), held=torch.from_numpy(held.astype(np.int32)), table=torch.from_numpy(table),
                         free=torch.from_numpy(order[used:]))
        self.owners = torch.tensor(p.row_owner_list, dtype=torch.int32, device=device)
        self.counts = torch.tensor([4, 1, 3], dtype=torch.int32, device=device)
        self.rope = kvip.Rotary(torch, 64, device, layout="half", scaling={"kind": "yarn", "factor": 4.0, "original": 2048})
        self.rope_query = kvip.Rotary(torch, 64, device, layout="interleaved")
        self.cache = torch.zeros((BATCH * HISTORY, 128), dtype=torch.bfloat16, device=device)      # the model's paged Index keys
        self.attend = kvip.SlotAttention(torch, device, tokens=tokens, heads=HEADS)
        self.verify = kvip.DraftVerifier(torch, device, batch=BATCH, depth=QUERIES - 1)
        self.selector = kvip.IndexSelector(torch, inputs=p.workspace.inputs, rotating=p.rotating, update=p.update,
                                           logical_ids=p.storage.logical_ids, row_owners=p.workspace.inputs.row_owners, forward=p.forward,
                                           rotary=self.rope)
        self.model = {}
        self.new_inputs(g)

    def new_inputs(self, g):
        """What the model would compute for the step's tokens; written in place, so that a captured graph reads it."""
        tokens, device = BATCH * QUERIES, self.p.device
        starts = np.concatenate(([0], np.cumsum(self.counts.cpu().numpy())))
        packed = np.concatenate([np.arange(-1, n - 1) for n in np.diff(starts)] + [np.full(tokens - starts[-1], -1)]).astype(np.int32)
        target = torch.softmax(torch.randn((tokens, VOCABULARY), generator=g, device=device) * 2, 1)
        new = dict(
            index_query=torch.randn((tokens, 64, 128), generator=g, device=device).to(torch.bfloat16),
            index_key=torch.randn((tokens, 128), generator=g, device=device).to(torch.bfloat16),
            weights=(torch.randn((tokens, 64), generator=g, device=device) / 8).to(torch.bfloat16),
            query=torch.randn((tokens, HEADS, 576), generator=g, device=device).to(torch.bfloat16),
            row=torch.randn((tokens, 576), generator=g, device=device).to(torch.bfloat16),
            target=target, draft=torch.softmax(target.log() + torch.randn((tokens, VOCABULARY), generator=g, device=device), 1),
            tokens=torch.randint(0, VOCABULARY, (tokens,), generator=g, device=device),
            parents=torch.from_numpy(packed).to(device), accept=torch.rand(tokens, generator=g, device=device) ** 4,
            sample=torch.rand(BATCH, generator=g, device=device))
        for name, value in new.items():
            if name in self.model:
                self.model[name].copy_(value)
            else:
                self.model[name] = value
        self.pristine = {k: v.clone() for k, v in self.model.items()}

    def __call__(self):
        p, m, tables, inputs = self.p, self.model, self.tables, self.p.workspace.inputs
        tables.plan(self.counts)
        inputs.prepare_device(tables.layout, self.owners)
        positions = tables.positions
        inputs.bind_positions(positions)
        p.workspace.key_lengths.copy_(tables.ends)
        self.rope(positions, m["index_key"][:, :64])
        self.rope_query(positions, m["query"][..., 512:], m["row"][:, 512:])
        self.cache.index_copy_(0, tables.slot_mapping.clamp(min=0), m["index_key"])
        p.storage.ingest_decode((self.cache, None), SimpleNamespace(slot_mapping=tables.slot_mapping.clamp(min=0)), inputs, inputs.row_owners)
        self.selector.positions = positions
        logical = self.selector(m["index_query"], m["weights"], SimpleNamespace(k_cache=None), None)
        self.out, self.lse = self.selector.attend(self.attend, m["query"], scale=0.08, tables=tables, draft=m["row"])
        accepted = self.verify(m["target"], m["draft"], m["tokens"], m["parents"], tables.starts, m["accept"], m["sample"])
        return logical, accepted

    def check(self, before):
        """Everything the step has left on the device, against the restatements."""
        torch.cuda.synchronize()
        t, p, m = self.tables, self.p, self.model
        expected = reference.slot_maps(before["lengths"], self.counts.cpu().numpy(), before["held"], before["table"], t.free.cpu().numpy(),
                                       before["head"], block=128, tokens=BATCH * QUERIES, queries=QUERIES)
        for name, value in expected.items():
            if name != "status":
                assert np.array_equal(getattr(t, name).cpu().numpy(), value), name
        total = int(expected["starts"][-1])
        positions = expected["positions"][:total]
        turned, size = reference.rotary(host(self.pristine["query"])[:total, :, 512:], positions, 64, "interleaved")
        assert (np.abs(host(m["query"])[:total, :, 512:] - turned) <= size * 2.0 ** -20 + np.abs(turned) * 2.0 ** -8).all()
        ends = p.workspace.inputs.query_ends.cpu().numpy().reshape(BATCH, QUERIES)
        for b in range(BATCH):
            n, first = int(expected["starts"][b + 1] - expected["starts"][b]), int(expected["starts"][b])
            assert ends[b].tolist() == [int(x) + 1 for x in positions[first:first + n]] + [0] * (QUERIES - n)
        case = dict(query=m["query"], pool=p.pool_hbm.view(torch.bfloat16), slots=p.update.slot_output[:, 0], requests=t.requests,
                    row_owners=self.owners, output_stride=RESIDENT, scale=0.08, starts=t.starts, draft=m["row"], ancestors=None)
        slots = p.update.slot_output[:total].cpu().numpy()
        assert (slots >= 0).all()                      # contexts are longer than 2048: full lists
        check_attention(case, self.out, self.lse, tokens=range(total))
        checked = reference.verify(*(host(m[k])[:total] for k in ("target", "draft")),
                                   *(m[k].cpu().numpy()[:total] for k in ("tokens", "parents")), expected["starts"],
                                   *(m[k].cpu().numpy() for k in ("accept", "sample")), QUERIES - 1)
        for got, want in zip((self.verify.tokens, self.verify.nodes, self.verify.counts), checked):
            assert np.array_equal(got.cpu().numpy(), want)
        assert int(self.attend.status) == int(self.verify.status) == int(t.status) == 0
        assert int(p.forward.li_status) == 0 and int(p.update.status.abs().max()) == 0
        return checked[2]

    def state(self):
        t = self.tables
        return dict(lengths=t.lengths.cpu().numpy(), held=t.held.cpu().numpy(), table=t.table.cpu().numpy(), head=int(t.head))


@pytest.mark.parametrize("captured", [False, True])
def test_speculative_steps(device, captured):
    step = Step(device)
    g = torch.Generator(device=device)
    g.manual_seed(99)
    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        graph = None
        kept_more = 0
        for turn in range(4):
            before = step.state()
            if captured and turn == 1:
                graph = torch.cuda.CUDAGraph()
                stream.synchronize()
                with torch.cuda.graph(graph, stream=stream):
                    step()
            if graph is not None:
                graph.replay()
            else:
                step()
            kept = step.check(before)
            kept_more += int((kept > 1).sum())
            step.tables.commit(step.verify.counts)
            after = step.state()
            assert np.array_equal(after["lengths"], before["lengths"] + kept)
            step.counts.copy_(torch.tensor([[2, 4, 1], [4, 4, 4], [1, 3, 4], [4, 1, 3]][turn], dtype=torch.int32))
            step.new_inputs(g)
            stream.synchronize()
        assert kept_more > 0            # some drafted tokens were accepted on the way
    del graph


def test_query_inputs_prepare_device_equals_prepare(device):
    import kvip_b200 as kvip
    counts, owners = (2, 0, 4, 1), (3, 1, 0, 2)
    one = kvip.QueryInputs(torch, 4, device, history=512, queries=4)
    one.prepare(counts, query_owners=owners)
    two = kvip.QueryInputs(torch, 4, device, history=512, queries=4)
    tables = kvip.BlockTables(torch, device, batch=4, pages=4, blocks=16, tokens=16, queries=4)
    tables.plan(torch.tensor(counts, dtype=torch.int32, device=device))
    two.prepare_device(tables.layout, torch.tensor(owners, dtype=torch.int32, device=device))
    torch.cuda.synchronize()
    assert torch.equal(one.metadata, two.metadata) and torch.equal(one.block_table, two.block_table) and two.token_count == 16
    with pytest.raises(ValueError):
        two.prepare_device(tables.layout[:, :8], two.row_owners)
    with pytest.raises(ValueError):
        two.prepare_device(tables.layout, two.row_owners[:3])
