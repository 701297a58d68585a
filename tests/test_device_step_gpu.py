"""Decode steps with drafted tokens, from lengths on the GPU to the lengths of the next step, against the definition over the tokens
themselves: which keys a token sees is told by the tokens that were committed and by the tree it stands in, with rows kept on the host, not
by the lists and pools of the step. So a key that is seen twice, one of a rejected token, or one whose row has moved shows."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import step_reference as reference
from test_step_operators_gpu import HALF_STEP, host

pytestmark = pytest.mark.gpu

QUERIES, HEADS, HISTORY, RESIDENT, VOCABULARY, SCALE, BLOCKS = 4, 16, 16384, 8192, 61, 0.05, 128
LENGTHS = [9000, 700, 2046, 1, 0]           # longer than the resident rows, shorter than a list, about to pass its end, one cached token, none
OWNERS = [3, 1, 5, 2, 4]                    # owner 0 takes the padding rows
BATCH = len(LENGTHS)


class Loop:
    def __init__(self, device, seed, own_owners=False):
        import kvip_b200 as kvip
        from decode_harness import DecodePipeline
        self.kvip, self.device, self.rng = kvip, device, np.random.default_rng(seed)
        self.g = torch.Generator(device=device)
        self.g.manual_seed(seed)
        tokens = self.tokens = BATCH * QUERIES
        self.p = p = DecodePipeline(device, batch=BATCH, queries=QUERIES, heads=64, history=HISTORY, resident=RESIDENT, len_lo=8, len_hi=9, seed=seed,
                                    owners=BATCH + 1, host_pool=False, gather=False)
        p.lru.resize(RESIDENT, [min(n, RESIDENT) for n in LENGTHS])      # victims among cached tokens alone
        self.source = p.source.view(torch.bfloat16).view(BATCH + 1, HISTORY, 576)
        self.source.copy_(torch.randn(self.source.shape, generator=self.g, device=device))
        self.rows = [host(self.source[o, :n]) for o, n in zip(OWNERS, LENGTHS)]                    # of the committed tokens
        self.keys = [p.storage.keys[o, :n].cpu().numpy() for o, n in zip(OWNERS, LENGTHS)]
        self.scales = [p.storage.scales[o, :n].cpu().numpy() for o, n in zip(OWNERS, LENGTHS)]
        pages = HISTORY // 128
        self.tables = kvip.BlockTables(torch, device, batch=BATCH, pages=pages, blocks=BLOCKS, tokens=tokens, queries=QUERIES)
        held = [-(-n // 128) for n in LENGTHS]
        order = self.rng.permutation(BLOCKS).astype(np.int32)
        table, used = np.full((BATCH, pages), -1, np.int32), np.cumsum([0] + held)
        for b in range(BATCH):
            table[b, :held[b]] = order[used[b]:used[b + 1]]
        self.tables.load(lengths=torch.tensor(LENGTHS), held=torch.tensor(held), table=torch.from_numpy(table), free=torch.from_numpy(order[used[-1]:]))
        self.owners = torch.tensor(OWNERS, dtype=torch.int32, device=device)
        self.cache = torch.zeros((BLOCKS * 128 + 1, 128), dtype=torch.bfloat16, device=device)  # the model's paged Index keys; the last row: no slot
        self.rope = kvip.Rotary(torch, 64, device, layout="half")
        self.rope_query = kvip.Rotary(torch, 64, device, layout="interleaved")
        self.attend = kvip.SlotAttention(torch, device, tokens=tokens, heads=HEADS)
        self.verify = kvip.DraftVerifier(torch, device, batch=BATCH, depth=QUERIES - 1)
        row_owners = torch.zeros(BATCH, dtype=torch.int32, device=device) if own_owners else p.workspace.inputs.row_owners
        self.select = kvip.IndexSelector(torch, inputs=p.workspace.inputs, rotating=p.rotating, update=p.update, logical_ids=p.storage.logical_ids,
                                         row_owners=row_owners, storage=p.storage, forward=p.forward, rotary=self.rope)
        self.model, self.jumps = {}, 0
        self.new_inputs([4, 3, 4, 2, 4], tree=False)

    def new_inputs(self, counts, tree):
        """What the model computes for the step's tokens, in place, so that a captured graph reads it."""
        device, g, tokens, self.tree = self.device, self.g, self.tokens, tree
        parents, depths, masks, drafted = (np.zeros(tokens, np.int64) for _ in range(4))
        t = 0
        for n in counts:
            for j in range(n):
                up = -1 if j == 0 else j - 1 if not tree else int(self.rng.integers(0, j))
                parents[t + j], depths[t + j] = up, 0 if j == 0 else depths[t + up] + 1
                masks[t + j] = (1 << j) | (masks[t + up] if j else 0)
            t += n
        target = torch.softmax(torch.randn((tokens, VOCABULARY), generator=g, device=device) * 3, 1)
        drafted[:] = self.rng.integers(0, VOCABULARY, tokens)
        new = dict(
            counts=torch.tensor(counts, dtype=torch.int32, device=device),
            index_query=torch.randn((tokens, 64, 128), generator=g, device=device).to(torch.bfloat16),
            index_key=torch.randn((tokens, 128), generator=g, device=device).to(torch.bfloat16),
            weights=(torch.randn((tokens, 64), generator=g, device=device) / 8).to(torch.bfloat16),
            query=torch.randn((tokens, HEADS, 576), generator=g, device=device).to(torch.bfloat16),
            row=torch.randn((tokens, 576), generator=g, device=device).to(torch.bfloat16),
            target=target, draft=torch.softmax(target.log() + torch.randn((tokens, VOCABULARY), generator=g, device=device), 1),
            drafted=torch.from_numpy(drafted).to(device), parents=torch.from_numpy(parents.astype(np.int32)).to(device),
            depths=torch.from_numpy(depths.astype(np.int32)).to(device), masks=torch.from_numpy(masks).to(device),
            accept=torch.rand(tokens, generator=g, device=device) ** 6, sample=torch.rand(BATCH, generator=g, device=device))
        for name, value in new.items():
            if name in self.model:
                self.model[name].copy_(value)
            else:
                self.model[name] = value
        self.pristine = {k: v.clone() for k, v in self.model.items()}

    def __call__(self):
        m, t, p = self.model, self.tables, self.p
        t.plan(m["counts"])
        positions = self.prepare()
        self.rope(positions, m["index_key"][:, :64])
        self.rope_query(positions, m["query"][..., 512:], m["row"][:, 512:])
        self.cache.index_copy_(0, torch.where(t.slot_mapping >= 0, t.slot_mapping, self.cache.shape[0] - 1), m["index_key"])
        self.logical = self.select(m["index_query"], m["weights"], SimpleNamespace(k_cache=SimpleNamespace(kv_cache=(self.cache, None))),
                                   SimpleNamespace(slot_mapping=t.slot_mapping))
        self.out, self.lse = self.select.attend(self.attend, m["query"], scale=SCALE, tables=t, draft=m["row"], ancestors=m["masks"])
        self.verify(m["target"], m["draft"], m["drafted"], m["parents"], t.starts, m["accept"], m["sample"])
        self.keep()
        self.before = [x.clone() for x in (t.lengths, t.starts)]
        t.commit(self.verify.counts)

    def prepare(self):
        self.select.prepare_device(self.tables, self.owners, self.model["depths"] if self.tree else None)
        return self.select.positions

    def keep(self):
        """The rows and Index keys of the accepted nodes, root first, go behind the cached tokens of their request; what else was written there
        belongs to no token."""
        t, m, storage = self.tables, self.model, self.p.storage
        j = torch.arange(QUERIES, device=self.device)
        node = torch.where(j < self.verify.counts[:, None], self.verify.nodes, j).clamp(min=0).long()
        at, owner = t.lengths[:, None].long() + j, self.owners[:, None].long()
        self.source[owner, at] = m["row"][(t.starts[:-1, None] + node).clamp(max=self.tokens - 1)]
        storage.keys[owner, at] = storage.keys[owner, at - j + node]
        storage.scales[owner, at] = storage.scales[owner, at - j + node]

    def check(self):
        torch.cuda.synchronize()
        m, p, was = self.model, self.p, self.pristine
        lengths, starts = (x.cpu().numpy() for x in self.before)
        assert lengths.tolist() == [len(r) for r in self.rows]
        positions = np.repeat(lengths, np.diff(starts)) + was["depths"].cpu().numpy()[:starts[-1]]
        for name, part in (("query", m["query"]), ("row", m["row"][:, None])):
            x = host(was[name]).reshape(self.tokens, -1, 576)[:starts[-1], :, 512:]
            turned, size = reference.rotary(x, positions, 64, "interleaved")
            got = host(part)[:starts[-1], :, 512:]
            assert (np.abs(got - turned) <= size * 2.0 ** -20 + np.abs(turned) * HALF_STEP[torch.bfloat16]).all(), name
        key, _ = reference.rotary(host(was["index_key"])[:, None][:starts[-1]], positions, 64, "half")
        assert (np.abs(host(m["index_key"])[:starts[-1]] - key[:, 0]) <= np.abs(key[:, 0]) * 2.0 ** -8 + 2.0 ** -18).all()
        rows, logical = host(m["row"]), self.logical[:, 0].cpu().numpy()
        kept = []
        for b in range(BATCH):
            mask = was["masks"].cpu().numpy()
            for t in range(starts[b], starts[b + 1]):
                listed = logical[t][logical[t] >= 0]
                assert len(set(listed.tolist())) == len(listed) == min(2048, lengths[b]) and (listed < lengths[b]).all()
                seen = np.concatenate([self.rows[b][listed], rows[[starts[b] + j for j in range(starts[b + 1] - starts[b]) if mask[t] >> j & 1]]])
                expected, log_sum, weight, size = reference.attention(host(m["query"][t]), seen, SCALE)
                logit = 577 * 2.0 ** -24 * size      # as in the test of the operator alone
                step = HALF_STEP[torch.bfloat16]
                assert (np.abs(host(self.out[t]) - expected) <= weight * (2 * step + 2 * logit + 2.0 ** -18) + np.abs(expected) * step + 1e-7).all(), (b, t)
                assert (np.abs(host(self.lse[t]) - log_sum) <= logit + 2.0 ** -20 * (1 + np.abs(log_sum))).all()
            a, z = starts[b], starts[b + 1]
            local = np.array([0, z - a])
            _, nodes, counts, _ = reference.verify(*(host(was[k])[a:z] for k in ("target", "draft")),
                                                   *(was[k].cpu().numpy()[a:z] for k in ("drafted", "parents")), local,
                                                   was["accept"].cpu().numpy()[a:z], was["sample"].cpu().numpy()[b:b + 1], QUERIES - 1)
            assert int(self.verify.counts[b]) == counts[0] and np.array_equal(self.verify.nodes[b].cpu().numpy(), nodes[0])
            path = a + nodes[0, :counts[0]]
            kept.append(int(counts[0]))
            self.jumps += int((nodes[0, :counts[0]] != np.arange(counts[0])).any())
            self.rows[b] = np.concatenate([self.rows[b], rows[path]])
            x = host(m["index_key"])[path].astype(np.float32)
            scale = (np.abs(x).max(1) / np.float32(448)).astype(np.float32)
            code = torch.from_numpy(np.clip(x / scale[:, None], -448, 448).astype(np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
            self.keys[b], self.scales[b] = np.concatenate([self.keys[b], code]), np.concatenate([self.scales[b], scale])
        assert self.tables.lengths.tolist() == [len(r) for r in self.rows]
        for b, owner in enumerate(OWNERS):          # Index rows may have changed places, among the cached tokens alone
            n = len(self.rows[b])
            ids = p.storage.logical_ids[owner].cpu().numpy()
            assert np.array_equal(np.sort(ids[:n]), np.arange(n)) and np.array_equal(ids[n:], np.arange(n, HISTORY))
            assert np.array_equal(p.storage.keys[owner, :n].cpu().numpy(), self.keys[b][ids[:n]])
            assert np.array_equal(p.storage.scales[owner, :n].cpu().numpy(), self.scales[b][ids[:n]])
        for status in (self.attend.status, self.verify.status, self.tables.status, p.forward.li_status, p.update.status, p.storage.ingest_errors):
            assert int(status.abs().max()) == 0
        return kept


def run(loop, device, *, tree, captured, steps=5):
    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    more = less = 0
    with torch.cuda.stream(stream):
        graph = None
        for turn in range(steps):
            counts = [[4, 3, 4, 2, 4], [1, 4, 4, 4, 2], [4, 4, 2, 0, 3], [3, 1, 4, 4, 4], [4, 4, 4, 3, 1]][turn]
            loop.new_inputs(counts, tree)
            if captured and turn == 1:
                graph = torch.cuda.CUDAGraph()
                stream.synchronize()
                with torch.cuda.graph(graph, stream=stream):
                    loop()
            if graph is None:
                loop()
            else:
                graph.replay()
            kept = loop.check()
            more += sum(k > 1 for k in kept)
            less += sum(k < n for k, n in zip(kept, counts))
    assert more > 2 and less > 2                 # drafted tokens were accepted, and rejected
    del graph


@pytest.mark.parametrize("captured,own_owners", [(False, False), (True, False), (False, True)])
def test_every_key_of_a_chain_is_seen_once(device, captured, own_owners):
    run(Loop(device, 3, own_owners), device, tree=False, captured=captured)


@pytest.mark.parametrize("captured", [False, True])
def test_nodes_of_a_tree_turn_by_their_depth_and_see_their_ancestors(device, captured):
    """Trees of up to four nodes: siblings have one position and two places, a node selects none of the step's tokens, and the accepted path is
    the continuation of the request whichever nodes it runs through."""
    loop = Loop(device, 4)
    run(loop, device, tree=True, captured=captured)
    assert loop.jumps > 0                        # accepted paths that leave nodes out
