"""Cases of the operators round the selection path of a speculative decode step, with their plain forms.

Four operators: the slot maps of a step, rotary positions (with the FP8 form of the Index queries), attention of drafted
tokens over the selected cache slots, and the verification of drafted tokens. A case names its operator in "op"."""
import math

import torch

own = False

WIDTH, VALUE = 576, 512          # a cache row: 512 latent values, then 64 rotated ones
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
YARN = {"kind": "yarn", "factor": 32.0, "original": 4096, "beta_fast": 32.0, "beta_slow": 1.0}


def listed():
    return [
        # ---- attention: `batch` requests with up to `nodes` drafted tokens each, every token with its own list
        # one request, one token: the latency of a single user
        dict(name="attention one token", op="attention", batch=1, nodes=1, ragged=False, heads=128, entries=2048, stride=16384,
             context=16384, type="bf16"),
        # the decode step of the benchmark's batch, every list full
        dict(name="attention 64 requests", op="attention", batch=64, nodes=1, ragged=False, heads=128, entries=2048, stride=8192,
             context=8192, type="bf16"),
        # a tree of eight drafted tokens a request, heads split over eight GPUs
        dict(name="attention trees 16 heads", op="attention", batch=32, nodes=8, ragged=False, heads=16, entries=2048, stride=8192,
             context=8192, type="bf16"),
        # requests of different, short contexts: lists that end early, one to four tokens a request
        dict(name="attention short ragged", op="attention", batch=48, nodes=4, ragged=True, heads=64, entries=2048, stride=4096,
             context=1500, type="fp16"),
        # ---- rotary
        # Index queries of a decode step, rotated and quantised to FP8 for the selection
        dict(name="rotary fp8 decode", op="quantise", tokens=64, heads=64, dim=128, width=64, layout="half", scaled=False,
             longest=131072, type="bf16"),
        # the rotated part of the latent queries of a prefill chunk, inside their 576-wide rows, with the keys
        dict(name="rotary chunk 8192", op="rotary", tokens=8192, heads=128, row=576, width=64, layout="interleaved", scaled=True,
             longest=131072, type="bf16"),
        # Index queries of a long prefill chunk of odd length
        dict(name="rotary fp8 chunk 16411", op="quantise", tokens=16411, heads=64, dim=128, width=64, layout="half", scaled=True,
             longest=1048576, type="bf16"),
        # ---- verification
        # one request, three drafted tokens behind the last committed one
        dict(name="verify one request", op="verify", batch=1, nodes=4, tree=False, vocabulary=131072, draft=True, type="fp32"),
        # a decode batch with the same chains
        dict(name="verify 64 chains", op="verify", batch=64, nodes=4, tree=False, vocabulary=131072, draft=True, type="fp32"),
        # trees of sixteen nodes, an odd vocabulary
        dict(name="verify 48 trees", op="verify", batch=48, nodes=16, tree=True, vocabulary=100003, draft=True, type="bf16"),
        # ---- slot maps
        # a decode step: four tokens a request
        dict(name="slot maps decode", op="maps", batch=64, most=4, pages=1024, block=128, tokens=256),
        # a mixed batch: a thousand requests, most of them decoding, some in the middle of a prompt
        dict(name="slot maps mixed", op="maps", batch=1000, most=1024, pages=1024, block=128, tokens=131072),
    ]


def _spread(rng, low, high):
    """A size between low and high, spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "quantise", "rotary", "verify", "maps"])
    if op == "attention":
        nodes = rng.choice([1, 1, 2, 3, 4, 8, 13])
        heads = rng.choice([1, 8, 16, 32, 40, 64, 96, 128])
        entries = rng.choice([2048, 2048, 1000, 257, 64, 1])
        batch = _spread(rng, 1, max(1, 64 * 128 // (heads * nodes) if heads > 32 else 256 // nodes))
        stride = rng.choice([2048, 4096, 8192])
        return dict(op=op, batch=batch, nodes=nodes, ragged=rng.random() < 0.5, heads=heads, entries=entries, stride=stride,
                    context=_spread(rng, 1, stride), type=rng.choice(["bf16", "bf16", "fp16"]))
    if op == "quantise":
        return dict(op=op, tokens=_spread(rng, 1, 16384), heads=rng.choice([1, 32, 64]), dim=128, width=rng.choice([32, 64, 128]),
                    layout=rng.choice(["half", "interleaved"]), scaled=rng.random() < 0.5, longest=_spread(rng, 1024, 2 ** 21),
                    type=rng.choice(["bf16", "fp16", "fp32"] if rng.random() < 0.5 else ["bf16"]))
    if op == "rotary":
        width = rng.choice([32, 64, 96, 128])
        return dict(op=op, tokens=_spread(rng, 1, 8192), heads=rng.choice([1, 8, 16, 64, 128]), row=width + rng.choice([0, 64, 512]),
                    width=width, layout=rng.choice(["half", "interleaved"]), scaled=rng.random() < 0.5,
                    longest=_spread(rng, 1024, 2 ** 21), type=rng.choice(["bf16", "fp16"]))
    if op == "verify":
        tree = rng.random() < 0.5
        return dict(op=op, batch=_spread(rng, 1, 64), nodes=rng.choice([1, 2, 4, 7, 12] if tree else [1, 2, 3, 4]), tree=tree,
                    vocabulary=_spread(rng, 1000, 131072), draft=rng.random() < 0.75, type=rng.choice(["fp32", "bf16", "fp16"]))
    batch = _spread(rng, 1, 1024)
    most = rng.choice([1, 2, 4, 100, 1000])
    block = rng.choice([16, 64, 128])
    return dict(op=op, batch=batch, most=most, pages=_spread(rng, 64, 2048), block=block, tokens=batch * most)


# ---- inputs -------------------------------------------------------------------------------------------------------
def _parents(nodes, tree, cpu):
    """Local parent of every node of one request: a chain, or a tree whose nodes hang on an earlier one."""
    if not tree:
        return [j - 1 for j in range(nodes)]
    return [-1] + [int(torch.randint(max(0, (j - 1) // 3), (j + 1) // 2 + 1, (1,), generator=cpu).clamp(max=j - 1)) for j in range(1, nodes)]


def _masks(parents):
    masks = []
    for j, p in enumerate(parents):
        masks.append((1 << j) | (masks[p] if p >= 0 else 0))
    return masks


def prepare(case, seed):
    cuda = torch.device("cuda")
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    cpu = torch.Generator()
    cpu.manual_seed(seed)
    return {"attention": _prepare_attention, "quantise": _prepare_rotary, "rotary": _prepare_rotary, "verify": _prepare_verify,
            "maps": _prepare_maps}[case["op"]](case, cuda, g, cpu)


def _prepare_attention(case, cuda, g, cpu):
    batch, nodes, heads, entries, stride = case["batch"], case["nodes"], case["heads"], case["entries"], case["stride"]
    kind = TYPES[case["type"]]
    counts = [1 + (5 * b + b // nodes) % nodes if case["ragged"] else nodes for b in range(batch)]
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    tokens = starts[-1]
    masks = [m for n in counts for m in _masks(_parents(n, True, cpu))]
    requests = torch.tensor([r for r, n in enumerate(counts) for _ in range(n)], dtype=torch.int32, device=cuda)
    # latent rows have a mean of their own in every channel
    pool = torch.empty((batch * stride, WIDTH), dtype=kind, device=cuda)
    mean = torch.randn(WIDTH, generator=g, device=cuda) * 0.3
    for b in range(batch):
        pool[b * stride:(b + 1) * stride] = (torch.randn((stride, WIDTH), generator=g, device=cuda) + mean).to(kind)
    low = 1 if case["ragged"] else case["context"]
    context = torch.randint(low, case["context"] + 1, (batch,), generator=cpu).to(cuda)
    # every token's list: distinct slots of its request in any order, -1 behind the last one of a short context
    order = torch.rand((tokens, stride), generator=g, device=cuda)
    order.masked_fill_(torch.arange(stride, device=cuda)[None, :] >= context[requests.long()][:, None], 2.0)
    order, chosen = order.sort(dim=1)
    slots = torch.full((tokens, entries), -1, dtype=torch.int32, device=cuda)
    most = min(entries, stride)
    slots[:, :most] = torch.where(order[:, :most] < 1.5, chosen[:, :most], -1).to(torch.int32)
    owners = torch.randperm(batch, generator=cpu).to(torch.int32).to(cuda)
    state = dict(
        op="attention", query=torch.randn((tokens, heads, WIDTH), generator=g, device=cuda).to(kind), pool=pool, slots=slots,
        requests=requests, owners=owners, starts=torch.tensor(starts, dtype=torch.int32, device=cuda),
        draft=(torch.randn((tokens, WIDTH), generator=g, device=cuda) + mean).to(kind),
        ancestors=torch.tensor(masks, dtype=torch.int64, device=cuda), scale=192 ** -0.5, stride=stride, nodes=nodes)
    if own:
        import kvip_b200
        state["attend"] = kvip_b200.SlotAttention(torch, cuda, tokens=tokens, heads=heads, entries=entries, dtype=kind)
    return state


def _prepare_rotary(case, cuda, g, cpu):
    tokens, heads, width = case["tokens"], case["heads"], case["width"]
    kind = TYPES[case["type"]]
    # the tokens of a chunk follow one another somewhere in the context, those of a decode step come from anywhere
    if tokens > 1024:
        first = int(torch.randint(0, max(1, case["longest"] - tokens + 1), (1,), generator=cpu))
        positions = first + torch.arange(tokens, dtype=torch.int64, device=cuda)
    else:
        positions = torch.randint(0, case["longest"], (tokens,), generator=cpu).to(cuda)
    scaling = YARN if case["scaled"] else None
    state = dict(op=case["op"], positions=positions, width=width, layout=case["layout"], scaling=scaling)
    if case["op"] == "quantise":
        state["rows"] = torch.randn((tokens, heads, case["dim"]), generator=g, device=cuda).to(kind)
        if own:
            state["codes"] = torch.empty((tokens, heads, case["dim"]), dtype=torch.float8_e4m3fn, device=cuda)
            state["scales"] = torch.empty((tokens, heads), dtype=torch.float32, device=cuda)
    else:
        row = case["row"]
        state["query"] = torch.randn((tokens, heads, row), generator=g, device=cuda).to(kind)[..., row - width:]
        state["key"] = torch.randn((tokens, 1, row), generator=g, device=cuda).to(kind)[..., row - width:]
        if own:
            state["query_out"] = torch.empty((tokens, heads, width), dtype=kind, device=cuda)
            state["key_out"] = torch.empty((tokens, 1, width), dtype=kind, device=cuda)
    if own:
        import kvip_b200
        state["rotary"] = kvip_b200.Rotary(torch, width, cuda, layout=case["layout"], scaling=scaling)
    return state


def _prepare_verify(case, cuda, g, cpu):
    batch, nodes, vocabulary = case["batch"], case["nodes"], case["vocabulary"]
    kind = TYPES[case["type"]]
    counts = [nodes if not case["tree"] else int(torch.randint(1, nodes + 1, (1,), generator=cpu)) for _ in range(batch)]
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    parents = [p for n in counts for p in _parents(n, case["tree"], cpu)]
    rows = starts[-1]
    target = torch.empty((rows, vocabulary), dtype=kind, device=cuda)
    draft = torch.empty((rows, vocabulary), dtype=kind, device=cuda) if case["draft"] else None
    tokens = torch.zeros(rows, dtype=torch.int64, device=cuda)
    for b in range(batch):      # a request at a time: logits of a few likely tokens over a long tail, a draft that comes near
        a, z = starts[b], starts[b + 1]
        logits = torch.randn((z - a, vocabulary), generator=g, device=cuda) * 2.5
        target[a:z] = torch.softmax(logits, 1).to(kind)
        guess = torch.softmax(logits + 0.7 * torch.randn((z - a, vocabulary), generator=g, device=cuda), 1)
        if draft is not None:
            draft[a:z] = guess.to(kind)
        above = torch.tensor([max(0, p) for p in parents[a:z]], device=cuda)
        if draft is None:       # a draft without probabilities: its tokens are the target's likely ones, siblings differ
            tokens[a:z] = logits[above].topk(z - a, dim=1).indices.diagonal()
        else:
            tokens[a:z] = torch.multinomial(guess[above], 1, generator=g)[:, 0]
    state = dict(
        op="verify", target=target, draft=draft, tokens=tokens, parents=torch.tensor(parents, dtype=torch.int32, device=cuda),
        starts=torch.tensor(starts, dtype=torch.int32, device=cuda), nodes=nodes, depth=max(1, nodes - 1),
        accept=torch.rand(rows, generator=g, device=cuda), sample=torch.rand(batch, generator=g, device=cuda))
    if own:
        import kvip_b200
        state["verify"] = kvip_b200.DraftVerifier(torch, cuda, batch=batch, depth=max(1, nodes - 1))
    return state


def _prepare_maps(case, cuda, g, cpu):
    batch, pages, block, tokens = case["batch"], case["pages"], case["block"], case["tokens"]
    counts = torch.randint(1, case["most"] + 1, (batch,), generator=cpu)
    if case["most"] > 100:      # most requests of a mixed batch decode
        counts = torch.where(torch.rand(batch, generator=cpu) < 0.75, 1, counts)
    counts = torch.where(counts.cumsum(0) <= tokens, counts, 0)
    counts = counts.clamp(max=pages * block)
    lengths = (torch.rand(batch, generator=cpu) * (pages * block - counts + 1)).long()
    held = (lengths + block - 1) // block
    table = torch.full((batch, pages), -1, dtype=torch.int32)
    blocks = int(held.sum()) + int(((lengths + counts + block - 1) // block - held).sum()) + 5
    order = torch.randperm(blocks, generator=cpu).to(torch.int32)
    taken = torch.arange(pages)[None, :] < held[:, None]
    table[taken] = order[:int(held.sum())]
    free = order[int(held.sum()):].to(cuda)
    i32 = dict(dtype=torch.int32, device=cuda)
    state = dict(op="maps", counts=counts.to(**i32), lengths=lengths.to(**i32), held=held.to(**i32), table=table.to(cuda), free=free,
                 head=torch.zeros(1, **i32), block=block, tokens=tokens)
    if own:
        import kvip_b200
        state["tables"] = kvip_b200.BlockTables(torch, cuda, batch=batch, pages=pages, blocks=free.numel(), tokens=tokens, block=block)
        state["tables"].load(lengths=state["lengths"], held=state["held"], table=state["table"], free=free)
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    op = state["op"]
    if own:
        if op == "attention":
            return state["attend"](state["query"], state["pool"], state["slots"], scale=state["scale"], requests=state["requests"],
                                   row_owners=state["owners"], output_stride=state["stride"], starts=state["starts"],
                                   draft=state["draft"], ancestors=state["ancestors"])
        if op == "quantise":
            return state["rotary"].quantise(state["positions"], state["rows"], state["codes"], state["scales"])
        if op == "rotary":
            return state["rotary"](state["positions"], state["query"], state["key"], query_out=state["query_out"],
                                   key_out=state["key_out"])
        if op == "verify":
            return state["verify"](state["target"], state["draft"], state["tokens"], state["parents"], state["starts"],
                                   state["accept"], state["sample"])
        maps = state["tables"].plan(state["counts"])
        return (maps.positions, maps.slot_mapping, maps.requests, maps.starts, maps.ends, maps.held_after, maps.taken, maps.table)
    return {"attention": _attention, "quantise": _quantise, "rotary": _rotary, "verify": _verify, "maps": _maps}[op](state)


def _attention(s):
    query, pool, slots, draft = s["query"].float(), s["pool"], s["slots"], s["draft"].float()
    requests = s["requests"].long()
    base = s["owners"].long()[requests] * s["stride"]
    listed_rows = pool[(base[:, None] + slots.clamp(min=0)).reshape(-1)].float().view(slots.shape[0], slots.shape[1], WIDTH)
    node = torch.arange(s["nodes"], device=slots.device)
    begin, end = s["starts"].long()[requests], s["starts"].long()[requests + 1]
    here = begin[:, None] + node[None, :]
    seen = (here < end[:, None]) & ((s["ancestors"][:, None] >> node[None, :]) & 1).bool()
    drafted_rows = draft[torch.where(here < end[:, None], here, 0)]
    rows = torch.cat((listed_rows, drafted_rows), 1)
    visible = torch.cat((slots >= 0, seen), 1)
    logits = torch.bmm(query, rows.transpose(1, 2)) * s["scale"]
    logits = logits.masked_fill(~visible[:, None, :], -math.inf)
    top = logits.amax(2, keepdim=True).clamp(min=-1e30)
    weights = torch.exp(logits - top)
    total = weights.sum(2, keepdim=True)
    out = torch.bmm(weights, rows[:, :, :VALUE]) / total.clamp(min=1e-30)
    return out.to(s["query"].dtype), (top + torch.log(total))[:, :, 0]


def _angles(s):
    width, scaling = s["width"], s["scaling"]
    device = s["positions"].device
    index = torch.arange(0, width, 2, dtype=torch.float64, device=device)
    frequency = 10000.0 ** (-index / width)
    factor = 1.0
    if scaling:
        at = [width * math.log(scaling["original"] / (turns * 2 * math.pi)) / (2 * math.log(10000.0))
              for turns in (scaling["beta_fast"], scaling["beta_slow"])]
        low, high = max(0, math.floor(at[0])), min(width - 1, math.ceil(at[1]))
        ramp = ((index / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
        frequency = frequency * (1 - ramp) + frequency / scaling["factor"] * ramp
        factor = 0.1 * math.log(scaling["factor"]) + 1.0
    angle = s["positions"].double()[:, None] * frequency[None, :]
    return (torch.cos(angle) * factor).float()[:, None, :], (torch.sin(angle) * factor).float()[:, None, :]


def _turned(x, cos, sin, layout):
    x = x.float()
    half = x.shape[-1] // 2
    if layout == "half":
        a, b = x[..., :half], x[..., half:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)


def _rotary(s):
    cos, sin = _angles(s)
    return tuple(_turned(x, cos, sin, s["layout"]).to(x.dtype) for x in (s["query"], s["key"]))


def _quantise(s):
    cos, sin = _angles(s)
    rows, width = s["rows"], s["width"]
    turned = torch.cat((_turned(rows[..., :width], cos, sin, s["layout"]), rows[..., width:].float()), -1)
    most = turned.abs().amax(-1)
    scales = torch.where(most > 0, most / 448, 1.0)
    return (turned / scales[..., None]).to(torch.float8_e4m3fn), scales


def _verify(s):
    target, draft, starts = s["target"], s["draft"], s["starts"].long()
    batch, vocabulary, depth = starts.numel() - 1, target.shape[1], s["depth"]
    device = target.device
    count = starts[1:] - starts[:-1]

    def row_of(matrix, at):
        x = matrix[at].double()
        return torch.where(x > 0, x, 0.0)

    here = torch.arange(batch, device=device)
    current = torch.zeros(batch, dtype=torch.int64, device=device)
    length = torch.zeros(batch, dtype=torch.int64, device=device)
    dead = torch.zeros(batch, dtype=torch.bool, device=device)
    weight = torch.ones(batch, dtype=torch.float64, device=device)
    tokens = torch.full((batch, depth + 2), -1, dtype=torch.int64, device=device)
    path = torch.full((batch, depth + 2), -1, dtype=torch.int32, device=device)
    live = count > 0
    path[:, 0] = torch.where(live, 0, -1).to(torch.int32)
    root = torch.where(live, starts[:-1], 0)
    rest = row_of(target, root)
    for node in range(1, s["nodes"]):          # every node after its parent: the walk down the tree, one node at a time
        at = torch.where(node < count, starts[:-1] + node, 0)
        tested = (node < count) & (s["parents"].long()[at] == current) & ~dead & (length < depth)
        token = s["tokens"][at]
        if draft is None:
            guess = torch.zeros((batch, vocabulary), dtype=torch.float64, device=device)
            guess[here, token] = 1.0
        else:
            guess = row_of(draft, root + current)
        limit = s["accept"].double()[at] * guess[here, token] * weight
        good = tested & (limit < rest[here, token])
        bad = tested & ~good
        if draft is None:                      # a draft that is certain of its token: the rejected token alone is lost
            left = rest.clone()
            left[here, token] = 0.0
        else:
            left = (rest - weight[:, None] * guess).clamp(min=0.0)
        mass = left.sum(1)
        length = length + good
        tokens[here, torch.where(good, length - 1, depth + 1)] = token
        path[here, torch.where(good, length, depth + 1)] = node
        current = torch.where(good, node, current)
        dead = dead | (bad & (mass == 0))
        weight = torch.where(good, 1.0, torch.where(bad, mass, weight))
        fresh = (good | (bad & (mass == 0)))[:, None]
        rest = torch.where(fresh, row_of(target, root + current), torch.where(bad[:, None], left, rest))
    sums = rest.cumsum(1)
    limit = s["sample"].double() * rest.sum(1)
    last = (torch.arange(vocabulary, device=device)[None, :] * (rest > 0)).amax(1)
    drawn = torch.minimum((sums <= limit[:, None]).sum(1), last)
    tokens[here, torch.where(live, length, depth + 1)] = drawn
    return tokens[:, :depth + 1].contiguous(), path[:, :depth + 1].contiguous(), torch.where(live, length + 1, 0).to(torch.int32)


def _maps(s):
    counts, lengths, held, block = s["counts"].long(), s["lengths"].long(), s["held"].long(), s["block"]
    batch, tokens, device = counts.numel(), s["tokens"], counts.device
    starts = torch.zeros(batch + 1, dtype=torch.int64, device=device)
    starts[1:] = counts.cumsum(0)
    ends = lengths + counts
    fresh = ((ends + block - 1) // block - held).clamp(min=0)
    offset = fresh.cumsum(0) - fresh
    table, page = s["table"], torch.arange(s["table"].shape[1], device=device)[None, :]
    added = (page >= held[:, None]) & (page < (held + fresh)[:, None])
    source = (s["head"].long() + offset[:, None] + page - held[:, None]).clamp(0, s["free"].numel() - 1)
    table.copy_(torch.where(added, s["free"][source], table))
    token = torch.arange(tokens, device=device)
    request = torch.searchsorted(starts, token, right=True) - 1
    real = token < starts[-1]
    request = torch.where(real, request, 0)
    position = lengths[request] + token - starts[request]
    slot = table[request, torch.where(real, position // block, 0)].long() * block + position % block
    return (torch.where(real, position, -1), torch.where(real, slot, -1), torch.where(real, request, -1).to(torch.int32),
            starts.to(torch.int32), ends.to(torch.int32), (held + fresh).to(torch.int32), fresh.sum().view(1).to(torch.int32), table)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "attention":
        tokens = case["batch"] * (case["nodes"] + 1) / 2 if case["ragged"] else case["batch"] * case["nodes"]
        context = (case["context"] + 1) / 2 if case["ragged"] else case["context"]
        rows = min(case["entries"], context) + (case["nodes"] + 1) / 2
        size = SIZE[case["type"]]
        # lists of one request's tokens may meet in the cache: each cached row is read once at most
        once = min(tokens * rows, case["batch"] * (context + case["nodes"]))
        return {"bytes": once * WIDTH * size + tokens * (case["heads"] * ((WIDTH + VALUE) * size + 4) + case["entries"] * 4),
                "flops": 2 * tokens * case["heads"] * rows * (WIDTH + VALUE)}
    if op == "quantise":
        values = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": values * (SIZE[case["type"]] + 1) + case["tokens"] * (8 + 4 * case["heads"]), "flops": 6 * values}
    if op == "rotary":
        values = case["tokens"] * (case["heads"] + 1) * case["width"]
        return {"bytes": values * 2 * SIZE[case["type"]] + case["tokens"] * 8, "flops": 3 * values}
    if op == "verify":
        rows = case["batch"] * (2 if case["draft"] and case["nodes"] > 1 else 1)
        return {"bytes": rows * case["vocabulary"] * SIZE[case["type"]], "flops": 3 * rows * case["vocabulary"]}
    return {"bytes": case["tokens"] * 20 + case["batch"] * 28, "flops": 10 * case["tokens"]}


# ---- the same from the definitions, in 64 bits -----------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "attention":
        starts, requests, owners, ancestors = (s[k].tolist() for k in ("starts", "requests", "owners", "ancestors"))
        out, lse = [], []
        for t, r in enumerate(requests):
            picked = s["slots"][t]
            mine = [s["pool"][owners[r] * s["stride"] + picked[picked >= 0].long()]]
            mine += [s["draft"][starts[r] + j][None] for j in range(starts[r + 1] - starts[r]) if ancestors[t] >> j & 1]
            mine = torch.cat(mine).double()
            logits = s["query"][t].double() @ mine.T * s["scale"]
            lse.append(torch.logsumexp(logits, 1))
            out.append(torch.softmax(logits, 1) @ mine[:, :VALUE])
        return torch.stack(out), torch.stack(lse)
    if op in ("rotary", "quantise"):
        width, half = s["width"], s["width"] // 2
        frequency = [10000.0 ** (-2.0 * i / width) for i in range(half)]
        factor = 1.0
        if s["scaling"]:
            y = s["scaling"]
            edge = [width * math.log(y["original"] / (beta * 2 * math.pi)) / (2 * math.log(10000.0)) for beta in (y["beta_fast"], y["beta_slow"])]
            low, high = max(0, math.floor(edge[0])), min(width - 1, math.ceil(edge[1]))
            for i in range(half):
                share = min(1.0, max(0.0, (i - low) / max(high - low, 1e-3)))
                frequency[i] = frequency[i] * (1 - share) + frequency[i] / y["factor"] * share
            factor = 0.1 * math.log(y["factor"]) + 1.0
        angle = s["positions"].double()[:, None] * torch.tensor(frequency, dtype=torch.float64, device="cuda")
        turn = torch.polar(torch.full_like(angle, factor), angle)[:, None, :]      # a complex number per pair

        def turned(x):
            x = x.double()
            pairs = x.unflatten(-1, (half, 2)) if s["layout"] == "interleaved" else x.unflatten(-1, (2, half)).transpose(-1, -2)
            y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            return (y if s["layout"] == "interleaved" else y.transpose(-1, -2)).flatten(-2)

        if op == "rotary":
            return turned(s["query"]), turned(s["key"])
        whole = s["rows"].double()
        whole[..., :width] = turned(s["rows"][..., :width])
        scale = whole.abs().amax(-1) / 448
        return whole / scale[..., None], scale
    if op == "verify":
        import numpy
        target = s["target"].double().cpu().numpy()
        draft = None if s["draft"] is None else s["draft"].double().cpu().numpy()
        starts, parents, tokens, accept, sample = (s[k].tolist() for k in ("starts", "parents", "tokens", "accept", "sample"))
        out_tokens, out_path, out_count = [], [], []
        for b, a in enumerate(starts[:-1]):
            n, node, said, went = starts[b + 1] - a, 0, [], [0]
            while True:
                rest, mass, found = target[a + node], 1.0, None
                for child in [j for j in range(1, n) if parents[a + j] == node]:
                    if draft is None:
                        guess = numpy.zeros(rest.size)
                        guess[tokens[a + child]] = 1.0
                    else:
                        guess = draft[a + node]
                    if accept[a + child] * guess[tokens[a + child]] * mass < rest[tokens[a + child]]:
                        found = child
                        break
                    rest = numpy.maximum(rest - mass * guess, 0.0) if draft is not None else rest * (guess == 0)
                    mass = rest.sum()
                if found is None:
                    break
                node = found
                said.append(tokens[a + found])
                went.append(found)
            sums = numpy.cumsum(rest)
            said.append(int(min(numpy.searchsorted(sums, sample[b] * rest.sum(), side="right"), numpy.flatnonzero(rest > 0)[-1])))
            out_count.append(len(said))
            out_tokens.append(said + [-1] * (s["depth"] + 1 - len(said)))
            out_path.append(went + [-1] * (s["depth"] + 1 - len(went)))
        return (torch.tensor(out_tokens, device="cuda"), torch.tensor(out_path, dtype=torch.int32, device="cuda"),
                torch.tensor(out_count, dtype=torch.int32, device="cuda"))
    return None     # whole numbers: the plain form is the definition
