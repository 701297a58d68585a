"""Block tables of the paged caches, kept on the GPU, and the slot maps of a step made from the requests' lengths there.

The reference receives `metadata.slot_mapping`, positions and block tables from the serving framework's host code. A step
that follows a verification of drafted tokens knows its lengths only on the GPU; `BlockTables` makes the maps from
them in one launch, with no copy to the host and none from it: blocks from a free list, packed positions, slots and
requests, and (for `QueryInputs.prepare_device`) the layout of the query slots."""
from .. import _lib, _launch


class BlockTables:
    """State of `batch` requests over a pool of `blocks` blocks of `block` tokens: `table` [batch, pages] int32,
    `lengths` [batch] cached tokens, `held` [batch] blocks in the row, `free` [blocks] and `head` [1], the first entry of
    the free list that is still free. A step is

        tables.plan(counts)       # one launch: appends blocks, fills positions, slot_mapping, requests, starts, ends
        ...                       # the forward reads them
        tables.commit(kept)       # lengths += kept (the tokens that stay), the blocks of the plan become the request's

    `plan` changes nothing but the table entries behind `held`, so a step that is planned again plans the same. `commit`, `load` and
    `release` end a plan: until the next one there is nothing to commit. Outputs are
    persistent buffers of this object, sized by `tokens` (packed tokens per step at most): the captured graph of a
    step finds them at the same place. `status` collects KVIP_ERR_* bits (include/kvip_b200.h: KvipSlotMapsArgs)."""

    _planned = ()      # outputs of a plan that `commit` takes over, each with its value where nothing is planned (then it keeps nothing)

    def __init__(self, torch, device, *, batch, pages, blocks, tokens, block=_lib.BLOCK_TOKENS, queries=0):
        self.torch = torch
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("BlockTables live on a CUDA device (kvip_b200 has no CPU path)")
        if not 1 <= batch <= 1024 or pages < 1 or tokens < 1 or block < 1 or blocks < 0:
            raise ValueError("BlockTables: 1..1024 requests, at least one page, one token and one token per block")
        if pages * block > 0x7fffffff or batch * pages * block > 0xffffffff:
            raise ValueError("BlockTables: pages * block must fit int32, batch * pages * block 32 bits")
        if not 0 <= queries <= _lib.MAX_QUERIES:
            raise ValueError("BlockTables: zero to four query slots per request")
        self.batch, self.pages, self.blocks, self.tokens, self.block, self.queries = batch, pages, blocks, tokens, block, queries
        # one block of int32 and one of int64 words: a table is made in a few launches
        i32, i64 = dict(dtype=torch.int32, device=device), dict(dtype=torch.int64, device=device)
        words = torch.zeros(5 * batch + 5 + tokens, **i32)
        (self.lengths, self.held, self.ends, self.held_after, self.starts, self.head, self.taken, self.status, nothing, self.requests) = words.split(
            (batch, batch, batch, batch, batch + 1, 1, 1, 1, 1, tokens))
        self._planned = ((self.ends, self.lengths), (self.held_after, self.held), (self.taken, nothing))
        self.positions, self.slot_mapping = torch.full((2, tokens), -1, **i64).unbind(0)
        self.table = torch.full((batch, pages), -1, **i32)
        self.free = torch.arange(max(1, blocks), **i32)
        self.layout = torch.zeros((4, batch * queries), **i64) if queries else None
        self.device, self.index = self.table.device, self.table.get_device()
        self.launch, self.launch_commit = _launch.Launcher("kvip_b200_slot_maps"), _launch.Launcher("kvip_b200_commit_tables")
        self._commit = tuple(t.data_ptr() for t in (self.starts, self.held_after, self.lengths, self.held, self.ends, self.head, self.taken,
                                                    self.status)) + (batch, 0)
        outputs = (self.table, self.positions, self.slot_mapping, self.requests, self.starts, self.ends, self.held_after, self.taken,
                   self.status)
        pointers = tuple(t.data_ptr() for t in outputs) + (self.layout.data_ptr() if queries else 0,)
        # the record behind `counts`: every buffer is this object's own
        self._rest = (self.held.data_ptr(), self.free.data_ptr(), self.head.data_ptr(), *pointers, batch, pages, blocks, tokens,
                      block, queries)
        self._lengths = self.lengths.data_ptr()

    @property
    def nbytes(self):
        tensors = [self.lengths, self.held, self.table, self.free, self.head, self.positions, self.slot_mapping, self.requests,
                   self.starts, self.ends, self.held_after, self.taken, self.status]
        return sum(t.numel() * t.element_size() for t in tensors + ([self.layout] if self.queries else []))

    def load(self, *, lengths, held, table, free, head=0):
        """Take over a state made elsewhere (copies; the free list may be shorter than `blocks`)."""
        if free.numel() > self.blocks or not 0 <= head <= free.numel():
            raise ValueError("BlockTables.load: the free list does not fit")
        if tuple(table.shape) != (self.batch, self.pages) or lengths.numel() != self.batch or held.numel() != self.batch:
            raise ValueError("BlockTables.load: lengths, held and table must match the batch and its pages")
        self.lengths.copy_(lengths)
        self.held.copy_(held)
        self.table.copy_(table)
        gap = self.blocks - free.numel()          # the list ends where the storage ends
        self.free[gap:self.blocks].copy_(free)
        self.head.fill_(gap + head)
        self._end_plan()

    def plan(self, counts):
        """Maps of a step that adds counts[b] tokens to request b (int32 [batch] on the device): one launch, no host
        copy, capturable. Returns self."""
        if (counts.dtype != self.torch.int32 or counts.ndim != 1 or counts.numel() != self.batch or counts.get_device() != self.index
                or not counts.is_contiguous()):
            raise ValueError("BlockTables counts must be contiguous int32 [batch] on the tables' device")
        self.launch(self.index, self._lengths, counts.data_ptr(), *self._rest)
        return self

    def tree_positions(self, depths):
        """Positions in the text of the planned tokens of trees: `lengths` + depth, where `positions` are the places of the tokens in
        the caches, one for each. depths: int32 [tokens] (or longer), 0 for a request's first token and one more than its parent's
        for the others. A depth that is negative or above the token's number in its request is taken as the nearest that is not
        (KVIP_ERR_TOKEN_RANGE); -1 where a token has no position. int64 [tokens], new; between `plan` and `commit`, capturable."""
        torch = self.torch
        if depths.dtype != torch.int32 or depths.ndim != 1 or depths.numel() < self.tokens or depths.device != self.table.device:
            raise ValueError("BlockTables depths must be flat int32 with an entry per packed token, on the tables' device")
        live = self.positions >= 0
        length = self.lengths[self.requests.clamp(min=0).long()]
        number = self.positions - length
        depth = depths[:self.tokens].long().clamp(min=0).minimum(number)
        self.status.bitwise_or_((live & (depth != depths[:self.tokens])).any().to(torch.int32) * _lib.ERR_TOKEN_RANGE)
        return torch.where(live, length + depth, -1)

    def commit(self, kept):
        """The planned blocks become the requests' own and `kept` [batch] int32 of the planned tokens stay (all of them, or
        what a verification accepted): one launch, capturable. A request that keeps fewer holds its blocks for the tokens to come; one
        that the plan gave no place (KVIP_ERR_*: `ends` is its length), or whose tokens were dropped behind the last output row, keeps
        none of those. A plan is committed once: without another one a second call keeps nothing. `status` says KVIP_ERR_TOKEN_RANGE
        where more should have been kept than was planned."""
        if tuple(kept.shape) != (self.batch,) or kept.get_device() != self.index:
            raise ValueError("BlockTables kept counts must be [batch] on the tables' device")
        kept = kept.to(self.torch.int32).contiguous()
        self.launch_commit(self.index, kept.data_ptr(), *self._commit)

    def _end_plan(self):
        for output, state in self._planned:
            output.copy_(state)

    def release(self, rows):
        """Requests that have ended (host list of row numbers): their blocks return to the free list, their rows are
        empty. Fixed shapes, no device read on the host. Blocks that the list has no place for (rows of `load` that hold more than was
        taken from it, or a block twice) are dropped, entries that are no block (a row with holes) are passed over, and `status` says
        KVIP_ERR_NO_SLOT for either. A plan that has not been committed ends here: its blocks are in the list still, and stay there."""
        rows = sorted(set(int(r) for r in rows))
        if not rows:
            return
        if rows[0] < 0 or rows[-1] >= self.batch:
            raise IndexError("BlockTables.release: row out of range")
        torch = self.torch
        index = torch.tensor(rows, dtype=torch.int64, device=self.device)
        table, held = self.table[index], self.held[index]
        page = torch.arange(self.pages, dtype=torch.int32, device=self.device)
        listed = page[None, :] < held[:, None]
        mine = (listed & (table >= 0)).reshape(-1)
        order = mine.cumsum(0)
        total = order[-1:]
        # the list grows downwards from head; entries that are no block, and blocks that the list has no place for (a state
        # whose rows hold more than was taken from it), go to a place behind it
        place = self.head.long() - total + order - 1
        fits = mine & (place >= 0) & (place < self.blocks)
        longer = torch.cat((self.free[:self.blocks], self.free[:1]))
        longer.scatter_(0, torch.where(fits, place, self.blocks), torch.where(fits, table.reshape(-1), longer[-1]))
        self.free[:self.blocks].copy_(longer[:-1])
        self.head.sub_(total.to(torch.int32)).clamp_(min=0)
        lost = ((mine & ~fits).any() | (listed & (table < 0)).any()).to(torch.int32) * _lib.ERR_NO_SLOT
        self.status.bitwise_or_(lost)
        self.table[index] = -1
        self.held[index] = 0
        self.lengths[index] = 0
        self._end_plan()
