"""Attention over the slots that the selection returns, with the drafted tokens of a tree.

The reference leaves attention to the serving framework; `slot_output` and the resident pool are its interface to it.
`SlotAttention` reads both where they lie: no dense gather is needed, every token's rows go from the pool into the
kernel once."""
from .. import _lib, _launch

WIDTH, VALUE = _lib.ATTENTION_WIDTH, _lib.ATTENTION_VALUE


class SlotAttention:
    """Attention of up to `tokens` packed query tokens with up to `heads` heads over `entries` slots each.

    A cache row has 576 elements (bf16 or fp16), the first 512 are its value as well. The call takes the query
    [tokens, heads, 576] in latent space, the resident pool (uint8 [rows, 1152] as `CudaBinding` binds it, or
    [rows, 576]), the slots of every token ([tokens, entries] or `slot_output` [tokens, 1, entries] int32, -1 = none) and,
    for drafted tokens, their rows of this step with the mask of their tree:

        out, lse = attend(query, pool, slots, scale=s, requests=maps.requests, row_owners=inputs.row_owners,
                          output_stride=rotating.output_stride, starts=maps.starts, draft=rows, ancestors=masks)

    Token t sees pool rows `owner * output_stride + slot` and the drafted rows `starts[request] + j` for the set bits j of
    `ancestors[t]` (int64; its own bit included; without `ancestors` a chain: every drafted row up to its own). out
    [tokens, heads, 512] in the query's type, lse [tokens, heads] float32 natural logarithm. A token that sees nothing gets zeros and
    -inf; a token with a negative request is padding and its outputs are left as they are. `status` collects KVIP_ERR_*
    bits of slots or requests out of range, which are skipped.

    There is no workspace; the outputs belong to this object unless the call gives its own, so calls without `out` and `lse`,
    and graphs captured from them, must follow one another."""

    def __init__(self, torch, device, *, tokens, heads, entries=_lib.TOPK, dtype=None):
        self.torch = torch
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("SlotAttention works on a CUDA device (kvip_b200 has no CPU path)")
        self.dtype = torch.bfloat16 if dtype is None else dtype
        if self.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("SlotAttention rows are bfloat16 or float16")
        if tokens < 1 or not 1 <= heads <= 128 or not 1 <= entries <= 1 << 20:
            raise ValueError("SlotAttention: at least one token, 1..128 heads, 1..2^20 entries")
        self.tokens, self.heads, self.entries = tokens, heads, entries
        self.out = torch.zeros((tokens, heads, VALUE), dtype=self.dtype, device=device)
        self.lse = torch.full((tokens, heads), float("-inf"), dtype=torch.float32, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.device, self.index = self.out.device, self.out.get_device()
        self._out, self._lse, self._status = self.out.data_ptr(), self.lse.data_ptr(), self.status.data_ptr()
        self.kind = _lib.FLOAT_BF16 if self.dtype == torch.bfloat16 else _lib.FLOAT_FP16
        self.launch = _launch.Launcher("kvip_b200_slot_attention")

    @property
    def nbytes(self):
        return sum(t.numel() * t.element_size() for t in (self.out, self.lse, self.status))

    def _flat(self, tensor, name, dtype, least, exact=False):
        """Address of a contiguous tensor of at least (or exactly) `least` elements."""
        count = tensor.numel()
        if count < least or (exact and count != least) or tensor.dtype != dtype or tensor.get_device() != self.index or not tensor.is_contiguous():
            raise ValueError(f"SlotAttention {name} must be contiguous {dtype} with {least} elements on {self.device}")
        return tensor.data_ptr()

    def __call__(self, query, pool, slots, *, scale, output_stride, requests=None, row_owners=None, queries=1, starts=None,
                 draft=None, ancestors=None, out=None, lse=None, splits=0, wait_kilocycles=0):
        torch, index, dtype = self.torch, self.index, self.dtype
        shape, strides = query.shape, query.stride()
        if len(shape) != 3 or shape[2] != WIDTH or strides[2] != 1 or query.dtype != dtype or query.get_device() != index:
            raise ValueError(f"SlotAttention query must be {dtype} [tokens, heads, {WIDTH}], innermost stride 1, on {self.device}")
        tokens, heads, _ = shape
        if tokens > self.tokens or heads > self.heads or heads < 1:
            raise ValueError("SlotAttention query exceeds the bound tokens or heads")
        size = 1 if pool.dtype == torch.uint8 else 2
        rows, rest = divmod(pool.numel() * size, 2 * WIDTH)
        if (rest or pool.shape[-1] * size != 2 * WIDTH or (size == 2 and pool.dtype != dtype) or pool.get_device() != index
                or not pool.is_contiguous()):
            raise ValueError(f"SlotAttention pool must be contiguous uint8 [rows, {2 * WIDTH}] or {dtype} [rows, {WIDTH}]")
        listed = slots.shape
        entries = listed[-1]
        if (slots.dtype != torch.int32 or listed[0] != tokens or slots.numel() != tokens * entries or not 1 <= entries <= self.entries
                or slots.get_device() != index or not slots.is_contiguous()):
            raise ValueError("SlotAttention slots must be contiguous int32 [tokens, entries] (or [tokens, 1, entries]) within the bound entries")
        if not 1 <= output_stride <= rows:
            raise ValueError("SlotAttention output_stride must lie within the pool")
        if tokens == 0:
            return (self.out[:0, :heads] if out is None else out), (self.lse[:0, :heads] if lse is None else lse)
        batch = row_owners.numel() if row_owners is not None else starts.numel() - 1 if starts is not None else rows // output_stride
        if batch < 1:
            raise ValueError("SlotAttention needs at least one request")
        if requests is not None:
            requests_ptr = self._flat(requests, "requests", torch.int32, tokens)
        elif queries < 1 or batch * queries < tokens:
            raise ValueError("SlotAttention tokens without requests belong to request t // queries")
        else:
            requests_ptr = 0
        owners_ptr = 0 if row_owners is None else self._flat(row_owners, "row_owners", torch.int32, batch)
        draft_ptr = starts_ptr = ancestors_ptr = draft_token = 0
        if draft is not None:
            if starts is None:
                raise ValueError("SlotAttention draft rows need the requests' starts")
            starts_ptr = self._flat(starts, "starts", torch.int32, batch + 1, True)
            drafted = draft.shape
            if len(drafted) != 2 or drafted[0] < tokens or drafted[1] != WIDTH or draft.dtype != dtype or draft.get_device() != index:
                raise ValueError(f"SlotAttention draft must be {dtype} [tokens, {WIDTH}]")
            draft_token, inner = draft.stride()
            if inner != 1:
                raise ValueError("SlotAttention draft needs an innermost stride of 1")
            draft_ptr = draft.data_ptr()
            if ancestors is not None:
                ancestors_ptr = self._flat(ancestors, "ancestors", torch.int64, tokens)
        elif ancestors is not None:
            raise ValueError("SlotAttention ancestors need draft rows")
        whole = tokens == self.tokens and heads == self.heads
        if out is None:
            out = self.out if whole else self.out.view(-1)[:tokens * heads * VALUE].view(tokens, heads, VALUE)
            out_ptr = self._out
        else:
            out_ptr = self._flat(out, "out", dtype, tokens * heads * VALUE, True)
        if lse is None:
            lse = self.lse if whole else self.lse.view(-1)[:tokens * heads].view(tokens, heads)
            lse_ptr = self._lse
        else:
            lse_ptr = self._flat(lse, "lse", torch.float32, tokens * heads, True)
        self.launch(
            index, query.data_ptr(), pool.data_ptr(), slots.data_ptr(), requests_ptr, owners_ptr, starts_ptr, draft_ptr, ancestors_ptr,
            out_ptr, lse_ptr, self._status, strides[0], strides[1], draft_token, rows, tokens, heads, entries, batch, queries,
            output_stride, self.kind, splits, wait_kilocycles, scale, 0)
        return out, lse
