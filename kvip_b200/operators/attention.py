"""Attention over the slots that the selection returns, with the drafted tokens of a tree.

The reference leaves attention to the serving framework; `slot_output` and the resident pool are its interface to it.
`SlotAttention` reads both where they lie: no dense gather is needed, every token's rows go from the pool into the
kernel once."""
from .. import _lib, _launch


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
        self.out = torch.zeros((tokens, heads, _lib.ATTENTION_VALUE), dtype=self.dtype, device=device)
        self.lse = torch.full((tokens, heads), float("-inf"), dtype=torch.float32, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.device, self.index = self.out.device, self.out.get_device()
        self._status = self.status.data_ptr()
        self.launch = _launch.Launcher("kvip_b200_slot_attention")

    @property
    def nbytes(self):
        return sum(t.numel() * t.element_size() for t in (self.out, self.lse, self.status))

    def _flat(self, tensor, name, dtype, count):
        if tensor.dtype != dtype or tensor.numel() != count or tensor.get_device() != self.index or not tensor.is_contiguous():
            raise ValueError(f"SlotAttention {name} must be contiguous {dtype} with {count} elements on {self.device}")
        return tensor.data_ptr()

    def __call__(self, query, pool, slots, *, scale, output_stride, requests=None, row_owners=None, queries=1, starts=None,
                 draft=None, ancestors=None, out=None, lse=None, splits=0, wait_kilocycles=0):
        torch, index, width = self.torch, self.index, _lib.ATTENTION_WIDTH
        if query.ndim != 3 or query.shape[2] != width or query.dtype != self.dtype or query.stride(2) != 1 or query.get_device() != index:
            raise ValueError(f"SlotAttention query must be {self.dtype} [tokens, heads, {width}], innermost stride 1, on {self.device}")
        tokens, heads = query.shape[0], query.shape[1]
        if tokens > self.tokens or heads > self.heads or heads < 1:
            raise ValueError("SlotAttention query exceeds the bound tokens or heads")
        if (pool.shape[-1] * pool.element_size() != 2 * width or pool.dtype not in (torch.uint8, self.dtype) or pool.get_device() != index
                or not pool.is_contiguous()):
            raise ValueError(f"SlotAttention pool must be contiguous uint8 [rows, {2 * width}] or {self.dtype} [rows, {width}]")
        if slots.dtype != torch.int32 or not slots.is_contiguous() or slots.get_device() != index or slots.shape[0] != tokens:
            raise ValueError("SlotAttention slots must be contiguous int32 [tokens, entries]")
        entries = slots.shape[-1]
        if slots.numel() != tokens * entries or not 1 <= entries <= self.entries:
            raise ValueError("SlotAttention slots must be [tokens, entries] (or [tokens, 1, entries]) within the bound entries")
        rows = pool.numel() * pool.element_size() // (2 * width)
        if not 1 <= output_stride <= rows:
            raise ValueError("SlotAttention output_stride must lie within the pool")
        if tokens == 0:
            return (self.out[:0, :heads] if out is None else out), (self.lse[:0, :heads] if lse is None else lse)
        if row_owners is not None:
            batch = row_owners.numel()
        elif starts is not None:
            batch = starts.numel() - 1
        else:
            batch = rows // output_stride
        requests_ptr = 0 if requests is None else self._flat(requests, "requests", torch.int32, requests.numel())
        if requests is None:
            if queries < 1 or batch * queries < tokens:
                raise ValueError("SlotAttention tokens without requests belong to request t // queries")
        elif requests.numel() < tokens:
            raise ValueError("SlotAttention requests must cover the tokens")
        owners_ptr = 0 if row_owners is None else self._flat(row_owners, "row_owners", torch.int32, batch)
        draft_ptr = starts_ptr = ancestors_ptr = 0
        draft_token = 0
        if draft is not None:
            if starts is None:
                raise ValueError("SlotAttention draft rows need the requests' starts")
            starts_ptr = self._flat(starts, "starts", torch.int32, batch + 1)
            if draft.ndim != 2 or draft.shape[0] < tokens or draft.shape[1] != width or draft.dtype != self.dtype or draft.stride(1) != 1 \
                    or draft.get_device() != index:
                raise ValueError(f"SlotAttention draft must be {self.dtype} [tokens, {width}], innermost stride 1")
            draft_ptr, draft_token = draft.data_ptr(), draft.stride(0)
            if ancestors is not None:
                if ancestors.numel() < tokens:
                    raise ValueError("SlotAttention ancestors must cover the tokens")
                ancestors_ptr = self._flat(ancestors, "ancestors", torch.int64, ancestors.numel())
        elif ancestors is not None:
            raise ValueError("SlotAttention ancestors need draft rows")
        if out is None:
            out = self.out if tokens == self.tokens and heads == self.heads else self.out.view(-1)[
                :tokens * heads * _lib.ATTENTION_VALUE].view(tokens, heads, _lib.ATTENTION_VALUE)
            out_ptr = out.data_ptr()
        else:
            out_ptr = self._flat(out, "out", self.dtype, tokens * heads * _lib.ATTENTION_VALUE)
        if lse is None:
            lse = self.lse if tokens == self.tokens and heads == self.heads else self.lse.view(-1)[:tokens * heads].view(tokens, heads)
            lse_ptr = lse.data_ptr()
        else:
            lse_ptr = self._flat(lse, "lse", torch.float32, tokens * heads)
        self.launch(
            index, query.data_ptr(), pool.data_ptr(), slots.data_ptr(), requests_ptr, owners_ptr, starts_ptr, draft_ptr, ancestors_ptr,
            out_ptr, lse_ptr, self._status, query.stride(0), query.stride(1), draft_token, rows, tokens, heads, entries, batch,
            queries, output_stride, _lib.FLOAT_BF16 if self.dtype == torch.bfloat16 else _lib.FLOAT_FP16, splits,
            wait_kilocycles, scale, 0)
        return out, lse
