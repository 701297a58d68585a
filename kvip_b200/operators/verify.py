"""Verification of drafted tokens: which of them the target keeps, and the token drawn where the walk ends.

The reference's query slots carry up to four tokens of a speculative step and leave their verification to the serving
framework. `DraftVerifier` walks every request's tree of drafted tokens on the GPU in one launch; the counts it returns
are what `BlockTables.commit` and the next step's maps take."""
from .. import _lib, _launch


class DraftVerifier:
    """Up to `batch` requests, at most `depth` accepted tokens each (1..63).

        tokens, nodes, counts = verify(target, draft, tokens, parents, starts, accept, sample)

    target [rows, vocabulary] (fp32, bf16 or fp16): the target's probabilities behind every packed row; row 0 of a
    request is its last committed token, the others its drafted tokens, each behind its parent (`parents` [rows] int32,
    local index; at most 64 rows a request, `starts` [batch + 1] int32). draft: the distributions the children of each
    row were drawn from, or None where the draft was certain. accept [rows] and sample [batch]: uniform numbers in
    [0, 1), float32. The rule stands in include/kvip_b200.h (KvipVerifyArgs): the tokens that come out are distributed as the
    target's own. Returns tokens [batch, depth + 1] int64 (accepted ones, then the drawn one, then -1), nodes
    [batch, depth + 1] int32 (0, the accepted rows, then -1) and counts [batch] int32 (accepted + 1), buffers of this object."""

    def __init__(self, torch, device, *, batch, depth=_lib.MAX_QUERIES - 1):
        self.torch = torch
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("DraftVerifier works on a CUDA device (kvip_b200 has no CPU path)")
        if not 1 <= batch <= 65536 or not 1 <= depth < _lib.MAX_NODES:
            raise ValueError("DraftVerifier: 1..65536 requests, a depth of 1..63")
        self.batch, self.depth = batch, depth
        self.tokens = torch.full((batch, depth + 1), -1, dtype=torch.int64, device=device)
        self.nodes = torch.full((batch, depth + 1), -1, dtype=torch.int32, device=device)
        self.counts = torch.zeros(batch, dtype=torch.int32, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.device, self.index = self.counts.device, self.counts.get_device()
        self._outputs = tuple(t.data_ptr() for t in (self.tokens, self.nodes, self.counts, self.status))
        self.types = {torch.bfloat16: _lib.FLOAT_BF16, torch.float16: _lib.FLOAT_FP16, torch.float32: _lib.FLOAT_FP32}
        self.launch = _launch.Launcher("kvip_b200_verify_drafts")

    def _flat(self, tensor, name, dtype, count):
        if tensor.numel() < count or tensor.dtype != dtype or tensor.ndim != 1 or tensor.get_device() != self.index or not tensor.is_contiguous():
            raise ValueError(f"DraftVerifier {name} must be contiguous {dtype} with at least {count} elements on {self.device}")
        return tensor.data_ptr()

    def __call__(self, target, draft, tokens, parents, starts, accept, sample):
        torch, index, flat = self.torch, self.index, self._flat
        kind, shape, strides = self.types.get(target.dtype), target.shape, target.stride()
        if kind is None or len(shape) != 2 or strides[1] != 1 or target.get_device() != index:
            raise ValueError(f"DraftVerifier target must be [rows, vocabulary] float32, bfloat16 or float16, innermost stride 1, on {self.device}")
        rows, vocabulary = shape
        if rows < 1 or not 1 <= vocabulary <= 1 << 24:
            raise ValueError("DraftVerifier: at least one row, a vocabulary of 1..2^24")
        draft_ptr, draft_row = 0, 0
        if draft is not None:
            draft_row, inner = draft.stride() if draft.ndim == 2 else (0, 0)
            if draft.shape != shape or draft.dtype != target.dtype or inner != 1 or draft.get_device() != index:
                raise ValueError("DraftVerifier draft must match the target")
            draft_ptr = draft.data_ptr()
        if starts.numel() != self.batch + 1:
            raise ValueError("DraftVerifier starts must be [batch + 1]")
        self.launch(
            index, target.data_ptr(), draft_ptr, flat(tokens, "tokens", torch.int64, rows), flat(parents, "parents", torch.int32, rows),
            flat(starts, "starts", torch.int32, self.batch + 1), flat(accept, "accept", torch.float32, rows),
            flat(sample, "sample", torch.float32, self.batch), *self._outputs, strides[0], draft_row, rows, vocabulary,
            self.batch, self.depth, kind, 0)
        return self.tokens, self.nodes, self.counts
