"""Rotary positions of queries and keys, and the rotated FP8 form that `QueryInputs.pack` takes.

The reference receives its Index queries and keys rotated and quantised by the serving framework; there is nothing of
this kind in it. `Rotary` turns part of every row by its token's position: the whole of the rows it is given in place or
into other tensors (`__call__`, the 64-wide rope part of latent queries and keys, or the rotated part of Index keys
before `ingest_decode`), or the first `width` elements of longer Index rows that are quantised to FP8 e4m3 with one
scale per row in the same pass (`quantise`)."""
import math

from . import _lib, _launch

LAYOUTS = {"half": 0, "interleaved": 1}


def frequencies(width, base=10000.0, scaling=None):
    """Angle per position of every pair, in double precision, and the factor on the rotated elements.

    scaling: None; `{"kind": "linear", "factor": f}` (positions divided by f); or `{"kind": "yarn", "factor": f,
    "original": n, "beta_fast": 32, "beta_slow": 1, "attention_factor": None}`: pairs that turn less than beta_slow
    times over the original context are divided by f, pairs that turn more than beta_fast times are kept, and between the
    two (in pair numbers, rounded outwards) the share grows linearly; the factor defaults to 0.1 ln f + 1."""
    pairs = [float(base) ** (-2.0 * i / width) for i in range(width // 2)]
    if scaling is None:
        return pairs, 1.0
    kind, factor = scaling.get("kind"), float(scaling.get("factor", 1.0))
    if kind not in ("linear", "yarn") or not factor >= 1.0:
        raise ValueError("Rotary scaling is None, linear or yarn, with a factor of at least one")
    if kind == "linear":
        return [f / factor for f in pairs], 1.0
    original = scaling.get("original")
    fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
    if not original or not fast > slow > 0 or not base > 1:
        raise ValueError("Rotary yarn scaling needs the original context, beta_fast > beta_slow > 0 and a base above one")

    def pair_turning(times):
        return width * math.log(original / (times * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(0, math.floor(pair_turning(fast))), min(width - 1, math.ceil(pair_turning(slow)))
    mixed = []
    for i, f in enumerate(pairs):
        share = min(1.0, max(0.0, (i - low) / max(high - low, 1e-3)))
        mixed.append(f * (1 - share) + f / factor * share)
    attention = scaling.get("attention_factor")
    return mixed, 0.1 * math.log(factor) + 1.0 if attention is None else float(attention)


class Rotary:
    """`width` rotated elements per row, `layout` "half" (element i pairs with i + width / 2) or "interleaved" (2i with
    2i + 1). The frequency table is made once here; a call is one launch on the current stream of the rows' device."""

    def __init__(self, torch, width, device, *, layout="half", base=10000.0, scaling=None):
        self.torch, self.device = torch, torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("Rotary works on a CUDA device (kvip_b200 has no CPU path)")
        if type(width) is not int or width < 2 or width % 2 or width > 1024:
            raise ValueError("Rotary width is an even number up to 1024")
        if layout not in LAYOUTS:
            raise ValueError("Rotary layout is 'half' or 'interleaved'")
        pairs, self.factor = frequencies(width, base, scaling)
        self.width, self.layout = width, LAYOUTS[layout]
        self.turns = torch.tensor([f / (2 * math.pi) for f in pairs], dtype=torch.float64, device=self.device)
        self.index, self._table = self.turns.get_device(), self.turns.data_ptr()
        self.types = {torch.bfloat16: _lib.FLOAT_BF16, torch.float16: _lib.FLOAT_FP16, torch.float32: _lib.FLOAT_FP32}
        self.launch = _launch.Launcher("kvip_b200_rotary")

    def _rows(self, tensor, tokens, what, kind=None):
        """(pointer, token stride, head stride, heads) of rows [tokens, heads, width] or [tokens, width]."""
        shape, dims = tensor.shape, tensor.ndim
        if dims not in (2, 3) or shape[0] != tokens or shape[-1] != self.width or tensor.stride(-1) != 1:
            raise ValueError(f"Rotary {what} must be [tokens, heads, {self.width}] or [tokens, {self.width}], innermost stride 1")
        if tensor.get_device() != self.index or (kind is not None and tensor.dtype != kind):
            raise ValueError(f"Rotary {what} must have the query's type, on {self.turns.device}")
        if dims == 2:
            return tensor.data_ptr(), tensor.stride(0), 0, 1
        return tensor.data_ptr(), tensor.stride(0), tensor.stride(1), shape[1]

    def _tokens(self, positions):
        if positions.dtype != self.torch.int64 or positions.ndim != 1 or positions.get_device() != self.index or not positions.is_contiguous():
            raise ValueError(f"Rotary positions must be a flat int64 tensor on {self.turns.device}")
        return positions.numel()

    def __call__(self, positions, query, key=None, *, query_out=None, key_out=None):
        """Rotate `query` (and `key`), in place or into `query_out` / `key_out`. Rows are [tokens, heads, width] or
        [tokens, width] views with any strides (bf16, fp16 or fp32); positions int64 [tokens], and the rows of a token with
        a negative position (padding) are not written. Outputs that are not in place, and query and key, have no
        element in common. Returns (query_out, key_out)."""
        tokens = self._tokens(positions)
        kind = query.dtype
        if kind not in self.types:
            raise ValueError("Rotary rows are bfloat16, float16 or float32")
        query_out = query if query_out is None else query_out
        x0, xt0, xh0, heads0 = self._rows(query, tokens, "query")
        y0, yt0, yh0, out0 = self._rows(query_out, tokens, "query_out", kind)
        x1 = y1 = 0
        xt1 = xh1 = yt1 = yh1 = heads1 = out1 = 0
        if key is not None:
            key_out = key if key_out is None else key_out
            x1, xt1, xh1, heads1 = self._rows(key, tokens, "key", kind)
            y1, yt1, yh1, out1 = self._rows(key_out, tokens, "key_out", kind)
        elif key_out is not None:
            raise ValueError("Rotary key_out needs a key")
        if heads0 != out0 or heads1 != out1:
            raise ValueError("Rotary outputs must have their inputs' heads")
        if tokens == 0 or heads0 == 0:
            if tokens and heads1:
                raise ValueError("Rotary query needs at least one head")
            return query_out, key_out
        if heads1 == 0:
            x1 = y1 = 0
        self.launch(self.index, positions.data_ptr(), self._table, x0, x1, y0, y1, 0, 0, xt0, xt1, xh0, xh1, yt0, yt1, yh0, yh1,
                    heads0, heads1, tokens, self.width, self.width, self.layout, self.types[kind], self.factor)
        return query_out, key_out

    def quantise(self, positions, rows, codes=None, scales=None):
        """Rotate the first `width` elements of every row and quantise the whole row: rows [tokens, heads, dim] ->
        (codes [tokens, heads, dim] float8_e4m3fn, scales [tokens, heads] float32) with scale = amax / 448, at least 2^-126 (1 for a row of
        zeros), and codes of the quotients by it, the rule of `IndexCacheStorage.ingest_decode`. Rows of tokens with a negative position are not written.
        Without `codes` / `scales` the outputs are allocated."""
        torch = self.torch
        tokens = self._tokens(positions)
        if rows.dtype not in self.types:
            raise ValueError("Rotary rows are bfloat16, float16 or float32")
        if rows.ndim != 3 or rows.shape[0] != tokens or rows.shape[2] < self.width or rows.stride(2) != 1 or rows.get_device() != self.index:
            raise ValueError(f"Rotary rows must be [tokens, heads, dim >= {self.width}], innermost stride 1, on {self.turns.device}")
        heads, dim = rows.shape[1], rows.shape[2]
        if codes is None:
            codes = torch.empty((tokens, heads, dim), dtype=torch.float8_e4m3fn, device=rows.device)
        if scales is None:
            scales = torch.empty((tokens, heads), dtype=torch.float32, device=rows.device)
        if codes.shape != rows.shape or codes.dtype != torch.float8_e4m3fn or not codes.is_contiguous() or codes.get_device() != self.index:
            raise ValueError("Rotary codes must be contiguous float8_e4m3fn of the rows' shape")
        if scales.shape != (tokens, heads) or scales.dtype != torch.float32 or not scales.is_contiguous() or scales.get_device() != self.index:
            raise ValueError("Rotary scales must be contiguous float32 [tokens, heads]")
        if tokens == 0 or heads == 0:
            return codes, scales
        self.launch(self.index, positions.data_ptr(), self._table, rows.data_ptr(), 0, 0, 0, codes.data_ptr(), scales.data_ptr(),
                    rows.stride(0), 0, rows.stride(1), 0, 0, 0, 0, 0, heads, 0, tokens, self.width, dim, self.layout,
                    self.types[rows.dtype], self.factor)
        return codes, scales
