"""Decode-step operators beside the BF16 ones of ``kernels``: the quantized KV cache and attention
over it, attention of drafted token trees, and constrained greedy logits.

Every function runs on its first tensor's device, on that device's current stream, and allocates
what it returns and its workspace per call, so calls on several streams and captured graphs share
nothing but the device's status word (``scratch(device).check()`` reads it: indexes and lengths
that live on the device are checked by the kernels, which read or write nothing outside a tensor
and record a status instead).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from .native import _scratch, native, scratch

BLOCK = 16  # positions of a cache block
_SCALE_BYTES = 64  # 16 FP32 scales behind a page's codes

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


class _Launch:
    """The device a call runs on: its status word and current stream, and the device as the current
    one while the call allocates and launches."""

    __slots__ = ("index", "status", "stream", "_guard")

    def __init__(self, first: torch.Tensor, *others: torch.Tensor | None):
        index = first.get_device()
        if index < 0:
            raise ValueError("the operands must be CUDA tensors")
        for t in others:
            if t is not None and t.get_device() != index:
                raise ValueError("the operands must be on one CUDA device")
        self.index = index
        s = _scratch.get(index)
        if s is None:
            with torch.cuda.device(index):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("the device's first call cannot be captured: its status word is laid out then")
                s = scratch(first.device)
        self.status = s.status.data_ptr()
        self.stream = _raw_stream(index)
        self._guard = None

    def __enter__(self):
        if torch.cuda.current_device() != self.index:
            self._guard = torch.cuda.device(self.index)
            self._guard.__enter__()
        return self

    def __exit__(self, *exc):
        if self._guard is not None:
            self._guard.__exit__(*exc)
        return False


def _ints(t: torch.Tensor, shape: tuple, name: str) -> None:
    if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {list(shape)}")


def _heads(t: torch.Tensor, name: str) -> None:
    """BF16 [rows, heads, d] whose rows are packed, each row 16-byte aligned."""
    if t.dtype != torch.bfloat16 or t.dim() != 3:
        raise ValueError(f"{name} must be BF16 [rows, heads, head_dim]")
    _, h, d = t.shape
    if (t.stride(2) != 1 and d != 1) or (t.stride(1) != d and h != 1):
        raise ValueError(f"{name} must have its heads packed in each row")
    if t.shape[0] > 1 and (t.stride(0) < h * d or t.stride(0) % 8):
        raise ValueError(f"{name} must have rows a multiple of 8 elements apart")
    if t.data_ptr() % 16:
        raise ValueError(f"{name} must be 16-byte aligned")


@dataclass
class QuantizedCache:
    """One layer's KV cache in quantized pages: bytes [blocks, 2 (K, V), kv_heads, 16 * d + 64], a
    block's 16 rows of one head as E4M3 codes followed by their 16 FP32 scales. An element's value is
    code * scale, a row's scale its largest magnitude / 448 (never below 1e-10 / 448). A page takes
    (16 d + 64) / 32 d of its BF16 form's bytes: 0.516 for d = 128."""

    pages: torch.Tensor
    head_dim: int

    def __post_init__(self):
        p = self.pages
        if p.dtype != torch.uint8 or p.dim() != 4 or p.shape[1] != 2 or not p.is_contiguous():
            raise ValueError("pages must be a contiguous uint8 tensor [blocks, 2, kv_heads, 16 * head_dim + 64]")
        if self.head_dim not in (64, 128) or p.shape[3] != BLOCK * self.head_dim + _SCALE_BYTES:
            raise ValueError("a quantized page holds 16 * head_dim + 64 bytes for a head_dim of 64 or 128")
        if p.data_ptr() % 16:
            raise ValueError("pages must be 16-byte aligned")

    @classmethod
    def empty(cls, blocks: int, kv_heads: int, head_dim: int, device=None) -> "QuantizedCache":
        """A cache of zeros."""
        return cls(torch.zeros(blocks, 2, kv_heads, BLOCK * head_dim + _SCALE_BYTES, dtype=torch.uint8,
                               device=device if device is not None else "cuda"), head_dim)

    @property
    def codes(self) -> torch.Tensor:
        """The E4M3 codes as a uint8 view [blocks, 2, kv_heads, 16, head_dim]."""
        return self.pages[..., :BLOCK * self.head_dim].unflatten(-1, (BLOCK, self.head_dim))

    @property
    def scales(self) -> torch.Tensor:
        """The scales as an FP32 view [blocks, 2, kv_heads, 16]."""
        return self.pages[..., BLOCK * self.head_dim:].view(torch.float32)

    def dequantize(self) -> torch.Tensor:
        """The values the cache stands for, FP32 [blocks, 2, kv_heads, 16, head_dim]."""
        return self.codes.view(torch.float8_e4m3fn).float() * self.scales.unsqueeze(-1)


def store_rows(qkv, q_heads, kv_heads, head_dim, q_norm, k_norm, eps, positions, inv_freq, attention_factor,
               cache, slots, rotary_dim=None, interleaved=False):
    """``kernels.qk_norm_rope_cache`` over a QuantizedCache, or with a partial or interleaved rotation."""
    quantized = isinstance(cache, QuantizedCache)
    rotary_dim = head_dim if rotary_dim is None else rotary_dim
    if qkv.dtype != torch.bfloat16 or qkv.dim() != 2 or qkv.shape[1] != (q_heads + 2 * kv_heads) * head_dim:
        raise ValueError("qkv must be BF16 [rows, (q_heads + 2 * kv_heads) * head_dim]")
    rows = qkv.shape[0]
    if kv_heads < 1 or q_heads < 0 or head_dim not in (64, 128):
        raise ValueError("head_dim must be 64 or 128, with at least one key/value head")
    if qkv.stride(1) != 1 or (rows > 1 and (qkv.stride(0) < qkv.shape[1] or qkv.stride(0) % 8)) or qkv.data_ptr() % 16:
        raise ValueError("qkv must have unit column stride and 16-byte aligned rows")
    if rotary_dim % 16 or not 16 <= rotary_dim <= head_dim:
        raise ValueError("rotary_dim must be a multiple of 16, at most head_dim")
    if (q_norm is None) != (k_norm is None):
        raise ValueError("q_norm and k_norm come together")
    for w in (q_norm, k_norm):
        if w is not None and (w.dtype != torch.bfloat16 or w.shape != (head_dim,) or not w.is_contiguous() or w.data_ptr() % 16):
            raise ValueError("norm weights must be contiguous BF16 [head_dim], 16-byte aligned")
    _ints(positions, (rows,), "positions")
    _ints(slots, (rows,), "slots")
    if inv_freq.dtype != torch.float32 or inv_freq.shape != (rotary_dim // 2,) or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous FP32 tensor of rotary_dim / 2 frequencies")
    if quantized:
        pages = cache.pages
        if cache.head_dim != head_dim or pages.shape[2] != kv_heads:
            raise ValueError("the cache has other heads")
    else:
        pages = cache
        if pages.dtype != torch.bfloat16 or pages.dim() != 5 or pages.shape[1:] != (2, kv_heads, BLOCK, head_dim) \
                or not pages.is_contiguous() or pages.data_ptr() % 16:
            raise ValueError("the cache must be contiguous BF16 [blocks, 2, kv_heads, 16, head_dim]")
    with _Launch(qkv, positions, slots, inv_freq, pages, q_norm, k_norm) as at:
        q = torch.empty(rows, q_heads, head_dim, dtype=torch.bfloat16, device=qkv.device)
        native().ops.kv_store(
            qkv.data_ptr(), qkv.stride(0) if rows > 1 else qkv.shape[1], rows, q_heads, kv_heads, head_dim,
            0 if q_norm is None else q_norm.data_ptr(), 0 if k_norm is None else k_norm.data_ptr(), eps,
            positions.data_ptr(), inv_freq.data_ptr(), attention_factor, rotary_dim, bool(interleaved), q.data_ptr(),
            pages.data_ptr(), quantized, slots.data_ptr(), pages.shape[0] * BLOCK, at.status, at.stream)
    return q


def tree_mask(parents) -> torch.Tensor:
    """The ``mask`` of ``paged_tree`` for drafted trees, as int32 [rows, words] on the CPU.

    ``parents`` holds a list per segment: each node's parent as its index in the segment, or -1 for a
    node that follows the history. A parent comes before its children. A node sees its ancestors and
    itself."""
    words = max((len(p) + 31) // 32 for p in parents) if len(parents) else 1
    rows = []
    for tree in parents:
        seen = []
        for i, p in enumerate(tree):
            if not -1 <= p < i:
                raise ValueError(f"node {i} has parent {p}: parents come before their children")
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
        rows += [[(b >> 32 * w) & 0xFFFFFFFF for w in range(words)] for b in seen]
    return torch.tensor(rows, dtype=torch.int64).reshape(-1, max(words, 1)).to(torch.int32)


def paged_tree(q, cache, table, segments, kv_heads, max_keys, max_len, mask=None, scale=None, keys_per_split=None,
               out=None):
    """Attention of every segment's appended rows over its history and themselves.

    q: BF16 [rows, q_heads, d] (d 64 or 128); ``cache`` the layer's pages, BF16 [blocks, 2, kv_heads,
    16, d] or a QuantizedCache, which hold the appended rows' keys and values too. ``segments`` int32
    [n, 5] and ``table`` as for ``paged_prefill``. Row i of a segment sees the whole history
    (positions below ``cached``) and the appended rows j whose bit j is set in its words of ``mask``
    (int32 [rows, words], bit j % 32 of word j / 32: ``tree_mask`` makes it from drafted trees); with
    ``mask=None`` the rows j <= i, as in a chain of drafts or a prompt chunk. A row that sees nothing
    gets zeros. Rows of ``out`` that belong to no segment are left as they were.

    ``max_keys`` bounds every segment's cached + len and ``max_len`` its len: a segment that goes
    past one of them (or past its table or the rows) gets zeros and records a status. A history is
    split every ``keys_per_split`` keys (a multiple of 16), and the splits are joined in order; by
    default the width depends on the sizes of the call, so a fixed width is what keeps a row's bits
    the same in other batches."""
    _heads(q, "q")
    rows, q_heads, d = q.shape
    quantized = isinstance(cache, QuantizedCache)
    if quantized:
        pages = cache.pages
        if cache.head_dim != d or pages.shape[2] != kv_heads:
            raise ValueError("the cache has other heads than q")
    else:
        pages = cache
        if pages.dtype != torch.bfloat16 or pages.dim() != 5 or pages.shape[1:] != (2, kv_heads, BLOCK, d) \
                or not pages.is_contiguous() or pages.data_ptr() % 16:
            raise ValueError("the cache must be contiguous BF16 [blocks, 2, kv_heads, 16, d], or a QuantizedCache")
    if d not in (64, 128) or kv_heads < 1 or q_heads < 1 or q_heads % kv_heads:
        raise ValueError("head_dim must be 64 or 128, with query heads a multiple of the key/value heads")
    n = segments.shape[0]
    _ints(segments, (n, 5), "segments")
    _ints(table, (table.numel(),), "table")
    if max_keys < 1 or max_len < 1 or max_keys > 1 << 30 or max_len > 1 << 24:
        raise ValueError("max_keys must be in [1, 2^30] and max_len in [1, 2^24]")
    if keys_per_split is not None and (keys_per_split < BLOCK or keys_per_split % BLOCK or keys_per_split > 1 << 30):
        raise ValueError("keys_per_split must be a positive multiple of 16")
    words = 0
    if mask is not None:
        words = mask.shape[1] if mask.dim() == 2 else 0
        _ints(mask, (rows, words), "mask")
        if words < 1 or words > 1 << 20:
            raise ValueError("mask must have a word for every 32 appended rows")
    if out is not None:
        _heads(out, "out")
        if out.shape != q.shape:
            raise ValueError("out must have the shape of q")
    with _Launch(q, pages, table, segments, mask, out) as at:
        if out is None:
            out = torch.empty(rows, q_heads, d, dtype=torch.bfloat16, device=q.device)
        if n == 0 or rows == 0:
            return out
        ops = native().ops
        if keys_per_split is None:
            keys_per_split = ops.tree_attention_split(n, q_heads, kv_heads, d, quantized, max_keys, max_len)
        splits = -(-max_keys // keys_per_split)
        po = pl = 0
        need = 0
        if splits > 1:
            need = rows * q_heads * splits
            work = torch.empty(need * (d + 2), dtype=torch.float32, device=q.device)
            po = work.data_ptr()
            pl = po + need * d * 4
        ops.tree_attention(
            q.data_ptr(), q.stride(0) if rows > 1 else q_heads * d, out.data_ptr(),
            out.stride(0) if rows > 1 else q_heads * d, rows, pages.data_ptr(), quantized, pages.shape[0],
            table.data_ptr(), table.numel(), segments.data_ptr(), n, q_heads, kv_heads, d,
            d ** -0.5 if scale is None else scale, 0 if mask is None else mask.data_ptr(), words, max_keys, max_len,
            keys_per_split, po, pl, need, at.status, at.stream)
    return out


def _token_lists(lists, rows: int, name: str):
    """(tokens, starts): row r's tokens are tokens[starts[r]:starts[r + 1]]."""
    if lists is None:
        return None, None
    tokens, starts = lists[0], lists[-1]
    _ints(tokens, (tokens.numel(),), name + " tokens")
    _ints(starts, (rows + 1,), name + " starts")
    if tokens.numel() > 1 << 30:
        raise ValueError(f"{name} holds more than 2^30 tokens")
    return tokens, starts


def _per_row(t, rows: int, name: str) -> None:
    if t is not None and (t.dtype != torch.float32 or t.shape != (rows,) or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous FP32 tensor of one value a row")


def process_logits(logits, prompt=None, output=None, repetition=None, frequency=None, presence=None, bias=None,
                   allowed=None, out=None):
    """Penalties, biases and a token mask on logits [rows, vocab] (FP32 or BF16, unit column stride),
    and each row's greedy token: (index int32 [rows], value FP32 [rows]), the first of equal maxima.

    ``prompt`` and ``output`` are (tokens, starts), int32: row r's tokens are
    ``tokens[starts[r]:starts[r + 1]]``; a token outside the vocabulary (padding) is left out. Of a
    token with logit x that occurs n times in the row's output, in this order and in FP32:

    - listed in prompt or output: x / repetition when x > 0, else x * repetition;
    - n > 0: x - frequency * n, then x - presence;
    - named by ``bias`` (tokens, values FP32, starts): x + value (of a token named twice, the last);
    - bit t % 32 of word t / 32 of the row of ``allowed`` (int32 [rows, words]) unset: -inf.

    ``repetition``, ``frequency`` and ``presence`` are FP32 [rows]. ``out`` (the logits' shape and
    type; may be ``logits``) receives the adjusted logits. A logit that is NaN is never chosen; a row
    whose every token is -inf (or NaN) gives index -1 and value -inf."""
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("logits must be FP32 or BF16 [rows, vocab]")
    rows, vocab = logits.shape
    if vocab < 1 or vocab > 1 << 30 or rows > 1 << 24:
        raise ValueError("logits must have 1 to 2^30 columns and at most 2^24 rows")
    if (logits.stride(1) != 1 and vocab != 1) or (rows > 1 and logits.stride(0) < vocab):
        raise ValueError("logits must have unit column stride")
    prompt_t, prompt_s = _token_lists(prompt, rows, "prompt")
    output_t, output_s = _token_lists(output, rows, "output")
    bias_t, bias_s = _token_lists(bias, rows, "bias")
    values = None
    if bias is not None:
        values = bias[1]
        if len(bias) != 3 or values.dtype != torch.float32 or values.shape != bias_t.shape or not values.is_contiguous():
            raise ValueError("bias must be (tokens, FP32 values, starts)")
    _per_row(repetition, rows, "repetition")
    _per_row(frequency, rows, "frequency")
    _per_row(presence, rows, "presence")
    if allowed is not None and (allowed.dtype != torch.int32 or allowed.dim() != 2 or allowed.shape[0] != rows
                                or allowed.shape[1] < (vocab + 31) // 32 or (allowed.stride(1) != 1 and allowed.shape[1] != 1)):
        raise ValueError("allowed must be int32 [rows, at least vocab / 32] with unit column stride")
    if out is not None and (out.dtype != logits.dtype or out.shape != logits.shape or (out.stride(1) != 1 and vocab != 1)
                            or (rows > 1 and out.stride(0) < vocab)):
        raise ValueError("out must have the logits' shape and type, and unit column stride")
    with _Launch(logits, prompt_t, prompt_s, output_t, output_s, bias_t, bias_s, values, repetition, frequency, presence,
                 allowed, out) as at:
        index = torch.empty(rows, dtype=torch.int32, device=logits.device)
        value = torch.empty(rows, dtype=torch.float32, device=logits.device)
        if rows == 0:
            return index, value
        ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        size = lambda t: 0 if t is None else t.numel()  # noqa: E731
        ops = native().ops
        slices = ops.logits_slices(vocab)
        partial = torch.empty(rows * slices, 2, dtype=torch.float32, device=logits.device) if slices > 1 else None
        ops.process_logits(
            logits.data_ptr(), logits.stride(0), ptr(out), 0 if out is None else out.stride(0),
            logits.dtype == torch.bfloat16, rows, vocab, ptr(prompt_t), ptr(prompt_s), size(prompt_t), ptr(output_t),
            ptr(output_s), size(output_t), ptr(bias_t), ptr(bias_s), size(bias_t), ptr(values), ptr(repetition),
            ptr(frequency), ptr(presence), ptr(allowed), 0 if allowed is None else allowed.stride(0), index.data_ptr(),
            value.data_ptr(), ptr(partial), rows * slices, at.status, at.stream)
    return index, value
