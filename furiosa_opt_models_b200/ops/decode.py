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

from .native import _scratch, calls, scratch

BLOCK = 16  # positions of a cache block
_SCALE_BYTES = 64  # 16 FP32 scales behind a page's codes


def _status(first: torch.Tensor) -> int:
    """Address of the status word of the first operand's device (0 off the GPU, where the call is
    refused after its other checks)."""
    index = first.get_device()
    if index < 0:
        return 0
    s = _scratch.get(index)
    if s is None:
        with torch.cuda.device(index):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the device's first call cannot be captured: its status word is laid out then")
            s = scratch(first.device)
    return s.status_ptr


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
        return calls().codes(self.pages, self.head_dim)

    @property
    def scales(self) -> torch.Tensor:
        """The scales as an FP32 view [blocks, 2, kv_heads, 16]."""
        return calls().scales(self.pages, self.head_dim)

    def dequantize(self) -> torch.Tensor:
        """The values the cache stands for, FP32 [blocks, 2, kv_heads, 16, head_dim]."""
        return self.codes.view(torch.float8_e4m3fn).float() * self.scales.unsqueeze(-1)


def store_rows(qkv, q_heads, kv_heads, head_dim, q_norm, k_norm, eps, positions, inv_freq, attention_factor,
               cache, slots, rotary_dim=None, interleaved=False):
    """``kernels.qk_norm_rope_cache`` over a QuantizedCache, or with a partial or interleaved rotation."""
    quantized = isinstance(cache, QuantizedCache)
    return calls().kv_store(qkv, q_heads, kv_heads, head_dim, q_norm, k_norm, eps, positions, inv_freq, attention_factor,
                            cache.pages if quantized else cache, cache.head_dim if quantized else 0, slots,
                            head_dim if rotary_dim is None else rotary_dim, interleaved, _status(qkv))


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
    gets zeros; a row of q with an element that is not finite gets NaN from any key it sees. ``out`` is
    q itself or memory apart from it; its rows that belong to no segment are left as they were.

    ``max_keys`` bounds every segment's cached + len and ``max_len`` its len: a segment that goes
    past one of them (or past its table or the rows) gets zeros and records a status. A history is
    split into parts of at most ``keys_per_split`` keys (a multiple of 16), which are joined in order;
    by default the width depends on the sizes of the call, so a fixed width is what keeps a row's bits
    the same in other batches (of the same ``max_len``, which picks the kernel)."""
    quantized = isinstance(cache, QuantizedCache)
    return calls().tree_attention(q, cache.pages if quantized else cache, cache.head_dim if quantized else 0, table,
                                  segments, kv_heads, max_keys, max_len, mask, scale, keys_per_split, out, _status(q))


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
    type; ``logits`` itself, or memory apart from them) receives the adjusted logits. A logit that is
    NaN is never chosen; a row whose every token is -inf (or NaN) gives index -1 and value -inf."""
    return calls().process_logits(logits, prompt, output, repetition, frequency, presence, bias, allowed, out,
                                  _status(logits))
