"""Decode-step operators on the host: drafted-tree masks, the quantized cache's views, refusals."""

import pytest
import torch

from furiosa_opt_models_b200 import ops

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def test_tree_mask_holds_ancestors_and_the_node_itself():
    # 0 - 1 - 3, 0 - 2, and 4 a second root; a chain of 40 in the second segment (two words).
    mask = ops.tree_mask([[-1, 0, 0, 1, -1], [i - 1 for i in range(40)]])
    assert mask.shape == (45, 2) and mask.dtype == I32
    bits = [[j for j in range(64) if mask[r, j // 32].item() >> (j % 32) & 1] for r in range(45)]
    assert bits[:5] == [[0], [0, 1], [0, 2], [0, 1, 3], [4]]
    assert bits[5:] == [list(range(i + 1)) for i in range(40)]
    assert ops.tree_mask([]).shape == (0, 1)
    assert ops.tree_mask([[], [-1]]).tolist() == [[1]]


@pytest.mark.parametrize("parents", [[[0]], [[-1, 1]], [[-1, 2, 0]], [[-2]]])
def test_tree_mask_refuses_parents_that_do_not_come_before(parents):
    with pytest.raises(ValueError, match="parents come before"):
        ops.tree_mask(parents)


def test_quantized_cache_views():
    c = ops.QuantizedCache.empty(3, 2, 64, device="cpu")
    assert c.pages.shape == (3, 2, 2, 16 * 64 + 64)
    assert c.codes.shape == (3, 2, 2, 16, 64) and c.scales.shape == (3, 2, 2, 16)
    assert torch.count_nonzero(c.dequantize()) == 0
    c.codes[1, 0, 1, 5] = torch.full((64,), 1.5).to(torch.float8_e4m3fn).view(torch.uint8)
    c.scales[1, 0, 1, 5] = 0.25
    v = c.dequantize()
    assert torch.equal(v[1, 0, 1, 5], torch.full((64,), 0.375)) and torch.count_nonzero(v) == 64


@pytest.mark.parametrize("pages,d", [
    (torch.zeros(2, 2, 1, 16 * 64 + 64), 64),
    (torch.zeros(2, 2, 1, 16 * 64, dtype=torch.uint8), 64),
    (torch.zeros(2, 1, 1, 16 * 64 + 64, dtype=torch.uint8), 64),
    (torch.zeros(2, 2, 1, 16 * 96 + 64, dtype=torch.uint8), 96),
    (torch.zeros(2, 2, 2, 16 * 64 + 64, dtype=torch.uint8)[:, :, :1], 64),
    (torch.zeros(2 * 2 * (16 * 64 + 64) + 1, dtype=torch.uint8)[1:].view(2, 2, 1, 16 * 64 + 64), 64),
])
def test_quantized_cache_refuses_other_pages(pages, d):
    with pytest.raises(ValueError):
        ops.QuantizedCache(pages, d)


def _tree_args(d=64, q_heads=4, kv_heads=2, rows=3):
    return dict(q=torch.zeros(rows, q_heads, d, dtype=BF16), cache=torch.zeros(4, 2, kv_heads, 16, d, dtype=BF16),
                table=torch.zeros(4, dtype=I32), segments=torch.zeros(1, 5, dtype=I32), kv_heads=kv_heads, max_keys=64,
                max_len=rows)


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(3, 4, 64)), "q must be BF16"),
    (dict(q=torch.zeros(3, 256, dtype=BF16)), "q must be BF16"),
    (dict(q=torch.zeros(3, 64, 4, dtype=BF16).transpose(1, 2)), "heads packed"),
    (dict(q=torch.zeros(3, 4 * 64 + 4, dtype=BF16)[:, :256].view(3, 4, 64)), "multiple of 8"),
    (dict(q=torch.zeros(3 * 256 + 1, dtype=BF16)[1:].view(3, 4, 64)), "16-byte"),
    (dict(q=torch.zeros(3, 4, 96, dtype=BF16), cache=torch.zeros(4, 2, 2, 16, 96, dtype=BF16)), "head_dim"),
    (dict(q=torch.zeros(3, 5, 64, dtype=BF16)), "multiple of the key/value heads"),
    (dict(cache=torch.zeros(4, 2, 2, 16, 64)), "cache must be"),
    (dict(cache=torch.zeros(4, 2, 3, 16, 64, dtype=BF16)), "cache must be"),
    (dict(cache=ops.QuantizedCache.empty(4, 3, 64, device="cpu")), "other heads"),
    (dict(segments=torch.zeros(1, 4, dtype=I32)), "segments"),
    (dict(segments=torch.zeros(1, 5, dtype=torch.int64)), "segments"),
    (dict(table=torch.zeros(4, dtype=torch.int64)), "table"),
    (dict(max_keys=0), "max_keys"),
    (dict(max_len=0), "max_len"),
    (dict(keys_per_split=24), "multiple of 16"),
    (dict(keys_per_split=0), "multiple of 16"),
    (dict(mask=torch.zeros(2, 1, dtype=I32)), "mask"),
    (dict(mask=torch.zeros(3, 0, dtype=I32)), "mask"),
    (dict(mask=torch.zeros(3, dtype=I32)), "mask"),
    (dict(out=torch.zeros(3, 4, 128, dtype=BF16)), "out must have"),
    (dict(), "CUDA"),
])
def test_paged_tree_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        ops.paged_tree(**{**_tree_args(), **change})


def test_paged_decode_and_prefill_over_a_quantized_cache_refuse_bf16_options():
    cache = ops.QuantizedCache.empty(4, 2, 64, device="cpu")
    q, table, segs = torch.zeros(1, 4, 64, dtype=BF16), torch.zeros(4, dtype=I32), torch.zeros(1, 5, dtype=I32)
    for option in (dict(warps=2), dict(stages=2), dict(counters=torch.zeros(2, dtype=I32))):
        with pytest.raises(ValueError, match="BF16 pages"):
            ops.paged_decode(q, cache, table, segs, 2, 16, **option)
    with pytest.raises(ValueError, match="paged_tree"):
        ops.paged_prefill(q, cache, table, segs, 2, torch.zeros(1, 2, dtype=I32))


def _store_args(d=64, rows=3):
    return dict(qkv=torch.zeros(rows, 8 * d, dtype=BF16), q_heads=4, kv_heads=2, head_dim=d, q_norm=None, k_norm=None,
                eps=1e-6, positions=torch.zeros(rows, dtype=I32), inv_freq=torch.zeros(d // 2), attention_factor=1.0,
                cache=ops.QuantizedCache.empty(4, 2, d, device="cpu"), slots=torch.zeros(rows, dtype=I32))


@pytest.mark.parametrize("change,match", [
    (dict(qkv=torch.zeros(3, 512)), "qkv must be BF16"),
    (dict(qkv=torch.zeros(3, 511, dtype=BF16)), "qkv must be BF16"),
    (dict(qkv=torch.zeros(512, 3, dtype=BF16).T), "unit column stride"),
    (dict(qkv=torch.zeros(3, 516, dtype=BF16)[:, :512]), "aligned rows"),
    (dict(q_norm=torch.zeros(64, dtype=BF16)), "come together"),
    (dict(q_norm=torch.zeros(64), k_norm=torch.zeros(64)), "norm weights"),
    (dict(positions=torch.zeros(3, dtype=torch.int64)), "positions"),
    (dict(slots=torch.zeros(2, dtype=I32)), "slots"),
    (dict(inv_freq=torch.zeros(16)), "inv_freq"),
    (dict(rotary_dim=24), "rotary_dim"),
    (dict(rotary_dim=0), "rotary_dim"),
    (dict(rotary_dim=80), "rotary_dim"),
    (dict(cache=ops.QuantizedCache.empty(4, 3, 64, device="cpu")), "other heads"),
    (dict(cache=torch.zeros(4, 2, 2, 16, 64), interleaved=True), "cache must be"),
    (dict(head_dim=96), "qkv must be BF16"),
    (dict(), "CUDA"),
])
def test_store_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        ops.qk_norm_rope_cache(**{**_store_args(), **change})


@pytest.mark.parametrize("change,match", [
    (dict(logits=torch.zeros(2, 10, dtype=torch.float16)), "FP32 or BF16"),
    (dict(logits=torch.zeros(10)), "FP32 or BF16"),
    (dict(logits=torch.zeros(2, 0)), "columns"),
    (dict(logits=torch.zeros(10, 2).T), "unit column stride"),
    (dict(logits=torch.zeros(1, 10).expand(2, 10)), "unit column stride"),
    (dict(prompt=(torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=I32))), "prompt tokens"),
    (dict(output=(torch.zeros(3, dtype=I32), torch.zeros(2, dtype=I32))), "output starts"),
    (dict(bias=(torch.zeros(3, dtype=I32), torch.zeros(3, dtype=I32))), "bias must be"),
    (dict(bias=(torch.zeros(3, dtype=I32), torch.zeros(2), torch.zeros(3, dtype=I32))), "bias must be"),
    (dict(repetition=torch.zeros(3)), "repetition"),
    (dict(frequency=torch.zeros(2, dtype=BF16)), "frequency"),
    (dict(presence=torch.zeros(2, 1)), "presence"),
    (dict(allowed=torch.zeros(2, 0, dtype=I32)), "allowed"),
    (dict(allowed=torch.zeros(1, 1, dtype=I32)), "allowed"),
    (dict(out=torch.zeros(2, 10, dtype=BF16)), "out must have"),
    (dict(out=torch.zeros(1, 10).expand(2, 10)), "out must have"),
    (dict(), "CUDA"),
])
def test_process_logits_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        ops.process_logits(**{**dict(logits=torch.zeros(2, 10)), **change})


def _changed_cache(change):
    """A QuantizedCache of 4 blocks, 2 heads of 64, changed after its checks."""
    c = ops.QuantizedCache.empty(4, 2, 64, device="cpu")
    for name, value in change.items():
        setattr(c, name, value(c.pages) if callable(value) else value)
    return c


@pytest.mark.parametrize("change", [
    dict(head_dim=128),
    dict(head_dim=32),
    dict(pages=lambda p: p[..., :16 * 64]),                                 # without scales, and with holes
    dict(pages=lambda p: torch.zeros(4, 2, 2, 16 * 64, dtype=torch.uint8)),
    dict(pages=lambda p: torch.zeros(4, 1, 2, 16 * 64 + 64, dtype=torch.uint8)),
    dict(pages=lambda p: torch.zeros(4, 2, 4, 16 * 64 + 64, dtype=torch.uint8)[:, :, ::2]),
    dict(pages=lambda p: torch.zeros(4, 2, 2, 16 * 64 + 64, dtype=BF16)),
    dict(pages=lambda p: p[0]),
    dict(pages=lambda p: torch.zeros(4 * 2 * 2 * 1088 + 8, dtype=torch.uint8)[8:].view(4, 2, 2, 1088)),
    dict(pages=lambda p: None),
])
def test_a_quantized_cache_changed_after_its_checks_is_refused(change):
    c = _changed_cache(change)
    for use in (lambda: c.codes, lambda: c.scales,
                lambda: ops.paged_tree(**{**_tree_args(), "cache": c}),
                lambda: ops.paged_tree(**{**_tree_args(d=128), "cache": c}),
                lambda: ops.qk_norm_rope_cache(**{**_store_args(), "cache": c})):
        with pytest.raises((ValueError, TypeError), match="page|torch tensor"):
            use()


def test_a_quantized_cache_of_other_heads_than_the_rows_is_refused():
    c = ops.QuantizedCache.empty(4, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="other heads"):
        ops.paged_tree(**{**_tree_args(d=128), "cache": c})
    with pytest.raises(ValueError, match="other heads"):
        ops.qk_norm_rope_cache(**{**_store_args(d=128), "cache": c})


def test_first_calls_at_once_share_one_scratch(monkeypatch):
    """Kernels keep the address of a device's status word: no second one takes its place."""
    import importlib
    import threading
    import time

    native = importlib.import_module("furiosa_opt_models_b200.ops.native")
    made = []

    class Slow:
        def __init__(self, device):
            time.sleep(0.05)  # as an allocation may, with the interpreter released
            self.device = device
            made.append(self)

    monkeypatch.setattr(native, "Scratch", Slow)
    monkeypatch.setattr(native, "_scratch", {})
    start, got = threading.Barrier(8), []

    def call(i):
        start.wait()
        got.append(native.scratch(torch.device("cuda", i % 2)))

    threads = [threading.Thread(target=call, args=(i,)) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 2 and len(got) == 8
    assert all(s is native.scratch(s.device) for s in got)


def _parts(keys, width, even):
    from furiosa_opt_models_b200.ops.native import native

    return native().ops.history_parts(keys, width, even)


def test_parts_of_a_history_are_equal_in_whole_tiles():
    # Eight parts of 1024 keys, not seven of 1152 and one of 128.
    assert _parts(8192, 1152, True) == (1024, 8)
    assert _parts(4096, 1152, True) == (1024, 4) and _parts(768, 512, True) == (384, 2)
    for keys in [*range(1, 3000), 8191, 8192, 8193, 131072, (1 << 22) - 1, 1 << 22, (1 << 22) + 129, (1 << 30) - 5, 1 << 30]:
        for width in (128, 256, 384, 1152, 4096, 1 << 20):
            each, count = _parts(keys, width, True)
            least = -(-keys // width)  # as few parts as the width allows, or fewer where whole tiles do it
            assert each <= width and (each % 128 == 0 or count == 1) and 1 <= count <= least
            assert (count - 1) * each < keys <= count * each
            if count > 1:
                assert (each - 128) * least < keys  # one tile less would not do
    for keys, width in ((1, 16), (17, 16), (1000, 48), (129, 128), (1 << 30, 1 << 30)):
        assert _parts(keys, width, False) == (width, -(-keys // width))
        assert _parts(keys, 48, True) == (48, -(-keys // 48))  # no whole tiles: parts as given


@pytest.mark.parametrize("rows,of,out,fine", [
    (3, (0, 4 * 64), (0, 4 * 64), True),                # q itself
    (3, (0, 4 * 64), (3 * 4 * 64, 4 * 64), True),       # behind it
    (3, (0, 8 * 64), (4 * 64, 8 * 64), True),           # beside it, in the same rows
    (3, (4 * 64, 8 * 64), (0, 8 * 64), True),
    (1, (0, 8 * 64), (0, 4 * 64), True),                # one row: its stride says nothing
    (3, (0, 4 * 64), (4 * 64, 4 * 64), False),          # a row further
    (3, (0, 8 * 64), (2 * 64, 8 * 64), False),          # two heads further
    (3, (0, 8 * 64), (6 * 64, 8 * 64), False),          # into the next row
    (3, (0, 4 * 64), (0, 8 * 64), False),               # other strides
    (1, (0, 4 * 64), (8, 4 * 64), False),
])
def test_out_that_overlaps_q_is_refused(rows, of, out, fine):
    mem = torch.zeros(4096, dtype=BF16)
    view = lambda v: mem.as_strided((rows, 4, 64), (v[1], 64, 1), v[0])  # noqa: E731
    with pytest.raises(ValueError, match="CUDA" if fine else "overlap"):
        ops.paged_tree(**{**_tree_args(rows=rows), "q": view(of), "out": view(out)})


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,of,out,fine", [
    (3, (0, 10), (0, 10), True),
    (3, (0, 10), (30, 10), True),
    (3, (0, 25), (10, 25), True),
    (3, (15, 25), (0, 25), True),
    (1, (0, 25), (0, 10), True),
    (3, (0, 10), (10, 10), False),
    (3, (0, 10), (1, 10), False),
    (3, (1, 10), (0, 10), False),
    (3, (0, 25), (20, 25), False),
    (3, (0, 20), (0, 10), False),
])
def test_out_that_overlaps_the_logits_is_refused(rows, of, out, fine, dtype):
    mem = torch.zeros(200, dtype=dtype)
    view = lambda v: mem.as_strided((rows, 10), (v[1], 1), v[0])  # noqa: E731
    with pytest.raises(ValueError, match="CUDA" if fine else "overlap"):
        ops.process_logits(view(of), out=view(out))


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e39])
def test_a_scale_that_is_not_finite_is_refused(scale):
    with pytest.raises(ValueError, match="scale must be finite"):
        ops.paged_tree(**_tree_args(), scale=scale)
