"""The decode-step operators against plain 64-bit forms: the quantizing store, attention of decode
rows, chunks and drafted trees over BF16 and quantized pages, constrained logits, and one
speculative step of all of them."""

import random

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32, I32, F64 = torch.bfloat16, torch.float32, torch.int32, torch.float64
E4M3 = torch.float8_e4m3fn
DEV = "cuda"


def _ops():
    from furiosa_opt_models_b200 import ops

    return ops


def _half(dtype):
    """Largest relative error of one rounding."""
    return torch.finfo(dtype).eps / 2


def _check():
    torch.cuda.synchronize()
    _ops().scratch(torch.device("cuda", 0)).check()


def _status():
    s = _ops().scratch(torch.device("cuda", 0)).status
    torch.cuda.synchronize()
    code = int(s[0].item())
    s.zero_()
    return code


# ------------------------------------------------------------------------------- quantizing store


def _front64(qkv, hq, hk, d, qn, kn, eps, pos, inv_freq, factor, rot, interleaved):
    x = qkv.double().view(-1, hq + 2 * hk, d).cpu()
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    out = []
    for h, w in ((q, qn), (k, kn)):
        if w is not None:
            h = h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * w.double().cpu()
        h = h.clone()
        a = (pos.double().cpu()[:, None] * inv_freq.double().cpu())[:, None]
        i = torch.arange(rot // 2) * 2 if interleaved else torch.arange(rot // 2)
        j = i + 1 if interleaved else i + rot // 2
        xi, xj = h[..., i].clone(), h[..., j].clone()
        h[..., i] = (xi * a.cos() - xj * a.sin()) * factor
        h[..., j] = (xj * a.cos() + xi * a.sin()) * factor
        out.append(h)
    return out[0], out[1], v


@pytest.mark.parametrize("rows,hq,hk,d,rot,interleaved,norm,quantized", [
    (1, 16, 8, 128, 128, False, True, True),
    (7, 4, 2, 64, 64, False, True, True),
    (33, 14, 2, 64, 32, False, False, True),
    (5, 6, 3, 128, 96, False, True, True),   # a rotation partner 6 lanes away
    (9, 8, 1, 128, 16, True, True, True),
    (200, 5, 5, 64, 64, True, False, True),
    (3, 0, 2, 128, 128, False, False, True),  # keys and values alone
    (700, 32, 8, 128, 128, True, True, True),
    (6, 4, 2, 64, 32, True, True, False),
    (6, 12, 4, 128, 64, False, False, False),
])
def test_store(rows, hq, hk, d, rot, interleaved, norm, quantized):
    ops = _ops()
    torch.manual_seed(rows)
    wide = torch.randn(rows, (hq + 2 * hk) * d + 8, device=DEV).mul_(3).to(BF16)
    qkv = wide[:, 8:] if rows % 2 else wide[:, :-8]  # rows of a wider tensor
    qkv[0, -d:] = 0  # a value row of zeros
    qn, kn = ((1 + 0.2 * torch.randn(d, device=DEV)).to(BF16) for _ in range(2)) if norm else (None, None)
    pos = torch.randint(0, 131072, (rows,), device=DEV, dtype=I32)
    inv_freq = 5e5 ** (-torch.arange(0, rot, 2, device=DEV, dtype=F32) / rot)
    blocks = rows // 16 + 3
    slots = torch.randperm(blocks * 16, device=DEV)[:rows].to(I32)
    if rows > 4:
        slots[2] = -1
    if quantized:
        cache = ops.QuantizedCache(torch.randint(0, 255, (blocks, 2, hk, 16 * d + 64), device=DEV).to(torch.uint8), d)
        before = cache.pages.clone()
    else:
        cache = torch.randn(blocks, 2, hk, 16, d, device=DEV).to(BF16)
        before = cache.clone()
    q = ops.qk_norm_rope_cache(qkv, hq, hk, d, qn, kn, 1e-5, pos, inv_freq, 0.9, cache, slots, rotary_dim=rot,
                               interleaved=interleaved)
    _check()
    rq, rk, rv = _front64(qkv, hq, hk, d, qn, kn, 1e-5, pos, inv_freq, 0.9, rot, interleaved)
    # FP32 steps before the rounding: the norm's sum of d squares, its inverse root (2 ulp) and two
    # products, an angle reduced to within pi (2^-24 * pi), sine and cosine (2 ulp), two products and
    # a sum: under (d + 32) * 2^-24 of the pair's larger element, itself under the row's largest.
    def slack(y):
        return (d + 32) * 2.0 ** -24 * 2 * y.abs().amax(-1, keepdim=True)

    assert ((q.double().cpu() - rq).abs() <= _half(BF16) * rq.abs() + slack(rq)).all()
    touched = torch.zeros(blocks, 16, dtype=torch.bool)
    for r, s in enumerate(slots.tolist()):
        if s < 0:
            continue
        b, o = divmod(s, 16)
        touched[b, o] = True
        for which, y in ((0, rk[r]), (1, rv[r])):
            if quantized:
                scale = cache.scales[b, which, :, o].double().cpu()
                want = y.abs().amax(-1).clamp_min(1e-10) / 448
                assert ((scale - want).abs() <= want * (2 * (d + 32) * 2.0 ** -24 + 2.0 ** -22)).all()
                got = cache.dequantize()[b, which, :, o].double().cpu()
                # Half a step of the code: relative, or of the subnormal spacing 2^-9.
                step = torch.maximum(_half(E4M3) * y.abs(), 2.0 ** -10 * scale[:, None])
                assert ((got - y).abs() <= step * (1 + 2.0 ** -3) + slack(y)).all()
            else:
                got = cache[b, which, :, o].double().cpu()
                assert ((got - y).abs() <= _half(BF16) * y.abs() + slack(y)).all()
    # Every other slot is as it was.
    if quantized:
        old = ops.QuantizedCache(before, d)
        same = (cache.codes == old.codes).all(-1) & (cache.pages[..., 16 * d:].unflatten(-1, (16, 4))
                                                     == before[..., 16 * d:].unflatten(-1, (16, 4))).all(-1)
    else:
        same = (cache == before).all(-1)
    assert (same.permute(0, 3, 1, 2).cpu() | touched[:, :, None, None]).all()


def test_store_values_that_are_not_finite_and_bad_slots():
    ops = _ops()
    torch.manual_seed(1)
    qkv = torch.randn(3, 4 * 64, device=DEV).to(BF16)
    qkv[0, 2 * 64 + 3] = float("nan")  # the key head
    qkv[1, 3 * 64 + 5] = float("inf")  # the value head
    qkv[1, 3 * 64 + 6] = -float("inf")
    cache = ops.QuantizedCache.empty(2, 1, 64)
    slots = torch.tensor([3, 17, 32], device=DEV, dtype=I32)  # the last one lies past the cache
    zero = torch.zeros(3, device=DEV, dtype=I32)
    freq = torch.ones(8, device=DEV)
    ops.qk_norm_rope_cache(qkv, 2, 1, 64, None, None, 1e-6, zero, freq, 1.0, cache, slots, rotary_dim=16)
    assert _status() == 8
    v = cache.dequantize()
    # The rotation makes NaN of both elements of the NaN's pair, (3, 3 + 16 / 2).
    assert v[0, 0, 0, 3].isnan().nonzero().flatten().tolist() == [3, 11]
    assert v[1, 1, 0, 1].isnan().sum() == 2 and v[1, 1, 0, 1, 5:7].isnan().all()
    # The others keep a scale of the finite ones.
    y = qkv[1, 3 * 64:].double()
    y = torch.where(y.isfinite(), y, 0)
    keep = torch.arange(64, device=DEV)
    keep = (keep != 5) & (keep != 6)
    assert ((v[1, 1, 0, 1].double() - y).abs() <= 2.0 ** -4 * y.abs() + y.abs().max() * 2.0 ** -18)[keep].all()
    assert torch.count_nonzero(v.nan_to_num(1.0)[:, :, 0].amax(-1)) == 4  # two rows' keys and values, nothing else


# ------------------------------------------------------------------------------------- attention


def _paged(lens, cached, hk, d, quantized, gen, spare=3):
    """(cache, table, segments, values in 64 bits) with scattered blocks; the slots past each
    sequence's end and the spare blocks hold NaN."""
    ops = _ops()
    segs, row, start = [], 0, 0
    for n, c in zip(lens, cached):
        nb = (n + c + 15) // 16
        segs.append((row, n, c, start, nb))
        row, start = row + n, start + nb
    blocks = start + spare
    x = torch.randn(blocks, 2, hk, 16, d, generator=gen) * 0.7
    x[:, 1] *= torch.rand(blocks, hk, 16, 1, generator=gen) * 3 + 0.01  # values of unequal sizes
    table = torch.randperm(blocks, generator=gen)[:start]
    if quantized:
        pages = torch.zeros(blocks, 2, hk, 16 * d + 64, dtype=torch.uint8)
        scale = x.abs().amax(-1).clamp_min(1e-10) / 448
        codes = (x / scale[..., None]).clamp(-448, 448).to(E4M3)
        pages[..., :16 * d] = codes.view(torch.uint8).flatten(3)
        pages[..., 16 * d:] = scale.view(torch.uint8)
        values = codes.double() * scale.double()[..., None]
    else:
        pages = x.to(BF16)
        values = pages.double()
    used = torch.zeros(blocks, 16, dtype=torch.bool)
    for _, n, c, s, nb in segs:
        for b in range(nb):
            used[table[s + b], :max(0, min(16, n + c - 16 * b))] = True
    for b, o in (~used).nonzero().tolist():
        if quantized:
            pages[b, :, :, o * d:(o + 1) * d] = 0x7F
            pages[b, :, :, 16 * d + 4 * o:16 * d + 4 * o + 4] = torch.tensor(
                [float("nan")]).view(torch.uint8)
        else:
            pages[b, :, :, o] = float("nan")
    cache = ops.QuantizedCache(pages.to(DEV), d) if quantized else pages.to(DEV)
    return (cache, table.to(I32).to(DEV), torch.tensor(segs, dtype=I32).reshape(-1, 5).to(DEV), values, table, segs)


def _attend64(q, values, table, segs, scale, mask=None, causal=True):
    """(outputs, tolerances) of the formula in 64 bits. ``mask``: per segment, bool [len, len]."""
    rows, hq, d = q.shape
    hk = values.shape[2]
    out, weight, err, part = (torch.zeros(rows, hq, d, dtype=F64) for _ in range(4))
    for i, (row, n, c, start, nb) in enumerate(segs):
        if n == 0:
            continue
        pages = values[table[start:start + nb]]
        k, v = (pages[:, w].permute(0, 2, 1, 3).reshape(-1, hk, d)[:n + c] for w in (0, 1))
        see = torch.ones(n, n + c, dtype=torch.bool)
        see[:, c:] = torch.tril(torch.ones(n, n)).bool() if mask is None else mask[i]
        for h in range(hq):
            kh, vh = k[:, h * hk // hq], v[:, h * hk // hq]
            qh = q[row:row + n, h].double()
            s = (qh @ kh.T * scale).masked_fill(~see, -torch.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0) * see
            seen = torch.where(see.any(0)[:, None], vh, 0.0)
            p_v = torch.where(p[..., None] > 0, p[..., None] * seen, 0.0)
            out[row:row + n, h] = p_v.sum(1)
            weight[row:row + n, h] = p_v.abs().sum(1)
            mags = kh.abs().nan_to_num(0.0)
            err[row:row + n, h] = ((qh.abs() @ mags.T) * scale).masked_fill(~see, 0).amax(-1, keepdim=True)
            most = qh.abs().amax(-1, keepdim=True) * mags.sum(-1) * scale
            part[row:row + n, h] = most.masked_fill(~see, 0).amax(-1, keepdim=True)
    return out, weight, (err, part)


def _tolerance(ref, weight, err, d, quantized):
    """One rounding of the output, one of each weight (FP16 over codes, BF16 over BF16), and the
    scores' FP32 sums of d products (and two scalings), each off by 2^-24 of the sum of magnitudes;
    a weight and its sum feel that twice. ex2 and lg2 add 2^-21 each. Over codes q may enter as two
    E4M3 parts of a row scaled to [128, 256): BF16's 8 bits are two parts of 4, so only bits below
    E4M3's smallest step 2^-9 are rounded, by 2^-10 at most, which is 2^-17 of the row's largest."""
    err, part = err
    return _half(BF16) * ref.abs() + weight * (
        _half(torch.float16 if quantized else BF16) + 2 * (d + 4) * 2.0 ** -24 * err + 2.0 ** -20
        + (2 * 2.0 ** -17 * part if quantized else 0))


def _random_masks(lens, gen, empty=False):
    """Per segment bool [len, len]; random bits (not a tree), some rows empty."""
    ms = []
    for n in lens:
        m = torch.rand(n, n, generator=gen) < 0.5
        if empty and n:
            m[0] = False
        ms.append(m)
    return ms


def _pack(ms, extra=0):
    words = max([1] + [(m.shape[0] + 31) // 32 for m in ms]) + extra
    rows = []
    for m in ms:
        for r in m.tolist():
            b = sum(1 << j for j, x in enumerate(r) if x)
            rows.append([(b >> 32 * w) & 0xFFFFFFFF for w in range(words)])
    return torch.tensor(rows, dtype=torch.int64).to(I32).to(DEV)


HEADS = [(16, 8, 128), (32, 8, 128), (8, 8, 64), (14, 2, 64), (12, 1, 128), (64, 2, 64)]


@pytest.mark.parametrize("split", [None, 16, 64, 4096])
@pytest.mark.parametrize("hq,hk,d", HEADS)
def test_decode_over_quantized_pages(hq, hk, d, split):
    ops = _ops()
    gen = torch.Generator().manual_seed(hq * d)
    cached = [0, 1, 14, 15, 16, 100, 511, 1000, 2047]
    cache, table, segs, values, tab, sl = _paged([1] * len(cached), cached, hk, d, True, gen)
    q = (torch.randn(len(cached), hq, d, generator=gen) * 1.5).to(BF16)
    out = ops.paged_decode(q.to(DEV), cache, table, segs, hk, 2048, keys_per_split=split)
    _check()
    ref, weight, err = _attend64(q, values, tab, sl, d ** -0.5)
    assert ((out.double().cpu() - ref).abs() <= _tolerance(ref, weight, err, d, True)).all()


LENS = [([1, 2, 5, 16, 33, 64, 7], [0, 1, 15, 16, 100, 700, 257]), ([40, 130, 1], [0, 300, 31]), ([300], [5]), ([3], [0])]


@pytest.mark.parametrize("quantized", [True, False], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("split", [None, 32, 2048])
@pytest.mark.parametrize("hq,hk,d", HEADS)
def test_tree_masks(hq, hk, d, split, quantized):
    ops = _ops()
    for case, (lens, cached) in enumerate(LENS):
        gen = torch.Generator().manual_seed(hq + d + case)
        cache, table, segs, values, tab, sl = _paged(lens, cached, hk, d, quantized, gen)
        q = (torch.randn(sum(lens), hq, d, generator=gen) * 1.5).to(BF16)
        ms = _random_masks(lens, gen, empty=True)
        bound = max(n + c for n, c in zip(lens, cached))
        out = ops.paged_tree(q.to(DEV), cache, table, segs, hk, bound + 9 * case, max(lens) + case, mask=_pack(ms, case),
                             keys_per_split=split)
        _check()
        ref, weight, err = _attend64(q, values, tab, sl, d ** -0.5, mask=ms)
        assert ((out.double().cpu() - ref).abs() <= _tolerance(ref, weight, err, d, quantized)).all()
        if cached[0] == 0 and case != 2:
            assert torch.count_nonzero(out[0]) == 0  # a first token that sees nothing


@pytest.mark.parametrize("quantized", [True, False], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("hq,hk,d", HEADS)
def test_chunks_are_causal_without_a_mask(hq, hk, d, quantized):
    ops = _ops()
    gen = torch.Generator().manual_seed(5)
    lens, cached = [17, 1, 129, 40], [0, 64, 250, 1]
    cache, table, segs, values, tab, sl = _paged(lens, cached, hk, d, quantized, gen)
    wide = (torch.randn(sum(lens), hq + 1, d, generator=gen)).to(BF16)
    q = wide[:, :hq]  # rows of a wider tensor
    held = torch.full((sum(lens), hq + 2, d), 7.0, dtype=BF16, device=DEV)
    got = ops.paged_tree(q.to(DEV) if hq % 2 else wide.to(DEV)[:, :hq], cache, table, segs, hk, 400, 129, scale=0.2,
                         out=held[:, :hq])
    _check()
    assert got.data_ptr() == held.data_ptr() and (held[:, hq:] == 7).all()
    ref, weight, err = _attend64(q, values, tab, sl, 0.2)
    assert ((got.double().cpu() - ref).abs() <= _tolerance(ref, weight, err, d, quantized)).all()


@pytest.mark.parametrize("quantized", [True, False], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("n", [6, 70])
def test_what_a_row_does_not_see_does_not_reach_it(n, quantized):
    """NaN and infinities in drafted nodes stay with the rows that see them."""
    ops = _ops()
    gen = torch.Generator().manual_seed(3)
    hq, hk, d = 8, 2, 128
    lens, cached = [n], [37]
    cache, table, segs, values, tab, sl = _paged(lens, cached, hk, d, quantized, gen)
    key, value = cached[0] + 2, cached[0] + 4  # nodes 2 (a NaN key) and 4 (values)
    pages = cache.pages if quantized else cache

    def at(pos):
        return tab[pos // 16], pos % 16

    b, o = at(key)
    values[b, 0, :, o, 9] = float("nan")
    if quantized:
        pages[b, 0, :, o * d + 9] = 0x7F
    else:
        pages[b, 0, :, o, 9] = float("nan")
    b, o = at(value)
    values[b, 1, :, o, 11] = float("nan")
    if quantized:
        pages[b, 1, :, o * d + 11] = 0xFF
    else:
        pages[b, 1, :, o, 11] = float("nan")
        pages[b, 1, :, o, 12] = float("inf")
        values[b, 1, :, o, 12] = float("inf")
    ms = [torch.eye(n, dtype=torch.bool)]
    ms[0][1, 2] = ms[0][3, 4] = ms[0][n - 1, 0] = True  # row 1 sees the key, row 3 the values
    q = torch.randn(n, hq, d, generator=gen).to(BF16)
    for split in (None, 16):
        out = ops.paged_tree(q.to(DEV), cache, table, segs, hk, n + 37, n, mask=_pack(ms), keys_per_split=split).cpu()
        _check()
        clean = [r for r in range(n) if r not in (1, 2, 3, 4)]
        ref, weight, err = _attend64(q, values, tab, sl, d ** -0.5, mask=ms)
        tol = _tolerance(ref, weight, err, d, quantized)
        assert ((out.double() - ref).abs() <= tol)[clean].all()
        assert out[[1, 2]].isnan().all()
        for r in (3, 4):
            assert out[r, :, 11].isnan().all()
            fine = [c for c in range(d) if c != 11 and (quantized or c != 12)]
            assert ((out[r].double() - ref[r]).abs() <= tol[r])[:, fine].all()
            if not quantized:
                assert (out[r, :, 12] == float("inf")).all()


@pytest.mark.parametrize("n", [3, 6, 70, 150])
def test_a_large_value_stays_with_the_rows_that_see_it(n):
    """A drafted node whose values are 2^100 times the others': its scale is no other row's unit."""
    ops = _ops()
    gen = torch.Generator().manual_seed(5)
    hq, hk, d = 8, 2, 128
    lens, cached = [n], [300]
    cache, table, segs, values, tab, sl = _paged(lens, cached, hk, d, True, gen)
    b, o = tab[302 // 16], 302 % 16  # node 2
    values[b, 1, :, o] *= 2.0 ** 100
    at = slice(16 * d + 4 * o, 16 * d + 4 * o + 4)
    scale = cache.pages[b, 1, :, at].contiguous().view(F32) * 2.0 ** 100
    cache.pages[b, 1, :, at] = scale.view(torch.uint8)
    ms = [torch.eye(n, dtype=torch.bool)]
    ms[0][n - 1, 0] = True
    q = torch.randn(n, hq, d, generator=gen).to(BF16)
    ref, weight, err = _attend64(q, values, tab, sl, d ** -0.5, mask=ms)
    for split in (None, 16, 128):
        out = ops.paged_tree(q.to(DEV), cache, table, segs, hk, n + 300, n, mask=_pack(ms), keys_per_split=split).cpu()
        _check()
        assert ((out.double() - ref).abs() <= _tolerance(ref, weight, err, d, True)).all()


@pytest.mark.parametrize("quantized", [True, False], ids=["e4m3", "bf16"])
def test_scores_of_a_wide_range(quantized):
    """Scores that rise by hundreds along the keys, and rows of large and of tiny queries."""
    ops = _ops()
    gen = torch.Generator().manual_seed(11)
    hq, hk, d = 8, 2, 128
    for n, split in ((1, 256), (1, 4096), (40, 4096), (40, 512)):
        cache, table, segs, values, tab, sl = _paged([n], [1500], hk, d, quantized, gen)
        q = torch.randn(n, hq, d, generator=gen) * torch.logspace(-30, 2.5, hq)[:, None]
        q = q.to(BF16)
        out = ops.paged_tree(q.to(DEV), cache, table, segs, hk, 1540, n, keys_per_split=split)
        _check()
        ref, weight, err = _attend64(q, values, tab, sl, d ** -0.5)
        assert ((out.double().cpu() - ref).abs() <= _tolerance(ref, weight, err, d, quantized)).all()


@pytest.mark.parametrize("quantized", [True, False], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("n", [2, 48])
def test_segments_that_do_not_fit_the_call(n, quantized):
    """Fields past the call's bounds give zeros and a status; rows of no segment stay as they were."""
    ops = _ops()
    gen = torch.Generator().manual_seed(2)
    hq, hk, d = 16, 8, 64
    cache, table, segs, values, tab, sl = _paged([n, n, n], [20, 30, 200], hk, d, quantized, gen)
    q = torch.randn(3 * n + 2, hq, d, generator=gen).to(BF16).to(DEV)
    whole = ops.paged_tree(q, cache, table, segs, hk, 200 + n, n)
    _check()

    def call(change=None, max_keys=200 + n, max_len=n):
        s = segs.clone()
        if change:
            s[1, change[0]] = change[1]
        out = torch.full_like(q, 3.0)
        ops.paged_tree(q, cache, table, s, hk, max_keys, max_len, out=out)
        return out, _status()

    for change in ((2, -1), (2, 500), (3, -4), (3, 100000), (4, 1), (4, 1 << 30), (1, n + 1), (2, (1 << 31) - 1)):
        out, code = call(change)
        assert code == 7, change
        rows = slice(n, 2 * n + (1 if change[0] == 1 else 0))
        other = 2 * n + (1 if change[0] == 1 else 0)
        if change[0] != 1:  # (a longer segment also covers the next one's first row)
            assert torch.count_nonzero(out[rows]) == 0, change
        assert torch.equal(out[:n], whole[:n]) and torch.equal(out[other:3 * n], whole[other:3 * n])
        assert (out[3 * n:] == 3).all()
    for change in ((0, -1), (0, 3 * n + 2), (1, -3), (0, (1 << 31) - 1)):  # rows outside q: nothing is written for them
        out, code = call(change)
        assert code == 7, change
        assert (out[n:2 * n] == 3).all() and torch.equal(out[:n], whole[:n])
    out, code = call((1, 0))  # an empty segment is nothing
    assert code == 0 and (out[n:2 * n] == 3).all()
    out, code = call(max_keys=100 + n)
    assert code == 7 and torch.count_nonzero(out[2 * n:3 * n]) == 0
    # A block ID outside the cache reads as zeros.
    bad = table.clone()
    bad[sl[2][3]] = 1 << 20
    bad[sl[2][3] + 1] = -7
    out = ops.paged_tree(q, cache, bad, segs, hk, 200 + n, n)
    assert _status() == 8
    assert torch.isfinite(out[:3 * n].float()).all()
    assert torch.equal(out[:2 * n], whole[:2 * n])


def test_a_fixed_split_gives_the_same_bits_in_any_batch():
    ops = _ops()
    gen = torch.Generator().manual_seed(8)
    hq, hk, d = 32, 8, 128
    cache, table, segs, _, _, sl = _paged([1] * 5 + [20], [900, 40, 3, 1777, 512, 600], hk, d, True, gen)
    q = torch.randn(25, hq, d, generator=gen).to(BF16).to(DEV)
    whole = ops.paged_tree(q, cache, table, segs, hk, 1778, 20, keys_per_split=512)
    again = ops.paged_tree(q, cache, table, segs, hk, 1778, 20, keys_per_split=512)
    assert torch.equal(whole, again)
    one = ops.paged_tree(q, cache, table, segs[3:4].contiguous(), hk, 1778, 20, keys_per_split=512)
    _check()
    assert torch.equal(whole[3], one[3])


@pytest.mark.parametrize("quantized", [True, False], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("n", [20, 40])
def test_parts_of_histories_around_whole_tiles(n, quantized):
    """Histories that end on, before and behind a tile, in parts of one to five tiles."""
    ops = _ops()
    gen = torch.Generator().manual_seed(n)
    hq, hk, d = 8, 2, 128
    cached = [0, 127 - n, 128 - n, 129 - n, 255, 256 - n, 257, 640 - n, 641 - n, 900]
    lens = [n] * len(cached)
    cache, table, segs, values, tab, sl = _paged(lens, cached, hk, d, quantized, gen)
    masks = _random_masks(lens, gen)
    q = torch.randn(sum(lens), hq, d, generator=gen).to(BF16)
    ref, weight, err = _attend64(q, values, tab, sl, d ** -0.5, mask=masks)
    for split in (128, 256, 384, 640):
        out = ops.paged_tree(q.to(DEV), cache, table, segs, hk, max(cached) + n, n, mask=_pack(masks), keys_per_split=split)
        _check()
        assert ((out.double().cpu() - ref).abs() <= _tolerance(ref, weight, err, d, quantized)).all()


def test_a_long_row_of_many_splits_has_the_same_bits_in_any_batch():
    ops = _ops()
    gen = torch.Generator().manual_seed(8)
    hq, hk, d = 16, 4, 64
    lens, cached = [1] * 70, [16 * 40 - 1, 16 * 11 + 3] + [16 * 30] + [16 * (i % 19) + i % 7 for i in range(67)]
    cache, table, segs, values, tab, sl = _paged(lens, cached, hk, d, True, gen)
    q = torch.randn(70, hq, d, generator=gen).to(BF16).to(DEV)
    every = ops.paged_decode(q, cache, table, segs, hk, max(cached) + 1, keys_per_split=16)
    for i in range(4):
        alone = segs[i:i + 1].clone()
        alone[0, 0] = 0
        one = ops.paged_decode(q[i:i + 1], cache, table, alone, hk, cached[i] + 1, keys_per_split=16)
        assert torch.equal(one[0], every[i])
    _check()
    ref, weight, err = _attend64(q.cpu(), values, tab, sl, d ** -0.5)
    assert ((every.double().cpu() - ref).abs() <= _tolerance(ref, weight, err, d, True)).all()


def test_offsets_past_32_bits():
    """Pages beyond 2^32 bytes of the cache: a quantized cache of 4.6 GB whose last blocks are used."""
    ops = _ops()
    hq, hk, d = 16, 8, 128
    blocks = (1 << 32) // (2 * hk * (16 * d + 64)) + 9000
    pages = torch.zeros(blocks, 2, hk, 16 * d + 64, dtype=torch.uint8, device=DEV)
    cache = ops.QuantizedCache(pages, d)
    gen = torch.Generator().manual_seed(4)
    small, table, segs, values, tab, sl = _paged([1, 40], [70, 90], hk, d, True, gen)
    far = blocks - small.pages.shape[0]
    pages[far:] = small.pages
    q = torch.randn(41, hq, d, generator=gen).to(BF16)
    out = ops.paged_tree(q.to(DEV), cache, table + far, segs, hk, 130, 40)
    _check()
    ref, weight, err = _attend64(q, values, tab, sl, d ** -0.5)
    assert ((out.double().cpu() - ref).abs() <= _tolerance(ref, weight, err, d, True)).all()
    # The store reaches them too.
    qkv = torch.randn(2, (hq + 2 * hk) * d, device=DEV).to(BF16)
    slots = torch.tensor([blocks * 16 - 1, 5], device=DEV, dtype=I32)
    pos = torch.zeros(2, device=DEV, dtype=I32)
    ops.qk_norm_rope_cache(qkv, hq, hk, d, None, None, 1e-6, pos, torch.ones(64, device=DEV), 1.0, cache, slots)
    _check()
    y = qkv[0].view(-1, d)[-hk:].float()
    got = cache.codes[-1, 1, :, 15].view(E4M3).float() * cache.scales[-1, 1, :, 15, None]
    assert ((got - y).abs() <= 2.0 ** -4 * y.abs() + 2.0 ** -18 * y.abs().amax(-1, keepdim=True)).all()


# ---------------------------------------------------------------------------------------- logits


def _logits64(x, prompt, output, rep, freq, pres, bias, allowed):
    """Per row python lists; x [rows, vocab] FP64. Returns (values, magnitudes for the tolerance)."""
    x = x.clone()
    size = x.abs()
    rows, vocab = x.shape
    for r in range(rows):
        inside = [t for t in output[r] if 0 <= t < vocab]
        listed = set(inside) | {t for t in prompt[r] if 0 <= t < vocab} if rep is not None else set()
        for t in listed:
            x[r, t] = x[r, t] / rep[r] if x[r, t] > 0 else x[r, t] * rep[r]
            size[r, t] += x[r, t].abs()
        for t in set(inside):
            n = inside.count(t)
            f = freq[r] * n if freq is not None else 0.0
            g = pres[r] if pres is not None else 0.0
            x[r, t] -= f + g
            size[r, t] += abs(f) + abs(g)
        for t, v in dict(bias[r]).items():
            if 0 <= t < vocab:
                x[r, t] += v
                size[r, t] += abs(v)
        if allowed is not None:
            x[r, ~allowed[r]] = -torch.inf
    return x, size


def _csr(lists, kind=I32, pick=lambda v: v):
    flat = [pick(v) for row in lists for v in row]
    starts = [0]
    for row in lists:
        starts.append(starts[-1] + len(row))
    return torch.tensor(flat, dtype=kind, device=DEV), torch.tensor(starts, dtype=I32, device=DEV)


def _bits(allowed):
    rows, vocab = allowed.shape
    words = (vocab + 31) // 32
    full = torch.zeros(rows, words * 32, dtype=torch.int64)
    full[:, :vocab] = allowed.long()
    return (full.view(rows, words, 32) << torch.arange(32)).sum(-1).to(I32).to(DEV)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab,features", [
    (1, 1, "pb"), (3, 7, "pbm"), (2, 31, "m"), (5, 1000, "pbm"), (2, 1001, "p"), (3, 32000, "b"), (2, 151936, "pbm"),
    (2, 262145, "pbm"), (4, 50257, ""), (1, 700001, "pbm"), (2, 33, "f"), (2, 4099, "r"),
])
def test_process_logits(rows, vocab, features, dtype):
    ops = _ops()
    rng = random.Random(rows * vocab)
    gen = torch.Generator().manual_seed(vocab)
    pad = rng.randrange(0, 9)
    wide = torch.randn(rows, vocab + pad, generator=gen).mul(4).to(dtype).to(DEV)
    x = wide[:, pad:]  # rows that begin at any place
    if rows > 1 and vocab > 3:
        x[1, 2] = float("nan")
    few = [rng.randrange(vocab) for _ in range(20)]
    lists = lambda n: [[rng.choice(few) if rng.random() < 0.5 else rng.randrange(vocab) for _ in range(rng.randrange(n))]  # noqa: E731
                       + [vocab, -1, vocab + 5] for _ in range(rows)]
    prompt, output = lists(300), lists(2000)
    output[-1] = []
    rep = freq = pres = None
    if "p" in features or "r" in features:
        rep = torch.rand(rows, generator=gen) + 0.8
    if "p" in features or "f" in features:
        freq = torch.rand(rows, generator=gen) - 0.2
    if "p" in features:
        pres = torch.rand(rows, generator=gen)
    bias = [[(rng.randrange(-1, vocab + 1), rng.uniform(-9, 9)) for _ in range(rng.randrange(40))] for _ in range(rows)]
    if "b" not in features:
        bias = [[] for _ in range(rows)]
    elif vocab > 3:
        bias[0] += [(3, 1.0), (3, 2.0), (3, -0.5)]  # the last one counts
    bias = [[(t, float(torch.tensor(v, dtype=F32))) for t, v in row] for row in bias]
    allowed = None
    if "m" in features:
        allowed = torch.rand(rows, vocab, generator=gen) < torch.tensor([0.9, 0.01, 0.5, 0.0, 0.3])[:rows, None]
        if rows > 2:
            allowed[2] = False  # nothing is left
            allowed[0] = False
            allowed[0, vocab - 1] = True
    out = torch.full((rows, vocab + 3), 9.0, dtype=dtype, device=DEV)[:, :vocab]
    kw = dict(prompt=_csr(prompt), output=_csr(output), allowed=None if allowed is None else _bits(allowed))
    for name, v in (("repetition", rep), ("frequency", freq), ("presence", pres)):
        if v is not None:
            kw[name] = v.to(DEV)
    if "b" in features:
        bt, bs = _csr(bias, pick=lambda v: v[0])
        kw["bias"] = (bt, _csr(bias, kind=F32, pick=lambda v: v[1])[0], bs)
    index, value = ops.process_logits(x, out=out, **kw)
    greedy = ops.process_logits(x, **kw)
    _check()
    assert torch.equal(index, greedy[0]) and torch.equal(value, greedy[1])
    d64 = lambda v: None if v is None else v.double()  # noqa: E731
    ref, size = _logits64(x.double().cpu(), prompt, output, d64(rep), d64(freq), d64(pres), bias, allowed)
    # Five FP32 steps (a product, a quotient or product, two differences, a sum), and one rounding
    # of the stored logit.
    got = out.double().cpu()
    tol = 5 * 2.0 ** -24 * size + (_half(BF16) * ref.abs() if dtype == BF16 else 0)
    inf = ref == -torch.inf
    assert torch.equal(got == -torch.inf, inf) and torch.equal(got.isnan(), ref.isnan())
    real = ~inf & ~ref.isnan()
    assert ((got - ref).abs() <= tol)[real].all()
    assert torch.all(out.as_strided((rows, 3), (vocab + 3, 1), out.storage_offset() + vocab) == 9)
    for r in range(rows):
        ok = real[r]
        if not ok.any():
            assert index[r] == -1 and value[r] == -torch.inf
            continue
        i = int(index[r])
        assert ok[i] and (value[r].double().cpu() - ref[r, i]).abs() <= 5 * 2.0 ** -24 * size[r, i]
        assert (ref[r, ok] <= ref[r, i] + (5 * 2.0 ** -24 * size[r])[ok] + 5 * 2.0 ** -24 * size[r, i]).all()
        if dtype == F32:
            best = out[r].cpu()[ok].max()
            assert value[r].cpu() == best and i == int((out[r].cpu() == best).nonzero()[0])


def test_process_logits_ties_in_place_and_bad_lists():
    ops = _ops()
    x = torch.zeros(2, 5000, device=DEV)
    x[:, [17, 18, 4999]] = 3.0
    index, value = ops.process_logits(x)
    assert index.tolist() == [17, 17] and value.tolist() == [3.0, 3.0]
    # In place: the same as into another tensor.
    lists = (torch.tensor([17, 17, 40], device=DEV, dtype=I32), torch.tensor([0, 3, 3], device=DEV, dtype=I32))
    freq = torch.full((2,), 0.5, device=DEV)
    other = torch.empty_like(x)
    a = ops.process_logits(x, output=lists, frequency=freq, out=other)
    b = ops.process_logits(x, output=lists, frequency=freq, out=x)
    _check()
    assert torch.equal(x, other) and torch.equal(a[0], b[0]) and a[0].tolist() == [18, 17]
    assert x[0, 17] == 2.0 and x[0, 40] == -0.5 and x[1, 40] == 0.0
    # Starts that leave the list read as an empty list.
    for starts in ([0, 3, 4], [2, 1, 3], [-1, 2, 3]):
        bad = (lists[0], torch.tensor(starts, device=DEV, dtype=I32))
        ops.process_logits(x, output=bad, frequency=freq, out=other)
        assert _status() == 7
        rows = [r for r in range(2) if not 0 <= starts[r] <= starts[r + 1] <= 3]
        assert torch.equal(other[rows], x[rows])
    none = ops.process_logits(x[:0], out=other[:0])
    assert none[0].shape == (0,)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab,output,biases,padding", [
    (2, 20000, 30000, 9000, 0),  # most of the vocabulary listed
    (900, 8200, 40, 3, 0),       # more slices than the GPU holds at once
    (3, 9000, 4000, 3000, 1 << 21),  # lists whose counts and places need more than one word
])
def test_process_logits_long_lists_in_place(rows, vocab, output, biases, padding, dtype):
    ops = _ops()
    gen = torch.Generator().manual_seed(vocab)
    x = torch.randn(rows, vocab, generator=gen).mul(4).to(dtype)
    draw = lambda n: torch.randint(0, vocab, (rows, n), generator=gen)  # noqa: E731
    prompt, out_tokens = draw(output // 2), draw(output)
    out_tokens[0, : output // 2] = 5  # one token many times
    bias_tokens = torch.stack([torch.randperm(vocab, generator=gen)[:biases] for _ in range(rows)])
    bias_values = torch.randn(rows, biases, generator=gen)
    rep = torch.rand(rows, generator=gen) + 0.8
    freq, pres = torch.rand(rows, generator=gen) * 0.1, torch.rand(rows, generator=gen)
    allowed = torch.rand(rows, vocab, generator=gen) < 0.6

    def csr(tokens, extra=0):
        flat = torch.cat([tokens.flatten().to(I32), torch.full((extra,), vocab, dtype=I32)])
        return flat.to(DEV), (torch.arange(rows + 1) * tokens.shape[1]).to(I32).to(DEV)

    bt, bs = csr(bias_tokens)
    kw = dict(prompt=csr(prompt), output=csr(out_tokens, padding), repetition=rep.to(DEV), frequency=freq.to(DEV),
              presence=pres.to(DEV), bias=(bt, bias_values.flatten().to(DEV), bs), allowed=_bits(allowed))
    mine = x.to(DEV)
    index, value = ops.process_logits(mine, out=mine, **kw)
    _check()
    count = torch.zeros(rows, vocab, dtype=torch.float64).scatter_add_(1, out_tokens, torch.ones(rows, output, dtype=torch.float64))
    listed = (count > 0).scatter(1, prompt, torch.ones(rows, output // 2, dtype=torch.bool))
    col = lambda v: v.double()[:, None]  # noqa: E731
    ref = x.double()
    size = ref.abs()
    ref = torch.where(listed, torch.where(ref > 0, ref / col(rep), ref * col(rep)), ref)
    size = size + ref.abs() + (count > 0) * (col(freq) * count + col(pres))
    ref = ref - (count > 0) * (col(freq) * count + col(pres))
    ref = ref.scatter_add(1, bias_tokens, bias_values.double())
    size = size.scatter_add(1, bias_tokens, bias_values.double().abs())
    # Five FP32 steps, and one rounding of the stored logit.
    tol = 5 * 2.0 ** -24 * size
    got = mine.double().cpu()
    assert torch.equal(got == -torch.inf, ~allowed)
    assert ((got - ref).abs() <= tol + (_half(BF16) * ref.abs() if dtype == BF16 else 0))[allowed].all()
    i, row = index.long().cpu(), torch.arange(rows)
    assert allowed[row, i].all() and ((value.double().cpu() - ref[row, i]).abs() <= tol[row, i]).all()
    least = torch.where(allowed, ref - tol, torch.tensor(-torch.inf, dtype=torch.float64)).amax(1)
    assert (ref[row, i] + tol[row, i] >= least).all()


# ------------------------------------------------------------------------------- a run of them all


class _Step:
    """One speculative step of a one-layer model over a quantized cache: drafted rows are projected
    to q/k/v, stored, attended with their tree and scored under penalties and a grammar mask."""

    def __init__(self, seed, vocab=2048, hq=8, hk=2, d=64, hidden=256):
        g = torch.Generator().manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=g).mul(s[-1] ** -0.5).to(BF16).to(DEV)  # noqa: E731
        self.hq, self.hk, self.d, self.vocab = hq, hk, d, vocab
        self.emb = torch.randn(vocab, hidden, generator=g).to(BF16).to(DEV)
        self.w_qkv, self.w_o, self.head = rand((hq + 2 * hk) * d, hidden), rand(hidden, hq * d), rand(vocab, hidden)
        self.qn, self.kn = torch.ones(d, dtype=BF16, device=DEV), torch.ones(d, dtype=BF16, device=DEV)
        self.inv_freq = 1e4 ** (-torch.arange(0, d, 2, device=DEV, dtype=F32) / d)
        self.blocks = 24
        self.cache = _ops().QuantizedCache.empty(self.blocks, hk, d)

    def __call__(self, tokens, positions, slots, table, segments, max_keys, max_len, mask, **logit_args):
        ops = _ops()
        qkv = ops.gemm(ops.embedding(tokens, self.emb), self.w_qkv)
        q = ops.qk_norm_rope_cache(qkv, self.hq, self.hk, self.d, self.qn, self.kn, 1e-6, positions, self.inv_freq, 1.0,
                                   self.cache, slots)
        o = ops.paged_tree(q, self.cache, table, segments, self.hk, max_keys, max_len, mask=mask)
        logits = ops.gemm(ops.gemm(o.flatten(1), self.w_o), self.head, epilogue=ops.EPI_F32)
        return (o, logits) + ops.process_logits(logits, **logit_args)


def _step_inputs(step, seed):
    """Two sequences of 50 and 33 positions, a tree of 7 and one of 4 drafted nodes."""
    rng = random.Random(seed)
    hist = [50, 33]
    parents = [[-1, 0, 0, 1, 1, 2, 5], [-1, 0, 1, -1]]
    blocks = rng.sample(range(step.blocks), 10)
    tables = [blocks[:5], blocks[5:]]
    i32 = lambda v: torch.tensor(v, dtype=I32, device=DEV)  # noqa: E731
    slot = lambda s, p: tables[s][p // 16] * 16 + p % 16  # noqa: E731
    prompt = dict(
        tokens=i32([rng.randrange(step.vocab) for _ in range(sum(hist))]),
        positions=i32([p for n in hist for p in range(n)]),
        slots=i32([slot(s, p) for s, n in enumerate(hist) for p in range(n)]),
        table=i32(blocks), segments=i32([[0, 50, 0, 0, 4], [50, 33, 0, 5, 3]]), max_keys=64, max_len=50, mask=None)
    depth = []
    for tree in parents:
        d = []
        for p in tree:
            d.append(0 if p < 0 else d[p] + 1)
        depth.append(d)
    drafted = dict(
        tokens=i32([rng.randrange(step.vocab) for _ in range(11)]),
        positions=i32([hist[s] + x for s in range(2) for x in depth[s]]),
        slots=i32([slot(s, hist[s] + j) for s, t in enumerate(parents) for j in range(len(t))]),
        table=i32(blocks), segments=i32([[0, 7, 50, 0, 5], [7, 4, 33, 5, 5]]), max_keys=80, max_len=8,
        mask=_ops().tree_mask(parents).to(DEV))
    words = step.vocab // 32
    drafted.update(
        output=(i32([rng.randrange(step.vocab) for _ in range(11 * 6)]), i32([6 * r for r in range(12)])),
        presence=torch.rand(11, device=DEV), frequency=torch.rand(11, device=DEV),
        allowed=torch.randint(-2 ** 31, 2 ** 31, (11, words), device=DEV, dtype=torch.int64).to(I32))
    return prompt, drafted, parents


def test_a_speculative_step():
    ops = _ops()
    step = _Step(0)
    prompt, drafted, parents = _step_inputs(step, 0)
    step(**prompt)
    o, logits, index, value = step(**drafted)
    _check()
    # The drafted rows' attention from what the cache holds.
    qkv = ops.gemm(ops.embedding(drafted["tokens"], step.emb), step.w_qkv)
    rq, _, _ = _front64(qkv, step.hq, step.hk, step.d, step.qn, step.kn, 1e-6, drafted["positions"], step.inv_freq, 1.0,
                        step.d, False)
    values = (step.cache.codes.view(E4M3).double() * step.cache.scales.double()[..., None]).cpu()
    ms = [torch.zeros(len(t), len(t), dtype=torch.bool) for t in parents]
    for m, tree in zip(ms, parents):
        for i, p in enumerate(tree):
            if p >= 0:
                m[i] |= m[p]
            m[i, i] = True
    ref, weight, err = _attend64(rq.to(BF16), values, drafted["table"].cpu().long(), drafted["segments"].tolist(),
                                 step.d ** -0.5, mask=ms)
    # q rounds to BF16 in the kernel from FP32 and here from FP64: a step apart at most, which moves
    # each score by 2^-8 of its sum of magnitudes at worst.
    tol = _tolerance(ref, weight, err, step.d, True) + 2 * _half(BF16) * 2 * weight * err[0]
    assert ((o.double().cpu() - ref).abs() <= tol).all()
    lists = drafted["output"][0].view(11, 6).tolist()
    bits = (drafted["allowed"].cpu().long()[:, :, None] >> torch.arange(32)).flatten(1) & 1 == 1
    want, size = _logits64(logits.double().cpu(), [[]] * 11, lists, None, drafted["frequency"].double().cpu(),
                           drafted["presence"].double().cpu(), [[]] * 11, bits)
    top = want.amax(-1)
    assert ((value.double().cpu() - top).abs() <= 5 * 2.0 ** -24 * size.amax(-1)).all()
    assert bits[torch.arange(11), index.cpu().long()].all()


def test_a_captured_step_replays_on_other_inputs_and_streams():
    """Two graphs of the step, replayed in turn and side by side on two streams, against eager calls."""
    ops = _ops()
    ops.scratch(torch.device("cuda", 0))
    steps = [_Step(1), _Step(2)]
    ins = [_step_inputs(s, i) for i, s in enumerate(steps)]
    for s, (prompt, drafted, _) in zip(steps, ins):
        s(**prompt)
        s(**drafted)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s, (_, drafted, _) in zip(steps, ins):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s(**drafted))
        graphs.append(g)
    for seed in (5, 6):
        wants = []
        for s, (_, drafted, _) in zip(steps, ins):
            gen = torch.Generator().manual_seed(seed)
            drafted["tokens"].copy_(torch.randint(0, s.vocab, (11,), generator=gen).to(I32))
            before = s.cache.pages.clone()
            wants.append([t.clone() for t in s(**drafted)])
            s.cache.pages.copy_(before)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for _ in range(3):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for want, got in zip(wants, outs):
            assert all(torch.equal(a, b) for a, b in zip(want, got))
    _check()


def test_calls_run_on_the_current_stream():
    ops = _ops()
    gen = torch.Generator().manual_seed(9)
    cache, table, segs, _, _, _ = _paged([1] * 4, [500, 600, 700, 2000], 8, 128, True, gen)
    q = torch.randn(4, 16, 128, generator=gen).to(BF16).to(DEV)
    want = ops.paged_decode(q, cache, table, segs, 8, 2001)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    big = torch.randn(4096, 4096, device=DEV)
    late = torch.zeros_like(q)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            big = (big @ big).tanh()
        late.copy_(q)  # arrives behind the products
        got = ops.paged_decode(late, cache, table, segs, 8, 2001)
    side.synchronize()
    _check()
    assert torch.equal(want, got)


def test_a_first_call_is_not_captured(monkeypatch):
    """The device's status word is laid out by the first call, outside of any graph."""
    ops = _ops()
    monkeypatch.setattr("furiosa_opt_models_b200.ops.decode._scratch", {})
    x = torch.zeros(1, 8, device=DEV)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = x + 1  # noqa: F841
        with pytest.raises(RuntimeError, match="cannot be captured"):
            ops.process_logits(x)


@pytest.mark.parametrize("quantized", [True, False], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("n", [1, 3, 6, 20, 70])
def test_a_query_that_is_not_finite_gives_nan_in_any_split(n, quantized):
    """Its row is NaN whether one part of the history answers it or several, zeros where it sees no
    key; the other rows are as they would be."""
    ops = _ops()
    gen = torch.Generator().manual_seed(n)
    hq, hk, d = 8, 2, 128
    lens, cached = [n, n], [300, 0]
    cache, table, segs, values, tab, sl = _paged(lens, cached, hk, d, quantized, gen)
    ms = [torch.eye(n, dtype=torch.bool) for _ in lens]
    q = torch.randn(2 * n, hq, d, generator=gen).to(BF16)
    odd = q.clone()
    odd[0, 1, 5], odd[n, 6, 7], odd[2 * n - 1, 0, 100] = float("nan"), float("inf"), -float("inf")
    bad = torch.zeros(2 * n, hq, dtype=torch.bool)
    bad[0, 1] = bad[n, 6] = bad[2 * n - 1, 0] = True
    if n > 2:
        ms[1][1] = False
        odd[n + 1, 3, 0] = float("nan")
    ref, weight, err = _attend64(q, values, tab, sl, d ** -0.5, mask=ms)
    tol = _tolerance(ref, weight, err, d, quantized)
    for split in (None, 16, 128, 4096):
        out = ops.paged_tree(odd.to(DEV), cache, table, segs, hk, n + 300, n, mask=_pack(ms), keys_per_split=split).cpu()
        _check()
        assert out[bad].isnan().all(), split
        assert ((out.double() - ref).abs() <= tol)[~bad].all(), split
        if n > 2:
            assert torch.count_nonzero(out[n + 1]) == 0


@pytest.mark.parametrize("quantized", [True, False], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("n", [3, 20, 70])
def test_a_row_whose_only_key_is_nan(n, quantized):
    ops = _ops()
    gen = torch.Generator().manual_seed(n)
    hq, hk, d = 8, 2, 64
    cache, table, segs, values, tab, sl = _paged([n], [0], hk, d, quantized, gen)
    if quantized:
        cache.pages[tab[0], 0, :, 2 * d + 9] = 0x7F  # node 2's key
    else:
        cache[tab[0], 0, :, 2, 9] = float("nan")
    ms = [torch.eye(n, dtype=torch.bool)]
    q = torch.randn(n, hq, d, generator=gen).to(BF16)
    ref, weight, err = _attend64(q, values, tab, sl, d ** -0.5, mask=ms)
    tol = _tolerance(ref, weight, err, d, quantized)
    other = torch.arange(n) != 2
    for split in (None, 16, 4096):
        out = ops.paged_tree(q.to(DEV), cache, table, segs, hk, n, n, mask=_pack(ms), keys_per_split=split).cpu()
        _check()
        assert out[2].isnan().all() and ((out.double() - ref).abs() <= tol)[other].all()


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("n", [6, 20, 70])
def test_scales_that_are_not_finite_stay_with_the_rows_that_see_them(n, bad):
    ops = _ops()
    gen = torch.Generator().manual_seed(n)
    hq, hk, d = 8, 2, 128
    cache, table, segs, values, tab, sl = _paged([n], [37], hk, d, True, gen)
    for which, node in ((0, 2), (1, 4)):  # node 2's key, node 4's values
        b, o = tab[(37 + node) // 16], (37 + node) % 16
        cache.pages[b, which, :, 16 * d + 4 * o:16 * d + 4 * o + 4] = torch.tensor([bad]).view(torch.uint8).to(DEV)
    ms = [torch.eye(n, dtype=torch.bool)]
    ms[0][1, 2] = ms[0][3, 4] = ms[0][n - 1, 0] = True  # row 1 sees the key, row 3 the values
    q = torch.randn(n, hq, d, generator=gen).to(BF16)
    ref, weight, err = _attend64(q, values, tab, sl, d ** -0.5, mask=ms)
    tol = _tolerance(ref, weight, err, d, True)
    clean = [r for r in range(n) if r not in (1, 2, 3, 4)]
    for split in (None, 16, 128):
        out = ops.paged_tree(q.to(DEV), cache, table, segs, hk, n + 37, n, mask=_pack(ms), keys_per_split=split).cpu()
        _check()
        assert ((out.double() - ref).abs() <= tol)[clean].all(), split
        assert not out[[3, 4]].isfinite().any(), split
        if bad != bad:
            assert out[1:5].isnan().all(), split


def test_a_status_of_another_stream_outlives_the_first_call(monkeypatch):
    """The first call's stream is busy when its status word is laid out; a kernel of another stream
    records a status at once, and nothing erases it."""
    import importlib

    ops = _ops()
    fresh = {}
    for module in ("decode", "native"):
        monkeypatch.setattr(importlib.import_module("furiosa_opt_models_b200.ops." + module), "_scratch", fresh)
    x = torch.zeros(1, 64, device=DEV)
    tokens, starts = torch.zeros(1, dtype=I32, device=DEV), torch.tensor([0, 9], dtype=I32, device=DEV)  # past the list
    big = torch.randn(4096, 4096, device=DEV)
    torch.cuda.synchronize()
    busy, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(busy):
        for _ in range(200):
            big = (big @ big).tanh()
        ops.scratch(torch.device("cuda", 0))
    with torch.cuda.stream(other):
        ops.process_logits(x, output=(tokens, starts), presence=torch.ones(1, device=DEV))
    torch.cuda.synchronize()
    assert int(fresh[0].status[0].item()) == 7


@pytest.mark.parametrize("quantized", [True, False], ids=["e4m3", "bf16"])
def test_bounds_far_above_the_lengths(quantized):
    """max_len and max_keys at their largest, as a captured call may give them, and many empty segments:
    what is launched follows the rows that exist."""
    ops = _ops()
    gen = torch.Generator().manual_seed(1)
    hq, hk, d = 8, 2, 64
    lens, cached = [1, 3, 2], [40, 90, 7]
    cache, table, segs, values, tab, sl = _paged(lens, cached, hk, d, quantized, gen)
    many = torch.zeros(300, 5, dtype=I32, device=DEV)
    many[[0, 150, 299]] = segs
    q = torch.randn(6, hq, d, generator=gen).to(BF16)
    ref, weight, err = _attend64(q, values, tab, sl, d ** -0.5)
    tol = _tolerance(ref, weight, err, d, quantized)
    for split in (None, 64, 1 << 20):
        keys = 1 << 30 if split is None or split > 64 else 128
        out = ops.paged_tree(q.to(DEV), cache, table, many, hk, keys, 1 << 24, keys_per_split=split)
        _check()
        assert ((out.double().cpu() - ref).abs() <= tol).all()


@pytest.mark.parametrize("quantized", [True, False], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("n", [1, 6, 20, 70])
def test_attention_written_over_its_queries(n, quantized):
    ops = _ops()
    gen = torch.Generator().manual_seed(n)
    hq, hk, d = 8, 2, 128
    lens, cached = [n, (n + 1) // 2, n], [700, 30, 0]
    cache, table, segs, _, _, _ = _paged(lens, cached, hk, d, quantized, gen)
    q = torch.randn(sum(lens) + 1, hq, d, generator=gen).to(BF16).to(DEV)
    for split in (None, 128, 4096):
        want = q.clone()
        ops.paged_tree(q, cache, table, segs, hk, 700 + n, n, keys_per_split=split, out=want)
        for _ in range(5):
            got = q.clone()
            ops.paged_tree(got, cache, table, segs, hk, 700 + n, n, keys_per_split=split, out=got)
            assert torch.equal(got, want)
    # Beside the queries, in the rows of one tensor.
    both = torch.cat([q, torch.zeros_like(q)], 1)
    ops.paged_tree(both[:, :hq], cache, table, segs, hk, 700 + n, n, keys_per_split=128, out=both[:, hq:])
    apart = torch.zeros_like(q)
    ops.paged_tree(q, cache, table, segs, hk, 700 + n, n, keys_per_split=128, out=apart)
    _check()
    assert torch.equal(both[:, :hq], q) and torch.equal(both[:, hq:], apart)


@pytest.mark.parametrize("quantized", [True, False], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("n", [1, 6, 20, 70])
def test_a_negative_scale(n, quantized):
    ops = _ops()
    gen = torch.Generator().manual_seed(n)
    hq, hk, d = 8, 2, 64
    cache, table, segs, values, tab, sl = _paged([n], [200], hk, d, quantized, gen)
    q = torch.randn(n, hq, d, generator=gen).to(BF16)
    ref, weight, err = _attend64(q, values, tab, sl, -0.3)
    tol = _tolerance(ref, weight, tuple(e.abs() for e in _attend64(q, values, tab, sl, 0.3)[2]), d, quantized)
    for split in (None, 16, 128):
        out = ops.paged_tree(q.to(DEV), cache, table, segs, hk, n + 200, n, scale=-0.3, keys_per_split=split)
        _check()
        assert ((out.double().cpu() - ref).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tied", [
    [4, 5, 7], [13, 1024 + 8, 3], [2048 + 7, 2048 + 5], [8191, 9000, 20000], [20000, 16384], [0, 24999], [24999],
    [24998, 24999], list(range(25000)),
])
@pytest.mark.parametrize("pad", [0, 1, 5])
def test_the_first_of_equal_maxima_is_chosen(tied, pad, dtype):
    """Equal maxima inside a vector, across a thread's vectors, in a row's unaligned ends and in other
    slices, among values that are below them; with a list, a listed token may be one of them."""
    ops = _ops()
    vocab = 25000
    wide = torch.full((3, vocab + pad), -1.0, dtype=dtype, device=DEV)
    x = wide[:, pad:]
    x[:, tied] = 2.5
    index, value = ops.process_logits(x)
    assert index.tolist() == [min(tied)] * 3 and value.tolist() == [2.5] * 3
    # A listed token that ends at the same value, before and behind the others (3.5 - 1 = 2.5).
    for token in (1, 8190, vocab - 2):
        x[:, tied] = 2.5
        x[:, token] = 3.5
        lists = (torch.tensor([token], dtype=I32, device=DEV), torch.tensor([0, 1, 1, 1], dtype=I32, device=DEV))
        index, value = ops.process_logits(x, output=lists, presence=torch.ones(3, device=DEV))
        assert index.tolist() == [min([token] + tied), token, token] and value.tolist() == [2.5, 3.5, 3.5]
        x[:, token] = -1.0
    # The first is not allowed: the next one.
    if len(tied) > 1:
        x[:, tied] = 2.5
        allowed = torch.ones(3, vocab, dtype=torch.bool)
        allowed[1, min(tied)] = False
        index, _ = ops.process_logits(x, allowed=_bits(allowed))
        assert index.tolist() == [min(tied), sorted(tied)[1], min(tied)]
    _check()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_infinite_logits(dtype):
    ops = _ops()
    inf = float("inf")
    x = torch.randn(4, 9001, device=DEV).to(dtype)
    x[0, 8500] = x[0, 77] = inf
    x[1] = -inf
    x[2] = float("nan")
    x[3, :9000] = -inf
    one = lambda t: (torch.tensor([t], dtype=I32, device=DEV), torch.tensor([0, 1, 1, 1, 1], dtype=I32, device=DEV))  # noqa: E731
    for kw in ({}, dict(output=one(77), frequency=torch.ones(4, device=DEV))):
        out = torch.empty_like(x)
        index, value = ops.process_logits(x, out=out, **kw)
        assert index.tolist() == [77, -1, -1, 9000]
        assert value.tolist()[:3] == [inf, -inf, -inf] and value[3] == x[3, 9000]
        assert torch.equal(out.nan_to_num(5.0), x.nan_to_num(5.0))
    index, value = ops.process_logits(x, prompt=one(77), repetition=torch.full((4,), inf, device=DEV))
    assert index[0] == 8500 and value[0] == inf  # inf / inf is NaN and never chosen
    _check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [33, 20011])
def test_masks_that_are_wide_strided_or_shared(vocab, dtype):
    ops = _ops()
    gen = torch.Generator().manual_seed(vocab)
    x = torch.randn(5, vocab, generator=gen).to(dtype).to(DEV)
    allowed = torch.rand(5, vocab, generator=gen) < 0.3
    bits = _bits(allowed)
    words = bits.shape[1]
    want, best = torch.empty_like(x), x.masked_fill(~allowed.to(DEV), -torch.inf)
    i0, v0 = ops.process_logits(x, allowed=bits, out=want)
    assert torch.equal(want, best) and torch.equal(v0, best.float().amax(1))
    for extra, skip in ((1, 0), (7, 3), (64, 1)):  # wider than it must be, rows of a wider tensor
        wide = torch.full((5, skip + words + extra), -1, dtype=I32, device=DEV)
        wide[:, skip:skip + words] = bits
        for view in (wide[:, skip:], wide[:, skip:skip + words]):
            out = torch.empty_like(x)
            i, v = ops.process_logits(x, allowed=view, out=out)
            assert torch.equal(i, i0) and torch.equal(v, v0) and torch.equal(out, want)
    shared = bits[1:2].expand(5, words)  # one mask for every row
    _, v = ops.process_logits(x, allowed=shared)
    assert torch.equal(v, x.masked_fill(~allowed[1].to(DEV), -torch.inf).float().amax(1))
    _check()


def test_calls_from_several_threads():
    """The calls release the interpreter: four threads on streams of their own, each with its inputs."""
    import threading

    ops = _ops()
    hq, hk, d = 8, 2, 64
    jobs = []
    for i in range(4):
        gen = torch.Generator().manual_seed(i)
        n = (1, 5, 20, 40)[i]
        cache, table, segs, _, _, _ = _paged([n] * 3, [100, 900, 40], hk, d, True, gen)
        q = torch.randn(3 * n, hq, d, generator=gen).to(BF16).to(DEV)
        x = torch.randn(4, 30000 + i, generator=gen).to(DEV)
        jobs.append((q, cache, table, segs, n, x))

    def call(job):
        q, cache, table, segs, n, x = job
        return (ops.paged_tree(q, cache, table, segs, hk, 900 + n, n, keys_per_split=128),) + ops.process_logits(x)

    want = [call(j) for j in jobs]
    torch.cuda.synchronize()
    faults = []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(50):
                    got = call(jobs[i])
                    stream.synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, want[i]))
        except BaseException as e:  # noqa: BLE001
            faults.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    _check()
    assert not faults, faults[0]


def test_captured_calls_of_many_parts_and_slices_replay_side_by_side():
    """Two graphs of wide trees in several parts and of logits in several slices, on two streams at once."""
    ops = _ops()
    gen = torch.Generator().manual_seed(1)
    hk, vocab = 2, 40000
    jobs = []
    for quantized in (True, False):
        cache, table, segs, _, _, _ = _paged([40, 20, 33], [900, 2000, 5], hk, 128, quantized, gen)
        q = torch.randn(93, 8, 128, generator=gen).to(BF16).to(DEV)
        x = torch.randn(93, vocab, generator=gen).to(DEV)
        lists = (torch.randint(0, vocab, (93 * 50,), generator=gen).to(I32).to(DEV), (torch.arange(94) * 50).to(I32).to(DEV))
        ones = torch.ones(93, device=DEV)

        def call(q=q, cache=cache, table=table, segs=segs, x=x, lists=lists, ones=ones):
            o = ops.paged_tree(q, cache, table, segs, hk, 2040, 40, keys_per_split=256)
            out = torch.empty_like(x)
            return (o, out) + ops.process_logits(x, output=lists, frequency=ones, out=out)

        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = call()
        jobs.append((call, graph, outs, q, x))
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(3):
        for _, _, _, q, x in jobs:
            q.copy_(torch.randn(q.shape, device=DEV))
            x.copy_(torch.randn(x.shape, device=DEV))
        wants = [[t.clone() for t in call()] for call, _, _, _, _ in jobs]
        torch.cuda.synchronize()
        for _ in range(3):
            for (_, graph, _, _, _), stream in zip(jobs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for want, (_, _, outs, _, _) in zip(wants, jobs):
            assert all(torch.equal(a, b) for a, b in zip(want, outs))
    _check()
