"""The decode-step operators as measurable cases: the quantizing cache store, attention over the
quantized cache, attention of drafted token trees, and constrained greedy logits.

``run`` computes a case in its plain form (elementary torch operations in 32 bits, 64 for rotation
angles) or, with ``own`` set, through the public calls of ``furiosa_opt_models_b200.ops``;
``exact`` is the same result from the definition in 64 bits.

The paged cache is the framework's: pages of 16 positions, ``[blocks, 2 (K, V), kv_heads, 16, d]``
BF16, or quantized pages of bytes ``[blocks, 2, kv_heads, 16 * d + 64]``: 16 rows of E4M3 codes,
then the rows' 16 FP32 scales (value = code * scale, scale = largest magnitude / 448).
"""

import math
import random

import torch

own = False

E4M3 = torch.float8_e4m3fn
DEV = "cuda"


def listed():
    return [
        # One decode step's cache write of a batch of 64 (8B-class heads, per-head norms).
        dict(name="store-step", op="store", rows=64, q_heads=32, kv_heads=8, d=128, rotary=128,
             interleaved=False, norm=True, last=40960, theta=1e6),
        # A prompt call of the most rows that a forward takes.
        dict(name="store-prompt", op="store", rows=8192, q_heads=32, kv_heads=8, d=128, rotary=128,
             interleaved=False, norm=True, last=8192, theta=1e6),
        # Interleaved pairs on half of a 64-wide head, an odd chunk of a long context.
        dict(name="store-partial", op="store", rows=1777, q_heads=24, kv_heads=6, d=64, rotary=32,
             interleaved=True, norm=False, last=131072, theta=500000.0),
        # One short conversation: latency alone.
        dict(name="decode-one", op="decode", seqs=1, keys=1000, ragged=False, q_heads=16, kv_heads=8,
             d=128, pattern=1),
        # A serving batch with histories of every length up to 9216.
        dict(name="decode-batch", op="decode", seqs=64, keys=9216, ragged=True, q_heads=32, kv_heads=8,
             d=128, pattern=2),
        # A few very long contexts on a 70B-class layer (eight query heads a key/value head).
        dict(name="decode-long", op="decode", seqs=3, keys=131072, ragged=True, q_heads=64, kv_heads=8,
             d=128, pattern=3),
        # A small verification: four requests, 16 drafted nodes each, BF16 cache.
        dict(name="tree-small", op="tree", seqs=4, nodes=16, cached=2048, ragged=True, quantized=False,
             q_heads=16, kv_heads=8, d=128, pattern=4),
        # A verification step of a serving batch over the quantized cache.
        dict(name="tree-batch", op="tree", seqs=16, nodes=31, cached=8192, ragged=True, quantized=True,
             q_heads=32, kv_heads=8, d=128, pattern=5),
        # Wide trees over long histories: where the matrix work counts.
        dict(name="tree-large", op="tree", seqs=24, nodes=64, cached=16384, ragged=True, quantized=True,
             q_heads=32, kv_heads=8, d=128, pattern=6),
        # One request with penalties and a bias, the adjusted logits wanted too.
        dict(name="logits-one", op="logits", rows=1, vocab=151936, half=False, prompt=700, output=300,
             bias=20, mask=False, write=True, pattern=7),
        # A greedy step of a batch: penalties, biases and grammar masks, only the tokens wanted.
        dict(name="logits-batch", op="logits", rows=64, vocab=128256, half=False, prompt=4096, output=1024,
             bias=50, mask=True, write=False, pattern=8),
        # A large batch of BF16 logits under grammar masks, the adjusted logits handed to a sampler.
        dict(name="logits-grammar", op="logits", rows=256, vocab=151936, half=True, prompt=1024, output=512,
             bias=0, mask=True, write=True, pattern=9),
    ]


HEADS = [(16, 8), (32, 8), (64, 8), (8, 8), (12, 2), (28, 4), (8, 1)]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["store", "decode", "tree", "logits"])
    q_heads, kv_heads = rng.choice(HEADS)
    d = rng.choice([64, 128, 128])
    pattern = rng.randrange(1 << 20)
    if op == "store":
        return dict(op=op, rows=_log(rng, 1, 8192), q_heads=q_heads, kv_heads=kv_heads, d=d,
                    rotary=rng.choice([d, d, d // 2, d // 4]), interleaved=rng.random() < 0.4,
                    norm=rng.random() < 0.5, last=_log(rng, 8192, 131072),
                    theta=rng.choice([10000.0, 500000.0, 1e6]))
    if op == "decode":
        seqs = _log(rng, 1, 64)
        return dict(op=op, seqs=seqs, keys=_log(rng, 1, min(131072, 589824 // seqs)), ragged=rng.random() < 0.7,
                    q_heads=q_heads, kv_heads=kv_heads, d=d, pattern=pattern)
    if op == "tree":
        seqs, nodes = _log(rng, 1, 24), _log(rng, 1, 64)
        return dict(op=op, seqs=seqs, nodes=nodes, cached=_log(rng, 1, 16384), ragged=rng.random() < 0.7,
                    quantized=rng.random() < 0.6, q_heads=q_heads if q_heads < 64 else 32, kv_heads=kv_heads,
                    d=d, pattern=pattern)
    rows = _log(rng, 1, 256)
    return dict(op=op, rows=rows, vocab=_log(rng, 1000, 262144 if rows <= 64 else 151936), half=rng.random() < 0.5,
                prompt=_log(rng, 1, 8192), output=_log(rng, 1, 4096), bias=rng.choice([0, 7, 300]),
                mask=rng.random() < 0.5, write=rng.random() < 0.5, pattern=pattern)


# ---------------------------------------------------------------------------------- sizes of a case


def lengths(case):
    """(rows appended, positions cached before) of every sequence, from the case alone."""
    rng = random.Random(case["pattern"])
    out = []
    for i in range(case["seqs"]):
        if case["op"] == "decode":
            keys = case["keys"] if i == 0 or not case["ragged"] else _log(rng, max(1, case["keys"] // 8), case["keys"])
            out.append((1, keys - 1))
        else:
            n = case["nodes"] if i == 0 or not case["ragged"] else rng.randint((case["nodes"] + 1) // 2, case["nodes"])
            c = case["cached"] if i == 0 or not case["ragged"] else rng.randint(case["cached"] // 4, case["cached"])
            out.append((n, c))
    return out


def list_lengths(case):
    """Token counts of each row's prompt, output and bias lists."""
    rng = random.Random(case["pattern"])
    return [(rng.randint(0, case["prompt"]), rng.randint(0, case["output"]), case["bias"] and rng.randint(0, case["bias"]))
            if case["rows"] > 1 else (case["prompt"], case["output"], case["bias"]) for _ in range(case["rows"])]


def work(case):
    d = case.get("d")
    if case["op"] == "store":
        heads = case["q_heads"] + 2 * case["kv_heads"]
        per_row = heads * d * 2 + case["q_heads"] * d * 2 + 2 * case["kv_heads"] * (d + 4) + 8
        return {"bytes": case["rows"] * per_row, "flops": case["rows"] * heads * d * 8}
    if case["op"] in ("decode", "tree"):
        per_key = 2 * case["kv_heads"] * (d + 4 if case.get("quantized", True) else 2 * d)
        nbytes = flops = 0
        for n, c in lengths(case):
            nbytes += (n + c) * per_key + 2 * n * case["q_heads"] * d * 2 + (n + c + 15) // 16 * 4
            flops += 4 * n * (n + c) * case["q_heads"] * d
        return {"bytes": nbytes, "flops": flops}
    size = 2 if case["half"] else 4
    cells = case["rows"] * case["vocab"]
    lists = sum(4 * p + 4 * o + 8 * b for p, o, b in list_lengths(case))
    return {"bytes": cells * size * (2 if case["write"] else 1) + (cells // 8 if case["mask"] else 0) + lists,
            "flops": 3 * cells}


# ----------------------------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)


def _pages(g, blocks, kv_heads, d):
    """BF16 pages [blocks, 2, kv_heads, 16, d]: keys with a few loud channels, values of order one."""
    cache = _randn(g, blocks, 2, kv_heads, 16, d, dtype=torch.bfloat16)
    loud = 1 + 3 * (torch.rand(kv_heads, 1, d, generator=g, device=DEV) < 0.05)
    cache[:, 0] *= loud.to(torch.bfloat16)
    return cache


def _quantize(cache, out):
    """BF16 pages into quantized pages, a slice of blocks at a time."""
    blocks, _, heads, _, d = cache.shape
    step = max(1, (1 << 26) // (2 * heads * 16 * d))
    for b in range(0, blocks, step):
        x = cache[b:b + step].float()
        scale = x.abs().amax(-1).clamp_min(1e-10) * (1 / 448)
        codes = (x / scale[..., None]).clamp(-448, 448).to(E4M3)
        out[b:b + step, :, :, :16 * d] = codes.view(torch.uint8).flatten(3)
        out[b:b + step, :, :, 16 * d:] = scale.view(torch.uint8)
    return out


def _codes(pages, d):
    return pages[..., :16 * d].view(E4M3).unflatten(-1, (16, d))


def _scales(pages, d):
    return pages[..., 16 * d:].view(torch.float32)


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    d = case.get("d")
    if case["op"] == "store":
        rows, heads = case["rows"], case["q_heads"] + 2 * case["kv_heads"]
        s["qkv"] = _randn(g, rows, heads * d).mul_(2).bfloat16()
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"], s["k_norm"] = ((1 + 0.3 * _randn(g, d)).bfloat16() for _ in range(2))
        if rows <= 256:  # a step: every row another sequence
            s["positions"] = torch.randint(0, case["last"], (rows,), generator=g, device=DEV, dtype=torch.int32)
        else:  # a prompt chunk that ends at the last position
            first = max(0, case["last"] - rows)
            s["positions"] = torch.arange(first, first + rows, device=DEV, dtype=torch.int32)
        j = torch.arange(0, case["rotary"], 2, device=DEV, dtype=torch.float64)
        s["inv_freq"] = (case["theta"] ** (-j / case["rotary"])).float()
        blocks = (rows + 15) // 16 + 3
        s["slots"] = torch.randperm(blocks * 16, generator=g, device=DEV)[:rows].int()
        s["pages"] = _quantize(_pages(g, blocks, case["kv_heads"], d),
                               torch.empty(blocks, 2, case["kv_heads"], 16 * d + 64, dtype=torch.uint8, device=DEV))
    elif case["op"] in ("decode", "tree"):
        segs, row, start = [], 0, 0
        for n, c in lengths(case):
            nb = (n + c + 15) // 16
            segs.append((row, n, c, start, nb))
            row, start = row + n, start + nb
        s["max_keys"] = max(n + c for _, n, c, _, _ in segs)
        s["max_len"] = max(n for _, n, _, _, _ in segs)
        s["segments"] = torch.tensor(segs, dtype=torch.int32).to(DEV)
        blocks = start + 2
        s["table"] = torch.randperm(blocks, generator=g, device=DEV)[:start].int()
        s["q"] = _randn(g, row, case["q_heads"], d).mul_(1.5).bfloat16()
        s["cache"] = _pages(g, blocks, case["kv_heads"], d)
        if case.get("quantized", True):
            pages = torch.empty(blocks, 2, case["kv_heads"], 16 * d + 64, dtype=torch.uint8, device=DEV)
            s["cache"] = _quantize(s["cache"], pages)
        if case["op"] == "tree":
            # Random trees: a node's parent is one of the nodes before it, the first is the root.
            rng = random.Random(int(seed))
            words = (s["max_len"] + 31) // 32
            mask = []
            for _, n, _, _, _ in segs:
                seen = []
                for i in range(n):
                    seen.append((seen[rng.randrange(max(0, i - 8), i)] if i else 0) | 1 << i)
                mask += [[(b >> 32 * w) & 0xFFFFFFFF for w in range(words)] for b in seen]
            s["mask"] = torch.tensor(mask, dtype=torch.int64).to(torch.int32).to(DEV)
    else:
        rows, vocab = case["rows"], case["vocab"]
        s["logits"] = _randn(g, rows, vocab).mul_(3)
        if case["half"]:
            s["logits"] = s["logits"].bfloat16()
        counts = list_lengths(case)
        for name, k in (("prompt", 0), ("output", 1), ("bias", 2)):
            total = sum(c[k] for c in counts)
            # Token frequencies fall off as in text: most repeats are of few tokens.
            u = torch.rand(total, generator=g, device=DEV)
            s[name] = (vocab * u ** 3).int().clamp_(0, vocab - 1)
            starts = [0]
            for c in counts:
                starts.append(starts[-1] + c[k])
            s[name + "_starts"] = torch.tensor(starts, dtype=torch.int32).to(DEV)
        s["bias_values"] = _randn(g, s["bias"].numel()).mul_(4)
        if case["bias"]:  # a request's biases name each token once
            s["bias"] = torch.cat([torch.randperm(vocab, generator=g, device=DEV)[:c[2]] for c in counts]).int()
        s["repetition"] = 1 + torch.rand(rows, generator=g, device=DEV) * 0.5
        s["frequency"] = torch.rand(rows, generator=g, device=DEV) * 0.5
        s["presence"] = torch.rand(rows, generator=g, device=DEV)
        s["allowed"] = None
        if case["mask"]:
            words = (vocab + 31) // 32
            full = lambda: torch.randint(-2**31, 2**31, (rows, words), generator=g, device=DEV, dtype=torch.int64).int()  # noqa: E731
            free = full() | full() | full() | full()  # inside a string: nearly every token
            tight = full() & full() & full() & full() & full() & full() & full() & full()  # a key or a bracket
            pick = torch.rand(rows, 1, generator=g, device=DEV)
            s["allowed"] = torch.where(pick < 0.5, free, tight)
            if rows > 8:
                s["allowed"][rows // 2] = 0  # a dead end of the grammar
    return s


# ------------------------------------------------------------------------------------ plain forms


def _store_plain(s):
    c = s["case"]
    d, hq, hk, rot = c["d"], c["q_heads"], c["kv_heads"], c["rotary"]
    rows = s["qkv"].shape[0]
    x = s["qkv"].float().view(rows, hq + 2 * hk, d)
    qk, v = x[:, :hq + hk], x[:, hq + hk:]
    if s["q_norm"] is not None:
        w = torch.cat([s["q_norm"].expand(hq, d), s["k_norm"].expand(hk, d)]).float()
        qk = qk / (qk.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
    angle = s["positions"].double()[:, None, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float(), angle.sin().float()
    head, rest = qk[..., :rot], qk[..., rot:]
    if c["interleaved"]:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        head = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    qk = torch.cat([head, rest], -1)
    kv = torch.stack([qk[:, hq:], v], 1)  # [rows, 2, hk, d]
    scale = kv.abs().amax(-1).clamp_min(1e-10) * (1 / 448)
    codes = (kv / scale[..., None]).clamp(-448, 448).to(E4M3)
    block, at = s["slots"].long() // 16, s["slots"].long() % 16
    byte = s["pages"][..., :16 * d].unflatten(-1, (16, d))
    byte[block, :, :, at] = codes.view(torch.uint8)
    _scales(s["pages"], d)[block, :, :, at] = scale
    return qk[:, :hq].bfloat16(), _codes(s["pages"], d), _scales(s["pages"], d)


def _visible(s, n, keys):
    """[sequences, n, keys]: which keys each of a sequence's rows sees."""
    seg = s["segments"].long()
    at = torch.arange(keys, device=DEV) - seg[:, 2, None, None]  # place among the appended rows
    row = torch.arange(n, device=DEV)[None, :, None]
    real = (row < seg[:, 1, None, None]) & (at < seg[:, 1, None, None])
    if "mask" not in s:
        return real & (at <= row)
    rows = (seg[:, :1] + torch.arange(n, device=DEV)).clamp_max(s["q"].shape[0] - 1)
    words = s["mask"][rows].long() & 0xFFFFFFFF  # [sequences, n, words]
    inside = at.clamp(0, n - 1).expand(-1, n, -1)
    bit = (words.gather(2, inside >> 5) >> (inside & 31)) & 1
    return real & ((at < 0) | (bit == 1))


def _attend_plain(s):
    c = s["case"]
    d, hq, hk = c["d"], c["q_heads"], c["kv_heads"]
    seg, n, keys = s["segments"].long(), s["max_len"], s["max_keys"]
    nb = (keys + 15) // 16
    at = (seg[:, 3:4] + torch.arange(nb, device=DEV)).clamp_max(s["table"].numel() - 1)
    pages = s["cache"][s["table"].long()[at]]  # [sequences, nb, 2, hk, ...]
    if s["cache"].dtype == torch.uint8:
        kv = _codes(pages, d).float() * _scales(pages, d)[..., None]
    else:
        kv = pages.float()
    kv = kv.permute(2, 0, 3, 1, 4, 5).flatten(3, 4)[..., :keys, :]  # [2, sequences, hk, keys, d]
    rows = (seg[:, :1] + torch.arange(n, device=DEV)).clamp_max(s["q"].shape[0] - 1)
    q = s["q"][rows].float().unflatten(2, (hk, hq // hk)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = q @ kv[0].transpose(-1, -2) * d ** -0.5  # [sequences, hk, group * n, keys]
    seen = _visible(s, n, keys)[:, None, None].expand(-1, 1, hq // hk, -1, -1).flatten(2, 3)
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = torch.exp(score - top)
    o = p @ kv[1] / p.sum(-1, keepdim=True).clamp_min(1e-37)
    o = o.unflatten(2, (hq // hk, n)).permute(0, 3, 1, 2, 4).flatten(2, 3)  # [sequences, n, hq, d]
    return o[torch.arange(n, device=DEV) < seg[:, 1:2]].bfloat16()


def _logits_plain(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    row = torch.arange(rows, device=DEV)
    of = lambda name: torch.repeat_interleave(row, s[name + "_starts"].diff().long(), output_size=s[name].numel())  # noqa: E731
    cell = lambda name: of(name) * vocab + s[name].long()  # noqa: E731
    count = torch.zeros(rows * vocab, device=DEV)
    count.scatter_add_(0, cell("output"), torch.ones(s["output"].numel(), device=DEV))
    seen = count > 0
    listed_ = seen.scatter(0, cell("prompt"), torch.ones(s["prompt"].numel(), dtype=torch.bool, device=DEV))
    count, seen, listed_ = (t.view(rows, vocab) for t in (count, seen, listed_))
    r = s["repetition"][:, None]
    x = torch.where(listed_, torch.where(x > 0, x / r, x * r), x)
    x = torch.where(seen, x - s["frequency"][:, None] * count, x)
    x = torch.where(seen, x - s["presence"][:, None], x)
    if s["bias"].numel():
        x = x.flatten().scatter_add(0, cell("bias"), s["bias_values"]).view(rows, vocab)
    if s["allowed"] is not None:
        col = torch.arange(vocab, device=DEV)
        x = x.masked_fill((s["allowed"][:, col >> 5] >> (col & 31)) & 1 == 0, -math.inf)
    best = x.amax(-1)
    # The first of equal maxima; a row with no token left has none.
    first = torch.where(x == best[:, None], torch.arange(vocab, device=DEV), vocab).amin(-1)
    first = torch.where(best == -math.inf, -1, first).int()
    return (first, best, x.to(s["logits"].dtype)) if s["case"]["write"] else (first, best)


def run(s):
    c = s["case"]
    if own:
        from furiosa_opt_models_b200 import ops

        if c["op"] == "store":
            cache = ops.QuantizedCache(s["pages"], c["d"])
            q = ops.qk_norm_rope_cache(s["qkv"], c["q_heads"], c["kv_heads"], c["d"], s["q_norm"], s["k_norm"], 1e-6,
                                       s["positions"], s["inv_freq"], 1.0, cache, s["slots"],
                                       rotary_dim=c["rotary"], interleaved=c["interleaved"])
            return q, cache.codes.view(E4M3), cache.scales
        if c["op"] == "decode":
            return ops.paged_decode(s["q"], ops.QuantizedCache(s["cache"], c["d"]), s["table"], s["segments"],
                                    c["kv_heads"], s["max_keys"])
        if c["op"] == "tree":
            cache = ops.QuantizedCache(s["cache"], c["d"]) if c["quantized"] else s["cache"]
            return ops.paged_tree(s["q"], cache, s["table"], s["segments"], c["kv_heads"], s["max_keys"], s["max_len"],
                                  mask=s["mask"])
        out = torch.empty_like(s["logits"]) if c["write"] else None
        bias = (s["bias"], s["bias_values"], s["bias_starts"]) if c["bias"] else None
        first, best = ops.process_logits(s["logits"], prompt=(s["prompt"], s["prompt_starts"]),
                                         output=(s["output"], s["output_starts"]), repetition=s["repetition"],
                                         frequency=s["frequency"], presence=s["presence"], bias=bias,
                                         allowed=s["allowed"], out=out)
        return (first, best, out) if c["write"] else (first, best)
    return {"store": _store_plain, "decode": _attend_plain, "tree": _attend_plain, "logits": _logits_plain}[c["op"]](s)


# -------------------------------------------------------------------------- the definitions, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"store": _store_exact, "decode": _attend_exact, "tree": _attend_exact, "logits": _logits_exact}[case["op"]](case, s)


def _store_exact(c, s):
    d, hq, hk, rot = c["d"], c["q_heads"], c["kv_heads"], c["rotary"]
    x = s["qkv"].double().view(-1, hq + 2 * hk, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]

    def turn(h, w):
        if w is not None:
            h = h * (h.pow(2).sum(-1, keepdim=True) / d + 1e-6).pow(-0.5) * w.double()
        pairs = range(rot // 2)
        i = torch.tensor([2 * j if c["interleaved"] else j for j in pairs], device=DEV)
        j = torch.tensor([2 * j + 1 if c["interleaved"] else j + rot // 2 for j in pairs], device=DEV)
        # A pair is a complex number, turned by the position times its frequency.
        z = torch.complex(h[..., i], h[..., j])
        z = z * torch.polar(torch.ones_like(z.real), (s["positions"].double()[:, None] * s["inv_freq"].double())[:, None].expand_as(z.real))
        h = h.clone()
        h[..., i], h[..., j] = z.real, z.imag
        return h

    q, k = turn(q, s["q_norm"]), turn(k, s["k_norm"])
    codes, scales = _codes(s["pages"], d).double(), _scales(s["pages"], d).double()
    block, at = torch.div(s["slots"].long(), 16, rounding_mode="floor"), s["slots"].long() % 16
    for which, y in ((0, k), (1, v)):
        scale = y.abs().max(-1).values.clamp_min(1e-10) / 448
        scales[block, which, :, at] = scale
        codes[block, which, :, at] = (y / scale[..., None]).float().clamp(-448, 448).to(E4M3).double()
    return q, codes, scales


def _attend_exact(c, s):
    d, hq, hk = c["d"], c["q_heads"], c["kv_heads"]
    total = sum(n * (n + k) for n, k in lengths(c))
    if total * hq * d > 4e11:
        return None  # too long in 64 bits
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for row, n, cached, start, nb in s["segments"].tolist():
        pages = s["cache"][s["table"][start:start + nb].long()]
        if pages.dtype == torch.uint8:
            pages = _codes(pages, d).double() * _scales(pages, d).double()[..., None]
        seen = torch.ones(n, n + cached, dtype=torch.bool, device=DEV)
        if c["op"] == "tree":
            j = torch.arange(n, device=DEV)
            seen[:, cached:] = (s["mask"][row:row + n].long()[:, j // 32] >> (j % 32)) & 1 == 1
        for h in range(hk):
            k, v = (pages[:, w, h].double().reshape(-1, d)[:n + cached] for w in (0, 1))
            for g in range(h * (hq // hk), (h + 1) * (hq // hk)):
                score = s["q"][row:row + n, g].double() @ k.T / math.sqrt(d)
                p = torch.softmax(score.masked_fill(~seen, -math.inf), -1)
                out[row:row + n, g] = p @ v
    return out


def _logits_exact(c, s):
    x = s["logits"].double()
    rows, vocab = x.shape
    if rows * vocab > 5e7:
        return None
    for r in range(rows):
        cut = lambda name: s[name][int(s[name + "_starts"][r]):int(s[name + "_starts"][r + 1])].long()  # noqa: E731
        made = torch.bincount(cut("output"), minlength=vocab)
        named = made.clone()
        named[cut("prompt")] += 1
        y = x[r]
        rep = s["repetition"][r].double()
        y = torch.where(named > 0, torch.where(y > 0, y / rep, y * rep), y)
        y = y - s["frequency"][r].double() * made - s["presence"][r].double() * (made > 0)
        lo, hi = int(s["bias_starts"][r]), int(s["bias_starts"][r + 1])
        y[s["bias"][lo:hi].long()] += s["bias_values"][lo:hi].double()
        if s["allowed"] is not None:
            bits = (s["allowed"][r].long()[:, None] >> torch.arange(32, device=DEV)) & 1
            y[bits.flatten()[:vocab] == 0] = -math.inf
        x[r] = y
    best = x.max(-1).values
    return (None, best, x) if c["write"] else (None, best)
