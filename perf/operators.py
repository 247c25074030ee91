"""Operators around the paged cache that a serving program calls beside append,
attention and argmax: rotary positions on the way into the cache, 8-bit pools
with a scale for each block and KV head, eviction by accumulated attention
weight, and penalties, biases and masks on logits.

A case is a dict with an "op" and that op's sizes.  ``prepare`` makes what a
serving program holds before the call, ``run`` makes one pass -- in plain torch,
or through the library where ``own`` is set -- and ``exact`` repeats it in
float64, written apart.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
BS = 16  # tokens per block
TOP = {"int8": 127.0, "fp8": 448.0}
ELEM = {"f32": 4, "bf16": 2, "fp8": 1, "int8_block": 1, "fp8_block": 1}
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed() -> list[dict]:
    heads = dict(hq=32, hkv=8, d=128)  # Llama-3-8B's attention layer
    return [
        # one layer's rotation and append in a decode step of 64 sequences at
        # long positions, banded frequencies: latency
        dict(name="rope_step", op="rope_append", tokens=64, far=131072, rot=128, pairs="half",
             kv="bf16", magnitude=1.0, **heads),
        # the prompt of one request of 8,192 tokens, the same layer
        dict(name="rope_prompt", op="rope_append", tokens=8192, far=8192, rot=128, pairs="half",
             kv="bf16", magnitude=1.0, **heads),
        # interleaved pairs over half of a 64-wide head, stretched to a million
        # positions: the keys of a long document, rotated by themselves
        dict(name="rope_partial", op="rope", tokens=16384, heads=16, d=64, far=1 << 20, rot=32,
             pairs="interleaved", magnitude=1.2),
        # one user's chat turn over a block-scaled cache, its step's row appended
        dict(name="block_single", op="block_decode", seqs=1, lo=300, hi=300, kv="fp8_block",
             append=True, **heads),
        # a decode step of 64 sequences, append and attention
        dict(name="block_batch", op="block_decode", seqs=64, lo=512, hi=4096, kv="int8_block",
             append=True, **heads),
        # long documents, few sequences
        dict(name="block_long", op="block_decode", seqs=8, lo=16384, hi=65536, kv="fp8_block",
             append=False, **heads),
        # a 512-token chunk of 8 long prompts, appended and attended
        dict(name="block_chunk", op="block_prefill", seqs=8, new=512, cached=1536,
             kv="int8_block", **heads),
        # the 64-sequence decode step that also adds up each token's weight
        dict(name="weights_step", op="weights", seqs=64, lo=512, hi=4096, kv="bf16", **heads),
        # 16 sequences cut to 1,024 tokens in 8 layers
        dict(name="evict_batch", op="evict", layers=8, seqs=16, lo=1500, hi=4096, budget=1024,
             sinks=4, recent=256, kv="bf16", hkv=8, d=128),
        # one long sequence cut to a quarter in 2 layers of a block-scaled cache
        dict(name="evict_long", op="evict", layers=2, seqs=1, lo=32768, hi=32768, budget=8192,
             sinks=16, recent=1024, kv="int8_block", hkv=8, d=128),
        # one request with a grammar over a small vocabulary: latency
        dict(name="logits_single", op="logits", rows=1, vocab=32000, history=300, biases=8,
             mask=True),
        # 64 requests at Llama-3's vocabulary, a few thousand tokens behind each
        dict(name="logits_batch", op="logits", rows=64, vocab=128256, history=2048, biases=64,
             mask=True),
    ]


def _log(rng, lo: int, hi: int) -> int:
    """An integer spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    op = rng.choice(["rope_append", "rope", "block_decode", "block_decode", "block_prefill",
                     "weights", "evict", "logits"])
    hkv, group, d = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 4, 8]), rng.choice([64, 128])
    heads = dict(hq=hkv * group, hkv=hkv, d=d)
    pairs = rng.choice(["half", "interleaved"])
    if op == "rope_append":
        rot = rng.choice([d, d, d // 2, 2 * rng.randint(1, d // 2)])
        return dict(op=op, tokens=_log(rng, 1, 8192), far=_log(rng, 16, 1 << 20), rot=rot,
                    pairs=pairs, kv=rng.choice(["bf16", "f32", "fp8"]),
                    magnitude=rng.choice([1.0, round(rng.uniform(0.9, 1.4), 3)]), **heads)
    if op == "rope":
        d = rng.choice([32, 64, 80, 128, 192])
        rot = rng.choice([d, d // 2, 2 * rng.randint(1, d // 2)])
        return dict(op=op, tokens=_log(rng, 1, 16384), heads=rng.randint(1, 16), d=d,
                    far=_log(rng, 16, 1 << 20), rot=rot, pairs=pairs,
                    magnitude=rng.choice([1.0, round(rng.uniform(0.9, 1.4), 3)]))
    if op in ("block_decode", "weights"):
        fmt = rng.choice(["int8_block", "fp8_block"] if op == "block_decode" else
                         ["bf16", "bf16", "f32", "int8_block", "fp8_block"])
        hi = _log(rng, 16, 65536 if op == "block_decode" else 16384)
        most = 5.0e8 if op == "block_decode" else 2.0e8  # pool elements
        seqs = _log(rng, 1, max(1, min(64, int(most / (2 * hkv * d * hi)))))
        case = dict(op=op, seqs=seqs, lo=_log(rng, max(1, hi // 16), hi), hi=hi, kv=fmt, **heads)
        return dict(case, append=rng.random() < 0.5) if op == "block_decode" else case
    if op == "block_prefill":
        return dict(op=op, seqs=_log(rng, 1, 8), new=_log(rng, 2, 512),
                    cached=rng.choice([0, _log(rng, 1, 1536)]),
                    kv=rng.choice(["int8_block", "fp8_block"]), **heads)
    if op == "evict":
        hi = _log(rng, 32, 4096)
        budget = _log(rng, 8, max(8, hi // 2))
        recent = rng.randint(0, budget // 2)
        return dict(op=op, layers=rng.randint(1, 4), seqs=_log(rng, 1, 16),
                    lo=_log(rng, max(1, hi // 8), hi), hi=hi, budget=budget,
                    sinks=rng.randint(0, min(16, budget - recent)), recent=recent,
                    kv=rng.choice(["bf16", "f32", "fp8", "int8_block", "fp8_block"]), hkv=hkv,
                    d=d)
    return dict(op=op, rows=_log(rng, 1, 64), vocab=_log(rng, 1000, 128256),
                history=_log(rng, 1, 2048), biases=rng.choice([0, _log(rng, 1, 64)]),
                mask=rng.random() < 0.6)


# ---- inputs ------------------------------------------------------------------------

def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(1_000_003 * (seed % 1_000_000) + 29)


def _randn(shape, g, dtype=torch.float32) -> torch.Tensor:
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _lens(case: dict) -> list[int]:
    """Context lengths, uniform in [lo, hi]: part of the case, so that every
    seed of a case is the same amount of work."""
    if case["op"] == "block_prefill":
        return [case["cached"] + case["new"]] * case["seqs"]
    g = torch.Generator().manual_seed(7 * case["seqs"] + 31 * case["hi"] + case["lo"])
    return torch.randint(case["lo"], case["hi"] + 1, (case["seqs"],), generator=g).tolist()


def _tables(lens: list[int], spare: int, g):
    """Block tables over randomly permuted blocks, the lengths, the pool's block
    count and ``spare`` blocks that no table holds."""
    need = [-(-n // BS) for n in lens]
    nb = sum(need) + spare + 8
    perm = torch.randperm(nb, generator=g, device=DEV).to(torch.int32)
    tab = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        tab[b, :n] = perm[at:at + n]
        at += n
    return tab, torch.tensor(lens, dtype=torch.int32, device=DEV), nb, perm[at:at + spare]


def _frequencies(rot: int, far: int) -> torch.Tensor:
    """Angles per position of the rot / 2 pairs: base 500,000, stretched evenly
    beyond 8,192 positions in the pairs that turn slowly (a program keeps the
    table that its configuration gives)."""
    f = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    factor = max(1.0, far / 8192)
    wave = 2 * math.pi / f
    smooth = ((8192 / wave - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
    return ((1 - smooth) * f / factor + smooth * f).to(DEV)


def _block_pool(x: torch.Tensor, fmt: str):
    """Blocks [.., hkv, BS, d] as bytes and one scale per (block, KV head)."""
    amax = x.abs().amax((-1, -2))
    if fmt == "int8_block":
        s = amax / 127.0
        y = (x.double() / s.double()[..., None, None]).round()
        return y.clamp(-127, 127).to(torch.int8).view(torch.uint8), s
    s = torch.exp2(torch.ceil(torch.log2(amax.double() / 448.0))).float()
    return (x / s[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8), s


def _pools(shape, fmt: str, g):
    """K and V pools [.., hkv, BS, d]; keys with a few large channels.  The scale
    pools of the 8-bit formats, else None."""
    out, scales = [], []
    for name in "kv":
        x = _randn(shape, g)
        if name == "k":
            x = x * torch.exp(0.4 * _randn((shape[-3], 1, shape[-1]), g))
        if fmt in ("int8_block", "fp8_block"):
            x, s = _block_pool(x, fmt)
        elif fmt == "fp8":
            s = x.abs().amax(-1) / 448.0
            x = (x / s[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        else:
            x, s = x.to(TORCH[fmt]), None
        out.append(x)
        scales.append(s)
    return (*out, *scales)


def prepare(case: dict, seed: int) -> dict:
    g = _gen(seed)
    st, op = dict(case=case), case["op"]
    if op in ("rope_append", "rope"):
        t, d = case["tokens"], case["d"]
        st["pos"] = torch.randint(0, case["far"], (t,), generator=g, device=DEV,
                                  dtype=torch.int32)
        st["freq"] = _frequencies(case["rot"], case["far"])
        if op == "rope":
            st["x"] = _randn((t, case["heads"], d), g)
            st["out"] = torch.empty_like(st["x"])
            return st
        hq, hkv = case["hq"], case["hkv"]
        st["q"], st["kn"], st["vn"] = (_randn((t, h, d), g) for h in (hq, hkv, hkv))
        nb = -(-t // BS) + 8
        dt = TORCH.get(case["kv"], torch.uint8)
        st["k"], st["v"] = (torch.zeros((nb, hkv, BS, d), dtype=dt, device=DEV) for _ in range(2))
        st["ks"], st["vs"] = ((torch.zeros((nb, hkv, BS), device=DEV) for _ in range(2))
                              if case["kv"] == "fp8" else (None, None))
        st["slots"] = torch.randperm(nb * BS, generator=g, device=DEV)[:t].to(torch.int64)
        st["out"] = torch.empty_like(st["q"])
    elif op in ("block_decode", "block_prefill", "weights"):
        lens, hq, hkv, d = _lens(case), case["hq"], case["hkv"], case["d"]
        st["tab"], st["ctx"], nb, _ = _tables(lens, 0, g)
        st["k"], st["v"], st["ks"], st["vs"] = _pools((nb, hkv, BS, d), case["kv"], g)
        rows = case["seqs"] * case.get("new", 1)
        st["q"] = _randn((rows, hq, d), g)
        st["out"] = torch.empty_like(st["q"])
        st["start"] = torch.arange(0, rows + 1, case.get("new", 1), dtype=torch.int32, device=DEV)
        if op == "weights":
            st["w"] = torch.exp(2.0 * _randn((nb, hkv, BS), g) - 4.0)
        elif op == "block_prefill" or case["append"]:
            st["kn"], st["vn"] = (_randn((rows, hkv, d), g) for _ in range(2))
    elif op == "evict":
        lens, n, hkv, d = _lens(case), case["layers"], case["hkv"], case["d"]
        left = [-(-min(x, case["budget"]) // BS) for x in lens]
        st["tab"], st["ctx"], nb, spare = _tables(lens, sum(left), g)
        st["to"] = torch.full((len(lens), max(left)), -1, dtype=torch.int32, device=DEV)
        at = 0
        for b, m in enumerate(left):
            st["to"][b, :m] = spare[at:at + m]
            at += m
        st["k"], st["v"], st["ks"], st["vs"] = _pools((n, nb, hkv, BS, d), case["kv"], g)
        st["w"] = torch.exp(2.0 * _randn((n, nb, hkv, BS), g) - 4.0)
    else:
        r, v = case["rows"], case["vocab"]
        st["x"] = 3.0 * _randn((r, v), g)
        st["out"] = torch.empty_like(st["x"])
        # ragged histories that repeat themselves, a part of each the prompt
        c = torch.Generator().manual_seed(3 * r + case["history"])
        n = torch.randint(max(1, case["history"] // 2), case["history"] + 1, (r,), generator=c)
        st["start"] = torch.cat([torch.zeros(1), n.cumsum(0)]).to(torch.int32).to(DEV)
        st["prompt"] = (n // 3).to(torch.int32).to(DEV)
        words = torch.rand((int(n.sum()),), generator=g, device=DEV)
        st["history"] = (words ** 3 * v).to(torch.int32).clamp(max=v - 1)
        st["rep"] = 1.0 + 0.3 * torch.rand((r,), generator=g, device=DEV)
        st["freq"], st["pres"] = (0.5 * torch.rand((r,), generator=g, device=DEV)
                                  for _ in range(2))
        if case["biases"]:
            m = min(case["biases"], v)
            at = torch.rand((r, v), generator=g, device=DEV).argsort(1)[:, :m]
            st["bias_ids"] = at.reshape(-1).to(torch.int32)
            st["bias"] = 2.0 * _randn((r * m,), g)
            st["bias_start"] = torch.arange(0, r * m + 1, m, dtype=torch.int32, device=DEV)
        if case["mask"]:
            words = -(-v // 32)
            st["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (r, words), generator=g, device=DEV,
                                          dtype=torch.int64).to(torch.int32)
    return st


# ---- one pass ------------------------------------------------------------------------

def _rotate(x, pos, freq, pairs: str, magnitude: float):
    """Plain rotation of x [T, H, D]: angles in 64 bits, products in 32."""
    angle = pos.double()[:, None] * freq
    c, s = ((f.float() * magnitude)[:, None] for f in (angle.cos(), angle.sin()))
    n = freq.numel()
    if pairs == "half":
        a, b, rest = x[..., :n], x[..., n:2 * n], x[..., 2 * n:]
        return torch.cat([a * c - b * s, b * c + a * s, rest], -1)
    a, b, rest = x[..., 0:2 * n:2], x[..., 1:2 * n:2], x[..., 2 * n:]
    return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), rest], -1)


def _store(pool, scale, slots, rows):
    """Rows [T, hkv, d] to slots of a pool, in its format."""
    blk, row = slots // BS, slots % BS
    if scale is None:
        pool[blk, :, row] = rows.to(pool.dtype)
        return
    amax = rows.abs().amax(-1, keepdim=True)
    y = (rows * (448.0 / amax)).clamp(-448, 448)
    pool.view(torch.float8_e4m3fn)[blk, :, row] = y.to(torch.float8_e4m3fn)
    scale[blk, :, row] = (amax / 448.0)[..., 0]


def _byte_values(b: torch.Tensor, fmt: str) -> torch.Tensor:
    """Stored bytes as the numbers they are (before the scale)."""
    return b.view(torch.int8 if fmt.startswith("int8") else torch.float8_e4m3fn).float()


def _values(pool, scale, fmt: str) -> torch.Tensor:
    """A pool's (or some of its blocks') rows in 32 bits."""
    if scale is None:
        return pool.float()
    s = scale[..., None, None] if fmt.endswith("block") else scale[..., None]
    return _byte_values(pool, fmt) * s


def _bytes(x, s, fmt: str) -> torch.Tensor:
    """x / s rounded to the format's bytes (in 64 bits: borders), 0 where s is."""
    y = torch.where(s > 0, x.double() / s.double(), 0.0)
    if fmt.startswith("int8"):
        return y.round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
    return y.float().clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _scale_of(amax, fmt: str) -> torch.Tensor:
    if fmt.startswith("int8"):
        return amax / 127.0
    return torch.exp2(torch.ceil(torch.log2(amax.double() / 448.0))).float()


def _append_blocks(pool, scale, new, st, fmt: str) -> None:
    """The last new tokens of every sequence into their blocks: the block's
    scale grows to hold them, its older rows are brought to it."""
    ctx, start, tab = st["ctx"].long(), st["start"].long(), st["tab"].long()
    n = start[1:] - start[:-1]
    first = ctx - n
    j = torch.arange(-(-(st["case"].get("new", 1) + BS - 1) // BS), device=DEV)
    blocks = first[:, None] // BS + j                                      # [B, J]
    pos = blocks[..., None] * BS + torch.arange(BS, device=DEV)             # [B, J, 16]
    fresh = (pos >= first[:, None, None]) & (pos < ctx[:, None, None])
    old = pos < first[:, None, None]
    hit = fresh.any(-1)                                                    # blocks with a new row
    ids = tab.gather(1, blocks.clamp(max=tab.shape[1] - 1))
    src = (start[:-1, None, None] + pos - first[:, None, None]).clamp(0, new.shape[0] - 1)
    ids, src, fresh, old = ids[hit], src[hit], fresh[hit], old[hit]         # [N], [N, 16]
    rows = new[src].transpose(1, 2)                                        # [N, hkv, 16, d]
    fresh, old = fresh[:, None, :, None], old[:, None, :, None]
    amax = torch.where(fresh, rows.abs(), 0.0).amax((-1, -2))
    s_old = torch.where(old.any(2)[:, :, 0], scale[ids], 0.0)
    s_new = torch.maximum(s_old, _scale_of(amax, fmt))
    have, wide = pool[ids], s_new[..., None, None]
    kept = _bytes(_byte_values(have, fmt).double() * s_old.double()[..., None, None], wide, fmt)
    pool[ids] = torch.where(fresh, _bytes(rows, wide, fmt), torch.where(old, kept, have))
    scale[ids] = s_new


def _attend(st, weights: bool = False):
    """Softmax attention of every query row over its sequence's cache; row i of
    a sequence's n sees the positions up to its own."""
    case = st["case"]
    hq, hkv, d, fmt = case["hq"], case["hkv"], case["d"], case["kv"]
    B, n = case["seqs"], case.get("new", 1)
    ids = st["tab"].long().clamp(min=0)
    L = ids.shape[1] * BS

    def rows(pool, scale):
        x = _values(pool[ids], None if scale is None else scale[ids], fmt)
        return x.transpose(1, 2).reshape(B, hkv, L, d)

    q = st["q"].view(B, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(B, hkv, -1, d)
    s = (q @ rows(st["k"], st["ks"]).transpose(2, 3).contiguous()) / math.sqrt(d)
    s = s.view(B, hkv, hq // hkv, n, L)
    last = (st["ctx"].long() - n)[:, None] + torch.arange(n, device=DEV)
    seen = torch.arange(L, device=DEV) <= last[..., None]                   # [B, n, L]
    s = torch.where(seen[:, None, None], s, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = p.view(B, hkv, -1, L) @ rows(st["v"], st["vs"])
    o = o.view(B, hkv, hq // hkv, n, d).permute(0, 3, 1, 2, 4).reshape(-1, hq, d)
    return (o, p.sum((2, 3))) if weights else o


def _evict_plain(st):
    case, ctx, tab = st["case"], st["ctx"].long(), st["tab"].long()
    n, B, hkv, fmt = case["layers"], case["seqs"], case["hkv"], case["kv"]
    budget, ids = case["budget"], tab.clamp(min=0)
    L = tab.shape[1] * BS
    # the largest weights beside the first and the last tokens, ties to the
    # lower position
    w = st["w"][:, ids].transpose(2, 3).reshape(n, B, hkv, L)
    pos = torch.arange(L, device=DEV)
    held = (pos < case["sinks"]) | (pos >= ctx[:, None] - case["recent"])
    key = torch.where(held[:, None], math.inf, w)
    key = torch.where((pos < ctx[:, None])[:, None], key, -math.inf)
    order = key.sort(dim=-1, descending=True, stable=True)[1][..., :budget]
    lens = ctx.clamp(max=budget)
    take = torch.arange(budget, device=DEV) < lens[:, None]                # [B, budget]
    pad = budget - order.shape[-1]
    order = torch.nn.functional.pad(order, (0, pad)) if pad > 0 else order
    order = torch.where(take[:, None], order, L).sort(-1)[0]
    keep = torch.where(take[:, None], order, -1).to(torch.int32)
    # rows to their new places
    lay = torch.arange(n, device=DEV)[:, None, None, None]
    b = torch.arange(B, device=DEV)[:, None, None]
    h = torch.arange(hkv, device=DEV)[:, None]
    p = order.clamp(max=L - 1)
    sb, sr = tab[b, p // BS].clamp(min=0), p % BS                           # [n, B, hkv, budget]
    j = torch.arange(budget, device=DEV)
    db = st["to"].long()[:, (j // BS).clamp(max=st["to"].shape[1] - 1)]    # [B, budget]
    on = take[:, None].expand(n, B, hkv, budget)
    at = [x.expand(n, B, hkv, budget)[on] for x in (lay, db[:, None], h, j % BS)]
    for pool, scale in ((st["k"], st["ks"]), (st["v"], st["vs"])):
        x = pool[lay, sb, h, sr]
        if scale is not None and fmt.endswith("block"):
            s = torch.where(on, scale[lay, sb, h], 0.0)
            s = torch.nn.functional.pad(s, (0, -budget % BS))
            s_new = s.view(n, B, hkv, -1, BS).amax(-1)                     # [n, B, hkv, blocks]
            wide = s_new.repeat_interleave(BS, -1)[..., :budget, None]
            x = _bytes(_byte_values(x, fmt).double() * s[..., :budget, None].double(), wide, fmt)
            some = on[..., ::BS]
            to = [y.expand_as(some)[some] for y in
                  (lay, db[:, None, ::BS], h)]
            scale[to[0], to[1], to[2]] = s_new[some]
        elif scale is not None:
            scale[at[0], at[1], at[2], at[3]] = scale[lay, sb, h, sr][on]
        pool[at[0], at[1], at[2], at[3]] = x[on]
    st["w"][at[0], at[1], at[2], at[3]] = st["w"][lay, sb, h, sr][on]
    return keep, lens.to(torch.int32)


def _logits_plain(st):
    x, (r, v) = st["x"], st["x"].shape
    start, hist = st["start"].long(), st["history"].long()
    i = torch.arange(hist.numel(), device=DEV)
    row = torch.searchsorted(start, i, right=True) - 1
    made = i >= start[row] + st["prompt"][row]
    one = torch.ones(hist.numel(), device=DEV)
    seen = torch.zeros(r * v, device=DEV).index_add_(0, row * v + hist, one).view(r, v) > 0
    count = torch.zeros(r * v, device=DEV).index_add_(0, row * v + hist, made.float()).view(r, v)
    rep = st["rep"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - (st["freq"][:, None] * count + st["pres"][:, None] * (count > 0))
    if "bias" in st:
        b = torch.zeros((r, v), device=DEV)
        k = torch.arange(st["bias"].numel(), device=DEV)
        b[torch.searchsorted(st["bias_start"].long(), k, right=True) - 1,
          st["bias_ids"].long()] = st["bias"]
        x = x + b
    if "allowed" in st:
        c = torch.arange(v, device=DEV)
        x = torch.where((st["allowed"][:, c // 32] >> (c % 32)) & 1 > 0, x, -math.inf)
    top = x.amax(1, keepdim=True)
    pick = torch.where(x == top, torch.arange(v, device=DEV), -1).amax(1)
    return x, torch.where(top[:, 0] > -math.inf, pick, -1).to(torch.int32)


def _held(st):
    """The pools as numbers, with their scales."""
    kind = {"fp8": torch.float8_e4m3fn, "fp8_block": torch.float8_e4m3fn,
            "int8_block": torch.int8}.get(st["case"]["kv"])
    if kind is None:
        return st["k"], st["v"]
    return st["k"].view(kind), st["v"].view(kind), st["ks"], st["vs"]


def _run_own(st):
    from rustral_amd import kv, model
    case = st["case"]
    op = case["op"]
    if op == "rope":
        return kv.rope(st["x"], st["pos"], st["freq"], interleaved=case["pairs"] == "interleaved",
                       magnitude=case["magnitude"], out=st["out"])
    if op == "rope_append":
        kv.rope_append(st["q"], st["kn"], st["vn"], st["pos"], st["freq"], st["k"], st["v"],
                       st["slots"], k_scale=st["ks"], v_scale=st["vs"],
                       fmt=case["kv"] if case["kv"] == "fp8" else None,
                       interleaved=case["pairs"] == "interleaved", magnitude=case["magnitude"],
                       out=st["out"])
        return (st["out"], *_held(st))
    if op in ("block_decode", "block_prefill"):
        cache = (st["k"], st["v"], st["ks"], st["vs"])
        if "kn" in st:
            kv.append_block_q(*cache, st["kn"], st["vn"], st["start"], st["tab"], st["ctx"],
                              case["kv"], max_new=case.get("new", 1))
        if op == "block_decode":
            kv.decode_attention_q(st["q"], *cache, st["tab"], st["ctx"], None, case["kv"],
                                  out=st["out"])
        else:
            kv.prefill_attention_q(st["q"], *cache, st["tab"], st["start"], st["ctx"], None,
                                   case["kv"], max_q_len=case["new"], out=st["out"])
        return (st["out"], *_held(st)) if "kn" in st else (st["out"],)
    if op == "weights":
        w = st["w"].clone()  # the sums so far are kept for the next pass
        kv.decode_attention_weights(st["q"], st["k"], st["v"], w, st["tab"], st["ctx"], None,
                                    k_scale=st["ks"], v_scale=st["vs"],
                                    fmt=case["kv"] if case["kv"] not in TORCH else None,
                                    out=st["out"])
        return st["out"], w
    if op == "evict":
        keep, lens = kv.evict_select(st["w"], st["tab"], st["ctx"], case["budget"],
                                     sinks=case["sinks"], recent=case["recent"])
        kv.evict_compact(st["k"], st["v"], keep, lens, st["tab"], st["to"], k_scale=st["ks"],
                         v_scale=st["vs"], weights=st["w"],
                         fmt=case["kv"] if case["kv"] not in TORCH else None)
        return (keep, lens, st["w"], *_held(st))
    return model.process_logits(
        st["x"], history=st["history"], history_start=st["start"], prompt_lens=st["prompt"],
        repetition=st["rep"], frequency=st["freq"], presence=st["pres"],
        bias_ids=st.get("bias_ids"), bias=st.get("bias"), bias_start=st.get("bias_start"),
        allowed=st.get("allowed"), out=st["out"])


def run(st: dict):
    if own:
        return _run_own(st)
    case = st["case"]
    op = case["op"]
    if op == "rope":
        return _rotate(st["x"], st["pos"], st["freq"], case["pairs"], case["magnitude"])
    if op == "rope_append":
        q, k = (_rotate(st[x], st["pos"], st["freq"], case["pairs"], case["magnitude"])
                for x in ("q", "kn"))
        _store(st["k"], st["ks"], st["slots"], k)
        _store(st["v"], st["vs"], st["slots"], st["vn"])
        return (q, *_held(st))
    if op in ("block_decode", "block_prefill"):
        if "kn" not in st:
            return (_attend(st),)
        _append_blocks(st["k"], st["ks"], st["kn"], st, case["kv"])
        _append_blocks(st["v"], st["vs"], st["vn"], st, case["kv"])
        return (_attend(st), *_held(st))
    if op == "weights":
        out, p = _attend(st, weights=True)
        w, ids, ctx = st["w"].clone(), st["tab"].long(), st["ctx"].long()
        on = torch.arange(ids.shape[1], device=DEV) < (ctx[:, None] + BS - 1) // BS
        p = p.view(p.shape[0], p.shape[1], -1, BS).transpose(1, 2)          # [B, blocks, hkv, 16]
        w[ids[on]] += p[on]
        return out, w
    if op == "evict":
        keep, lens = _evict_plain(st)
        return (keep, lens, st["w"], *_held(st))
    return _logits_plain(st)


# ---- what a pass cannot do without -----------------------------------------------------

def work(case: dict) -> dict:
    op = case["op"]
    if op == "rope":
        n = case["tokens"] * case["heads"] * case["d"]
        return dict(bytes=8 * n + 4 * case["tokens"], flops=3 * n)
    if op == "rope_append":
        t, d, e = case["tokens"], case["d"], ELEM[case["kv"]]
        row = d * e + (4 if case["kv"] == "fp8" else 0)
        return dict(bytes=t * (8 * case["hq"] * d + 2 * case["hkv"] * (4 * d + row) + 12),
                    flops=3 * t * (case["hq"] + case["hkv"]) * d)
    if op == "logits":
        r, v = case["rows"], case["vocab"]
        extra = 4 * case["history"] * 3 // 4 + 8 * case["biases"] + (v // 8 if case["mask"] else 0)
        return dict(bytes=r * (8 * v + extra + 4), flops=4 * r * v)
    lens, hkv, d, e = _lens(case), case["hkv"], case["d"], ELEM[case["kv"]]
    scale = {"fp8": 4.0, "int8_block": 4 / BS, "fp8_block": 4 / BS}.get(case["kv"], 0.0)
    if op == "evict":
        kept = sum(min(x, case["budget"]) for x in lens)
        return dict(bytes=int(case["layers"] * hkv * (
            4 * sum(lens) + 4 * kept + kept * 2 * (2 * (d * e + scale) + 4))), flops=0)
    pool = sum(lens) * 2 * hkv * (d * e + scale)
    n = case.get("new", 1)
    fresh = case["seqs"] * n * 2 * hkv * (4 * d + d * e) if "append" not in case or \
        case["append"] else 0
    fresh = 0 if op == "weights" else fresh
    sums = 8 * sum(lens) * hkv if op == "weights" else 0
    pairs = sum(n * (x - n) + n * (n + 1) // 2 for x in lens)
    return dict(bytes=int(pool + fresh + sums + 8 * case["seqs"] * n * case["hq"] * d
                          + sum(lens) / 4), flops=4 * d * case["hq"] * pairs)


# ---- the same in float64 -----------------------------------------------------------------

def _turn64(x, st, case):
    """x's pairs as complex numbers, turned."""
    z = torch.polar(torch.tensor(case["magnitude"], dtype=torch.float64, device=DEV),
                    torch.outer(st["pos"].double(), st["freq"]))[:, None]
    y, n = x.double().clone(), st["freq"].numel()
    if case["pairs"] == "half":
        t = torch.complex(y[..., :n], y[..., n:2 * n]) * z
        y[..., :n], y[..., n:2 * n] = t.real, t.imag
    else:
        t = torch.complex(y[..., 0:2 * n:2].contiguous(), y[..., 1:2 * n:2].contiguous()) * z
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = t.real, t.imag
    return y


def _numbers64(bytes_, scale, fmt):
    kind = torch.int8 if fmt.startswith("int8") else torch.float8_e4m3fn
    return bytes_.view(kind).float().double() * scale.double()


def _to_bytes64(x, s, fmt):
    if s == 0:
        return torch.zeros(x.shape, dtype=torch.uint8, device=x.device)
    y = x / s.double()
    if fmt.startswith("int8"):
        return y.round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
    return y.float().clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _fill_block64(pool, scale, blk, h, lo, rows, fmt):
    """Rows lo .. of one (block, head) tile, written after the rows below lo."""
    a = float(rows.abs().max())
    if fmt == "int8_block":
        need = rows.abs().max().float() / 127.0
    else:
        m, e = math.frexp(a / 448.0)
        need = torch.tensor(math.ldexp(1.0, e - 1 if m == 0.5 else e), device=DEV)
    s0 = scale[blk, h].clone() if lo else torch.zeros((), device=DEV)
    s = torch.maximum(s0, need)
    tile = pool[blk, h]
    if lo and s > s0:
        tile[:lo] = _to_bytes64(_numbers64(tile[:lo], s0, fmt), s, fmt)
    tile[lo:lo + rows.shape[0]] = _to_bytes64(rows.double(), s, fmt)
    scale[blk, h] = s


def _sequence64(st, which: str, b: int, n: int):
    fmt, ids = st["case"]["kv"], st["tab"][b, :-(-n // BS)].long()
    x, s = st[which][ids], st[which + "s"]
    if s is not None:
        x = _numbers64(x, s[ids][..., None, None] if fmt.endswith("block") else s[ids][..., None],
                       fmt)
    return x.double().transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, :n]


def _attention64(st, b: int, length: int, n: int):
    """Sequence b's n last rows: outputs [n, hq, d] and the weights [hkv, length]."""
    case = st["case"]
    hkv, d, G = case["hkv"], case["d"], case["hq"] // case["hkv"]
    q = st["q"][b * n:(b + 1) * n].double()
    k, v = _sequence64(st, "k", b, length), _sequence64(st, "v", b, length)
    out = torch.empty_like(q)
    w = torch.zeros((hkv, length), dtype=torch.float64, device=DEV)
    late = torch.arange(length, device=DEV) > \
        (length - n) + torch.arange(n, device=DEV)[:, None]
    for h in range(case["hq"]):
        s = q[:, h] @ k[h // G].T.contiguous() * d ** -0.5
        p = s.masked_fill(late, -math.inf).softmax(-1)
        out[:, h] = p @ v[h // G]
        w[h // G] += p.sum(0)
    return out, w


def _evict64(st, case):
    n, hkv, fmt = case["layers"], case["hkv"], case["kv"]
    lens, B = st["ctx"].tolist(), case["seqs"]
    keep = torch.full((n, B, hkv, case["budget"]), -1, dtype=torch.int32)
    for b, length in enumerate(lens):
        ids = st["tab"][b, :-(-length // BS)].long()
        m = min(length, case["budget"])
        to = st["to"][b, :-(-m // BS)].long()
        for layer in range(n):
            w = st["w"][layer][ids].transpose(0, 1).reshape(hkv, -1)[:, :length].double()
            w[:, :case["sinks"]] = math.inf
            if case["recent"]:
                w[:, max(0, length - case["recent"]):] = math.inf
            top = w.sort(dim=1, descending=True, stable=True)[1][:, :m].sort(1)[0]
            keep[layer, b, :, :m] = top.cpu().to(torch.int32)
            for h in range(hkv):
                p = top[h]
                src, at = (ids[p // BS], p % BS), torch.arange(m, device=DEV)
                dst = (to[at // BS], at % BS)
                st["w"][layer, dst[0], h, dst[1]] = st["w"][layer, src[0], h, src[1]]
                for c in "kv":
                    pool, scale = st[c][layer], st[c + "s"]
                    x = pool[src[0], h, src[1]]
                    if fmt.endswith("block"):
                        s = scale[layer][src[0], h]
                        for j in range(to.numel()):
                            part = slice(j * BS, min(m, (j + 1) * BS))
                            most = s[part].max()
                            pool[to[j], h, :x[part].shape[0]] = _to_bytes64(
                                _numbers64(x[part], s[part, None], fmt), most, fmt)
                            scale[layer][to[j], h] = most
                        continue
                    if scale is not None:
                        scale[layer][dst[0], h, dst[1]] = scale[layer][src[0], h, src[1]]
                    pool[dst[0], h, dst[1]] = x
    left = torch.tensor([min(x, case["budget"]) for x in lens], dtype=torch.int32)
    return (keep.to(DEV), left.to(DEV), st["w"], *_held(st))


def _logits64(st, case):
    out = st["x"].double().clone()
    ends, v = st["start"].tolist(), case["vocab"]
    picks = []
    for r in range(case["rows"]):
        words = st["history"][ends[r]:ends[r + 1]].long()
        y, p = out[r], int(st["prompt"][r])
        ids = words.unique()
        rep = st["rep"][r].double()
        y[ids] = torch.where(y[ids] > 0, y[ids] / rep, y[ids] * rep)
        made, times = words[p:].unique(return_counts=True)
        y[made] -= st["freq"][r].double() * times + st["pres"][r].double()
        if "bias" in st:
            a, z = st["bias_start"][r:r + 2].tolist()
            y[st["bias_ids"][a:z].long()] += st["bias"][a:z].double()
        if "allowed" in st:
            bits = st["allowed"][r].cpu().numpy().view("uint8")
            ok = torch.from_numpy(bits).to(DEV)[:, None] >> torch.arange(8, device=DEV) & 1
            y[ok.reshape(-1)[:v] == 0] = -math.inf
        top = (y == y.max()).nonzero()[-1, 0] if y.max() > -math.inf else -1
        picks.append(int(top))
    return out, torch.tensor(picks, dtype=torch.int32, device=DEV)


def exact(case: dict, seed: int):
    op = case["op"]
    tiles = 0
    if op == "block_prefill":
        tiles = case["seqs"] * (case["new"] // BS + 2) * case["hkv"]
    elif op == "evict" and case["kv"].endswith("block"):
        tiles = case["layers"] * case["hkv"] * sum(
            min(x, case["budget"]) // BS + 1 for x in _lens(case))
    if tiles > 12000:  # a tile at a time: too long
        return None
    st = prepare(case, seed)
    if op == "rope":
        return _turn64(st["x"], st, case)
    if op == "rope_append":
        q, k = _turn64(st["q"], st, case), _turn64(st["kn"], st, case)
        pools = []
        for c, rows in (("k", k), ("v", st["vn"].double())):
            blk, at = st["slots"] // BS, st["slots"] % BS
            if case["kv"] == "fp8":
                a = rows.abs().amax(-1, keepdim=True)
                y = (rows * 448.0 / a).float().to(torch.float8_e4m3fn)
                st[c].view(torch.float8_e4m3fn)[blk, :, at] = y
                st[c + "s"][blk, :, at] = (a / 448.0)[..., 0].float()
                pools.append(st[c].view(torch.float8_e4m3fn).float().double())
            else:
                pool = st[c].double()
                pool[blk, :, at] = rows
                pools.append(pool)
        return (q, *pools) if case["kv"] != "fp8" else (q, *pools, st["ks"], st["vs"])
    if op in ("block_decode", "block_prefill", "weights"):
        lens, n = st["ctx"].tolist(), case.get("new", 1)
        if "kn" in st:
            for c in "kv":
                for b, length in enumerate(lens):
                    for j in range((length - n) // BS, (length - 1) // BS + 1):
                        lo, hi = max(length - n, j * BS), min(length, (j + 1) * BS)
                        at = b * n + lo - (length - n)
                        rows = st[c + "n"][at:at + hi - lo]
                        for h in range(case["hkv"]):
                            _fill_block64(st[c], st[c + "s"], int(st["tab"][b, j]), h, lo % BS,
                                          rows[:, h], case["kv"])
        got = [_attention64(st, b, x, n) for b, x in enumerate(lens)]
        out = torch.cat([o for o, _ in got])
        if op == "weights":
            w = st["w"].double()
            for b, (_, p) in enumerate(got):
                pos = torch.arange(p.shape[1], device=DEV)
                w[st["tab"][b, pos // BS].long(), :, pos % BS] += p.T
            return out, w
        return (out, *_held(st)) if "kn" in st else (out,)
    if op == "evict":
        return _evict64(st, case)
    return _logits64(st, case)
