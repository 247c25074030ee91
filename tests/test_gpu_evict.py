"""Eviction by accumulated weight on the GPU: the sums against 64 bits, the
selection and the move bit-exact."""
import math

import numpy as np
import pytest
import torch

import oracle
from rustral_amd import _lib, kv
from tests import op_refs as R
from tests.gpu_util import say, to_dev, to_np
from tests.helpers import contexts, make_tables
from tests.test_gpu_block_quant import filled

pytestmark = pytest.mark.gpu


def pools_of(rng, nb, hkv, d, kind):
    """(k, v, ks, vs) in storage and (k, v) as float64."""
    if kind.endswith("block"):
        k, v, ks, vs = filled(rng, nb, hkv, d, kind, 0.5)
        return (k, v, ks, vs), (R.dequantize(k, ks, kind), R.dequantize(v, vs, kind))
    x = [rng.standard_normal((nb, hkv, 16, d)).astype(np.float32) for _ in "kv"]
    if kind == "f32":
        return (*x, None, None), tuple(a.astype(np.float64) for a in x)
    if kind == "bf16":
        b = [oracle.bf16_from_f32(a) for a in x]
        return (*b, None, None), tuple((a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
                                       for a in b)
    p, s = [], []
    for a in x:
        m = np.abs(a).max(-1)
        top = 127 if kind == "int8" else 448
        s.append((m / np.float32(top)).astype(np.float32))
        y = a / s[-1][..., None]
        p.append(np.clip(np.rint(y), -127, 127).astype(np.int8).view(np.uint8) if kind == "int8"
                 else R.e4m3(y.astype(np.float32)))
    return (*p, *s), tuple(R.dequantize(a, c, kind) for a, c in zip(p, s))


KINDS = ["f32", "bf16", "int8", "fp8", "int8_block", "fp8_block"]
# hq, hkv, d, contexts
DECODES = [(4, 4, 64, (1, 1, 2)), (8, 4, 128, (1, 128, 6)), (32, 8, 128, (129, 500, 4)),
           (32, 8, 128, (400, 2500, 5)), (16, 2, 64, (700, 1600, 2)), (8, 1, 128, (6000, 6000, 1))]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", range(len(DECODES)))
def test_weights_and_attention(dev, kind, case):
    hq, hkv, d, (lo, hi, B) = DECODES[case]
    say(f"weights {kind} hq={hq} hkv={hkv} d={d} ctx={lo}..{hi} x {B}")
    rng = np.random.default_rng(10 * case + len(kind))
    ctx = contexts(rng, B, lo, hi)
    if B > 3:
        ctx[0] = 0
    nb = int(((ctx + 15) // 16).sum()) + 2
    tables = make_tables(rng, ctx, 16, nb)
    if B > 4:
        tables[1, 0] = -1
        tables[2, :] = nb
    (k, v, ks, vs), (fk, fv) = pools_of(rng, nb, hkv, d, kind)
    q = rng.standard_normal((B, hq, d)).astype(np.float32)
    w0 = rng.random((nb, hkv, 16)).astype(np.float32)
    want, bound, ws, wb = R.attend(q, fk, fv, tables, ctx, 1 / math.sqrt(d))
    sums, sbound = w0.astype(np.float64), np.abs(w0) * 2.0 ** -23
    for b in range(B):
        for p in range(max(0, int(ctx[b]))):
            blk = tables[b, p // 16]
            if 0 <= blk < nb:
                sums[blk, :, p % 16] += ws[b][:, p]
                sbound[blk, :, p % 16] += wb[b][:, p] + 2.0 ** -23 * ws[b][:, p]
    fmt = kind if kind not in ("f32", "bf16") else None
    scales = dict(k_scale=to_dev(ks, dev), v_scale=to_dev(vs, dev)) if fmt else {}
    w = to_dev(w0, dev)
    args = (to_dev(tables, dev), to_dev(ctx, dev), None)
    gk, gv = to_dev(k, dev), to_dev(v, dev)
    out = kv.decode_attention_weights(to_dev(q, dev), gk, gv, w, *args, fmt=fmt, **scales)
    R.assert_within(to_np(out), want, bound, "attention")
    R.assert_within(to_np(w), sums, sbound, "weights")
    # the same bits again (no block is shared)
    w2 = to_dev(w0, dev)
    out2 = kv.decode_attention_weights(to_dev(q, dev), gk, gv, w2, *args, fmt=fmt, **scales)
    assert torch.equal(out, out2) and torch.equal(w, w2)


def test_weights_of_shared_blocks_add_up(dev):
    """Two sequences over one prefix, one of them twice in the call: every one's
    weight arrives."""
    say("weights shared")
    rng = np.random.default_rng(3)
    hq, hkv, d, nb = 8, 2, 64, 12
    tables = np.array([[1, 2, 3, 4], [1, 2, 3, 5], [1, 2, 3, 4], [6, 6, 6, 7]], np.int32)
    ctx = np.array([60, 50, 60, 49], np.int32)
    (k, v, _, _), (fk, fv) = pools_of(rng, nb, hkv, d, "bf16")
    q = rng.standard_normal((4, hq, d)).astype(np.float32)
    q[2] = q[0]
    _, _, ws, wb = R.attend(q, fk, fv, tables, ctx, 1 / math.sqrt(d))
    sums, bound = np.zeros((nb, hkv, 16)), np.full((nb, hkv, 16), 1e-7)
    for b in range(4):
        for p in range(ctx[b]):
            sums[tables[b, p // 16], :, p % 16] += ws[b][:, p]
            bound[tables[b, p // 16], :, p % 16] += wb[b][:, p] + 2.0 ** -21 * ws[b][:, p]
    w = torch.zeros((nb, hkv, 16), device=dev)
    kv.decode_attention_weights(to_dev(q, dev), to_dev(k, dev), to_dev(v, dev), w,
                                to_dev(tables, dev), to_dev(ctx, dev))
    R.assert_within(to_np(w), sums, bound, "shared")
    assert abs(float(w.sum()) - 4 * hq) < 1e-2     # every head's weights add up to 1


@pytest.mark.parametrize("lo,hi,B,budget,sinks,recent", [
    (1, 40, 6, 16, 0, 0), (1, 40, 6, 16, 4, 12), (100, 1000, 4, 64, 4, 20),
    (900, 4000, 3, 1000, 1, 0), (3000, 9000, 2, 700, 4, 256), (20000, 40000, 1, 5000, 0, 1),
    (70000, 70000, 1, 3333, 16, 100), (5, 5, 3, 200, 4, 4), (1024, 1024, 2, 1023, 0, 0)])
def test_select(dev, lo, hi, B, budget, sinks, recent):
    say(f"select {lo}..{hi} x {B} budget={budget} sinks={sinks} recent={recent}")
    rng = np.random.default_rng(lo + hi + budget)
    hkv, layers = 2, 2
    ctx = contexts(rng, B, lo, hi)
    nb = int(((ctx + 15) // 16).sum()) + 2
    tables = make_tables(rng, ctx, 16, nb)
    if B > 3:
        ctx[0] = 0
        tables[1, 0] = -1
    w = np.exp(3 * rng.standard_normal((layers, nb, hkv, 16))).astype(np.float32)
    # ties, zeros of both signs, infinities and NaN among them
    w[0][rng.random(w[0].shape) < 0.3] = 0.5
    w[1][rng.random(w[1].shape) < 0.2] = 0.0
    w[1][rng.random(w[1].shape) < 0.2] = -0.0
    w[1][rng.random(w[1].shape) < 0.05] = np.nan
    w[1][rng.random(w[1].shape) < 0.01] = np.inf
    w[1][rng.random(w[1].shape) < 0.01] = -np.inf
    w[1][rng.random(w[1].shape) < 0.05] *= -1
    keep, lens = kv.evict_select(to_dev(w, dev), to_dev(tables, dev), to_dev(ctx, dev), budget,
                                 sinks=sinks, recent=recent)
    for i in range(layers):
        want, want_lens = R.select(w[i], tables, ctx, budget, sinks, recent)
        assert np.array_equal(to_np(lens), want_lens)
        assert np.array_equal(to_np(keep)[i], want), i


def test_select_equal_weights_and_caps(dev):
    say("select ties")
    nb, hkv = 300, 1
    ctx = np.array([4001, 17, -3, 16], np.int32)
    tables = make_tables(np.random.default_rng(0), np.maximum(ctx, 0), 16, nb)
    w = np.full((nb, hkv, 16), 0.25, np.float32)
    keep, lens = kv.evict_select(to_dev(w, dev), to_dev(tables, dev), to_dev(ctx, dev), 100,
                                 sinks=3, recent=7)
    got = to_np(keep)
    assert to_np(lens).tolist() == [100, 17, 0, 16]
    # all equal: the lower positions, and the last seven
    assert got[0, 0].tolist() == list(range(93)) + list(range(3994, 4001))
    assert got[1, 0].tolist() == list(range(17)) + [-1] * 83 and (got[2] == -1).all()
    want, want_lens = R.select(w, tables, ctx, 30, 2, 4, cap=50)
    keep, lens = kv.evict_select(to_dev(w, dev), to_dev(tables, dev), to_dev(ctx, dev), 30,
                                 sinks=2, recent=4, max_context=50)
    assert np.array_equal(to_np(keep), want) and np.array_equal(to_np(lens), want_lens)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hkv,d,layers", [(2, 64, 2), (8, 128, 1), (3, 32, 2), (1, 128, 3)])
def test_compact(dev, kind, hkv, d, layers):
    say(f"compact {kind} hkv={hkv} d={d} layers={layers}")
    rng = np.random.default_rng(hkv + d + layers)
    B, budget = 4, 50
    ctx = np.array([300, 47, 0, 90], np.int32)
    nb = 60
    tables = make_tables(rng, ctx, 16, nb)
    free = np.setdiff1d(np.arange(nb, dtype=np.int32), tables[tables >= 0])
    dst = np.full((B, 4), -1, np.int32)
    dst[0], dst[1, :3], dst[3] = free[:4], free[4:7], free[7:11]
    dst[3, 1] = nb                                  # a destination that is not there
    sets = [pools_of(rng, nb, hkv, d, kind)[0] for _ in range(layers)]
    k, v = (np.stack([s[i] for s in sets]) for i in range(2))
    ks, vs = (None if sets[0][2] is None else np.stack([s[i] for s in sets]) for i in (2, 3))
    w = rng.random((layers, nb, hkv, 16)).astype(np.float32)
    fmt = kind if kind not in ("f32", "bf16") else None
    g = [None if a is None else to_dev(a, dev) for a in (k, v, ks, vs, w)]
    keep, lens = kv.evict_select(g[4], to_dev(tables, dev), to_dev(ctx, dev), budget, sinks=2,
                                 recent=10)
    kv.evict_compact(g[0], g[1], keep, lens, to_dev(tables, dev), to_dev(dst, dev), k_scale=g[2],
                     v_scale=g[3], weights=g[4], fmt=fmt)
    nk, nl = to_np(keep), to_np(lens)
    for i in range(layers):
        want, _ = R.select(w[i], tables, ctx, budget, 2, 10)
        assert np.array_equal(nk[i], want)
        R.compact(k[i], v[i], None if ks is None else ks[i], None if vs is None else vs[i], w[i],
                  nk[i], nl, tables, dst, fmt)
    torch.cuda.synchronize()
    for got, want, name in zip(g, (k, v, ks, vs, w), ("k", "v", "ks", "vs", "w")):
        if want is not None:
            assert np.array_equal(to_np(got).view(np.uint8), want.view(np.uint8)), name


def test_compact_any_head_width_and_bad_positions(dev):
    """head_dim 40 (no unrolled build), without sums, positions the table does not
    hold."""
    say("compact any")
    rng = np.random.default_rng(1)
    nb, hkv, d = 8, 2, 40
    k, v = (rng.standard_normal((nb, hkv, 16, d)).astype(np.float32) for _ in "kv")
    src, dst = np.array([[0, 9]], np.int32), np.array([[3]], np.int32)
    keep = np.array([[[0, 5, 16, 40], [-7, 3, 15, 2]]], np.int32)
    lens = np.array([4], np.int32)
    gk, gv = to_dev(k, dev), to_dev(v, dev)
    kv.evict_compact(gk, gv, to_dev(keep, dev), to_dev(lens, dev), to_dev(src, dev), to_dev(dst, dev))
    R.compact(k, v, None, None, None, keep, lens, src, dst, None)
    torch.cuda.synchronize()
    assert np.array_equal(to_np(gk), k) and np.array_equal(to_np(gv), v)


def test_evict_front_end_refuses(dev):
    w = torch.zeros((4, 2, 16), device=dev)
    tab = torch.zeros((1, 2), dtype=torch.int32, device=dev)
    ctx = torch.zeros(1, dtype=torch.int32, device=dev)
    k = torch.zeros((4, 2, 16, 64), device=dev)
    q = torch.zeros((1, 4, 64), device=dev)
    with pytest.raises(ValueError):
        kv.evict_select(w, tab[0], ctx, 8)
    with pytest.raises(ValueError):
        kv.evict_select(w, tab, ctx, 8, keep=torch.zeros((1, 2, 9), dtype=torch.int32, device=dev))
    with pytest.raises(ValueError):
        kv.decode_attention_weights(q, k, k, w[:3], tab, ctx)
    with pytest.raises(ValueError):
        kv.decode_attention_weights(q, k.to(torch.uint8), k.to(torch.uint8), w, tab, ctx, fmt="int8")
    keep = torch.zeros((1, 2, 8), dtype=torch.int32, device=dev)
    with pytest.raises(ValueError):
        kv.evict_compact(k, k, keep[:, :1], ctx, tab, tab)
    with pytest.raises(ValueError):
        kv.evict_compact(k, k, keep, ctx, tab, tab, weights=w[:2])


def _sums(rng, kind, shape):
    x = rng.standard_normal(shape)
    w = {"spread": lambda: np.exp(2 * x),              # a few hundred keys a first digit
         "close": lambda: 1 + 1e-4 * x,                # nearly all keys in one first digit
         "steps": lambda: np.round(np.exp(x) * 4) / 4,  # ties at every threshold
         "nan": lambda: np.where(x > -0.5, np.nan, x),  # the threshold among the NaN
         "tiny": lambda: x * 1e-42}[kind]()            # subnormal sums, both signs
    return w.astype(np.float32)


@pytest.mark.parametrize("kind", ["spread", "close", "steps", "nan", "tiny"])
@pytest.mark.parametrize("length,B,layers", [(1, 2, 1), (300, 2, 1), (1500, 3, 1), (6000, 1, 2),
                                             (33000, 1, 1), (150, 80, 4), (2500, 2, 150)])
def test_select_distributions(dev, kind, length, B, layers):
    """Where the threshold falls decides how the kernel comes to it: in a first digit of
    few keys or of many, among ties, among the lowest keys; for few workgroups and for
    many, with budgets of one row, a part and all but one."""
    say(f"select {kind} {length} x {B} x {layers}")
    rng = np.random.default_rng(length + B)
    hkv = 2
    ctx = contexts(rng, B, max(1, length - 40), length)
    nb = int(((ctx + 15) // 16).sum()) + 1
    tables = make_tables(rng, ctx, 16, nb)
    one = _sums(rng, kind, (2, nb, hkv, 16))
    w = one[np.arange(layers) % 2]
    for budget in sorted({1, int(ctx.max()) // 3 + 1, max(1, int(ctx.min()) - 1)}):
        keep, lens = kv.evict_select(to_dev(w, dev), to_dev(tables, dev), to_dev(ctx, dev), budget,
                                     sinks=min(2, budget - 1), recent=0)
        for i in range(min(2, layers)):
            want, want_lens = R.select(one[i], tables, ctx, budget, min(2, budget - 1), 0)
            assert np.array_equal(to_np(lens), want_lens)
            got = to_np(keep)[i::2]
            assert all(np.array_equal(g, want) for g in got), (budget, i)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 4, 64), (16, 2, 64), (4, 2, 128)])
def test_what_no_table_names_is_not_seen(dev, kind, hq, hkv, d):
    """Block 0 (what an invalid id is read as), a block past every table and the rows behind
    each context hold NaN and infinities, scales too; tables have holes, ids too large,
    a context past its table's valid part and one of length 0."""
    say(f"unseen {kind} hq={hq} hkv={hkv} d={d}")
    rng = np.random.default_rng(21)
    ctx = np.array([37, 0, 700, 130, 16], np.int32)
    nb = 60
    ids = rng.permutation(np.arange(1, nb - 1))
    tables = np.full((5, 45), -1, np.int32)
    o = 0
    for b, n in enumerate(ctx):
        m = -(-int(n) // 16)
        if b == 2:
            m = 30                              # the rest of its context has no blocks
        tables[b, :m] = ids[o:o + m]
        o += m
    tables[2, 3], tables[3, 0], tables[3, 4] = -1, nb, 2 ** 31 - 1
    (k, v, ks, vs), (fk, fv) = pools_of(rng, nb, hkv, d, kind)
    bad = {"f32": np.float32("nan"), "bf16": np.uint16(0x7fc0)}.get(kind, np.uint8(0x7f))
    inf = {"f32": np.float32("inf"), "bf16": np.uint16(0xff80)}.get(kind, np.uint8(0xff))
    for blk in (0, nb - 1):
        k[blk], v[blk] = bad, inf
        if ks is not None:
            ks[blk], vs[blk] = np.nan, np.inf
    for b, n in enumerate(ctx):
        if n % 16 and 0 <= tables[b, n // 16] < nb:
            k[tables[b, n // 16], :, n % 16:] = bad
            v[tables[b, n // 16], :, n % 16:] = inf
            if kind in ("int8", "fp8"):
                ks[tables[b, n // 16], :, n % 16:] = np.nan
                vs[tables[b, n // 16], :, n % 16:] = np.inf
    fk, fv = np.nan_to_num(fk), np.nan_to_num(fv)
    q = rng.standard_normal((5, hq, d)).astype(np.float32)
    fmt = kind if kind not in ("f32", "bf16") else None
    scales = dict(k_scale=to_dev(ks, dev), v_scale=to_dev(vs, dev)) if fmt else {}
    want, bound, ws, _ = R.attend(q, fk, fv, tables, ctx, 1 / math.sqrt(d))
    w = torch.zeros((nb, hkv, 16), device=dev)
    gk, gv, gt, gc = (to_dev(a, dev) for a in (k, v, tables, ctx))
    out = kv.decode_attention_weights(to_dev(q, dev), gk, gv, w, gt, gc, fmt=fmt, **scales)
    R.assert_within(to_np(out), want, bound, "attention with weights")
    w = to_np(w)
    assert np.isfinite(w).all() and not w[0].any() and not w[nb - 1].any()
    assert abs(w.sum() - 4 * hq) < 1e-2
    if kind.endswith("block"):
        args = (gk, gv, scales["k_scale"], scales["v_scale"], gt)
        for ps in (0, 64, 128):
            got = kv.decode_attention_q(to_dev(q, dev), *args, gc, None, fmt, partition_size=ps)
            R.assert_within(to_np(got), want, bound, f"decode {ps}")
        n = np.array([37, 0, 90, 100, 16], np.int32)
        start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        qq = rng.standard_normal((int(start[-1]), hq, d)).astype(np.float32)
        got = kv.prefill_attention_q(to_dev(qq, dev), *args, to_dev(start, dev), gc, None, fmt)
        want, bound, _, _ = R.attend(qq, fk, fv, tables, ctx, 1 / math.sqrt(d), n, start)
        R.assert_within(to_np(got), want, bound, "prefill")


@pytest.mark.parametrize("kind", ["bf16", "int8", "fp8", "int8_block", "fp8_block"])
@pytest.mark.parametrize("hq,hkv,d", [(16, 2, 128), (16, 4, 64), (4, 2, 128), (2, 2, 64)])
def test_precision_of_the_products(dev, kind, hq, hkv, d):
    """Queries and weights enter the matrix cores with 24 bits at every group size.  What is
    left are the roundings of some 128 fp32 additions of partial sums of about 1: 11 steps
    of 2^-25 when they are independent, 3.4e-7; 2^-20 is three times that, and two bf16
    terms (2^-17 of each of 128 products, as many independent) would be 3e-6 off."""
    say(f"precision {kind} hq={hq} hkv={hkv} d={d}")
    rng = np.random.default_rng(5)
    ctx = np.array([400, 1300], np.int32)
    nb = 110
    tables = make_tables(rng, ctx, 16, nb)
    (k, v, ks, vs), (fk, fv) = pools_of(rng, nb, hkv, d, kind)
    q = rng.standard_normal((2, hq, d)).astype(np.float32)
    want, _, ws, _ = R.attend(q, fk, fv, tables, ctx, 1 / math.sqrt(d))
    fmt = kind if kind != "bf16" else None
    scales = dict(k_scale=to_dev(ks, dev), v_scale=to_dev(vs, dev)) if fmt else {}
    w = torch.zeros((nb, hkv, 16), device=dev)
    gk, gv, gt, gc = (to_dev(a, dev) for a in (k, v, tables, ctx))
    outs = [kv.decode_attention_weights(to_dev(q, dev), gk, gv, w, gt, gc, fmt=fmt, **scales)]
    if kind.endswith("block"):
        outs.append(kv.decode_attention_q(to_dev(q, dev), gk, gv, *scales.values(), gt, gc, fmt=fmt))
    for o in outs:
        assert np.linalg.norm(to_np(o) - want) <= 2.0 ** -20 * np.linalg.norm(want)
    w = to_np(w)
    for b in range(2):
        p = np.arange(ctx[b])
        got = w[tables[b, p // 16], :, p % 16].T
        assert np.linalg.norm(got - ws[b]) <= 2.0 ** -20 * np.linalg.norm(ws[b])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("hq,hkv,lo,hi", [(4, 4, 1, 90), (8, 4, 100, 600), (8, 1, 700, 2100)])
def test_weights_of_narrow_heads(dev, kind, hq, hkv, lo, hi):
    say(f"weights d=32 {kind} hq={hq} hkv={hkv}")
    rng = np.random.default_rng(hi)
    ctx = contexts(rng, 3, lo, hi)
    nb = int(((ctx + 15) // 16).sum()) + 1
    tables = make_tables(rng, ctx, 16, nb)
    (k, v, _, _), (fk, fv) = pools_of(rng, nb, hkv, 32, kind)
    q = rng.standard_normal((3, hq, 32)).astype(np.float32)
    want, bound, ws, wb = R.attend(q, fk, fv, tables, ctx, 1 / math.sqrt(32))
    w = torch.zeros((nb, hkv, 16), device=dev)
    out = kv.decode_attention_weights(to_dev(q, dev), to_dev(k, dev), to_dev(v, dev), w,
                                      to_dev(tables, dev), to_dev(ctx, dev))
    R.assert_within(to_np(out), want, bound, "attention")
    w = to_np(w)
    for b in range(3):
        p = np.arange(ctx[b])
        R.assert_within(w[tables[b, p // 16], :, p % 16].T, ws[b], wb[b] + 2.0 ** -23 * ws[b], "sums")


def test_shapes_without_a_kernel_are_refused(dev):
    say("no kernel")
    z = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device=dev)
    tab, ctx = z(1, 2, t=torch.int32), torch.full((1,), 5, dtype=torch.int32, device=dev)
    w = z(4, 2, 16)
    for hq, d, fmt in ((6, 64, None), (32, 64, None), (2, 48, None), (2, 32, "int8_block"),
                       (6, 64, "fp8_block"), (2, 32, "int8")):
        t = torch.float32 if fmt is None else torch.uint8
        k, v = z(4, 2, 16, d, t=t), z(4, 2, 16, d, t=t)
        s = {}
        if fmt:
            shape = (4, 2) if fmt.endswith("block") else (4, 2, 16)
            s = dict(k_scale=z(*shape), v_scale=z(*shape), fmt=fmt)
        with pytest.raises(_lib.RkvError):
            kv.decode_attention_weights(z(1, hq, d), k, v, w, tab, ctx, **s)
        if fmt and fmt.endswith("block"):
            with pytest.raises(_lib.RkvError):
                kv.decode_attention_q(z(1, hq, d), k, v, s["k_scale"], s["v_scale"], tab, ctx,
                                      fmt=fmt)
            with pytest.raises(_lib.RkvError):
                kv.prefill_attention_q(z(1, hq, d), k, v, s["k_scale"], s["v_scale"], tab,
                                       torch.tensor([0, 1], dtype=torch.int32, device=dev), ctx,
                                       fmt=fmt)
    with pytest.raises(ValueError):      # the fused append takes row-scaled pools
        kv.decode_attention_append_q(z(1, 2, 64), z(4, 2, 16, 64, t=torch.uint8),
                                     z(4, 2, 16, 64, t=torch.uint8), z(4, 2), z(4, 2), z(1, 2, 64),
                                     z(1, 2, 64), tab, ctx, fmt="int8_block")
