"""8-bit pools with one scale a (block, KV head) tile on the GPU: append_block_q
bytes and scales bit-exact against the formulas, gather, decode and prefill
attention against 64 bits on the dequantized pools."""
import math

import numpy as np
import pytest
import torch

from rustral_amd import _lib, kv
from tests import op_refs as R
from tests.gpu_util import say, to_dev, to_np
from tests.helpers import contexts, make_tables

pytestmark = pytest.mark.gpu

FMTS = ["int8_block", "fp8_block"]


def filled(rng, nb, hkv, d, fmt, spread=0.0):
    """Random pools with sensible tiles, as numpy."""
    out = []
    for _ in "kv":
        x = rng.standard_normal((nb, hkv, 16, d)).astype(np.float32)
        if spread:
            x *= np.exp(spread * rng.standard_normal((nb, hkv, 1, 1))).astype(np.float32)
        p, s = np.zeros((nb, hkv, 16, d), np.uint8), np.zeros((nb, hkv), np.float32)
        for i in range(nb):
            for h in range(hkv):
                s[i, h] = R.tile_scale(np.abs(x[i, h]).max(), fmt)
                p[i, h] = R.tile_bytes(x[i, h], s[i, h], fmt)
        out.append((p, s))
    return out[0][0], out[1][0], out[0][1], out[1][1]


# new rows a sequence, contexts after them: fresh blocks, one row at a time, runs
# that start and end inside a block, empty ones, a context shorter than its new
# rows, several blocks
APPENDS = [([1, 1, 1, 1], [1, 16, 17, 40]), ([5, 0, 40, 16], [5, 33, 47, 16]),
           ([3, 100, 17, 1], [300, 100, 33, 2]), ([20, 7, 2, 2], [13, 7, 2, -1])]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hkv,d,layers", [(8, 128, 1), (2, 64, 3), (1, 32, 2), (3, 128, 1)])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append_block_q_bitexact(dev, fmt, hkv, d, layers, case):
    say(f"append_block_q {fmt} hkv={hkv} d={d} layers={layers} case={case}")
    rng = np.random.default_rng(100 * case + hkv + d)
    n, ctx = (np.array(x, np.int32) for x in APPENDS[case])
    start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    nb = 40
    tables = make_tables(rng, np.maximum(ctx, 1), 16, nb)
    if case == 2:
        tables[0, -1] = nb            # the block of sequence 0's last rows is not there
        tables[1, 2] = -1
    pools = [filled(rng, nb, hkv, d, fmt) for _ in range(layers)]
    k, v, ks, vs = (np.stack([p[i] for p in pools]) for i in range(4))
    ks[:, tables[0, 0]] = 1e30        # what a reused block's memory may hold
    kn = (rng.standard_normal((layers, max(1, int(start[-1])), hkv, d)) *
          np.exp(rng.standard_normal((layers, 1, hkv, 1)))).astype(np.float32)
    vn = rng.standard_normal(kn.shape).astype(np.float32)
    g = [to_dev(a, dev) for a in (k, v, ks, vs)]
    one = (lambda t: t[0]) if layers == 1 else (lambda t: t)
    kv.append_block_q(*(one(t) for t in g), one(to_dev(kn, dev)), one(to_dev(vn, dev)),
                      to_dev(start, dev), to_dev(tables, dev), to_dev(ctx, dev), fmt)
    for i in range(layers):
        R.append_block(k[i], ks[i], kn[i], start, tables, ctx, fmt)
        R.append_block(v[i], vs[i], vn[i], start, tables, ctx, fmt)
    torch.cuda.synchronize()
    for got, want, name in zip(g, (k, v, ks, vs), ("k", "v", "ks", "vs")):
        assert np.array_equal(to_np(got).view(np.uint8), want.view(np.uint8)), name


@pytest.mark.parametrize("fmt", FMTS)
def test_append_block_q_one_row_at_a_time(dev, fmt):
    """Forty steps of growing and shrinking rows: every growth of a scale brings
    the older rows along, and max_new bounds what a call writes."""
    say(f"append_block_q steps {fmt}")
    rng = np.random.default_rng(8)
    B, hkv, d, nb = 3, 2, 64, 16
    k, v = (rng.integers(0, 255, (nb, hkv, 16, d), dtype=np.uint8) for _ in "kv")
    ks, vs = np.full((nb, hkv), np.nan, np.float32), np.full((nb, hkv), np.inf, np.float32)
    g = [to_dev(a, dev) for a in (k, v, ks, vs)]
    tables = make_tables(rng, [48] * B, 16, nb)
    start = np.arange(B + 1, dtype=np.int32)
    for step in range(40):
        ctx = np.full(B, step + 1, np.int32)
        size = np.exp(2 * rng.standard_normal((B, hkv, 1))) * (1 + step % 5)
        kn = (rng.standard_normal((B, hkv, d)) * size).astype(np.float32)
        vn = (rng.standard_normal((B, hkv, d)) / size).astype(np.float32)
        kv.append_block_q(*g, to_dev(kn, dev), to_dev(vn, dev), to_dev(start, dev),
                          to_dev(tables, dev), to_dev(ctx, dev), fmt, max_new=1)
        R.append_block(k, ks, kn, start, tables, ctx, fmt)
        R.append_block(v, vs, vn, start, tables, ctx, fmt)
    torch.cuda.synchronize()
    for got, want in zip(g, (k, v, ks, vs)):
        assert np.array_equal(to_np(got).view(np.uint8), want.view(np.uint8))
    many, vmany = (rng.standard_normal((9, hkv, d)).astype(np.float32) for _ in "kv")
    start = np.array([0, 3, 6, 9], np.int32)
    ctx = np.full(B, 43, np.int32)
    kv.append_block_q(*g, to_dev(many, dev), to_dev(vmany, dev), to_dev(start, dev),
                      to_dev(tables, dev), to_dev(ctx, dev), fmt, max_new=2)
    R.append_block(k, ks, many, start, tables, ctx, fmt, max_new=2)
    R.append_block(v, vs, vmany, start, tables, ctx, fmt, max_new=2)
    torch.cuda.synchronize()
    for got, want in zip(g, (k, v, ks, vs)):
        assert np.array_equal(to_np(got).view(np.uint8), want.view(np.uint8))


@pytest.mark.parametrize("fmt", FMTS)
def test_append_block_q_borders(dev, fmt):
    """Ties, zeros, tiny tiles, infinities, NaN, values at the ends."""
    say(f"append_block_q borders {fmt}")
    hkv, d, nb = 1, 64, 12
    f = np.float32
    rows = np.zeros((10, 4, hkv, d), f)
    rows[0, 0, 0, :5] = [127, 0.5, 1.5, -2.5, 126.5]          # int8 scale 1: ties to even
    rows[1] = 0                                               # zeros
    rows[2, :, 0, 3] = 2.0 ** -111                            # below the smallest tile
    rows[3, 0, 0, 3], rows[3, 1, 0, 4] = 2.0 ** -110, 2.0 ** -111
    rows[4, 0, 0, :4] = [np.inf, -np.inf, np.nan, 3.0]
    rows[5, :, 0, 0] = np.inf                                 # nothing finite but zeros
    rows[6, 0, 0, :3] = [448, 447, 1.9999]
    rows[7, 0, 0, :3] = [449, 448.0001, -0.001]               # needs the next power of two
    rows[8, 0, 0, :3] = [3e38, 1.0, -3e38]
    rows[9] = np.linspace(-5, 5, 4 * d).reshape(4, hkv, d)
    seqs = len(rows)
    k = np.random.default_rng(1).integers(0, 256, (nb, hkv, 16, d), dtype=np.uint8)
    v, ks, vs = k.copy(), np.ones((nb, hkv), f), np.ones((nb, hkv), f)
    tables = np.arange(seqs, dtype=np.int32)[:, None]
    start = (4 * np.arange(seqs + 1)).astype(np.int32)
    for at, by in ((0, 1.0), (6, 1.0), (10, 24.0)):   # fresh, behind six rows, a growth
        ctx = np.full(seqs, at + 4, np.int32)
        with np.errstate(over="ignore"):
            new = (rows * f(by)).reshape(-1, hkv, d)
        g = [to_dev(a, dev) for a in (k, v, ks, vs)]
        kv.append_block_q(*g, to_dev(new, dev), to_dev(new[::-1].copy(), dev), to_dev(start, dev),
                          to_dev(tables, dev), to_dev(ctx, dev), fmt, max_new=4)
        R.append_block(k, ks, new, start, tables, ctx, fmt)
        R.append_block(v, vs, new[::-1].copy(), start, tables, ctx, fmt)
        torch.cuda.synchronize()
        for got, want, name in zip(g, (k, v, ks, vs), ("k", "v", "ks", "vs")):
            assert np.array_equal(to_np(got).view(np.uint8), want.view(np.uint8)), (at, name)


@pytest.mark.parametrize("fmt", FMTS)
def test_gather_of_block_pools(dev, fmt):
    say(f"gather {fmt}")
    rng = np.random.default_rng(4)
    hkv, d, nb = 8, 128, 80
    ctx = np.array([0, 1, 15, 16, 17, 300, 555], np.int32)
    tables = make_tables(rng, ctx, 16, nb)
    k, v, ks, vs = filled(rng, nb, hkv, d, fmt, 1.0)
    ko, vo = kv.gather_q(*(to_dev(a, dev) for a in (k, v, ks, vs)), to_dev(tables, dev),
                         to_dev(ctx, dev), fmt, max_ctx=560)
    want_k, want_v = R.dequantize(k, ks, fmt).astype(np.float32), R.dequantize(v, vs, fmt).astype(np.float32)
    for got, want in ((to_np(ko), want_k), (to_np(vo), want_v)):
        for b, L in enumerate(ctx):
            pos = np.arange(L)
            rows = want[tables[b, pos // 16], :, pos % 16].transpose(1, 0, 2)
            assert np.array_equal(got[b, :, :L], rows)
            assert not got[b, :, L:].any()


# hq, hkv, d, contexts (low, high, sequences): every group size, one partition and
# many, one token
DECODES = [(8, 8, 64, (1, 1, 3)), (8, 4, 128, (1, 40, 5)), (32, 8, 128, (100, 128, 4)),
           (32, 8, 128, (300, 2000, 6)), (16, 2, 64, (500, 1500, 3)), (4, 1, 128, (9000, 9000, 1)),
           (2, 2, 64, (3000, 5000, 2)), (8, 1, 128, (513, 700, 2)), (64, 8, 64, (17, 400, 9))]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("case", range(len(DECODES)))
def test_decode_over_block_pools(dev, fmt, case):
    hq, hkv, d, (lo, hi, B) = DECODES[case]
    say(f"decode {fmt} hq={hq} hkv={hkv} d={d} ctx={lo}..{hi} x {B}")
    rng = np.random.default_rng(case)
    ctx = contexts(rng, B, lo, hi)
    if B > 3:
        ctx[1] = 0
    nb = int(((ctx + 15) // 16).sum()) + 3
    tables = make_tables(rng, ctx, 16, nb)
    if B > 4:
        tables[2, 0] = nb + 5                 # a block that is not there
        tables[3, :] = -1                     # nothing left of this sequence
    k, v, ks, vs = filled(rng, nb, hkv, d, fmt, 0.5)
    used = np.zeros(nb, bool)
    used[tables[(tables >= 0) & (tables < nb)]] = True
    ks[~used], vs[~used] = np.nan, np.nan     # never read
    for b in range(B):                        # rows behind a sequence: any bytes
        if ctx[b] % 16 and 0 <= tables[b, ctx[b] // 16] < nb:
            k[tables[b, ctx[b] // 16], :, ctx[b] % 16:] = 0x7f
            v[tables[b, ctx[b] // 16], :, ctx[b] % 16:] = 0xff
    q = rng.standard_normal((B, hq, d)).astype(np.float32)
    g = [to_dev(a, dev) for a in (k, v, ks, vs, tables, ctx)]
    scale = 1 / math.sqrt(d)
    ref_ks, ref_vs = np.where(used[:, None], ks, 0), np.where(used[:, None], vs, 0)
    with np.errstate(invalid="ignore"):
        dk, dv = np.nan_to_num(R.dequantize(k, ref_ks, fmt)), np.nan_to_num(R.dequantize(v, ref_vs, fmt))
    want, bound, _, _ = R.attend(q, dk, dv, tables, ctx, scale)
    for ps in (0, 64, 640):
        got = to_np(kv.decode_attention_q(to_dev(q, dev), *g, None, fmt, partition_size=ps))
        R.assert_within(got, want, bound, f"partition_size={ps}")
        assert np.linalg.norm(got - want) <= 2.0 ** -15 * max(np.linalg.norm(want), 1e-9)


# hq, hkv, d, new rows, contexts
PREFILLS = [(8, 8, 64, [1, 5], [1, 5]), (8, 4, 128, [40, 3, 17], [40, 70, 33]),
            (32, 8, 128, [128, 0, 60], [128, 20, 300]), (16, 2, 64, [33, 200], [500, 200]),
            (8, 1, 128, [16, 1], [16, 129]), (64, 8, 128, [70], [70]),
            (2, 1, 64, [9, 7], [5, 7]), (4, 4, 128, [150, 2], [150, 31])]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("case", range(len(PREFILLS)))
def test_prefill_over_block_pools(dev, fmt, case):
    hq, hkv, d, n, ctx = PREFILLS[case]
    say(f"prefill {fmt} hq={hq} hkv={hkv} d={d} n={n} ctx={ctx}")
    rng = np.random.default_rng(50 + case)
    n, ctx = np.array(n, np.int32), np.array(ctx, np.int32)
    start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    nb = int(((ctx + 15) // 16).sum()) + 3
    tables = make_tables(rng, ctx, 16, nb)
    if case == 3:
        tables[0, 4] = -1                     # a hole in the cached prefix
    k, v, ks, vs = filled(rng, nb, hkv, d, fmt, 0.5)
    used = np.zeros(nb, bool)
    used[tables[tables >= 0]] = True
    ks[~used], vs[~used] = np.nan, np.inf
    k[~used], v[~used] = 0x7f, 0xff
    for b in range(len(ctx)):                 # rows behind a sequence: any bytes, a NaN too
        if ctx[b] % 16:
            k[tables[b, ctx[b] // 16], :, ctx[b] % 16:] = 0x7f
            v[tables[b, ctx[b] // 16], :, ctx[b] % 16:] = 0xff
    q = rng.standard_normal((max(1, int(start[-1])), hq, d)).astype(np.float32)
    g = [to_dev(a, dev) for a in (k, v, ks, vs, tables, start, ctx)]
    with np.errstate(invalid="ignore"):
        dk = np.nan_to_num(R.dequantize(k, np.where(used[:, None], ks, 0), fmt))
        dv = np.nan_to_num(R.dequantize(v, np.where(used[:, None], vs, 0), fmt))
    want, bound, _, _ = R.attend(q, dk, dv, tables, ctx, 1 / math.sqrt(d), n, start)
    out = torch.full((len(q) + 1, hq, d), 7.0, device=dev)
    kv.prefill_attention_q(to_dev(q, dev), *g, None, fmt, out=out[:-1])
    got = to_np(out)
    assert (got[-1] == 7.0).all()             # behind the last sequence
    R.assert_within(got[:-1], want, bound, "prefill")
    assert np.linalg.norm(got[:-1] - want) <= 2.0 ** -15 * max(np.linalg.norm(want), 1e-9)


@pytest.mark.parametrize("fmt", FMTS)
def test_last_prefill_row_is_the_decode_of_that_row(dev, fmt):
    """A prompt appended and attended, then its last row by decode."""
    say(f"prefill then decode {fmt}")
    rng = np.random.default_rng(6)
    hq, hkv, d, n = 8, 2, 128, np.array([77, 16, 130], np.int32)
    start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    nb = 20
    tables = make_tables(rng, n, 16, nb)
    pools = [torch.zeros((nb, hkv, 16, d), dtype=torch.uint8, device=dev) for _ in "kv"] + \
        [torch.zeros((nb, hkv), device=dev) for _ in "kv"]
    kn, vn = (to_dev(rng.standard_normal((int(start[-1]), hkv, d)).astype(np.float32), dev)
              for _ in "kv")
    q = to_dev(rng.standard_normal((int(start[-1]), hq, d)).astype(np.float32), dev)
    st, tb, cx = to_dev(start, dev), to_dev(tables, dev), to_dev(n, dev)
    kv.append_block_q(*pools, kn, vn, st, tb, cx, fmt)
    all_rows = kv.prefill_attention_q(q, *pools, tb, st, cx, None, fmt)
    last = torch.from_numpy(start[1:].astype(np.int64) - 1).to(dev)
    one = kv.decode_attention_q(q[last].contiguous(), *pools, tb, cx, None, fmt)
    err = (all_rows[last] - one).abs().max().item()
    # both within 2^-14 max |v| or so of the exact rows (op_refs.attend's bound)
    assert err < 2e-3, err


def test_block_front_end_refuses(dev):
    k = torch.zeros((4, 2, 16, 64), dtype=torch.uint8, device=dev)
    s, rows = torch.zeros((4, 2), device=dev), torch.zeros((4, 2, 16), device=dev)
    x = torch.zeros((3, 2, 64), device=dev)
    st = torch.tensor([0, 3], dtype=torch.int32, device=dev)
    tab, ctx = torch.zeros((1, 2), dtype=torch.int32, device=dev), st[1:]
    with pytest.raises(ValueError, match="scale pools"):
        kv.append_block_q(k, k, rows, rows, x, x, st, tab, ctx)
    with pytest.raises(ValueError, match="format"):
        kv.append_block_q(k, k, s, s, x, x, st, tab, ctx, "int8")
    with pytest.raises(ValueError):
        kv.append_block_q(k, k, s, s, x, x, st[:1], tab, ctx)
    with pytest.raises(ValueError):
        kv.append_block_q(k, k, s, s, x[:, :1], x[:, :1], st, tab, ctx)
    q = torch.zeros((1, 4, 64), device=dev)
    with pytest.raises(ValueError, match="scale pools"):
        kv.decode_attention_q(q, k, k, rows, rows, tab, ctx, None, "int8_block")
    with pytest.raises(ValueError, match="scale pools"):
        kv.gather_q(k, k, rows, rows, tab, ctx, "fp8_block")
    with pytest.raises(ValueError):
        kv.prefill_attention_q(q, k, k, s, s, tab, st[:1], ctx)
    with pytest.raises(ValueError, match="format"):
        kv.decode_attention_append_q(q, k, k, s, s, x[:1], x[:1], tab, ctx, None, "int8_block")
    with pytest.raises(_lib.RkvError):
        kv.prefill_attention_q(torch.zeros((3, 6, 64), device=dev), k, k, s, s, tab, st, ctx)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("bad", [np.nan, np.inf, 2.0 ** 100])
def test_prefill_rows_before_a_tile_do_not_see_its_scales(dev, fmt, bad):
    """The tile of positions 32 .. 47 gets scales of NaN, infinity or 2^100: the rows
    before it keep every bit, whichever wave and iteration they share with it."""
    say(f"prefill before a bad tile {fmt} {bad}")
    rng = np.random.default_rng(9)
    for ctx0, hq, hkv, d in [(40, 8, 2, 128), (70, 8, 8, 64), (48, 8, 1, 128)]:
        for cached in (0, 10, 27):
            n, ctx = np.array([ctx0 - cached], np.int32), np.array([ctx0], np.int32)
            nb = 6
            tables = make_tables(rng, ctx, 16, nb)
            k, v, ks, vs = filled(rng, nb, hkv, d, fmt, 0.5)
            q = rng.standard_normal((int(n[0]), hq, d)).astype(np.float32)
            outs = []
            for scale in (None, bad):
                if scale is not None:
                    ks[tables[0, 2]], vs[tables[0, 2]] = scale, scale
                g = [to_dev(a, dev) for a in (k, v, ks, vs, tables, np.array([0, n[0]], np.int32),
                                              ctx)]
                outs.append(to_np(kv.prefill_attention_q(to_dev(q, dev), *g, None, fmt)))
            rows = 32 - cached
            assert np.isfinite(outs[1][:rows]).all()
            assert np.array_equal(outs[0][:rows], outs[1][:rows]), (ctx0, cached)
