"""The operators around the cache as a serving program runs them together: rotary
positions, append, attention that adds up weights, logits, and now and then an
eviction into fresh blocks; the same step captured in a graph; calls on two
streams at once."""
import math

import numpy as np
import pytest
import torch

from rustral_amd import kv, model
from tests import op_refs as R
from tests.gpu_util import say, to_dev, to_np

pytestmark = pytest.mark.gpu

HQ, HKV, D, VOCAB = 8, 2, 64, 5000
SCALE = 1 / math.sqrt(D)


def new_pools(dev, nb, fmt):
    if fmt is None:
        return [torch.zeros((nb, HKV, 16, D), dtype=torch.bfloat16, device=dev) for _ in "kv"], {}
    pools = [torch.zeros((nb, HKV, 16, D), dtype=torch.uint8, device=dev) for _ in "kv"]
    scales = [torch.zeros((nb, HKV), device=dev) for _ in "kv"]
    return pools, dict(k_scale=scales[0], v_scale=scales[1], fmt=fmt)


def values(pools, extra):
    """The pools' rows in float64."""
    if not extra:
        return [p.float().cpu().numpy().astype(np.float64) for p in pools]
    return [R.dequantize(to_np(p), to_np(s), extra["fmt"])
            for p, s in zip(pools, (extra["k_scale"], extra["v_scale"]))]


@pytest.mark.parametrize("fmt", [None, "int8_block", "fp8_block"])
def test_decode_with_eviction(dev, fmt):
    """Three sequences decode 60 steps from prompts of their own; at steps 20 and 40
    each is cut to 32 rows in fresh blocks of the device block manager.  Attention,
    sums and kept rows are checked against 64 bits at every step, from the pools as
    the library wrote them."""
    say(f"decode with eviction fmt={fmt}")
    rng = np.random.default_rng(4)
    B, nb = 3, 48
    man = kv.DeviceBlockManager(nb, 16, max_seqs=2 * B, max_blocks_per_seq=8, device=dev)
    freq, mag = kv.rope_frequencies(D, 10000.0, scaling="parts", factor=4.0, original_context=64,
                                    device=dev)
    pools, extra = new_pools(dev, nb, fmt)
    sums = torch.zeros((nb, HKV, 16), device=dev)
    lens = np.array([33, 5, 48], np.int32)     # prompt tokens; then what the cache holds
    seen = lens.copy()                         # positions so far, evicted ones too
    slots = np.arange(B)
    man.reserve(slots, lens)

    def append(x, v, n_new, cache_lens, positions, tables):
        start = np.concatenate([[0], np.cumsum(n_new)]).astype(np.int32)
        if fmt is None:
            where = np.concatenate([np.arange(c - n, c) for c, n in zip(cache_lens, n_new)])
            owner = np.repeat(slots, n_new)
            at = man.slot_mapping(owner, where)
            q = torch.zeros((len(where), HQ, D), device=dev)
            kv.rope_append(q, x, v, positions, freq, *pools, at, magnitude=mag)
            return start
        kr = kv.rope(x, positions, freq, magnitude=mag)
        kv.append_block_q(*pools, extra["k_scale"], extra["v_scale"], kr, v, to_dev(start, dev),
                          tables, to_dev(np.asarray(cache_lens, np.int32), dev), fmt,
                          max_new=int(max(n_new)))
        return start

    def randn(*shape):
        return to_dev(rng.standard_normal(shape).astype(np.float32), dev)

    # the prompts, appended and attended by the prefill
    tables = man.batch_tables(slots, 8)
    total = int(lens.sum())
    pos = to_dev(np.concatenate([np.arange(n) for n in lens]).astype(np.int32), dev)
    start = append(randn(total, HKV, D), randn(total, HKV, D), lens, lens, pos, tables)
    q = kv.rope(randn(total, HQ, D), pos, freq, magnitude=mag)
    ctx = to_dev(lens, dev)
    if fmt is None:
        out = kv.prefill_attention(q, *pools, tables, to_dev(start, dev), ctx)
    else:
        out = kv.prefill_attention_q(q, *pools, extra["k_scale"], extra["v_scale"], tables,
                                     to_dev(start, dev), ctx, None, fmt)
    want, bound, _, _ = R.attend(to_np(q), *values(pools, extra), to_np(tables), lens, SCALE, lens,
                                 start)
    R.assert_within(to_np(out), want, bound, "prompt")

    history = [list(rng.integers(0, VOCAB, n)) for n in seen]
    prompts = to_dev(seen.copy(), dev)
    for step in range(60):
        if step in (20, 40):
            old = man.batch_tables(slots, 8)
            fresh = slots + B if slots[0] < B else slots - B
            ctx = to_dev(lens, dev)
            keep, left = kv.evict_select(sums, old, ctx, 32, sinks=2, recent=8)
            ref_keep, ref_left = R.select(to_np(sums), to_np(old), lens, 32, 2, 8)
            assert np.array_equal(to_np(keep), ref_keep) and np.array_equal(to_np(left), ref_left)
            man.reserve(fresh, ref_left)
            to = man.batch_tables(fresh, 8)
            before = [to_np(t).copy() for t in (*pools, sums)]
            scales = [to_np(extra[n]).copy() if fmt else None for n in ("k_scale", "v_scale")]
            kv.evict_compact(*pools, keep, left, old, to, weights=sums, **extra)
            R.compact(before[0], before[1], *scales, before[2], ref_keep, ref_left, to_np(old),
                      to_np(to), fmt)
            for got, ref in zip((*pools, sums), before):
                assert np.array_equal(to_np(got).view(np.uint8), ref.view(np.uint8))
            man.free(slots)
            slots, lens = fresh, ref_left.copy()
        lens += 1
        man.reserve(slots, lens)
        tables = man.batch_tables(slots, 8)
        grown = to_np(tables)[np.arange(B), (lens - 1) // 16][(lens - 1) % 16 == 0]
        sums[torch.from_numpy(grown.astype(np.int64)).to(dev)] = 0   # blocks handed out now
        pos = to_dev(seen.astype(np.int32), dev)
        append(randn(B, HKV, D), randn(B, HKV, D), np.ones(B, int), lens, pos, tables)
        q = kv.rope(randn(B, HQ, D), pos, freq, magnitude=mag)
        seen += 1
        w0, fk_fv = to_np(sums).astype(np.float64), values(pools, extra)
        out = kv.decode_attention_weights(q, *pools, sums, tables, to_dev(lens, dev), **extra)
        want, bound, ws, wb = R.attend(to_np(q), *fk_fv, to_np(tables), lens, SCALE)
        R.assert_within(to_np(out), want, bound, f"step {step}")
        wbound, tb = np.abs(w0) * 2.0 ** -23, to_np(tables)
        for b in range(B):
            p = np.arange(lens[b])
            w0[tb[b, p // 16], :, p % 16] += ws[b].T
            wbound[tb[b, p // 16], :, p % 16] += (wb[b] + 2.0 ** -22 * ws[b]).T
        R.assert_within(to_np(sums), w0, wbound + 1e-30, f"sums {step}")
        # the step's tokens: no token three times, a grammar of every third word
        logits = randn(B, VOCAB)
        words = np.zeros(-(-VOCAB // 32) * 32, bool)
        words[step % 3:VOCAB:3] = True
        allowed = np.packbits(words, bitorder="little").view(np.int32)
        ends = np.concatenate([[0], np.cumsum([len(h) for h in history])]).astype(np.int32)
        args = dict(history=np.concatenate(history).astype(np.int32), start=ends,
                    prompt=to_np(prompts), repetition=np.full(B, 1.2, np.float32),
                    presence=np.full(B, 100.0, np.float32),
                    allowed=np.tile(allowed, (B, 1)))
        names = dict(start="history_start", prompt="prompt_lens")
        _, pick = model.process_logits(logits, **{names.get(k, k): to_dev(v, dev)
                                                  for k, v in args.items()}, out=logits.clone())
        _, picks, _ = R.logits(to_np(logits), **args)
        assert np.array_equal(to_np(pick), picks)
        for b in range(B):
            assert picks[b] % 3 == step % 3
            history[b].append(int(picks[b]))
    made = [h[int(n):] for h, n in zip(history, to_np(prompts))]
    assert all(len(set(m)) == len(m) for m in made)   # a presence of 100 forbids repeats
    assert man.status()[1] == 0
    man.close()


@pytest.mark.parametrize("fmt", [None, "int8_block", "fp8_block"])
def test_step_in_a_graph(dev, fmt):
    """A step captured once and replayed, with eager work on the same pools and
    workspaces of its own in between: the same bits as the eager step."""
    say(f"graph fmt={fmt}")
    rng = np.random.default_rng(11)
    B, nb, mbs = 4, 260, 64
    lens = np.array([1000, 17, 0, 513], np.int32)
    tables = np.full((B, mbs), -1, np.int32)
    o = 0
    for b, n in enumerate(lens):
        m = -(-int(n) // 16)
        tables[b, :m] = np.arange(o, o + m)
        o += m
    dst = np.full((B, 4), -1, np.int32)
    for b, n in enumerate(lens):
        m = -(-min(int(n), 50) // 16)
        dst[b, :m] = np.arange(o, o + m)
        o += m
    pools, extra = new_pools(dev, nb, fmt)
    if fmt is None:
        for p in pools:
            p.copy_(torch.randn(p.shape, device=dev))
    else:
        for p in pools:
            p.random_(0, 100)
        for s in (extra["k_scale"], extra["v_scale"]):
            s.copy_(2.0 ** -torch.randint(5, 9, s.shape, device=dev).float())
    first = [p.clone() for p in pools]
    scales = [extra[n].clone() for n in ("k_scale", "v_scale")] if fmt else []
    w0 = torch.rand((nb, HKV, 16), device=dev)
    sums = w0.clone()
    freq, _ = kv.rope_frequencies(D, device=dev)
    q0, kn, vn = (to_dev(rng.standard_normal((B, h, D)).astype(np.float32), dev)
                  for h in (HQ, HKV, HKV))
    pos, ctx, tab, to = (to_dev(a, dev) for a in (lens - 1, lens, tables, dst))
    slots = to_dev(np.array([tables[b, (n - 1) // 16] * 16 + (n - 1) % 16 if n else -1
                             for b, n in enumerate(lens)], np.int64), dev)
    start = to_dev(np.array([0, 1, 2, 2, 3], np.int32), dev)
    logits = to_dev(rng.standard_normal((B, 9000)).astype(np.float32), dev)
    hist = to_dev(rng.integers(0, 9000, 100).astype(np.int32), dev)
    ends = to_dev(np.array([0, 50, 50, 80, 100], np.int32), dev)
    pen = to_dev(np.full(B, 1.3, np.float32), dev)

    def step():
        if fmt is None:
            q = kv.rope_append(q0, kn, vn, pos, freq, *pools, slots)
        else:
            q = kv.rope(q0, pos, freq)
            kr = kv.rope(kn, pos, freq)
            kv.append_block_q(*pools, extra["k_scale"], extra["v_scale"], kr, vn, start, tab, ctx,
                              fmt, max_new=1)
        a = kv.decode_attention_weights(q, *pools, sums, tab, ctx, **extra)
        keep, left = kv.evict_select(sums, tab, ctx, 50, sinks=2, recent=10)
        kv.evict_compact(*pools, keep, left, tab, to, weights=sums, **extra)
        y, pick = model.process_logits(logits, history=hist, history_start=ends, repetition=pen)
        return a, keep, left, y, pick

    def reset():
        for p, f in zip(pools, first):
            p.copy_(f)
        for n, s in zip(("k_scale", "v_scale"), scales):
            extra[n].copy_(s)
        sums.copy_(w0)

    def state(got):
        return [t.clone() for t in (*got, *pools, sums)]

    reset()
    eager = state(step())
    reset()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        reset()
        if i % 2:   # the program's own work between replays
            step()
            torch.cuda.synchronize()
            reset()
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(state(got), eager):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), i


def test_two_streams_at_once(dev):
    """Two streams with their own inputs and workspaces, many calls in flight:
    each gets what it gets alone."""
    say("two streams")
    rng = np.random.default_rng(3)
    sets = []
    for i in range(2):
        nb, lens = 300, np.array([2000, 900 + 64 * i, 700], np.int32)
        tables = np.full((3, 128), -1, np.int32)
        o = 0
        for b, n in enumerate(lens):
            m = -(-int(n) // 16)
            tables[b, :m] = np.arange(o, o + m)
            o += m
        pools = [to_dev(rng.standard_normal((nb, HKV, 16, D)).astype(np.float32), dev).bfloat16()
                 for _ in "kv"]
        sets.append(dict(pools=pools, tab=to_dev(tables, dev), ctx=to_dev(lens, dev),
                         q=to_dev(rng.standard_normal((3, HQ, D)).astype(np.float32), dev),
                         w=torch.zeros((nb, HKV, 16), device=dev),
                         x=to_dev(rng.standard_normal((3, 20000)).astype(np.float32), dev)))

    def work(s):
        s["w"].zero_()
        a = kv.decode_attention_weights(s["q"], *s["pools"], s["w"], s["tab"], s["ctx"])
        keep, left = kv.evict_select(s["w"], s["tab"], s["ctx"], 200, sinks=4, recent=20)
        y, pick = model.process_logits(s["x"])
        return a, s["w"].clone(), keep, left, y, pick

    alone = [work(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(work(sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for run in got[i]:
            for a, b in zip(run, alone[i]):
                assert torch.equal(a, b)


def small(dev):
    """Tensors of a small call of every entry point, by name, and the calls."""
    rng = np.random.default_rng(8)
    lens = np.array([20, 37], np.int32)
    tables = np.array([[0, 1, -1], [2, 3, 4]], np.int32)
    t = {n: to_dev(rng.standard_normal(s).astype(np.float32), dev)
         for n, s in dict(q=(2, HQ, D), kn=(2, HKV, D), vn=(2, HKV, D), x=(2, 5000)).items()}
    t.update(tab=to_dev(tables, dev), ctx=to_dev(lens, dev), pos=to_dev(lens - 1, dev),
             dst=to_dev(np.array([[5, 6], [7, 8]], np.int32), dev),
             start=to_dev(np.array([0, 1, 2], np.int32), dev),
             slots=to_dev(np.array([19, 4 * 16 + 4], np.int64), dev),
             k=torch.zeros((9, HKV, 16, D), device=dev), v=torch.zeros((9, HKV, 16, D), device=dev),
             w=torch.zeros((9, HKV, 16), device=dev))
    t.update({n: torch.zeros((9, HKV, 16, D), dtype=torch.uint8, device=dev) for n in ("k8", "v8")})
    t.update({n: torch.zeros((9, HKV), device=dev) for n in ("ks", "vs")})
    freq, _ = kv.rope_frequencies(D, device=dev)

    def run():
        a = kv.rope_append(t["q"], t["kn"], t["vn"], t["pos"], freq, t["k"], t["v"], t["slots"])
        b = kv.rope(t["kn"], t["pos"], freq)
        q8 = (t["k8"], t["v8"], t["ks"], t["vs"])
        kv.append_block_q(*q8, b, t["vn"], t["start"], t["tab"], t["ctx"], max_new=1)
        c = kv.decode_attention_q(t["q"], *q8, t["tab"], t["ctx"], fmt="int8_block")
        e = kv.prefill_attention_q(t["q"], *q8, t["tab"], t["start"], t["ctx"], max_q_len=1)
        f = kv.decode_attention_weights(t["q"], t["k"], t["v"], t["w"], t["tab"], t["ctx"])
        keep, left = kv.evict_select(t["w"], t["tab"], t["ctx"], 18, sinks=1, recent=2)
        kv.evict_compact(t["k"], t["v"], keep, left, t["tab"], t["dst"], weights=t["w"])
        y, pick = model.process_logits(t["x"])
        return [u.clone() for u in (a, b, c, e, f, keep, left, y, pick, t["k"], t["v"], t["w"],
                                    t["k8"], t["v8"], t["ks"], t["vs"])]

    return t, freq, run


def test_on_a_device_that_is_not_current(dev, monkeypatch):
    """The calls make their tensors' device the current one: seen from another
    current device (here as far as the front end can tell) the results are the same."""
    say("another current device")
    want = small(dev)[2]()
    seen = []
    real = torch.cuda.device
    monkeypatch.setattr(kv, "_current_device", lambda: 1)
    monkeypatch.setattr(torch.cuda, "device", lambda d: seen.append(d) or real(d))
    got = small(dev)[2]()
    assert seen == [0] * 9
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_front_end_refuses_outputs_and_workspaces(dev):
    """Buffers a kernel would write past, or that the device cannot reach."""
    say("refusals")
    t, freq, _ = small(dev)
    q8 = (t["k8"], t["v8"], t["ks"], t["vs"])
    for bad, err in ((t["q"][:1].clone(), ValueError), (t["q"].double(), TypeError),
                     (t["q"].cpu(), ValueError)):
        with pytest.raises(err):
            kv.prefill_attention_q(t["q"], *q8, t["tab"], t["start"], t["ctx"], max_q_len=1, out=bad)
        with pytest.raises(err):
            kv.decode_attention_weights(t["q"], t["k"], t["v"], t["w"], t["tab"], t["ctx"], out=bad)
        with pytest.raises((ValueError, TypeError)):
            kv.rope(t["q"], t["pos"], freq, out=bad)
        with pytest.raises(ValueError):
            kv.rope_append(t["q"], t["kn"], t["vn"], t["pos"], freq, t["k"], t["v"], t["slots"],
                           out=bad)
    host = torch.zeros(1 << 20, dtype=torch.uint8)
    with pytest.raises(ValueError):
        kv.decode_attention_weights(t["q"], t["k"], t["v"], t["w"], t["tab"], t["ctx"],
                                    workspace=host)
    with pytest.raises(ValueError):
        model.process_logits(t["x"], workspace=host)
    with pytest.raises(ValueError):
        model.process_logits(t["x"], out=t["x"][:, :4999].clone())


def test_one_token_of_any_stride(dev):
    """One token's rows may come from tensors of different token strides."""
    say("one token")
    t, freq, _ = small(dev)
    wide = torch.zeros((1, HKV + 3, D), device=dev)
    wide[:, :HKV] = t["vn"][:1]
    pools = [[torch.zeros_like(t["k"]) for _ in "kv"] for _ in range(2)]
    for v, p in ((t["vn"][:1], pools[0]), (wide[:, :HKV], pools[1])):
        kv.rope_append(t["q"][:1], t["kn"][:1], v, t["pos"][:1], freq, *p, t["slots"][:1])
    assert all(torch.equal(a, b) for a, b in zip(*pools)) and pools[0][1].any()


@pytest.mark.parametrize("fmt", [None, "int8_block", "fp8_block"])
def test_pools_past_32_bit_offsets(dev, fmt):
    """Two layers of 70,000 blocks of 8 x 128 (2.3e9 elements), the blocks in use at their
    ends: the same bits as in pools that hold only those."""
    say(f"large pools fmt={fmt}")
    hkv, d, hq, big = 8, 128, 16, 70_000
    ids = np.array([big - 1, 3, big - 2, 65_600, big - 5, 1, big - 9, 40_001, big - 7], np.int64)
    few = len(ids)
    ctx = np.array([33, 20], np.int32)
    tab = np.array([[0, 1, 2], [3, 4, -1]], np.int32)      # places in ids
    dst = np.array([[5, 6], [7, 8]], np.int32)
    rng = np.random.default_rng(2)
    total = int(ctx.sum())
    kn, vn = (to_dev(rng.standard_normal((2, total, hkv, d)).astype(np.float32), dev) for _ in "kv")
    q = to_dev(rng.standard_normal((2, hq, d)).astype(np.float32), dev)
    qq = to_dev(rng.standard_normal((total, hq, d)).astype(np.float32), dev)
    start = to_dev(np.array([0, 33, 53], np.int32), dev)
    gctx = to_dev(ctx, dev)
    freq, _ = kv.rope_frequencies(d, device=dev)
    pos = to_dev(np.concatenate([np.arange(n) for n in ctx]).astype(np.int32), dev)
    results = []
    for nb in (few, big):
        name = np.arange(few) if nb == few else ids
        to = lambda t: to_dev(np.where(t >= 0, name[t], -1).astype(np.int32), dev)
        dt = torch.bfloat16 if fmt is None else torch.uint8
        k, v = (torch.zeros((2, nb, hkv, 16, d), dtype=dt, device=dev) for _ in "kv")
        w = torch.zeros((2, nb, hkv, 16), device=dev)
        ks, vs = (torch.zeros((2, nb, hkv), device=dev) for _ in "kv")
        gt, gd = to(tab), to(dst)
        out = []
        if fmt is None:
            slots = np.concatenate([name[tab[b, np.arange(n) // 16]] * 16 + np.arange(n) % 16
                                    for b, n in enumerate(ctx)])
            for i in range(2):
                out.append(kv.rope_append(qq, kn[i], vn[i], pos, freq, k[i], v[i],
                                          to_dev(slots.astype(np.int64), dev)))
            sc = [{}] * 2
        else:
            kv.append_block_q(k, v, ks, vs, kn, vn, start, gt, gctx, fmt)
            sc = [dict(k_scale=ks[i], v_scale=vs[i], fmt=fmt) for i in range(2)]
        for i in range(2):
            out.append(kv.decode_attention_weights(q, k[i], v[i], w[i], gt, gctx, **sc[i]))
            if fmt:
                out.append(kv.decode_attention_q(q, k[i], v[i], ks[i], vs[i], gt, gctx, fmt=fmt))
                out.append(kv.prefill_attention_q(qq, k[i], v[i], ks[i], vs[i], gt, start, gctx,
                                                  fmt=fmt))
                out += kv.gather_q(k[i], v[i], ks[i], vs[i], gt, gctx, fmt=fmt)
        keep, left = kv.evict_select(w, gt, gctx, 18, sinks=2, recent=3)
        kv.evict_compact(k, v, keep, left, gt, gd, weights=w,
                         **(dict(k_scale=ks, v_scale=vs, fmt=fmt) if fmt else {}))
        at = torch.from_numpy(name).to(dev)
        out += [keep, left] + [t[:, at].contiguous() for t in (k, v, w, ks, vs)]
        results.append(out)
        del k, v
    assert results[0][-5].any() and results[0][-3].any()
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_a_smaller_v_pool_is_refused(dev):
    """The kernels index V by K's shape."""
    say("smaller v pool")
    t, freq, _ = small(dev)
    v8, vs, v = t["v8"][:5].clone(), t["vs"][:5].clone(), t["v"][:5].clone()
    q8 = (t["k8"], v8, t["ks"], vs)
    keep = torch.zeros((2, HKV, 4), dtype=torch.int32, device=dev)
    left = torch.full((2,), 4, dtype=torch.int32, device=dev)
    for call in (
            lambda: kv.append_block_q(*q8, t["kn"], t["vn"], t["start"], t["tab"], t["ctx"]),
            lambda: kv.decode_attention_q(t["q"], *q8, t["tab"], t["ctx"], fmt="int8_block"),
            lambda: kv.prefill_attention_q(t["q"], *q8, t["tab"], t["start"], t["ctx"]),
            lambda: kv.gather_q(*q8, t["tab"], t["ctx"], fmt="fp8_block"),
            lambda: kv.decode_attention_weights(t["q"], t["k"], v, t["w"], t["tab"], t["ctx"]),
            lambda: kv.evict_compact(t["k"], v, keep, left, t["tab"], t["dst"]),
            lambda: kv.rope_append(t["q"], t["kn"], t["vn"], t["pos"], freq, t["k"], v, t["slots"])):
        with pytest.raises(ValueError):
            call()
