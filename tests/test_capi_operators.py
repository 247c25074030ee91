"""CPU checks of the operators around the cache: refusals on the host before any
launch, workspace sizes, and the frequency tables."""
import math

import numpy as np
import pytest

from rustral_amd import _lib, kv
from rustral_amd._lib import (RKV_BF16, RKV_ERR_INVALID_ARG, RKV_ERR_UNSUPPORTED,
                              RKV_ERR_WORKSPACE, RKV_F32, RKV_FP8, RKV_FP8_BLOCK, RKV_I8,
                              RKV_I8_BLOCK)

BAD, NOT_BUILT, WORK = RKV_ERR_INVALID_ARG, RKV_ERR_UNSUPPORTED, RKV_ERR_WORKSPACE


def call(name, defaults, **kw):
    args = dict(defaults)
    unknown = set(kw) - set(args)
    assert not unknown, unknown
    args.update(kw)
    return getattr(_lib.lib(), name)(*args.values())


ROPE = dict(out=16, x=32, positions=16, inv_freq=16, n=2, heads=4, d=64, rot=64, ots=256, ohs=64,
            ts=256, hs=64, inter=0, mag=1.0, stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(d=60), NOT_BUILT), (dict(d=2048, rot=64), NOT_BUILT), (dict(rot=63), BAD),
    (dict(rot=66), BAD), (dict(rot=0), BAD), (dict(heads=0), BAD), (dict(n=-1), BAD),
    (dict(n=1 << 31), BAD), (dict(x=None), BAD), (dict(out=None), BAD),
    (dict(positions=None), BAD), (dict(inv_freq=None), BAD), (dict(ts=255), BAD),
    (dict(ohs=66), BAD), (dict(x=8), BAD), (dict(out=32, ots=512), BAD),
])
def test_rope_refuses(kw, code):
    assert call("rkv_rope", ROPE, **kw) == code
    assert _lib.lib().rkv_last_error().decode()


def test_rope_of_no_tokens_is_a_no_op():
    assert call("rkv_rope", ROPE, n=0, x=None, out=None) == 0


ROPE_APPEND = dict(q_out=16, k=16, v=16, ks=None, vs=None, q=32, kn=16, vn=16, ots=256, ohs=64,
                   qts=256, qhs=64, sts=128, shs=64, positions=16, inv_freq=16, slots=16, n=2,
                   hq=4, hkv=2, d=64, rot=64, inter=0, mag=1.0, bs=16, nb=8, dt=RKV_BF16,
                   stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(dt=RKV_I8), BAD), (dict(dt=RKV_I8_BLOCK), BAD), (dict(dt=9), BAD),
    (dict(dt=RKV_FP8, ks=16, vs=16, d=80, rot=64), NOT_BUILT), (dict(hkv=0), BAD),
    (dict(bs=0), BAD), (dict(nb=-1), BAD), (dict(slots=None), BAD), (dict(vn=None), BAD),
    (dict(shs=62), BAD), (dict(kn=20), BAD), (dict(d=68), NOT_BUILT), (dict(rot=128), BAD),
    (dict(q_out=32, ots=512), BAD),
])
def test_rope_append_refuses(kw, code):
    assert call("rkv_rope_append", ROPE_APPEND, **kw) == code


APPEND = dict(k=16, v=16, ks=16, vs=16, pls=0, kn=16, vn=16, sls=0, sts=128, shs=64, start=16,
              tab=16, mbs=4, ctx=16, B=2, layers=1, hkv=2, d=64, bs=16, nb=8, max_new=3,
              dt=RKV_I8_BLOCK, stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(dt=RKV_I8), BAD), (dict(dt=RKV_BF16), BAD), (dict(bs=32), NOT_BUILT),
    (dict(d=48), NOT_BUILT), (dict(B=-1), BAD), (dict(max_new=-1), BAD), (dict(mbs=-1), BAD),
    (dict(hkv=0), BAD), (dict(ks=None), BAD), (dict(start=None), BAD), (dict(ctx=None), BAD),
    (dict(sts=127), BAD), (dict(vn=24), BAD), (dict(layers=2, pls=100), BAD),
    (dict(B=70000), BAD),
])
def test_append_block_q_refuses(kw, code):
    assert call("rkv_append_block_q", APPEND, **kw) == code


@pytest.mark.parametrize("kw", [dict(B=0), dict(max_new=0), dict(layers=0), dict(mbs=0)])
def test_append_block_q_of_nothing(kw):
    assert call("rkv_append_block_q", APPEND, k=None, **kw) == 0


PREFILL = dict(out=16, q=16, k=16, v=16, ks=16, vs=16, tab=16, mbs=4, start=16, ctx=16, B=2, hq=8,
               hkv=2, d=64, bs=16, nb=8, max_q=3, scale=0.1, dt=RKV_FP8_BLOCK, stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(dt=RKV_I8), NOT_BUILT), (dict(dt=RKV_FP8), NOT_BUILT), (dict(dt=RKV_F32), BAD),
    (dict(d=32), NOT_BUILT), (dict(hq=6), NOT_BUILT), (dict(hq=7), BAD), (dict(bs=8), NOT_BUILT),
    (dict(ks=None), BAD), (dict(nb=0), BAD), (dict(max_q=-1), BAD), (dict(out=24), BAD),
])
def test_prefill_attention_q_refuses(kw, code):
    assert call("rkv_prefill_attention_q", PREFILL, **kw) == code


def test_decode_attention_q_takes_block_scales_only_with_scale_pools():
    args = dict(out=16, q=16, k=16, v=16, ks=16, vs=16, tab=16, mbs=4, ctx=16, B=2, hq=8, hkv=2,
                d=128, bs=16, nb=10, maxc=64, scale=0.1, dt=RKV_I8_BLOCK, ps=0, ws=None, wsb=0,
                stream=None)
    for kw, code in [(dict(ks=None), BAD), (dict(d=32), NOT_BUILT), (dict(dt=6), BAD),
                     (dict(dt=RKV_BF16), BAD), (dict(ps=100), NOT_BUILT),
                     (dict(maxc=4096, mbs=256), WORK)]:
        assert call("rkv_decode_attention_q", args, **kw) == code, kw
    gather = dict(ko=16, vo=16, k=16, v=16, ks=16, vs=16, tab=16, mbs=4, ctx=16, off=None, B=2,
                  hkv=2, d=64, bs=32, nb=8, max_ctx=64, dt=RKV_FP8_BLOCK, stream=None)
    assert call("rkv_gather_q", gather) == NOT_BUILT      # 16-row tiles
    assert call("rkv_gather_q", gather, bs=16, dt=6) == BAD


WEIGHTS = dict(out=16, w=16, q=16, k=16, v=16, ks=None, vs=None, tab=16, mbs=4, ctx=16, B=2, hq=8,
               hkv=2, d=64, bs=16, nb=8, maxc=64, scale=0.1, dt=RKV_BF16, ws=256, wsb=1 << 20,
               stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(w=None), BAD), (dict(dt=RKV_I8_BLOCK), BAD), (dict(hq=6), NOT_BUILT), (dict(hq=7), BAD),
    (dict(d=48), NOT_BUILT), (dict(bs=32), NOT_BUILT), (dict(ws=None), WORK), (dict(wsb=100), WORK),
    (dict(ws=8), BAD), (dict(nb=0), BAD), (dict(maxc=-1), BAD), (dict(q=None), BAD),
    (dict(hkv=0), BAD),
])
def test_decode_attention_weights_refuses(kw, code):
    assert call("rkv_decode_attention_weights", WEIGHTS, **kw) == code


def test_decode_attention_weights_workspace_holds_every_shape():
    """The size function's answer is enough for every cap a call may have up to
    max_context (the check is made before any launch: a launch would need the
    GPU, so what is looked at is that no call is refused for its workspace)."""
    L = _lib.lib()
    for B, hkv, g in [(1, 1, 1), (1, 8, 4), (2, 8, 4), (3, 2, 8), (16, 1, 4), (64, 8, 4), (300, 1, 1)]:
        for maxc in (1, 16, 128, 129, 512, 513, 640, 1000, 4096, 16384, 32768, 65536, 131072):
            need = L.rkv_decode_weights_workspace_bytes(B, g * hkv, hkv, 128, maxc)
            assert need > 0
            for cap in {maxc, max(1, maxc - 1), max(1, maxc // 2), min(maxc, 520)}:
                # a null query is reported after the workspace of the partials, the
                # scores' share is checked by arithmetic
                p = L.rkv_decode_partition_size_for(0, B, g * hkv, hkv, 128, RKV_BF16, cap)
                p = 128 if cap <= 128 else 512 if cap <= 512 else p
                parts = -(-cap // p)
                rows = B * g * hkv
                pad = lambda x: -(-x // 256) * 256  # noqa: E731
                used = pad(rows * parts * 128 * 4) + pad(rows * parts * 8) + rows * parts * p * 4
                assert used <= need, (B, hkv, g, maxc, cap)


SELECT = dict(keep=16, lens=16, w=16, wls=0, tab=16, mbs=4, ctx=16, B=2, layers=1, hkv=2, bs=16,
              nb=8, budget=8, sinks=2, recent=4, maxc=64, stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(budget=0), BAD), (dict(budget=5), BAD), (dict(sinks=-1), BAD), (dict(recent=-1), BAD),
    (dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1), BAD), (dict(bs=8), NOT_BUILT), (dict(hkv=0), BAD),
    (dict(B=-1), BAD), (dict(keep=None), BAD), (dict(lens=None), BAD), (dict(w=None), BAD),
    (dict(tab=None), BAD), (dict(w=8), BAD), (dict(layers=2, wls=6), BAD), (dict(maxc=-1), BAD),
    (dict(B=70000), BAD), (dict(mbs=1 << 28), BAD),
])
def test_evict_select_refuses(kw, code):
    assert call("rkv_evict_select", SELECT, **kw) == code


COMPACT = dict(k=16, v=16, ks=None, vs=None, w=None, pls=0, wls=0, keep=16, lens=16, budget=8,
               src=16, sb=4, dst=16, db=2, B=2, layers=1, hkv=2, d=64, bs=16, nb=8, dt=RKV_BF16,
               stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(dt=-1), BAD), (dict(dt=6), BAD), (dict(dt=RKV_I8), BAD), (dict(dt=RKV_I8_BLOCK), BAD),
    (dict(dt=RKV_FP8, ks=16, vs=16, d=80), NOT_BUILT), (dict(d=60), NOT_BUILT),
    (dict(bs=32), NOT_BUILT), (dict(budget=0), BAD), (dict(keep=None), BAD), (dict(dst=None), BAD),
    (dict(k=24), BAD), (dict(layers=2, pls=100), BAD),
    (dict(layers=2, pls=1040, dt=RKV_I8_BLOCK, ks=16, vs=16), BAD), (dict(B=70000), BAD),
    (dict(sb=-1), BAD),
])
def test_evict_compact_refuses(kw, code):
    assert call("rkv_evict_compact", COMPACT, **kw) == code


LOGITS = dict(out=16, ots=100, pick=16, x=32, ts=100, rows=2, n=100, hist=16, hs=16, pl=None,
              rep=16, freq=None, pres=None, bi=None, bv=None, bst=None, allowed=None, als=0,
              ws=None, wsb=0, stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(n=0), BAD), (dict(rows=-1), BAD), (dict(rows=65536), BAD), (dict(x=None), BAD),
    (dict(out=None, pick=None), BAD), (dict(hist=None), BAD), (dict(hs=None), BAD),
    (dict(bi=16), BAD), (dict(bi=16, bv=16), BAD), (dict(ts=99), BAD), (dict(ots=99), BAD),
    (dict(allowed=16, als=3), BAD), (dict(out=32, ots=104), BAD),
    (dict(n=5000, ts=5000, ots=5000), WORK), (dict(n=5000, ts=5000, ots=5000, ws=16, wsb=8), WORK),
    (dict(n=5000, ts=5000, ots=5000, ws=12, wsb=64), BAD), (dict(n=2 ** 31 - 1, ts=2 ** 31), BAD),
])
def test_process_logits_refuses(kw, code):
    assert call("rkv_process_logits", LOGITS, **kw) == code


def test_process_logits_workspace():
    L = _lib.lib()
    assert L.rkv_process_logits_workspace_bytes(1, 4096) == 0
    assert L.rkv_process_logits_workspace_bytes(3, 4097) == 3 * 2 * 8
    assert L.rkv_process_logits_workspace_bytes(0, 100000) == 0


# ---- the front end's own checks (shapes the kernels index by) -----------------------------

def test_front_end_refuses_host_tensors_and_unknown_formats():
    import torch
    from rustral_amd import model
    z = torch.zeros(4, 2, 64)
    with pytest.raises(ValueError, match="device"):
        kv.rope(z, torch.zeros(4, dtype=torch.int32), torch.zeros(32, dtype=torch.float64))
    with pytest.raises(ValueError, match="scaling"):
        kv.rope_frequencies(64, scaling="other")
    for fn in (kv._bcode, kv._anycode):
        with pytest.raises(ValueError, match="format"):
            fn("int4")
    with pytest.raises(ValueError, match="format"):
        kv._bcode("int8")
    with pytest.raises(ValueError, match="device"):
        model.process_logits(torch.zeros(2, 8))
    with pytest.raises(ValueError, match="device"):
        kv.evict_select(torch.zeros(4, 2, 16), None, None, 8)


# ---- frequency tables ------------------------------------------------------------------------

def table(rot, base=10000.0, **kw):
    f, m = kv.rope_frequencies(rot, base, device="cpu", **kw)
    return f.numpy(), m


@pytest.mark.parametrize("rot,base", [(2, 10000.0), (64, 10000.0), (128, 500000.0), (100, 10.0)])
def test_frequencies_plain_linear_base(rot, base):
    i = np.arange(rot // 2)
    want = base ** (-2.0 * i / rot)
    got, m = table(rot, base)
    assert m == 1.0 and np.allclose(got, want, rtol=1e-14)
    got, m = table(rot, base, scaling="linear", factor=8)
    assert m == 1.0 and np.allclose(got, want / 8, rtol=1e-14)
    if rot > 2:
        got, m = table(rot, base, scaling="base", factor=4)
        wide = base * 4 ** (rot / (rot - 2))
        assert m == 1.0 and np.allclose(got, wide ** (-2.0 * i / rot), rtol=1e-13)
        # the slowest pair turns factor times slower, the fastest as before
        assert np.isclose(got[-1], want[-1] / 4, rtol=1e-12) and got[0] == 1.0


def test_frequencies_by_parts():
    rot, base, factor, ctx = 128, 10000.0, 16.0, 4096
    plain, _ = table(rot, base)
    got, m = table(rot, base, scaling="parts", factor=factor, original_context=ctx)
    assert np.isclose(m, 0.1 * math.log(factor) + 1, rtol=1e-6)
    turns = ctx * plain / (2 * math.pi)
    # a pair well above 32 turns keeps its frequency, one well below 1 is divided
    assert np.allclose(got[turns > 40], plain[turns > 40], rtol=1e-13)
    assert np.allclose(got[turns < 0.8], plain[turns < 0.8] / factor, rtol=1e-13)
    share = got / plain
    assert (np.diff(share) <= 1e-12).all() and ((share > 1 / factor - 1e-9) & (share <= 1)).all()


def test_frequencies_in_bands():
    rot, base, factor, ctx, low, high = 128, 500000.0, 8.0, 8192, 1.0, 4.0
    plain, _ = table(rot, base)
    got, m = table(rot, base, scaling="bands", factor=factor, original_context=ctx, low=low,
                   high=high)
    assert m == 1.0
    for f, g in zip(plain, got):
        wave = 2 * math.pi / f
        if wave < ctx / high:
            want = f
        elif wave > ctx / low:
            want = f / factor
        else:
            smooth = (ctx / wave - low) / (high - low)
            want = (1 - smooth) * f / factor + smooth * f
        assert np.isclose(g, want, rtol=1e-12)


@pytest.mark.parametrize("kw", [
    dict(rot=63), dict(rot=0), dict(rot=64, base=1.0), dict(rot=64, scaling="linear", factor=0.5),
    dict(rot=64, scaling="linear", factor=math.inf), dict(rot=64, scaling="linear", factor=math.nan),
    dict(rot=64, scaling="parts", factor=2), dict(rot=2, scaling="base", factor=2),
    dict(rot=64, scaling="bands", factor=2, original_context=100, low=4, high=4),
    dict(rot=64, scaling="bands", factor=2, original_context=100, low=0, high=4),
])
def test_frequencies_refuse(kw):
    with pytest.raises(_lib.RkvError):
        table(**kw)
