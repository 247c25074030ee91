"""Rotary positions on the GPU: kv.rope against the formula in 64 bits, and
kv.rope_append against rope followed by append / append_q, bit for bit."""
import numpy as np
import pytest
import torch

from rustral_amd import _lib, kv
from tests import op_refs as R
from tests.gpu_util import say, to_dev, to_np

pytestmark = pytest.mark.gpu


def freqs(dev, rot, base=10000.0):
    return kv.rope_frequencies(rot, base, device=dev)[0]


def positions(rng, t, far):
    p = rng.integers(0, far, t).astype(np.int32)
    p[:2] = (0, far - 1)[:t]
    return p


# D, rotary_dim, heads, tokens: whole heads, parts of them, pair offsets off a
# 16-byte boundary (half = 3, 10, 31), one token, odd head widths
SHAPES = [(128, 128, 8, 1), (128, 128, 40, 67), (64, 32, 3, 300), (64, 6, 5, 9), (80, 20, 2, 33),
          (64, 62, 7, 17), (32, 32, 1, 2100), (192, 192, 4, 5), (128, 2, 2, 3), (8, 8, 3, 70),
          (1024, 512, 2, 3), (96, 96, 9, 2050)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot,h,t", SHAPES)
def test_rope_against_the_formula(dev, d, rot, h, t, interleaved):
    say(f"rope d={d} rot={rot} h={h} t={t} interleaved={interleaved}")
    rng = np.random.default_rng(d + rot + h + t)
    x = rng.standard_normal((t, h, d)).astype(np.float32)
    pos = positions(rng, t, 1 << 20)
    f = freqs(dev, rot)
    got = to_np(kv.rope(to_dev(x, dev), to_dev(pos, dev), f, interleaved=interleaved,
                        magnitude=1.25))
    want = R.rope(x, pos, f.cpu().numpy(), interleaved, 1.25)
    R.assert_within(got, want, R.rope_bound(x, pos, f.cpu().numpy(), interleaved, 1.25), "rope")
    assert np.array_equal(got[..., rot:].view(np.uint32), x[..., rot:].view(np.uint32))


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_far_positions(dev, interleaved):
    """int32's whole range, negative positions too: angles of 2^31 rad."""
    say(f"rope far interleaved={interleaved}")
    rng = np.random.default_rng(5)
    pos = np.array([0, 1, -1, 2**31 - 1, -2**31, 2**30 + 7, 123456789, -5], np.int32)
    x = rng.standard_normal((len(pos), 2, 64)).astype(np.float32)
    f = freqs(dev, 64, 500000.0)
    got = to_np(kv.rope(to_dev(x, dev), to_dev(pos, dev), f, interleaved=interleaved))
    R.assert_within(got, R.rope(x, pos, f.cpu().numpy(), interleaved),
                    R.rope_bound(x, pos, f.cpu().numpy(), interleaved), "far")
    back = kv.rope(to_dev(got, dev), to_dev(-pos, dev), f, interleaved=interleaved)
    keep = pos != -2**31  # its negative is not an int32
    assert np.abs(to_np(back) - x)[keep].max() < 1e-5


def test_rope_position_zero_and_passed_elements_are_exact(dev):
    """Position 0 turns nothing; elements past rotary_dim pass whatever they are."""
    say("rope exact")
    x = np.random.default_rng(0).standard_normal((3, 2, 64)).astype(np.float32)
    x[0, 0, 40], x[1, 1, 41], x[2, 0, 63], x[2, 1, 50] = np.inf, np.nan, -0.0, -np.inf
    for inter in (False, True):
        for rot in (32, 36, 2):
            got = to_np(kv.rope(to_dev(x, dev), to_dev(np.zeros(3, np.int32), dev), freqs(dev, rot),
                                interleaved=inter))
            assert np.array_equal(got[..., rot:].view(np.uint32), x[..., rot:].view(np.uint32))
            assert np.array_equal(got[..., :rot], x[..., :rot])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_strides_and_in_place(dev, interleaved):
    """q, k and v as slices of one projection's output, and the rotation in place."""
    say(f"rope strides interleaved={interleaved}")
    rng = np.random.default_rng(9)
    t, hq, hkv, d = 37, 6, 2, 64
    fused = rng.standard_normal((t, (hq + 2 * hkv) * d)).astype(np.float32)
    g = to_dev(fused, dev)
    pos, f = to_dev(positions(rng, t, 5000), dev), freqs(dev, d)
    q, k = g[:, :hq * d].view(t, hq, d), g[:, hq * d:(hq + hkv) * d].view(t, hkv, d)
    want_q = kv.rope(q.contiguous(), pos, f, interleaved=interleaved)
    want_k = kv.rope(k.contiguous(), pos, f, interleaved=interleaved)
    # heads before tokens
    swapped = kv.rope(q.contiguous().transpose(0, 1).contiguous().transpose(0, 1), pos, f,
                      interleaved=interleaved)
    assert torch.equal(swapped, want_q)
    kv.rope(q, pos, f, interleaved=interleaved, out=q)
    kv.rope(k, pos, f, interleaved=interleaved, out=k)
    torch.cuda.synchronize()
    assert torch.equal(q, want_q) and torch.equal(k, want_k)
    assert np.array_equal(to_np(g)[:, (hq + hkv) * d:], fused[:, (hq + hkv) * d:])


@pytest.mark.parametrize("kind", ["f32", "bf16", "int8", "fp8"])
@pytest.mark.parametrize("hq,hkv,d,rot,t,interleaved", [
    (32, 8, 128, 128, 64, False), (32, 8, 128, 128, 64, True), (4, 4, 32, 32, 5, False),
    (8, 1, 64, 32, 130, False), (8, 1, 64, 20, 130, False), (2, 2, 64, 30, 1, True),
    (8, 2, 128, 6, 2100, False), (3, 1, 128, 128, 3, False)])
def test_rope_append_equals_rope_then_append(dev, kind, hq, hkv, d, rot, t, interleaved):
    say(f"rope_append {kind} hq={hq} hkv={hkv} d={d} rot={rot} t={t} interleaved={interleaved}")
    rng = np.random.default_rng(hq + d + rot + t)
    nb = (t + 15) // 16 + 4
    q, k, v = (to_dev(rng.standard_normal((t, h, d)).astype(np.float32), dev)
               for h in (hq, hkv, hkv))
    pos, f = to_dev(positions(rng, t, 100000), dev), freqs(dev, rot)
    slots = rng.permutation(nb * 16)[:t].astype(np.int64)
    slots[t // 2] = -1                       # padding: q rotated, nothing stored
    if t > 4:
        slots[1] = nb * 16                   # past the pool
    slots = to_dev(slots, dev)
    quant = kind in ("int8", "fp8")
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}.get(kind, torch.uint8)

    def pools():
        g = torch.Generator().manual_seed(3)
        p = [torch.randint(0, 100, (nb, hkv, 16, d), generator=g).to(dt).to(dev) for _ in "kv"]
        s = [torch.full((nb, hkv, 16), 7.0, device=dev) for _ in "kv"] if quant else [None, None]
        return p, s

    (k1, v1), (ks1, vs1) = pools()
    (k2, v2), (ks2, vs2) = pools()
    out = kv.rope_append(q, k, v, pos, f, k1, v1, slots, k_scale=ks1, v_scale=vs1,
                         fmt=kind if quant else None, interleaved=interleaved, magnitude=1.1)
    qr = kv.rope(q, pos, f, interleaved=interleaved, magnitude=1.1)
    kr = kv.rope(k, pos, f, interleaved=interleaved, magnitude=1.1)
    if quant:
        kv.append_q(k2, v2, ks2, vs2, kr, v, slots, kind)
    else:
        kv.append(k2, v2, kr, v, slots)
    torch.cuda.synchronize()
    assert torch.equal(out, qr)
    assert torch.equal(k1, k2) and torch.equal(v1, v2)
    if quant:
        assert torch.equal(ks1, ks2) and torch.equal(vs1, vs2)


def test_rope_append_from_a_fused_projection(dev):
    """k_new and v_new as slices with one stride, q rotated in place."""
    say("rope_append slices")
    rng = np.random.default_rng(2)
    t, hq, hkv, d, nb = 19, 8, 2, 64, 6
    g = to_dev(rng.standard_normal((t, (hq + 2 * hkv) * d)).astype(np.float32), dev)
    q = g[:, :hq * d].view(t, hq, d)
    k = g[:, hq * d:(hq + hkv) * d].view(t, hkv, d)
    v = g[:, (hq + hkv) * d:].view(t, hkv, d)
    pos, f = to_dev(positions(rng, t, 900), dev), freqs(dev, d)
    slots = to_dev(rng.permutation(nb * 16)[:t].astype(np.int64), dev)
    pools = [torch.zeros((nb, hkv, 16, d), dtype=torch.bfloat16, device=dev) for _ in range(4)]
    want = kv.rope(q.contiguous(), pos, f)
    kv.append(pools[0], pools[1], kv.rope(k.contiguous(), pos, f), v.contiguous(), slots)
    kv.rope_append(q, k, v, pos, f, pools[2], pools[3], slots, out=q)
    torch.cuda.synchronize()
    assert torch.equal(q, want)
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])


def test_rope_front_end_refuses(dev):
    x = torch.zeros((4, 2, 64), device=dev)
    pos, f = torch.zeros(4, dtype=torch.int32, device=dev), freqs(dev, 64)
    with pytest.raises(TypeError):
        kv.rope(x.half(), pos, f)
    with pytest.raises(TypeError):
        kv.rope(x, pos.long(), f)
    with pytest.raises(TypeError):
        kv.rope(x, pos, f.float())
    with pytest.raises(ValueError):
        kv.rope(x, pos[:3], f)
    with pytest.raises(ValueError):
        kv.rope(x, pos, freqs(dev, 66))
    with pytest.raises(ValueError):
        kv.rope(x.transpose(1, 2), pos, f)
    with pytest.raises(_lib.RkvError):   # rows off a 16-byte boundary
        kv.rope(torch.zeros(4 * 2 * 64 + 1, device=dev)[1:].view(4, 2, 64), pos, f)
    p = torch.zeros((4, 2, 16, 64), device=dev)
    slots = torch.zeros(4, dtype=torch.int64, device=dev)
    with pytest.raises(ValueError):
        kv.rope_append(x, x[:, :1], x[:, :1], pos, f, p, p, slots)
    with pytest.raises(ValueError):
        kv.rope_append(x, x, x, pos, f, p, p, slots[:2])
    with pytest.raises(ValueError):
        kv.rope_append(x, x, x, pos, f, p.to(torch.uint8), p.to(torch.uint8), slots, fmt="int8")
    assert kv.rope(x[:0], pos[:0], f).shape == (0, 2, 64)


@pytest.mark.parametrize("d,rot", [(8, 8), (24, 24), (40, 18), (1024, 1024), (128, 2)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_negative_positions_and_odd_widths(dev, d, rot, interleaved):
    """Positions down to -2^31, every head width the call takes; a turn there and back."""
    say(f"rope negative d={d} rot={rot} interleaved={interleaved}")
    rng = np.random.default_rng(d)
    pos = np.array([-1, 0, -2 ** 31, 2 ** 31 - 1, -77777, 5], np.int32)
    f, _ = kv.rope_frequencies(rot, device=dev)
    x = rng.standard_normal((len(pos), 3, d)).astype(np.float32)
    y = kv.rope(to_dev(x, dev), to_dev(pos, dev), f, interleaved=interleaved)
    freq = f.cpu().numpy()
    R.assert_within(to_np(y), R.rope(x, pos, freq, interleaved),
                    R.rope_bound(x, pos, freq, interleaved), "negative")
    some = pos[[0, 1, 4, 5]]
    back = to_np(kv.rope(y[[0, 1, 4, 5]].contiguous(), to_dev(-some, dev), f,
                         interleaved=interleaved))
    x = x[[0, 1, 4, 5]]
    # the first turn's errors on a pair reach each element (2 bounds), and the second's
    # own is that of a pair sqrt(2) as large at most
    R.assert_within(back, x.astype(np.float64), 3.5 * R.rope_bound(x, some, freq, interleaved),
                    "there and back")
