"""process_logits on the GPU against the formulas in 64 bits."""
import math

import numpy as np
import pytest
import torch

from rustral_amd import _lib, model
from tests import op_refs as R
from tests.gpu_util import say, to_dev, to_np

pytestmark = pytest.mark.gpu


def make(rng, rows, n, hist, biases, mask):
    x = (3 * rng.standard_normal((rows, n))).astype(np.float32)
    lens = rng.integers(0, hist + 1, rows)
    start = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    a = dict(history=rng.integers(0, max(1, n // 3), max(1, int(start[-1]))).astype(np.int32),
             start=start, prompt=(lens // 2).astype(np.int32),
             repetition=(0.8 + rng.random(rows)).astype(np.float32),
             frequency=rng.standard_normal(rows).astype(np.float32),
             presence=rng.standard_normal(rows).astype(np.float32))
    a["history"][::17] = -1                  # ids outside the vocabulary
    a["history"][5::23] = n
    if biases:
        a["bias_start"] = (biases * np.arange(rows + 1)).astype(np.int32)
        a["bias_ids"] = rng.integers(-1, n + 1, rows * biases).astype(np.int32)  # some twice
        a["bias"] = (4 * rng.standard_normal(rows * biases)).astype(np.float32)
    if mask:
        a["allowed"] = rng.integers(-2**31, 2**31, (rows, -(-n // 32) + mask - 1)).astype(np.int32)
    return x, a


def call(dev, x, a, **kw):
    names = dict(start="history_start", prompt="prompt_lens")
    return model.process_logits(x if isinstance(x, torch.Tensor) else to_dev(x, dev),
                                **{names.get(k, k): to_dev(v, dev) for k, v in a.items()}, **kw)


def check(got, pick, x, a):
    want, picks, bound = R.logits(x, **a)
    got, pick = to_np(got), to_np(pick)
    low = np.isneginf(want)
    assert np.array_equal(np.isneginf(got), low)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fin = np.isfinite(want)
    R.assert_within(got[fin], want[fin], bound[fin], "logits")
    assert np.array_equal(got[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)])
    for r in range(len(pick)):               # the best of the computed row, the last of equals
        z = np.where(np.isnan(got[r]), -np.inf, got[r])
        assert pick[r] == (np.nonzero(z == z.max())[0][-1] if z.max() > -np.inf else -1)
        if pick[r] != picks[r]:              # two entries nearer than their rounding
            assert abs(want[r, pick[r]] - want[r, picks[r]]) <= 2 * bound[r].max()
    return picks


@pytest.mark.parametrize("rows,n,hist,biases,mask", [
    (1, 1, 3, 1, 1), (2, 31, 10, 2, 0), (3, 1000, 40, 0, 1), (5, 4096, 300, 7, 1),
    (4, 4097, 300, 7, 2), (7, 32000, 900, 64, 1), (2, 128256, 2000, 16, 1), (3, 50257, 77, 3, 1),
    (64, 8200, 100, 4, 0), (2, 5000, 0, 3, 0)])
def test_against_the_formulas(dev, rows, n, hist, biases, mask):
    say(f"logits rows={rows} n={n} hist={hist} biases={biases} mask={mask}")
    rng = np.random.default_rng(rows + n)
    x, a = make(rng, rows, n, hist, biases, mask)
    check(*call(dev, x, a), x, a)


@pytest.mark.parametrize("drop", [
    ("repetition",), ("frequency", "presence"), ("prompt",), ("bias_ids", "bias", "bias_start"),
    ("allowed",), ("repetition", "frequency", "presence", "history", "start", "prompt"),
    ("repetition", "frequency", "presence", "history", "start", "prompt", "bias_ids", "bias",
     "bias_start", "allowed")])
def test_parts_left_out(dev, drop):
    say(f"logits without {drop}")
    x, a = make(np.random.default_rng(4), 3, 9001, 200, 5, 1)
    a = {k: v for k, v in a.items() if k not in drop}
    got, pick = call(dev, x, a)
    check(got, pick, x, a)
    if not a:
        assert np.array_equal(to_np(got), x)
        assert np.array_equal(to_np(pick), to_np(model.argmax(to_dev(x, dev))))


def test_rows_with_nothing_left_infinities_and_ties(dev):
    say("logits corners")
    n = 6000
    x = np.zeros((6, n), np.float32)
    x[1, 7] = np.inf
    x[2, :] = -np.inf
    x[3, 100], x[3, 5000], x[3, 200] = 2.0, 2.0, np.nan
    x[4, 10] = np.nan
    x[5, :] = np.nan
    allowed = np.full((6, -(-n // 32)), -1, np.int32)
    allowed[0] = 0                            # a mask that leaves nothing
    a = dict(allowed=allowed)
    got, pick = call(dev, x, a)
    check(got, pick, x, a)
    assert to_np(pick).tolist() == [-1, 7, -1, 5000, n - 1, -1]
    allowed[3, 5000 // 32] &= ~np.int32(1 << (5000 % 32))
    _, pick = call(dev, x, a)
    assert to_np(pick)[3] == 100
    # a penalised infinity, a bias on a masked token
    a = dict(history=np.array([7, 7, 3], np.int32), start=np.array([0, 0, 2, 2, 3, 3, 3], np.int32),
             repetition=np.full(6, 2.0, np.float32), bias_ids=np.array([100], np.int32),
             bias=np.array([5.0], np.float32), bias_start=np.array([0, 0, 0, 0, 1, 1, 1], np.int32),
             allowed=allowed)
    check(*call(dev, x, a), x, a)


def test_strides_in_place_and_pick_alone(dev):
    say("logits strides")
    rng = np.random.default_rng(8)
    x, a = make(rng, 4, 5001, 60, 4, 1)
    want, want_pick = call(dev, x, a)
    wide = torch.full((4, 6000), 9.0, device=dev)
    view = wide[:, 3:5004]                    # off a 16-byte boundary
    view.copy_(to_dev(x, dev))
    got, pick = call(dev, view, a, out=view)
    torch.cuda.synchronize()
    assert got.data_ptr() == view.data_ptr()
    assert torch.equal(got, want) and torch.equal(pick, want_pick)
    assert (wide[:, :3] == 9).all() and (wide[:, 5004:] == 9).all()
    aligned = torch.empty((4, 6000), device=dev)[:, :5001]
    got, pick = call(dev, x, a, out=aligned)
    assert torch.equal(got, want) and torch.equal(pick, want_pick)
    only = torch.empty(4, dtype=torch.int32, device=dev)
    g, ws = to_dev(x, dev), torch.empty(4096, dtype=torch.uint8, device=dev)
    rc = _lib.lib().rkv_process_logits(None, 0, only.data_ptr(), g.data_ptr(), 5001, 4, 5001, None,
                                       None, None, None, None, None, None, None, None, None, 0,
                                       ws.data_ptr(), 4096, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert torch.equal(only, model.argmax(g))
    assert np.array_equal(to_np(g), x)


def test_front_end_refuses(dev):
    x = torch.zeros((2, 100), device=dev)
    i = torch.zeros(3, dtype=torch.int32, device=dev)
    with pytest.raises(TypeError):
        model.process_logits(x.half())
    with pytest.raises(ValueError):
        model.process_logits(x[0])
    with pytest.raises(ValueError):
        model.process_logits(x, allowed=torch.zeros((2, 3), dtype=torch.int32, device=dev))
    with pytest.raises(ValueError):
        model.process_logits(x, repetition=torch.ones(3, device=dev), history=i, history_start=i)
    with pytest.raises(_lib.RkvError):
        model.process_logits(x, repetition=torch.ones(2, device=dev))
    with pytest.raises(ValueError):
        model.process_logits(x, bias_ids=i)
    got, pick = model.process_logits(x[:0])
    assert got.shape == (0, 100) and pick.shape == (0,)


@pytest.mark.parametrize("rows", [1, 3, 257])
@pytest.mark.parametrize("n", [4097, 16381, 16384, 16385, 32000, 32767, 32768, 32769])
def test_borders_of_slices_and_rows(dev, rows, n):
    """Lengths on both sides of multiples of a slice, for few rows and for more than the
    chip has CUs; rows on and off a 16-byte boundary give the same bits."""
    say(f"logits rows={rows} n={n}")
    rng = np.random.default_rng(rows + n)
    x, a = make(rng, rows, n, 300, 5, 1)
    got, pick = call(dev, x, a)
    wide = torch.zeros((rows, n + 5), device=dev)
    wide[:, 1:n + 1] = to_dev(x, dev)
    off, off_pick = call(dev, wide[:, 1:n + 1], a)
    assert torch.equal(got.view(torch.int32), off.view(torch.int32)) and torch.equal(pick, off_pick)
    some = min(rows, 3)                       # the formulas on the first rows
    b = {k: v[:some] if len(v) == rows else v for k, v in a.items()}
    b["start"], b["bias_start"] = a["start"][:some + 1], a["bias_start"][:some + 1]
    check(got[:some], pick[:some], x[:some], b)
    best = torch.where(got.isnan(), -math.inf, got).max(1).values
    assert torch.equal(got.gather(1, pick.long()[:, None])[:, 0], best)
