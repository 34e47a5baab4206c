"""Relative position tables with values of any size: what a program writes there to hide or to force a bucket (1e9, the type's
lowest and largest value) instead of -inf.  A row's softmax does not change by a constant, so rows that see such keys only have the
softmax of their scores without a bias, and rows that see others have none of the hidden ones."""
import math

import pytest
import torch

from mint_amd import attention as A
from tests import test_gpu_attention_ops as T

pytestmark = pytest.mark.gpu
LOW, TOP = torch.finfo(torch.float32).min, torch.finfo(torch.float32).max


def _inputs(seed, B, nq, nk, H, Hkv, dh):
    gen = torch.Generator().manual_seed(seed)
    q, k, v = T._rand(gen, B, nq, H, dh), T._rand(gen, B, nk, Hkv, dh), T._rand(gen, B, nk, Hkv, dh)
    return gen, q, k, v, T._rand(gen, B, nq, H, dh)


def _compare(q, k, v, do, ref, **kw):
    out = A.attention(q, k, v, **kw)
    T._within("out", out, ref["out"])
    o, saved = A.attention(q, k, v, training=True, **kw)
    T._within("out (training)", o, ref["out"])
    for name, g in zip(("dq", "dk", "dv", "drel"), A.attention_backward(do, q, k, v, o, saved, **kw)):
        if name in ref:
            T._within(name, g, ref[name])
    return saved


@pytest.mark.parametrize("value", [-3e4, -1e9, LOW, 1e9, TOP])
@pytest.mark.parametrize("nq,nk,window,sinks", [(77, 77, (-1, -1), 0), (130, 130, (40, 0), 3), (3, 300, (-1, -1), 0)])
def test_rows_that_see_nothing_but_such_keys(value, nq, nk, window, sinks, monkeypatch):
    """Values count up to 2^14.  There a score is rounded by 2^-24 of it, 2^-10, once for each of the 32 products of dh 32 and for
    the bias, the scale and the reference point at the most: 35 * 2^-10 to either side, so a probability is off by less than
    exp(2 * 35 * 2^-10) - 1 = 0.071 of itself.  Its log-sum-exp, near 2^14 log2(e), and the probabilities that the backward takes
    from it, by another 2^-9: 0.08, in place of the 32-bit arithmetic's share of the bounds."""
    monkeypatch.setattr(T, "F32", 0.08)
    gen, q, k, v, do = _inputs(5, 2, nq, nk, 4, 2, 32)
    t, m = T._table(gen, 4)
    t[:] = value
    ref = T._reference(q, k, v, 32 ** -0.5, window=window, sinks=sinks, dout=do)
    saved = _compare(q, k, v, do, ref, rel_table=t, rel_map=m, window=window, sinks=sinks, scale=32 ** -0.5)
    assert torch.isfinite(saved.lse).all()


@pytest.mark.parametrize("value", [-3e4, -1e9, LOW])
@pytest.mark.parametrize("dh", [32, 80, 128])
@pytest.mark.parametrize("side", ["before", "after"])
def test_a_bucket_hidden_by_a_finite_value(value, dh, side):
    """The keys farthest to one side, whole tiles of them before or after the ones that count: as if the value were -inf, with the
    bounds of every other call."""
    gen, q, k, v, do = _inputs(dh, 2, 203, 203, 2, 2, dh)
    t, m = T._table(gen, 2)
    bucket = int(m[0] if side == "before" else m[-1])
    hidden = t.clone()
    hidden[bucket] = -math.inf
    kw = dict(rel_map=m, scale=dh ** -0.5)
    ref = T._reference(q, k, v, kw["scale"], rel_table=hidden, rel_map=m, dout=do)
    t[bucket] = value
    saved = _compare(q, k, v, do, ref, rel_table=t, **kw)
    assert (saved.lse.double() - ref["lse"][0]).abs().max() <= 64 * 2.0 ** -18
    one = A.attention(q[:, 150:151], k, v, rel_table=t, q_start=torch.full((2,), 150, dtype=torch.int32, device=T.DEV), **kw)
    T._within("one row", one, tuple(x[:, 150:151] for x in ref["out"]))


def test_infinities_and_numbers_that_are_none_keep_their_meaning():
    gen, q, k, v, do = _inputs(9, 1, 64, 64, 2, 2, 64)
    t, m = T._table(gen, 2)
    t[int(m[24 + 2])] = -math.inf
    T._check(q, k, v, 0.125, train=False, rel_table=t, rel_map=m)
    t[int(m[24]), 1] = float("nan")  # distance 0, the second head
    out = A.attention(q, k, v, rel_table=t, rel_map=m)
    assert torch.isfinite(out[:, :, 0]).all() and out[:, :, 1].isnan().all()
