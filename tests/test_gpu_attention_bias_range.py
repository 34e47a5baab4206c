"""Relative position tables with values of any size: what a program writes there to hide or to force a bucket (1e9, the type's
lowest value) instead of -inf.  Rows that see other keys as well have none of the hidden ones."""
import math

import pytest
import torch

from mint_amd import attention as A
from tests import test_gpu_attention_ops as T

pytestmark = pytest.mark.gpu
LOW = torch.finfo(torch.float32).min


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
