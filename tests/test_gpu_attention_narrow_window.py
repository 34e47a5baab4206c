"""Rows that see few keys of a long sequence: their gradients get the exact row sums that short sequences have (the rounding of the
output, 2^-8 of it, is a large share of dP - dO . O where few probabilities are averaged)."""
import pytest
import torch

from mint_amd import attention as A
from tests import test_gpu_attention_ops as T

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,sinks", [((1, 0), 0), ((0, 1), 0), ((2, 2), 0), ((1, 0), 4), ((31, 31), 0), ((40, 0), 23)])
@pytest.mark.parametrize("nq,nk,H,Hkv,dh", [(700, 700, 2, 2, 32), (520, 1100, 4, 2, 80), (3, 900, 4, 2, 128)])
def test_narrow_windows_of_long_sequences(window, sinks, nq, nk, H, Hkv, dh, monkeypatch):
    """The bounds of a call with 24-bit probabilities and outputs in its row sums."""
    gen = torch.Generator().manual_seed(nq + window[0])
    q, k, v, do = (T._rand(gen, 1, n, h, dh) for n, h in ((nq, H), (nk, Hkv), (nk, Hkv), (nq, H)))
    kw = dict(scale=dh ** -0.5, window=window, sinks=sinks)
    with monkeypatch.context() as m:
        m.setattr(A, "EXACT_KEYS", nk)  # (what the reference takes its bounds by)
        ref = T._reference(q, k, v, dout=do, **kw)
    o, saved = A.attention(q, k, v, training=True, **kw)
    T._within("out", o, ref["out"])
    for name, g in zip(("dq", "dk", "dv"), A.attention_backward(do, q, k, v, o, saved, **kw)):
        T._within(name, g, ref[name])


def test_wide_windows_of_long_sequences_do_without():
    q = torch.zeros(1, 700, 1, 32, dtype=torch.bfloat16, device="cuda")
    for window, sinks, lo in (((31, 32), 0, True), ((32, 32), 0, False), ((31, 31), 2, False), ((5, -1), 0, False), ((-1, 5), 0, False),
                              ((2 ** 31 - 1, 2 ** 31 - 1), 2 ** 31 - 1, False)):
        assert (A.attention(q, q, q, training=True, window=window, sinks=sinks)[1].out_lo is not None) == lo, window
