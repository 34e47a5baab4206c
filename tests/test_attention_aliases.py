"""Outputs of the attention operators that stand where another tensor of the call does: refused before anything is launched, but
for the places that the kernels read before they write (no GPU needed: the pointers are never read)."""
import ctypes as C

import pytest

from mint_amd import _lib as L
from tests.test_attention_args import BIAS, _attention, _norm, lib  # noqa: F401

NORM_TENSORS = ("q", "k", "q_out", "k_out", "dq_out", "dk_out", "dq", "dk")
NORM_FORWARD = {("q_out", "q"), ("k_out", "k")}
NORM_BACKWARD = {("dq", "dq_out"), ("dk", "dk_out"), ("dq", "q"), ("dk", "k")}


def _norm_says(lib, backward, **kw):
    n = C.c_size_t(0)
    rc = lib.fact_qk_norm_workspace(C.byref(_norm(**kw)), backward, C.byref(n))
    return rc, lib.fact_last_error().decode() if rc else ""


@pytest.mark.parametrize("backward,outputs,inputs,allowed", [
    (0, ("q_out", "k_out"), ("q", "k"), NORM_FORWARD),
    (1, ("dq", "dk"), ("q", "k", "dq_out", "dk_out"), NORM_BACKWARD)])
def test_norm_outputs(lib, backward, outputs, inputs, allowed):  # noqa: F811
    place = {n: getattr(_norm(), n) for n in NORM_TENSORS}
    for out in outputs:
        for other in outputs + inputs:
            if other == out:
                continue
            rc, why = _norm_says(lib, backward, **{out: place[other]})
            if (out, other) in allowed:
                assert rc == 0, (out, other, why)
                # the same place with its heads and tokens swapped: rows of other workgroups are overwritten
                rc, why = _norm_says(lib, backward, **{out: place[other], out + "_stride": (8 * 256, 64, 512)})
            assert rc == -1 and "another tensor" in why, (out, other)
    # both inputs in one place (shared queries and keys), written over by either side
    rc, why = _norm_says(lib, backward, q=4096, k=4096, **{outputs[0]: 4096})
    assert rc == -1 and "another tensor" in why
    assert _norm_says(lib, backward, q=4096, k=4096)[0] == 0


def test_norm_strides_of_single_elements_do_not_matter(lib):  # noqa: F811
    assert _norm_says(lib, 0, q_out=4096, B=1, q_out_stride=(8, 256, 64))[0] == 0
    assert _norm_says(lib, 1, dq=4096, n=1, dq_stride=(8 * 256, 8, 64))[0] == 0


def test_norm_gain_gradients(lib):  # noqa: F811
    gains = dict(q_gamma=1 << 20, k_gamma=1 << 21, dq_gamma=1 << 22, dk_gamma=1 << 23, positions=1 << 24)
    assert _norm_says(lib, 1, **gains)[0] == 0
    for kw in (dict(dk_gamma=1 << 22), dict(dq_gamma=1 << 20), dict(dk_gamma=1 << 20), dict(dq_gamma=1 << 24), dict(dk_gamma=4096),
               dict(dq_gamma=7 * 4096)):
        rc, why = _norm_says(lib, 1, **dict(gains, **kw))
        assert rc == -1 and "another tensor" in why, kw
    assert _norm_says(lib, 1, **dict(gains, k_gamma=1 << 20))[0] == 0  # one gain for both


def test_norm_calls_refuse_too(lib):  # noqa: F811
    a = _norm(q_out=2 * 4096)
    assert lib.fact_qk_norm(C.byref(a), None, 0, None) == -1
    a = _norm(dk=7 * 4096)
    assert lib.fact_qk_norm_backward(C.byref(a), 1 << 26, 1 << 20, None) == -1


def _attention_says(lib, backward, **kw):
    n = C.c_size_t(0)
    rc = lib.fact_attention_workspace(C.byref(_attention(**kw)), backward, C.byref(n))
    return rc, lib.fact_last_error().decode() if rc else ""


def test_attention_in_place_of_the_queries_needs_their_strides(lib):  # noqa: F811
    assert _attention_says(lib, 0, out=4096)[0] == 0
    for strides in ((64, 256, 2048), (8 * 256, 64, 512), (8 * 512, 512, 64)):
        rc, why = _attention_says(lib, 0, out=4096, out_stride=strides)
        assert rc == -1 and "another tensor" in why, strides
    assert _attention_says(lib, 0, out=4096, out_stride=(8, 256, 64), B=1)[0] == 0  # one sequence: its stride is never used
    assert _attention_says(lib, 0, out=4096, nq=1, out_stride=(8 * 256, 8, 64))[0] == 0
    a = _attention(out=4096, out_stride=(64, 256, 2048))
    assert lib.fact_attention(C.byref(a), None, 0, None) == -1


@pytest.mark.parametrize("backward", [0, 1])
def test_attention_outputs_beside_the_heads(lib, backward):  # noqa: F811
    """The fp32 outputs and the tables: drel over rel_table would be read as the bias by the kernel that follows."""
    kw = dict(BIAS, kv_len=1 << 23, q_start=1 << 24, out_lo=1 << 25, lse=1 << 26)
    assert _attention_says(lib, backward, **kw)[0] == 0
    small = ["drel"] if backward else ["out_lo", "lse"]
    others = ["q", "k", "v", "out", "rel_table", "rel_map", "kv_len", "q_start", "out_lo", "lse"]
    others += ["dout", "dq", "dk", "dv"] if backward else []
    place = _attention(**kw)
    for out in small:
        for other in others:
            if other != out:
                rc, why = _attention_says(lib, backward, **dict(kw, **{out: getattr(place, other)}))
                assert rc == -1 and "another tensor" in why, (out, other)
    for out in ("dq", "dk", "dv") if backward else ("out",):
        for other in ("rel_table", "rel_map", "kv_len", "q_start"):
            rc, why = _attention_says(lib, backward, **dict(kw, **{out: getattr(place, other)}))
            assert rc == -1 and "another tensor" in why, (out, other)
