"""What the attention operators refuse, and the bucket map, without a GPU: the C entry points check their arguments before they
touch the device (the pointers below are never read)."""
import ctypes as C
import math
import os
from fractions import Fraction

import pytest
import torch

from mint_amd import _lib as L
from mint_amd import attention as A

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(L.LIB_PATH):
        import __graft_entry__ as g
        g.build()
    return L.lib()


def _attention(backward=True, **kw):
    a = L.FactAttention(B=2, H=4, Hkv=2, nq=8, nk=24, dh=64, window_left=-1, window_right=-1, scale=0.125)
    for i, n in enumerate(("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv")):
        setattr(a, n, 4096 * (i + 1))
    for n in ("q", "out", "dout", "dq"):
        getattr(a, n + "_stride")[:] = (8 * 256, 256, 64)
    for n in ("k", "v", "dk", "dv"):
        getattr(a, n + "_stride")[:] = (24 * 128, 128, 64)
    for n, v in kw.items():
        if n.endswith("_stride"):
            getattr(a, n)[:] = v
        else:
            setattr(a, n, v)
    return a


BIAS = dict(rel_table=1 << 20, rel_map=1 << 21, rel_buckets=32, rel_max_distance=128, drel=1 << 22)


def test_struct_sizes_match_the_header(lib, tmp_path):
    """The ctypes mirrors against a C compiler's layout of include/fact_hip.h."""
    import subprocess
    src = tmp_path / "s.c"
    fields = [("FactAttention", f) for f, _ in L.FactAttention._fields_] + [("FactQkNorm", f) for f, _ in L.FactQkNorm._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "fact_hip.h"\nint main(void){printf("%zu %zu\\n",'
                   "sizeof(FactAttention),sizeof(FactQkNorm));"
                   + "".join('printf("%%zu\\n",offsetof(%s,%s));' % f for f in fields) + "return 0;}\n")
    exe = str(tmp_path / "s")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe])
    got = subprocess.check_output([exe], text=True).split()
    assert [int(x) for x in got[:2]] == [C.sizeof(L.FactAttention), C.sizeof(L.FactQkNorm)]
    assert [int(x) for x in got[2:]] == [getattr(getattr(L, s), f).offset for s, f in fields]


@pytest.mark.parametrize("kw,rc,word", [
    (dict(B=0), -1, "positive"), (dict(nk=0), -1, "positive"), (dict(Hkv=3), -1, "multiple"), (dict(dh=72), -3, "head dim"),
    (dict(dh=48), -3, "head dim"), (dict(nq=1 << 30), -1, "2^30"), (dict(B=1 << 20, H=1 << 12, Hkv=1 << 12), -1, "too many"),
    (dict(scale=0.0), -1, "scale"), (dict(scale=-1.0), -1, "scale"), (dict(scale=math.nan), -1, "scale"),
    (dict(scale=math.inf), -1, "scale"), (dict(scale=1e-9), -1, "scale"), (dict(sinks=-1), -1, "sinks"),
    (dict(q=None), -1, "null"), (dict(v=4096 + 8), -1, "aligned"), (dict(out_lo=4096 + 2), -1, "aligned"),
    (dict(k_stride=(24 * 128, 132, 64)), -1, "multiples of 8"), (dict(dq_stride=(8 * 256, 0, 64)), -1, "broadcast"),
    (dict(v_stride=(1 << 40, (1 << 25) + 8, 64)), -1, "2^25"), (dict(q_stride=(1 << 40, -64, 64)), -1, "2^25"),
    (dict(dk_stride=(0, 128, 64)), -1, "broadcast"), (dict(dq=4096), -1, "another tensor"), (dict(dk=8 * 4096, dv=8 * 4096), -1, "another tensor"),
    (dict(dv=6 * 4096), -1, "another tensor"), (dict(B=1 << 19, nk=64 * 64), -1, "too many"), (dict(nq=1 << 29, B=1 << 3), -1, "too many"), (dict(lse=None), -1, "lse"),
    (dict(BIAS, rel_map=None), -1, "rel_map"), (dict(BIAS, rel_buckets=0), -1, "rel_buckets"),
    (dict(BIAS, rel_buckets=257), -1, "rel_buckets"), (dict(BIAS, rel_max_distance=0), -1, "rel_max_distance"),
    (dict(BIAS, rel_max_distance=1025), -1, "rel_max_distance"), (dict(BIAS, drel=None), -1, "drel")])
def test_attention_refuses(lib, kw, rc, word):
    a = _attention(**kw)
    n = C.c_size_t(0)
    assert lib.fact_attention_workspace(C.byref(a), 1, C.byref(n)) == rc
    assert word in lib.fact_last_error().decode()
    assert lib.fact_attention_backward(C.byref(a), 1 << 23, 1 << 40, None) == rc


def test_attention_asks_for_its_workspace(lib):
    n = C.c_size_t(0)
    a = _attention()
    assert lib.fact_attention_workspace(C.byref(a), 0, C.byref(n)) == 0 and n.value == 0
    assert lib.fact_attention_workspace(C.byref(a), 1, C.byref(n)) == 0 and n.value >= 2 * 4 * 8 * 4
    assert lib.fact_attention_backward(C.byref(a), None, 0, None) == -4
    assert lib.fact_attention_backward(C.byref(a), 4096, n.value - 1, None) == -4
    assert lib.fact_attention_backward(C.byref(a), 4100, n.value, None) == -1
    # broadcast inputs are fine, an output with a zero stride over one element too
    assert lib.fact_attention_workspace(C.byref(_attention(k_stride=(0, 128, 0), dq_stride=(0, 256, 64), B=1)), 1, C.byref(n)) == 0
    # one row against a long cache: split over workgroups, so partial rows are kept
    a = _attention(nq=1, nk=1 << 20)
    assert lib.fact_attention_workspace(C.byref(a), 0, C.byref(n)) == 0 and n.value > 0
    assert lib.fact_attention(C.byref(a), None, 0, None) == -4
    assert lib.fact_attention_workspace(None, 0, C.byref(n)) == -1 and lib.fact_attention(None, None, 0, None) == -1


def test_an_output_is_not_an_input(lib):
    n = C.c_size_t(0)
    for name in ("k", "v"):
        a = _attention(out=getattr(_attention(), name))
        assert lib.fact_attention_workspace(C.byref(a), 0, C.byref(n)) == -1 and "another tensor" in lib.fact_last_error().decode()
    assert lib.fact_attention_workspace(C.byref(_attention(out=4096)), 0, C.byref(n)) == 0  # in place of q


def test_workspace_of_blocks_with_sinks_stays_small(lib):
    """The partial sums of the blocks that all queries see are bounded by the work that runs beside them."""
    n = C.c_size_t(0)
    for B, H, nq in ((1, 4, 16384), (32, 12, 16384), (4, 12, 1440), (1, 1, 1 << 20)):
        a = _attention(B=B, H=H, Hkv=H, nq=nq, nk=nq, dh=128, window_left=255, window_right=0, sinks=4)
        assert lib.fact_attention_workspace(C.byref(a), 1, C.byref(n)) == 0
        assert n.value <= 4 * B * H * nq + (1 << 28), (B, H, nq, n.value)


def _norm(**kw):
    a = L.FactQkNorm(B=2, n=8, H=4, Hkv=2, dh=64, rotary_dim=64, base=10000.0, eps=1e-6)
    for i, n in enumerate(("q", "k", "q_out", "k_out", "dq_out", "dk_out", "dq", "dk")):
        setattr(a, n, 4096 * (i + 1))
        getattr(a, n + "_stride")[:] = (8 * 256, 256, 64)
    for n, v in kw.items():
        if n.endswith("_stride"):
            getattr(a, n)[:] = v
        else:
            setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw,rc,word", [
    (dict(B=0), -1, "positive"), (dict(Hkv=0), -1, "positive"), (dict(n=1 << 30, B=1 << 10), -1, "too many"),
    (dict(n=1 << 16, B=1 << 10), -1, "too many"),
    (dict(dh=132), -3, "head dim"), (dict(dh=20), -3, "head dim"), (dict(rotary_dim=72), -1, "rotary_dim"),
    (dict(rotary_dim=-8), -1, "rotary_dim"), (dict(rotary_dim=12), -1, "rotary_dim"), (dict(dtype=2), -1, "dtype"),
    (dict(eps=-1.0), -1, "eps"), (dict(eps=math.nan), -1, "eps"), (dict(base=0.0), -1, "base"), (dict(base=math.nan), -1, "base"),
    (dict(position0=(1 << 31) - 5), -1, "position"), (dict(k=None), -1, "null"), (dict(dq=4096 + 4), -1, "aligned"), (dict(q_gamma=4096 + 4), -1, "aligned"),
    (dict(q_stride=(8 * 256, 252, 64)), -1, "multiples of 8"), (dict(dk_stride=(8 * 256, 0, 64)), -1, "broadcast")])
def test_norm_refuses(lib, kw, rc, word):
    n = C.c_size_t(0)
    a = _norm(**kw)
    assert lib.fact_qk_norm_workspace(C.byref(a), 1, C.byref(n)) == rc
    assert word in lib.fact_last_error().decode()
    assert lib.fact_qk_norm_backward(C.byref(a), 1 << 23, 1 << 40, None) == rc


def test_norm_asks_for_its_workspace(lib):
    n = C.c_size_t(0)
    assert lib.fact_qk_norm_workspace(C.byref(_norm()), 0, C.byref(n)) == 0 and n.value == 0
    assert lib.fact_qk_norm_workspace(C.byref(_norm()), 1, C.byref(n)) == 0 and n.value > 0
    assert lib.fact_qk_norm_backward(C.byref(_norm()), None, 0, None) == -4
    assert lib.fact_qk_norm(None, None, 0, None) == -1


@pytest.mark.parametrize("buckets,dist,both", [(32, 128, True), (32, 128, False), (64, 512, True), (8, 20, True), (2, 5, False),
                                               (4, 100, True), (256, 1024, False), (256, 1000, True), (6, 7, False), (18, 77, True)])
def test_bucket_map_against_exact_powers(lib, buckets, dist, both):
    m = A.relative_buckets(buckets, dist, both).tolist()
    n = buckets // 2 if both else buckets
    e = n // 2
    for d in range(-dist, dist + 1):
        far = abs(d) if both else max(-d, 0)
        if far < e:
            b = far
        else:  # floor(log(far / e) / log(dist / e) * (n - e)) in exact arithmetic
            t = 0
            while t + 1 < n - e and Fraction(far, e) ** (n - e) >= Fraction(dist, e) ** (t + 1):
                t += 1
            b = e + t
        assert m[d + dist] == b + (n if both and d > 0 else 0), d


@pytest.mark.parametrize("args", [(1, 10, False), (3, 10, True), (258, 1000, False), (32, 8, True), (32, 1025, True), (0, 5, False),
                                  (2, 1, False)])
def test_bucket_map_refuses(lib, args):
    with pytest.raises(L.FactError):
        A.relative_buckets(*args)


@pytest.mark.parametrize("args", [(32, 1 << 33, True), ((1 << 32) + 32, 128, True), (32, (1 << 32) + 128, False)])
def test_bucket_map_refuses_what_ctypes_would_cut(lib, args):
    with pytest.raises(ValueError, match="32 bits"):
        A.relative_buckets(*args)


def test_python_calls_refuse_host_tensors():
    q = torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: A.attention(q, q, q), lambda: A.qk_norm_rope(q, q), lambda: A.attention(None, q, q),
                 lambda: A.attention(q[0], q, q)):
        with pytest.raises(ValueError):
            call()


def test_operator_sources_hold_nothing_that_a_graph_cannot_replay():
    """Calls are captured into graphs: no memset nodes, no allocation, no synchronisation on the way."""
    for f in ("rel_attention.hip", "qk_norm.hip"):
        text = open(os.path.join(ROOT, "mint_amd", "csrc", f)).read()
        assert "hipMemset" not in text and "hipMalloc" not in text and "Synchronize" not in text


def _model_cfg(**at):
    st = lambda seq, feat: L.FactStackCfg(seq, feat, 800, 2, 10, 1600)
    cfg = L.FactConfig(st(120, 225), st(240, 35), st(0, 0), 225, 1e-5)
    return cfg, (L.FactAttnCfg * 3)(L.FactAttnCfg(), L.FactAttnCfg(), L.FactAttnCfg(**at))


def test_model_options_add_their_variables(lib):
    n0, t0, n, t = C.c_size_t(0), C.c_int(0), C.c_size_t(0), C.c_int(0)
    cfg, none = _model_cfg()
    assert lib.fact_arena_size(C.byref(cfg), C.byref(n0), C.byref(t0)) == 0
    assert lib.fact_arena_size_ex(C.byref(cfg), none, C.byref(n), C.byref(t)) == 0 and (n.value, t.value) == (n0.value, t0.value)
    assert lib.fact_arena_size_ex(C.byref(cfg), None, C.byref(n), C.byref(t)) == 0 and (n.value, t.value) == (n0.value, t0.value)
    cfg, at = _model_cfg(qk_norm=1, rel_buckets=32, rel_max_distance=128, window=64, sinks=4)
    assert lib.fact_arena_size_ex(C.byref(cfg), at, C.byref(n), C.byref(t)) == 0 and t.value == t0.value + 2 * 3


@pytest.mark.parametrize("at,word", [
    (dict(qk_norm=2), "qk_norm"), (dict(rotary_dim=16), "qk_norm"), (dict(qk_norm=1, rotary_dim=12), "rotary_dim"),
    (dict(qk_norm=1, rotary_dim=88), "rotary_dim"), (dict(qk_norm=1, rotary_base=math.nan), "rotary_base"), (dict(window=-1), "window"),
    (dict(sinks=3), "sinks"), (dict(window=4, sinks=-1), "sinks"), (dict(rel_buckets=300), "buckets"),
    (dict(rel_buckets=32), "distance"), (dict(rel_buckets=31, rel_max_distance=128), "even"),
    (dict(rel_buckets=32, rel_max_distance=8), "largest distance"), (dict(rel_buckets=32, rel_max_distance=5000), "distance")])
def test_model_options_refuse(lib, at, word):
    cfg, a = _model_cfg(**at)
    assert lib.fact_arena_size_ex(C.byref(cfg), a, None, None) == -1
    assert word in lib.fact_last_error().decode()
    assert lib.fact_create_ex(C.byref(cfg), a, 1, 0, None, C.byref(C.c_void_p())) == -1


def test_options_parse_from_a_text_config():
    from mint_amd import protos
    m = protos.Merge("""fact_model { cross_modal_model { transformer { hidden_size: 800 qk_norm: true rotary_dim: 80
        attention_window: 64 attention_sinks: 4 relative_attention_num_buckets: 32 } } }""", protos.MultiModalModel())
    t = m.fact_model.cross_modal_model.transformer
    assert t.qk_norm and (t.rotary_dim, t.rotary_base, t.attention_window, t.attention_sinks) == (80, 10000.0, 64, 4)
    assert (t.relative_attention_num_buckets, t.relative_attention_max_distance) == (32, 128)
    again = protos.Merge(protos.MessageToString(m), protos.MultiModalModel())
    assert again == m
