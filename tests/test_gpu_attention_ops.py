"""Attention with window, sinks and relative position bias, and the per-head q / k norm with rotation (mint_amd/attention.py),
against plain implementations in 64 bits.

Bounds are elementwise and follow the roundings the kernels make (half a step of bf16: h = 2^-8 of the value):
  out   the probabilities enter P V as bf16 (h each), the result is rounded (h)         h (sum_j P |V| + |out|)
  D     = rowsum(dO . out), with out off by the above                                    sum_d |dO| d(out)
  dS    = P (dP - D) enters its products as bf16                                         h |dS| + P d(D)
  dq    scale sum_j d(dS) |K| + h |dq|;  dk likewise;  dv  h (P^T |dO| + |dv|)
With a bias (and up to 512 keys) the probabilities and the output are carried to 24 bits for D (d(out) = 2^-20 of the same sum)
and the table's gradient sums dS unrounded.  fp32 arithmetic adds at most 2^-15 of the absolute sums (128 terms, exp2 of |x| < 64).
"""
import math

import pytest
import torch

from mint_amd import attention as A

pytestmark = pytest.mark.gpu
DEV = "cuda"
H8, F32 = 2.0 ** -8, 2.0 ** -15


def _rand(gen, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=gen) * std).to(dtype).to(DEV)


def _seen(B, nq, nk, window, sinks, kv_len, q_start):
    j = torch.arange(nk, device=DEV)[None, None]
    p = torch.arange(nq, device=DEV)[None, :, None].expand(B, nq, 1)
    if q_start is not None:
        p = p + q_start.long()[:, None, None]
    d = j - p
    ok = torch.ones(B, nq, nk, dtype=torch.bool, device=DEV)
    if window[1] >= 0:
        ok &= d <= window[1]
    if window[0] >= 0:
        ok &= (d >= -window[0]) | (j < sinks)
    if kv_len is not None:
        ok &= j < kv_len.long()[:, None, None]
    return ok, d


def _reference(q, k, v, scale, window=(-1, -1), sinks=0, rel_table=None, rel_map=None, kv_len=None, q_start=None, dout=None):
    """Everything in float64 with its elementwise error bound: {name: (value, bound)}."""
    B, nq, H, dh = q.shape
    nk, Hkv = k.shape[1:3]
    g = H // Hkv
    ok, d = _seen(B, nq, nk, window, sinks, kv_len, q_start)
    q, k, v = (t.double() for t in (q, k, v))
    if kv_len is not None:  # rows past the length may hold anything
        live = (torch.arange(nk, device=DEV)[None] < kv_len.long()[:, None])[:, :, None, None]
        k, v = torch.where(live, k, 0.0), torch.where(live, v, 0.0)
    qh = q.permute(0, 2, 1, 3)
    kh, vh = (t.permute(0, 2, 1, 3).repeat_interleave(g, 1) for t in (k, v))
    s = scale * qh @ kh.transpose(-1, -2)
    if rel_table is not None:
        D = rel_map.numel() // 2
        bucket = rel_map.long().clamp(0, rel_table.shape[0] - 1)[d.clamp(-D, D) + D]
        s = s + rel_table.double()[bucket].permute(0, 3, 1, 2)
    s = s.masked_fill(~ok[:, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    e = (s - torch.where(m.isinf(), 0.0, m)).exp()
    l = e.sum(-1, keepdim=True)
    P = e / torch.where(l == 0, 1.0, l)
    out = P @ vh
    Av = P @ vh.abs()
    res = {"out": (out.permute(0, 2, 1, 3), (H8 * (Av + out.abs()) + F32 * Av).permute(0, 2, 1, 3))}
    res["lse"] = ((m + l.log()).squeeze(-1) / math.log(2), None)
    if dout is None:
        return res
    do = dout.double().permute(0, 2, 1, 3)
    dP = do @ vh.transpose(-1, -2)
    Dr = (do * out).sum(-1, keepdim=True)
    dS = P * (dP - Dr)
    h_out = 2.0 ** -20 if rel_table is not None or nk <= A.EXACT_KEYS else H8
    dD = (do.abs() * (h_out * (Av + out.abs()) + F32 * Av)).sum(-1, keepdim=True)
    e32 = F32 * P * (do.abs() @ vh.abs().transpose(-1, -2) + (do.abs() * Av).sum(-1, keepdim=True))
    edS = H8 * dS.abs() + P * dD + e32

    def kv(t):  # sum over the heads of a group
        return t.view(B, Hkv, g, nk, dh).sum(2).permute(0, 2, 1, 3)

    dq = scale * dS @ kh
    dk, dv = kv(scale * dS.transpose(-1, -2) @ qh), kv(P.transpose(-1, -2) @ do)
    res["dq"] = (dq.permute(0, 2, 1, 3), (scale * edS @ kh.abs() + H8 * dq.abs()).permute(0, 2, 1, 3))
    res["dk"] = (dk, kv(scale * edS.transpose(-1, -2) @ qh.abs()) + H8 * dk.abs())
    res["dv"] = (dv, (H8 + F32) * kv(P.transpose(-1, -2) @ do.abs()) + H8 * dv.abs())
    if rel_table is not None:
        nb = rel_table.shape[0]
        eT = P * dD + e32
        got = torch.zeros(2, H, nb, dtype=torch.float64, device=DEV)
        flat = bucket[:, None].expand(B, H, nq, nk).permute(1, 0, 2, 3).reshape(H, -1)
        got[0].scatter_add_(1, flat, dS.permute(1, 0, 2, 3).reshape(H, -1))
        got[1].scatter_add_(1, flat, eT.permute(1, 0, 2, 3).reshape(H, -1))
        res["drel"] = (got[0].t(), got[1].t())
    return res


def _within(name, got, ref):
    value, bound = ref
    err = (got.double() - value).abs()
    bad = ~(err <= bound * 1.0001 + 1e-30)
    assert not bad.any(), "%s: %d of %d outside, worst %.3g of its bound" % (
        name, int(bad.sum()), bad.numel(), float((err / (bound + 1e-300)).nan_to_num(float("inf")).max()))


def _check(q, k, v, scale, train=True, seed=5, **kw):
    gen = torch.Generator().manual_seed(seed)
    dout = _rand(gen, *q.shape) if train else None
    ref = _reference(q, k, v, scale, dout=dout, **kw)
    out = A.attention(q, k, v, scale=scale, **kw)
    _within("out", out, ref["out"])
    if not train:
        return out
    o, saved = A.attention(q, k, v, scale=scale, training=True, **kw)
    _within("out (training)", o, ref["out"])
    lse, want = saved.lse.double(), ref["lse"][0]
    assert torch.equal(lse == math.inf, want == -math.inf)  # rows without keys
    fine = want != -math.inf
    assert (lse - want)[fine].abs().max() <= 64 * 2.0 ** -18 if fine.any() else True
    grads = A.attention_backward(dout, q, k, v, o, saved, scale=scale, **kw)
    for name, g in zip(("dq", "dk", "dv", "drel"), grads):
        assert g.dtype == (torch.float32 if name == "drel" else torch.bfloat16)
        _within(name, g, ref[name])
    return o, saved, grads


def _table(gen, H, buckets=16, dist=24, both=True, std=1.0):
    return _rand(gen, buckets, H, std=std, dtype=torch.float32), A.relative_buckets(buckets, dist, both, device=DEV)


@pytest.mark.parametrize("dh", [32, 64, 80, 96, 128])
@pytest.mark.parametrize("bias", [False, True])
def test_full_attention_every_head_dim(dh, bias):
    gen = torch.Generator().manual_seed(dh)
    B, n, H = 2, 77, 3
    q, k, v = (_rand(gen, B, n, H, dh) for _ in range(3))
    kw = {}
    if bias:
        kw["rel_table"], kw["rel_map"] = _table(gen, H)
    _check(q, k, v, dh ** -0.5, **kw)


@pytest.mark.parametrize("nq,nk", [(1, 1), (1, 2), (2, 1), (16, 33), (17, 31), (31, 64), (32, 32), (33, 65), (127, 129), (128, 128),
                                   (129, 40), (257, 300)])
@pytest.mark.parametrize("bias", [False, True])
def test_lengths(nq, nk, bias):
    gen = torch.Generator().manual_seed(nq * 1000 + nk)
    q, k, v = _rand(gen, 2, nq, 2, 64), _rand(gen, 2, nk, 2, 64), _rand(gen, 2, nk, 2, 64)
    kw = {}
    if bias:
        kw["rel_table"], kw["rel_map"] = _table(gen, 2, buckets=8, dist=9)
    _check(q, k, v, 0.125, **kw)


@pytest.mark.parametrize("window,sinks", [((0, 0), 0), ((5, 0), 0), ((5, 3), 2), ((40, 0), 4), ((64, 64), 33), ((-1, 0), 0),
                                          ((-1, 7), 3), ((9, -1), 1), ((300, 0), 0), ((31, 0), 200), ((2 ** 31 - 1, 2 ** 31 - 1), 5)])
@pytest.mark.parametrize("bias", [False, True])
def test_windows_and_sinks(window, sinks, bias):
    gen = torch.Generator().manual_seed(7)
    B, n, H = 2, 203, 2
    q, k, v = (_rand(gen, B, n, H, 32) for _ in range(3))
    kw = {"window": window, "sinks": sinks}
    if bias:
        kw["rel_table"], kw["rel_map"] = _table(gen, H)
    _check(q, k, v, 32 ** -0.5, **kw)


@pytest.mark.parametrize("H,Hkv", [(4, 4), (4, 2), (6, 1), (12, 4)])
@pytest.mark.parametrize("bias", [False, True])
def test_shared_key_heads(H, Hkv, bias):
    gen = torch.Generator().manual_seed(H * 10 + Hkv)
    q, k, v = _rand(gen, 2, 150, H, 80), _rand(gen, 2, 150, Hkv, 80), _rand(gen, 2, 150, Hkv, 80)
    kw = {"window": (70, 0), "sinks": 3}
    if bias:
        kw["rel_table"], kw["rel_map"] = _table(gen, H, both=False)
    _check(q, k, v, 80 ** -0.5, **kw)


@pytest.mark.parametrize("bias", [False, True])
def test_ragged_batch_with_empty_sequences_and_garbage_past_the_end(bias):
    gen = torch.Generator().manual_seed(3)
    B, n, H = 5, 140, 2
    q, k, v = (_rand(gen, B, n, H, 64) for _ in range(3))
    kv_len = torch.tensor([140, 0, 1, 37, 96], dtype=torch.int32, device=DEV)
    for b in range(B):
        k[b, int(kv_len[b]):] = float("nan")
        v[b, int(kv_len[b]):] = float("inf")
    kw = {"kv_len": kv_len}
    if bias:
        kw["rel_table"], kw["rel_map"] = _table(gen, H)
    out, saved, grads = _check(q, k, v, 0.125, **kw)
    assert (out[1] == 0).all() and all((g[1] == 0).all() for g in grads[:3])
    for b in range(B):
        assert (grads[1][b, int(kv_len[b]):] == 0).all() and (grads[2][b, int(kv_len[b]):] == 0).all()
    _check(q, k, v, 0.125, window=(12, 2), sinks=1, **kw)  # later rows see nothing but the sink, or nothing at all


@pytest.mark.parametrize("nq,nk,start,window,sinks", [(1, 500, 333, (-1, 0), 0), (1, 500, 333, (40, 0), 3), (2, 70, 40, (5, 0), 0),
                                                      (100, 400, 250, (60, 0), 4), (100, 400, 250, (-1, 0), 0), (64, 300, 100, (20, 9), 0),
                                                      (150, 800, 500, (-1, -1), 0), (40, 500, 300, (33, 0), 70), (17, 90, -5, (3, 2), 0)])
@pytest.mark.parametrize("bias", [False, True])
def test_keys_that_no_query_sees_may_hold_anything(nq, nk, start, window, sinks, bias):
    """Places of a cache that are not written yet, or have left the window: nothing of them reaches a result."""
    gen = torch.Generator().manual_seed(nq + nk)
    B, H, Hkv, dh = 2, 4, 2, 80
    q, k, v = _rand(gen, B, nq, H, dh), _rand(gen, B, nk, Hkv, dh), _rand(gen, B, nk, Hkv, dh)
    kw = dict(window=window, sinks=sinks, q_start=torch.tensor([start, start + 3], dtype=torch.int32, device=DEV))
    if bias:
        kw["rel_table"], kw["rel_map"] = _table(gen, H)
    hidden = ~_seen(B, nq, nk, window, sinks, None, kw["q_start"])[0].any(1)
    assert hidden.any() or window == (-1, -1)
    zk, zv = (t.masked_fill(hidden[:, :, None, None], 0.0) for t in (k, v))
    k[hidden], v[hidden] = float("nan"), float("inf")
    do = _rand(gen, B, nq, H, dh)
    want, ws = A.attention(q, zk, zv, training=True, **kw)
    got, gs = A.attention(q, k, v, training=True, **kw)
    assert torch.equal(got, want) and torch.equal(gs.lse, ws.lse)
    for x, y in zip(A.attention_backward(do, q, k, v, got, gs, **kw), A.attention_backward(do, q, zk, zv, want, ws, **kw)):
        assert torch.equal(x, y)
    assert torch.equal(A.attention(q, k, v, **kw), A.attention(q, zk, zv, **kw))
    _check(q, zk, zv, dh ** -0.5, **kw)


def test_lengths_out_of_range_are_clamped():
    gen = torch.Generator().manual_seed(4)
    q, k, v = (_rand(gen, 3, 20, 1, 32) for _ in range(3))
    over = torch.tensor([1000, -5, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    inside = torch.tensor([20, 0, 20], dtype=torch.int32, device=DEV)
    assert torch.equal(A.attention(q, k, v, kv_len=over), A.attention(q, k, v, kv_len=inside))
    far = torch.tensor([2 ** 31 - 1, -2 ** 31, 0], dtype=torch.int32, device=DEV)
    got = A.attention(q, k, v, q_start=far, window=(3, 3))
    assert (got[:2] == 0).all() and got[2].abs().sum() > 0


@pytest.mark.parametrize("nq,H,Hkv", [(1, 2, 2), (1, 8, 2), (3, 4, 1), (16, 2, 2), (5, 6, 2), (17, 2, 2), (1, 40, 2)])
@pytest.mark.parametrize("nk", [5, 300, 4099])
@pytest.mark.parametrize("bias", [False, True])
def test_few_rows_against_a_cache(nq, H, Hkv, nk, bias):
    gen = torch.Generator().manual_seed(nq + nk)
    B = 3
    q, k, v = _rand(gen, B, nq, H, 128), _rand(gen, B, nk, Hkv, 128), _rand(gen, B, nk, Hkv, 128)
    kv_len = torch.tensor([nk, max(nq, nk // 2), nk - 1], dtype=torch.int32, device=DEV)
    start = kv_len - nq
    kw = {"kv_len": kv_len, "q_start": start}
    if bias:
        kw["rel_table"], kw["rel_map"] = _table(gen, H, both=False)
    for window, sinks in (((-1, 0), 0), ((100, 0), 4), ((-1, -1), 0)):
        _check(q, k, v, 128 ** -0.5, train=nk <= 300, window=window, sinks=sinks, **kw)


def test_few_rows_agree_with_the_rows_of_the_whole():
    gen = torch.Generator().manual_seed(1)
    q, k, v = _rand(gen, 2, 90, 2, 80), _rand(gen, 2, 90, 2, 80), _rand(gen, 2, 90, 2, 80)
    t, m = _table(gen, 2)
    whole = A.attention(q, k, v, window=(30, 0), sinks=2, rel_table=t, rel_map=m)
    for i in (0, 1, 29, 89):
        one = A.attention(q[:, i:i + 1], k, v, window=(30, 0), sinks=2, rel_table=t, rel_map=m,
                          q_start=torch.full((2,), i, dtype=torch.int32, device=DEV))
        assert (one[:, 0].float() - whole[:, i].float()).abs().max() <= 3 * H8 * v.float().abs().max()


def test_bias_edges_distances_and_a_hidden_key():
    gen = torch.Generator().manual_seed(2)
    n = 400
    q, k, v = (_rand(gen, 1, n, 2, 32) for _ in range(3))
    for dist, buckets in ((1, 2), (31, 8), (32, 32), (300, 64), (1024, 256)):
        m = torch.randint(-3, buckets + 3, (2 * dist + 1,), generator=gen, dtype=torch.int32).to(DEV)  # any map, clamped
        t = _rand(gen, buckets, 2, std=2.0, dtype=torch.float32)
        _check(q, k, v, 32 ** -0.5, rel_table=t, rel_map=m)
    # the widest map beside the widest head: more than 64 KB of LDS
    q, k, v = (_rand(gen, 1, 1100, 2, 128) for _ in range(3))
    _check(q, k, v, 128 ** -0.5, rel_table=_rand(gen, 256, 2, dtype=torch.float32),
           rel_map=torch.randint(0, 256, (2 * 1024 + 1,), generator=gen, dtype=torch.int32).to(DEV))
    q, k, v = (_rand(gen, 1, n, 2, 32) for _ in range(3))
    t, m = _table(gen, 2)
    t[int(m[24 + 3])] = -math.inf  # hides every key whose distance lies in that bucket
    ref = _reference(q, k, v, 0.2, rel_table=t, rel_map=m)
    _within("out", A.attention(q, k, v, scale=0.2, rel_table=t, rel_map=m), ref["out"])
    t[:] = -math.inf
    assert (A.attention(q, k, v, rel_table=t, rel_map=m) == 0).all()


def test_strides_packed_views_broadcast_and_unaligned_inputs():
    gen = torch.Generator().manual_seed(9)
    B, n, H, dh = 2, 75, 4, 80
    packed = _rand(gen, B, n, 3, H, dh)
    q, k, v = packed.unbind(2)
    base = A.attention(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(A.attention(q, k, v), base)
    heads_first = [t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (q, k, v)]
    assert torch.equal(A.attention(*heads_first), base)
    odd = torch.empty(B * n * H * dh + 3, dtype=torch.bfloat16, device=DEV)[3:].view(B, n, H, dh).copy_(q)
    assert odd.data_ptr() % 16 and torch.equal(A.attention(odd, k, v), base)
    wide = torch.empty(B, n, H, dh + 1, dtype=torch.bfloat16, device=DEV)[..., :dh].copy_(k)
    assert torch.equal(A.attention(q, wide, v), base)
    one = k[:, :, :1].expand(B, n, H, dh)  # a broadcast key head
    assert torch.equal(A.attention(q, one, v), A.attention(q, one.contiguous(), v))
    for nq in (75, 3):  # in place of the queries
        x = q[:, :nq].contiguous()
        want = A.attention(x, k, v)
        assert A.attention(x, k, v, out=x).data_ptr() == x.data_ptr() and torch.equal(x, want)
    # packed destinations; nothing around them is touched
    dst = torch.full((B, n, 3, H, dh), 7.0, dtype=torch.bfloat16, device=DEV)
    base, _ = A.attention(q.contiguous(), k.contiguous(), v.contiguous(), training=True)
    o, saved = A.attention(q, k, v, training=True, out=dst[:, :, 1])
    assert o.data_ptr() == dst[:, :, 1].data_ptr() and torch.equal(dst[:, :, 1], base)
    assert (dst[:, :, 0] == 7).all() and (dst[:, :, 2] == 7).all()
    do = _rand(gen, B, n, H, dh)
    want = A.attention_backward(do, q, k, v, base, saved)
    A.attention_backward(do, q, k, v, o, saved, dq=dst[:, :, 0], dk=dst[:, :, 1].clone(), dv=dst[:, :, 2])
    assert torch.equal(dst[:, :, 0], want[0]) and torch.equal(dst[:, :, 2], want[2])


@pytest.mark.parametrize("stride", [1 << 24, 1 << 25, 1 << 26])
def test_offsets_past_32_bits(stride):
    """Element offsets beyond 2^31 in one sequence, carried by the token stride (the widest is copied by the call)."""
    n = 200 if stride < 1 << 25 else 100 if stride < 1 << 26 else 40
    big = torch.empty((n - 1) * stride + 4096, dtype=torch.bfloat16, device=DEV)
    gen = torch.Generator().manual_seed(6)
    src = _rand(gen, 2, n, 2, 64)
    k = big.as_strided((1, n, 2, 64), (n * stride, stride, 64, 1))
    v = big.as_strided((1, n, 2, 64), (n * stride, stride, 64, 1), 2048)
    k.copy_(src[:1])
    v.copy_(src[1:])
    for nq in (1, 40):
        q = _rand(gen, 1, nq, 2, 64)
        assert torch.equal(A.attention(q, k, v), A.attention(q, src[:1], src[1:]))
    do = _rand(gen, 1, n, 2, 64)
    grads = []
    for x, y in ((k, v), (src[:1], src[1:])):
        o, saved = A.attention(x, x, y, training=True)
        grads.append((o,) + A.attention_backward(do, x, x, y, o, saved))
    assert all(torch.equal(x, y) for x, y in zip(*grads))


def test_results_repeat_exactly():
    gen = torch.Generator().manual_seed(8)
    q, k, v = (_rand(gen, 2, 600, 4, 80) for _ in range(3))
    t, m = _table(gen, 4, buckets=32, dist=128)
    do = _rand(gen, 2, 600, 4, 80)
    kw = dict(rel_table=t, rel_map=m)

    def once():
        o, saved = A.attention(q, k, v, training=True, **kw)
        return (o,) + tuple(A.attention_backward(do, q, k, v, o, saved, **kw))

    first = once()
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, once()))


def test_rows_with_one_key_have_no_score_gradient():
    """A softmax over one key is constant: dq, dk and the table's gradient are exactly zero, dv is dout."""
    gen = torch.Generator().manual_seed(30)
    q, k, v, do = (_rand(gen, 3, 50, 4, 80) for _ in range(4))
    t, m = _table(gen, 4)
    for kw in (dict(window=(0, 0)), dict(kv_len=torch.ones(3, dtype=torch.int32, device=DEV)), dict(window=(0, -1), kv_len=torch.ones(3, dtype=torch.int32, device=DEV), sinks=1)):
        for bias in ({}, dict(rel_table=t, rel_map=m)):
            o, saved = A.attention(q, k, v, training=True, **kw, **bias)
            g = A.attention_backward(do, q, k, v, o, saved, **kw, **bias)
            assert (g[0] == 0).all() and (g[1] == 0).all() and (len(g) < 4 or (g[3] == 0).all())
            if kw.get("window") == (0, 0):
                assert torch.equal(o, v) and torch.equal(g[2], do)


def test_gradients_against_differences():
    """Directional derivative of sum(out . w) by central differences of the float64 definition, along random directions."""
    gen = torch.Generator().manual_seed(12)
    B, n, H, dh = 1, 40, 2, 32
    q, k, v = (_rand(gen, B, n, H, dh) for _ in range(3))
    t, m = _table(gen, H, buckets=8, dist=12)
    w = _rand(gen, B, n, H, dh)
    kw = dict(window=(15, 4), sinks=2, rel_map=m)
    o, saved = A.attention(q, k, v, scale=0.3, training=True, rel_table=t, **kw)
    g = A.attention_backward(w, q, k, v, o, saved, scale=0.3, rel_table=t, **kw)
    for i, x in enumerate((q, k, v, t)):
        u = torch.randn(x.shape, generator=gen, dtype=torch.float64).to(DEV)

        def f(step):
            a = [z.double() for z in (q, k, v, t)]
            a[i] = a[i] + step * u
            return float((_reference(*a[:3], 0.3, rel_table=a[3], **kw)["out"][0] * w.double()).sum())

        num = (f(1e-4) - f(-1e-4)) / 2e-4
        ana = float((g[i].double() * u).sum())
        # bf16 gradients of |g| ~ rms: the projection of their roundings on u is below h |g| |u| (norms)
        slack = 3 * H8 * float(g[i].double().norm()) * 4 if i < 3 else 1e-4 * float((g[i].double().norm() * u.norm()))
        assert abs(num - ana) <= slack, (i, num, ana, slack)


def test_capture_replay_on_two_streams():
    gen = torch.Generator().manual_seed(14)
    q, k, v, do = (_rand(gen, 2, 300, 4, 64) for _ in range(4))
    q1, k1, v1 = _rand(gen, 2, 1, 4, 64), _rand(gen, 2, 5000, 4, 64), _rand(gen, 2, 5000, 4, 64)
    t, m = _table(gen, 4)
    kw = dict(rel_table=t, rel_map=m, window=(64, 64), sinks=2)

    def step():
        a, b = A.qk_norm_rope(q, k)
        o, saved = A.attention(a, b, v, training=True, **kw)
        g = A.attention_backward(do, a, b, v, o, saved, **kw)
        r = A.qk_norm_rope_backward(g[0], g[1], q, k)
        return (o, g[2], g[3], r[0], r[1], r[2], A.attention(q1, k1, v1, rel_table=t, rel_map=m))

    want = [x.clone() for x in step()]
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                got = step()
        graphs.append((g, s, got))
    for rep in range(3):
        for g, s, got in graphs:
            for x in got:
                x.zero_()
        torch.cuda.synchronize()
        for g, s, got in graphs:  # both at once
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for g, s, got in graphs:
            assert all(torch.equal(x, y) for x, y in zip(got, want)), rep
        assert all(torch.equal(x, y) for x, y in zip(step(), want))


def test_empty_tensors():
    z = torch.zeros(0, 4, 2, 64, dtype=torch.bfloat16, device=DEV)
    assert A.attention(z, z, z).shape == z.shape
    q, none = torch.ones(2, 3, 2, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(2, 0, 2, 64, dtype=torch.bfloat16, device=DEV)
    o, saved = A.attention(q, none, none, training=True)
    assert (o == 0).all() and (saved.lse == math.inf).all()
    g = A.attention_backward(q, q, none, none, o, saved)
    assert (g[0] == 0).all() and g[1].shape == none.shape
    a, b = A.qk_norm_rope(z, z)
    assert a.shape == z.shape and b.shape == z.shape


def test_refusals():
    q = torch.zeros(2, 20, 4, 64, dtype=torch.bfloat16, device=DEV)
    t, m = torch.zeros(8, 4, device=DEV), A.relative_buckets(8, 20, device=DEV)
    for call in (lambda: A.attention(q.float(), q, q), lambda: A.attention(q, q[:, :, :3], q[:, :, :3]),
                 lambda: A.attention(q, q, q[:, :5]), lambda: A.attention(q, q.cpu(), q), lambda: A.attention(q[0], q, q),
                 lambda: A.attention(q, q, q, rel_table=t), lambda: A.attention(q, q, q, rel_table=t.half(), rel_map=m),
                 lambda: A.attention(q, q, q, rel_table=t[:, :3], rel_map=m), lambda: A.attention(q, q, q, rel_table=t, rel_map=m[:-1]),
                 lambda: A.attention(q, q, q, kv_len=torch.zeros(2, device=DEV)),
                 lambda: A.attention(q, q, q, q_start=torch.zeros(3, dtype=torch.int32, device=DEV)),
                 lambda: A.attention(q, q, q, out=q[:1].expand(2, 20, 4, 64)), lambda: A.attention(q, q, q, out=q.float()),
                 lambda: A.qk_norm_rope(q.half(), q.half()), lambda: A.qk_norm_rope(q, q.float()),
                 lambda: A.qk_norm_rope(q, q, q_gamma=torch.ones(63, device=DEV)),
                 lambda: A.qk_norm_rope(q, q, positions=torch.zeros(2, 20, device=DEV)),
                 lambda: A.qk_norm_rope(q, q[:, :5]), lambda: A.attention(q, q, q, window=(1 << 32, 0)),
                 lambda: A.attention(q, q, q, window=(5, -(1 << 33))), lambda: A.attention(q, q, q, window=(5, 0, 0)),
                 lambda: A.attention(q, q, q, window=(5, 0), sinks=(1 << 32) + 1), lambda: A.qk_norm_rope(q, q, position0=1 << 32),
                 lambda: A.qk_norm_rope(q, q, rotary_dim=(1 << 32) + 64)):
        with pytest.raises(ValueError):
            call()
    from mint_amd._lib import FactError
    odd = torch.zeros(2, 20, 4, 48, dtype=torch.bfloat16, device=DEV)
    for call in (lambda: A.attention(odd, odd, odd), lambda: A.attention(q, q, q, scale=0.0), lambda: A.attention(q, q, q, sinks=-1),
                 lambda: A.attention(q, q, q, scale=float("nan")), lambda: A.qk_norm_rope(q, q, rotary_dim=65),
                 lambda: A.qk_norm_rope(q, q, rotary_dim=12), lambda: A.qk_norm_rope(q, q, eps=-1.0),
                 lambda: A.qk_norm_rope(q, q, base=0.0), lambda: A.qk_norm_rope(q, q, position0=(1 << 31) - 10),
                 lambda: A.attention(q, q.clone(), q.clone(), out=q, window=(1, 1), sinks=-2),
                 lambda: (lambda k: A.attention(q, k, q.clone(), out=k))(q.clone())):
        with pytest.raises(FactError):
            call()


# ---- norm of queries and keys with rotation ---------------------------------------------------------------------------
def _norm_reference(q, k, gq, gk, eps, rot, base, inter, pos, dq=None, dk=None):
    leaves = [t.double().requires_grad_(True) for t in (q, k, gq, gk)]
    dh = q.shape[-1]

    def one(x, g):
        y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * g
        if not rot:
            return y
        i = torch.arange(rot // 2, device=x.device)
        a, b = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
        ang = pos.double()[..., None] * base ** (-2.0 * i.double() / rot)
        c, s = ang.cos()[:, :, None], ang.sin()[:, :, None]
        z = y.clone()
        z[..., a] = y[..., a] * c - y[..., b] * s
        z[..., b] = y[..., b] * c + y[..., a] * s
        return z

    zq, zk = one(leaves[0], leaves[2]), one(leaves[1], leaves[3])
    got = [zq.detach(), zk.detach()]
    if dq is not None:
        got += torch.autograd.grad((zq, zk), leaves, (dq.double(), dk.double()))
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dh,rot,inter", [(8, 8, False), (24, 16, True), (32, 0, False), (64, 64, True), (80, 80, False), (80, 40, False),
                                          (96, 96, True), (128, 128, False), (128, 64, True), (120, 8, False)])
@pytest.mark.parametrize("B,n,H,Hkv", [(1, 1, 1, 1), (2, 37, 5, 2), (3, 130, 20, 1)])
def test_norm_and_rotation(dtype, dh, rot, inter, B, n, H, Hkv):
    """One rounding of each result (half a step of its type) on 32-bit arithmetic: a row sum of dh terms, an angle exact to 2^-22."""
    gen = torch.Generator().manual_seed(dh + rot + n)
    packed = _rand(gen, B, n, H + Hkv, dh, dtype=dtype, std=3.0)
    q, k = packed[:, :, :H], packed[:, :, H:]
    gq, gk = (1 + _rand(gen, dh, dtype=torch.float32, std=0.3) for _ in range(2))
    dq, dk = _rand(gen, B, n, H, dh, dtype=dtype), _rand(gen, B, n, Hkv, dh, dtype=dtype)
    pos = torch.randint(-1000, 3_000_000, (B, n), generator=gen, dtype=torch.int32).to(DEV)
    kw = dict(eps=1e-5, rotary_dim=rot, base=5000.0, interleaved=inter, positions=pos)
    want = _norm_reference(q, k, gq, gk, 1e-5, rot, 5000.0, inter, pos, dq, dk)
    got = list(A.qk_norm_rope(q, k, gq, gk, **kw))
    dxq, dxk, dgq, dgk = A.qk_norm_rope_backward(dq, dk, q, k, gq, gk, **kw)
    got += [dxq, dxk, dgq, dgk]
    half = H8 if dtype == torch.bfloat16 else 2.0 ** -24
    for i, (x, y) in enumerate(zip(got, want)):
        # size of the terms behind a value: its row's largest (a rotation mixes two, a mean mixes all)
        if i < 4:
            size = y.abs().amax(-1, keepdim=True)
            assert ((x.double() - y).abs() <= half * y.abs() + 2.0 ** -18 * size + 1e-12).all(), i
        else:  # sum over B n heads of products: 2^-20 of the sum of their absolute values, bounded by sqrt(count) * norm
            heads = H if i == 4 else Hkv
            assert x.dtype == torch.float32
            assert (x.double() - y).abs().max() <= 2.0 ** -18 * B * n * heads * 12, i


def test_norm_in_place_defaults_and_repeats():
    gen = torch.Generator().manual_seed(4)
    q, k = _rand(gen, 2, 50, 4, 64), _rand(gen, 2, 50, 2, 64)
    a, b = A.qk_norm_rope(q, k, position0=7)
    pos = torch.arange(7, 57, dtype=torch.int32, device=DEV)
    ones = torch.ones(64, device=DEV)
    c, d = A.qk_norm_rope(q, k, ones, ones, positions=pos)
    assert torch.equal(a, c) and torch.equal(b, d)
    q2, k2 = q.clone(), k.clone()
    A.qk_norm_rope(q2, k2, position0=7, q_out=q2, k_out=k2)
    assert torch.equal(q2, a) and torch.equal(k2, b)
    dq, dk = _rand(gen, 2, 50, 4, 64), _rand(gen, 2, 50, 2, 64)
    want = A.qk_norm_rope_backward(dq, dk, q, k)
    again = A.qk_norm_rope_backward(dq, dk, q, k)
    assert all(torch.equal(x, y) for x, y in zip(want, again))
    A.qk_norm_rope_backward(dq, dk, q, k, dq=dq, dk=dk)
    assert torch.equal(dq, want[0]) and torch.equal(dk, want[1])


def test_norm_of_zero_rows_stays_finite():
    z = torch.zeros(1, 3, 2, 64, dtype=torch.bfloat16, device=DEV)
    a, b = A.qk_norm_rope(z, z, eps=1e-6)
    assert (a == 0).all() and (b == 0).all()
    g = A.qk_norm_rope_backward(torch.ones_like(z), torch.ones_like(z), z, z, eps=1e-6)
    assert all(torch.isfinite(x).all() for x in g)


def test_norm_attention_run_as_a_block():
    """The run a transformer layer makes - norm, attention, both backwards - against float64 of the whole."""
    gen = torch.Generator().manual_seed(21)
    B, n, H, dh = 2, 60, 2, 64
    q, k, v, do = (_rand(gen, B, n, H, dh) for _ in range(4))
    gq, gk = (1 + _rand(gen, dh, dtype=torch.float32, std=0.2) for _ in range(2))
    t, m = _table(gen, H)
    kw = dict(window=(20, 20), sinks=2, rel_table=t, rel_map=m)
    a, b = A.qk_norm_rope(q, k, gq, gk)
    o, saved = A.attention(a, b, v, training=True, **kw)
    da, db, dv, dt = A.attention_backward(do, a, b, v, o, saved, **kw)
    dq, dk, dgq, dgk = A.qk_norm_rope_backward(da, db, q, k, gq, gk)
    leaves = [x.double().requires_grad_(True) for x in (q, k, v, gq, gk, t)]
    pos = torch.arange(n, device=DEV).double()
    i = torch.arange(dh // 2, device=DEV)
    c, s = (pos[:, None] * 10000.0 ** (-2.0 * i / dh)).cos(), (pos[:, None] * 10000.0 ** (-2.0 * i / dh)).sin()

    def norm(x, g):
        y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * g
        y0, y1 = y[..., :dh // 2], y[..., dh // 2:]
        c4, s4 = c[None, :, None], s[None, :, None]
        return torch.cat((y0 * c4 - y1 * s4, y1 * c4 + y0 * s4), -1).permute(0, 2, 1, 3)

    ok, d = _seen(B, n, n, (20, 20), 2, None, None)
    D = m.numel() // 2
    x = norm(leaves[0], leaves[3]) @ norm(leaves[1], leaves[4]).transpose(-1, -2) * dh ** -0.5
    x = x + leaves[5][m.long()[d.clamp(-D, D) + D]].permute(0, 3, 1, 2)
    y = (x.masked_fill(~ok[:, None], -math.inf).softmax(-1) @ leaves[2].permute(0, 2, 1, 3)).permute(0, 2, 1, 3)
    ref = torch.autograd.grad(y, leaves, do.double())
    # a and b are rounded on the way (h each): scores move by 2 h |q| |k| scale ~ 2 h sqrt(dh), P by as much of itself, and
    # the gradients, products of at most four such factors, by 4 times it in norm
    tol = 4 * 2 * H8 * math.sqrt(dh) * 0.25
    for got, want, name in ((o, y, "out"), (dq, ref[0], "dq"), (dk, ref[1], "dk"), (dv, ref[2], "dv"), (dgq, ref[3], "dgq"),
                            (dgk, ref[4], "dgk"), (dt, ref[5], "dtable")):
        assert float((got.double() - want).norm() / want.norm()) <= tol, name


def test_a_second_call_of_a_geometry_checks_and_computes_like_the_first():
    """Calls of one geometry share their checks; alignment, copies and types are still looked at, and results follow the tensors."""
    gen = torch.Generator().manual_seed(40)
    B, n, H, dh = 2, 40, 2, 64
    t, m = _table(gen, H)
    for rep in range(3):
        q, k, v, do = (_rand(gen, B, n, H, dh) for _ in range(4))
        kw = dict(rel_table=t, rel_map=m, window=[9, 9], sinks=rep)
        _check(q, k, v, 0.2, seed=rep, **kw)
        want = A.attention(q, k, v, **kw)
        odd = torch.empty(q.numel() + 4, dtype=torch.bfloat16, device=DEV)[4:].view(q.shape).copy_(q)
        assert odd.data_ptr() % 16 == 8 and odd.stride() == q.stride()
        assert torch.equal(A.attention(odd, k, v, **kw), want)
        dst = torch.zeros_like(q)
        assert A.attention(q, k, v, out=dst, **kw) is dst and torch.equal(dst, want)
        with pytest.raises(ValueError):
            A.attention(q, k, v, out=odd, **kw)
        with pytest.raises(ValueError):
            A.attention(q, k.float(), v, **kw)
        a, b = A.qk_norm_rope(q, k, position0=rep)
        c, d = A.qk_norm_rope(odd, k, position0=rep)
        assert torch.equal(a, c) and torch.equal(b, d)
        g = A.qk_norm_rope_backward(do, do, q, k, position0=rep)
        h = A.qk_norm_rope_backward(do, do, odd, k, position0=rep)
        assert all(torch.equal(x, y) for x, y in zip(g, h))
