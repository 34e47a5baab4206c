"""The attention operators have a backward of their own and record no graph: tensors that require grad are refused under grad mode."""
import pytest
import torch

from mint_amd import attention as A


def _raises(call):
    with pytest.raises(ValueError, match="requires grad"):
        call()


def test_heads_that_require_grad_are_refused():
    """The check comes before the one for the device, so it can be seen here."""
    x = torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16)
    g = x.clone().requires_grad_(True)
    saved = A.AttentionSaved(torch.zeros(2, 2, 4), None)
    for call in (lambda: A.attention(g, x, x), lambda: A.attention(g * 1, x, x), lambda: A.qk_norm_rope(g, x),
                 lambda: A.attention_backward(x, g, x, x, x, saved), lambda: A.qk_norm_rope_backward(x, x, g, x)):
        _raises(call)
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):  # the next check
            call()
    with pytest.raises(ValueError, match="CUDA"):
        A.attention(g.detach(), x, x)


@pytest.mark.gpu
def test_every_tensor_that_requires_grad_is_refused():
    """Also by the later calls of a geometry, which share the first one's checks, and also where no_grad calls came first."""
    gen = torch.Generator().manual_seed(3)
    q, k, v, do = (torch.randn(2, 20, 2, 64, generator=gen).bfloat16().cuda() for _ in range(4))
    t, m = torch.randn(8, 2, generator=gen).cuda(), A.relative_buckets(8, 12, device="cuda")
    gq, gk = torch.ones(64, device="cuda"), torch.ones(64, device="cuda")
    att = dict(q=q, k=k, v=v, rel_table=t, out=torch.empty_like(q))
    fixed = dict(rel_map=m)
    o, saved = A.attention(q, k, v, training=True, rel_table=t, **fixed)
    back = dict(dout=do, q=q, k=k, v=v, out=o, rel_table=t, dq=torch.empty_like(q), dk=torch.empty_like(q), dv=torch.empty_like(q))
    norm = dict(q=q, k=k, q_gamma=gq, k_gamma=gk, q_out=torch.empty_like(q), k_out=torch.empty_like(q))
    nback = dict(dq_out=do, dk_out=v, q=q, k=k, q_gamma=gq, k_gamma=gk, dq=torch.empty_like(q), dk=torch.empty_like(q))
    for call, kw, more in ((A.attention, att, fixed), (A.attention_backward, back, dict(fixed, saved=saved)),
                           (A.qk_norm_rope, norm, {}), (A.qk_norm_rope_backward, nback, {})):
        call(**kw, **more)
        for name in kw:
            asks = dict(kw, **{name: kw[name].detach().requires_grad_(True)})
            for _ in range(2):
                with torch.no_grad():
                    got = call(**asks, **more)
                assert all(not x.requires_grad for x in (got if isinstance(got, tuple) else (got,)) if x is not asks[name])
                _raises(lambda: call(**asks, **more))
        call(**kw, **more)
    for i in range(2):
        asks = A.AttentionSaved(*(x.detach().requires_grad_(j == i) for j, x in enumerate(saved)))
        _raises(lambda: A.attention_backward(saved=asks, **dict(back, **fixed)))
