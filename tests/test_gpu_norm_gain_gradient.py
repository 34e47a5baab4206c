"""The gain gradients of the q / k norm against float64, bounded by the sum of the absolute values of the terms behind each.

A term is dz turned back times x r.  Its own roundings, in 2^-24 of |turned parts| |x r|: the sum of up to 128 squares behind r (8
values a lane, then 4 moves: 12 additions, halved by the root), the root itself (2), x r and the product (2), the turn (3) and its
cosine and sine (an angle rounded to 2^-24 of half a turn, pi, and 2 of the functions): 20.  A gradient adds its terms in the
wave (at these sizes up to 3 units of 3 heads a lane), its lane groups (4), waves (3), rows of partial sums (16 a thread, then 31):
63 additions.  Together 83 * 2^-24 < 2^-17 of the sum of absolute values.

Roundings point either way, so over the dh gradients the error's norm stays far below that: each of the terms adds at random, 20
roundings of 2^-24 each at the most, and each of the 63 additions one of a partial sum that random terms leave below sqrt(count)
of their size: (20 + 63) * 2^-24 * sqrt(count) < 2^-17 sqrt(count) of a term's root mean square, sqrt(dh) of that in norm.  Terms
kept in bf16 would be 2^-9 / sqrt(3) sqrt(count) off, 150 times as much."""
import math

import pytest
import torch

from mint_amd import attention as A

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dh,rot,inter", [(8, 8, False), (32, 0, False), (80, 80, False), (80, 40, True), (128, 128, False), (128, 64, True)])
@pytest.mark.parametrize("B,n,H,Hkv", [(1, 1, 1, 1), (2, 37, 5, 2), (3, 130, 20, 1), (16, 360, 10, 10)])
def test_gain_gradients(dtype, dh, rot, inter, B, n, H, Hkv):
    gen = torch.Generator().manual_seed(dh + rot + n)
    q, k, dq, dk = ((torch.randn(B, n, h, dh, generator=gen) * std).to(dtype).cuda() for h, std in ((H, 3.0), (Hkv, 3.0), (H, 1.0), (Hkv, 1.0)))
    gq, gk = ((1 + 0.3 * torch.randn(dh, generator=gen)).cuda() for _ in range(2))
    pos = torch.randint(-1000, 3_000_000, (B, n), generator=gen, dtype=torch.int32).cuda()
    got = A.qk_norm_rope_backward(dq, dk, q, k, gq, gk, eps=1e-5, rotary_dim=rot, base=5000.0, interleaved=inter, positions=pos)[2:]
    i = torch.arange(rot // 2, device="cuda")
    a, b = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
    angle = pos.double()[..., None, None] * 5000.0 ** (-2.0 * i.double() / max(rot, 1))
    c, s = angle.cos(), angle.sin()
    for x, dz, grad in ((q, dq, got[0]), (k, dk, got[1])):
        x, dz = x.double(), dz.double()
        xr = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)
        dy, parts = dz.clone(), dz.abs()
        if rot:
            dy[..., a], dy[..., b] = dz[..., a] * c + dz[..., b] * s, dz[..., b] * c - dz[..., a] * s
            parts[..., a] = parts[..., b] = dz[..., a].abs() + dz[..., b].abs()
        term = dy * xr
        want, total = term.sum((0, 1, 2)), (parts * xr.abs()).sum((0, 1, 2))
        err = (grad.double() - want).abs()
        assert grad.dtype == torch.float32 and (err <= 2.0 ** -17 * total).all(), float((err / total).max())
        rms = float((parts * xr.abs()).square().mean().sqrt())
        assert float(err.norm()) <= 2.0 ** -17 * math.sqrt(x[..., 0].numel()) * rms * math.sqrt(dh)
