"""GPU: a prompt gets the same bits in any company, rows whose scores rise steeply among them.

What a prompt is packed with decides how its rows are spread over workgroups and waves and how many keys a tile holds; the reference point
of a row (see csrc/prompt.hip) has to move at the same keys in all of them."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def attend(K, lens, rows, heads, dtype):
    """The first ``rows`` outputs of a call over prompts of ``lens``; ``rows`` = (q, k, v) of the first one, noise for the others."""
    N = sum(lens)
    g = torch.Generator(device='cuda').manual_seed(5)
    parts = []
    for x in rows:
        y = torch.randn((N, x.shape[1]), generator=g, device='cuda').to(dtype)
        y[:x.shape[0]] = x
        parts.append(y)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    out = torch.empty_like(parts[0])
    K.attn_prompt(*parts, torch.tensor(cu, dtype=torch.int32, device='cuda'), out, *heads, scale=1.0)
    return out[:lens[0]].clone()


# natural units per key: 64 keys stay below 2^60; 64 pass it; 32 pass it; 64 pass 2^127; 32 pass 2^127; falling
@pytest.mark.parametrize('growth', [0.5, 0.8, 1.45, 1.9, 2.9, 40.0, -1.3])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('heads,kv_heads,dh', [(8, 8, 32), (8, 8, 64), (8, 2, 64), (8, 8, 128), (8, 2, 128), (4, 1, 256), (8, 8, 40)])
def test_steep_rows_have_the_same_bits_in_any_company(heads, kv_heads, dh, growth, dtype):
    import tst_amd  # noqa: F401
    from tst_amd import kernels as K
    L, g = 203, torch.Generator(device='cuda').manual_seed(dh)
    q, k, v = (torch.randn((L, n * dh), generator=g, device='cuda') for n in (heads, kv_heads, kv_heads))
    for h in range(heads):
        q[:, h * dh] = 1.0 + 0.1 * h
    for h in range(kv_heads):
        k[:, h * dh] = torch.arange(L, device='cuda') * growth
    rows = [x.to(dtype) for x in (q, k, v)]
    alone = attend(K, [L], rows, (heads, kv_heads), dtype)
    assert torch.isfinite(alone).all()
    for lens in ([L, 300, 17], [L, 1, 2, 3, 4, 5], [L] + [3] * 200, [L] + [40] * 160, [L] + [90] * 130):
        got = attend(K, lens, rows, (heads, kv_heads), dtype)
        assert torch.equal(got, alone), (lens[:3], len(lens), int((got != alone).any(1).sum()))
    # A score (dh products of three pieces each) is off by (3 dh + 2) half steps of fp32 of sum|q k|, a weight by twice that, by 4 half steps of
    # its distance from the largest score and by 4 of its own, a sum of L weights by L; numerator and denominator each.  bf16 rounds
    # the weights and the result once more.
    q, k, v = (x.double()[:, :dh] for x in rows)
    dead = torch.ones(L, L, dtype=torch.bool, device='cuda').triu(1)
    p, mag = (q @ k.t()).masked_fill(dead, -math.inf), (q.abs() @ k.abs().t()).masked_fill(dead, 0.0).amax(1, keepdim=True)
    w = torch.softmax(p, 1)
    wide = torch.where(w > 1e-12, p.amax(1, keepdim=True) - p, torch.zeros_like(p)).amax(1, keepdim=True)
    tol = 2 * (2 * (3 * dh + 2) * mag + 4 * wide + 4 + 2 * L) * 2.0 ** -24 * (w @ v.abs()) + 2.0 ** -24 * (w @ v).abs()
    if dtype == torch.bfloat16:
        tol += 2.0 ** -8 * (w @ v.abs() + (w @ v).abs())
    assert ((alone[:, :dh].double() - w @ v).abs() <= tol).all()
