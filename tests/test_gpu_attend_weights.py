"""GPU: attention over the 4-bit cache keeps its weights beyond bf16: the output's rounding is the only one to 8 bits."""
import pytest
import torch

from test_gpu_prompted import K, U32, UBF, attend64, filled_cache, i32  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('heads,kv_heads,dh', [(8, 8, 32), (8, 2, 64), (16, 4, 128), (4, 1, 256)])
@pytest.mark.parametrize('lens', [[1, 2, 3, 5], [40, 64, 65], [300, 700], [5000]], ids=str)
def test_bf16_weights_are_not_rounded_to_bf16(K, heads, kv_heads, dh, lens):  # noqa: F811
    """Values that nearly cancel show what the weights lost: with two bf16 pieces a weight is off by 2^-8 of 2^-8 of it, half a step each
    (numerator only: the sum is of the whole weights); the scores' and sums' errors as everywhere, the result rounded once."""
    cache, table, vals = filled_cache(K, lens, kv_heads, dh, 32, seed=dh)
    q = torch.randn((len(lens), heads * dh), generator=torch.Generator(device='cuda').manual_seed(7), device='cuda').to(torch.bfloat16)
    out = torch.empty_like(q)
    K.attn_cache4(q, cache, table, i32(lens), out, len(lens), heads, max(lens))
    per, w = heads // kv_heads, kv_heads * dh
    for r, n in enumerate(lens):
        for h in range(heads):
            g = h // per
            want, absv, rel = attend64(q[r:r + 1, h * dh:(h + 1) * dh], vals[r][:n, g * dh:(g + 1) * dh], vals[r][:n, w + g * dh:w + (g + 1) * dh],
                                       dh ** -0.5, False)
            tol = (rel + UBF ** 2) * absv + UBF * want.abs() + 1e-30
            err = (out[r:r + 1, h * dh:(h + 1) * dh].double() - want).abs()
            assert not (err > tol).any(), (r, h, (err / tol).max().item())
