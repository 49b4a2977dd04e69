"""GPU: bf16 prompt attention divides by the sum of the weights that it multiplied the values with."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def K():
    import tst_amd  # noqa: F401
    from tst_amd import kernels
    return kernels


def cu_of(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device='cuda')


@pytest.mark.parametrize('heads,kv_heads,dh', [(2, 2, 32), (8, 2, 64), (4, 4, 128), (4, 1, 256), (2, 2, 40), (2, 1, 96)])
@pytest.mark.parametrize('lens', [[400], [400] + [5] * 200], ids=['alone', 'beside short ones'])
@pytest.mark.parametrize('at', [3, 40, 333])
def test_a_row_that_one_key_takes_gets_that_value(K, heads, kv_heads, dh, lens, at):
    """One key scores at least 60 natural units above the others: their weights are below 400 e^-60 of its own, so the exact result is its value but
    for 1e-23, and 1 + 3 half steps of fp32 (sum, reciprocal, product) do not move a bf16 number.  The key's own weight is any number: the
    scores differ from row to row."""
    N, g = sum(lens), torch.Generator(device='cuda').manual_seed(dh + at)
    q, k = torch.randn((N, heads * dh), generator=g, device='cuda') * 0.05, torch.randn((N, kv_heads * dh), generator=g, device='cuda') * 0.05
    v = torch.randn((N, kv_heads * dh), generator=g, device='cuda').to(torch.bfloat16)
    q.view(N, heads, dh)[:, :, 0] = 1 + torch.rand((N, heads), generator=g, device='cuda')
    k.view(N, kv_heads, dh)[:, :, 0] = 0
    k.view(N, kv_heads, dh)[at, :, 0] = 70.0
    q, k = q.to(torch.bfloat16), k.to(torch.bfloat16)
    out = torch.empty((N, heads * dh), dtype=torch.bfloat16, device='cuda')
    K.attn_prompt(q, k, v, cu_of(lens), out, heads, kv_heads, scale=1.0)
    want = v.view(N, kv_heads, dh)[at].repeat_interleave(heads // kv_heads, 0).reshape(-1)
    got = out[at:lens[0]]
    assert torch.equal(got, want.expand_as(got)), int((got != want).sum())


@pytest.mark.parametrize('dh', [32, 64, 128, 256])
@pytest.mark.parametrize('L', [60, 300, 2000])
def test_peaked_rows_lose_little_more_than_the_results_rounding(K, dh, L):
    """Rounded weights w (1 + d), |d| <= 2^-8, in numerator and denominator: the result is off by at most 2^-8 sum w |v - out|, which a peaked row
    makes small, and by its own rounding (scores and sums in fp32: as in the other tests)."""
    g = torch.Generator(device='cuda').manual_seed(L)
    q, k, v = (torch.randn((L, dh), generator=g, device='cuda').to(torch.bfloat16) for _ in range(3))
    out, scale = torch.empty_like(q), 30.0 / math.sqrt(dh)
    K.attn_prompt(q, k, v, cu_of([L]), out, 1, scale=scale)
    qd, kd, vd = q.double(), k.double(), v.double()
    dead = torch.ones((L, L), dtype=torch.bool, device='cuda').triu(1)
    s, mag = ((qd @ kd.t()) * scale).masked_fill(dead, -math.inf), ((qd.abs() @ kd.abs().t()) * scale).masked_fill(dead, 0.0).amax(1, keepdim=True)
    w = torch.softmax(s, 1)
    want, wide = w @ vd, torch.where(w > 1e-12, s.amax(1, keepdim=True) - s, torch.zeros_like(s)).amax(1, keepdim=True)
    rel = 2 * (2 * (3 * dh + 2) * mag + 4 * wide + 4 + 2 * L) * 2.0 ** -24
    apart = torch.stack([(w @ (vd[:, e:e + 1] - want[:, e].unsqueeze(0)).abs()).diagonal() for e in range(dh)], 1)     # sum_j w_ij |v_je - out_ie|
    tol = 2.0 ** -8 * (apart * (1 + 2.0 ** -7) + want.abs()) + rel * (w @ vd.abs()) + 1e-30
    err = (out.double() - want).abs()
    assert not (err > tol).any(), (err / tol).max().item()
