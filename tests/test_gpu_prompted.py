"""GPU: the operators of prompted decoding against plain statements of their definitions in 64 bits: packed prompt attention, page
tables and slot maps, the 4-bit cache (stored, read back, attended to), the rules on logits and the grammar step.

Tolerances count roundings (u = 2^-24 for fp32, 2^-8 for bf16).  A score is a sum of n = dh products scaled once: it is off by at most
d = (n + 2) u32 * scale * sum|q k|.  exp(s - m) is off by 2 d from its argument, by |s - m| u32 * 4 from forming the argument in fp32
(its difference, its product with log2 e) and by 4 u32 of its own.  Summing L weights adds L u32.  An output is a weighted mean of
values: off by (those relative errors, twice for numerator and denominator) * sum w|v|, L u32 for its own sum.  bf16 adds u_bf16 *
sum w|v| for the weights' rounding and u_bf16 * |out| for the result's.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U32, UBF = 2.0 ** -24, 2.0 ** -8


@pytest.fixture(scope='module')
def K():
    import tst_amd  # noqa: F401
    assert torch.cuda.is_available()
    from tst_amd import kernels
    return kernels


def gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device='cuda')


def attend64(q, k, v, scale, causal):
    """q [Lq, dh], k, v [Lk, dh] in 64 bits -> (out, the bound's parts: sum w|v|, relative error of the weights)"""
    q, k, v = q.double(), k.double(), v.double()
    s = (q @ k.t()) * scale
    mag = (q.abs() @ k.abs().t()) * scale
    if causal:
        dead = torch.ones_like(s, dtype=torch.bool).triu(1)
        s = s.masked_fill(dead, -math.inf)
        mag = mag.masked_fill(dead, 0.0)
    w = torch.softmax(s, 1)
    wide = torch.where(w > 1e-12, s.amax(1, keepdim=True) - s, torch.zeros_like(s)).amax(1, keepdim=True)
    rel = 2 * (2 * (q.shape[1] * 3 + 2) * U32 * mag.amax(1, keepdim=True) + (4 * wide + 4 + 2 * k.shape[0]) * U32)
    return w @ v, w @ v.abs(), rel


def check(got, want, absv, rel, bf16):
    tol = rel * absv + 1e-30
    if bf16:
        tol = tol + UBF * absv + UBF * want.abs()
    else:
        tol = tol + U32 * want.abs()
    err = (got.double() - want).abs()
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert not (err > tol).any() and not torch.isnan(got).any(), worst


# ---- packed prompt attention ----------------------------------------------------------------------------------------------------
def prompt_case(K, lens, heads, kv_heads, dh, dtype, seed=0, before=0, behind=0, pad=0, scale=None):
    g = gen(seed)
    cu = [before]
    for n in lens:
        cu.append(cu[-1] + n)
    N = cu[-1] + behind
    width = (heads + 2 * kv_heads) * dh + pad
    qkv = torch.randn((N, width), generator=g, device='cuda').to(dtype)
    a, b = heads * dh, (heads + kv_heads) * dh
    q, k, v = qkv[:, :a], qkv[:, a:b], qkv[:, b:b + kv_heads * dh]
    out = torch.full((N, a), 7.0, device='cuda', dtype=dtype)
    K.attn_prompt(q, k, v, i32(cu), out, heads, kv_heads, scale=scale)
    return q, k, v, cu, out


def check_prompt(q, k, v, cu, out, heads, kv_heads, dh, dtype, scale=None):
    per = heads // kv_heads
    for b in range(len(cu) - 1):
        r = slice(cu[b], cu[b + 1])
        if cu[b] == cu[b + 1]:
            continue
        for h in range(heads):
            g = h // per
            want, absv, rel = attend64(q[r, h * dh:(h + 1) * dh], k[r, g * dh:(g + 1) * dh], v[r, g * dh:(g + 1) * dh],
                                       dh ** -0.5 if scale is None else scale, True)
            check(out[r, h * dh:(h + 1) * dh], want, absv, rel, dtype == torch.bfloat16)


LENS = [[1], [0, 1, 2, 0], [15, 16, 17], [31, 33, 32], [63, 64, 65], [127, 129, 1, 128], [255, 257], [3, 300, 0, 511, 7], [1000]]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('lens', LENS, ids=str)
def test_prompt_lengths(K, lens, dtype):
    q, k, v, cu, out = prompt_case(K, lens, 4, 2, 64, dtype, seed=len(lens) + sum(lens))
    check_prompt(q, k, v, cu, out, 4, 2, 64, dtype)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('heads,kv_heads,dh', [(1, 1, 8), (2, 2, 128), (8, 8, 64), (4, 1, 256), (6, 3, 32), (3, 1, 24), (2, 1, 40), (2, 2, 96),
                                               (5, 5, 200), (16, 4, 128), (12, 2, 64), (1, 1, 16), (10, 5, 72)])
def test_prompt_heads(K, heads, kv_heads, dh, dtype):
    q, k, v, cu, out = prompt_case(K, [70, 1, 150], heads, kv_heads, dh, dtype, seed=dh)
    check_prompt(q, k, v, cu, out, heads, kv_heads, dh, dtype)


@pytest.mark.parametrize('dh', [4, 12, 20, 252])
def test_prompt_fp32_heads_of_four(K, dh):
    q, k, v, cu, out = prompt_case(K, [70, 1, 150], 2, 1, dh, torch.float32, seed=dh)
    check_prompt(q, k, v, cu, out, 2, 1, dh, torch.float32)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_prompt_rows_outside_stay(K, dtype):
    """Rows before the first and behind the last sequence are neither read nor written; strides wider than the heads."""
    heads, kv_heads, dh = 4, 2, 64
    g = gen(5)
    cu, N = [37, 100, 100, 175], 230
    q, k, v = (torch.randn((N, w * dh + 16), generator=g, device='cuda').to(dtype) for w in (heads, kv_heads, kv_heads))
    for t in (q, k, v):
        t[:37] = math.nan
        t[175:] = math.inf
        t[:, t.shape[1] - 16:] = math.nan
    out = torch.full((N, heads * dh + 32), 7.0, device='cuda', dtype=dtype)
    K.attn_prompt(q[:, :heads * dh], k[:, :kv_heads * dh], v[:, :kv_heads * dh], i32(cu), out[:, :heads * dh], heads, kv_heads)
    assert (out[:37] == 7).all() and (out[175:] == 7).all() and (out[:, heads * dh:] == 7).all()
    check_prompt(q, k, v, cu, out, heads, kv_heads, dh, dtype)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('bad', [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize('at', [0, 5, 63, 64, 100, 149])
def test_prompt_nonfinite_reaches_only_what_attends_to_it(K, dtype, bad, at):
    heads, dh, L = 2, 64, 150
    g = gen(at)
    q, k, v = (torch.randn((2 * L, heads * dh), generator=g, device='cuda').to(dtype) for _ in range(3))
    cu = [0, L, 2 * L]
    v[at, 3] = bad                # first sequence: a value; second: a key
    k[L + at, dh + 3] = bad
    q[L:, dh + 3] = q[L:, dh + 3].abs() + 0.5
    out = torch.empty_like(q)
    K.attn_prompt(q, k, v, i32(cu), out, heads)
    # rows in front of `at` and the untouched heads: as if nothing were there
    for r, h in ((slice(0, at), 0), (slice(0, L), 1), (slice(L, L + at), 1), (slice(L, 2 * L), 0)):
        if r.stop > r.start:
            c = slice(h * dh, (h + 1) * dh)
            want, absv, rel = attend64(q[r, c], k[r, c], v[r, c], dh ** -0.5, True)
            keep = torch.ones(dh, dtype=torch.bool, device='cuda')
            check(out[r, c][:, keep], want, absv, rel, dtype == torch.bfloat16)
    hit = out[at:L, :dh].float()
    assert (torch.isnan(hit[:, 3]) if math.isnan(bad) else hit[:, 3] == bad).all()
    others = torch.ones(dh, dtype=torch.bool, device='cuda')
    others[3] = False
    r, c = slice(0, L), slice(0, dh)
    v2 = v.clone()
    v2[at, 3] = 0
    want, absv, rel = attend64(q[r, c], k[r, c], v2[r, c], dh ** -0.5, True)
    check(out[r, c][:, others], want[:, others], absv[:, others], rel, dtype == torch.bfloat16)
    hit = out[L + at:, dh:].float()
    if bad == -math.inf:          # a key that no row weighs: rows that attend to others too go on without it
        if at > 0:
            r, c = slice(L, 2 * L), slice(dh, 2 * dh)
            ks = torch.cat([k[L:L + at, c], k[L + at + 1:, c]])
            assert torch.isfinite(hit).all() and ks.shape[0] == L - 1
        else:
            assert torch.isnan(hit[0]).all() and torch.isfinite(hit[1:]).all()
    else:
        assert torch.isnan(hit).all()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_prompt_large_scores_and_scale(K, dtype):
    """Scores far apart (one key takes all) and a scale of the caller's."""
    q, k, v, cu, out = prompt_case(K, [200, 33], 2, 1, 64, dtype, seed=9, scale=3.0)
    check_prompt(q, k, v, cu, out, 2, 1, 64, dtype, scale=3.0)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('size', [1.0, 2.0 ** 100])
@pytest.mark.parametrize('growth', [0.25, 1.0, 6.0, -1.0])
@pytest.mark.parametrize('dh', [64, 128, 256])
def test_prompt_scores_that_outgrow_the_first_tiles(K, dh, growth, size, dtype):
    """Scores that rise or fall along the keys by up to thousands of powers of two, on values small and near the top of the range."""
    heads, L = 2, 330
    g = gen(dh)
    q, k, v = (torch.randn((L, heads * dh), generator=g, device='cuda') for _ in range(3))
    for h in range(heads):
        q[:, h * dh] = 1.0
        k[:, h * dh] = torch.arange(L, device='cuda') * growth
    q, k, v = q.to(dtype), k.to(dtype), (v * size).to(dtype)
    out = torch.empty_like(q)
    K.attn_prompt(q, k, v, i32([0, L]), out, heads, scale=1.0)
    check_prompt(q, k, v, [0, L], out, heads, heads, dh, dtype, scale=1.0)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('heads,kv_heads,dh', [(4, 2, 32), (4, 4, 64), (8, 2, 128), (2, 1, 256)])
def test_prompt_short_alone_and_beside_a_long_one(K, heads, kv_heads, dh, dtype):
    """Short prompts among themselves (rows spread differently over the GPU) and in front of a long one: right, and the same bits."""
    short = [20, 33, 1, 0, 64, 7, 100, 32, 65, 2]
    q, k, v, cu, out = prompt_case(K, short + [900], heads, kv_heads, dh, dtype, seed=dh)
    check_prompt(q, k, v, cu, out, heads, kv_heads, dh, dtype)
    n = cu[len(short)]
    alone = torch.empty_like(out[:n])
    K.attn_prompt(q[:n], k[:n], v[:n], i32(cu[:len(short) + 1]), alone, heads, kv_heads)
    assert torch.equal(alone, out[:n])


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('heads,kv_heads,dh', [(8, 4, 32), (8, 8, 24), (8, 2, 64), (16, 4, 128), (8, 1, 72), (8, 1, 256), (12, 2, 128)])
def test_prompt_many_short(K, heads, kv_heads, dh, dtype):
    """Enough short prompts to fill the GPU several times; some longer than a tile, some empty."""
    lens = ([3, 17, 0, 32, 33, 1, 66, 8] * 17)[:130]
    q, k, v, cu, out = prompt_case(K, lens, heads, kv_heads, dh, dtype, seed=dh, before=2, behind=2)
    first = 8
    check_prompt(q, k, v, cu[:first + 1], out, heads, kv_heads, dh, dtype)
    for b in range(first, len(lens), first):                 # the rest against calls of eight at a time: the same bits
        e = min(b + first, len(lens))
        part = out.clone()
        K.attn_prompt(q, k, v, i32(cu[b:e + 1]), part, heads, kv_heads)
        assert torch.equal(part, out)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('B', [3, 150])
@pytest.mark.parametrize('heads,kv_heads,dh', [(8, 2, 64), (8, 8, 128), (8, 2, 128), (4, 1, 256), (8, 8, 32)])
def test_prompt_short_nonfinite_and_steep(K, heads, kv_heads, dh, B, dtype):
    """Short prompts, few and many: an infinity in the middle of one reaches only what attends to it; scores that rise by thousands of
    powers of two, on values near the top of the range."""
    L, w = 41, kv_heads * dh
    g = gen(B)
    q, k, v = (torch.randn((B * L, n), generator=g, device='cuda') for n in (heads * dh, w, w))
    for h in range(heads):
        q[L:2 * L, h * dh] = 1.0
    for h in range(kv_heads):
        k[L:2 * L, h * dh] = torch.arange(L, device='cuda') * 40.0
    v[L:2 * L] *= 2.0 ** 100
    k[20, 3], v[2 * L + 33, 1] = math.inf, math.nan
    q[:L, 3] = q[:L, 3].abs() + 0.5
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    cu = list(range(0, B * L + 1, L))
    out = torch.empty_like(q)
    K.attn_prompt(q, k, v, i32(cu), out, heads, kv_heads, scale=1.0)
    check_prompt(q[:20], k[:20], v[:20], [0, 20], out[:20], heads, kv_heads, dh, dtype, scale=1.0)
    check_prompt(q, k, v, [L, 2 * L], out, heads, kv_heads, dh, dtype, scale=1.0)
    check_prompt(q, k, v, [2 * L, 2 * L + 33], out, heads, kv_heads, dh, dtype, scale=1.0)
    assert torch.isnan(out[20:L, :dh]).all() and torch.isnan(out[2 * L + 33:3 * L, 1]).all()
    if kv_heads > 1:
        last = (heads - 1) * dh
        assert torch.isfinite(out[:L, last:]).all() and torch.isfinite(out[2 * L:3 * L, last:]).all()
    if B > 3:
        check_prompt(q, k, v, [(B - 1) * L, B * L], out, heads, kv_heads, dh, dtype, scale=1.0)


@pytest.mark.parametrize('heads,kv_heads,dh,dtype', [(256, 64, 256, torch.bfloat16), (256, 64, 128, torch.float32), (128, 128, 128, torch.bfloat16),
                                                     (80, 80, 128, torch.float32)])
def test_prompt_short_with_wide_rows(K, heads, kv_heads, dh, dtype):
    """Short prompts whose keys do not fit an L2 together: the other work order."""
    lens, per = [40, 33, 70, 1, 50, 64], heads // kv_heads
    q, k, v, cu, out = prompt_case(K, lens, heads, kv_heads, dh, dtype, seed=heads)
    for h in (0, 1, per - 1, per, heads // 2 + 3, heads - per, heads - 1):
        one, g = slice(h * dh, (h + 1) * dh), slice(h // per * dh, (h // per + 1) * dh)
        check_prompt(q[:, one], k[:, g], v[:, g], cu, out[:, one], 1, 1, dh, dtype)
    assert not (out == 7).all(1).any()


@pytest.mark.parametrize('B', [63, 64, 65, 130, 4097])
def test_prompt_many_sequences(K, B):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 5, (B,), generator=g).tolist()
    lens[0], lens[B // 2], lens[-1] = 3, 40, 2
    q, k, v, cu, out = prompt_case(K, lens, 2, 1, 32, torch.bfloat16, seed=B, behind=3)
    assert (out[cu[-1]:] == 7).all()
    rows = torch.arange(cu[-1], device='cuda')
    start = torch.repeat_interleave(torch.tensor(cu[:-1], device='cuda'), torch.tensor(lens, device='cuda'))
    live = (rows.unsqueeze(0) <= rows.unsqueeze(1)) & (rows.unsqueeze(0) >= start.unsqueeze(1))
    for h in range(2):
        qd, kd, vd = q[:cu[-1], 32 * h:32 * h + 32].double(), k[:cu[-1]].double(), v[:cu[-1]].double()
        s = (qd @ kd.t()) * 32 ** -0.5
        mag = (qd.abs() @ kd.abs().t()) * 32 ** -0.5
        s, mag = s.masked_fill(~live, -math.inf), mag.masked_fill(~live, 0.0)
        w = torch.softmax(s, 1)
        wide = torch.where(w > 1e-12, s.amax(1, keepdim=True) - s, torch.zeros_like(s)).amax(1, keepdim=True)
        rel = 2 * (2 * (32 * 3 + 2) * U32 * mag.amax(1, keepdim=True) + (4 * wide + 4 + 2 * 40) * U32)
        check(out[:cu[-1], 32 * h:32 * h + 32], w @ vd, w @ vd.abs(), rel, True)


def test_prompt_offsets_beyond_32_bits(K):
    buf = torch.empty((33000, 1 << 16), device='cuda', dtype=torch.bfloat16)     # 4.3 GB, 2.16e9 elements
    cu = [32770, 33000]
    g = gen(3)
    for i in range(4):
        buf[cu[0]:, i * 256:i * 256 + 128] = torch.randn((230, 128), generator=g, device='cuda').to(torch.bfloat16)
    q, k, v = (buf[:, i * 256:i * 256 + 128] for i in range(3))
    out = torch.empty((33000, 128), device='cuda', dtype=torch.bfloat16)
    K.attn_prompt(q, k, v, i32(cu), out, 2)
    check_prompt(q, k, v, cu, out, 2, 2, 64, torch.bfloat16)


def test_prompt_same_bits_again_and_in_any_company(K):
    """A sequence's result depends neither on the run nor on what is packed around it (at the same place in the tiles)."""
    q, k, v, cu, out = prompt_case(K, [130, 256, 90], 4, 2, 128, torch.bfloat16, seed=2)
    again = torch.empty_like(out)
    K.attn_prompt(q, k, v, i32(cu), again, 4, 2)
    assert torch.equal(out, again)
    alone = torch.empty_like(out)
    K.attn_prompt(q, k, v, i32([130, 386]), alone, 4, 2)
    assert torch.equal(alone[130:386], out[130:386])


# ---- page tables ----------------------------------------------------------------------------------------------------------------
def plan_plain(lens, room, pages, page, width):
    need = [min(-(-(max(a, 0) + max(b, 0)) // page), width) for a, b in zip(lens, room)]
    table, cu, slots, pos, seq, at = [], [0], [], [], [], 0
    for b, (n, m) in enumerate(zip(lens, need)):
        row = [pages[at + j] if j < m and at + j < len(pages) else -1 for j in range(width)]
        table.append(row)
        for p in range(max(n, 0)):
            pg = row[p // page] if p // page < width else -1
            slots.append(pg * page + p % page if pg >= 0 else -1)
            pos.append(p)
            seq.append(b)
        cu.append(cu[-1] + max(n, 0))
        at += m
    return table, cu, slots, pos, seq, at


@pytest.mark.parametrize('page', [8, 16, 64, 128])
@pytest.mark.parametrize('B,top', [(0, 1), (1, 1), (1, 5000), (3, 0), (64, 90), (65, 200), (1500, 40), (3000, 70)])
def test_page_plan(K, B, top, page):
    g = torch.Generator().manual_seed(B + top + page)
    lens = torch.randint(0, top + 1, (B,), generator=g).tolist()
    room = torch.randint(0, 60, (B,), generator=g).tolist()
    need = [-(-(a + b) // page) for a, b in zip(lens, room)]
    width = max(need, default=0) + 2
    pages = torch.randperm(sum(need) + 5, generator=g).tolist()
    want = plan_plain(lens, room, pages, page, width)
    total = sum(lens)
    out = [torch.full((B, width), 99, dtype=torch.int32, device='cuda'), torch.full((B + 1,), 99, dtype=torch.int32, device='cuda')]
    out += [torch.full((total + 9,), 99, dtype=torch.int32, device='cuda') for _ in range(3)] + [torch.full((1,), 99, dtype=torch.int32, device='cuda')]
    K.page_plan(i32(lens), i32(room), i32(pages), page, *out)
    assert out[0].tolist() == want[0] and out[1].tolist() == want[1] and out[5].tolist() == [want[5]]
    for t, w in zip(out[2:5], want[2:5]):
        assert t[:total].tolist() == w and (t[total:] == 99).all()


def test_page_plan_short_lists_negative_lengths_no_room(K):
    lens, page, width = [10, -3, 40, 0, 25], 8, 4
    pages = list(range(100, 106))
    want = plan_plain(lens, [0] * 5, pages, page, width)
    out = [torch.empty((5, width), dtype=torch.int32, device='cuda'), i32([0] * 6)] + [i32([99] * 60) for _ in range(3)] + [i32([0])]
    K.page_plan(i32(lens), None, i32(pages), page, *out)      # 40 tokens want 5 pages of a 4-wide row; the list runs out
    assert [out[0].tolist(), out[1].tolist(), out[5].item()] == [want[0], want[1], want[5]] and want[5] == 2 + 4 + 4
    assert out[2][:75].tolist() == want[2][:60] and -1 in want[2]
    small = [torch.empty((5, width), dtype=torch.int32, device='cuda'), i32([0] * 6)] + [i32([99] * 20) for _ in range(3)] + [i32([0])]
    K.page_plan(i32(lens), None, i32(pages), page, *small)     # fewer entries than tokens: what fits
    assert small[2].tolist() == want[2][:20] and small[1].tolist() == want[1]


@pytest.mark.parametrize('B', [3, 1030])
def test_page_plan_room_beyond_31_bits(K, B):
    """A length and a room whose sum passes 2^31: as many pages as the table is wide."""
    top = 2 ** 31 - 1
    lens, room, width, page = [5, 40, 0] + [1] * (B - 3), [top, top, top] + [0] * (B - 3), 4, 32
    pages = list(range(100, 100 + 3 * width + B))
    table, cu, slots, pos, seq, used = (torch.empty(s, dtype=torch.int32, device='cuda') for s in ((B, width), B + 1, sum(lens), sum(lens), sum(lens), 1))
    K.page_plan(i32(lens), i32(room), i32(pages), page, table, cu, slots, pos, seq, used)
    want = [pages[width * b:width * b + width] for b in range(3)] + [[pages[3 * width + b], -1, -1, -1] for b in range(B - 3)]
    assert table.tolist() == want and used.item() == 3 * width + B - 3
    assert slots.tolist()[:45] == [pages[0] * page + i for i in range(5)] + [pages[width + i // page] * page + i % page for i in range(40)]


def test_page_step(K):
    table = i32([[5, 9, -1], [7, -1, -1], [2, 3, 4]])
    base, sent = i32([14, 16, 0]), i32([2, 0, 1, 9, -1, 0])
    slots, pos, lens = (i32([99] * 8) for _ in range(3))
    K.page_step(base, sent, 3, table, 16, slots, pos, lens, 6)
    assert pos.tolist() == [3, 17, 19, 0, 0, 17, 99, 99] and lens.tolist() == [4, 18, 20, 0, 0, 18, 99, 99]
    assert slots.tolist() == [35, 145, -1, -1, -1, 145, 99, 99]
    K.page_step(base, None, 40, table, 16, slots, pos, lens, 3)
    assert pos.tolist()[:3] == [54, 56, 40] and slots.tolist()[:3] == [-1, -1, 72]


# ---- the 4-bit cache -------------------------------------------------------------------------------------------------------------
GRID = [0, .5, 1, 1.5, 2, 3, 4, 6]


def quantise64(x):
    """The values that rows x [..., 32 * n] stand for after storing, by the definition, in 64 bits."""
    y = x.double().reshape(-1, 32)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    top = y.abs().amax(1, keepdim=True)
    unit = torch.full_like(top, 2.0 ** -126)
    for e in range(-125, 127):
        unit = torch.where(top > 6 * unit, torch.full_like(top, 2.0 ** e), unit)
    dist = (y.abs().unsqueeze(-1) / unit.unsqueeze(-1) - grid).abs()
    key = torch.where(dist == dist.amin(-1, keepdim=True), torch.arange(8, device=x.device) & 1, 2)
    out = grid[key.argmin(-1)] * unit * torch.sign(y)
    return torch.where(torch.isfinite(y).all(1, keepdim=True), out, torch.full_like(out, math.nan)).reshape(x.shape)


def same(a, b):
    a, b = a.double(), b.double()
    return torch.equal(torch.nan_to_num(a, nan=1e300), torch.nan_to_num(b, nan=1e300))


def rows_of(kind, n, w, g):
    x = torch.randn((n, w), generator=g, device='cuda')
    if kind == 'wide':       # every power of two, ties among them: multiples of a quarter of the unit
        x = torch.round(x * 8) / 4 * torch.exp2(torch.randint(-130, 120, (n, w // 32), generator=g, device='cuda').float()).repeat_interleave(32, 1)
    if kind == 'odd':
        x[torch.rand((n, w), generator=g, device='cuda') < 0.5] = 0
        x[0] = 0
        x[-1, 5] = math.nan
        x[-1, w - 1] = -math.inf
        x[n // 2, :32] = 3e38
        x[n // 3, :32] = 1e-42
    return x


@pytest.mark.parametrize('kind', ['normal', 'wide', 'odd'])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('n,kv_heads,dh,page', [(1, 1, 32, 16), (100, 8, 64, 32), (130, 3, 128, 64), (70, 2, 256, 128), (64, 5, 32, 128), (257, 1, 64, 16)])
def test_cache_store_and_read(K, n, kv_heads, dh, page, dtype, kind):
    g = gen(n + dh)
    w = kv_heads * dh
    kv = torch.cat([rows_of(kind, n, w, g), rows_of(kind, n, w, g)], 1).to(dtype)
    pages = -(-n // page) + 2
    slots = torch.randperm(pages * page, generator=g, device='cuda')[:n].to(torch.int32)
    slots[n // 2] = -1 if n > 1 else slots[0]
    cache = K.Cache4(pages, page, kv_heads, dh)
    K.cache4_write(cache, kv[:, :w], kv[:, w:], slots, n)
    back = torch.full((n + 2, 2 * w), 7.0, device='cuda', dtype=dtype)
    K.cache4_read(cache, slots, back[:, :w], back[:, w:], n)
    want = quantise64(kv)
    if n > 1:
        want[n // 2] = 0
    if dtype == torch.bfloat16:
        want = want.to(dtype)
    else:
        want = want.float()
    assert same(back[:n], want) and (back[n:] == 7).all()
    # the documented layout, byte by byte, for one token
    i = 0
    s = int(slots[i])
    t, p = s % page, s // page
    codes = cache.kc[p, :, t].int()
    unit = torch.where(cache.ks[p, :, t] == 255, math.nan, torch.exp2(cache.ks[p, :, t].double() - 127)).repeat_interleave(32, 1)
    sign = torch.tensor([1.0] * 8 + [-1.0] * 8, dtype=torch.float64, device='cuda')
    grid = torch.tensor(GRID * 2, dtype=torch.float64, device='cuda') * sign
    vals = torch.stack((grid[(codes & 15).long()], grid[(codes >> 4).long()]), -1).reshape(kv_heads, dh) * unit
    assert same(vals.reshape(-1).to(dtype), want[i, :w])
    codes = cache.vc[p, :, :, t].int()
    unit = torch.where(cache.vs[p, :, :, t] == 255, math.nan, torch.exp2(cache.vs[p, :, :, t].double() - 127)).repeat_interleave(32, 1)
    vals = torch.stack((grid[(codes & 15).long()], grid[(codes >> 4).long()]), -1).reshape(kv_heads, dh) * unit
    assert same(vals.reshape(-1).to(dtype), want[i, w:])


def test_cache_write_leaves_the_rest(K):
    cache = K.Cache4(6, 32, 2, 64)
    for t in (cache.kc, cache.ks, cache.vc, cache.vs):
        t.random_(0, 200, generator=gen(1))
    before = [t.clone() for t in (cache.kc, cache.ks, cache.vc, cache.vs)]
    kv = torch.randn((5, 256), generator=gen(2), device='cuda')
    slots = i32([33, 100, -1, 6 * 32, 2 ** 31 - 1])
    K.cache4_write(cache, kv[:, :128], kv[:, 128:], slots, 5)
    for s in (33, 100):
        p, t = divmod(s, 32)
        for a, b, ax in zip((cache.kc, cache.ks, cache.vc, cache.vs), before, (2, 2, 3, 3)):
            a.select(ax, t)[p].copy_(b.select(ax, t)[p])
    for a, b in zip((cache.kc, cache.ks, cache.vc, cache.vs), before):
        assert torch.equal(a, b)


def filled_cache(K, lens, kv_heads, dh, page, seed, width=None):
    """A cache whose sequences (shuffled pages) hold random rows; the values they stand for, per sequence, in 64 bits."""
    g = gen(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(max(need, default=0), 1) if width is None else width
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    cache = K.Cache4(pages, page, kv_heads, dh)
    for t in (cache.kc, cache.vc):
        t.random_(0, 256, generator=g)
    for t in (cache.ks, cache.vs):                       # what no sequence holds: anything, NaN scales among it
        t.random_(100, 256, generator=g)
        t[t > 140] = 255
    w, at, vals = kv_heads * dh, 0, []
    for b, n in enumerate(lens):
        table[b, :need[b]] = torch.tensor(perm[at:at + need[b]], dtype=torch.int32)
        at += need[b]
        kv = torch.randn((n, 2 * w), generator=g, device='cuda')
        kv[:, w:] *= 2
        p = torch.arange(n)
        slots = (table[b, p // page].long() * page + p % page).to(torch.int32).cuda()
        K.cache4_write(cache, kv[:, :w], kv[:, w:], slots, n)
        vals.append(quantise64(kv))
    return cache, table.cuda(), vals


def check_attend(q, vals, lens, out, heads, kv_heads, dh, dtype, seq=None, scale=None):
    per, w = heads // kv_heads, kv_heads * dh
    for r in range(q.shape[0]):
        s = r if seq is None else seq[r]
        n = lens[r]
        if n <= 0:
            assert (out[r] == 0).all()
            continue
        for h in range(heads):
            g = h // per
            want, absv, rel = attend64(q[r:r + 1, h * dh:(h + 1) * dh], vals[s][:n, g * dh:(g + 1) * dh],
                                       vals[s][:n, w + g * dh:w + (g + 1) * dh], dh ** -0.5 if scale is None else scale, False)
            check(out[r:r + 1, h * dh:(h + 1) * dh], want, absv, rel, dtype == torch.bfloat16)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('page', [16, 32, 64, 128])
@pytest.mark.parametrize('heads,kv_heads,dh', [(1, 1, 32), (8, 8, 64), (16, 4, 128), (4, 1, 256), (16, 1, 128), (40, 2, 64), (34, 2, 32)])
def test_attend_lengths(K, heads, kv_heads, dh, page, dtype):
    lens = [0, 1, 15, 16, 17, 63, 64, 65, 128, 129, 200, 1000]
    cache, table, vals = filled_cache(K, lens, kv_heads, dh, page, seed=dh + page)
    q = torch.randn((len(lens), heads * dh), generator=gen(1), device='cuda').to(dtype)
    out = torch.full_like(q, 7.0)
    K.attn_cache4(q, cache, table, i32(lens), out, len(lens), heads, 1000)
    check_attend(q, vals, lens, out, heads, kv_heads, dh, dtype)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('rows,length', [(1, 70000), (2, 5000), (3, 1023)])
def test_attend_long(K, rows, length, dtype):
    lens = [length - 37 * i for i in range(rows)]
    cache, table, vals = filled_cache(K, lens, 2, 128, 64, seed=length)
    q = torch.randn((rows, 4 * 128), generator=gen(2), device='cuda').to(dtype)
    out = torch.empty_like(q)
    K.attn_cache4(q, cache, table, i32(lens), out, rows, 4, length)
    check_attend(q, vals, lens, out, 4, 2, 128, dtype)
    again = torch.empty_like(q)
    K.attn_cache4(q, cache, table, i32(lens), again, rows, 4, length)
    assert torch.equal(out, again)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_attend_rows_of_shared_sequences_strides_scale(K, dtype):
    """Several rows of one sequence at different lengths, rows of none, wider strides, rows behind the last left alone."""
    cache, table, vals = filled_cache(K, [300, 90], 2, 64, 32, seed=4, width=12)
    seq, lens = [1, 0, 0, 1, 5, -1, 0], [90, 300, 7, 1, 50, 50, 0]
    g = gen(6)
    q = torch.randn((9, 4 * 64 + 8), generator=g, device='cuda').to(dtype)
    out = torch.full((9, 4 * 64 + 16), 7.0, device='cuda', dtype=dtype)
    K.attn_cache4(q[:, :256], cache, table, i32(lens), out[:, :256], 7, 4, 300, seq=i32(seq), scale=0.3)
    eff = [n if 0 <= s < 2 else 0 for n, s in zip(lens, seq)]
    check_attend(q[:7, :256], vals, eff, out[:, :256], 4, 2, 64, dtype, seq=seq, scale=0.3)
    assert (out[7:] == 7).all() and (out[:, 256:] == 7).all()


def test_attend_cut_lengths_and_bad_pages(K):
    """Lengths beyond max_len or the table are cut; pages outside the cache count as nothing."""
    cache, table, vals = filled_cache(K, [200, 200, 200], 1, 64, 32, seed=8)
    q = torch.randn((3, 128), generator=gen(7), device='cuda')
    out = torch.empty_like(q)
    K.attn_cache4(q, cache, table, i32([10 ** 9, 200, 150]), out, 3, 2, 150)
    check_attend(q, vals, [150, 150, 150], out, 2, 1, 64, torch.float32)
    K.attn_cache4(q, cache, table[:, :4].contiguous(), i32([200] * 3), out, 3, 2, 200)
    check_attend(q, vals, [128] * 3, out, 2, 1, 64, torch.float32)
    bad = table.clone()
    bad[0, 1], bad[1, 0], bad[2] = -7, cache.pages, 2 ** 31 - 1
    K.attn_cache4(q, cache, bad, i32([200] * 3), out, 3, 2, 200)
    cut = [torch.cat([vals[0][:32], vals[0][64:]]), vals[1][32:], vals[2]]
    check_attend(q, cut, [168, 168, 0], out, 2, 1, 64, torch.float32)


def test_attend_nonfinite_in_and_out_of_reach(K):
    """A NaN group inside the length reaches its elements; behind the length it reaches nothing (filled_cache puts NaN scales there)."""
    for dtype in (torch.bfloat16, torch.float32):
        cache, table, vals = filled_cache(K, [70, 70, 70], 1, 64, 32, seed=9)
        kv = torch.zeros((2, 128), device='cuda')
        kv[0, 64 + 40] = math.nan               # value elements 32..63 of token 40 of sequence 0
        kv[1, 3] = math.inf                     # keys 0..31 of token 40 of sequence 1
        slots = (table[:2, 1] * 32 + 8).contiguous()
        K.cache4_write(cache, kv[:, :64], kv[:, 64:], slots, 2)
        q = torch.randn((3, 64), generator=gen(3), device='cuda').to(dtype)
        out = torch.empty_like(q)
        K.attn_cache4(q, cache, table, i32([70, 70, 70]), out, 3, 1, 70)
        assert torch.isnan(out[0, 32:]).all() and torch.isfinite(out[0, :32]).all() and torch.isnan(out[1]).all()
        check_attend(q[2:], vals[2:], [70], out[2:], 1, 1, 64, dtype)
        K.attn_cache4(q, cache, table, i32([40, 40, 40]), out, 3, 1, 70)
        check_attend(q, vals, [40] * 3, out, 1, 1, 64, dtype)


def test_cache_offsets_beyond_32_bits(K):
    pages, page, kv_heads, dh = 33100, 128, 8, 256            # kc and vc of 4.3 GB each
    cache = K.Cache4(pages, page, kv_heads, dh)
    n = 300
    table = i32([[pages - 1, 0, pages - 2], [pages - 3, 32800, 1]])
    g = gen(1)
    vals = []
    for b in range(2):
        kv = torch.randn((n, 2 * kv_heads * dh), generator=g, device='cuda')
        p = torch.arange(n, device='cuda')
        slots = (table[b].long()[p // page] * page + p % page).to(torch.int32)
        K.cache4_write(cache, kv[:, :kv_heads * dh], kv[:, kv_heads * dh:], slots, n)
        back = torch.empty_like(kv)
        K.cache4_read(cache, slots, back[:, :kv_heads * dh], back[:, kv_heads * dh:], n)
        vals.append(quantise64(kv))
        assert same(back, vals[-1].float())
    q = torch.randn((2, kv_heads * dh), generator=g, device='cuda').to(torch.bfloat16)
    out = torch.empty_like(q)
    K.attn_cache4(q, cache, table, i32([n, n - 1]), out, 2, kv_heads, n)
    check_attend(q, vals, [n, n - 1], out, kv_heads, kv_heads, dh, torch.bfloat16)


def test_attend_captured_graphs_with_their_own_work(K):
    """Two captured calls and an eager one, replayed with eager work between, give the eager bits each time."""
    cache, table, vals = filled_cache(K, [3000, 2500], 2, 64, 64, seed=12)
    qs = [torch.randn((2, 256), generator=gen(i), device='cuda').to(torch.bfloat16) for i in range(2)]
    lens = i32([3000, 2500])
    want, graphs, outs = [], [], []
    side = torch.cuda.Stream()
    for q in qs:
        o = torch.empty_like(q)
        K.attn_cache4(q, cache, table, lens, o, 2, 4, 3000)
        want.append(o)
        work = K.attn_cache4_work(2, 4, 2, 64, 3000)
        out = torch.zeros_like(q)
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            K.attn_cache4(q, cache, table, lens, out, 2, 4, 3000, work=work)
            with torch.cuda.graph(graph, stream=side):
                K.attn_cache4(q, cache, table, lens, out, 2, 4, 3000, work=work)
        torch.cuda.current_stream().wait_stream(side)
        graphs.append((graph, work))
        outs.append(out)
    for _ in range(3):
        for out in outs:
            out.zero_()
        for graph, _w in graphs:
            graph.replay()
        eager = torch.empty_like(qs[0])
        K.attn_cache4(qs[0], cache, table, lens, eager, 2, 4, 3000)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0]) and all(torch.equal(a, b) for a, b in zip(outs, want))


# ---- rules on logits --------------------------------------------------------------------------------------------------------------
def rules_plain(x, V, params, hist, hist_len, prompt, cu, sent, bias, bias_row, mask, mask_row):
    """fp32 arithmetic in the documented order, row by row."""
    y = x.float().cpu().clone()
    for r in range(y.shape[0]):
        s = r if sent is None else sent[r]
        if params is not None and 0 <= s < len(params):
            rp, fp, pp = params[s]
            gen_toks = [] if hist is None else [t for t in hist[r][:min(hist_len[r], len(hist[r])) if hist_len is not None else len(hist[r])] if 0 <= t < V]
            old = [] if prompt is None else [t for t in prompt[max(cu[s], 0):cu[s + 1]] if 0 <= t < V]
            for t in set(gen_toks) | set(old):
                y[r, t] = y[r, t] / rp if y[r, t] > 0 else y[r, t] * rp
            for t in set(gen_toks):
                y[r, t] = (y[r, t] - torch.tensor(float(gen_toks.count(t))) * fp) - pp
        b = -1 if bias is None else (0 if bias_row is None else bias_row[r])
        if bias is not None and 0 <= b < len(bias):
            y[r] = y[r] + bias[b, :V]
        m = -1 if mask is None else (0 if mask_row is None else mask_row[r])
        if mask is not None and 0 <= m < len(mask):
            ok = ((mask[m].unsqueeze(1) >> torch.arange(32, dtype=torch.int32)) & 1).flatten()[:V].bool()
            y[r, ~ok] = -math.inf
    return y


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('V,ld', [(1, 1), (31, 40), (33, 33), (100, 104), (997, 1000), (8192, 8192), (8193, 8200), (20001, 20001)])
@pytest.mark.parametrize('parts', ['all', 'penalties', 'bias', 'mask', 'none', 'sent'])
@pytest.mark.parametrize('inplace', [False, True])
def test_logit_rules(K, V, ld, parts, dtype, inplace):
    R = 7
    g = torch.Generator().manual_seed(V + len(parts))
    x = torch.randn((R, ld), generator=g).mul(3).to(dtype)
    x[0, 0], x[1, V - 1], x[2, V // 2] = math.inf, -math.inf, math.nan
    x[3, :V // 2 + 1] = 0
    use = lambda *names: parts == 'all' or parts in names       # noqa: E731
    params = hist = hist_len = prompt = cu = sent = bias = bias_row = mask = mask_row = None
    if use('penalties', 'sent'):
        n = 3 if parts == 'sent' else R
        params = torch.rand((n, 3), generator=g) + 0.5
        hist = torch.randint(-1, min(V, 60) + 1, (R, 50), generator=g, dtype=torch.int32)
        hist_len = torch.tensor([0, 50, 1, 20, 99, -4, 33], dtype=torch.int32)
        cu = torch.tensor([0] + torch.randint(0, 30, (n,), generator=g).cumsum(0).tolist(), dtype=torch.int32)
        prompt = torch.randint(-2, V + 2, (int(cu[-1]) + 4,), generator=g, dtype=torch.int32)
        prompt[:3] = V - 1
        if parts == 'sent':
            sent = torch.tensor([2, 0, 0, 1, 3, -1, 2], dtype=torch.int32)
            hist_len = None
    if use('bias'):
        bias = torch.randn((2, ld), generator=g)
        bias_row = torch.tensor([0, 1, -1, 1, 2, 0, 0], dtype=torch.int32) if parts == 'all' else None
    if use('mask'):
        mask = torch.randint(-2 ** 31, 2 ** 31, (3, (V + 31) // 32), generator=g).to(torch.int32)
        mask[1] = 0
        mask_row = torch.tensor([2, 1, -1, 0, 3, 2, 0], dtype=torch.int32)
    dev = lambda t: None if t is None else t.cuda()       # noqa: E731
    logits = dev(x).clone()
    out = logits if inplace else torch.full((R + 1, ld), 7.0, device='cuda', dtype=dtype)
    K.adjust_logits(logits, R, V, out, params=dev(params), sent=dev(sent), hist=dev(hist), hist_len=dev(hist_len), prompt=dev(prompt),
                    prompt_cu=dev(cu), bias=dev(bias), bias_row=dev(bias_row), mask=dev(mask), mask_row=dev(mask_row))
    want = rules_plain(x[:, :V], V, params, None if hist is None else hist.tolist(), None if hist_len is None else [max(0, i) for i in hist_len.tolist()],
                       None if prompt is None else prompt.tolist(), None if cu is None else cu.tolist(), None if sent is None else sent.tolist(), bias,
                       None if bias_row is None else bias_row.tolist(), mask, None if mask_row is None else mask_row.tolist()).to(dtype)
    assert same(out[:R, :V].cpu(), want)
    if inplace:
        assert same(out[:, V:].cpu(), x[:, V:])
    else:
        assert (out[R:] == 7).all() and (out[:, V:] == 7).all() and same(logits.cpu(), x)


def test_logit_rules_many_rows(K):
    """More rows than one grid holds."""
    R, V = 70001, 40
    x = torch.randn((R, V), generator=gen(1), device='cuda')
    hist = torch.randint(0, V, (R, 3), generator=gen(2), device='cuda', dtype=torch.int32)
    params = torch.rand((R, 3), generator=gen(3), device='cuda') + 1
    out = torch.empty_like(x)
    K.adjust_logits(x, R, V, out, params=params, hist=hist)
    c = torch.zeros_like(x).scatter_add_(1, hist.long(), torch.ones((R, 3), device='cuda'))
    y = torch.where(c > 0, torch.where(x > 0, x / params[:, :1], x * params[:, :1]), x)
    y = torch.where(c > 0, (y - c * params[:, 1:2]) - params[:, 2:3], y)
    assert torch.equal(out, y)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('R,n_hist', [(513, 9000), (300, 2500), (40, 9000), (520, 2049)])
def test_logit_rules_long_histories(K, R, n_hist, dtype):
    """Histories with more different tokens than a chunk's list holds, and just about as many."""
    V = 9001
    x = torch.randn((R, V), generator=gen(1), device='cuda').to(dtype)
    hist = torch.randint(0, V, (R, n_hist), generator=gen(2), device='cuda', dtype=torch.int32)
    hist[0] = torch.arange(n_hist, device='cuda', dtype=torch.int32) % V
    hist[1] = 5
    params = torch.rand((R, 3), generator=gen(3), device='cuda') + 1
    out = torch.empty_like(x)
    K.adjust_logits(x, R, V, out, params=params, hist=hist)
    c = torch.zeros((R, V), device='cuda').scatter_add_(1, hist.long(), torch.ones((R, n_hist), device='cuda'))
    f = x.float()
    y = torch.where(c > 0, torch.where(f > 0, f / params[:, :1], f * params[:, :1]), f)
    y = torch.where(c > 0, (y - c * params[:, 1:2]) - params[:, 2:3], y).to(dtype)
    assert torch.equal(out, y)


def test_grammar_next(K):
    table = i32([[1, -1, 2], [0, 2, 2], [-1, -1, -1]])
    state = i32([0, 1, 2, -1])
    out = i32([9] * 6)
    K.grammar_next(table, state, i32([1, 1, 0, 3, 7]), i32([2, 0, 5, 0, 0]), out, 5)
    assert out.tolist() == [2, 0, -1, -1, -1, 9]
    K.grammar_next(table, state, None, i32([2, 1, 0, 0]), out, 4)
    assert out.tolist()[:4] == [2, 2, -1, -1]


# ---- the operators in a row -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_prefill_then_steps(K, dtype):
    """Plan, prompt attention, store, then single tokens over the cache on a side stream: as a server would run them."""
    heads, kv_heads, dh, page, steps = 4, 2, 64, 32, 5
    lens = [40, 1, 0, 97, 32]
    B, w = len(lens), kv_heads * dh
    g = gen(33)
    total = sum(lens)
    room = i32([steps] * B)
    need = sum(-(-(n + steps) // page) for n in lens)
    width = max(-(-(n + steps) // page) for n in lens)
    table = torch.empty((B, width), dtype=torch.int32, device='cuda')
    cu, slots, pos, seq, used = (torch.empty(n, dtype=torch.int32, device='cuda') for n in (B + 1, total, total, total, 1))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    qkv = torch.randn((total, (heads + 2 * kv_heads) * dh), generator=g, device='cuda').to(dtype)
    new = torch.randn((steps, B, (heads + 2 * kv_heads) * dh), generator=g, device='cuda').to(dtype)
    a, b = heads * dh, heads * dh + w
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        K.page_plan(i32(lens), room, torch.randperm(need, device='cuda').to(torch.int32), page, table, cu, slots, pos, seq, used)
        out = torch.empty((total, a), device='cuda', dtype=dtype)
        K.attn_prompt(qkv[:, :a], qkv[:, a:b], qkv[:, b:], cu, out, heads, kv_heads)
        cache = K.Cache4(need, page, kv_heads, dh)
        K.cache4_write(cache, qkv[:, a:b], qkv[:, b:], slots, total)
        res = torch.empty((steps, B, a), device='cuda', dtype=dtype)
        s1, p1, l1 = (torch.empty(B, dtype=torch.int32, device='cuda') for _ in range(3))
        work = K.attn_cache4_work(B, heads, kv_heads, dh, max(lens) + steps)
        for t in range(steps):
            K.page_step(i32(lens), None, t, table, page, s1, p1, l1, B)
            K.cache4_write(cache, new[t, :, a:b], new[t, :, b:], s1, B)
            K.attn_cache4(new[t, :, :a], cache, table, l1, res[t], B, heads, max(lens) + steps, work=work)
    torch.cuda.current_stream().wait_stream(side)
    assert used.item() == need
    check_prompt(qkv[:, :a], qkv[:, a:b], qkv[:, b:], cu.tolist(), out, heads, kv_heads, dh, dtype)
    at = cu.tolist()
    for t in range(steps):
        vals = [quantise64(torch.cat([qkv[at[i]:at[i + 1], a:], new[:t + 1, i, a:]])) for i in range(B)]
        check_attend(new[t, :, :a], vals, [n + t + 1 for n in lens], res[t], heads, kv_heads, dh, dtype)


# ---- all of them together --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_a_step_of_all_operators_captured_and_replayed(K, dtype):
    """Plan, prompt attention, cache, one decode step, rules and grammar in one graph on a stream of its own: replays over new inputs, with
    eager work between them, give the bits of eager calls."""
    heads, kv_heads, dh, page, V, B, states = 4, 2, 64, 32, 1003, 5, 4
    wq, wk = heads * dh, kv_heads * dh
    width, N = 8, 700

    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        lens = torch.randint(0, 140, (B,), generator=g)
        lens[seed % B] = 0
        d = dict(lens=lens.int(), room=torch.full((B,), 3, dtype=torch.int32), pages=torch.randperm(B * width, generator=g).int(),
                 qkv=torch.randn((N, wq + 2 * wk), generator=g).to(dtype), step=torch.randn((B, wq + 2 * wk), generator=g).to(dtype),
                 logits=torch.randn((B, V), generator=g).to(dtype), hist=torch.randint(0, V, (B, 9), generator=g).int(),
                 params=torch.rand((B, 3), generator=g) + 0.5, bias=torch.randn((1, V), generator=g),
                 mask=torch.randint(-2 ** 31, 2 ** 31 - 1, (states, (V + 31) // 32), generator=g).int(),
                 state=torch.randint(0, states, (B,), generator=g).int(), tok=torch.randint(0, V, (B,), generator=g).int(),
                 next=torch.randint(-1, states, (states, V), generator=g).int())
        return {k: v.cuda() for k, v in d.items()}

    def buffers():
        z = lambda *s, t=torch.int32: torch.zeros(s, dtype=t, device='cuda')       # noqa: E731
        return dict(table=z(B, width), cu=z(B + 1), slots=z(N), pos=z(N), seq=z(N), used=z(1), out=z(N, wq, t=dtype), s_slots=z(B), s_pos=z(B),
                    s_lens=z(B), att=z(B, wq, t=dtype), y=z(B, V, t=dtype), after=z(B), cache=K.Cache4(B * width, page, kv_heads, dh),
                    work=K.attn_cache4_work(B, heads, kv_heads, dh, width * page, 'cuda'))

    def run(i, b):
        K.page_plan(i['lens'], i['room'], i['pages'], page, b['table'], b['cu'], b['slots'], b['pos'], b['seq'], b['used'])
        q, k, v = i['qkv'][:, :wq], i['qkv'][:, wq:wq + wk], i['qkv'][:, wq + wk:]
        K.attn_prompt(q, k, v, b['cu'], b['out'], heads, kv_heads)
        K.cache4_write(b['cache'], k, v, b['slots'], N)
        K.page_step(i['lens'], None, 0, b['table'], page, b['s_slots'], b['s_pos'], b['s_lens'], B)
        K.cache4_write(b['cache'], i['step'][:, wq:wq + wk], i['step'][:, wq + wk:], b['s_slots'], B)
        K.attn_cache4(i['step'][:, :wq], b['cache'], b['table'], b['s_lens'], b['att'], B, heads, width * page, work=b['work'])
        K.adjust_logits(i['logits'], B, V, b['y'], params=i['params'], hist=i['hist'], bias=i['bias'], mask=i['mask'], mask_row=i['state'])
        K.grammar_next(i['next'], i['state'], None, i['tok'], b['after'], B)

    fixed, mine = inputs(0), buffers()
    mine['slots'].fill_(-1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(fixed, mine)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run(fixed, mine)
    names = ('table', 'cu', 'used', 's_slots', 's_pos', 's_lens', 'att', 'y', 'after')
    for seed in (3, 1, 2, 3):
        new, plain = inputs(seed), buffers()
        plain['slots'].fill_(-1)
        run(new, plain)
        mine['slots'].fill_(-1)                          # entries behind the last token stay as they are: no slot
        for k in fixed:
            fixed[k].copy_(new[k])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        n = int(plain['cu'][-1])
        for k in names:
            assert torch.equal(mine[k], plain[k]), (seed, k)
        for k in ('slots', 'pos', 'seq', 'out'):
            assert torch.equal(mine[k][:n], plain[k][:n]), (seed, k)
        assert n == int(new['lens'].sum()) and not torch.isnan(mine['att'].float()).any()


# ---- what the wrappers refuse (nothing is launched) -----------------------------------------------------------------------------------
def test_wrappers_refuse(K):
    from tst_amd import TstError
    z = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device='cuda')            # noqa: E731
    iz = lambda *s: z(*s, t=torch.int32)                                               # noqa: E731
    rows = z(8, 256)

    def each(call, ok, bad):
        call(**ok)
        for name, value, kind, why in bad:
            with pytest.raises(kind, match=why):
                call(**dict(ok, **{name: value}))

    shifted = z(8 * 128 + 4)[1:8 * 128 + 1].view(8, 128)                               # rows off their 16-byte boundaries
    for t in (torch.float32, torch.bfloat16):
        r = z(8, 512, t=t)
        other = torch.bfloat16 if t is torch.float32 else torch.float32
        each(K.attn_prompt, dict(q=r[:, :128], k=r[:, 128:192], v=r[:, 192:256], cu=iz(2), out=z(8, 128, t=t), heads=2, kv_heads=1), [
            ('q', z(8, 128, t=torch.float16), ValueError, 'q must be fp32 or bf16'), ('k', z(8, 64, t=other), ValueError, 'k must be a 2-D'),
            ('q', torch.zeros(8, 128, dtype=t), ValueError, 'on the current GPU'), ('q', z(8, 130, t=t), ValueError, 'not a multiple'),
            ('q', z(8, 2, 64, t=t), ValueError, 'q must be'), ('v', z(7, 64, t=t), ValueError, 'v must hold'), ('k', z(8, 56, t=t), ValueError, 'k must hold'),
            ('k', z(64, 8, t=t).t(), ValueError, 'inner stride'), ('k', z(1, 64, t=t).expand(8, 64), ValueError, 'overlap'),
            ('k', z(8, 66, t=t)[:, :64], ValueError, '16 bytes'), ('out', r[:, :128], ValueError, 'out must not overlap'),
            ('out', r[:, 64:192], ValueError, 'out must not overlap'), ('cu', iz(2).long(), ValueError, 'cu must be'), ('cu', None, TypeError, 'cu must be a tensor'),
            ('cu', iz(4)[::2], ValueError, 'cu must be'), ('cu', iz(0), ValueError, 'cu must be'), ('heads', 3, ValueError, 'heads'), ('heads', 0, ValueError, 'heads'),
            ('kv_heads', 0, ValueError, 'heads'), ('heads', 1.5, TypeError, 'heads must be an integer'), ('q', None, TypeError, 'q must be a tensor'),
            ('q', [1], TypeError, 'q must be a tensor'), ('scale', math.nan, TstError, 'not finite'), ('scale', 'x', TypeError, 'real number|float')])
    with pytest.raises(ValueError, match='16-byte'):
        K.attn_prompt(shifted, rows[:, :128], rows[:, 128:], iz(2), z(8, 128), 1)
    plan = dict(lens=iz(3), room=None, pages=iz(5), page=32, table=iz(3, 4), cu=iz(4), slots=iz(9), pos=iz(9), seq=iz(9), used=iz(1))
    each(K.page_plan, plan, [
        ('lens', None, TypeError, 'lens'), ('lens', iz(3, 1), ValueError, 'lens must be'), ('room', iz(2), ValueError, 'room must be'), ('pages', None, TypeError, 'pages'),
        ('page', 24, TstError, 'power of two'), ('page', 'a', TypeError, 'page must be an integer'), ('table', iz(2, 4), ValueError, 'table must be'),
        ('table', iz(3, 8)[:, :4], ValueError, 'table must be'), ('cu', iz(3), ValueError, 'cu must be'), ('pos', iz(8), ValueError, 'pos must be'),
        ('seq', z(9), ValueError, 'seq must be'), ('used', iz(0), ValueError, 'used must be'), ('used', None, TstError, 'null pointer'), ('slots', None, TypeError, 'slots')])
    each(K.page_step, dict(base=iz(3), sent=None, t=0, table=iz(3, 4), page=32, slots=iz(3), pos=iz(3), lens=iz(3), n_rows=3), [
        ('base', iz(2), ValueError, 'base must be'), ('sent', iz(2), ValueError, 'sent must be'), ('lens', iz(2), ValueError, 'lens must be'),
        ('n_rows', -1, TstError, 'negative'), ('t', None, TypeError, 't must be an integer'), ('table', iz(3), ValueError, 'table must be'),
        ('n_rows', 1 << 70, TypeError, 'integer')])
    cache = K.Cache4(3, 32, 2, 64)
    no = iz(8) - 1
    each(K.cache4_write, dict(cache=cache, k=rows[:, :128], v=rows[:, 128:], slots=no, n_rows=8), [
        ('k', z(8, 120), ValueError, 'k must hold'), ('v', z(8, 128, t=torch.bfloat16), ValueError, 'v must be a 2-D'), ('slots', no[:7], ValueError, 'slots must be'),
        ('n_rows', 9, ValueError, 'must hold'), ('k', z(8, 128).double(), ValueError, 'rows must be fp32 or bf16'), ('slots', None, TstError, 'null pointer')])
    each(K.cache4_read, dict(cache=cache, k=z(8, 128), v=z(8, 128), slots=no, n_rows=8), [
        ('k', z(8, 120), ValueError, 'k must hold'), ('slots', no.long(), ValueError, 'slots must be'), ('v', shifted, ValueError, '16-byte')])
    cache.dev += 1                                                                     # as if it were on another device
    for call, a in ((K.cache4_write, (rows[:, :128], rows[:, 128:], no, 8)), (K.cache4_read, (no, rows[:, :128], rows[:, 128:], 8))):
        with pytest.raises(ValueError, match='the current device is'):
            call(cache, *a)
    cache.dev -= 1
    each(K.attn_cache4, dict(q=rows, cache=cache, table=iz(8, 3), lens=iz(8), out=z(8, 256), n_rows=8, heads=4, max_len=96), [
        ('heads', 3, ValueError, 'multiple of the cache'), ('q', rows[:, :248], ValueError, 'q must hold'), ('out', rows, ValueError, 'overlap'),
        ('table', iz(8), ValueError, 'table must be'), ('seq', iz(7), ValueError, 'seq must be'), ('lens', iz(7), ValueError, 'lens must be'),
        ('lens', None, TstError, 'null pointer'), ('work', z(9)[1:].double(), ValueError, 'work must be'), ('max_len', -1, ValueError, 'bad sizes'),
        ('scale', math.inf, TstError, 'not finite')])
    with pytest.raises(TstError, match='are needed'):
        K.attn_cache4(rows, cache, iz(8, 300), iz(8), z(8, 256), 8, 4, 9000, work=z(4))
    x = z(8, 100)
    full = dict(logits=x, n_rows=8, n_cols=100, out=x, params=z(8, 3), hist=iz(8, 5), hist_len=iz(8), prompt=iz(6), prompt_cu=iz(9), bias=z(1, 100),
                bias_row=None, mask=iz(2, 4), mask_row=iz(8))
    each(K.adjust_logits, full, [
        ('out', z(8, 100, t=torch.bfloat16), ValueError, 'one type'), ('out', z(7, 100), ValueError, 'out must hold'), ('n_cols', 101, ValueError, 'logits must hold'),
        ('params', z(7, 3), ValueError, 'params must be'), ('params', None, ValueError, 'need params'), ('params', z(8, 4), ValueError, 'params must be'),
        ('hist', iz(7, 5), ValueError, 'hist must be'), ('hist', iz(5, 8).t(), ValueError, 'hist must be'), ('hist_len', iz(7), ValueError, 'hist_len must be'),
        ('prompt_cu', None, ValueError, 'needs prompt_cu'), ('prompt_cu', iz(8), ValueError, 'prompt_cu must be'), ('bias', z(1, 99), ValueError, 'bias must be'),
        ('bias', z(1, 100).half(), ValueError, 'bias must be'), ('mask', iz(2, 3), ValueError, 'mask must be'), ('mask_row', iz(7), ValueError, 'mask_row must be'),
        ('logits', x.half(), ValueError, 'fp32 or bf16'), ('sent', iz(7), ValueError, 'sent must be')])
    wide = z(16, 100)
    with pytest.raises(ValueError, match='out must be logits or not overlap it'):
        K.adjust_logits(wide[:8], 8, 100, wide[4:12])
    state = iz(4)
    each(K.grammar_next, dict(table=iz(2, 7), state=state, parent=None, tok=iz(4), out=iz(4), n_rows=4), [
        ('out', state, ValueError, 'out must not be state'), ('state', None, TypeError, 'state'), ('tok', iz(3), ValueError, 'tok must be'),
        ('tok', None, TstError, 'null pointer'), ('table', iz(7), ValueError, 'table must be'), ('parent', iz(3), ValueError, 'parent must be')])
    torch.cuda.synchronize()
