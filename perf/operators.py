"""Operators of prompted decoding, in their plain form and through this package's kernels.

Attention over whole prompts (packed, causal, grouped heads), page tables and slot maps of a paged cache, a key/value cache
held in 4 bits (written, read back, attended to by single tokens), and penalties / biases / grammar masks on logits.

The 4-bit format: groups of 32 elements along the head share a power of two 2^E, E the smallest exponent in [-126, 126] with
max|x| <= 6 * 2^E; an element is the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code) times its sign and 2^E; a
group that holds a NaN or an infinity stands for NaN.  Keys: codes [page][head][token][dh / 2], two elements to a byte (the
even one in the low half), scales E + 127 [page][head][token][dh / 32]; values: codes [page][head][dh / 2][token], scales
[page][head][dh / 32][token].
"""
import math
import random

import torch

own = False

BIG = 1 << 28          # elements of the largest temporary of the plain forms
DT = {'fp32': torch.float32, 'bf16': torch.bfloat16}


def _kernels():
    import tst_amd  # noqa: F401
    from tst_amd import kernels
    return kernels


# ---- cases -------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a handful of short prompts at the sizes of the fp32 translation decoder (2 heads of 128): the latency of a small prefill
        dict(name='prompt_fp32_few_short', op='prompt', dtype='fp32', heads=2, kv_heads=2, dh=128, seqs=16, longest=60, even=0, salt=1),
        # a serving batch of ragged prompts through the 512-wide language model (8 heads of 64)
        dict(name='prompt_bf16_ragged_batch', op='prompt', dtype='bf16', heads=8, kv_heads=8, dh=64, seqs=256, longest=512, even=0, salt=2),
        # two long documents, four query heads to a key head
        dict(name='prompt_bf16_long_grouped', op='prompt', dtype='bf16', heads=16, kv_heads=4, dh=128, seqs=2, longest=8191, even=1, salt=3),
        # requests of an interactive service entering a batch
        dict(name='plan_48_requests', op='plan', seqs=48, longest=90, room=50, page=16, spare=7, salt=4),
        # a bulk job's 8192 requests planned at once, two million prompt tokens
        dict(name='plan_8192_requests', op='plan', seqs=8192, longest=512, room=64, page=64, spare=100, salt=5),
        # the new keys and values of one decode step, 8 heads of 64
        dict(name='cache_step_bf16', op='store', dtype='bf16', tokens=256, kv_heads=8, dh=64, page=32, salt=6),
        # the keys and values of a whole prefill, fp32 activations
        dict(name='cache_prefill_fp32', op='store', dtype='fp32', tokens=65521, kv_heads=8, dh=128, page=64, salt=7),
        # one step of 64 sentences with short contexts at the language model's sizes, fp32
        dict(name='attend_fp32_short', op='attend', dtype='fp32', heads=8, kv_heads=8, dh=64, rows=64, longest=100, page=32, salt=8),
        # one step of a full serving batch, grouped heads, contexts of up to 8000 tokens
        dict(name='attend_bf16_batch', op='attend', dtype='bf16', heads=32, kv_heads=8, dh=128, rows=256, longest=8000, page=64, salt=9),
        # one step of three very long contexts: few rows, work only along the context
        dict(name='attend_bf16_few_long', op='attend', dtype='bf16', heads=16, kv_heads=4, dh=128, rows=3, longest=131001, page=64, salt=10),
        # constrained decoding of a small interactive batch over a 32000-token vocabulary
        dict(name='logits_fp32_small', op='logits', dtype='fp32', rows=16, V=32000, generated=40, prompt=60, masks=12, bias=1, salt=11),
        # the same for a large batch with long histories, bf16 logits
        dict(name='logits_bf16_large', op='logits', dtype='bf16', rows=2048, V=32000, generated=500, prompt=800, masks=64, bias=1, salt=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(8, 8, 64), (2, 2, 128), (16, 4, 128), (32, 8, 128), (12, 2, 64), (4, 1, 256), (8, 8, 32), (16, 1, 128), (10, 5, 64)]


def draw(rng):
    salt = rng.randrange(1 << 30)
    op = rng.choice(['prompt', 'prompt', 'plan', 'store', 'attend', 'attend', 'logits'])
    dtype = rng.choice(['bf16', 'bf16', 'fp32'])
    h, g, dh = rng.choice(HEADS)
    if op == 'prompt':
        while True:
            c = dict(op=op, dtype=dtype, heads=h, kv_heads=g, dh=dh, seqs=_log(rng, 1, 256), longest=_log(rng, 1, 8191),
                     even=rng.randrange(2), salt=salt)
            if work(c)['flops'] <= (4e11 if dtype == 'bf16' else 2e10) and sum(_lens(c)) * h * dh <= 1 << 27:
                return c
    if op == 'plan':
        while True:
            c = dict(op=op, seqs=_log(rng, 1, 8192), longest=_log(rng, 1, 4096), room=_log(rng, 1, 512), page=rng.choice([16, 32, 64, 128]),
                     spare=rng.choice([0, 1, 50]), salt=salt)
            if c['seqs'] * (c['longest'] + c['room']) <= 8192 * 576:
                return c
    if op == 'store':
        return dict(op=op, dtype=dtype, tokens=min(_log(rng, 1, 65521), (1 << 26) // (g * dh)), kv_heads=g, dh=dh,
                    page=rng.choice([16, 32, 64, 128]), salt=salt)
    if op == 'attend':
        while True:
            c = dict(op=op, dtype=dtype, heads=h, kv_heads=g, dh=dh, rows=_log(rng, 1, 512), longest=_log(rng, 1, 131001),
                     page=rng.choice([16, 32, 64, 128]), salt=salt)
            if c['rows'] * c['longest'] * g * dh <= 256 * 8000 * 8 * 128 and c['rows'] * c['longest'] * h <= 256 * 8000 * 32:
                return c
    while True:
        c = dict(op=op, dtype=dtype, rows=_log(rng, 1, 2048), V=_log(rng, 100, 60000), generated=_log(rng, 1, 2000), prompt=_log(rng, 1, 2000),
                 masks=rng.choice([0, 1, 30]), bias=rng.randrange(2), salt=salt)
        if c['rows'] * c['V'] * (1 if dtype == 'bf16' else 2) <= 2048 * 32000:
            return c


def _lens(case):
    """The lengths of a case's sequences: spread over 1 .. longest (even: near the longest), the longest among them."""
    rng = random.Random(case['salt'])
    n, top = case.get('seqs', case.get('rows')), case['longest']
    low = max(1, top * 7 // 10) if case.get('even') else 1
    lens = [rng.randint(low, top) for _ in range(n)]
    lens[rng.randrange(n)] = top
    return lens


def work(case):
    op = case['op']
    e = 2 if case.get('dtype') == 'bf16' else 4
    if op == 'prompt':
        lens = _lens(case)
        h, g, dh = case['heads'], case['kv_heads'], case['dh']
        return dict(bytes=sum(lens) * (2 * h + 2 * g) * dh * e, flops=4 * dh * h * sum(n * (n + 1) // 2 for n in lens))
    if op == 'plan':
        lens = _lens(case)
        width, need = _plan_sizes(case)
        return dict(bytes=4 * (3 * len(lens) + need + len(lens) * width + 3 * sum(lens)), flops=0)
    if op == 'store':
        n = 2 * case['tokens'] * case['kv_heads'] * case['dh']          # read the rows, write the codes, read them back, write the rows
        return dict(bytes=2 * n * e + 2 * n * 17 // 32, flops=0)
    if op == 'attend':
        total = sum(_lens(case))
        h, g, dh = case['heads'], case['kv_heads'], case['dh']
        return dict(bytes=total * g * 2 * dh * 17 // 32 + 2 * case['rows'] * h * dh * e, flops=4 * dh * h * total)
    R, V = case['rows'], case['V']
    return dict(bytes=2 * R * V * e + 4 * V * case['bias'] + case['masks'] * ((V + 31) // 32) * 4 + 2 * R * (case['generated'] + case['prompt']),
                flops=0)


# ---- inputs ------------------------------------------------------------------------------------------------------------------
def _gen(seed, salt):
    g = torch.Generator(device='cuda')
    g.manual_seed((seed * 1000003 + salt) % (1 << 62))
    return g


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


def _plan_sizes(case):
    need = [-(-(n + case['room']) // case['page']) for n in _lens(case)]
    return max(need), sum(need)


def _quantise(x):
    """x [..., dh] -> (codes uint8 [..., dh / 2], scales uint8 [..., dh / 32])"""
    grp = x.float().unflatten(-1, (-1, 32))
    top = grp.abs().amax(-1)
    m, ex = torch.frexp(top)
    E = (ex - 3 + (m > 0.75).int()).clamp(-126, 126)
    E = torch.where(top > 0, E, torch.full_like(E, -126))
    bad = ~torch.isfinite(grp).all(-1)
    y = torch.ldexp(grp, -E.unsqueeze(-1))
    a = y.abs()
    mag = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int()
           + (a > 5.0).int())
    code = (mag + 8 * (y < 0).int()).flatten(-2)
    scale = torch.where(bad, torch.full_like(E, 255), E + 127)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), scale.to(torch.uint8)


def _values(codes, scales):
    """The values of codes [..., dh / 2] and scales [..., dh / 32]: [..., dh]"""
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    c = codes.int()
    v = grid[torch.stack((c & 15, c >> 4), -1).flatten(-2)].unflatten(-1, (-1, 32))
    s = scales.int()
    f = torch.ldexp(torch.ones((), device=codes.device), s - 127)
    f = torch.where(s == 255, torch.full_like(f, float('nan')), f)
    return (v * f.unsqueeze(-1)).flatten(-2)


def _inputs(case, seed):
    op = case['op']
    g = _gen(seed, case['salt'])
    dev = 'cuda'
    if op == 'prompt':
        lens = _lens(case)
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        width = (case['heads'] + 2 * case['kv_heads']) * case['dh']
        qkv = torch.randn((cu[-1], width), generator=g, device=dev).to(DT[case['dtype']])     # the fused projection's output
        a, b = case['heads'] * case['dh'], (case['heads'] + case['kv_heads']) * case['dh']
        return dict(q=qkv[:, :a], k=qkv[:, a:b], v=qkv[:, b:], cu=_i32(cu), lens=lens,
                    out=torch.empty((cu[-1], a), dtype=DT[case['dtype']], device=dev))
    if op == 'plan':
        # the lengths are the case's, in an order that the seed draws, so that tables and outputs keep their sizes
        lens = _lens(case)
        width, need = _plan_sizes(case)
        order = torch.randperm(len(lens), generator=g, device=dev)
        total = sum(lens)
        i32 = dict(dtype=torch.int32, device=dev)
        return dict(lens=_i32(lens)[order].contiguous(), room=torch.full((len(lens),), case['room'], **i32),
                    pages=torch.randperm(need + case['spare'], generator=g, device=dev).to(torch.int32),
                    table=torch.empty((len(lens), width), **i32), cu=torch.empty(len(lens) + 1, **i32), slots=torch.empty(total, **i32),
                    pos=torch.empty(total, **i32), seq=torch.empty(total, **i32), used=torch.empty(1, **i32))
    if op == 'store':
        n, w = case['tokens'], case['kv_heads'] * case['dh']
        kv = torch.randn((n, 2 * w), generator=g, device=dev)
        kv *= torch.exp(0.7 * torch.randn((1, 2 * w), generator=g, device=dev))            # channels differ in size, as projections do
        kv = kv.to(DT[case['dtype']])
        pages = (n + case['page'] - 1) // case['page'] + 3
        slots = torch.randperm(pages, generator=g, device=dev)[torch.arange(n, device=dev) // case['page']] * case['page'] + (
            torch.arange(n, device=dev) % case['page'])
        return dict(k=kv[:, :w], v=kv[:, w:], slots=slots.to(torch.int32), pages=pages,
                    k_out=torch.empty((n, w), dtype=kv.dtype, device=dev), v_out=torch.empty((n, w), dtype=kv.dtype, device=dev))
    if op == 'attend':
        lens, page, hk, dh = _lens(case), case['page'], case['kv_heads'], case['dh']
        need = [-(-n // page) for n in lens]
        pages = sum(need) + 5
        perm = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
        at = torch.zeros(len(lens), dtype=torch.int64)
        at[1:] = torch.tensor(need).cumsum(0)[:-1]
        at, need_t = at.to(dev), torch.tensor(need, device=dev)
        cols = torch.arange(max(need), device=dev).unsqueeze(0)
        table = torch.where(cols < need_t.unsqueeze(1), perm[(at.unsqueeze(1) + cols).clamp(max=pages - 1)], torch.full((), -1, dtype=torch.int32, device=dev))
        u8 = dict(dtype=torch.uint8, device=dev)
        kc, ks = torch.empty((pages, hk, page, dh // 2), **u8), torch.empty((pages, hk, page, dh // 32), **u8)
        vc, vs = torch.empty((pages, hk, dh // 2, page), **u8), torch.empty((pages, hk, dh // 32, page), **u8)
        step = max(1, (1 << 26) // (hk * page * dh))
        size = torch.exp(0.5 * torch.randn((1, hk, 1, dh), generator=g, device=dev))
        for p in range(0, pages, step):
            m = min(step, pages - p)
            c, s = _quantise(torch.randn((m, hk, page, dh), generator=g, device=dev) * size)
            kc[p:p + m], ks[p:p + m] = c, s
            c, s = _quantise(torch.randn((m, hk, page, dh), generator=g, device=dev))
            vc[p:p + m], vs[p:p + m] = c.transpose(2, 3), s.transpose(2, 3)
        q = torch.randn((case['rows'], case['heads'] * dh), generator=g, device=dev).to(DT[case['dtype']])
        return dict(q=q, kc=kc, ks=ks, vc=vc, vs=vs, table=table.contiguous(), lens=_i32(lens), longest=max(lens), out=torch.empty_like(q))
    R, V, M = case['rows'], case['V'], case['masks']
    logits = (3 * torch.randn((R, V), generator=g, device=dev)).to(DT[case['dtype']])
    few = lambda shape: (V * torch.rand(shape, generator=g, device=dev) ** 3).int().clamp(max=V - 1)     # noqa: E731  frequent tokens repeat
    hist = few((R, case['generated']))
    hist_len = torch.randint(0, case['generated'] + 1, (R,), generator=g, device=dev, dtype=torch.int32)
    plen = torch.randint(0, case['prompt'] + 1, (R,), generator=g, device=dev)
    prompt_cu = torch.zeros(R + 1, dtype=torch.int32, device=dev)
    prompt_cu[1:] = plen.cumsum(0)
    prompt = few((R * case['prompt'],))
    params = torch.stack((1 + 0.5 * torch.rand(R, generator=g, device=dev), torch.rand(R, generator=g, device=dev),
                          torch.rand(R, generator=g, device=dev)), 1).contiguous()
    bias = mask = mask_row = None
    if case['bias']:
        bias = torch.where(torch.rand((1, V), generator=g, device=dev) < 0.01, 5 * torch.randn((1, V), generator=g, device=dev),
                           torch.zeros((), device=dev))
    if M:
        # grammar states from strict (a few tokens allowed) to loose; -1: the row is unconstrained
        share = torch.rand((M, 1), generator=g, device=dev)
        bits = torch.rand((M, (V + 31) // 32, 32), generator=g, device=dev) < share.unsqueeze(-1)
        mask = (bits.long() << torch.arange(32, device=dev)).sum(-1).to(torch.int32)
        mask_row = torch.randint(-1, M, (R,), generator=g, device=dev, dtype=torch.int32)
    return dict(logits=logits, hist=hist, hist_len=hist_len, prompt=prompt, prompt_cu=prompt_cu, params=params, bias=bias, mask=mask,
                mask_row=mask_row, out=torch.empty_like(logits))


def prepare(case, seed):
    s = _inputs(case, seed)
    s['case'] = case
    if own and case['op'] == 'store':
        s['cache'] = _kernels().Cache4(s['pages'], case['page'], case['kv_heads'], case['dh'])
    if own and case['op'] == 'attend':
        K = _kernels()
        s['cache'] = K.Cache4(s['kc'].shape[0], case['page'], case['kv_heads'], case['dh'], tensors=(s['kc'], s['ks'], s['vc'], s['vs']))
        s['work'] = K.attn_cache4_work(case['rows'], case['heads'], case['kv_heads'], case['dh'], s['longest'])
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------------
def run(s):
    op = s['case']['op']
    return (_run_own if own else _run_plain)(op, s['case'], s)


def _run_own(op, c, s):
    K = _kernels()
    if op == 'prompt':
        K.attn_prompt(s['q'], s['k'], s['v'], s['cu'], s['out'], c['heads'], c['kv_heads'])
        return s['out']
    if op == 'plan':
        K.page_plan(s['lens'], s['room'], s['pages'], c['page'], s['table'], s['cu'], s['slots'], s['pos'], s['seq'], s['used'])
        return [s[n] for n in ('table', 'cu', 'slots', 'pos', 'seq', 'used')]
    if op == 'store':
        K.cache4_write(s['cache'], s['k'], s['v'], s['slots'], c['tokens'])
        K.cache4_read(s['cache'], s['slots'], s['k_out'], s['v_out'], c['tokens'])
        return [s['k_out'], s['v_out']]
    if op == 'attend':
        K.attn_cache4(s['q'], s['cache'], s['table'], s['lens'], s['out'], c['rows'], c['heads'], s['longest'], work=s['work'])
        return s['out']
    K.adjust_logits(s['logits'], c['rows'], c['V'], s['out'], params=s['params'], hist=s['hist'], hist_len=s['hist_len'], prompt=s['prompt'],
                    prompt_cu=s['prompt_cu'], bias=s['bias'], mask=s['mask'], mask_row=s['mask_row'])
    return s['out']


def _run_plain(op, c, s):
    if op == 'prompt':
        return _prompt_plain(c, s)
    if op == 'plan':
        return _plan_plain(c, s)
    if op == 'store':
        hk, dh = c['kv_heads'], c['dh']
        res = []
        for x in (s['k'], s['v']):
            res.append(_values(*_quantise(x.unflatten(1, (hk, dh)))).flatten(1).to(x.dtype))
        return res
    if op == 'attend':
        return _attend_plain(c, s)
    return _logits_plain(c, s)


def _prompt_plain(c, s):
    h, g, dh = c['heads'], c['kv_heads'], c['dh']
    lens, dev = s['lens'], 'cuda'
    out = s['out']
    q, k, v = (s[n].unflatten(1, (-1, dh)) for n in 'qkv')
    b0, at = 0, 0
    while b0 < len(lens):
        b1, top = b0, 0                          # sequences b0 .. b1 - 1 together, padded to the longest of them
        while b1 < len(lens) and (b1 == b0 or (b1 + 1 - b0) * h * max(top, lens[b1]) ** 2 <= BIG):
            top = max(top, lens[b1])
            b1 += 1
        n = torch.tensor(lens[b0:b1], device=dev)
        start = at + n.cumsum(0) - n
        cols = torch.arange(top, device=dev)
        live = cols.unsqueeze(0) < n.unsqueeze(1)
        rows = start.unsqueeze(1) + cols.unsqueeze(0).minimum(n.unsqueeze(1) - 1)
        future = cols.unsqueeze(0) > cols.unsqueeze(1)
        kk = k[rows].float().permute(0, 2, 3, 1)                 # [b, g, dh, t]
        vv = v[rows].float().transpose(1, 2)                     # [b, g, t, dh]
        res = torch.empty((b1 - b0, top, h, dh), device=dev)
        step = h if b1 - b0 > 1 else max(1, min(h, BIG // (top * top)))
        for h0 in range(0, h, step):
            hs = torch.arange(h0, min(h, h0 + step), device=dev)
            gs = hs // (h // g)
            qq = q[rows][:, :, hs].float().transpose(1, 2)       # [b, heads, t, dh]
            sc = torch.matmul(qq, kk[:, gs]) * (1.0 / math.sqrt(dh))
            sc.masked_fill_(future, float('-inf'))
            sc = torch.exp(sc - sc.amax(-1, keepdim=True))
            sc = sc / sc.sum(-1, keepdim=True)
            res[:, :, hs] = torch.matmul(sc, vv[:, gs]).transpose(1, 2)
        out[rows[live]] = res[live].flatten(1).to(out.dtype)
        at += sum(lens[b0:b1])
        b0 = b1
    return out


def _plan_plain(c, s):
    page, lens, dev = c['page'], s['lens'].long(), 'cuda'
    B, W = s['table'].shape
    need = (lens + s['room'].long() + page - 1) // page
    first = need.cumsum(0) - need
    cols = torch.arange(W, device=dev).unsqueeze(0)
    idx = (first.unsqueeze(1) + cols).clamp(max=s['pages'].numel() - 1)
    table = torch.where(cols < need.unsqueeze(1), s['pages'][idx], torch.full((), -1, dtype=torch.int32, device=dev))
    cu = torch.zeros(B + 1, dtype=torch.int64, device=dev)
    cu[1:] = lens.cumsum(0)
    N = s['slots'].numel()
    i = torch.arange(N, device=dev)
    seq = torch.bucketize(i, cu[1:], right=True)
    pos = i - cu[seq]
    slots = table[seq, pos // page].long() * page + pos % page
    return [table, cu.int(), slots.int(), pos.int(), seq.int(), need.sum().int().view(1)]


def _gather(s, rows, top, c):
    """Keys and values [row, head, token, dh] of the first `top` tokens of the given rows (pages beyond a row's own: page 0)."""
    page = c['page']
    ids = s['table'][rows, :(top + page - 1) // page].long().clamp(min=0)
    k = _values(s['kc'][ids], s['ks'][ids])                                              # [r, n, head, page, dh]
    v = _values(s['vc'][ids].transpose(-1, -2), s['vs'][ids].transpose(-1, -2))
    return [x.transpose(1, 2).flatten(2, 3)[:, :, :top] for x in (k, v)]


def _attend_plain(c, s):
    R, h, g, dh = c['rows'], c['heads'], c['kv_heads'], c['dh']
    lens = _lens(c)
    out = torch.empty_like(s['q'])
    r0 = 0
    while r0 < R:
        r1, top = r0, 0
        while r1 < R and (r1 == r0 or (r1 + 1 - r0) * max(top, lens[r1]) * max(g * dh, h) <= BIG * 2):
            top = max(top, lens[r1])
            r1 += 1
        rows = torch.arange(r0, r1, device='cuda')
        k, v = _gather(s, rows, top, c)
        q = s['q'][r0:r1].float().view(r1 - r0, g, h // g, dh)
        sc = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(dh))
        dead = torch.arange(top, device='cuda').unsqueeze(0) >= s['lens'][r0:r1].unsqueeze(1)
        sc.masked_fill_(dead[:, None, None], float('-inf'))
        sc = torch.exp(sc - sc.amax(-1, keepdim=True))
        sc = sc / sc.sum(-1, keepdim=True)
        out[r0:r1] = torch.matmul(sc, v).reshape(r1 - r0, h * dh).to(out.dtype)
        r0 = r1
    return out


def _counts(c, s):
    R, V = c['rows'], c['V']
    gen = torch.zeros((R, V + 1), device='cuda')
    live = torch.arange(s['hist'].shape[1], device='cuda').unsqueeze(0) < s['hist_len'].unsqueeze(1)
    gen.scatter_add_(1, torch.where(live, s['hist'].long(), V), torch.ones_like(s['hist'], dtype=torch.float32))
    cu = s['prompt_cu'].long()
    n = s['prompt'].numel()
    at = torch.arange(n, device='cuda')
    row = torch.bucketize(at, cu[1:], right=True)
    used = row < R
    seen = torch.zeros((R + 1, V), dtype=torch.bool, device='cuda')
    seen[torch.where(used, row, R), s['prompt'].long()] = True
    return gen[:, :V], seen[:R]


def _logits_plain(c, s):
    V = c['V']
    gen, seen = _counts(c, s)
    rp, fp, pp = (s['params'][:, i:i + 1] for i in range(3))
    y = s['logits'].float()
    y = torch.where(seen | (gen > 0), torch.where(y > 0, y / rp, y * rp), y)
    y = torch.where(gen > 0, (y - gen * fp) - pp, y)
    if s['bias'] is not None:
        y = y + s['bias']
    if s['mask'] is not None:
        bits = (s['mask'].unsqueeze(-1) >> torch.arange(32, device='cuda', dtype=torch.int32)) & 1
        bits = bits.flatten(1)[:, :V].bool()
        ok = bits[s['mask_row'].long().clamp(min=0)] | (s['mask_row'] < 0).unsqueeze(1)
        y = torch.where(ok, y, torch.full((), float('-inf'), device='cuda'))
    return y.to(s['logits'].dtype)


# ---- in 64 bits, from the definitions ------------------------------------------------------------------------------------------
def _decode64(codes, scales):
    """The numbers of 4-bit codes from the fields of the format: sign, two exponent bits, one mantissa bit."""
    byte = codes.long()
    parts = []
    for nibble in (byte % 16, byte // 16):
        sign, e, m = 1.0 - 2.0 * (nibble // 8).double(), (nibble // 2 % 4).double(), (nibble % 2).double()
        parts.append(sign * torch.where(e > 0, (1 + m / 2) * 2.0 ** (e - 1), m / 2))
    x = torch.empty(codes.shape[:-1] + (2 * codes.shape[-1],), dtype=torch.float64, device=codes.device)
    x[..., 0::2], x[..., 1::2] = parts
    return x * (2.0 ** (scales.double() - 127)).repeat_interleave(32, dim=-1)


def exact(case, seed):
    op, s = case['op'], _inputs(case, seed)
    if op == 'prompt':
        h, g, dh = case['heads'], case['kv_heads'], case['dh']
        res = torch.empty(s['out'].shape, dtype=torch.float64, device='cuda')
        at = 0
        for n in s['lens']:
            for kv in range(g):
                k = s['k'][at:at + n, kv * dh:(kv + 1) * dh].double()
                v = s['v'][at:at + n, kv * dh:(kv + 1) * dh].double()
                for head in range(kv * (h // g), (kv + 1) * (h // g)):
                    q = s['q'][at:at + n, head * dh:(head + 1) * dh].double() / math.sqrt(dh)
                    p = torch.softmax((q @ k.t()).masked_fill(torch.ones((n, n), dtype=torch.bool, device='cuda').triu(1), -math.inf), 1)
                    res[at:at + n, head * dh:(head + 1) * dh] = p @ v
            at += n
        return res
    if op == 'plan':
        return None            # whole numbers
    if op == 'store':
        grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device='cuda')
        odd = torch.arange(8, device='cuda') & 1
        res = []
        for x in (s['k'], s['v']):
            parts = []
            for part in x.split(max(1, (1 << 24) // x.shape[1])):
                y = part.double().reshape(-1, 32)
                top = y.abs().amax(1, keepdim=True)
                unit = torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, torch.ones_like(top)) / 6)).clamp(-126, 126))
                # log2 may land one step beside the border: take the smallest power of two whose six-fold holds the group
                unit = torch.where(top <= 3 * unit, unit / 2, torch.where(top > 6 * unit, unit * 2, unit))
                dist = (y.abs().unsqueeze(-1) / unit.unsqueeze(-1) - grid).abs()
                near = torch.where(dist == dist.amin(-1, keepdim=True), odd, 2).argmin(-1)
                parts.append((grid[near] * unit * torch.sign(y)).reshape(part.shape))
            res.append(torch.cat(parts))
        return res
    if op == 'attend':
        h, g, dh = case['heads'], case['kv_heads'], case['dh']
        res = torch.empty(s['q'].shape, dtype=torch.float64, device='cuda')
        for r, n in enumerate(_lens(case)):
            ids = s['table'][r, :(n + case['page'] - 1) // case['page']].long()
            k = _decode64(s['kc'][ids], s['ks'][ids]).permute(1, 0, 2, 3).reshape(g, -1, dh)[:, :n]
            v = _decode64(s['vc'][ids].transpose(2, 3), s['vs'][ids].transpose(2, 3)).permute(1, 0, 2, 3).reshape(g, -1, dh)[:, :n]
            q = s['q'][r].double().view(g, h // g, dh) / math.sqrt(dh)
            res[r] = (torch.softmax(q @ k.transpose(1, 2), -1) @ v).flatten()
        return res
    R, V = case['rows'], case['V']
    res = torch.empty((R, V), dtype=torch.float64, device='cuda')
    cu, hl = s['prompt_cu'].tolist(), s['hist_len'].tolist()
    rows = s['mask_row'].tolist() if s['mask'] is not None else [-1] * R
    shift = torch.arange(32, device='cuda')
    for r in range(R):
        gen = torch.bincount(s['hist'][r, :hl[r]].long(), minlength=V).double()
        old = torch.bincount(s['prompt'][cu[r]:cu[r + 1]].long(), minlength=V)
        rp, fp, pp = s['params'][r].double()
        y = s['logits'][r].double()
        y = torch.where((old + gen) > 0, torch.where(y > 0, y / rp, y * rp), y) - gen * fp - (gen > 0) * pp
        if s['bias'] is not None:
            y = y + s['bias'][0].double()
        if rows[r] >= 0:
            y[((s['mask'][rows[r]].long().unsqueeze(1) >> shift) & 1).flatten()[:V] == 0] = -math.inf
        res[r] = y
    return res
