"""GPU: the decode loop over prompts of different lengths, a cache in 4 bits and rules on the logits, end to end.

Logits are compared under the tolerances the package states: fp32 1e-4 relative (``helpers.logits_close``), bf16 2e-2 of a row's largest
magnitude.  The 4-bit cache is compared with a model in 64 bits that attends to exactly what the cache holds (read back), so that a tie
in the 4-bit rounding cannot hide or show anything; what it holds is compared with the unrounded keys and values: an element is off by
at most half the widest step, 2^E, and 2^E < amax / 3 of its group of 32.
"""
import math

import pytest
import torch

from helpers import logits_close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def T():
    import tst_amd
    assert torch.cuda.is_available()
    return tst_amd


def make_lm(T, dtype, d=128, heads=2, layers=2, V=203, pe_max_len=400, seed=1):
    from tst_amd import synthetic
    vocab = T.Vocab.synthetic(V)
    lm = T.TransformerLM(T.HP(dict(model_size=d, n_layers=layers, n_heads=heads, d_ff=2 * d, pe_max_len=pe_max_len)), vocab, dtype=dtype)
    lm.load_state_dict(synthetic.synthetic_state_dict(lm, 3, 1.0, 2.0, seed=seed))
    return lm, vocab


def ragged(V, lens, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(4, V, (n,), generator=g) for n in lens]


class Model64:
    """The language model in 64 bits over one token sequence; with bf16 weights where the model stores them so."""

    def __init__(self, lm):
        self.P = {k: v.double() for k, v in lm.state_dict().items()}
        if lm.dtype == 'bf16':
            for k, v in self.P.items():
                if k.endswith('weight') and v.dim() == 2 and k != 'embed.weight':
                    self.P[k] = v.to(torch.bfloat16).double()
        self.lm, self.dh = lm, lm.d // lm.heads

    def ln(self, x, name):
        return torch.nn.functional.layer_norm(x, (self.lm.d,), self.P[name + '.weight'], self.P[name + '.bias'])

    def lin(self, x, name):
        return x @ self.P[name + '.weight'].t() + self.P[name + '.bias']

    def run(self, z, toks, first=0, held=None):
        """Logits of positions first ..; ``held``: per layer the (keys, values) [length, d] that stand in for the model's own."""
        lm, dh = self.lm, self.dh
        toks = toks.cuda()
        x = self.P['embed.weight'][toks] * math.sqrt(lm.d) + self.P['pe'][first:first + len(toks)] + z.double()
        kv = []
        for i in range(lm.n_layers):
            p = 'layers.%d.' % i
            h = self.ln(x, p + 'ln1')
            q, k, v = (self.lin(h, p + 'self_attn.' + n) for n in 'qkv')
            kv.append((k, v))
            if held is not None:
                k, v = held[i]
            t = torch.arange(first, first + len(toks), device='cuda')
            dead = torch.arange(k.shape[0], device='cuda').unsqueeze(0) > t.unsqueeze(1)
            out = []
            for j in range(lm.heads):
                c = slice(j * dh, (j + 1) * dh)
                s = (q[:, c] @ k[:, c].t() / math.sqrt(dh)).masked_fill(dead, -math.inf)
                out.append(torch.softmax(s, 1) @ v[:, c])
            x = x + self.lin(torch.cat(out, 1), p + 'self_attn.o')
            x = x + self.lin(torch.relu(self.lin(self.ln(x, p + 'ln2'), p + 'ff.w1')), p + 'ff.w2')
        return self.lin(self.ln(x, 'ln'), 'out'), kv


def assert_logits(got, want, dtype):
    got, want = got.double().cpu(), want.double().cpu()
    if dtype == 'fp32':
        ok, worst = logits_close(got.numpy(), want.numpy())
        assert ok, worst
    else:
        assert ((got - want).abs().amax(-1) <= 2e-2 * want.abs().amax(-1)).all()


@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
@pytest.mark.parametrize('d,heads', [(128, 2), (96, 3), (256, 2)])
def test_prompt_logits_of_ragged_sequences(T, dtype, d, heads):
    lm, vocab = make_lm(T, dtype, d=d, heads=heads)
    lens = [1, 70, 0, 33, 200]
    seqs = ragged(203, lens, 3)
    z = torch.randn((5, d), generator=torch.Generator().manual_seed(5)).cuda() * 0.1
    got = lm.prompt_logits(z, seqs)
    assert [tuple(g.shape) for g in got] == [(n, 203) for n in lens]
    m = Model64(lm)
    for i, s in enumerate(seqs):
        if len(s):
            assert_logits(got[i], m.run(z[i], s)[0], dtype)
    steps = lm(z[1:2], seqs[1].unsqueeze(0))
    assert_logits(got[1], steps[0], dtype)
    assert lm.prompt_logits(z[:0], []) == [] and lm.prompt_logits(z[:1], [torch.empty(0, dtype=torch.int64)])[0].shape == (0, 203)


@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
@pytest.mark.parametrize('d,heads,page', [(128, 2, 32), (64, 2, 16), (256, 2, 64), (256, 1, 128)])
def test_paged_session_against_a_model_that_attends_to_what_the_cache_holds(T, dtype, d, heads, page):
    from tst_amd import kernels as K
    lm, vocab = make_lm(T, dtype, d=d, heads=heads)
    lens = [1, 40, 2, 130, 33]
    prompts = ragged(203, lens, 4)
    z = torch.randn((5, d), generator=torch.Generator().manual_seed(6)).cuda() * 0.1
    steps = 4
    sess = lm.paged_session(z, prompts, steps, page=page)
    new = ragged(203, [steps] * 5, 9)
    rows = K.RowState(5, steps, torch.device('cuda', 0), False, 0)
    order = torch.tensor([3, 0, 4, 1, 2], dtype=torch.int32, device='cuda')        # rows need not be in sentence order
    rows.sent.copy_(order)
    m = Model64(lm)
    for t in range(steps):
        feed = [prompts[s][-1] if t == 0 else new[s][t - 1] for s in order.tolist()]
        rows.tok.copy_(torch.stack(feed))
        logits = sess.step(rows, 5, t)[:5, :203].clone()
        for r, s in enumerate(order.tolist()):
            n = lens[s] + t
            toks = torch.cat([prompts[s], new[s][:t]])
            p = torch.arange(n, device='cuda')
            slots = (sess.table[s].long()[p // page] * page + p % page).to(torch.int32)
            held = []
            for c in sess.caches:
                k, v = (torch.empty((n, d), device='cuda') for _ in range(2))
                K.cache4_read(c, slots, k, v, n)
                held.append((k.double(), v.double()))
            want, _ = m.run(z[s], toks[-1:], first=n - 1, held=held)
            assert_logits(logits[r:r + 1], want, dtype)
            if t == 0:
                own = m.run(z[s], toks)[1]
                slack = 1e-3 if dtype == 'fp32' else 6e-2     # what the model's own arithmetic is off by before the rounding
                for have, true in zip(held, own):
                    for a, b in zip(have, true):
                        top = b.reshape(n, -1, 32).abs().amax(-1, keepdim=True)
                        assert ((a - b).reshape(n, -1, 32).abs() <= top * (1 / 3 + slack)).all()


@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
def test_decode_over_ragged_prompts(T, dtype):
    """InferenceState over a list of prompts: results start with the prompts, tokens follow the session's own logits, and one sentence
    alone gives the same first logits."""
    lm, vocab = make_lm(T, dtype, layers=3)
    lens = [5, 1, 64, 17, 2, 100]
    prompts = ragged(203, lens, 7)
    z = torch.randn((6, 128), generator=torch.Generator().manual_seed(8)).cuda() * 0.1
    st = T.InferenceState({'model': lm, 'inputs': z, 'vocab': vocab, 'max_len': 12, 'kv_cache': 'fp4', 'active_seqs': prompts, 'return_logits': True})
    out = st.inference()
    eos = vocab.stoi['<eos>']
    for i, (p, o) in enumerate(zip(prompts, out)):
        assert o[:len(p)].tolist() == p.tolist() and len(p) <= len(o) <= len(p) + 12
        for t, (lg, sent) in enumerate(st.step_logits):
            at = (sent == i).nonzero().flatten().tolist()
            assert (len(at) == 1) == (t <= len(o) - len(p)) or t == len(o) - len(p)
            if at and t < len(o) - len(p):
                assert int(lg[at[0]].float().argmax()) == int(o[len(p) + t])
            elif at:
                assert int(lg[at[0]].float().argmax()) == eos or t == 12
    for i in (2, 5):
        alone = T.InferenceState({'model': lm, 'inputs': z[i:i + 1], 'vocab': vocab, 'max_len': 12, 'kv_cache': 'fp4', 'active_seqs': [prompts[i]],
                                  'return_logits': True})
        alone.inference()
        assert_logits(alone.step_logits[0][0][:1], st.step_logits[0][0][i:i + 1], dtype)
    packed = T.InferenceState({'model': lm, 'inputs': z, 'vocab': vocab, 'max_len': 12, 'kv_cache': 'fp4', 'active_seqs': prompts})
    tok, n, _ = packed.decode_packed()
    assert [p.tolist()[:-1] + tok[i, :int(n[i])].tolist() for i, p in enumerate(prompts)] == [o.tolist() for o in out]


def test_decode_4bit_without_prompts_sampling_and_streams(T):
    lm, vocab = make_lm(T, 'bf16')
    z = torch.randn((40, 128), generator=torch.Generator().manual_seed(8)).cuda() * 0.1
    args = {'model': lm, 'inputs': z, 'vocab': vocab, 'max_len': 15, 'kv_cache': 'fp4'}
    a = [s.tolist() for s in T.InferenceState(dict(args)).inference()]
    b = [s.tolist() for s in T.InferenceState(dict(args, active_seqs=torch.full((40, 1), vocab.stoi['<bos>']))).inference()]
    assert a == b and all(s[0] == vocab.stoi['<bos>'] for s in a)
    jobs = [lambda: [s.tolist() for s in T.InferenceState(dict(args)).inference()] for _ in range(3)]
    assert T.run_on_streams(jobs) == [a] * 3
    smp = dict(args, sample_type='sample', seed=11, temperature=0.8)
    c, d = ([s.tolist() for s in T.InferenceState(dict(smp)).inference()] for _ in range(2))
    assert c == d and c != a


# ---- rules ----------------------------------------------------------------------------------------------------------------------
class TableModel:
    """A foreign model: the logits after a token are a row of a table (and it keeps that memory)."""

    def __init__(self, V, seed):
        self.table = (3 * torch.randn((V, V), generator=torch.Generator().manual_seed(seed))).cuda()

    def __call__(self, inputs, active_seqs, *args, **kw):
        return self.table[active_seqs[:, -1:]]


def plain_rules(x, V, prompt, generated, rep=1.0, freq=0.0, pres=0.0, bias=None, ok=None):
    y = x.clone()
    f = lambda v: torch.tensor(float(v), dtype=torch.float32)     # noqa: E731
    for v in set(prompt) | set(generated):
        y[v] = y[v] / f(rep) if y[v] > 0 else y[v] * f(rep)
    for v in set(generated):
        y[v] = (y[v] - f(generated.count(v)) * f(freq)) - f(pres)
    if bias is not None:
        y = y + bias
    if ok is not None:
        y[~ok] = -math.inf
    return y


def plain_greedy(table, start, eos, max_len, rules, grammar=None, state=0):
    out, gen = list(start), []
    for _ in range(max_len):
        ok = None if grammar is None else grammar[state] >= 0
        y = plain_rules(table[out[-1]], table.shape[0], start, gen, ok=ok if ok is not None else rules.get('ok'),
                        **{k: v for k, v in rules.items() if k != 'ok'})
        v = int(y.argmax())
        if v == eos:
            break
        out.append(v)
        gen.append(v)
        if grammar is not None:
            state = int(grammar[state, v])
    return out


def plain_beam(table, start, eos, max_len, k, rules, grammar=None, state=0):
    """Beam search over the table in 64 bits: k best continuations by summed log-probability, finished ones kept."""
    beams = [(0.0, list(start), [], False, state)]
    for _ in range(max_len):
        offers = []
        for b, (score, toks, gen, fin, st) in enumerate(beams):
            if fin:
                offers.append((score, b, 0, beams[b]))
                continue
            ok = None if grammar is None or st < 0 else grammar[st] >= 0
            y = plain_rules(table[toks[-1]], table.shape[0], start, gen, ok=ok if ok is not None else rules.get('ok'),
                            **{n: v for n, v in rules.items() if n != 'ok'}).double()
            lp = y - torch.logsumexp(y, 0)
            for rank, v in enumerate(torch.sort(lp, descending=True, stable=True).indices[:k].tolist()):
                nst = st if grammar is None else (-1 if st < 0 else int(grammar[st, v]))
                offers.append((score + float(lp[v]), b, rank, (score + float(lp[v]), toks + [v], gen + [v], v == eos, nst)))
        offers.sort(key=lambda o: (-o[0], o[1], o[2]))
        beams = [(o[0],) + o[3][1:] for o in offers[:k]]
        if beams[0][3]:
            break
    best = beams[0][1]
    return best[:-1] if beams[0][3] else best


V = 97
CASES = {
    'repetition': dict(repetition_penalty=1.7),
    'frequency': dict(frequency_penalty=0.9, presence_penalty=0.4),
    'all': dict(repetition_penalty=1.3, frequency_penalty=0.5, presence_penalty=-0.2),
}


def to_plain(rules, i):
    return {a: (rules[b][i] if isinstance(rules[b], (list, torch.Tensor)) else rules[b])
            for a, b in (('rep', 'repetition_penalty'), ('freq', 'frequency_penalty'), ('pres', 'presence_penalty')) if b in rules}


@pytest.mark.parametrize('beam', [1, 4])
@pytest.mark.parametrize('case', sorted(CASES))
def test_penalties_follow_every_hypothesis(T, case, beam):
    vocab = T.Vocab.synthetic(V)
    model, table = TableModel(V, 3), TableModel(V, 3).table.cpu()
    kept = model.table.clone()
    B, bos, eos = 9, vocab.stoi['<bos>'], vocab.stoi['<eos>']
    start = torch.randint(4, V, (B, 3), generator=torch.Generator().manual_seed(2))
    st = T.InferenceState({'model': model, 'inputs': torch.zeros((B, 1), device='cuda'), 'vocab': vocab, 'max_len': 14, 'beam_size': beam,
                           'active_seqs': start.cuda(), **CASES[case]})
    got = [s.tolist() for s in st.inference()]
    for i in range(B):
        p = to_plain(CASES[case], i)
        want = (plain_greedy(table, start[i].tolist(), eos, 14, p) if beam == 1 else plain_beam(table, start[i].tolist(), eos, 14, beam, p))
        assert got[i] == want, (i, got[i], want)
    assert torch.equal(model.table, kept), 'the foreign model\'s memory was written'


@pytest.mark.parametrize('beam', [1, 4])
def test_rules_per_sentence_biases_and_masks(T, beam):
    vocab = T.Vocab.synthetic(V)
    model, table = TableModel(V, 4), TableModel(V, 4).table.cpu()
    B, bos, eos = 6, vocab.stoi['<bos>'], vocab.stoi['<eos>']
    g = torch.Generator().manual_seed(1)
    rules = dict(repetition_penalty=(1 + torch.rand(B, generator=g)).tolist(), presence_penalty=torch.rand(B, generator=g).tolist())
    bias = torch.randn((B, V), generator=g)
    ok = torch.rand((B, V), generator=g) < 0.3
    ok[:, 50] = True
    ok[1] = False
    ok[1, 60] = True                                    # one token only: fewer than the beams
    args = {'model': model, 'inputs': torch.zeros((B, 1), device='cuda'), 'vocab': vocab, 'max_len': 10, 'beam_size': beam}
    got = [s.tolist() for s in T.InferenceState(dict(args, logit_bias=bias, allowed_tokens=ok, **rules)).inference()]
    run = plain_greedy if beam == 1 else (lambda *a, **kw: plain_beam(*a[:4], beam, *a[4:], **kw))
    for i in range(B):
        p = dict(to_plain(rules, i), bias=bias[i], ok=ok[i])
        assert got[i] == run(table, [bos], eos, 10, p)
    got = [s.tolist() for s in T.InferenceState(dict(args, logit_bias={7: 50.0, 3: -100.0})).inference()]
    one = torch.zeros(V)
    one[7], one[3] = 50.0, -100.0
    assert got == [run(table, [bos], eos, 10, dict(bias=one))] * B and got[0] == [bos] + [7] * 10


@pytest.mark.parametrize('B', [5, 3000])
@pytest.mark.parametrize('beam', [1, 3])
def test_grammar(T, beam, B):
    """A grammar's state follows each row through retirement and beam reorders (3000 sentences: the loop that reads exact counts)."""
    vocab = T.Vocab.synthetic(V)
    model, table = TableModel(V, 5), TableModel(V, 5).table.cpu()
    bos, eos = vocab.stoi['<bos>'], vocab.stoi['<eos>']
    g = torch.Generator().manual_seed(6)
    S = 7
    nxt = torch.where(torch.rand((S, V), generator=g) < 0.25, torch.randint(0, S, (S, V), generator=g), torch.tensor(-1))
    nxt[:, 10] = 2
    nxt[2, :] = -1
    nxt[2, 11] = 0                                      # a state with a single way on
    nxt[:, eos] = torch.where(torch.arange(S) % 3 == 0, 0, -1)
    start = torch.randint(0, S, (B,), generator=g)
    grammar = T.Grammar(nxt, start)
    got = [s.tolist() for s in T.InferenceState({'model': model, 'inputs': torch.zeros((B, 1), device='cuda'), 'vocab': vocab, 'max_len': 12,
                                                 'beam_size': beam, 'grammar': grammar, 'frequency_penalty': 0.3}).inference()]
    run = plain_greedy if beam == 1 else (lambda *a, **kw: plain_beam(*a[:4], beam, *a[4:], **kw))
    seen = {}
    for i in range(B):
        s = int(start[i])
        if s not in seen:
            seen[s] = run(table, [bos], eos, 12, dict(freq=0.3), grammar=nxt, state=s)
        assert got[i] == seen[s], i
    assert len(seen) == min(S, len(set(start.tolist())))


@pytest.mark.parametrize('kind', ['transformer', 'rnnlm', 'lm_bf16', 'lm_4bit'])
def test_rules_on_the_packages_own_models(T, kind):
    """The token of every step is the best of the plainly adjusted logits of that step (histories from the results)."""
    from tst_amd import synthetic
    V2 = 203
    vocab = T.Vocab.synthetic(V2)
    B, extra = 12, {}
    g = torch.Generator().manual_seed(3)
    if kind == 'transformer':
        hp = dict(d_model=64, dropout=0.1, n_layers=2, pe_max_len=60, n_heads=2, d_ff=128)
        m = T.Transformer(T.HP(hp), vocab, vocab)
        m.load_state_dict(synthetic.synthetic_state_dict(m, 3, 1.0, 2.0, seed=4))
        model, inputs = m.decoder, torch.randn((B, 9, 64), generator=g).cuda()
    elif kind == 'rnnlm':
        model = T.RNNLM(64, vocab, 2)
        model.load_state_dict(synthetic.synthetic_state_dict(model, 3, 1.0, 2.0, seed=5))
        inputs, extra = torch.randn((2, B, 64), generator=g).cuda(), {'substitute_inputs': True, 'inputs_batch_dim': 1, 'kwargs': {'return_z': True}}
    else:
        model, vocab = make_lm(T, 'bf16', V=V2)
        inputs = torch.randn((B, 128), generator=g).cuda() * 0.1
        extra = {'kv_cache': 'fp4'} if kind == 'lm_4bit' else {}
    bias = torch.randn(V2, generator=g)
    st = T.InferenceState({'model': model, 'inputs': inputs, 'vocab': vocab, 'max_len': 10, 'return_logits': True, 'repetition_penalty': 1.5,
                           'frequency_penalty': 0.7, 'logit_bias': bias, **extra})
    out = [s.tolist() for s in st.inference()]
    bos, eos = vocab.stoi['<bos>'], vocab.stoi['<eos>']
    for t, (lg, sent) in enumerate(st.step_logits):
        low = lg.dtype == torch.bfloat16
        for r, s in enumerate(sent.tolist()):
            gen = out[s][1:1 + t]
            if len(gen) < t:
                continue
            y = plain_rules(lg[r].float().cpu(), V2, [bos], gen, 1.5, 0.7, 0.0, bias)
            y = y.to(lg.dtype).float() if low else y
            want = int((y == y.max()).nonzero()[0])
            assert want == (out[s][1 + t] if len(out[s]) > 1 + t else eos), (t, s)


def test_default_calls_are_what_they_were(T):
    """Neutral rules change nothing: same tokens as without them, and no rule object in the loop."""
    lm, vocab = make_lm(T, 'fp32')
    z = torch.randn((7, 128), generator=torch.Generator().manual_seed(8)).cuda() * 0.1
    args = {'model': lm, 'inputs': z, 'vocab': vocab, 'max_len': 9}
    a = T.InferenceState(dict(args))
    b = T.InferenceState(dict(args, repetition_penalty=1.0, frequency_penalty=0.0, presence_penalty=0))
    assert [s.tolist() for s in a.inference()] == [s.tolist() for s in b.inference()] and a.loop.rules is None and b.loop.rules is None


@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
def test_fewer_rows_of_long_contexts(T, dtype):
    """A batch whose long contexts stay whole with all rows and are cut over workgroups once few are left."""
    from tst_amd import kernels as K
    lm, vocab = make_lm(T, dtype, d=128, heads=4, layers=1, pe_max_len=1500)
    lens = [1400, 3] + [20] * 30
    prompts = ragged(203, lens, 8)
    z = torch.randn((32, 128), generator=torch.Generator().manual_seed(6)).cuda() * 0.1
    sess = lm.paged_session(z, prompts, 2)
    rows = K.RowState(32, 2, torch.device('cuda', 0), False, 0)
    rows.sent.copy_(torch.arange(32, dtype=torch.int32))
    rows.tok.copy_(torch.stack([p[-1] for p in prompts]))
    every = sess.step(rows, 32, 0)[:32, :203].clone()
    for n in (5, 2, 1):
        assert_logits(sess.step(rows, n, 0)[:n, :203], every[:n], dtype)


def test_paged_session_refusals(T):
    lm, vocab = make_lm(T, 'fp32', layers=1, pe_max_len=50)
    z = torch.zeros((2, 128), device='cuda')
    ok = ragged(203, [5, 7], 1)
    for args, why in [((z[:0], [], 3), 'at least one prompt'), ((z, ok, 0), 'max_new'), ((z, ok[:1], 3), 'conditioning vectors'), ((z[:, :64], ok, 3), 'model_size'),
                      ((z, [ok[0], ok[1][:0]], 3), 'at least 1'), ((z, [ok[0], ok[1].float()], 3), '1-D tensor'), ((z, [ok[0], ok[1].view(1, -1)], 3), '1-D tensor'),
                      ((z, ragged(203, [5, 49], 1), 3), 'positions exceed'), ((z, ok, 3, 24), 'page')]:
        with pytest.raises(ValueError, match=why):
            lm.paged_session(*args)
    with pytest.raises(IndexError):
        lm.paged_session(z, [ok[0], torch.tensor([1, 203])], 3)
    lm.paged_session(z, ragged(203, [5, 48], 1), 3)                              # 48 + 3 - 1 positions
    with pytest.raises(ValueError, match='head size'):
        make_lm(T, 'fp32', d=96, heads=2, layers=1)[0].paged_session(z[:, :96].contiguous(), ok, 3)
