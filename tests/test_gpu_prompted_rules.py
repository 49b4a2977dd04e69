"""GPU: rules on logits where a row has nothing left to pick, and together with the soft mode, end to end."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

V = 97


@pytest.fixture(scope='module')
def T():
    import tst_amd
    assert torch.cuda.is_available()
    return tst_amd


class Walk:
    """A foreign model whose logits depend on the step only: rows of a table, -inf where it says so."""

    def __init__(self, rows):
        self.rows = rows.cuda()

    def __call__(self, inputs, active_seqs, *args, **kw):
        return self.rows[active_seqs.shape[1] - 1].expand(active_seqs.shape[0], 1, -1)


@pytest.mark.parametrize('B', [2, 2500])
def test_a_row_that_the_model_leaves_nothing_stays_under_its_grammar(T, B):
    """State 0 allows 10 and 11.  At step 1 the model itself gives both -inf: whatever is picked there, the steps behind it follow state 0."""
    vocab = T.Vocab.synthetic(V)
    rows = torch.randn((6, V), generator=torch.Generator().manual_seed(4))
    rows[1, 10:12] = -math.inf
    rows[:, 40] = 9.0                                   # what the model likes best is never allowed
    nxt = torch.full((1, V), -1)
    nxt[0, 10:12] = 0
    st = T.InferenceState({'model': Walk(rows), 'inputs': torch.zeros((B, 1), device='cuda'), 'vocab': vocab, 'max_len': 5,
                           'grammar': T.Grammar(nxt)})
    for s in st.inference():
        got = s.tolist()
        assert len(got) == 6 and all(v in (10, 11) for t, v in enumerate(got[1:]) if t != 1), got
        assert [got[1 + t] for t in (0, 2, 3, 4)] == [10 + int(rows[t, 10:12].argmax()) for t in (0, 2, 3, 4)]


def test_gumbel_with_neutral_rules_runs_and_with_rules_is_refused(T):
    vocab = T.Vocab.synthetic(V)
    model = Walk(torch.randn((6, V), generator=torch.Generator().manual_seed(4)))
    args = {'model': model, 'inputs': torch.zeros((3, 1), device='cuda'), 'vocab': vocab, 'max_len': 1, 'gumbel': True}
    torch.manual_seed(5)
    a = T.InferenceState(dict(args)).inference()
    torch.manual_seed(5)
    b = T.InferenceState(dict(args, repetition_penalty=1.0)).inference()
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    with pytest.raises(NotImplementedError, match='gumbel'):
        T.InferenceState(dict(args, allowed_tokens=torch.arange(V) < 50)).inference()


@pytest.mark.parametrize('kind,beam', [(k, b) for k in ('transformer', 'rnnlm', 'lm_fp32', 'lm_bf16') for b in (1, 4)] + [('lm_4bit', 1)])
def test_rules_that_change_no_logit_change_no_result(T, kind, beam):
    """With rules the selection reads the whole rows of logits instead of what a model's own projection left for it: the same results."""
    from tst_amd import synthetic
    vocab, B, extra = T.Vocab.synthetic(1203), 600, {}
    g = torch.Generator().manual_seed(3)
    if kind == 'transformer':
        m = T.Transformer(T.HP(dict(d_model=64, dropout=0.1, n_layers=2, pe_max_len=60, n_heads=2, d_ff=128)), vocab, vocab)
        model, x = m.decoder, torch.randn((B, 9, 64), generator=g).cuda()
    elif kind == 'rnnlm':
        m = model = T.RNNLM(64, vocab, 2)
        x, extra = torch.randn((2, B, 64), generator=g).cuda(), {'substitute_inputs': True, 'inputs_batch_dim': 1, 'kwargs': {'return_z': True}}
    else:
        m = model = T.TransformerLM(T.HP(dict(model_size=128, n_layers=2, n_heads=2, d_ff=256, pe_max_len=60)), vocab,
                                    dtype='fp32' if kind == 'lm_fp32' else 'bf16')
        x, extra = torch.randn((B, 128), generator=g).cuda() * 0.1, {'kv_cache': 'fp4'} if kind == 'lm_4bit' else {}
    m.load_state_dict(synthetic.synthetic_state_dict(m, 3, 1.0, 2.0, seed=4))
    args = {'model': model, 'inputs': x, 'vocab': vocab, 'max_len': 10, 'beam_size': beam, **extra}
    tok, n, _ = T.InferenceState(dict(args)).decode_packed()
    for rule in (dict(logit_bias=torch.zeros(1203)), dict(allowed_tokens=torch.ones(B, 1203, dtype=torch.bool)),
                 dict(grammar=T.Grammar(torch.zeros(1, 1203, dtype=torch.int64)))):
        got = T.InferenceState(dict(args, **rule)).decode_packed()
        assert torch.equal(got[0], tok) and torch.equal(got[1], n), list(rule)
