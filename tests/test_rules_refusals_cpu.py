"""CPU: combinations of logit rules that cannot be kept are refused before anything runs (nothing here touches a GPU)."""
import pytest
import torch

import tst_amd as T
from tst_amd import engine


class _Session:
    """What DecodeLoop asks a session before it allocates anything."""
    needs_anc = False
    takes_soft = True
    incremental = True

    def __init__(self, V):
        self.V = V


V = 20
RULES = {
    'repetition': dict(repetition_penalty=1.2),
    'frequency': dict(frequency_penalty=[0.0, 0.1]),
    'presence': dict(presence_penalty=torch.tensor([0.5, 0.5])),
    'bias': dict(logit_bias={3: -1.0}),
    'mask': dict(allowed_tokens=torch.arange(V) < 10),
    'grammar': dict(grammar=engine.Grammar(torch.zeros(1, V, dtype=torch.int64))),
}


@pytest.mark.parametrize('rule', sorted(RULES))
def test_rules_do_not_combine_with_gumbel(rule):
    """The soft step adds noise after the softmax: a token of probability 0 would keep its noise, so no mask, bias or penalty holds."""
    vocab = T.Vocab.synthetic(V)
    state = {'model': lambda *a: None, 'inputs': torch.zeros(2, 4), 'vocab': vocab, 'gumbel': True}
    with pytest.raises(NotImplementedError, match='gumbel'):
        T.InferenceState(dict(state, **RULES[rule])).inference()
    rules = engine.LogitRules(V, 2, 1, 'cpu', **RULES[rule])
    with pytest.raises(NotImplementedError, match='gumbel'):
        engine.DecodeLoop(_Session(V), 2, 1, 5, 2, 3, 0, device=torch.device('cpu'), gumbel=(1.0, torch.zeros(2, V), None), rules=rules)


def test_neutral_rules_pass_beside_gumbel():
    """Penalties that change nothing are no rules: such a call goes on to ask for its GPU (or runs)."""
    neutral = dict(repetition_penalty=1.0, frequency_penalty=[0.0, 0.0], presence_penalty=0)
    assert not engine.any_rule(2, **neutral) and not engine.any_rule(2)
    assert all(engine.any_rule(2, **r) for r in RULES.values())
    state = {'model': lambda *a: None, 'inputs': torch.zeros(2, 4), 'vocab': T.Vocab.synthetic(V), 'gumbel': True}
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match='needs a GPU'):
            T.InferenceState(dict(state, **neutral)).inference()


INF = float('-inf')


def bias_of(forbidden, n=None):
    """A bias that forbids the given tokens: [V], or [n, V] from a list of n lists."""
    if n is None:
        b = torch.zeros(V)
        b[list(forbidden)] = INF
        return b
    return torch.stack([bias_of(f) for f in forbidden])


def test_biases_that_forbid_every_token_are_refused():
    everything = range(V)
    for b in (bias_of(everything), bias_of([[1], everything], 2), {v: INF for v in everything}, torch.full((V,), torch.finfo(torch.float32).min),
              torch.full((V,), -1e300, dtype=torch.float64)):       # the last two round to -inf, in bf16 and in fp32
        with pytest.raises(ValueError, match='leaves a sentence no token'):
            engine.LogitRules(V, 2, 1, 'cpu', logit_bias=b)
    engine.LogitRules(V, 2, 1, 'cpu', logit_bias=bias_of(range(1, V)))
    engine.LogitRules(V, 2, 1, 'cpu', logit_bias=bias_of([range(1, V), range(V - 1)], 2))


def test_biases_and_masks_that_leave_nothing_together_are_refused():
    one, per = torch.zeros(V, dtype=torch.bool), torch.zeros(2, V, dtype=torch.bool)
    one[[3, 5]] = True
    per[0, 3], per[1, 5] = True, True
    for ok, b in ((one, bias_of([3, 5])), (one, bias_of([[3], [3, 5]], 2)), (per, bias_of([5])), (per, bias_of([[5], [5]], 2))):
        with pytest.raises(ValueError, match='leaves a sentence no token'):
            engine.LogitRules(V, 2, 1, 'cpu', logit_bias=b, allowed_tokens=ok)
    for ok, b in ((one, bias_of([3])), (one, bias_of([[3], [5]], 2)), (per, bias_of([7])), (per, bias_of([[5], [3]], 2))):
        assert engine.LogitRules(V, 2, 1, 'cpu', logit_bias=b, allowed_tokens=ok).active


def chain():
    """State s goes to s + 1 on token 4 + s, state 0 also to 3 on token 10; state 3 allows token 11 and the end."""
    nxt = torch.full((4, V), -1)
    nxt[0, 4], nxt[1, 5], nxt[2, 6], nxt[0, 10], nxt[3, 11], nxt[3, 3] = 1, 2, 3, 3, 3, 2
    return nxt


def test_biases_that_leave_a_state_of_the_grammar_nothing_are_refused():
    for start, b in ((0, bias_of([4, 10])), (0, bias_of([5])), (0, bias_of([6])), (0, bias_of([11, 3])), ([0, 3], bias_of([[5], []], 2)),
                     ([3, 0], bias_of([11, 3]))):
        with pytest.raises(ValueError, match='of the grammar no token'):
            engine.LogitRules(V, 2, 1, 'cpu', logit_bias=b, grammar=engine.Grammar(chain(), start), eos=3)
    # what is never met may be left without a token: states before the start, behind a forbidden token, behind the end
    for start, b in ((0, bias_of([12])), (3, bias_of([4, 10, 5])), ([2, 3], bias_of([5])), (0, bias_of([4, 5, 6])), ([0, 3], bias_of([[], [5]], 2)), (3, bias_of([6])),
                     (0, {4: INF, 5: INF})):
        assert engine.LogitRules(V, 2, 1, 'cpu', logit_bias=b, grammar=engine.Grammar(chain(), start), eos=3).active
    with pytest.raises(ValueError, match='of the grammar no token'):     # without an end token 3 is a token like any other
        engine.LogitRules(V, 2, 1, 'cpu', logit_bias=bias_of([6]), grammar=engine.Grammar(chain(), 3))


def test_a_forbidden_token_leaves_the_grammar_state_where_it_is():
    """Beams and models with logits of -inf can pick a token that the state forbids: the row goes on under that state's rules, not under none."""
    table, mask, start = engine.Grammar(chain(), [0, 2]).on('cpu', 2, V)
    assert table.dtype == torch.int32 and table.is_contiguous()
    want = torch.where(chain() < 0, torch.arange(4).unsqueeze(1), chain())
    assert torch.equal(table.long(), want) and start.tolist() == [0, 2]
    assert torch.equal(mask, engine.pack_mask(chain() >= 0))


def test_rules_for_another_vocabulary_than_the_models_are_refused():
    """Columns behind the rules' vocabulary would pass as they are, forbidden or not."""
    for n in (V - 1, V + 3):
        rules = engine.LogitRules(V, 2, 1, 'cpu', allowed_tokens=torch.arange(V) < 5)
        with pytest.raises(ValueError, match='%d tokens, the model has %d' % (V, n)):
            engine.DecodeLoop(_Session(n), 2, 1, 5, 2, 3, 0, device=torch.device('cpu'), rules=rules)
