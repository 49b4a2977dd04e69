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
