"""GPU: rows of a paged step that stand behind the end, or belong to no sentence, touch nothing."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
def test_rows_behind_the_end_or_of_no_sentence_store_and_read_nothing(dtype):
    import tst_amd as T
    from tst_amd import kernels as K, synthetic
    vocab = T.Vocab.synthetic(203)
    lm = T.TransformerLM(T.HP(dict(model_size=64, n_layers=2, n_heads=2, d_ff=128, pe_max_len=42)), vocab, dtype=dtype)
    lm.load_state_dict(synthetic.synthetic_state_dict(lm, 3, 1.0, 2.0, seed=1))
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(4, 203, (n,), generator=g) for n in (40, 1, 9)]
    z = torch.randn((3, 64), generator=g).cuda() * 0.1
    sess = lm.paged_session(z, prompts, 3, page=16)
    assert sess.max_len == 42                                                    # the positional table ends there
    rows = K.RowState(3, 3, torch.device('cuda', 0), False, 0)
    rows.tok.copy_(torch.tensor([7, 8, 9], dtype=torch.int32))

    def step(sent, t):
        rows.sent.copy_(torch.tensor(sent, dtype=torch.int32))
        sess.plan.run(rows, 3, t)
        return sess.logits[:3, :203].clone()
    held = [[x.clone() for x in (c.kc, c.ks, c.vc, c.vs)] for c in sess.caches]
    out = step([0, 0, 0], 3)                                                     # 39 + 3 = 42: one position too many
    assert sess.plan.pos.tolist() == [0] * 3 and sess.plan.lens.tolist() == [0] * 3 and sess.plan.slots.tolist() == [-1] * 3
    assert bool(torch.isfinite(out).all())
    out = step([3, -1, 1 << 30], 0)
    assert sess.plan.pos.tolist() == [0] * 3 and sess.plan.lens.tolist() == [0] * 3 and sess.plan.slots.tolist() == [-1] * 3
    assert bool(torch.isfinite(out).all())
    for c, kept in zip(sess.caches, held):
        assert all(torch.equal(a, b) for a, b in zip((c.kc, c.ks, c.vc, c.vs), kept))
    # beside such rows the others get what they get alone
    mixed = step([0, 1, 5], 4)[1]
    assert sess.plan.pos.tolist() == [0, 4, 0] and sess.plan.lens.tolist() == [0, 5, 0]
    assert bool(torch.isfinite(mixed).all()) and torch.equal(mixed, step([5, 1, 0], 4)[1])
    with pytest.raises(ValueError, match='made for 3 new tokens'):
        sess.step(rows, 3, 3)
