"""CPU: refusals of the prompted-decoding entry points and wrappers, and the host-side helpers (nothing here touches a GPU)."""
import pytest
import torch

from tst_amd import _lib, engine, kernels as K


def cache(**kw):
    return _lib.TstCache4(**dict(dict(kc=16, ks=16, vc=16, vs=16, pages=4, page=32, kv_heads=2, dh=64, reserved=0), **kw))


def refused(match, name, *args):
    with pytest.raises(_lib.TstError, match=match):
        _lib.call(name, *args)


def test_page_plan_refusals():
    ok = [16, 16, 2, 16, 9, 32, 16, 4, 16, 16, 16, 16, 50, 16, None]
    for i, v, why in [(0, None, 'null pointer'), (3, None, 'null pointer'), (6, None, 'null pointer'), (8, None, 'null pointer'), (13, None, 'null pointer'),
                      (2, -1, 'negative'), (4, -1, 'negative'), (7, -1, 'negative'), (12, -1, 'negative'), (5, 0, 'power of two'), (5, 24, 'power of two'),
                      (5, 4, 'power of two'), (5, 2048, 'power of two'), (2, 1 << 31, 'exceeds'), (12, 1 << 31, 'exceeds')]:
        refused(why, 'tst_page_plan', *(ok[:i] + [v] + ok[i + 1:]))
    step = [16, None, 3, 16, 4, 2, 32, 16, 16, 16, 5, None]
    for i, v, why in [(0, None, 'null pointer'), (3, None, 'null pointer'), (7, None, 'null pointer'), (2, -1, 'negative'), (10, -1, 'negative'),
                      (6, 12, 'power of two'), (10, 1 << 31, 'exceeds')]:
        refused(why, 'tst_page_step', *(step[:i] + [v] + step[i + 1:]))


@pytest.mark.parametrize('name,unit', [('tst_attn_prompt_f32', 4), ('tst_attn_prompt_bf16', 8)])
def test_attn_prompt_refusals(name, unit):
    ok = [16, 128, 16, 64, 16, 64, 16, 2, 16, 128, 100, 2, 1, 64, 0.1, None]
    for i, v, why in [(0, None, 'null pointer'), (2, None, 'null pointer'), (4, None, 'null pointer'), (6, None, 'null pointer'), (8, None, 'null pointer'),
                      (1, 120, 'hold the heads'), (1, 129, 'hold the heads'), (3, 56, 'hold the heads'), (5, 66, 'hold the heads'), (9, 120, 'hold the heads'),
                      (11, 3, 'hold the heads'), (12, 0, 'multiple of kv_heads'), (11, 0, 'multiple of kv_heads'), (13, unit - 1, 'head size'),
                      (13, 0, 'head size'), (13, 264, 'head size'), (10, -1, 'negative'), (7, -1, 'negative'), (10, 1 << 31, 'exceeds'), (0, 24, '16-byte'),
                      (8, 20, '16-byte'), (3, (1 << 22) + 64, 'exceeds 2.22'), (5, (1 << 22) + 64, 'exceeds 2.22'), (14, float('nan'), 'not finite'),
                      (14, float('inf'), 'not finite')]:
        refused(why, name, *(ok[:i] + [v] + ok[i + 1:]))
    refused('multiple of kv_heads', name, *(ok[:11] + [3, 2] + ok[13:]))
    refused('too many', name, *(ok[:1] + [4096 * 8] + ok[2:3] + [4096 * 8] + ok[4:5] + [4096 * 8] + ok[6:9] + [4096 * 8, 1 << 30, 4096, 4096, 8, 0.1, None]))


@pytest.mark.parametrize('ty', ['f32', 'bf16'])
def test_cache_refusals(ty):
    rows = [16, 128, 16, 128, 16, 10, None]
    for bad, why in [(dict(dh=48), 'head size 48'), (dict(dh=512), 'head size'), (dict(page=8), 'page 8'), (dict(page=256), 'page 256'),
                     (dict(kv_heads=0), 'sizes'), (dict(pages=-1), 'sizes'), (dict(pages=1 << 27), 'sizes'), (dict(pages=1 << 40), 'exceeds'),
                     (dict(kc=None), 'null cache array'), (dict(vs=None), 'null cache array'), (dict(vc=24), '16-byte')]:
        refused(why, 'tst_cache4_write_' + ty, cache(**bad), *rows)
        refused(why, 'tst_cache4_read_' + ty, cache(**bad), 16, 16, 128, 16, 128, 10, None)
        refused(why, 'tst_attn_cache4_' + ty, cache(**bad), 16, 128, 16, 4, 3, None, 16, 100, 16, 128, 3, 2, 0.1, None, 0, None)
    refused('null cache', 'tst_cache4_write_' + ty, None, *rows)
    for i, v, why in [(0, None, 'null pointer'), (2, None, 'null pointer'), (4, None, 'null pointer'), (1, 120, 'kv_heads'), (3, 129, 'kv_heads'),
                      (5, -1, 'negative'), (5, 1 << 31, 'exceeds'), (0, 8, '16-byte')]:
        refused(why, 'tst_cache4_write_' + ty, cache(), *(rows[:i] + [v] + rows[i + 1:]))
    att = [16, 256, 16, 4, 3, None, 16, 100, 16, 256, 3, 4, 0.1, None, 0, None]
    for i, v, why in [(0, None, 'null pointer'), (2, None, 'null pointer'), (6, None, 'null pointer'), (8, None, 'null pointer'), (1, 250, 'hold heads'),
                      (9, 128, 'hold heads'), (11, 3, 'multiple of kv_heads'), (11, 0, 'multiple of kv_heads'), (10, -1, 'negative'), (7, -1, 'negative'),
                      (3, -1, 'negative'), (4, -1, 'negative'), (10, 1 << 31, 'exceeds'), (7, 1 << 31, 'exceeds'), (0, 8, '16-byte'), (13, 8, '16-byte'),
                      (7, 100000, 'are needed'), (12, float('nan'), 'not finite'), (12, float('-inf'), 'not finite')]:
        refused(why, 'tst_attn_cache4_' + ty, cache(), *(att[:i] + [v] + att[i + 1:]))


def test_attn_cache4_work_is_a_pure_size_rule():
    f = _lib._dll.tst_attn_cache4_work
    assert f(3, 4, 2, 64, 100) == 0 and f(0, 4, 2, 64, 100000) == 0 and f(1, 4, 2, 64, 100000) > 0
    for bad in [(-1, 4, 2, 64, 1), (1, 0, 2, 64, 1), (1, 4, 0, 64, 1), (1, 4, 3, 64, 1), (1, 4, 2, 0, 1), (1, 4, 2, 64, -1), (1 << 31, 4, 2, 64, 1)]:
        assert f(*bad) == -1
    with pytest.raises(ValueError, match='bad sizes'):
        K.attn_cache4_work(1, 4, 3, 64, 1)


def test_attn_cache4_work_covers_fewer_rows_and_tokens():
    """What a call asks for (its refusal says so) never exceeds what the size rule gives for at least as many rows and tokens."""
    import random
    rng, f = random.Random(3), _lib._dll.tst_attn_cache4_work

    def wanted(r, heads, kv, dh, n):
        with pytest.raises(_lib.TstError, match='are needed|not finite') as e:        # the scale is looked at after the scratch
            _lib.call('tst_attn_cache4_f32', cache(kv_heads=kv, dh=dh), 16, heads * dh, 16, 4, 3, None, 16, n, 16, heads * dh, r, heads, float('nan'), None, 0,
                      None)
        text = str(e.value)
        return int(text.split('floats, ')[1].split()[0]) if 'are needed' in text else 0

    cut = 0
    for _ in range(3000):
        kv, dh = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([32, 64, 128, 256])
        heads = kv * rng.choice([1, 2, 4, 16, 17, 40])
        R, n = int(2 ** rng.uniform(0, 11)), int(2 ** rng.uniform(0, 18))
        most = f(R, heads, kv, dh, n)
        for r in {1, min(2, R), R, max(1, R // 2), rng.randint(1, R), min(R, max(1, 128 // kv)), min(R, max(1, 255 // kv)), min(R, max(1, 511 // kv))}:
            for m in {n, rng.randint(1, n), max(1, n // 2), min(n, 1025), min(n, 2049), min(n, 4097), min(n, 8193)}:
                need = wanted(r, heads, kv, dh, m)
                cut += need > 0
                assert need <= most, (r, R, heads, kv, dh, m, n)
    assert cut > 1000


@pytest.mark.parametrize('ty', ['f32', 'bf16'])
def test_adjust_logits_refusals(ty):
    R = _lib.TstLogitRules

    def call(rules, logits=16, ld=100, n=3, V=100, out=16, ldo=100):
        _lib.call('tst_adjust_logits_' + ty, logits, ld, n, V, rules, out, ldo, None)
    for kw, why in [(dict(rules=None), 'null rules'), (dict(logits=None), 'null pointer'), (dict(out=None), 'null pointer'), (dict(ld=99), 'hold V'),
                    (dict(ldo=99), 'hold V'), (dict(n=-1), 'negative'), (dict(V=-1), 'negative'), (dict(n=1 << 31), 'exceeds'), (dict(ldo=108), 'in place'),
                    (dict(rules=R(hist=16, ld_hist=4, n_hist=4)), 'need params'), (dict(rules=R(prompt=16, prompt_cu=16)), 'need params'),
                    (dict(rules=R(params=16, n_sent=3, prompt=16)), 'prompt_cu'), (dict(rules=R(params=16, n_sent=2)), 'must hold 3 rows'),
                    (dict(rules=R(params=16, n_sent=3, hist=16, ld_hist=3, n_hist=4)), 'ld_hist'), (dict(rules=R(bias=16, n_bias=1, ld_bias=99)), 'ld_bias'),
                    (dict(rules=R(mask=16, n_masks=1, ld_mask=3)), 'ld_mask'), (dict(rules=R(n_bias=-1)), 'negative'), (dict(rules=R(n_hist=1 << 31)), 'exceeds')]:
        with pytest.raises(_lib.TstError, match=why):
            call(**dict(dict(rules=R()), **kw))
    refused('null pointer', 'tst_grammar_next', None, 3, 10, 16, 4, None, 16, 32, 4, None)
    refused('out must not be state', 'tst_grammar_next', 16, 3, 10, 16, 4, None, 16, 16, 4, None)
    refused('negative', 'tst_grammar_next', 16, -3, 10, 16, 4, None, 16, 32, 4, None)


def test_paged_step_refusals():
    layers = (_lib.TstTfmLayer * 1)()
    for f in ('wqkv', 'wo', 'w1', 'w2'):
        setattr(layers[0], f, 16)
    caches = (_lib.TstCache4 * 1)(cache(kv_heads=2, dh=32))
    step = dict(n_layers=1, d=64, heads=2, d_ff=128, V=10, n_pos=50, slab_rows=3, layers=layers, x=16, h=16, a=16, ff=16, logits=16, emb=16, pe=16, wout=16)
    plan = dict(caches=caches, table=16, width=2, n_seq=3, base=16, slots=16, pos=16, lens=16, qkv=16, max_len=40)

    def call(s={}, p={}, n=2, t=0, sent=16):
        st = _lib.TstTfmStep(**dict(step, **s))
        _lib.call('tst_paged_step_run', _lib.TstPagedStep(step=_lib.ctypes.pointer(st), **dict(plan, **p)), 16, sent, n, t, None)
    refused('null plan', 'tst_paged_step_run', None, 16, 16, 1, 0, None)
    for kw, why in [(dict(n=4), 'buffers hold 3'), (dict(t=-1), 'max_len'), (dict(p=dict(max_len=51)), 'max_len'), (dict(p=dict(max_len=0)), 'max_len'),
                    (dict(p=dict(qkv=None)), 'work buffer'), (dict(s=dict(logits=None)), 'work buffer'), (dict(p=dict(base=None)), 'null input'),
                    (dict(s=dict(wout=None)), 'null input'), (dict(s=dict(z=16), sent=None), 'z without sent'), (dict(s=dict(heads=3)), 'sizes'),
                    (dict(p=dict(caches=(_lib.TstCache4 * 1)(cache(kv_heads=2, dh=64)))), 'does not fit')]:
        with pytest.raises(_lib.TstError, match=why):
            call(**kw)


def test_wrappers_refuse_cpu_tensors_and_bad_shapes():
    f, i = torch.zeros(4, 64), torch.zeros(4, dtype=torch.int32)
    with pytest.raises((ValueError, RuntimeError)):
        K.attn_prompt(f, f, f, i, f.clone(), 1)
    for kw in (dict(head_size=48), dict(page=24), dict(kv_heads=0), dict(pages=-1), dict(pages=1 << 26, page=64)):
        with pytest.raises(ValueError):
            K.Cache4(**dict(dict(pages=2, page=32, kv_heads=1, head_size=64, device='cpu'), **kw))
    with pytest.raises(ValueError, match='on the GPU'):
        K.Cache4(2, 32, 1, 64, device='cpu')


def test_grammar_and_masks_on_the_host():
    bits = engine.pack_mask(torch.tensor([[True] * 33, [False] * 32 + [True], [i % 2 == 0 for i in range(33)]]))
    assert bits.dtype == torch.int32 and (bits.to(torch.int64) & 0xffffffff).tolist() == [[0xffffffff, 1], [0, 1], [0x55555555, 1]]
    with pytest.raises(ValueError, match='state 1 allows no token'):
        engine.Grammar([[0, 1], [-1, -1]])
    with pytest.raises(ValueError, match='outside'):
        engine.Grammar([[0, 2]])
    with pytest.raises(ValueError, match='integers'):
        engine.Grammar(torch.zeros(2, 2))
    g = engine.Grammar([[0, 1], [1, -1]], start=[0, 1])
    with pytest.raises(ValueError, match='vocabulary 3'):
        g.on('cpu', 2, 3)
    with pytest.raises(ValueError, match='start'):
        g.on('cpu', 3, 2)
    with pytest.raises(ValueError, match='start'):
        engine.Grammar([[0, 0]], start=1).on('cpu', 1, 2)
    table, mask, start = g.on('cpu', 2, 2)
    assert mask.tolist() == [[3], [1]] and start.tolist() == [0, 1]


@pytest.mark.parametrize('kw,why', [
    (dict(repetition_penalty=0.0), 'repetition_penalty'), (dict(repetition_penalty=float('nan')), 'repetition_penalty'),
    (dict(frequency_penalty=[1.0]), 'frequency_penalty'), (dict(presence_penalty=float('inf')), 'presence_penalty'),
    (dict(logit_bias=torch.zeros(4)), 'logit_bias'), (dict(logit_bias=torch.full((5,), float('nan'))), 'logit_bias'),
    (dict(logit_bias=torch.full((5,), float('inf'))), 'logit_bias'), (dict(allowed_tokens=torch.zeros(5, dtype=torch.bool)), 'leaves a sentence'),
    (dict(allowed_tokens=torch.ones(5)), 'boolean'), (dict(allowed_tokens=torch.ones(3, 5, dtype=torch.bool)), 'boolean'),
    (dict(allowed_tokens=torch.ones(5, dtype=torch.bool), grammar=1), 'grammar')])
def test_rules_are_checked_before_anything_runs(kw, why):
    with pytest.raises(ValueError, match=why):
        engine.LogitRules(5, 2, 1, 'cpu', **kw)
    with pytest.raises(IndexError):
        engine.LogitRules(5, 2, 1, 'cpu', logit_bias={5: 1.0})


def test_neutral_rules_are_inactive_and_prompts_are_packed():
    assert not engine.LogitRules(5, 2, 1, 'cpu', prompts=[[1], [2, 3]]).active
    r = engine.LogitRules(5, 2, 1, 'cpu', repetition_penalty=[1.0, 2.0], prompts=[[1], [2, 3]])
    assert r.active and r.prompt.tolist() == [1, 2, 3] and r.prompt_cu.tolist() == [0, 1, 3]
    assert r.params.tolist() == [[1.0, 0.0, 0.0], [2.0, 0.0, 0.0]]
    assert engine.LogitRules(5, 2, 1, 'cpu', frequency_penalty=1.0, prompts=[[1], [2]]).prompt is None


class _NoModel:
    pass


def test_inference_state_refusals():
    import tst_amd as T
    vocab = T.Vocab.synthetic(20)
    base = {'model': _NoModel(), 'inputs': torch.zeros(2, 4), 'vocab': vocab}
    for kw, err in [(dict(kv_cache='int3'), ValueError), (dict(kv_cache='fp4'), NotImplementedError),
                    (dict(active_seqs=[torch.tensor([1]), torch.tensor([1, 2])]), NotImplementedError)]:
        with pytest.raises(err):
            T.InferenceState(dict(base, **kw)).inference()

    class Paged(_NoModel):
        paged_session = None
    for kw, err in [(dict(beam_size=2), NotImplementedError), (dict(gumbel=True), NotImplementedError), (dict(active_seqs=[torch.tensor([1])]), ValueError),
                    (dict(active_seqs=[torch.tensor([1]), torch.tensor([], dtype=torch.long)]), ValueError),
                    (dict(active_seqs=[torch.tensor([1]), torch.tensor([20])]), IndexError),
                    (dict(active_seqs=[torch.tensor([1]), torch.tensor([1.0])]), ValueError)]:
        with pytest.raises(err):
            T.InferenceState(dict(base, model=Paged(), kv_cache='fp4', **kw)).inference()
