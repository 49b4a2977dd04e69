"""CPU: a paged step behind the end that its session was made for is refused (nothing here touches a GPU)."""
import pytest

from tst_amd import _lib
from tst_amd.lm import PagedLMSession


def run(t, max_len=40, n_seq=3, rows=2):
    layers = (_lib.TstTfmLayer * 1)()
    for f in ('wqkv', 'wo', 'w1', 'w2'):
        setattr(layers[0], f, 16)
    caches = (_lib.TstCache4 * 1)(_lib.TstCache4(kc=16, ks=16, vc=16, vs=16, pages=4, page=32, kv_heads=2, dh=32, reserved=0))
    step = _lib.TstTfmStep(n_layers=1, d=64, heads=2, d_ff=128, V=10, n_pos=50, slab_rows=3, layers=layers, x=16, h=16, a=16, ff=16, logits=16, emb=16, pe=16,
                           wout=16)
    plan = _lib.TstPagedStep(step=_lib.ctypes.pointer(step), caches=caches, table=16, width=2, n_seq=n_seq, base=16, slots=16, pos=16, lens=16, qkv=16,
                             max_len=max_len)
    _lib.call('tst_paged_step_run', plan, 16, 16, rows, t, None)


def test_steps_behind_max_len_are_refused():
    for t in (40, 41, 50, 1 << 30):
        with pytest.raises(_lib.TstError, match='outside 0 .. max_len'):
            run(t, rows=0)
    with pytest.raises(_lib.TstError, match='outside 0 .. max_len'):
        run(1, max_len=1, rows=0)
    with pytest.raises(_lib.TstError, match='max_len'):
        run(0, n_seq=-1, rows=0)
    run(39, rows=0)                       # the last step; no rows, so nothing is launched


def test_a_session_refuses_steps_behind_its_new_tokens():
    s = object.__new__(PagedLMSession)
    s.max_new, s.logits = 3, None

    class Plan:
        def run(self, rows, n, t):
            self.t = t
    s.plan = Plan()
    for t in (-1, 3, 100):
        with pytest.raises(ValueError, match='made for 3 new tokens'):
            s.step(None, 1, t)
    s.step(None, 1, 2)
    assert s.plan.t == 2


def test_a_paged_step_on_another_device_is_refused(monkeypatch):
    """Like the wrappers: the kernels run on the current device, so the session has to live there."""
    import torch
    from tst_amd import kernels as K
    plan = object.__new__(K.PagedPlan)
    plan.dev = 1
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: 0)
    with pytest.raises(ValueError, match='the session is on cuda:1, the current device is cuda:0'):
        plan.run(None, 1, 0)
