"""CPU: sizes near the end of 32 bits that the kernels' counters cannot walk are refused (nothing here touches a GPU)."""
import pytest

from tst_amd import _lib

TOP = 0x7fffffff


def cache():
    return _lib.TstCache4(kc=16, ks=16, vc=16, vs=16, pages=4, page=32, kv_heads=2, dh=64, reserved=0)


@pytest.mark.parametrize('ty', ['f32', 'bf16'])
def test_attention_over_contexts_near_two_to_the_31(ty):
    """Positions are counted in steps of up to 512 tokens: behind the last step the counter has to fit, or the loop would not end."""
    def call(max_len):
        _lib.call('tst_attn_cache4_' + ty, cache(), 16, 256, 16, TOP, 3, None, 16, max_len, 16, 256, 0, 4, 0.1, 16, 0, None)
    for n in (TOP, TOP - 511, TOP - 1023):
        with pytest.raises(_lib.TstError, match='max_len exceeds'):
            call(n)
        assert _lib._dll.tst_attn_cache4_work(1, 4, 2, 64, n) == -1
    call(TOP - 1024)                        # no rows: nothing is launched
    assert _lib._dll.tst_attn_cache4_work(1, 4, 2, 64, TOP - 1024) > 0


@pytest.mark.parametrize('ty', ['f32', 'bf16'])
def test_rules_on_rows_near_two_to_the_31(ty):
    """Columns are counted in chunks of up to 8192 from up to 7 in front of the row."""
    def call(V):
        _lib.call('tst_adjust_logits_' + ty, 16, TOP, 0, V, _lib.TstLogitRules(), 16, TOP, None)
    for V in (TOP, TOP - 8191, TOP - 16383):
        with pytest.raises(_lib.TstError, match='columns exceed'):
            call(V)
    call(TOP - 16384)


def test_scratch_of_calls_that_would_be_refused():
    """rows * heads of a call fit 31 bits; beyond, the product of the scratch rule would not fit 64."""
    f = _lib._dll.tst_attn_cache4_work
    assert f(TOP, 4096, 1, 256, 1 << 30) == -1 and f(TOP, TOP, TOP, 256, 1 << 30) == -1 and f(1 << 20, 4096, 1, 256, 1 << 30) == -1
    assert f((1 << 19) - 1, 4096, 1, 256, 1 << 30) > 0 and f(TOP, 1, 1, 32, 100) == 0 and f(TOP, 1, 1, 32, 1 << 30) > 0
