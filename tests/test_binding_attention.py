"""The CPython binding's attention side: what it leaves to the Python layer (host code only: CPU
tensors are never launched on)."""
import pytest
import torch

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def mod(pkg):
    from fagq_mi355x import _lib
    if _lib.fast_launch() is None:
        pytest.skip("binding not built")
    return _lib


def test_cpu_tensors_and_odd_arguments_are_left_to_python(pkg, mod):
    b, err = mod._fast_mod, mod.FAST_ARG_ERROR
    q, w = torch.zeros(3, 2, 64, dtype=BF16), torch.zeros(64, dtype=BF16)
    cos, pos = torch.zeros(4, 32), torch.zeros(3, dtype=torch.int64)
    a = [q, q, w, w, cos, cos, pos, 1e-6, False]
    assert b.rope(*a, None, None, 0) == err and b.rope(*a, None, None, None) == err
    assert b.rope_bwd(*a, q, q, None, None, 0) == err
    for i, v in ((0, None), (6, 3), (7, "1"), (8, 1)):
        assert b.rope(*a[:i], v, *a[i + 1:], None, None, 0) == err
    c, s = pkg.empty_kv_cache(2, 2, 16, 64, device="cpu")
    i32 = torch.zeros(1, 2, dtype=torch.int32)
    assert b.cache_write(q, None, pos, c, None, s, None, 0) == err
    assert b.cache_write(q, q, pos, c, None, s, None, 0) == err
    assert b.cache_read(c, None, s, None, i32, i32[0], q, None, 0) == err
    assert b.attention(q[None], c, c, s, s, i32, i32[0, :1], 0.1, None, 0, None, None, 0) == err
    assert b.attention(q[None], c, c, s, s, i32, i32[0, :1], 0.1, None, True, None, None, 0) == err
    for fn, n in ((b.rope, 12), (b.rope_bwd, 14), (b.cache_write, 8), (b.cache_read, 9),
                  (b.attention, 13), (b.bind_attention, 7)):
        with pytest.raises(TypeError):
            fn(*[0] * (n - 1))
    with pytest.raises(ValueError):
        b.bind_attention(*[0] * 7)
