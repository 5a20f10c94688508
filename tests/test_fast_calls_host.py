"""The compiled host path without a GPU: what it is not made for it leaves alone."""

import pytest
import torch

from kohakufa_cute import cache, native


def test_host_tensors_and_wrong_arguments_are_left_to_python():
    if native.fast is None:
        pytest.skip("the optional module is not built")
    native.library()  # binds the module
    q = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16)
    held = cache.QuantizedCache(*(torch.zeros(1, 2, 4, *tail, dtype=t) for tail, t in
                                  (((32,), torch.uint8), ((1, 2), torch.bfloat16)) * 2))
    for call in (lambda f: f.window_attention(q, q, q, 4, 0, 0, None), lambda f: f.window_attention(None, 1, "x", 4, 0, 0, None),
                 lambda f: f.window_attention(), lambda f: f.cache_write(held, q, q, 0, None), lambda f: f.cache_write(q, q, q, 0, None),
                 lambda f: f.cache_read(held, 0, None), lambda f: f.cache_attention(q, held, 0, None, 0, None),
                 lambda f: f.cache_attention(q, (1, 2, 3, 4), 0, None, 0, None)):
        assert call(native.fast) is None
    with pytest.raises(KeyError):
        native.fast.bind({}, native._check)
    with pytest.raises(TypeError):
        native.fast.allow("0")
    import kohakufa_cute

    with pytest.raises(ValueError, match="CUDA"):
        kohakufa_cute.sliding_window_attention(q, q, q, window=4)
