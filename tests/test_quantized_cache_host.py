"""The 4-bit key/value cache, the parts that need no GPU: construction and refusals."""

import pytest
import torch

import kohakufa_cute
from kohakufa_cute import cache as qc


def cpu_cache(**kwargs):
    return kohakufa_cute.quantized_cache(2, 3, 40, 128, device="cpu", **kwargs)


def test_an_empty_cache_has_the_documented_shapes():
    cache = cpu_cache(dtype=torch.float16)
    assert cache.k_codes.shape == cache.v_codes.shape == (2, 3, 40, 64) and cache.k_codes.dtype == torch.uint8
    assert cache.k_params.shape == cache.v_params.shape == (2, 3, 40, 2, 2) and cache.k_params.dtype == torch.float16
    assert all(not t.any() for t in cache)


@pytest.mark.parametrize("arguments", ((0, 1, 1, 64), (1, -1, 1, 64), (1, 1, 1.0, 64), (1, 1, True, 64), (1, 1, 1, 96),
                                       (1, 1, 1, 576)))
def test_bad_sizes_are_refused(arguments):
    with pytest.raises(ValueError, match="quantized_cache"):
        kohakufa_cute.quantized_cache(*arguments, device="cpu")


def test_a_type_other_than_16_bits_is_refused():
    with pytest.raises(ValueError, match="FP16 or BF16"):
        cpu_cache(dtype=torch.float32)


def test_caches_that_are_none_are_refused():
    good = cpu_cache()
    bad = [None, good[:3], (*good[:3], None), good._replace(k_codes=good.k_codes.int()),
           good._replace(v_codes=good.v_codes[:, :, 1:]), good._replace(v_params=good.v_params.half()),
           good._replace(k_params=good.k_params[..., :1]), good._replace(k_codes=good.k_codes[..., :40]), good]
    for cache in bad:  # the last one lives on the CPU
        with pytest.raises(ValueError, match="cache"):
            qc._check_cache("f", cache)


@pytest.mark.parametrize("value", (-1, 2**31, 1.0, True, None, torch.zeros(2, dtype=torch.int64),
                                   torch.zeros(3, dtype=torch.int32)))
def test_bad_positions_are_refused(value):
    with pytest.raises(ValueError, match="f: "):
        qc._positions("f", "start", value, 2, torch.device("cpu"))


def test_gradients_are_refused():
    with pytest.raises(ValueError, match="inference only"):
        qc._no_gradient("f", torch.zeros(1, requires_grad=True))
    with torch.no_grad():
        qc._no_gradient("f", torch.zeros(1, requires_grad=True))


def test_overlaps_are_found_by_their_strides():
    """Against enumeration: what shares memory is found, and ordinary layouts are not suspected."""
    import itertools

    base = torch.zeros(4000)
    for sizes in ((2, 3, 4), (1, 5, 2), (3, 1, 1), (2, 2, 2, 2, 2)):
        for strides in itertools.product((0, 1, 2, 3, 5, 8, 24), repeat=min(len(sizes), 3)):
            strides = strides + tuple(30 * 2**i for i in range(len(sizes) - 3))
            t = base.as_strided(sizes, strides)
            places = {sum(i * s for i, s in zip(at, strides)) for at in itertools.product(*map(range, sizes))}
            if len(places) < t.numel():
                assert qc._may_overlap(t), (sizes, strides)
    whole = torch.zeros(3, 4, 5, 8)
    for t in (whole, whole.transpose(1, 2), whole[1:, ::2, 1:3], whole.permute(3, 1, 0, 2), whole[..., :1], whole[:1].expand(1, 4, 5, 8),
              torch.zeros(1, 4, 5, 8).as_strided((1, 4, 5, 8), (0, 40, 8, 1))):
        assert not qc._may_overlap(t)
    for t in (whole[:1].expand(2, 4, 5, 8), whole.as_strided((2, 4, 5, 8), (20, 40, 8, 1)), whole.as_strided((3, 4), (4, 2))):
        assert qc._may_overlap(t)
