"""Dimensions that the kernels' int32 counts do not hold are refused, not cut off."""
import numpy as np
import pytest

from tests.test_decoder_refusals import cache_inputs, info, refused
from tfjs_b200.kernels import decoder

BIG = (1 << 32) + 5          # as int32: 5


@pytest.mark.parametrize("change", [
    dict(kCache=info([BIG, 1, 1, 1]), vCache=info([BIG, 1, 1, 1])),
    dict(pageTable=info([3, BIG], "int32")), dict(lengths=info([BIG], "int32")),
])
def test_caches(change):
    refused(decoder._paged_attention, dict(cache_inputs(), q=info([3, 4, 1, 64]), **change), {}, "2^31")


def test_tokens_and_heads():
    new = [3, 2, BIG, 64]
    refused(decoder._paged_cache_append, dict(cache_inputs(), k=info(new), v=info(new)), {}, "2^31")
    refused(decoder._paged_attention, dict(cache_inputs(), q=info([3, BIG + 1, 1, 64])), {}, "2^31")
    for shape in ([1, 1, BIG, 1], [BIG, 1, 1, 1], [1, BIG, 1, 1]):
        inp = {n: info(shape) for n in "qkv"}
        refused(decoder._linear_attention, dict(inp, logDecay=info([shape[1]])), {}, "2^31")
    assert np.int32(np.int64(BIG) & 0xffffffff) == 5


@pytest.mark.parametrize("attrs", [dict(budget=7.5), dict(budget=8, recent=2.5), dict(budget=float("inf")),
                                   dict(budget=float("nan"))])
def test_budgets_are_whole_numbers(attrs):
    inp = dict(cache_inputs(), weights=info([3, 2, 64]))
    with pytest.raises((ValueError, OverflowError)):
        decoder._paged_cache_evict({"inputs": inp, "attrs": attrs, "backend": None})
