"""What the operators of a decoder's memory refuse, before anything is allocated or launched:
a stand-in for the backend fails the test on any call."""
import ctypes

import numpy as np
import pytest

from tfjs_b200 import _cabi
from tfjs_b200.backend import CudaBackend, DataId, TensorInfo
from tfjs_b200.kernels import decoder
from tests import decoder_cases as dc


class Untouched(object):
    def __getattr__(self, name):
        raise AssertionError("the backend was asked for %s" % name)


def info(shape, dtype="float32"):
    return TensorInfo(DataId(), shape, dtype)


def cache_inputs():
    return {"kCache": info([9, 2, 16, 64]), "vCache": info([9, 2, 16, 64]),
            "pageTable": info([3, 4], "int32"), "lengths": info([3], "int32")}


def refused(kernel, inputs, attrs=None, word=""):
    with pytest.raises(ValueError) as e:
        kernel({"inputs": inputs, "attrs": attrs or {}, "backend": Untouched()})
    assert word in str(e.value), str(e.value)


APPEND = dict(k=[3, 2, 5, 64], v=[3, 2, 5, 64])


@pytest.mark.parametrize("change,word", [
    (dict(kCache=info([9, 2, 16])), "kCache"),
    (dict(kCache=info([9, 2, 16, 64], "int32")), "kCache"),
    (dict(vCache=info([9, 2, 16, 32])), "vCache"),
    (dict(pageTable=info([4, 4], "int32")), "pageTable"),
    (dict(pageTable=info([3, 4])), "pageTable"),
    (dict(pageTable=info([3, 0], "int32")), "pageTable"),
    (dict(lengths=info([3])), "lengths"),
    (dict(lengths=info([3, 1], "int32")), "lengths"),
    (dict(lengths=info([0], "int32")), "lengths"),
])
def test_a_cache_that_is_none(change, word):
    for kernel, more, attrs in (
            (decoder._paged_cache_append, {n: info(s) for n, s in APPEND.items()}, {}),
            (decoder._paged_attention, {"q": info([3, 4, 1, 64])}, {}),
            (decoder._paged_cache_evict, {"weights": info([3, 2, 64])}, {"budget": 8})):
        refused(kernel, dict(cache_inputs(), **more, **change), attrs, word)


def test_one_pool_for_keys_and_values():
    inp = cache_inputs()
    inp["vCache"] = inp["kCache"]
    refused(decoder._paged_attention, dict(inp, q=info([3, 4, 1, 64])), {}, "same tensor")


@pytest.mark.parametrize("change,word", [
    (dict(k=info([3, 4, 5, 64])), "k must"), (dict(k=info([2, 2, 5, 64])), "k must"),
    (dict(k=info([3, 2, 0, 64])), "k has"), (dict(v=info([3, 2, 4, 64])), "v must"),
    (dict(counts=info([2], "int32")), "counts"), (dict(counts=info([3])), "counts"),
])
def test_append_refusals(change, word):
    inp = dict(cache_inputs(), **{n: info(s) for n, s in APPEND.items()})
    refused(decoder._paged_cache_append, dict(inp, **change), {}, word)


def test_append_of_a_pool_to_itself():
    inp = dict(cache_inputs(), v=info([3, 2, 16, 64]))
    inp["kCache"] = info([3, 2, 16, 64])
    inp["vCache"] = info([3, 2, 16, 64])
    inp["k"] = TensorInfo(inp["kCache"].dataId, [3, 2, 16, 64], "float32")
    refused(decoder._paged_cache_append, inp, {}, "one of the pools")


@pytest.mark.parametrize("change,word", [
    (dict(q=info([3, 4, 2, 64])), "q must"), (dict(q=info([3, 4, 1, 32])), "q must"),
    (dict(q=info([3, 3, 1, 64])), "evenly"), (dict(q=info([3, 1, 1, 64])), "evenly"),
    (dict(mask=info([3, 63])), "mask"), (dict(mask=info([3, 64], "bool")), "mask"),
    (dict(weights=info([3, 4, 64])), "weights"),
])
def test_attention_refusals(change, word):
    refused(decoder._paged_attention, dict(cache_inputs(), q=info([3, 4, 1, 64]), **{
        k: v for k, v in change.items() if k != "q"}) if "q" not in change else
        dict(cache_inputs(), **change), {}, word)


@pytest.mark.parametrize("change,attrs,word", [
    (dict(weights=info([3, 2, 63])), {}, "weights"), (dict(positions=info([3, 2, 64])), {}, "positions"),
    (dict(total=info([2], "int32")), {}, "total"), ({}, dict(budget=0), "budget"),
    ({}, dict(budget=-3), "budget"), ({}, dict(recent=9), "budget"), ({}, dict(recent=-1), "budget"),
])
def test_evict_refusals(change, attrs, word):
    inp = dict(cache_inputs(), weights=info([3, 2, 64]))
    inp.update(change)
    refused(decoder._paged_cache_evict, inp, dict(dict(budget=8, recent=2), **attrs), word)


@pytest.mark.parametrize("change,word", [
    (dict(q=info([2, 3, 64])), "q must"), (dict(q=info([2, 3, 0, 64])), "q has"),
    (dict(k=info([2, 3, 5, 32])), "k must"),
    (dict(v=info([2, 3, 4, 64])), "v must"), (dict(logDecay=info([2])), "logDecay"),
    (dict(state=info([2, 3, 64, 32])), "state"), (dict(lengths=info([2])), "lengths"),
])
def test_linear_refusals(change, word):
    inp = {"q": info([2, 3, 5, 64]), "k": info([2, 3, 5, 64]), "v": info([2, 3, 5, 64]), "logDecay": info([3])}
    refused(decoder._linear_attention, dict(inp, **change), {}, word)


class Foreign(object):
    def __init__(self, shape=(2, 3), typestr="<f4", strides=None, ptr=4096):
        self.__cuda_array_interface__ = {"shape": shape, "typestr": typestr, "strides": strides,
                                         "data": (ptr, False), "version": 2}


@pytest.mark.parametrize("values,shape,dtype", [
    (Foreign(typestr="<f2"), None, None), (Foreign(typestr="<f4"), None, "int32"),
    (Foreign(strides=(4, 8)), None, None), (Foreign(strides=(24, 4)), None, None),
    (Foreign(), [7], None),
])
def test_foreign_memory_refusals(values, shape, dtype):
    backend = CudaBackend.__new__(CudaBackend)       # no context: any call of the library fails
    backend.ctx = None
    with pytest.raises(ValueError):
        backend.createTensorFromGPUData(values, shape, dtype)


def test_null_contexts():
    lib = _cabi.load()
    p, lp = _cabi.PagedParams(), _cabi.LinearAttentionParams()
    assert lib.tfjs_cuda_paged_cache_append(None, ctypes.byref(p), *[0] * 8) == 1
    assert lib.tfjs_cuda_paged_attention(None, ctypes.byref(p), *[0] * 9) == 1
    assert lib.tfjs_cuda_paged_cache_evict(None, ctypes.byref(p), *[0] * 11) == 1
    assert lib.tfjs_cuda_linear_attention(None, ctypes.byref(lp), *[0] * 8) == 1
    out = ctypes.c_int32(5)
    assert lib.tfjs_cuda_from_device(None, None, 0, ctypes.byref(out)) == 1
    assert lib.tfjs_cuda_wait_stream(None, None) == 1 and lib.tfjs_cuda_signal_stream(None, None) == 1


def test_the_references_agree_with_each_other():
    """Eviction at a budget of the whole row, attention over one slot, one token of the
    recurrence: cases whose answers are plain."""
    cache = dc.Cache(1, 2, 8, 4, [6, 1])
    w = np.random.default_rng(1).random((2, 2, cache.capacity)).astype(np.float32)
    ow, op, ol, kept, k, v = dc.evict(cache, w, [6, 1], 6, 0)
    assert np.array_equal(ow[0, :, :6], w[0, :, :6]) and list(ol) == [6, 1] and list(kept[1, 0]) == [0] + [-1] * 5
    q = np.ones((2, 2, 1, 8), np.float32)
    out, _, _, _ = dc.attention(q, cache, [6, 1])
    assert np.allclose(out[1, 0], cache.rows(cache.v, 1, 1)[0])
    one = np.ones((1, 1, 1, 2), np.float32)
    o, s, _, _ = dc.linear(one, one, one, np.zeros(1, np.float32))
    assert np.array_equal(o.ravel(), [2.0, 2.0]) and np.array_equal(s.ravel(), [1.0] * 4)


def test_parameter_structs_match_the_header_and_the_typescript_packers():
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    header = open(os.path.join(root, "include", "tfjs_cuda.h")).read()
    ts = open(os.path.join(root, "tfjs_b200", "ts", "src", "binding.ts")).read()
    for cls, name, size in ((_cabi.PagedParams, "tfjs_cuda_paged_params", 48),
                            (_cabi.LinearAttentionParams, "tfjs_cuda_linear_attention_params", 28)):
        assert ctypes.sizeof(cls) == size and "new ArrayBuffer(%d)" % size in ts
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, header, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = [f for line in re.findall(r"(?:int32_t|float) ([^;]*);", body) for f in re.split(r",\s*", line)]
        assert fields == [f for f, _ in cls._fields_]
        assert "v.setFloat32(%d, scale ?? 1, true)" % cls.scale.offset in ts
