"""What a decoder keeps between tokens: a paged key-value cache (append, attention of one new
token, eviction by accumulated weight) and the state of linear attention with a decay.

The kernels are this backend's own; the reference has no counterpart.  The pools of the
cache are the one thing too large to copy and are updated in place; every other tensor is a
value, as everywhere else.
"""
from ctypes import byref

from .. import _cabi
from ..kernel_registry import KernelConfig
from .common import BACKEND, dev


_MOST = (1 << 31) - 1      # of a dimension: the kernels count in int32


def _want(name, what, info, shape, dtype):
    """`shape` holds sizes, or None where any size goes."""
    got = info.shape
    if info.dtype == dtype:
        if got == shape:
            if 0 not in got:
                return
        elif len(got) == len(shape):
            for w, g in zip(shape, got):
                if g <= 0 or g > _MOST or (w is not None and g != w):
                    break
            else:
                return
    if 0 in got and info.dtype == dtype and len(got) == len(shape) and \
            all(w is None or g == w for w, g in zip(shape, got)):
        raise ValueError("%s: %s has an empty dimension: %s" % (name, what, list(got)))
    if got and max(got) > _MOST:
        raise ValueError("%s: %s has a dimension above 2^31 - 1: %s" % (name, what, list(got)))
    raise ValueError("%s: %s must be %s %s, but got %s %s" %
                     (name, what, dtype, ["any" if w is None else w for w in shape],
                      info.dtype, list(got)))


def _paged(name, inp):
    """Checks the pools, the table and the lengths; the parameters and the rows' capacity."""
    kc, vc, table, lengths = inp["kCache"], inp["vCache"], inp["pageTable"], inp["lengths"]
    _want(name, "kCache", kc, [None] * 4, "float32")
    _want(name, "vCache", vc, kc.shape, "float32")
    if kc.dataId is vc.dataId:
        raise ValueError("%s: kCache and vCache are the same tensor" % name)
    _want(name, "lengths", lengths, [None], "int32")
    batch = lengths.shape[0]
    _want(name, "pageTable", table, [batch, None], "int32")
    num_pages, kv_heads, page_size, head_dim = kc.shape
    max_pages = table.shape[1]
    return _cabi.PagedParams(batch, 0, kv_heads, head_dim, num_pages, page_size, max_pages), \
        max_pages * page_size


def _not_a_pool(name, inp, names):
    for n in names:
        t = inp.get(n)
        if t is not None and (t.dataId is inp["kCache"].dataId or t.dataId is inp["vCache"].dataId):
            raise ValueError("%s: %s is one of the pools" % (name, n))


def _scale(p, scale):
    if scale is not None:
        p.has_scale, p.scale = 1, scale      # (a c_float: rounded to float32 on the way)


def _outputs(backend, shapes, call):
    """Allocates the outputs, makes the call with their device ids, and gives them back;
    nothing is left behind when it fails."""
    outs = []
    try:
        for shape, dtype in shapes:
            outs.append(backend.make_output(shape, dtype))
        backend.check(call([backend.data[o.dataId].dev for o in outs]))
    except Exception:
        for o in outs:
            backend.disposeData(o.dataId)
        raise
    return outs


def _paged_cache_append(args):
    backend, inp = args["backend"], args["inputs"]
    name = "_PagedCacheAppend"
    p, _ = _paged(name, inp)
    k, v, counts = inp["k"], inp["v"], inp.get("counts")
    _want(name, "k", k, [p.batch, p.kv_heads, None, p.head_dim], "float32")
    _want(name, "v", v, k.shape, "float32")
    if counts is not None:
        _want(name, "counts", counts, [p.batch], "int32")
    _not_a_pool(name, inp, ("k", "v"))
    p.tokens = k.shape[2]
    reads = [dev(backend, t) for t in (k, v, inp["pageTable"], inp["lengths"], counts)]
    pools = [backend.device_id_for_update(inp[n].dataId) for n in ("kCache", "vCache")]
    return _outputs(backend, [([p.batch], "int32")],
                    lambda out: backend.lib.tfjs_cuda_paged_cache_append(
                        backend.ctx, byref(p), *pools, *reads, *out))[0]


def _paged_attention(args):
    backend, inp = args["backend"], args["inputs"]
    name = "_PagedAttention"
    p, capacity = _paged(name, inp)
    q, mask, weights = inp["q"], inp.get("mask"), inp.get("weights")
    _want(name, "q", q, [p.batch, None, 1, p.head_dim], "float32")
    p.heads = q.shape[1]
    if p.heads % p.kv_heads:
        raise ValueError("%s: %d query heads do not share %d key-value heads evenly" %
                         (name, p.heads, p.kv_heads))
    if mask is not None:
        _want(name, "mask", mask, [p.batch, capacity], "float32")
    if weights is not None:
        _want(name, "weights", weights, [p.batch, p.kv_heads, capacity], "float32")
    _scale(p, args["attrs"].get("scale"))
    reads = [dev(backend, t) for t in (q, inp["kCache"], inp["vCache"], inp["pageTable"],
                                       inp["lengths"], mask, weights)]
    shapes = [([p.batch, 1, p.heads, p.head_dim], "float32")]
    if weights is not None:
        shapes.append((list(weights.shape), "float32"))
    outs = _outputs(backend, shapes, lambda out: backend.lib.tfjs_cuda_paged_attention(
        backend.ctx, byref(p), *reads, out[0], out[1] if weights is not None else 0))
    return outs if weights is not None else outs[0]


def _paged_cache_evict(args):
    backend, inp, at = args["backend"], args["inputs"], args["attrs"]
    name = "_PagedCacheEvict"
    p, capacity = _paged(name, inp)
    weights, positions, total = inp["weights"], inp.get("positions"), inp.get("total")
    slots = [p.batch, p.kv_heads, capacity]
    _want(name, "weights", weights, slots, "float32")
    if positions is not None:
        _want(name, "positions", positions, slots, "int32")
    if total is not None:
        _want(name, "total", total, [p.batch], "int32")
    _not_a_pool(name, inp, ("weights",))
    budget, recent = int(at["budget"]), int(at.get("recent", 0))
    if not 0 < budget < 1 << 30 or not 0 <= recent <= budget or \
            budget != at["budget"] or recent != at.get("recent", 0):
        raise ValueError("%s: the budget must be a positive whole number and hold the recent slots, "
                         "but got budget %s, recent %s" % (name, at["budget"], at.get("recent", 0)))
    p.budget, p.recent = budget, recent
    reads = [dev(backend, t) for t in (weights, inp["pageTable"], inp["lengths"], positions, total)]
    pools = [backend.device_id_for_update(inp[n].dataId) for n in ("kCache", "vCache")]
    return _outputs(backend, [(slots, "float32"), (slots, "int32"), ([p.batch], "int32"),
                              ([p.batch, p.kv_heads, budget], "int32")],
                    lambda out: backend.lib.tfjs_cuda_paged_cache_evict(
                        backend.ctx, byref(p), *pools, *reads, *out))


def _linear_attention(args):
    backend, inp = args["backend"], args["inputs"]
    name = "_LinearAttention"
    q, k, v, decay = inp["q"], inp["k"], inp["v"], inp["logDecay"]
    state, lengths = inp.get("state"), inp.get("lengths")
    _want(name, "q", q, [None] * 4, "float32")
    batch, heads, seq, dim_k = q.shape
    _want(name, "k", k, q.shape, "float32")
    _want(name, "v", v, [batch, heads, seq, None], "float32")
    dim_v = v.shape[3]
    _want(name, "logDecay", decay, [heads], "float32")
    states = [batch, heads, dim_k, dim_v]
    if state is not None:
        _want(name, "state", state, states, "float32")
    if lengths is not None:
        _want(name, "lengths", lengths, [batch], "int32")
    p = _cabi.LinearAttentionParams(batch, heads, seq, dim_k, dim_v)
    _scale(p, args["attrs"].get("scale"))
    reads = [dev(backend, t) for t in (q, k, v, decay, state, lengths)]
    return _outputs(backend, [([batch, seq, heads, dim_v], "float32"), (states, "float32")],
                    lambda out: backend.lib.tfjs_cuda_linear_attention(
                        backend.ctx, byref(p), *reads, *out))


CONFIGS = [
    KernelConfig("_PagedCacheAppend", BACKEND, _paged_cache_append),
    KernelConfig("_PagedAttention", BACKEND, _paged_attention),
    KernelConfig("_PagedCacheEvict", BACKEND, _paged_cache_evict),
    KernelConfig("_LinearAttention", BACKEND, _linear_attention),
]
