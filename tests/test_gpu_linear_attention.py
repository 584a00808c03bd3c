"""Linear attention with a decay for each head against its recurrence in 64 bits
(tests/decoder_cases.py, which derives the tolerances): single tokens, prompts of every
remainder, padded batches, prompts in pieces."""
import numpy as np
import pytest

from tests import decoder_cases as dc

pytestmark = pytest.mark.gpu


@pytest.fixture
def tf(cuda_engine):
    from tfjs_b200 import ops
    before = cuda_engine.backend.numDataIds()
    yield ops
    cuda_engine.backend.sync()
    assert cuda_engine.backend.numDataIds() == before


def inputs(seed, b, h, n, dk, dv):
    r = np.random.default_rng(seed)
    q, k, v = (r.standard_normal((b, h, n, d)).astype(np.float32) for d in (dk, dk, dv))
    return q, k / np.float32(np.sqrt(dk)), v, r.standard_normal((b, h, dk, dv)).astype(np.float32)


def decays(h):
    return np.log1p(-np.exp2(-np.linspace(1.0, 10.0, h))).astype(np.float32)


def call(tf, *args, **kw):
    ts = [tf.tensor(a) if isinstance(a, np.ndarray) else a for a in args]
    kw = {k: tf.tensor(a) if isinstance(a, np.ndarray) else a for k, a in kw.items()}
    outs = tf.linear_attention(*ts, **kw)
    got = [t.arraySync() for t in outs]
    for t in ts + list(kw.values()) + outs:
        if hasattr(t, "dispose"):
            t.dispose()
    return got


def check(got, ref):
    for g, r, off in zip(got, ref[:2], ref[2:]):
        assert g.shape == r.shape
        assert np.all(np.abs(g - r) <= off), (np.max(np.abs(g - r)), np.max(np.abs(g - r) / off))


@pytest.mark.parametrize("b,h,n,dk,dv", [
    (1, 1, 1, 1, 1), (1, 12, 1, 64, 64), (3, 4, 1, 128, 128), (2, 3, 1, 33, 50), (1, 2, 1, 256, 256),
    (2, 2, 2, 64, 64), (1, 3, 17, 16, 32), (2, 2, 63, 64, 64), (2, 2, 64, 64, 64), (1, 2, 65, 64, 64),
    (1, 2, 127, 128, 128), (1, 1, 129, 128, 64), (1, 2, 200, 33, 50), (1, 1, 300, 256, 100),
    (2, 3, 513, 32, 64), (1, 2, 700, 96, 128), (1, 1, 150, 7, 3), (1, 1, 260, 100, 256),
    (40, 4, 70, 64, 64),
])
def test_against_the_recurrence(tf, b, h, n, dk, dv):
    q, k, v, s = inputs(n + dk, b, h, n, dk, dv)
    ld = decays(h)
    check(call(tf, q, k, v, ld), dc.linear(q, k, v, ld))
    lengths = np.random.default_rng(n).integers(0, n + 1, b).astype(np.int32)
    check(call(tf, q, k, v, ld, state=s, scale=0.125, lengths=lengths),
          dc.linear(q, k, v, ld, s, 0.125, lengths))


@pytest.mark.parametrize("log_decay", [0.0, -1e-6, -0.7, -30.0, -200.0, -np.inf])
def test_decays_from_none_to_all(tf, log_decay):
    """A decay of 1 keeps everything, one of 0 leaves the token itself (e^-inf = 0; what
    0 * -inf would be must not enter)."""
    b, h, n, dk, dv = 1, 2, 200, 64, 64
    q, k, v, s = inputs(3, b, h, n, dk, dv)
    ld = np.full(h, log_decay, np.float32)
    check(call(tf, q, k, v, ld, state=s), dc.linear(q, k, v, ld, s))


def test_a_prompt_in_pieces_and_tokens(tf):
    """Handing the state on gives what one call gives."""
    b, h, n, d = 2, 3, 333, 64
    q, k, v, s = inputs(4, b, h, n, d, d)
    ld = decays(h)
    ref = dc.linear(q, k, v, ld, s, 0.125)
    at, outs = 0, []
    for piece in (200, 1, 1, 64, 67):
        cut = [np.ascontiguousarray(x[:, :, at:at + piece]) for x in (q, k, v)]
        o, s = call(tf, *cut, ld, state=s, scale=0.125)
        outs.append(o)
        at += piece
    assert at == n
    check([np.concatenate(outs, axis=1), s], ref)


def test_behind_a_rows_end_nothing_counts(tf):
    """NaN and infinities behind a row's tokens do not enter; a row without tokens keeps its
    state."""
    b, h, n, d = 3, 2, 150, 64
    q, k, v, s = inputs(5, b, h, n, d, d)
    lengths = np.array([0, 70, 149], np.int32)
    for i, m in enumerate(lengths):
        q[i, :, m:], k[i, :, m:], v[i, :, m:] = np.nan, np.inf, np.nan
    ld = decays(h)
    clean = [np.where(np.isfinite(x), x, 0).astype(np.float32) for x in (q, k, v)]
    got = call(tf, q, k, v, ld, state=s, lengths=lengths)
    check(got, dc.linear(*clean, ld, s, None, lengths))
    assert np.array_equal(got[1][0], s[0]) and np.all(got[0][1, 70:] == 0.0)
    got = call(tf, *[np.ascontiguousarray(x[:, :, 149:]) for x in (q, k, v)], ld, state=s,
               lengths=np.array([0, 0, 0], np.int32))
    assert np.all(got[0] == 0.0) and np.array_equal(got[1], s)


def test_bad_lengths_are_reported(tf, cuda_engine):
    from tfjs_b200 import _cabi
    q, k, v, s = inputs(6, 2, 1, 80, 32, 32)
    ld = decays(1)
    ts = [tf.tensor(x) for x in (q, k, v, ld, np.array([-1, 81], np.int32))]
    outs = tf.linear_attention(*ts[:4], lengths=ts[4])
    with pytest.raises(_cabi.CudaError) as e:
        cuda_engine.backend.sync()
    assert e.value.code == 1 and "length" in str(e.value)
    check([t.arraySync() for t in outs], dc.linear(q, k, v, ld, None, None, [0, 80]))
    for t in ts + outs:
        t.dispose()


def test_captured_prompts_replay(tf, cuda_engine):
    """Two captured prompts of different sizes, replayed in turn with an eager one in between: each
    has a workspace of its own."""
    backend = cuda_engine.backend
    made = []
    for seed, n, d in ((8, 300, 64), (9, 150, 128)):
        q, k, v, s = inputs(seed, 2, 2, n, d, d)
        ld = decays(2)
        ts = [tf.tensor(x) for x in (q, k, v, ld, s)]
        for t in ts:
            backend.device_id(t.dataId)
        backend.sync()
        backend.capture_begin(64 << 20)
        outs = tf.linear_attention(*ts, scale=0.125)
        made.append((backend.capture_end(), outs, ts, dc.linear(q, k, v, ld, s, 0.125)))
    for i in range(6):
        backend.graph_launch(made[i % 2][0])
        if i == 3:
            call(tf, *[np.zeros((1, 1, 700, 32), np.float32)] * 3, decays(1))
    for graph, outs, ts, ref in made:
        check([t.arraySync() for t in outs], ref)
        backend.graph_destroy(graph)
        for t in ts + outs:
            t.dispose()


def test_captured_tokens_replay(tf, cuda_engine):
    """A captured token whose new state is copied over the old one: a replay a token."""
    backend = cuda_engine.backend
    b, h, d = 2, 3, 64
    q, k, v, s = inputs(7, b, h, 1, d, d)
    ld = decays(h)
    ts = [tf.tensor(x) for x in (q, k, v, ld, s)]
    for t in ts:
        backend.device_id(t.dataId)
    backend.sync()
    backend.capture_begin(16 << 20)
    out, new = tf.linear_attention(*ts, scale=0.125)
    backend.copy(new.dataId, ts[4].dataId)
    new.dispose()
    graph = backend.capture_end()
    for _ in range(5):
        backend.graph_launch(graph)
    rep = [np.ascontiguousarray(np.repeat(x, 5, axis=2)) for x in (q, k, v)]
    ref = dc.linear(*rep, ld, s, 0.125)
    got = out.arraySync()
    assert np.all(np.abs(got[:, 0] - ref[0][:, 4]) <= ref[2][:, 4])
    backend.graph_destroy(graph)
    for t in ts + [out]:
        t.dispose()
