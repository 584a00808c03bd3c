"""Linear attention with infinities in its state, and over many chunks."""
import numpy as np
import pytest

from tests import decoder_cases as dc
from tests.test_gpu_linear_attention import call, check, decays, inputs, tf  # noqa: F401  (tf: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 3, 200])
@pytest.mark.parametrize("log_decay", [0.0, -0.5, -1e-3])
def test_an_infinite_state_stays_infinite(tf, n, log_decay):
    """An infinity times a decay is that infinity, and so it leaves in the new state, single tokens and
    prompts alike; the elements beside it keep their values."""
    h, d = 2, 32
    q, k, v, s = inputs(n, 1, h, n, d, d)
    s[0, 0, 3, 5], s[0, 1, 30, 31] = np.inf, -np.inf
    ld = np.full(h, log_decay, np.float32)
    _, got = call(tf, q, k, v, ld, state=s)
    clean = np.where(np.isfinite(s), s, 0).astype(np.float32)
    _, ref, _, off = dc.linear(q, k, v, ld, clean)
    assert got[0, 0, 3, 5] == np.inf and got[0, 1, 30, 31] == -np.inf
    there = np.isfinite(s)
    assert np.all(np.abs(got - ref)[there] <= off[there])


def test_long_rows_keep_their_first_state(tf):
    """128 chunks of tokens whose keys are zero leave exp(log_decay)^16384 times the first state.
    A decay for a whole chunk that is one float is off the same way in every chunk, by half a unit in its
    last place or more: 64 EPS in all and more for these.  What remains with the decay in two
    parts is the rounding of each chunk's step, at most EPS and to either side: over 128 steps its standard
    deviation is below 128 ** 0.5 * EPS / 3 ** 0.5 = 6.6 EPS, over the mean of 1024 elements 0.21 EPS.
    2 EPS is over nine of those."""
    h, n, d = 8, 16384, 32
    r = np.random.default_rng(21)
    q = np.zeros((1, h, n, d), np.float32)
    s = (1.0 + r.random((1, h, d, d))).astype(np.float32)
    ld = (-np.geomspace(1e-6, 1e-4, h)).astype(np.float32)
    _, got = call(tf, q, q, q, ld, state=s)
    ref = s.astype(np.float64) * np.exp(ld.astype(np.float64) * n)[None, :, None, None]
    drift = np.mean(got / ref - 1.0, axis=(0, 2, 3)) / dc.EPS
    assert np.all(np.abs(drift) <= 2.0), drift
    # the largest error: 128 roundings of EPS each and the two products of a step
    assert np.max(np.abs(got / ref - 1.0)) <= 132 * dc.EPS


@pytest.mark.parametrize("n", [1100, 1152, 2047, 2049, 4200])
def test_many_chunks(tf, n):
    """9, 16, 17 and 33 chunks: beyond the first eight that the scan has in flight, its second batch,
    and its second time around; ragged rows."""
    b, h, dk, dv = 2, 2, 16, 32
    q, k, v, s = inputs(n, b, h, n, dk, dv)
    ld = np.array([-1e-4, -0.01], np.float32)
    lengths = np.array([n, n - 700], np.int32)
    check(call(tf, q, k, v, ld, state=s, scale=0.25, lengths=lengths),
          dc.linear(q, k, v, ld, s, 0.25, lengths))


@pytest.mark.parametrize("b,h,n,dk,dv,spots", [
    (2, 2, 400, 64, 64, [(0, 1, 200, 9)]),
    (1, 1, 33, 64, 64, [(0, 0, 32, 63)]),
    (2, 3, 300, 33, 50, [(0, 0, 0, 49), (1, 2, 299, 0)]),
    (1, 2, 260, 128, 256, [(0, 0, 130, 3), (0, 1, 259, 200), (0, 1, 128, 200)]),
    (40, 8, 150, 16, 32, [(i, i % 8, 149 - i, i % 32) for i in range(40)]),
])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_what_is_not_finite_comes_after_its_token(tf, b, h, n, dk, dv, spots, value):
    """A NaN or an infinity in v enters its column of out with its token and not before, in prompts as in
    single tokens, and its column of the state; everything else keeps its value."""
    q, k, v, s = inputs(17 + n, b, h, n, dk, dv)
    ld = decays(h)
    clean = dc.linear(q, k, v, ld, s, 0.125)
    v = v.copy()
    there, inside = np.ones(clean[0].shape, bool), np.ones(clean[1].shape, bool)
    for i, j, t, d in spots:
        v[i, j, t, d] = value
        there[i, t:, j, d] = inside[i, j, :, d] = False
    out, state = call(tf, q, k, v, ld, state=s, scale=0.125)
    assert np.all(np.abs(out - clean[0])[there] <= clean[2][there])
    assert np.all(np.abs(state - clean[1])[inside] <= clean[3][inside])
    assert not np.any(np.isfinite(out[~there])) and not np.any(np.isfinite(state[~inside]))


def test_values_next_to_the_largest(tf):
    """Finite values of v beyond 2^127: the outputs of their chunk are right, earlier tokens' among them.
    At decays of 1/2 such a value still counts 115 tokens later, with a weight of 5e-39: below 2^-126 the
    operands of the tensor core are spaced 2^-136, so a weight is off by up to that, times the value."""
    b, h, n, d = 1, 2, 300, 64
    q, k, v, s = inputs(5, b, h, n, d, d)
    v[0, 0, 140, 7], v[0, 1, 290, 63] = 3.4e38, np.finfo(np.float32).max
    k[0, :, [140, 290]] *= 0.01
    q *= np.float32(0.01)
    ld = decays(h)
    lengths = np.array([295], np.int32)
    ref = dc.linear(q, k, v, ld, s, None, lengths)
    out, state = call(tf, q, k, v, ld, state=s, lengths=lengths)
    ref[2][:, 140:256, 0, 7] += 2.0 ** -136 * 3.4e38
    first = np.s_[:, :256]                  # (the chunk of the first; the second's begins at 256)
    assert np.all(np.abs(out - ref[0])[first] <= ref[2][first])
    assert np.all(np.abs(out - ref[0])[:, 256:, 1] <= ref[2][:, 256:, 1])
