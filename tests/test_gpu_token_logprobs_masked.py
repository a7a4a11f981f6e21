"""GPU tests of iomx_launch_token_logprobs on rows whose logits lie far apart, each row with a tolerance of
its own: forbidden tokens at the type's lowest finite value, rows of nothing else, rows at either end of the range."""
import numpy as np
import pytest

from iom_amd import iomx
from packed_cases import decode, encode
from test_gpu_token_logprobs import run

pytestmark = pytest.mark.gpu

BF16, F16, F32 = iomx.DT_BF16, iomx.DT_F16, iomx.DT_F32
LOWEST = {BF16: -3.3895313892515355e38, F16: -65504.0, F32: -3.4028234663852886e38}


@pytest.fixture(scope="module", autouse=True)
def _device():
    assert iomx.device_count() >= 1
    iomx.check(iomx.lib().iomx_set_device(0))
    yield


def exact(x, tokens, K):
    """log probabilities, entropy, ids and log probabilities of the likeliest: everything by differences from the
    row's largest logit, so that nothing is lost next to a logit of 1e38."""
    top = x.max(-1, keepdims=True)
    with np.errstate(over="ignore"):
        d = x - top
        e = np.exp(d)
        total = e.sum(-1, keepdims=True)
        logs = d - np.log(total)
        entropy = np.log(total) - np.where(e > 0, d * e, 0).sum(-1, keepdims=True) / total
    ids = np.argsort(-x, axis=-1, kind="stable")[:, :K]
    return np.take_along_axis(logs, tokens, 1), entropy, ids, np.take_along_axis(logs, ids, 1)


def allowed(x, want):
    """By row.  An exponential is of consequence for differences d from the row's largest logit down to -104: the
    difference and its product with log2 e are rounded (104 * 2^-23 together), the function is off by 2^-22, its
    terms are added in F32 in chains of at most V / 64 + 64.  Each rounding is half a step (2^-24 of what it rounds), and
    two steps' worth is granted.  The logarithm moves with the sum's relative error, the entropy with that of sum d e^d
    too (its size relative to the sum is at most log V).  What is added to them (d itself, the result) is rounded once to
    F32: 2^-24 of the result."""
    V = x.shape[-1]
    spread = np.minimum(104.0, x.max(-1, keepdims=True) - x.min(-1, keepdims=True))
    total = spread * 2.0 ** -22 + 2.0 ** -21 + (V / 64 + 64) * 2.0 ** -24
    return (2 + np.log(V)) * total + 2.0 ** -24 * np.abs(want)


def masked(rng, V, lowest):
    """Rows of ordinary logits, each with other ones allowed, and rows at the ends of the range."""
    x = rng.standard_normal((40, V)) * 3
    for r in range(24):
        x[r, rng.permutation(V)[:V - 1 - r * (V - 1) // 24]] = lowest     # from one allowed token upwards
    x[24] = lowest                                          # none: all equally likely
    x[25] = -lowest
    x[26] = np.where(np.arange(V) % 2 == 0, lowest, -lowest)
    x[27, :V // 2] = lowest                                 # the larger ones come late
    x[28, V // 2:] = lowest
    x[29] = lowest
    x[29, V - 1] = lowest / 2
    x[30] = -lowest
    x[30, 0] = 1.0
    x[31] = np.sort(x[31])
    x[32] = np.sort(x[32])[::-1]
    x[33] = 0.75 * lowest
    return x


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("V", [1, 40, 700, 2433, 9001, 40000])
def test_masks_of_the_lowest_value(dtype, V):
    rng = np.random.default_rng(21)
    raw = encode(dtype, masked(rng, V, LOWEST[dtype]))
    x = decode(dtype, raw)
    for K in {1, min(20, V), min(32, V)}:
        tokens = rng.integers(0, V, (40, 3))
        given, entropy, ids, tops = exact(x, tokens, K)
        got = run(dtype, raw, tokens, K)
        assert np.array_equal(got["top_ids"], ids)
        for name, want in (("logprobs", given), ("entropy", entropy), ("top_logprobs", tops)):
            far = np.broadcast_to(allowed(x, want), want.shape)
            # F32 ends at (2 - 2^-23) 2^127: what lies half a step past it rounds to an infinity
            want = np.where(want <= -(2.0 ** 128 - 2.0 ** 103), -np.inf, want)
            fine = np.isfinite(want)
            assert np.array_equal(got[name][~fine], want[~fine]), name
            assert (far[fine & (np.abs(want) < 1e3)] < 1e-2).all()            # the bound is a sharp one
            off = np.abs(got[name] - want) - far
            worst = np.unravel_index(np.argmax(np.where(fine, off, -np.inf)), off.shape)
            assert not fine.any() or off[worst] <= 0, (name, worst, got[name][worst], want[worst], far[worst])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_of_one_value(dtype):
    """Any value, of whatever size: every token has the log probability -log V, and the entropy is log V."""
    V = 5000
    top = -LOWEST[dtype]
    values = np.array([0.0, 1.0, -7.5, 60000.0, -60000.0, top, -top, top / 2, -top / 2, 1e-6])
    raw = encode(dtype, np.repeat(values[:, None], V, 1))
    got = run(dtype, raw, np.tile([0, V - 1], (len(values), 1)), 4)
    assert np.array_equal(got["top_ids"], np.tile(np.arange(4), (len(values), 1)))
    # a sum of V ones is exact; a logarithm, a difference and a result rounded to F32
    for name, want in (("logprobs", -np.log(V)), ("top_logprobs", -np.log(V)), ("entropy", np.log(V))):
        assert (np.abs(got[name] - want) <= 3 * 2.0 ** -24 * np.log(V)).all(), (name, got[name])
