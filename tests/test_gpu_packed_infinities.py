"""GPU tests of iomx_launch_sdpa_packed with infinite values that a row sees, against its definition in 64 bits:
whatever the token's probability, also where it is far below what a matrix product keeps, the feature is that
infinity (a NaN of both signs), in every division of the work and on both kernels."""
import numpy as np
import pytest

from iom_amd import iomx
from packed_cases import Attention, decode, encode

pytestmark = pytest.mark.gpu

BF16, F16 = iomx.DT_BF16, iomx.DT_F16


@pytest.fixture(scope="module", autouse=True)
def _device():
    assert iomx.device_count() >= 1
    iomx.check(iomx.lib().iomx_set_device(0))
    yield


# 4 query heads on one KV head: rows of a block are 4 times these
DIVISIONS = [(D, rows, ctx) for D in (64, 128, 192) for rows in (1, 8, 12, 33, 200) for ctx in (100, 2300)]


def both(case):
    for path in (0, 1):
        raw = case.run(path=path)
        case.check(raw)
    return decode(case.dtype, raw)


def far_away(case, s, x, by):
    """Moves the score of cached token x of sequence s to about `by` (q is all ones then)."""
    page, r = case.table[s, x // case.P], x % case.P
    case.k_pages[page, :, r] = encode(case.dtype, by / np.sqrt(case.D))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,rows,ctx", DIVISIONS)
@pytest.mark.parametrize("by", [-160.0, 160.0])
def test_infinities_of_any_probability(dtype, D, rows, ctx, by):
    """Token 3 holds an infinity in feature 7, token 20 the other one in features 9 and 11, token 21 the same
    as token 3 in feature 11.  Their probabilities are e^-160 of the others' (`by` below zero), or one token
    at the end of the context takes all of the probability (above)."""
    case = Attention(63, dtype, (4, 1), D, 64, [rows, 1], [ctx, 64])
    case.q[:] = encode(dtype, 1.0)
    if by < 0:
        for x in (3, 20, 21):
            far_away(case, 0, x, by)
    else:
        far_away(case, 0, ctx - 1, by)
    for x, feature, value in ((3, 7, np.inf), (20, 9, -np.inf), (20, 11, -np.inf), (21, 11, np.inf)):
        case.v_pages[case.table[0, x // 64], 0, x % 64, feature] = encode(dtype, value)
    out = both(case).reshape(-1, 4, D)[:rows]
    assert np.isposinf(out[:, :, 7]).all() and np.isneginf(out[:, :, 9]).all() and np.isnan(out[:, :, 11]).all()
    assert np.isfinite(np.delete(out, [7, 9, 11], -1)).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_an_infinity_behind_the_first_rows(dtype):
    """Row 100 of a prompt holds one: rows before it are finite, it and those behind it are not, however small
    its probability."""
    case = Attention(64, dtype, (4, 2), 64, 16, [300, 40], [0, 30])
    case.q[:] = encode(dtype, 1.0)
    case.k[:, 100] = encode(dtype, -160.0 / 8)
    case.v[:, 100, 5] = encode(dtype, np.inf)
    out = both(case).reshape(-1, 4, 64)
    assert np.isfinite(out[:100]).all() and np.isposinf(out[100:300, :, 5]).all() and np.isfinite(out[300:]).all()
    assert np.isfinite(np.delete(out, 5, -1)).all()
