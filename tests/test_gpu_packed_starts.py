"""GPU tests of iomx_launch_cache_append_packed with starts outside the entries and starts that fall:
what they mean is what they mean to the attention (starts clamped to the axis)."""
import numpy as np
import pytest

from iom_amd import iomx
from packed_cases import ints, tensor
from test_gpu_packed_rows import Append

pytestmark = pytest.mark.gpu

BF16, F32 = iomx.DT_BF16, iomx.DT_F32


@pytest.fixture(scope="module", autouse=True)
def _device():
    assert iomx.device_count() >= 1
    iomx.check(iomx.lib().iomx_set_device(0))
    yield


def appended(case, starts):
    """The pools after entry e of every sequence s with clamp(starts[s]) <= e < clamp(starts[s + 1]) is written
    (of two sequences that claim an entry, the first writes it)."""
    kp, vp = case.k_pages.copy(), case.v_pages.copy()
    E = case.T if case.rows is None else len(case.rows)
    at = np.clip(starts, 0, E)
    taken = set()
    for s, c in enumerate(case.ctx):
        for e in range(at[s], at[s + 1]):
            if e in taken:
                continue
            taken.add(e)
            x, row = c + e - at[s], e if case.rows is None else case.rows[e]
            if x < case.M * case.P and 0 <= case.table[s, x // case.P] < case.N:
                page = case.table[s, x // case.P]
                kp[page, :, x % case.P], vp[page, :, x % case.P] = case.k[:, row], case.v[:, row]
    return kp, vp


STARTS = [
    [-7, 20, 40, 60],                   # the first one before the axis
    [-2 ** 31, -5, 20, 2 ** 31 - 1],    # a sequence before the axis has no rows, the last one ends with the axis
    [0, 50, 20, 20],                    # falling: the second has no rows, the first keeps its own
    [0, 30, 10, 10],
    [40, 10, 30, 60],                   # the first has none
    [60, 0, 60, 0],
    [0, 30, 10, 50],                    # entries 10 .. 29 are claimed twice
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("starts", STARTS)
@pytest.mark.parametrize("listed", [None, "any"])
def test_starts_that_are_clamped_or_fall(dtype, starts, listed):
    case = Append(8, dtype, 2, 60, 32, 16, [60, 60, 60], [0, 5, 30], None)
    case.starts = np.array([0, 20, 40, 60])
    if listed:
        case.rows = np.random.default_rng(8).permutation(60)[:57]
    t = [tensor(dtype, a) for a in (case.k, case.v, case.k_pages, case.v_pages)]
    small = [ints([starts]), ints(case.table), ints([case.ctx])]
    rows = ints([case.rows]) if listed else None
    iomx.check(iomx.cache_append_packed(*[x.view() for x in t + small], rows.view() if rows else None), "append")
    iomx.synchronize()
    kp, vp = appended(case, np.array(starts))
    assert np.array_equal(t[2].view().to_host(), kp) and np.array_equal(t[3].view().to_host(), vp)


def test_starts_of_many_sequences_that_fall():
    """More starts than lanes, the falls in both groups of 64."""
    rng = np.random.default_rng(9)
    S = 150
    case = Append(9, BF16, 2, 400, 32, 16, [3] * S, list(rng.integers(0, 40, S)), None, spare=300)
    starts = np.arange(S + 1) * 2
    starts[[5, 63, 64, 65, 140]] = [-3, 0, 500, 1, 2 ** 31 - 1]
    case.table = rng.permutation(case.N)[:S].reshape(S, 1)      # a page each
    case.M = 1
    case.ctx = list(rng.integers(0, 10, S))
    t = [tensor(BF16, a) for a in (case.k, case.v, case.k_pages, case.v_pages)]
    small = [ints([starts]), ints(case.table), ints([case.ctx])]
    iomx.check(iomx.cache_append_packed(*[x.view() for x in t + small]), "append")
    iomx.synchronize()
    kp, vp = appended(case, starts)
    assert np.array_equal(t[2].view().to_host(), kp) and np.array_equal(t[3].view().to_host(), vp)
