"""GPU tests of iomx_launch_sdpa_packed with values at the end of BF16's range, against its definition in 64 bits:
their weighted mean is finite while their sum is not, in every division of the work and on both kernels."""
import numpy as np
import pytest

from iom_amd import iomx
from packed_cases import Attention, decode, encode

pytestmark = pytest.mark.gpu

BF16 = iomx.DT_BF16


@pytest.fixture(scope="module", autouse=True)
def _device():
    assert iomx.device_count() >= 1
    iomx.check(iomx.lib().iomx_set_device(0))
    yield


# 4 query heads on one KV head: rows of a block are 4 times these
DIVISIONS = [(D, rows, ctx) for D in (64, 128, 192) for rows in (1, 8, 12, 33, 200) for ctx in (100, 2300)]


def with_values(case, change):
    """Replaces the values of tokens (NaN slots of the pages stay), `change` on float64 [.., D]."""
    case.v = encode(case.dtype, change(decode(case.dtype, case.v)))
    old = decode(case.dtype, case.v_pages)
    case.v_pages = encode(case.dtype, np.where(np.isnan(old), np.nan, change(old)))


def both(case):
    for path in (0, 1):
        raw = case.run(path=path)
        case.check(raw)
    return decode(case.dtype, raw)


@pytest.mark.parametrize("D,rows,ctx", DIVISIONS)
@pytest.mark.parametrize("scale", [0.0, 1.0, 6.0])
def test_large_values_whose_mean_is_finite(D, rows, ctx, scale):
    """Values around 1e38 in some features (four of them pass F32's range), ordinary and small ones in others.
    A feature's tolerance is relative to its own values."""
    size = np.ones(D)
    size[:16] = 1e38
    size[16:24] = 1e20
    size[24:32] = 1e-18
    case = Attention(60, BF16, (4, 1), D, 64, [rows, 1, 0], [ctx, 64, 9], scale=scale)
    with_values(case, lambda v: np.clip(np.abs(v) + 0.25, 0.25, 2.0) * size)
    assert np.isfinite(both(case)).all()


@pytest.mark.parametrize("tree", [False, True])
def test_large_values_of_either_sign(tree):
    """Heads, trees and rows without a cache; the mean of values of either sign is far below them."""
    for heads, D, rows, ctx in (((8, 2), 64, [70, 5], [40, 900]), ((6, 6), 80, [9, 300], [3000, 0]), ((2, 1), 40, [9, 30], [70, 0])):
        case = Attention(61, BF16, heads, D, 16, rows, ctx, tree=tree, scale=0.5)
        with_values(case, lambda v: np.clip(v, -3, 3) * 1e38)
        assert np.isfinite(both(case)).all()
    case = Attention(62, BF16, (4, 2), 64, 16, [150, 20], [0, 0], cache=False, tree=tree, scale=0.5)
    with_values(case, lambda v: np.clip(v, -3, 3) * 1e38)
    assert np.isfinite(both(case)).all()


@pytest.mark.parametrize("rows,ctx", [([1, 2], [2300, 40]), ([90, 7], [30, 0])])
def test_a_recorded_step_with_large_values(rows, ctx):
    """Rows that are taken again in a replayed graph: ordinary and large values in turn, each as the eager call."""
    cases = [Attention(65, BF16, (8, 2), 64, 16, rows, ctx) for _ in range(2)]
    with_values(cases[0], lambda v: np.clip(np.abs(v) + 0.25, 0.25, 2.0) * 1e38)
    t = cases[0].upload()
    views = {n: x.view() for n, x in t.items()}
    rc, nbytes, _ = iomx.sdpa_packed_workspace(max_rows=cases[0].max_rows, **views)
    iomx.check(rc)
    ws = iomx.Buffer(nbytes) if nbytes else None
    st = iomx.Stream()
    iomx.synchronize()
    st.begin_capture()
    rc = iomx.sdpa_packed(max_rows=cases[0].max_rows, workspace=ws, stream=st, **views)
    graph = st.end_capture()
    iomx.check(rc)
    for case in (cases[0], cases[1], cases[0], cases[1], cases[0]):
        for name in ("v", "v_pages"):
            t[name].view().from_host(getattr(case, name))
        t["out"].buf.fill(0x5A)
        iomx.synchronize()
        graph.launch(st)
        st.synchronize()
        got = t["out"].view().to_host()
        case.check(got)
        assert np.array_equal(got, case.run())
    graph.close()
    st.close()
