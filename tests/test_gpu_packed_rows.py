"""GPU tests of iomx_launch_rope_packed and iomx_launch_cache_append_packed."""
import numpy as np
import pytest

from iom_amd import iomx
from packed_cases import HALF_STEP, decode, encode, ints, starts_of, tensor

pytestmark = pytest.mark.gpu

BF16, F16, F32 = iomx.DT_BF16, iomx.DT_F16, iomx.DT_F32


@pytest.fixture(scope="module", autouse=True)
def _device():
    assert iomx.device_count() >= 1
    iomx.check(iomx.lib().iomx_set_device(0))
    yield


def rope_exact(x, positions, theta):
    D = x.shape[-1]
    angle = positions[:, None].astype(np.longdouble) * np.longdouble(theta) ** (-2 * np.arange(D // 2, dtype=np.longdouble) / D)
    cos, sin = np.cos(angle).astype(np.float64), np.sin(angle).astype(np.float64)
    lo, hi = x[..., :D // 2], x[..., D // 2:]
    return np.concatenate([lo * cos - hi * sin, hi * cos + lo * sin], -1), np.concatenate([np.hypot(lo, hi)] * 2, -1)


def rope_far(dtype, exact, size):
    """Half a step of the result; of the larger component, two F32 roundings of the products and the
    sum (3 * 2^-24), the error of sine and cosine (2^-23 for F32: two units in the last place; 2^-18
    for the 16-bit leaves: the hardware's), and the angle's own: a fraction of a turn rounded to F32
    (2^-26 of a turn) times 2 pi, and 2^31 * 2^-53 turns of the binary64 product."""
    angle = 2 * np.pi * (2.0 ** -26 + 2.0 ** -22 * 0.5)
    trig = 2.0 ** -22 if dtype == F32 else 2.0 ** -17
    least = {BF16: 2.0 ** -133, F16: 2.0 ** -24, F32: 2.0 ** -149}[dtype]
    return HALF_STEP[dtype] * np.abs(exact) * 1.01 + (3 * 2.0 ** -24 + trig + angle) * size + least


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("H,T,D", [(1, 1, 16), (4, 16, 32), (32, 5, 64), (3, 100, 80), (8, 33, 128), (2, 17, 96), (1, 40, 512), (70, 3, 48)])
def test_rope_packed(dtype, H, T, D):
    rng = np.random.default_rng(H * T + D)
    x = encode(dtype, rng.standard_normal((H, T, D)))
    positions = rng.integers(0, 4000, T)
    positions[:: 7] = rng.integers(0, 2 ** 31 - 1, positions[:: 7].size)
    positions[-1] = 0
    if T > 4:
        positions[2] = -1
        positions[3] = 2 ** 31 - 1
    tx, out = tensor(dtype, x), iomx.DeviceTensor(dtype, (H, T, D), fill=0x5A)
    iomx.check(iomx.rope_packed(tx.view(), out.view(), ints([positions]).view(), 10000.0), "rope_packed")
    iomx.synchronize()
    raw = out.view().to_host()
    exact, size = rope_exact(decode(dtype, x), positions, 10000.0)
    there = positions >= 0
    got = decode(dtype, raw)
    assert (np.abs(got - exact) <= rope_far(dtype, exact, size))[:, there].all(), np.max(np.abs(got - exact)[:, there])
    assert np.array_equal(raw[:, positions == 0], x[:, positions == 0])          # nothing to turn
    assert (raw[:, ~there].view(np.uint8) == 0x5A).all()
    if T % 16:
        whole = out.raw().reshape(H, -(-T // 16), D // 16, 16, 16)
        assert (np.ascontiguousarray(whole[:, -1, :, T % 16:]).view(np.uint8) == 0x5A).all()


@pytest.mark.parametrize("theta", [1.0, 500000.0, 3.0e38])
def test_rope_packed_bases(theta):
    rng = np.random.default_rng(9)
    x = encode(F32, rng.standard_normal((2, 20, 64)))
    positions = rng.integers(0, 100000, 20)
    tx, out = tensor(F32, x), iomx.DeviceTensor(F32, (2, 20, 64))
    iomx.check(iomx.rope_packed(tx.view(), out.view(), ints([positions]).view(), theta))
    iomx.synchronize()
    exact, size = rope_exact(decode(F32, x), positions, theta)
    assert (np.abs(decode(F32, out.view().to_host()) - exact) <= rope_far(F32, exact, size)).all()


def test_rope_packed_of_rows_in_order_is_rope():
    """Positions a, a+1, ...: iomx_launch_rope's rows, within a step of BF16 and its F32 angles."""
    rng = np.random.default_rng(10)
    x = encode(BF16, rng.standard_normal((4, 50, 64)))
    tx, one, two = tensor(BF16, x), iomx.DeviceTensor(BF16, (4, 50, 64)), iomx.DeviceTensor(BF16, (4, 50, 64))
    iomx.check(iomx.rope(tx.view(), one.view(), 37, 10000.0))
    iomx.check(iomx.rope_packed(tx.view(), two.view(), ints([np.arange(37, 87)]).view(), 10000.0))
    iomx.synchronize()
    a, b = (decode(BF16, t.view().to_host()) for t in (one, two))
    _, size = rope_exact(decode(BF16, x), np.zeros(50, np.int64), 1.0)
    # both round once (half a step each); iomx_launch_rope's angle, up to 87 in binary32, is off by up to 2^-18
    assert (np.abs(a - b) <= 2.0 ** -8 * (np.abs(a) + np.abs(b)) * 1.01 + 2.0 ** -15 * size).all()


def test_rope_packed_on_views():
    """Every other head of a tensor into another order of heads."""
    rng = np.random.default_rng(11)
    x = encode(F16, rng.standard_normal((6, 30, 64)))
    src, dst = iomx.DeviceTensor(F16, (12, 30, 64), fill=0xFF), iomx.DeviceTensor(F16, (2, 3, 30, 64), fill=0x5A)
    sv = src.view().slice(0, 1, 6, 2)
    sv.from_host(x)
    positions = rng.integers(0, 999, 30)
    plain = iomx.DeviceTensor(F16, (6, 30, 64))
    for s in range(2):
        iomx.check(iomx.rope_packed(sv.slice(0, s, 3, 2), dst.view().select(0, s), ints([positions]).view(), 10000.0))
    iomx.check(iomx.rope_packed(tensor(F16, x).view(), plain.view(), ints([positions]).view(), 10000.0))
    iomx.synchronize()
    want = plain.view().to_host()
    got = dst.view().to_host()
    assert np.array_equal(got[0], want[0::2]) and np.array_equal(got[1], want[1::2])


# ---------------------------------------------------------------------------
# cache_append_packed
# ---------------------------------------------------------------------------

class Append:
    def __init__(self, seed, dtype, Hkv, T, D, P, counts, ctx, listed, first=0, spare=2):
        rng = np.random.default_rng(seed)
        carrier, bits = iomx.carrier(dtype), iomx.LEAF_BITS[dtype]
        raw = lambda dims: rng.integers(0, 2 ** bits, dims, np.uint64).astype(carrier)
        self.dtype, self.P, self.T, self.ctx = dtype, P, T, list(ctx)
        self.k, self.v = raw((Hkv, T, D)), raw((Hkv, T, D))
        used = [-(-(c + n) // P) for c, n in zip(ctx, counts)]
        self.M, self.N = max(1, max(used)), sum(used) + spare
        order = list(rng.permutation(self.N))
        self.table = np.full((len(ctx), self.M), -1, np.int64)
        for s, n in enumerate(used):
            for m in range(n):
                self.table[s, m] = order.pop()
        self.k_pages, self.v_pages = raw((self.N, Hkv, P, D)), raw((self.N, Hkv, P, D))
        self.starts = starts_of(counts, first)
        self.rows = rng.permutation(T)[:self.starts[-1]] if listed else None
        if listed == "sorted":
            self.rows = np.sort(self.rows)

    def expected(self):
        kp, vp = self.k_pages.copy(), self.v_pages.copy()
        E = self.T if self.rows is None else len(self.rows)
        for s, c in enumerate(self.ctx):
            for e in range(max(0, self.starts[s]), min(E, self.starts[s + 1])):
                x = max(0, c) + e - self.starts[s]
                row = e if self.rows is None else self.rows[e]
                if x >= self.M * self.P or not 0 <= row < self.T:
                    continue
                page = self.table[s, x // self.P]
                if 0 <= page < self.N:
                    kp[page, :, x % self.P] = self.k[:, row]
                    vp[page, :, x % self.P] = self.v[:, row]
        return kp, vp

    def check(self, stream=None):
        t = [tensor(self.dtype, a) for a in (self.k, self.v, self.k_pages, self.v_pages)]
        small = [ints([self.starts]), ints(self.table), ints([self.ctx])]
        rows = None if self.rows is None else ints([self.rows])
        padding = t[2].raw().copy()
        iomx.check(iomx.cache_append_packed(*[x.view() for x in t + small], rows.view() if rows else None, stream), "append")
        iomx.synchronize()
        kp, vp = self.expected()
        assert np.array_equal(t[2].view().to_host(), kp) and np.array_equal(t[3].view().to_host(), vp)
        want = tensor(self.dtype, kp)
        assert np.array_equal(t[2].raw(), want.raw())            # padding slots as they were
        assert padding.shape == want.raw().shape
        for x in t + small + [want] + ([rows] if rows else []):
            x.free()


APPENDS = [
    (1, 1, 16, 16, [1], [0]), (2, 40, 64, 16, [7, 0, 20, 1], [0, 5, 9, 47]), (8, 100, 128, 64, [33, 17, 50], [63, 0, 100]),
    (3, 30, 80, 48, [10, 20], [40, 41]), (1, 70, 32, 7, [30, 40], [3, 20]), (4, 17, 96, 1, [9, 8], [2, 0])]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Hkv,T,D,P,counts,ctx", APPENDS)
@pytest.mark.parametrize("listed", [None, "sorted", "any"])
def test_append(dtype, Hkv, T, D, P, counts, ctx, listed):
    Append(1, dtype, Hkv, T, D, P, counts, ctx, listed).check()


@pytest.mark.parametrize("dtype", range(23))
def test_append_of_every_leaf(dtype):
    Append(2, dtype, 2, 40, 48, 16, [7, 0, 20, 1], [0, 5, 9, 47], "any").check()


def test_append_many_sequences():
    """More than one wave's worth of starts; a token each, and none for some."""
    rng = np.random.default_rng(3)
    counts = rng.integers(0, 3, 300)
    Append(3, BF16, 2, int(counts.sum()) + 5, 32, 16, counts, rng.integers(0, 40, 300), None).check()
    Append(3, BF16, 2, 200, 32, 16, [1] * 130, rng.integers(0, 40, 130), "any", first=9).check()


def test_append_skips_what_has_no_place():
    case = Append(4, F16, 2, 60, 64, 16, [20, 20, 20], [0, 5, 30], "any")
    case.table[0, 1], case.table[1, 0] = -1, case.N
    case.table[2, -1] = -2 ** 31
    case.rows[[3, 30]] = [-1, 60]
    case.check()
    case = Append(5, F16, 2, 60, 64, 16, [20, 20, 20], [0, 5, 30], None)
    case.ctx = [-4, 2 ** 31 - 1, case.M * 16 - 3]           # before the table, past it, over its end
    case.check()
    case = Append(6, F16, 2, 60, 64, 16, [20, 20], [0, 5], None, first=7)   # entries of no sequence on either side
    case.check()


def test_append_captured():
    st = iomx.Stream()
    case = Append(7, BF16, 2, 40, 64, 16, [7, 20, 1], [0, 9, 47], None)
    t = [tensor(BF16, a) for a in (case.k, case.v, case.k_pages, case.v_pages)]
    small = [ints([case.starts]), ints(case.table), ints([case.ctx])]
    iomx.synchronize()
    st.begin_capture()
    rc = iomx.cache_append_packed(*[x.view() for x in t + small], None, st)
    graph = st.end_capture()
    iomx.check(rc)
    for i in range(3):
        for tt, data in zip(t[2:], (case.k_pages, case.v_pages)):
            tt.view().from_host(data)
        case.ctx = [[0, 9, 47], [2, 3, 4], [10, 0, 20]][i]
        small[2].view().from_host(np.array([case.ctx], np.uint32))
        iomx.synchronize()
        graph.launch(st)
        st.synchronize()
        kp, vp = case.expected()
        assert np.array_equal(t[2].view().to_host(), kp) and np.array_equal(t[3].view().to_host(), vp)
    graph.close()
    st.close()
