"""GPU tests of iomx_launch_sdpa_packed against its definition in 64 bits (packed_cases.Attention,
whose tolerances count the roundings): prompts, single tokens and trees, every head layout and
page size, what is not seen, lengths that the device holds, graphs and streams."""
import numpy as np
import pytest

from iom_amd import iomx
from packed_cases import Attention, decode, encode, ints, starts_of, tensor

pytestmark = pytest.mark.gpu

BF16, F16 = iomx.DT_BF16, iomx.DT_F16


@pytest.fixture(scope="module", autouse=True)
def _device():
    assert iomx.device_count() >= 1
    iomx.check(iomx.lib().iomx_set_device(0))
    yield


def both(case):
    """Path 0 and the one-wave-per-row kernel."""
    case.check(case.run())
    kernel = iomx.last_launch().kernel.decode()
    case.check(case.run(path=1))
    return kernel


# heads, D, P, rows, ctx
PROMPTS = [
    ((1, 1), 16, 16, [1], [0]),
    ((4, 4), 32, 16, [17, 3, 40], [0, 5, 31]),
    ((8, 2), 64, 32, [1, 70, 0, 15, 16], [33, 0, 9, 64, 1]),
    ((32, 4), 64, 16, [33, 5], [100, 0]),
    ((6, 2), 80, 48, [29, 64, 2], [47, 48, 49]),
    ((12, 4), 96, 64, [100, 7], [1, 130]),
    ((8, 8), 128, 16, [40, 90], [17, 0]),
    ((16, 1), 128, 64, [65], [250]),
    ((5, 1), 112, 32, [31, 33], [63, 65]),
    ((6, 2), 40, 16, [20, 9], [30, 2]),            # heads of no whole tiles
    ((4, 2), 64, 7, [20, 9], [30, 21]),            # pages of no whole tiles
    ((4, 2), 64, 1, [5], [9]),
    ((2, 1), 136, 16, [9, 3], [20, 0]),
    ((2, 2), 256, 32, [21], [40]),
    ((3, 3), 8, 16, [11], [18]),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,D,P,rows,ctx", PROMPTS)
def test_prompts(dtype, heads, D, P, rows, ctx):
    both(Attention(1, dtype, heads, D, P, rows, ctx))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,D,P,rows,ctx", PROMPTS)
def test_trees(dtype, heads, D, P, rows, ctx):
    both(Attention(2, dtype, heads, D, P, rows, ctx, tree=True, first=3, tail=21))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,D,P", [((32, 4), 64, 16), ((8, 8), 64, 64), ((16, 2), 128, 32), ((71, 1), 64, 16), ((4, 2), 80, 16)])
@pytest.mark.parametrize("ctx", [[0], [1, 15, 16, 17, 31, 32, 33, 0], [700, 3, 1025, 64, 2049]])
def test_single_tokens(dtype, heads, D, P, ctx):
    both(Attention(3, dtype, heads, D, P, [1] * len(ctx), ctx))


@pytest.mark.parametrize("tree", [False, True])
def test_longer_ones(tree):
    """Blocks of rows that start inside a tile, several of them per sequence, and scores that span a wide range."""
    both(Attention(4, BF16, (8, 2), 64, 32, [257, 300, 31], [511, 0, 1000], tree=tree, first=5, scale=4.0))
    both(Attention(5, F16, (4, 4), 128, 64, [190, 129], [0, 333], tree=tree, scale=8.0))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows", [[1, 1, 1], [40, 3, 75], [200]])
def test_without_a_cache(dtype, rows):
    both(Attention(6, dtype, (8, 2), 64, 16, rows, [0] * len(rows), cache=False, tail=4))
    both(Attention(6, dtype, (8, 2), 64, 16, rows, [0] * len(rows), cache=False, tree=True))


def test_rows_of_no_sequence_and_rows_past_the_bound_are_left_as_they_were():
    case = Attention(7, BF16, (4, 2), 64, 16, [10, 0, 30, 4], [20, 3, 0, 50], first=17, tail=40, max_rows=12)
    both(case)
    case = Attention(7, BF16, (4, 2), 64, 16, [10, 0, 30, 4], [20, 3, 0, 50], first=17, tail=40, max_rows=1000)
    both(case)


def test_rows_that_see_nothing_are_zero():
    case = Attention(8, BF16, (8, 2), 64, 16, [6, 33], [0, 40], tree=True)
    case.tree[:] = 0
    case.tree[2] = 1 << 4
    assert both(case)
    out = decode(BF16, case.run())
    assert not out[:2].any() and not np.signbit(out[:2]).any() and out[2].any() and out[6:].any()
    # the same for a sequence whose pages are all absent
    case = Attention(8, F16, (8, 2), 64, 16, [6, 33], [64, 40], tree=True)
    case.tree[:] = 0
    case.table[0] = [case.N, -1, 2 ** 31 - 1, -2 ** 31]
    both(case)
    assert not decode(F16, case.run())[:6].any()


def test_absent_pages_are_not_seen():
    for rows in ([1, 1], [50, 20]):
        case = Attention(9, BF16, (8, 2), 64, 32, rows, [200, 70])
        case.table[0, [0, 3]] = [-1, case.N]
        case.table[1, 1] = case.N + 5
        both(case)


def test_bits_past_the_last_word_and_past_the_rows_are_not_seen():
    case = Attention(10, BF16, (8, 2), 64, 16, [70, 5], [20, 20], tree=True)
    case.tree[:] = 0xFFFFFFFF
    both(case)
    case.tree = np.ascontiguousarray(case.tree[:, :1])     # rows 32.. have no bit
    both(case)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("rows", [[4, 1], [90, 40]])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_what_a_row_does_not_see_does_not_reach_it(dtype, tree, rows, value):
    """The last row's key or value is not finite and only that row sees it."""
    for which in "kv":
        case = Attention(11, dtype, (8, 2), 64, 16, rows, [37, 0], tree=tree)
        last = [n - 1 for n in rows]
        for s, j in enumerate(last):
            t = case.starts[s] + j
            getattr(case, which)[:, t, 3] = encode(dtype, value)
            if tree:
                case.tree[case.starts[s]:t, j >> 5] &= ~np.uint32(1 << (j & 31))
                case.tree[t, j >> 5] |= np.uint32(1 << (j & 31))
        both(case)
        got = decode(dtype, case.run())
        for s, j in enumerate(last):
            assert np.isfinite(got[case.starts[s]:case.starts[s] + j]).all()
            # a value of infinity at the row itself, a key of either sign of it or NaN: visible there, and not in finite form
            if which == "v" or np.isnan(value):
                assert not np.isfinite(got[case.starts[s] + j]).all()


@pytest.mark.parametrize("rows", [[1], [40]])
def test_special_values_that_are_seen(rows):
    """A NaN score makes the row NaN; an infinite value shows in its feature alone."""
    case = Attention(12, BF16, (4, 2), 64, 16, rows, [100])
    page, r = case.table[0, 3], 5
    case.v_pages[page, 0, r, 7] = encode(BF16, np.inf)
    case.k_pages[page, 1, r, 7] = encode(BF16, np.nan)
    both(case)
    got = decode(BF16, case.run()).reshape(-1, 4, 64)
    assert np.isposinf(got[:, :2, 7]).all() and np.isfinite(np.delete(got[:, :2], 7, -1)).all() and np.isnan(got[:, 2:]).all()


def test_huge_and_tiny_operands():
    for dtype, big in ((BF16, 1e30), (F16, 6e4)):
        case = Attention(13, dtype, (4, 2), 64, 16, [40, 1], [70, 30])
        case.v[:] = encode(dtype, decode(dtype, case.v) * (big / 8))
        both(case)
        # scores of thousands: one token takes all
        case = Attention(13, dtype, (4, 2), 64, 16, [40, 1], [70, 30], scale=3000.0)
        both(case)
        # subnormal values
        case = Attention(13, dtype, (4, 2), 64, 16, [40, 1], [70, 30])
        case.v[:] &= 0x807F if dtype == BF16 else 0x83FF
        case.v_pages[:] &= 0x807F if dtype == BF16 else 0x83FF
        both(case)


def test_lengths_and_starts_are_clamped():
    """Device values past the tensors are clamped: the same as the clamped ones."""
    case = Attention(14, BF16, (8, 2), 64, 16, [20, 30], [48, 40])
    t = case.upload()
    want = case.run(t=t)
    t["starts"].view().from_host(np.array([[-7, 20, 2 ** 31 - 1]], np.int64).astype(np.int32).view(np.uint32))
    t["lengths"].view().from_host(np.array([[2 ** 31 - 1, 40]], np.int64).astype(np.int32).view(np.uint32))
    for path in (0, 1):
        t["out"].buf.fill(0x5A)
        got = case.run(t=t, path=path)
        case.check(got)
    t["lengths"].view().from_host(np.array([[-3, -2 ** 31]], np.int64).astype(np.int32).view(np.uint32))
    case.ctx = [0, 0]
    for path in (0, 1):
        case.check(case.run(t=t, path=path))
    # starts that fall: their sequence has no rows
    t["starts"].view().from_host(np.array([[30, 20, 50]], np.uint32))
    t["out"].buf.fill(0x5A)
    got = case.run(t=t)
    assert (got[:20] == 0x5A5A).all() and (got[20:] != 0x5A5A).any()
    assert want.shape == got.shape


def test_views_with_strides():
    """Pools that are slices of one tensor [layers, 2, N, Hkv, P, D], heads in another order, an
    output plane inside a larger tensor."""
    case = Attention(15, BF16, (4, 2), 64, 16, [40, 1, 20], [70, 30, 0], tree=True, tail=2)
    t = case.upload()
    pool = iomx.DeviceTensor(BF16, (2, 2, case.N, case.Hkv, case.P, case.D), fill=0xFF)
    kp, vp = pool.view().select(0, 1).select(0, 0), pool.view().select(0, 1).select(0, 1)
    kp.from_host(case.k_pages)
    vp.from_host(case.v_pages)
    # one tensor [T-rows planes: q heads doubled, every other one in use]
    wide = iomx.DeviceTensor(BF16, (2 * case.Hq, case.T, case.D), fill=0xFF)
    q = wide.view().slice(0, 1, case.Hq, 2)
    q.from_host(case.q)
    # heads outside the pages: [Hkv, N, P, D] permuted
    turned = iomx.DeviceTensor(BF16, (case.Hkv, case.N, case.P, case.D), fill=0xFF)
    tv = turned.view().permute([1, 0])
    tv.from_host(case.v_pages)
    outs = iomx.DeviceTensor(BF16, (3, case.T, case.Hq * case.D), fill=0x5A)
    views = {n: x.view() for n, x in t.items()}
    for v_view in (vp, tv):
        views.update(q=q, k_pages=kp, v_pages=v_view, out=outs.view().select(0, 1))
        for path in (0, 1):
            outs.buf.fill(0x5A)
            case.check(case.run(t=views, path=path))
            assert (outs.view().select(0, 0).to_host() == 0x5A5A).all()
            assert (outs.view().select(0, 2).to_host() == 0x5A5A).all()


def test_a_dense_cache_is_a_pool():
    """A cache [S, Hkv, C, D] as the framework's other attention has it, two sequences of three in use."""
    case = Attention(16, BF16, (8, 2), 64, 96, [1, 1], [90, 33])
    case.N, case.table = 3, np.array([[2], [0]])
    old = case.k_pages, case.v_pages
    case.k_pages = np.full((3, 2, 96, 64), 0x7FC0, np.uint16)
    case.v_pages = case.k_pages.copy()
    for s, page in enumerate((2, 0)):
        for new, pool in zip((case.k_pages, case.v_pages), old):
            new[page, :, :case.ctx[s]] = pool[case.table[s, 0] if pool.shape[0] > 2 else 0, :, :case.ctx[s]]
    rng = np.random.default_rng(5)
    for s, page in enumerate((2, 0)):
        for new in (case.k_pages, case.v_pages):
            new[page, :, :case.ctx[s]] = encode(BF16, rng.standard_normal((2, case.ctx[s], 64)))
    both(case)


def test_agrees_with_the_attention_of_equal_lengths():
    """iomx_launch_sdpa at position 0 on one sequence: the same operation, other roundings."""
    case = Attention(17, BF16, (8, 2), 64, 16, [50], [0], cache=False)
    got = decode(BF16, case.run())
    dims = {"q": (8, 50, 64), "k": (2, 50, 64), "v": (2, 50, 64)}
    t = [tensor(BF16, getattr(case, n)) for n in dims] + [iomx.DeviceTensor(BF16, (50, 512), fill=0)]
    views = [x.view() for x in t]
    rc, nbytes, _ = iomx.sdpa_workspace(*views, 0, 50)
    ws = iomx.Buffer(nbytes)
    iomx.check(iomx.sdpa(*views, 0, 50, ws), "sdpa")
    iomx.synchronize()
    other = decode(BF16, t[3].view().to_host())
    _, far, _ = case.exact()
    assert (np.abs(got - other) <= 2 * far + 2.0 ** -10).all()


@pytest.mark.parametrize("rows", [[1, 1, 1], [33, 60, 5]])
def test_the_same_result_every_time(rows):
    case = Attention(18, F16, (8, 2), 128, 16, rows, [900, 40, 700], tree=True)
    first = case.run()
    for _ in range(3):
        assert np.array_equal(first, case.run())


@pytest.mark.parametrize("rows", [[1, 1], [40, 9]])
def test_a_recorded_step_follows_the_lengths(rows):
    """Recorded once, replayed after the lengths, the table and the rows have changed, with eager work between."""
    cases = [Attention(20 + i, BF16, (8, 2), 64, 16, rows, ctx) for i, ctx in enumerate(([700, 90], [30, 500], [0, 16]))]
    M, N = max(c.M for c in cases), max(c.N for c in cases)
    for c in cases:
        c.table = np.pad(c.table, ((0, 0), (0, M - c.M)), constant_values=-1)
        c.k_pages, c.v_pages = (np.pad(p, ((0, N - c.N), (0, 0), (0, 0), (0, 0))) for p in (c.k_pages, c.v_pages))
        c.N, c.M = N, M
    t = cases[0].upload()
    views = {n: x.view() for n, x in t.items()}
    rc, nbytes, _ = iomx.sdpa_packed_workspace(max_rows=cases[0].max_rows, **views)
    iomx.check(rc)
    ws = iomx.Buffer(nbytes) if nbytes else None
    st = iomx.Stream()
    st.begin_capture()
    rc = iomx.sdpa_packed(max_rows=cases[0].max_rows, workspace=ws, stream=st, **views)
    graph = st.end_capture()
    iomx.check(rc)
    for c in cases + cases[::-1]:
        for name in ("q", "k", "v", "k_pages", "v_pages"):
            t[name].view().from_host(getattr(c, name))
        for name, value in (("table", c.table), ("lengths", [c.ctx])):
            t[name].view().from_host(np.asarray(value).astype(np.int32).view(np.uint32))
        t["out"].buf.fill(0x5A)
        iomx.synchronize()
        graph.launch(st)
        st.synchronize()
        got = t["out"].view().to_host()
        c.check(got)
        assert np.array_equal(got, c.run())     # the eager result, with a workspace of its own
    graph.close()
    st.close()


def test_two_streams_at_once():
    cases = [Attention(30 + i, BF16, (8, 2), 64, 16, rows, ctx) for i, (rows, ctx) in
             enumerate((([1, 1, 1], [2000, 3, 900]), ([200, 40], [0, 77])))]
    want = [c.run() for c in cases]
    streams = [iomx.Stream() for _ in cases]
    held = []
    for c in cases:
        t = c.upload()
        views = {n: x.view() for n, x in t.items()}
        rc, nbytes, _ = iomx.sdpa_packed_workspace(max_rows=c.max_rows, **views)
        held.append((t, views, iomx.Buffer(nbytes) if nbytes else None))
    iomx.synchronize()
    for _ in range(5):
        for c, st, (t, views, ws) in zip(cases, streams, held):
            iomx.check(iomx.sdpa_packed(max_rows=c.max_rows, workspace=ws, stream=st, **views))
    for st in streams:
        st.synchronize()
    for w, (t, views, ws) in zip(want, held):
        assert np.array_equal(w, views["out"].to_host())
    for st in streams:
        st.close()


def test_a_pool_of_more_than_four_gigabytes():
    """Page numbers whose bytes pass 32 bits."""
    P, Hkv, D, N = 64, 8, 128, 36000                       # 128 KiB a page, 4.4 GiB a pool
    case = Attention(40, F16, (8, 8), D, P, [1, 20], [150, 70])
    old_table, used = case.table.copy(), [int(x) for x in case.table[case.table >= 0]]
    far = {page: N - 1 - 7 * i for i, page in enumerate(used)}
    pools = [iomx.DeviceTensor(F16, (N, Hkv, P, D), fill=None) for _ in range(2)]
    for pool, data in zip(pools, (case.k_pages, case.v_pages)):
        for page in used:
            pool.view().select(0, far[page]).from_host(data[page])
    t = case.upload()
    t.update(k_pages=pools[0], v_pages=pools[1],
             table=ints([[far[x] if x >= 0 else -1 for x in row] for row in old_table]))
    for path in (0, 1):
        case.check(case.run(t=t, path=path))
    for x in t.values():
        x.free()


def test_padding_of_the_output_is_left_as_it_was():
    case = Attention(41, BF16, (3, 1), 16, 16, [5, 9], [3, 20])
    t = case.upload()
    case.run(t=t)
    raw = t["out"].raw().reshape(1, 3, 16, 16)              # 14 rows of 16
    assert (raw[0, :, 14:] == 0x5A5A).all()


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F16, 128), (BF16, 80), (F16, 32)])
@pytest.mark.parametrize("rows", [4, 8, 16, 32, 33, 70])
@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("tree", [False, True])
def test_every_division_of_the_work(dtype, D, rows, long, tree):
    """4 query heads on one KV head: 16 rows per KV head and fewer, up to 32, 64, 128 and more, each with
    contexts whose tokens stay with one workgroup and with ones that are shared out."""
    ctx = [2300, 0, 700, 1537] if long else [200, 0, 31, 64]
    case = Attention(50, dtype, (4, 1), D, 64, [rows, 1, rows - 1, rows // 2], ctx, tree=tree, tail=1)
    case.check(case.run())


@pytest.mark.parametrize("dtype,D", [(BF16, 144), (F16, 160), (BF16, 192), (F16, 208), (F16, 240), (BF16, 256)])
@pytest.mark.parametrize("rows", [4, 8, 16, 32, 33, 70])
@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("tree", [False, True])
def test_every_division_of_the_work_of_wide_heads(dtype, D, rows, long, tree):
    ctx = [2300, 0, 700, 1537] if long else [200, 0, 31, 64]
    case = Attention(54, dtype, (4, 1), D, 64, [rows, 1, rows - 1, rows // 2], ctx, tree=tree, tail=1)
    case.check(case.run())
    assert iomx.last_launch().kernel.decode() != "sdpa_packed_rows"


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_more_sequences_than_lanes(dtype):
    """The shares of 150 sequences, most of them short or without rows."""
    rng = np.random.default_rng(51)
    rows = rng.integers(0, 3, 150)
    ctx = rng.integers(0, 90, 150)
    ctx[[3, 64, 65, 149]] = [1900, 1500, 1100, 1300]
    rows[[3, 64, 149]] = [1, 2, 2]
    case = Attention(51, dtype, (2, 1), 64, 64, list(rows), list(ctx), tail=2)
    case.check(case.run())
    case = Attention(52, dtype, (2, 1), 64, 64, [1] * 150, list(ctx))
    case.check(case.run())


def test_a_long_context_of_one_sequence():
    """A piece for nearly every workgroup, and a context that ends just after a piece."""
    for ctx in (16384, 9001):
        case = Attention(53, BF16, (4, 2), 128, 128, [1], [ctx])
        case.check(case.run())
        case = Attention(53, F16, (4, 2), 64, 128, [12], [ctx], tree=True)
        case.check(case.run())


def test_a_table_wider_than_the_contexts():
    """Room for far more pages than there are: the work is divided by the lengths."""
    case = Attention(54, BF16, (8, 2), 64, 16, [1, 5, 0, 1], [300, 2, 9, 1111])
    case.table = np.pad(case.table, ((0, 0), (0, 3000)), constant_values=-1)
    case.M += 3000
    case.check(case.run())
