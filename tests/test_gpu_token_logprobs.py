"""GPU tests of iomx_launch_token_logprobs against its definition in 64 bits."""
import numpy as np
import pytest

from iom_amd import iomx
from packed_cases import decode, encode, tensor

pytestmark = pytest.mark.gpu

BF16, F16, F32, I32 = iomx.DT_BF16, iomx.DT_F16, iomx.DT_F32, iomx.DT_I32


@pytest.fixture(scope="module", autouse=True)
def _device():
    assert iomx.device_count() >= 1
    iomx.check(iomx.lib().iomx_set_device(0))
    yield


def exact(x, tokens, K):
    """log probabilities, entropy, ids and log probabilities of the likeliest, in 64 bits"""
    V = x.shape[-1]
    flat = x.reshape(-1, V)
    with np.errstate(all="ignore"):
        top = flat.max(-1, keepdims=True)
        bad = np.isnan(flat).any(-1) | np.isposinf(flat).any(-1) | np.isneginf(flat).all(-1)
        e = np.exp(flat - top)
        total = e.sum(-1, keepdims=True)
        whole = top + np.log(total)
        p = e / total
        entropy = (np.log(total) - np.where(e > 0, (flat - top) * p, 0).sum(-1, keepdims=True))
        logs = flat - whole
    logs[bad], entropy[bad] = np.nan, np.nan
    t = tokens.reshape(flat.shape[0], -1)
    inside = (t >= 0) & (t < V)
    given = np.where(inside, np.take_along_axis(logs, np.where(inside, t, 0), 1), -np.inf)
    ids = np.argsort(-flat, axis=-1, kind="stable")[:, :K]
    tops = np.take_along_axis(logs, ids, 1)
    ids[bad] = -1
    lead = x.shape[:-1]
    return given.reshape(*lead, -1), entropy.reshape(*lead, 1), ids.reshape(*lead, K), tops.reshape(*lead, K)


def allowed(x, want):
    """Distance of a log probability or an entropy.  With r = the spread of the finite logits: an
    exponential's argument is off by a rounding of the difference and one of its product with log2 e
    (r * 2^-23 together), the function by 2^-22, a sum of V of them in F32, in chains of at most
    V / 64 + 64, by that many half steps in the worst case; what is left over is the roundings of the
    logarithm, the maximum and the result."""
    V = x.shape[-1]
    finite = np.where(np.isfinite(x), x, 0)
    r = min(104.0, float(np.ptp(finite)) if x.size else 0.0)      # past that an exponential is zero
    big = float(np.abs(finite).max(initial=0))
    total = r * 2.0 ** -22 + 2.0 ** -21 + (V / 64 + 64) * 2.0 ** -24
    return (2 + np.log(V)) * total + 2.0 ** -21 * (big + np.abs(np.where(np.isfinite(want), want, 0)))


def run(dtype, raw, tokens=None, K=0, entropy=True, lead_view=None):
    dims = raw.shape[:-1]
    t = {"logits": tensor(dtype, raw)}
    if tokens is not None:
        t["tokens"] = tensor(I32, tokens.astype(np.int32).view(np.uint32))
        t["logprobs"] = iomx.DeviceTensor(F32, tokens.shape, fill=0x5A)
    if entropy:
        t["entropy"] = iomx.DeviceTensor(F32, dims + (1,), fill=0x5A)
    if K:
        t["top_ids"] = iomx.DeviceTensor(I32, dims + (K,), fill=0x5A)
        t["top_logprobs"] = iomx.DeviceTensor(F32, dims + (K,), fill=0x5A)
    views = {n: x.view() for n, x in t.items()}
    rc, nbytes, _ = iomx.token_logprobs_workspace(**views)
    iomx.check(rc)
    ws = iomx.Buffer(nbytes) if nbytes else None
    if ws:
        ws.fill(0xFF)
    iomx.check(iomx.token_logprobs(workspace=ws, **views), "token_logprobs")
    iomx.synchronize()
    got = {n: views[n].to_host() for n in t if n not in ("logits", "tokens")}
    for n in got:       # padding slots are as they were
        raw_out = t[n].raw()
        rows, cols = dims[-1], t[n].dims[-1]
        tiles = raw_out.reshape(-1, -(-rows // 16), -(-cols // 16), 16, 16).transpose(0, 1, 3, 2, 4)
        tiles = tiles.reshape(-1, -(-rows // 16) * 16, -(-cols // 16) * 16)
        assert (tiles[:, rows:] == 0x5A5A5A5A).all() and (tiles[:, :, cols:] == 0x5A5A5A5A).all(), n
    for x in t.values():
        x.free()
    if ws:
        ws.free()
    return {n: (a.view(np.float32).astype(np.float64) if n != "top_ids" else a.view(np.int32)) for n, a in got.items()}


def close(got, want, far, what):
    # F32 ends at (2 - 2^-23) 2^127: what lies half a step (2^103) past it rounds to an infinity (the
    # distance of the type's lowest value from its highest is twice that)
    want = np.where(want <= -(2.0 ** 128 - 2.0 ** 103), -np.inf, want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert np.array_equal(np.isneginf(got), np.isneginf(want)), what
    fine = np.isfinite(want)
    off = np.abs(got - want)[fine]
    assert (off <= np.broadcast_to(far, want.shape)[fine]).all(), (what, off.max(), np.min(far))


def check(dtype, raw, tokens, K, entropy=True):
    x = decode(dtype, raw)
    got = run(dtype, raw, tokens, K, entropy)
    given, ent, ids, tops = exact(x, tokens if tokens is not None else np.zeros(raw.shape[:-1] + (1,), np.int64), K)
    if tokens is not None:
        close(got["logprobs"], given, allowed(x, given), "logprobs")
    if entropy:
        close(got["entropy"], ent, allowed(x, ent), "entropy")
    if K:
        assert np.array_equal(got["top_ids"], ids)
        close(got["top_logprobs"], tops, allowed(x, tops), "top_logprobs")


def make(seed, dtype, dims, scale=3.0):
    rng = np.random.default_rng(seed)
    return encode(dtype, rng.standard_normal(dims) * scale), rng


SHAPES = [(1, 1), (1, 2), (16, 16), (3, 33), (17, 255), (16, 4096), (5, 4097), (40, 1000), (1, 32000), (33, 8192), (2, 60001),
          (4, 1, 777), (3, 2, 19, 300), (70, 1, 5000)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dims", SHAPES)
def test_rows(dtype, dims):
    raw, rng = make(1, dtype, dims)
    V = dims[-1]
    for K, G in ((1, 1), (min(8, V), 3), (min(32, V), 17), (0, 2)):
        tokens = rng.integers(-2, V + 2, dims[:-1] + (G,))
        check(dtype, raw, tokens, K)


def test_each_output_alone():
    raw, rng = make(2, BF16, (20, 3000))
    tokens = rng.integers(0, 3000, (20, 2))
    check(BF16, raw, tokens, 0, entropy=False)
    check(BF16, raw, None, 5, entropy=False)
    check(BF16, raw, None, 0, entropy=True)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_ties_go_to_the_lowest_id(dtype):
    rng = np.random.default_rng(3)
    raw = encode(dtype, rng.integers(0, 3, (18, 5000)))            # three different logits
    check(dtype, raw, rng.integers(0, 5000, (18, 1)), 32)
    raw = encode(dtype, np.zeros((3, 700)))
    check(dtype, raw, rng.integers(0, 700, (3, 1)), 32)
    raw = encode(dtype, np.where(rng.integers(0, 2, (3, 700)), 0.0, -0.0))    # equal zeros of either sign
    check(dtype, raw, rng.integers(0, 700, (3, 1)), 32)
    # the largest at the ends, and in an order that gets better or worse all along
    ramp = encode(dtype, np.stack([np.arange(2000), -np.arange(2000)] * 3) / 64)
    check(dtype, ramp, rng.integers(0, 2000, (6, 1)), 32)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_masked_logits(dtype):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((20, 2500)) * 4
    x[:, 2400:] = -np.inf
    x[3, rng.permutation(2500)[:2480]] = -np.inf                   # twenty left, 32 asked for
    x[4, :] = -np.inf
    x[4, 1777] = 1.5                                               # one left: log probability 0, entropy 0
    x[5, :] = -np.inf                                              # nothing left
    x[6, :1200] = -np.inf                                          # nothing in the first half
    x[7, 9], x[8, 2499], x[9, 0] = np.nan, np.inf, np.inf
    x[10, :] = np.nan
    lowest = {BF16: -3.3895313892515355e38, F16: -65504.0, F32: -3.4028234663852886e38}[dtype]
    x[11, 100:] = lowest                                           # masked with the lowest value instead
    x[12, :] = lowest                                              # all of them equal
    x[13, :] = 6.0e4                                               # far from zero
    tokens = rng.integers(0, 2500, (20, 4))
    tokens[4, 0] = 1777
    check(dtype, encode(dtype, x), tokens, 32)


def test_far_apart_logits():
    """Distributions with almost all of the probability in one token, and nearly even ones."""
    rng = np.random.default_rng(5)
    for scale in (1e-3, 30.0, 1e4):
        raw = encode(F32, rng.standard_normal((17, 3000)) * scale)
        check(F32, raw, rng.integers(0, 3000, (17, 2)), 8)


def test_views_with_strides():
    raw, rng = make(6, BF16, (3, 10, 900))
    owner = iomx.DeviceTensor(BF16, (6, 2, 10, 900), fill=0xFF)
    view = owner.view().select(1, 1).slice(0, 0, 3, 2)
    view.from_host(raw)
    outs = iomx.DeviceTensor(F32, (2, 3, 10, 1), fill=0x5A)
    ids = iomx.DeviceTensor(I32, (3, 10, 4), fill=0x5A)
    tops = iomx.DeviceTensor(F32, (3, 10, 4), fill=0x5A)
    views = dict(logits=view, entropy=outs.view().select(0, 1), top_ids=ids.view(), top_logprobs=tops.view())
    rc, nbytes, _ = iomx.token_logprobs_workspace(**views)
    iomx.check(rc)
    iomx.check(iomx.token_logprobs(workspace=iomx.Buffer(nbytes) if nbytes else None, **views))
    iomx.synchronize()
    x = decode(BF16, raw)
    _, ent, want, _ = exact(x, np.zeros((3, 10, 1), np.int64), 4)
    close(outs.view().select(0, 1).to_host().view(np.float32).astype(np.float64), ent, allowed(x, ent), "entropy")
    assert (outs.view().select(0, 0).to_host() == 0x5A5A5A5A).all()
    assert np.array_equal(ids.view().to_host().view(np.int32), want)


def test_the_same_result_every_time_and_recorded():
    raw, rng = make(7, F32, (50, 20000))
    tokens = rng.integers(0, 20000, (50, 1))
    first = run(F32, raw, tokens, 20)
    second = run(F32, raw, tokens, 20)
    assert all(np.array_equal(first[n], second[n]) for n in first)
    t = {"logits": tensor(F32, raw), "tokens": tensor(I32, tokens.astype(np.int32).view(np.uint32)),
         "logprobs": iomx.DeviceTensor(F32, (50, 1)), "entropy": iomx.DeviceTensor(F32, (50, 1)),
         "top_ids": iomx.DeviceTensor(I32, (50, 20)), "top_logprobs": iomx.DeviceTensor(F32, (50, 20))}
    views = {n: x.view() for n, x in t.items()}
    rc, nbytes, _ = iomx.token_logprobs_workspace(**views)
    ws = iomx.Buffer(nbytes) if nbytes else None
    st = iomx.Stream()
    iomx.synchronize()
    st.begin_capture()
    rc = iomx.token_logprobs(workspace=ws, stream=st, **views)
    graph = st.end_capture()
    iomx.check(rc)
    for replay in range(3):
        shifted = np.roll(raw, replay * 17, axis=-1)
        t["logits"].view().from_host(shifted)
        for n in first:
            t[n].buf.fill(0x5A)
        iomx.synchronize()
        graph.launch(st)
        st.synchronize()
        want = run(F32, shifted, tokens, 20)
        for n in first:
            got = views[n].to_host()
            got = got.view(np.int32) if n == "top_ids" else got.view(np.float32).astype(np.float64)
            assert np.array_equal(got, want[n]), (replay, n)
    graph.close()
    st.close()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [40000, 300001])
def test_large_vocabularies_of_few_and_of_equal_logits(dtype, V):
    """Rows with fewer finite logits than places (a grammar that allows a few tokens), rows of equal
    logits, equal largest logits in many cells, in one cell, and just more of them than places."""
    rng = np.random.default_rng(8)
    x = rng.standard_normal((12, V)) * 2
    x[0, :] = -np.inf
    x[0, rng.permutation(V)[:10]] = rng.standard_normal(10)
    x[1, :] = -np.inf
    x[1, rng.permutation(V)[:200]] = rng.standard_normal(200)
    x[2, :] = 0.25
    x[3, rng.permutation(V)[:400]] = 20.0
    x[4, 777:1400] = 20.0
    x[5, rng.permutation(V)[:33]] = 20.0
    x[6, rng.permutation(V)[:31]] = 20.0
    x[7, :] = -np.inf
    x[7, 5:300] = 1.0                                              # in one or two cells
    x[8, :] = -np.inf
    x[8, V - 20:] = 1.0
    x[9, :] = np.where(np.arange(V) % 3 == 0, -np.inf, -7.0)
    x[10, V - 1] = 30.0
    for K in (1, 20, 32):
        check(dtype, encode(dtype, x), rng.integers(0, V, (12, 2)), K)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("V", [100, 686, 2560, 2561, 40000, 150001])
def test_masks_of_the_lowest_value(dtype, V):
    """Forbidden tokens at the type's lowest finite value: fewer allowed ones than places, in every row a
    different number; and rows of two values, of which the larger is rarer than the places are many."""
    lowest = {BF16: -3.3895313892515355e38, F16: -65504.0, F32: -3.4028234663852886e38}[dtype]
    rng = np.random.default_rng(11)
    x = np.full((18, V), lowest)
    for r in range(12):
        some = rng.permutation(V)[:3 * r]
        x[r, some] = rng.standard_normal(len(some)) * 2
    x[12] = np.where(np.arange(V) % 2 == 0, lowest, -np.inf)
    x[13, 7] = -lowest
    x[14, rng.permutation(V)[:9]] = lowest / 2
    x[15, rng.permutation(V)[:9]] = -lowest
    x[16] = rng.standard_normal(V) * 2
    x[17] = np.sort(rng.standard_normal(V))
    for K in (1, 20, 32):
        check(dtype, encode(dtype, x), rng.integers(0, V, (18, 2)), K)


@pytest.mark.parametrize("dtype,V,K", [(BF16, 64, 1), (F16, 65, 1), (BF16, 1024, 20), (F32, 1025, 20), (F16, 1472, 20),
                                       (BF16, 1473, 20), (BF16, 2432, 32), (F16, 2433, 32), (F32, 2433, 32)])
def test_vocabularies_of_few_cells(dtype, V, K):
    """On both sides of the sizes up to which a row's logits are picked from without cells."""
    rng = np.random.default_rng(13)
    x = rng.standard_normal((40, V)) * 2
    x[3] = 0.25
    x[4] = -np.inf
    x[4, V // 2] = 1.0
    x[5, :V // 2] = -np.inf
    x[6] = np.sort(x[6])
    x[7] = np.sort(x[7])[::-1]
    x[8] = np.round(x[8])
    check(dtype, encode(dtype, x), rng.integers(0, V, (40, 1)), K)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows", [512, 513])
def test_few_and_many_rows(dtype, rows):
    """The last number of rows from which several waves pick, and one more; ordinary rows, equal logits,
    few finite ones, and more candidates than are held."""
    V = 9001
    rng = np.random.default_rng(12)
    x = rng.standard_normal((rows, V)) * 2
    for r in range(0, 60, 6):
        x[r] = 0.25
        x[r + 1, rng.permutation(V)[:40 * r + 3]] = 20.0
        x[r + 2] = -np.inf
        x[r + 2, rng.permutation(V)[:r + 1]] = rng.standard_normal(r + 1)
        x[r + 3] = -65504.0
        x[r + 3, rng.permutation(V)[:r]] = 1.5
        x[r + 4, 17 * r:17 * r + 300] = 20.0
        x[r + 5] = np.sort(x[r + 5])
    check(dtype, encode(dtype, x), rng.integers(0, V, (rows, 1)), 32)


def test_the_workspace_has_to_be_there():
    t = {"logits": iomx.DeviceTensor(BF16, (3, 500)), "entropy": iomx.DeviceTensor(F32, (3, 1), fill=0x5A)}
    views = {n: x.view() for n, x in t.items()}
    rc, nbytes, align = iomx.token_logprobs_workspace(**views)
    assert rc == 0 and nbytes > 0 and align == 256
    small = iomx.Buffer(nbytes - 1)
    assert iomx.token_logprobs(**views) == iomx.ERR_INVALID
    assert iomx.token_logprobs(workspace=small, **views) == iomx.ERR_INVALID
    off = iomx.Buffer(nbytes + 256)
    assert iomx.token_logprobs(workspace=iomx.Buffer.at(off.ptr.value + 64, nbytes), **views) == iomx.ERR_INVALID
    iomx.synchronize()
    assert (t["entropy"].view().to_host() == 0x5A5A5A5A).all()
