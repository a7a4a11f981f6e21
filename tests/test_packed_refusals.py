"""What the operations on packed rows refuse, and the workspace queries: host code only, no GPU
(every request here is turned down before a launch)."""
import ctypes as C

import pytest

from iom_amd import iomx
from test_sdpa_workspace_query import dense_view

BF16, F16, F32, F64, I8 = iomx.DT_BF16, iomx.DT_F16, iomx.DT_F32, iomx.DT_F64, iomx.DT_I8
INVALID, UNSUPPORTED, OVERFLOW = iomx.ERR_INVALID, iomx.ERR_UNSUPPORTED, iomx.ERR_OVERFLOW


def ref(v):
    return None if v is None else C.byref(v)


def attention_views(Hq=8, Hkv=2, T=20, D=64, S=3, N=9, P=32, M=4, W=1):
    return {"q": dense_view((Hq, T, D), 0), "k": dense_view((Hkv, T, D), 1), "v": dense_view((Hkv, T, D), 2),
            "out": dense_view((T, Hq * D), 3), "starts": dense_view((1, S + 1), 4),
            "k_pages": dense_view((N, Hkv, P, D), 5), "v_pages": dense_view((N, Hkv, P, D), 6),
            "table": dense_view((S, M), 7), "lengths": dense_view((1, S), 8), "tree": dense_view((T, W), 9)}


ORDER = ("q", "k", "v", "out", "starts", "k_pages", "v_pages", "table", "lengths", "tree")


def query(views, dtype=BF16, max_rows=20):
    nbytes, align = C.c_uint64(77), C.c_uint64(78)
    rc = iomx.lib().iomx_sdpa_packed_workspace(dtype, *[ref(views[n]) for n in ORDER], max_rows, C.byref(nbytes),
                                               C.byref(align))
    return rc, nbytes.value, align.value


def launch(views, dtype=BF16, max_rows=20, workspace=None, nbytes=0, path=0):
    return iomx.lib().iomx_launch_sdpa_packed(dtype, *[ref(views[n]) for n in ORDER], max_rows, workspace, nbytes,
                                              path, None)


def changed(**dims):
    """The views with other extents for some of them (None: left out)."""
    views = attention_views()
    for slot, name in enumerate(ORDER):
        if name in dims:
            views[name] = None if dims[name] is None else dense_view(dims[name], slot)
    return views


NO_CACHE = dict(k_pages=None, v_pages=None, table=None, lengths=None)


@pytest.mark.parametrize("views", [attention_views(), changed(tree=None), changed(**NO_CACHE), changed(tree=None, **NO_CACHE),
                                   attention_views(Hq=6, Hkv=6, D=40, P=7)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_the_query_accepts(views, dtype):
    rc, nbytes, align = query(views, dtype)
    assert rc == 0 and align >= 1 and (nbytes == 0) == (align == 1)


@pytest.mark.parametrize("dims,want", [
    (dict(q=(7, 20, 64), out=(20, 448)), INVALID),          # seven query heads on two
    (dict(q=(20, 64)), INVALID),
    (dict(k=(2, 21, 64)), INVALID),                         # another number of rows
    (dict(v=(2, 20, 48)), INVALID),
    (dict(out=(20, 500)), INVALID),
    (dict(out=(1, 20, 512)), INVALID),
    (dict(starts=(2, 4)), INVALID),
    (dict(starts=(1, 1)), INVALID),                         # no sequence
    (dict(starts=(1, 5)), INVALID),                         # four sequences, three table rows
    (dict(table=(2, 4)), INVALID),
    (dict(lengths=(3, 1)), INVALID),
    (dict(k_pages=(9, 1, 32, 64)), INVALID),
    (dict(v_pages=(9, 2, 16, 64)), INVALID),
    (dict(k_pages=(2, 32, 64), v_pages=(2, 32, 64)), INVALID),
    (dict(tree=(19, 1)), INVALID),
    (dict(v_pages=None), INVALID),                          # half a cache
    (dict(table=None), INVALID),
    (dict(lengths=None, k_pages=None, v_pages=None), INVALID),
    (dict(q=None), INVALID),
    (dict(out=None), INVALID),
    (dict(starts=None), INVALID),
    (dict(q=(8, 20, 272), k=(2, 20, 272), v=(2, 20, 272), out=(20, 8 * 272), k_pages=(9, 2, 32, 272),
          v_pages=(9, 2, 32, 272)), UNSUPPORTED),           # heads wider than 256
])
def test_attention_refuses_extents(dims, want):
    assert query(changed(**dims))[0] == want
    assert launch(changed(**dims)) == want


def test_attention_refuses_the_rest():
    assert query(attention_views(), F32)[0] == UNSUPPORTED and launch(attention_views(), F64) == UNSUPPORTED
    assert query(attention_views(), max_rows=0)[0] == INVALID
    assert launch(attention_views(), path=7) == INVALID and launch(attention_views(), path=-1) == INVALID
    for name in ORDER:
        if name == "out":
            continue
        views = attention_views()
        views["out"].base = views[name].base
        assert launch(views) == INVALID, name
    views = attention_views()
    views["k"].base += 8                                    # storages are 16-byte aligned
    assert launch(views) == INVALID
    assert launch(attention_views(P=1 << 20, M=1 << 20)) == OVERFLOW
    assert iomx.lib().iomx_sdpa_packed_workspace(BF16, *[ref(attention_views()[n]) for n in ORDER], 20, None, None) == INVALID


def rope(dtype=BF16, x=(4, 20, 64), out=(4, 20, 64), positions=(1, 20), theta=10000.0, same=False):
    views = [dense_view(x, 0), dense_view(out, 0 if same else 1), dense_view(positions, 2)]
    return iomx.lib().iomx_launch_rope_packed(dtype, *map(ref, views), theta, None)


@pytest.mark.parametrize("kw,want", [
    (dict(out=(4, 21, 64)), INVALID), (dict(x=(20, 64), out=(20, 64)), INVALID), (dict(positions=(1, 19)), INVALID),
    (dict(positions=(20, 1)), INVALID), (dict(theta=0.5), INVALID), (dict(theta=float("nan")), INVALID),
    (dict(theta=1e39), INVALID), (dict(same=True), INVALID), (dict(dtype=F64), UNSUPPORTED), (dict(dtype=I8), UNSUPPORTED),
    (dict(dtype=99), UNSUPPORTED), (dict(x=(4, 20, 40), out=(4, 20, 40)), UNSUPPORTED),
    (dict(x=(4, 20, 528), out=(4, 20, 528)), UNSUPPORTED)])
def test_rope_packed_refuses(kw, want):
    assert rope(**kw) == want


def append(dtype=BF16, alias=None, **dims):
    full = dict(k=(2, 20, 64), v=(2, 20, 64), k_pages=(9, 2, 32, 64), v_pages=(9, 2, 32, 64), starts=(1, 4), table=(3, 4),
                lengths=(1, 3), rows=(1, 11))
    full.update(dims)
    views = {n: None if d is None else dense_view(d, i) for i, (n, d) in enumerate(full.items())}
    if alias:
        views[alias[0]].base = views[alias[1]].base
    return iomx.lib().iomx_launch_cache_append_packed(dtype, *map(ref, views.values()), None)


@pytest.mark.parametrize("kw,want", [
    (dict(v=(2, 21, 64)), INVALID), (dict(k=None), INVALID), (dict(v_pages=None), INVALID), (dict(table=None), INVALID),
    (dict(k_pages=(9, 3, 32, 64), v_pages=(9, 3, 32, 64)), INVALID), (dict(v_pages=(9, 2, 32, 80)), INVALID),
    (dict(starts=(1, 3)), INVALID), (dict(lengths=(1, 4)), INVALID), (dict(rows=(2, 11)), INVALID),
    (dict(alias=("k", "k_pages")), INVALID), (dict(alias=("v", "k_pages")), INVALID), (dict(alias=("rows", "v_pages")), INVALID),
    (dict(dtype=99), UNSUPPORTED),
    (dict(k=(2, 20, 40), v=(2, 20, 40), k_pages=(9, 2, 32, 40), v_pages=(9, 2, 32, 40)), UNSUPPORTED),
    (dict(k_pages=(9, 2, 1 << 20, 64), v_pages=(9, 2, 1 << 20, 64), table=(3, 1 << 20)), OVERFLOW)])
def test_cache_append_packed_refuses(kw, want):
    assert append(**kw) == want


LOGPROBS = dict(logits=(2, 5, 100), tokens=(2, 5, 3), logprobs=(2, 5, 3), entropy=(2, 5, 1), top_ids=(2, 5, 8),
                top_logprobs=(2, 5, 8))


def logprobs_views(alias=None, **dims):
    full = dict(LOGPROBS, **dims)
    views = {n: None if d is None else dense_view(d, i) for i, (n, d) in enumerate(full.items())}
    if alias:
        views[alias[0]].base = views[alias[1]].base
    return views


def logprobs(dtype=BF16, **kw):
    views = logprobs_views(**kw)
    rc = iomx.lib().iomx_launch_token_logprobs(dtype, *map(ref, views.values()), None, 0, None)
    nbytes, align = C.c_uint64(0), C.c_uint64(0)
    assert iomx.lib().iomx_token_logprobs_workspace(dtype, *map(ref, views.values()), C.byref(nbytes), C.byref(align)) == rc
    return rc


@pytest.mark.parametrize("kw,want", [
    (dict(logprobs=None), INVALID), (dict(tokens=None), INVALID), (dict(top_ids=None), INVALID), (dict(logits=None), INVALID),
    (dict(tokens=None, logprobs=None, entropy=None, top_ids=None, top_logprobs=None), INVALID),
    (dict(tokens=(2, 5, 2)), INVALID), (dict(entropy=(2, 5, 2)), INVALID), (dict(entropy=(5, 1)), INVALID),
    (dict(entropy=(2, 4, 1)), INVALID), (dict(tokens=(1, 5, 3), logprobs=(1, 5, 3)), INVALID),
    (dict(logits=(2, 5, 7)), INVALID),                                              # eight of seven
    (dict(top_ids=(2, 5, 33), top_logprobs=(2, 5, 33)), UNSUPPORTED),
    (dict(logits=(1, 1, 1 << 24), tokens=None, logprobs=None, entropy=(1, 1, 1), top_ids=None, top_logprobs=None), UNSUPPORTED),
    (dict(alias=("logprobs", "logits")), INVALID), (dict(alias=("top_logprobs", "logprobs")), INVALID),
    (dict(alias=("entropy", "tokens")), INVALID),
    (dict(dtype=F64), UNSUPPORTED), (dict(dtype=I8), UNSUPPORTED), (dict(dtype=-1), UNSUPPORTED)])
def test_token_logprobs_refuses(kw, want):
    assert logprobs(**kw) == want


def test_attention_needs_its_workspace():
    views = attention_views(M=64)                    # room for 2048 tokens: their parts are joined
    rc, nbytes, align = query(views)
    assert rc == 0 and nbytes > 0 and align == 256
    aligned = 0x7E0000000000
    assert launch(views) == INVALID
    assert launch(views, workspace=aligned, nbytes=nbytes - 1) == INVALID
    assert launch(views, workspace=aligned + 64, nbytes=nbytes) == INVALID
    assert query(attention_views(M=4))[1:] == (0, 1)  # 128 tokens stay with their workgroups


def test_token_logprobs_needs_its_workspace():
    views = logprobs_views()
    nbytes, align = C.c_uint64(0), C.c_uint64(0)
    assert iomx.lib().iomx_token_logprobs_workspace(BF16, *map(ref, views.values()), C.byref(nbytes), C.byref(align)) == 0
    assert nbytes.value > 0 and align.value == 256
    for workspace, given in ((None, 0), (0x7E0000000000, nbytes.value - 1), (0x7E0000000000 + 16, nbytes.value)):
        assert iomx.lib().iomx_launch_token_logprobs(BF16, *map(ref, views.values()), workspace, given, None) == INVALID
    assert iomx.lib().iomx_token_logprobs_workspace(BF16, *map(ref, views.values()), None, None) == INVALID


def test_borrowed_memory_is_left_alone():
    """Tensors, buffers and streams of another library: no allocation is made for them, none is freed."""
    t = iomx.DeviceTensor.at(0x7E0000000000, BF16, (3, 20, 40))
    assert t.nbytes == 3 * 32 * 48 * 2 and t.view().cview().base == 0x7E0000000000
    t.free()
    assert t.view().cview().base is None
    stream = iomx.Stream.at(0)
    assert not stream.h
    stream.close()
    b = iomx.Buffer.at(0x7E0000000000, 64)
    b.free()
    assert not b.ptr
