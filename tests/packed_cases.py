"""Plain 64-bit forms of the operations on packed rows, and the device operands of a case."""
import numpy as np

import datagen
from iom_amd import iomx

HALF_STEP = {iomx.DT_BF16: 2.0 ** -8, iomx.DT_F16: 2.0 ** -11, iomx.DT_F32: 2.0 ** -24}


def encode(dtype, values):
    """float values -> raw elements of the leaf, round to nearest even."""
    values = np.asarray(values, np.float32)
    if dtype == iomx.DT_F32:
        return values.view(np.uint32)
    if dtype == iomx.DT_F16:
        return values.astype(np.float16).view(np.uint16)
    return datagen.bf16_rne(values).reshape(values.shape)


def decode(dtype, raw):
    """raw elements -> float64, exactly."""
    if dtype == iomx.DT_F32:
        return raw.view(np.float32).astype(np.float64)
    if dtype == iomx.DT_F16:
        return raw.view(np.float16).astype(np.float64)
    return (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def tensor(dtype, raw, fill=0xFF):
    """A device tensor of these raw elements; its padding slots hold `fill` bytes (0xFF..: NaN in
    the floating leaves, -1 in the integers)."""
    raw = np.asarray(raw)
    t = iomx.DeviceTensor(dtype, raw.shape, fill=fill)
    t.view().from_host(raw)
    return t


def ints(rows):
    return tensor(iomx.DT_I32, np.atleast_2d(np.asarray(rows, np.int64)).astype(np.int32).view(np.uint32))


def starts_of(rows, first=0):
    return np.concatenate([[first], first + np.cumsum(rows)])


class Attention:
    """One request: packed rows, a pool of pages and who sees whom, with its 64-bit result.

    rows, ctx: per sequence.  first / tail: rows before the first and behind the last sequence.
    """

    def __init__(self, seed, dtype, heads, D, P, rows, ctx, tree=False, first=0, tail=0, cache=True, scale=1.0,
                 spare_pages=2, max_rows=None):
        rng = np.random.default_rng(seed)
        self.dtype, (self.Hq, self.Hkv), self.D, self.P = dtype, heads, D, P
        self.rows, self.ctx = list(rows), list(ctx) if cache else [0] * len(rows)
        self.S, self.cache = len(rows), cache
        self.starts = starts_of(rows, first)
        self.T = int(max(1, self.starts[-1] + tail))
        self.max_rows = max(1, max(rows)) if max_rows is None else max_rows
        draw = lambda dims, s=1.0: encode(dtype, rng.standard_normal(dims) * s)
        self.q = draw((self.Hq, self.T, D), scale)
        self.k, self.v = draw((self.Hkv, self.T, D)), draw((self.Hkv, self.T, D))
        used = [-(-c // P) for c in self.ctx]
        self.M = max(1, max(used))
        self.N = max(1, sum(used) + spare_pages)
        order = list(rng.permutation(self.N))
        self.table = np.full((self.S, self.M), -1, np.int64)
        for s, n in enumerate(used):
            for m in range(n):
                self.table[s, m] = order.pop()
        # slots that hold no token are NaN
        nan = encode(dtype, np.full((self.N, self.Hkv, P, D), np.nan))
        self.k_pages, self.v_pages = nan.copy(), nan.copy()
        for s, c in enumerate(self.ctx):
            for x in range(0, c, P):
                n = min(P, c - x)
                for pool in (self.k_pages, self.v_pages):
                    pool[self.table[s, x // P], :, :n] = draw((self.Hkv, n, D))
        self.tree = None
        if tree:
            words = max(1, -(-max(rows) // 32))
            self.tree = np.zeros((self.T, words), np.uint32)
            for s, n in enumerate(rows):
                seen = []
                for j in range(n):
                    parent = int(rng.integers(max(-1, j - 4), j)) if j else -1
                    seen.append((seen[parent] if parent >= 0 else 0) | 1 << j)
                    for w in range(words):
                        self.tree[self.starts[s] + j, w] = seen[-1] >> 32 * w & 0xFFFFFFFF

    def sees(self, s, i):
        """Own rows that row i of sequence s sees."""
        n = self.rows[s]
        if self.tree is None:
            return np.arange(n) <= i
        j = np.arange(n)
        bits = self.tree[self.starts[s] + i]
        inside = j < 32 * bits.size
        return inside & ((bits[np.where(inside, j >> 5, 0)] >> (j & 31)) & 1 != 0)

    def exact(self):
        """(out [T, Hq*D] with NaN where nothing is written, the allowed distance, rows written)"""
        dec = lambda raw: decode(self.dtype, raw)
        q, k, v, kp, vp = map(dec, (self.q, self.k, self.v, self.k_pages, self.v_pages))
        u, G = HALF_STEP[self.dtype], self.Hq // self.Hkv
        out = np.full((self.T, self.Hq * self.D), np.nan)
        far = np.zeros_like(out)
        written = np.zeros(self.T, bool)
        for s in range(self.S):
            n, c = self.rows[s], self.ctx[s]
            a = self.starts[s]
            x = np.arange(c)
            slots = self.table[s, x // self.P] if c else x
            present = (slots >= 0) & (slots < self.N)
            x, slots = x[present], slots[present]
            todo = range(min(n, self.max_rows))
            if not n:
                continue
            mask = np.array([np.concatenate([np.ones(len(x), bool), self.sees(s, i)]) for i in todo])
            for h in range(self.Hkv):
                kk = np.concatenate([kp[slots, h, x % self.P], k[h, a:a + n]])
                vv = np.concatenate([vp[slots, h, x % self.P], v[h, a:a + n]])
                for g in range(h * G, h * G + G):
                    qq = q[g, a:a + len(todo)]
                    with np.errstate(all="ignore"):
                        scores = np.where(mask, qq @ kk.T / np.sqrt(self.D), -np.inf)
                        top = scores.max(-1, keepdims=True)
                        e = np.exp(scores - np.where(np.isneginf(top), 0, top))
                        e = np.where(mask, e, 0)
                        total = e.sum(-1, keepdims=True)
                        p = e / np.where(total == 0, 1, total)
                    cols = slice(g * self.D, (g + 1) * self.D)
                    for i in todo:
                        m = mask[i]
                        with np.errstate(all="ignore"):
                            o = p[i, m] @ vv[m] if m.any() else np.zeros(self.D)
                            weight = p[i, m] @ np.abs(vv[m]) if m.any() else np.zeros(self.D)
                            # a score is a sum of D exact products in F32 (D roundings of partial sums no larger than
                            # sum |q k|), scaled and subtracted (4 more): it moves its probability by that much,
                            # and the normaliser as much again
                            # (an infinite score is exact)
                            wide = np.abs(qq[i]) @ np.abs(kk[m]).T
                            wide = np.where(np.isfinite(wide), wide, 0).max(initial=0) / np.sqrt(self.D)
                        moved = 2 * (self.D + 4) * 2.0 ** -24 * wide
                        # probabilities round to the leaf (u), exponentials and sums to F32, the result to the leaf (u);
                        # F16 probabilities below 2^-14 of the largest round to steps of 2^-24
                        tiny = m.sum() * 2.0 ** -25 * np.abs(vv[m]).max(0, initial=0) if self.dtype == iomx.DT_F16 else 0
                        out[a + i, cols] = o
                        far[a + i, cols] = (u * np.abs(o) + (u * 1.02 + moved + (m.sum() + 64) * 2.0 ** -24) * weight
                                            + tiny + (2.0 ** -25 if self.dtype == iomx.DT_F16 else 2.0 ** -133))
            written[a:a + len(todo)] = True
        return out, far, written

    def upload(self):
        """The device operands, in the order of iomx.sdpa_packed's arguments."""
        t = {"q": tensor(self.dtype, self.q), "k": tensor(self.dtype, self.k), "v": tensor(self.dtype, self.v),
             "out": iomx.DeviceTensor(self.dtype, (self.T, self.Hq * self.D), fill=0x5A), "starts": ints(self.starts)}
        if self.cache:
            t.update(k_pages=tensor(self.dtype, self.k_pages), v_pages=tensor(self.dtype, self.v_pages),
                     table=ints(self.table), lengths=ints(self.ctx))
        if self.tree is not None:
            t["tree"] = tensor(iomx.DT_U32, self.tree)
        return t

    def run(self, path=0, t=None, keep=False):
        """The raw logical result [T, Hq*D]."""
        own = t is None
        t = t or self.upload()
        views = {n: x.view() if isinstance(x, iomx.DeviceTensor) else x for n, x in t.items()}
        rc, nbytes, align = iomx.sdpa_packed_workspace(max_rows=self.max_rows, **views)
        iomx.check(rc, "workspace")
        assert align in (1, 16, 64, 256)
        ws = iomx.Buffer(nbytes) if nbytes else None
        if ws:
            ws.fill(0xFF)
        iomx.check(iomx.sdpa_packed(max_rows=self.max_rows, workspace=ws, path=path, **views), "sdpa_packed")
        iomx.synchronize()
        out = views["out"].to_host()
        if ws:
            ws.free()
        if own and not keep:
            for x in t.values():
                x.free()
        return out

    def check(self, raw):
        out, far, written = self.exact()
        got = decode(self.dtype, raw)
        assert np.array_equal(raw[~written], np.full_like(raw[~written], 0x5A5A)), "rows of no sequence were written"
        got, want, far = got[written], out[written], far[written]
        special = ~np.isfinite(want)
        assert np.array_equal(np.isnan(got[special]), np.isnan(want[special]))
        inf = special & ~np.isnan(want)
        assert np.array_equal(got[inf], want[inf])
        off = np.where(special, 0, np.abs(got - want) - far)
        worst = np.unravel_index(np.argmax(np.where(np.isnan(off), np.inf, off)), off.shape) if off.size else None
        assert not off.size or off[worst] <= 0, (worst, got[worst], want[worst], far[worst])
        finite = ~special
        if finite.any():
            return float(np.max(np.abs(got - want)[finite] / np.maximum(far[finite], 1e-300)))
        return 0.0
