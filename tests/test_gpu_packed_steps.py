"""The operations on packed rows together, as a server with drafted tokens runs them: prompts of
different lengths in one step, then trees of drafted tokens, verified and accepted, on one growing
cache in pages.

A model of one attention layer (embedding, head-planar projections, rotary encoding at each row's
position, attention over pages, output projection to logits), BF16, random weights.  Every step's
operations are checked on the operands they met on the device: attention against its definition in
64 bits, appended rows bit for bit, log probabilities and likeliest tokens against the logits, and the
tokens of the whole run against the same model one token at a time.
"""
import numpy as np
import pytest

from iom_amd import iomx
from packed_cases import Attention, decode, encode, ints, starts_of, tensor
from test_gpu_token_logprobs import allowed, close, exact

pytestmark = pytest.mark.gpu

BF16, I32, F32, U32 = iomx.DT_BF16, iomx.DT_I32, iomx.DT_F32, iomx.DT_U32
HQ, HKV, D, VOCAB, PAGE, PAGES, SLOTS, THETA = 8, 2, 64, 700, 16, 100, 20, 10000.0
HIDDEN = 128


class Server:
    def __init__(self, sequences):
        rng = np.random.default_rng(99)
        mat = lambda rows, cols, s=1.0: tensor(BF16, encode(BF16, s * rng.standard_normal((rows, cols)) / np.sqrt(cols)))
        self.table = tensor(BF16, encode(BF16, rng.standard_normal((VOCAB, HIDDEN))))
        self.wq, self.wk, self.wv = mat(HQ * D, HIDDEN, 2.0), mat(HKV * D, HIDDEN, 2.0), mat(HKV * D, HIDDEN)
        self.wo = mat(VOCAB, HQ * D, 8.0)
        self.k_pages, self.v_pages = (iomx.DeviceTensor(BF16, (PAGES, HKV, PAGE, D), fill=0xFF) for _ in range(2))
        free = list(rng.permutation(PAGES))
        self.pages = np.array([[free.pop() for _ in range(SLOTS)] for _ in range(sequences)])
        self.page_table = ints(self.pages)
        self.lengths = [0] * sequences
        self.kept = [([], []) for _ in range(sequences)]      # raw key and value rows of each sequence

    def step(self, tokens, positions, starts, tree=None, children=None, top=4):
        """One forward pass over packed rows; returns their log probabilities and likeliest tokens, and
        what append() needs."""
        T, S = len(tokens), len(self.lengths)
        ids = tensor(U32, np.asarray(tokens, np.uint32).reshape(1, 1, T))
        x = iomx.DeviceTensor(BF16, (1, T, HIDDEN))
        status = iomx.Buffer(16)
        iomx.check(iomx.embedding(self.table.view(), ids.view(), x.view(), status))
        heads = {}
        for name, w, H in (("q", self.wq, HQ), ("k", self.wk, HKV), ("v", self.wv, HKV)):
            out = iomx.DeviceTensor(BF16, (1, H, T, D))
            iomx.check(iomx.linear(x.view(), w.view(), out.view(), 0, T, True, H, D), name)
            heads[name] = out.view().select(0, 0)
        at = ints([positions])
        turned = {}
        for name in "qk":
            out = iomx.DeviceTensor(BF16, heads[name].dims, fill=0xFF)
            iomx.check(iomx.rope_packed(heads[name], out.view(), at.view(), THETA))
            turned[name] = out.view()
        first, lengths = ints([starts]), ints([self.lengths])
        out = iomx.DeviceTensor(BF16, (T, HQ * D), fill=0x5A)
        masks = tensor(U32, tree) if tree is not None else None
        operands = dict(q=turned["q"], k=turned["k"], v=heads["v"], out=out.view(), starts=first.view(),
                        k_pages=self.k_pages.view(), v_pages=self.v_pages.view(), table=self.page_table.view(),
                        lengths=lengths.view(), tree=masks.view() if masks else None, max_rows=int(np.diff(starts).max()))
        rc, nbytes, _ = iomx.sdpa_packed_workspace(**operands)
        iomx.check(rc)
        iomx.check(iomx.sdpa_packed(workspace=iomx.Buffer(nbytes) if nbytes else None, **operands))
        logits = iomx.DeviceTensor(BF16, (1, T, VOCAB))
        rows = iomx.DeviceTensor.at(out.buf.ptr.value, BF16, (1, T, HQ * D))
        iomx.check(iomx.linear(rows.view(), self.wo.view(), logits.view(), 0, T, False, 1, VOCAB))
        given = tensor(I32, np.asarray(children, np.int32).view(np.uint32)) if children is not None else None
        results = {"logprobs": iomx.DeviceTensor(F32, given.dims) if given else None, "entropy": iomx.DeviceTensor(F32, (T, 1)),
                   "top_ids": iomx.DeviceTensor(I32, (T, top)), "top_logprobs": iomx.DeviceTensor(F32, (T, top))}
        views = {n: t.view() if t else None for n, t in results.items()}
        views.update(logits=logits.view().select(0, 0), tokens=given.view() if given else None)
        rc, nbytes, _ = iomx.token_logprobs_workspace(**views)
        iomx.check(rc)
        iomx.check(iomx.token_logprobs(workspace=iomx.Buffer(nbytes), **views))
        iomx.synchronize()
        self.check_attention(operands, starts, tree, out)
        got = {n: v.view().to_host() for n, v in results.items() if v}
        x_logits = decode(BF16, logits.view().select(0, 0).to_host())
        some = np.asarray(children) if children is not None else np.zeros((T, 1), np.int64)
        want_given, entropy, want_ids, tops = exact(x_logits, some, top)
        assert np.array_equal(got["top_ids"].view(np.int32), want_ids)
        as_float = lambda raw: raw.view(np.float32).astype(np.float64)
        close(as_float(got["top_logprobs"]), tops, allowed(x_logits, tops), "top")
        close(as_float(got["entropy"]), entropy, allowed(x_logits, entropy), "entropy")
        if given:
            close(as_float(got["logprobs"]), want_given, allowed(x_logits, want_given), "given")
        self.spread = np.abs(decode(BF16, out.view().to_host())) @ np.abs(decode(BF16, self.wo.view().to_host())).T
        return want_ids, x_logits, (turned["k"], heads["v"])

    def check_attention(self, operands, starts, tree, out):
        case = Attention.__new__(Attention)
        case.dtype, case.Hq, case.Hkv, case.D, case.P = BF16, HQ, HKV, D, PAGE
        case.rows, case.ctx, case.S = list(np.diff(starts)), self.lengths, len(self.lengths)
        case.starts, case.T, case.max_rows = np.asarray(starts), out.dims[0], operands["max_rows"]
        case.N, case.table, case.tree = PAGES, self.pages, tree
        for name in ("q", "k", "v", "k_pages", "v_pages"):
            setattr(case, name, operands[name].to_host())
        case.check(out.view().to_host())

    def append(self, kv, starts, rows=None):
        """The listed rows (or all) of a step to the cache, and what they were to the host's record."""
        k, v = kv
        listed = ints([rows]) if rows is not None else None
        iomx.check(iomx.cache_append_packed(k, v, self.k_pages.view(), self.v_pages.view(), ints([starts]).view(),
                                            self.page_table.view(), ints([self.lengths]).view(), listed.view() if listed else None))
        iomx.synchronize()
        raw_k, raw_v = k.to_host(), v.to_host()
        for s in range(len(self.lengths)):
            for e in range(starts[s], starts[s + 1]):
                row = e if rows is None else rows[e]
                self.kept[s][0].append(raw_k[:, row])
                self.kept[s][1].append(raw_v[:, row])
            self.lengths[s] += starts[s + 1] - starts[s]
        for pool, which in ((self.k_pages.view().to_host(), 0), (self.v_pages.view().to_host(), 1)):
            for s, n in enumerate(self.lengths):
                x = np.arange(n)
                assert np.array_equal(pool[self.pages[s, x // PAGE], :, x % PAGE], np.array(self.kept[s][which]))


def test_prompts_then_drafted_trees():
    rng = np.random.default_rng(7)
    prompts = [list(rng.integers(0, VOCAB, n)) for n in (37, 1, 90, 16)]
    S = len(prompts)
    server = Server(S)
    starts = [int(x) for x in starts_of([len(p) for p in prompts])]
    ids, logits, kv = server.step([t for p in prompts for t in p], [i for p in prompts for i in range(len(p))], starts)
    server.append(kv, starts)
    # the next token of each sequence, and its alternatives
    text = [list(p) for p in prompts]
    pending = []
    for s in range(S):
        row = starts[s + 1] - 1
        pending.append(int(ids[row, 0]))
    accepted_more = False
    for turn in range(4):
        # a tree for each sequence: its pending token, some guesses after it, guesses after those
        tokens, positions, masks, parents, counts = [], [], [], [], []
        for s in range(S):
            nodes, parent = [pending[s]], [-1]
            for j in range(1, 3 + 3 * s + turn):
                parent.append(int(rng.integers(max(-1, j - 3), j)))
                if parent[-1] < 0:
                    parent[-1] = 0
                nodes.append(int(rng.integers(0, VOCAB)))
            seen = []
            for j, p in enumerate(parent):
                seen.append((seen[p] if p >= 0 else 0) | 1 << j)
            depth = [bin(m).count("1") - 1 for m in seen]
            tokens.append(nodes); parents.append(parent); masks += seen; counts.append(len(nodes))
            positions += [server.lengths[s] + d for d in depth]
        first = [int(x) for x in starts_of(counts)]
        tree = np.array([[m & 0xFFFFFFFF] for m in masks], np.uint32)
        flat = [t for nodes in tokens for t in nodes]
        # a first pass proposes: the second node of each tree becomes the token that follows the root
        ids, _, _ = server.step(flat, positions, first, tree)
        for s in range(S):
            if counts[s] > 1:
                flat[first[s] + 1] = int(ids[first[s], 0])
        children = np.full((len(flat), 2), -1)
        for s in range(S):
            for j, p in enumerate(parents[s]):
                if p >= 0:
                    children[first[s] + p, 0 if children[first[s] + p, 0] < 0 else 1] = flat[first[s] + j]
        ids, logits, kv = server.step(flat, positions, first, tree, children)
        # greedy acceptance: from the root, follow the child that is the likeliest token
        accepted, keep = [], []
        for s in range(S):
            node, path = 0, [0]
            while True:
                best = int(ids[first[s] + node, 0])
                follow = [j for j, p in enumerate(parents[s]) if p == node and flat[first[s] + j] == best]
                if not follow:
                    pending[s] = best
                    break
                node = follow[0]
                path.append(node)
            accepted_more = accepted_more or len(path) > 1
            text[s] += [flat[first[s] + j] for j in path]
            keep.append(len(path))
            accepted += [first[s] + j for j in path]
        kept = [int(x) for x in starts_of(keep)]
        server.append(kv, kept, accepted)
        assert [server.lengths[s] for s in range(S)] == [len(t) for t in text]
    assert accepted_more
    # the same text, a sequence at a time in one causal pass: each token is the likeliest, or as near to
    # it as other roundings can bring it.  Of the two logits each rounds to BF16 in either pass (4 half
    # steps of the largest); each component of the attention's result may lie 4 half steps apart (its
    # own rounding in either pass, and those of the keys, values and queries it is made of, which are
    # half a step each of components that it averages), so a logit by 4 half steps of the sum of its
    # terms' magnitudes.
    for s in range(S):
        alone = Server(1)
        ids, logits, _ = alone.step(text[s], list(range(len(text[s]))), [0, len(text[s])])
        begin = len(prompts[s])
        for i in range(begin, len(text[s])):
            row = logits[i - 1]
            gap = row[ids[i - 1, 0]] - row[text[s][i]]
            assert gap <= 2.0 ** -8 * (4 * np.abs(row).max() + 2 * 4 * alone.spread[i - 1].max()), (s, i, gap)
