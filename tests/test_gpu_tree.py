"""The operators of a pass over drafted trees -- plan, attention,
verification, cache commit and fork -- against plain implementations in 64
bits, at the sizes and masks where they can go wrong; their run together in
QwenModel; and a captured pass replayed."""
import ctypes
import math

import numpy as np
import pytest
import torch

from golem_amd import capi, synth
from golem_amd.qwen import QwenModel, rope_tables
from tests.gpu_util import log

pytestmark = pytest.mark.gpu
vp = capi.vp


def offsets(sizes):
    return np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)


def random_parents(g, sizes, fanout):
    """Parents of every tree: chains for fanout 1, else an earlier node not far before."""
    out = []
    for t in sizes:
        for i in range(t):
            out.append(-1 if i == 0 else i - 1 if fanout == 1 else int(g.integers(max(0, (i - 1) // fanout - 1), i)))
    return np.array(out, np.int32).reshape(-1)


# ---- the plan -----------------------------------------------------------------


def plan_reference(sizes, parents, prefix, context, max_nodes, M):
    words = (max_nodes + 31) // 32
    rows, positions = np.full(M, -1, np.int32), np.full(M, -1, np.int32)
    mask = np.zeros((M, words), np.uint32)
    first = offsets(sizes)
    for b, t in enumerate(sizes):
        seen = {}
        for i in range(min(t, max_nodes)):
            m, p = first[b] + i, parents[first[b] + i]
            if p == -1:
                seen[i] = [i]
            elif 0 <= p < i and p in seen:
                seen[i] = seen[p] + [i]
            else:
                continue
            at = int(prefix[b]) + len(seen[i]) - 1
            if prefix[b] < 0 or at >= context:
                continue
            rows[m], positions[m] = m, at
            for j in seen[i]:
                mask[m, j // 32] |= np.uint32(1 << (j % 32))
    return rows, positions, mask


def run_plan(dev, sizes, parents, prefix, context, half, max_nodes, M):
    g = synth.rng(3)
    cos, sin = g.standard_normal((2, context, half)).astype(np.float32)
    words = (max_nodes + 31) // 32
    out = [dev.full((M,), 77, np.int32), dev.full((M,), 77, np.int32), dev.full((M, words), 77, np.int32),
           dev.full((M, half), 77.0), dev.full((M, half), 77.0)]
    held = [dev.put(x) for x in (offsets(sizes), np.append(parents, 0).astype(np.int32),
                                 np.append(prefix, 0).astype(np.int32), cos, sin)]
    capi.call("gx_qwen_tree_plan", dev.ctx.ptr, len(sizes), M, max_nodes, *map(vp, held), half, context,
              *map(vp, out))
    rows, positions, mask, oc, os = [dev.get(x) for x in out]
    wr, wp, wm = plan_reference(sizes, parents, prefix, context, max_nodes, M)
    np.testing.assert_array_equal(rows, wr)
    np.testing.assert_array_equal(positions, wp)
    np.testing.assert_array_equal(mask.view(np.uint32), wm)
    np.testing.assert_array_equal(oc, np.where(wp[:, None] >= 0, cos[np.maximum(wp, 0)], 0))
    np.testing.assert_array_equal(os, np.where(wp[:, None] >= 0, sin[np.maximum(wp, 0)], 0))


@pytest.mark.parametrize("sizes,fanout,max_nodes,pad", [
    ([1], 1, 1, 0), ([5], 1, 5, 0), ([6, 1, 4], 2, 6, 3), ([0, 3, 0, 0, 2, 0], 2, 3, 0), ([64, 33, 31, 32], 3, 64, 1),
    ([65, 96], 4, 96, 0), ([512, 200], 1, 512, 0), ([511], 7, 512, 5), ([40] * 70, 3, 40, 9), ([], 1, 4, 6),
])
def test_plan(dev, sizes, fanout, max_nodes, pad):
    g = synth.rng(1)
    parents = random_parents(g, sizes, fanout)
    prefix = g.integers(0, 50, len(sizes))
    run_plan(dev, sizes, parents, prefix, 600, 32, max_nodes, sum(sizes) + pad)


@pytest.mark.parametrize("half", [1, 5, 12, 64, 128])
def test_plan_rotation_rows(dev, half):
    """Head widths off the 16-byte pieces, and rows past one workgroup's."""
    sizes = [70, 3, 33]
    run_plan(dev, sizes, random_parents(synth.rng(2), sizes, 3), np.array([9, 0, 4]), 100, half, 70, 110)


def test_plan_leaves_out_what_has_no_place(dev):
    # a later parent, itself, below -1, and everything below those; a second
    # root; positions past the context; a negative prefix; more nodes than max_nodes
    parents = np.array([-1, 0, 2, 2, 3, 7, 1, -1, 7, -5, 9] + [-1, 0, 1, 2] + [-1, 0] + [-1, 0, 1, 2, 3, 4], np.int32)
    run_plan(dev, [11, 4, 2, 6], parents, np.array([3, 18, -1, 0]), 20, 16, 11, 25)
    run_plan(dev, [6], np.array([-1, 0, 1, 2, 3, 4], np.int32), np.array([0]), 20, 16, 4, 6)


# ---- attention -----------------------------------------------------------------


def long_context(n, max_nodes, heads, kv):
    """A context past which a call is for the kernel whose workgroups have several tiles, and a little more."""
    tiles = n * kv * ((max_nodes * (heads // kv) + 31) // 32)
    return 32 * (7 * 8 * max(min(64, 256 // tiles), 1) + 2)


class Attention:
    """A case's arrays: caches of nslots conversations filled with NaN past
    each prefix, draft buffers filled with NaN past the last token."""

    def __init__(self, seed, sizes, prefix, heads, kv, hd, fanout=3, nslots=None, pad=0, max_nodes=None, spread=2.0,
                 long=False):
        g = synth.rng(seed)
        self.sizes, self.prefix = list(sizes), np.array(prefix, np.int32)
        self.heads, self.kv, self.hd = heads, kv, hd
        self.n, self.tokens = len(sizes), sum(sizes)
        self.M = self.tokens + pad
        self.max_nodes = max_nodes or max(max(sizes), 1)
        self.words = (self.max_nodes + 31) // 32
        self.nslots = nslots or self.n
        self.slots = g.permutation(self.nslots)[:self.n].astype(np.int32)
        self.context = (int(max(prefix)) + 8) // 8 * 8
        self.dctx = (max(self.M, 1) + 7) // 8 * 8
        f16 = np.float16
        self.q = (spread * g.standard_normal((self.M, heads, hd))).astype(f16)
        self.k = g.standard_normal((self.nslots, kv, self.context, hd)).astype(f16)
        self.v = g.standard_normal((self.nslots, kv, self.context, hd)).astype(f16)
        self.kd = g.standard_normal((kv, self.dctx, hd)).astype(f16)
        self.vd = g.standard_normal((kv, self.dctx, hd)).astype(f16)
        for s in range(self.nslots):
            p = int(self.prefix[list(self.slots).index(s)]) if s in self.slots else 0
            self.k[s, :, p:], self.v[s, :, p:] = np.nan, np.nan
        self.kd[:, self.tokens:], self.vd[:, self.tokens:] = np.nan, np.nan
        if long:  # a context, launched for in whole, that has the tiles of a tree side by side in a workgroup
            short, self.context = self.context, long_context(self.n, self.max_nodes, heads, kv)
            more = ((0, 0), (0, 0), (0, self.context - short), (0, 0))
            self.k, self.v = (np.pad(x, more, constant_values=np.nan) for x in (self.k, self.v))
        self.long = long
        self.first = offsets(sizes)
        parents = random_parents(g, sizes, fanout)
        self.mask = plan_reference(sizes, parents, self.prefix, 1 << 30, self.max_nodes, self.M)[2]

    def sees(self, b, i):
        return [j for j in range(self.sizes[b]) if self.mask[self.first[b] + i, j // 32] >> np.uint32(j % 32) & 1]

    def reference(self):
        """The definition in float64, and for each output its tolerances: see `tolerance`."""
        out = np.zeros((self.M, self.heads, self.hd))
        tol = np.zeros((self.M, self.heads, 2))
        group = self.heads // self.kv
        with np.errstate(invalid="ignore", over="ignore"):
            for b in range(self.n):
                s, p = self.slots[b], max(int(self.prefix[b]), 0)
                for i in range(self.sizes[b]):
                    m, on = self.first[b] + i, self.first[b] + np.array(self.sees(b, i), int)
                    for h in range(self.heads):
                        c = h // group
                        k = np.concatenate([self.k[s, c, :p], self.kd[c, on]]).astype(np.float64)
                        v = np.concatenate([self.v[s, c, :p], self.vd[c, on]]).astype(np.float64)
                        if len(k) == 0:
                            continue
                        q = self.q[m, h].astype(np.float64)
                        x = (k * q).sum(1) / math.sqrt(self.hd)
                        w = np.exp(x - x.max())
                        out[m, h] = (w[:, None] * v).sum(0) / w.sum()
                        tol[m, h] = self.tolerance(np.abs(k * q).sum(1).max() / math.sqrt(self.hd), len(k),
                                                   np.abs(x).max(), np.abs(v[np.isfinite(v)]).max())
        return out, tol

    def tolerance(self, dot, count, top, vmax):
        """A score is a float32 sum of hd exact products, hd roundings of at
        most 2^-24 of `dot`, and the factor's and product's two of |x|; in base
        2 the difference to the maximum adds two more; e^ takes these absolute
        errors as relative ones, twice (numerator and sum).  exp2 is within
        2^-22, the probability's two fp16 parts within 2^-22 of it, and every
        sum of `count` positive terms within count * 2^-24 (products: of their
        magnitudes), three of them with the shares' joins.  All of it times the
        largest value.  That is the worst of every element; the root of a row's
        mean square has roundings of either sign, N of them adding up to the
        root of N, and a second bound with those."""
        e = 2.0 ** -24
        return [vmax * (2 * (hd * dot + 4 * (top + 12)) * e + 2 * 2 ** -22 + 3 * n * e)
                for hd, n in ((self.hd, count + 64), (self.hd ** 0.5, (count + 64) ** 0.5))]

    def run(self, dev, max_prefix=None, q8=False, fill=77.0, lone=False, nslots=None, skew=0):
        M, width = self.M, self.heads * self.hd
        kc = self.k.reshape(self.nslots, self.kv, self.context, self.hd // 8, 8).transpose(0, 1, 3, 2, 4)
        kd = self.kd.reshape(self.kv, self.dctx, self.hd // 8, 8).transpose(0, 2, 1, 3)
        h = [dev.put(np.ascontiguousarray(x).view(np.int16)) for x in (
            self.q, kc, self.v.transpose(0, 1, 3, 2), kd, self.vd.transpose(0, 2, 1))]
        first, mask, prefix, slots = (dev.put(x) for x in (self.first, self.mask.view(np.int32), self.prefix, self.slots))
        out = dev.full((M * width + skew,), fill)[skew:]
        q, sc, qs = (dev.full((M * width + skew,), 55, np.int8)[skew:].reshape(M, width), dev.full((M, width // 32), 55.0),
                     dev.full((M, width // 32), 55, np.int32)) if q8 else (None, None, None)
        mp = max_prefix if max_prefix is not None else self.context if self.long else int(max(self.prefix.max(), 0))
        size = capi.size_out("gx_qwen_attention_tree_workspace_bytes", self.n, M, self.max_nodes, self.heads, self.kv,
                             self.hd, mp)
        ws = dev.full((max(size, 256),), 0xFF, np.uint8)
        capi.call("gx_qwen_attention_tree", dev.ctx.ptr, vp(h[0]), self.n, M, self.max_nodes, vp(first), vp(mask),
                  vp(prefix), mp, self.heads, self.kv, self.hd, vp(h[1]), vp(h[2]), self.context, vp(h[3]), vp(h[4]),
                  self.dctx, vp(out), vp(q), vp(sc), vp(qs), vp(ws), size, None if lone else vp(slots),
                  nslots or self.nslots)
        o = dev.get(out).reshape(M, self.heads, self.hd)
        return (o, dev.get(q), dev.get(sc), dev.get(qs)) if q8 else o

    def check(self, dev, **kw):
        got, (want, tol) = self.run(dev, **kw), self.reference()
        got, tail = got[:self.tokens], got[self.tokens:]
        off, tol = np.abs(got - want[:self.tokens]), tol[:self.tokens]
        rms = np.sqrt((off ** 2).mean(2))
        log(f"  sizes {self.sizes[:6]} prefix {self.prefix[:6]}: worst {(off / np.maximum(tol[..., :1], 1e-30)).max():.3f}, "
            f"rows' rms {(rms / np.maximum(tol[..., 1], 1e-30)).max():.3f} of the tolerances")
        assert np.all(off <= tol[..., :1]) and np.all(rms <= tol[..., 1])
        assert np.all(tail == 77.0)
        return got


# A tile a workgroup that covers the keys, the keys over several, and several tiles a workgroup.
FORMS = [(70, None, False), (1100, None, False), (70, 64, True)]
HEADS = [(4, 2, 64), (8, 2, 32), (6, 2, 96), (8, 2, 128), (3, 3, 64), (16, 1, 128), (5, 1, 32), (32, 8, 128)]


@pytest.mark.parametrize("heads,kv,hd", HEADS)
@pytest.mark.parametrize("sizes,prefix", [([1], [0]), ([1], [1]), ([7], [45]), ([33, 1, 12], [64, 200, 31])])
def test_attention_heads(dev, heads, kv, hd, sizes, prefix):
    Attention(10, sizes, prefix, heads, kv, hd).check(dev)


@pytest.mark.parametrize("heads,kv,hd", HEADS)
@pytest.mark.parametrize("sizes,prefix", [([65], [0]), ([40, 1, 70], [64, 200, 31])])
def test_attention_heads_of_long_contexts(dev, heads, kv, hd, sizes, prefix):
    Attention(10, sizes, prefix, heads, kv, hd, long=True).check(dev)


@pytest.mark.parametrize("prefix", [0, 1, 7, 8, 31, 32, 33, 63, 64, 65, 127, 128, 129, 500, 1023, 2050])
def test_attention_prefixes(dev, prefix):
    Attention(11, [5, 9], [prefix, max(prefix - 3, 0)], 4, 2, 64).check(dev)
    Attention(11, [5, 37], [prefix, max(prefix - 3, 0)], 4, 2, 64, long=True).check(dev)


@pytest.mark.parametrize("sizes", [[31], [32], [33], [64, 2], [3, 64, 30], [100], [129, 5], [1] * 11, [0, 4, 0, 3]])
def test_attention_trees(dev, sizes):
    g = synth.rng(12)
    prefix = list(g.integers(0, 90, len(sizes)))
    for long in (False, True):
        Attention(12, sizes, prefix, 4, 2, 64, nslots=len(sizes) + 2, pad=3, long=long).check(dev)


def test_attention_chain_of_512(dev):
    for long in (False, True):
        Attention(13, [512], [40], 2, 1, 32, fanout=1, long=long).check(dev)


def test_attention_many_trees(dev):
    g = synth.rng(14)
    Attention(14, list(g.integers(1, 5, 130)), list(g.integers(0, 70, 130)), 2, 1, 32).check(dev)


@pytest.mark.parametrize("sizes,max_nodes", [([9, 4], 70), ([9, 4], 40), ([8, 4], None), ([9, 4], 512)])
def test_attention_launched_for_a_longer_prefix(dev, sizes, max_nodes):
    """max_prefix above every prefix (a captured pass), and rows of more mask words than the trees need."""
    a = Attention(15, sizes, [100, 3], 8, 2, 128, max_nodes=max_nodes)
    a.k = np.concatenate([a.k, np.full_like(a.k, np.nan)] * 20, 2)
    a.v = np.concatenate([a.v, np.full_like(a.v, np.nan)] * 20, 2)
    a.context = a.k.shape[2]
    a.check(dev, max_prefix=a.context)


def test_attention_large_scores(dev):
    """Scores of hundreds: one key takes all, as the maximum moves from tile to tile."""
    for long in (False, True):
        Attention(16, [20], [700], 4, 2, 64, spread=60.0, long=long).check(dev)


@pytest.mark.parametrize("heads,kv,hd,prefix", [(4, 2, 32, 3), (32, 8, 128, 300), (4, 4, 96, 40), (8, 2, 128, 1500),
                                                (8, 1, 64, 5000)])
def test_attention_one_tile(dev, heads, kv, hd, prefix):
    """Trees that fill a tile of rows, and fill it but for a few, beside empty ones and shorter prefixes."""
    most = 32 * kv // heads
    Attention(25, [most, 0, 1, max(most - 1, 1)], [prefix, 5, prefix // 2, 0], heads, kv, hd, pad=2).check(dev)
    Attention(26, [1, most], [prefix, prefix + 9], heads, kv, hd, fanout=1, max_nodes=most).check(dev)


@pytest.mark.parametrize("sizes,prefix,long", [([11, 30], [333, 60], False), ([11, 30], [333, 60], True),
                                               ([10, 3], [333, 60], False), ([10, 3], [1333, 60], False)])
def test_attention_q8_form_is_the_floats(dev, orc, sizes, prefix, long):
    a = Attention(17, sizes, prefix, 6, 2, 96, pad=2, long=long)
    o, q, sc, qs = a.run(dev, q8=True)
    b = orc.Batch(np.ascontiguousarray(o[:a.tokens].reshape(a.tokens, -1))).quantize()
    np.testing.assert_array_equal(q[:a.tokens], b.q_rows())
    scale = np.abs(o[:a.tokens].reshape(a.tokens, -1, 32)).max(2).astype(np.float32) / np.float32(127)
    np.testing.assert_array_equal(sc[:a.tokens], scale.astype(np.float16).astype(np.float32))
    np.testing.assert_array_equal(qs[:a.tokens], q[:a.tokens].reshape(a.tokens, -1, 32).sum(2, dtype=np.int32))
    assert np.all(q[a.tokens:] == 55) and np.all(sc[a.tokens:] == 55.0) and np.all(qs[a.tokens:] == 55)


@pytest.mark.parametrize("prefix,max_nodes,long", FORMS)
def test_attention_outputs_of_any_alignment(dev, prefix, max_nodes, long):
    """Outputs off the alignment of their wide stores: floats by 4 bytes, bytes by 1."""
    a = Attention(24, [7, 2], [prefix, 9], 4, 2, 64, max_nodes=max_nodes, pad=1, long=long)
    for x, y in zip(a.run(dev, q8=True), a.run(dev, q8=True, skew=1)):
        np.testing.assert_array_equal(x, y)


@pytest.mark.parametrize("long", [False, True])
def test_attention_masks_of_any_kind(dev, long):
    """Bits that are no tree's, bits past the tree's nodes, and nodes that see nothing."""
    a = Attention(18, [40, 6, 3], [50, 0, 0], 4, 2, 64, max_nodes=64, long=long)
    g = synth.rng(19)
    a.mask[:] = g.integers(0, 1 << 32, a.mask.shape, dtype=np.uint64).astype(np.uint32)
    a.mask[a.first[1] + 2] = 0
    a.mask[a.first[2]:a.first[2] + 3] = np.uint32(0xFFFFFFF8)  # past its three nodes only
    a.mask[a.first[2]:, 1] = 0
    got = a.check(dev)
    assert np.all(got[a.first[1] + 2] == 0) and np.all(got[a.first[2]:] == 0)


@pytest.mark.parametrize("prefix,max_nodes,long", FORMS)
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_attention_hidden_values_stay_hidden(dev, bad, prefix, max_nodes, long):
    """Infinite and NaN keys and values of nodes that a node does not see
    reach nothing of it; those it sees reach it as they would in float64.  An
    element that shares its tile with a hidden one is summed again key by key,
    another order of the same sum: within the same tolerance of the float64
    result; every other keeps its bits."""
    a = Attention(20, [6, 5], [prefix, 9], 4, 2, 64, fanout=1, max_nodes=max_nodes, long=long)
    a.mask[:] = 0
    for b in range(2):
        for i in range(a.sizes[b]):  # nodes see themselves and the next but one before
            a.mask[a.first[b] + i, 0] = (1 << i) | (1 << max(i - 2, 0))
    clean = a.run(dev)
    a.vd[0, 3, 7] = bad          # node 3 of tree 0, seen by 3 and 5
    a.kd[1, a.first[1] + 1] = bad  # node 1 of tree 1, seen by 1 and 3
    got, (want, tol) = a.run(dev), a.reference()
    touched = np.zeros(got.shape, bool)
    touched[[3, 5], :2, 7] = True
    touched[[a.first[1] + 1, a.first[1] + 3], 2:] = True
    again = np.zeros(got.shape, bool)
    again[:6, :2, 7] = True
    np.testing.assert_array_equal(got[~touched & ~again], clean[~touched & ~again])
    near = again & ~touched
    assert np.all(np.abs(got[near] - want[near]) <= np.broadcast_to(tol[..., :1], got.shape)[near])
    np.testing.assert_array_equal(got[[3, 5], :2, 7], want[[3, 5], :2, 7])
    rows = a.first[1] + np.array([1, 3])
    assert np.all(np.isnan(got[rows, 2:])) and np.all(np.isnan(want[rows, 2:]))


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("heads,hd,nodes", [(4, 64, 80), (8, 128, 47), (2, 32, 190)])
def test_attention_tiles_in_halves(dev, heads, hd, nodes, long):
    """Trees of five and six tiles of rows, the last ones by halves of each
    step: prefixes that end in either half, a NaN query and hidden NaN and
    infinite values in the last tile."""
    kv = heads // 4 if heads > 4 else heads // 2
    for prefix in (0, 20, 40, 64, 333):
        Attention(27, [nodes, 3], [prefix, 50], heads, kv, hd, long=True).check(dev)
    a = Attention(28, [nodes], [77], heads, kv, hd, long=long)
    clean = a.run(dev)
    a.q[nodes - 2] = np.nan
    a.vd[:, nodes - 1] = np.nan
    a.vd[0, nodes - 3, 5] = np.inf
    seen = [nodes - 3 in a.sees(0, i) for i in range(nodes)]
    got, (want, tol) = a.run(dev), a.reference()
    assert np.all(np.isnan(got[nodes - 2:]))
    group = heads // a.kv
    for i in range(nodes - 2):
        off = np.zeros((heads, hd), bool)
        off[:group, 5] = seen[i]
        assert np.all(got[i][off] == np.inf)
        assert np.all(np.abs(got[i][~off] - want[i][~off]) <= np.broadcast_to(tol[i, :, :1], off.shape)[~off])
    assert np.isfinite(clean).all() and not all(seen)


@pytest.mark.parametrize("prefix,max_nodes,long", [(100, None, False), (1100, None, False), (100, 64, True)])
def test_attention_infinite_cached_values(dev, prefix, max_nodes, long):
    a = Attention(21, [3], [prefix], 4, 2, 64, max_nodes=max_nodes, long=long)
    a.v[a.slots[0], 0, 41, 5], a.v[a.slots[0], 1, 99, 0] = np.inf, -np.inf
    got, (want, tol) = a.run(dev), a.reference()
    fine = np.isfinite(want)
    assert (~fine).sum() == 3 * 4
    np.testing.assert_array_equal(got[~fine], want[~fine])
    assert np.all(np.abs(got - np.where(fine, want, 0))[fine] <= np.broadcast_to(tol[..., :1], got.shape)[fine])


@pytest.mark.parametrize("prefix,max_nodes,long", FORMS)
def test_attention_nan_query_is_its_own(dev, prefix, max_nodes, long):
    a = Attention(22, [9], [prefix], 4, 2, 64, max_nodes=max_nodes, long=long)
    clean = a.run(dev)
    a.q[4] = np.nan
    got = a.run(dev)
    assert np.all(np.isnan(got[4]))
    rest = np.arange(9) != 4
    np.testing.assert_array_equal(got[rest], clean[rest])


def test_attention_one_conversation_and_clamped_slots(dev):
    """slots NULL: every tree over one conversation's caches, each with its
    prefix; a slot out of range reads the nearest; a prefix past max_prefix is
    cut to it and a negative one sees nothing."""
    a = Attention(23, [4, 7], [60, 60], 4, 2, 64)
    a.slots[:] = 0
    a.k[0], a.v[0] = np.where(np.isnan(a.k[0]), 0, a.k[0]), np.where(np.isnan(a.v[0]), 0, a.v[0])
    a.prefix[1] = 33
    a.check(dev, lone=True)
    a.slots[:] = [-4, 9]
    got = a.run(dev, nslots=1)
    a.slots[:] = 0
    want = a.run(dev)
    np.testing.assert_array_equal(got, want)
    a.prefix[:] = [1 << 30, -5]
    got = a.run(dev, max_prefix=50)
    a.prefix[:] = [50, 0]
    np.testing.assert_array_equal(got, a.run(dev, max_prefix=50))


@pytest.mark.parametrize("max_nodes,max_prefix", [(5, 300), (64, 300), (64, 262144)])
def test_attention_past_32_bits(dev, max_nodes, max_prefix):
    """A conversation whose cache begins past 2^32 bytes (and 2^31 elements)."""
    kv, hd, ctx, nslots = 2, 64, 262144, 68
    n = nslots * kv * hd * ctx  # 2.3e9 elements
    t = dev.torch
    kc = t.zeros(n, dtype=t.float16, device="cuda").view(nslots, kv, hd // 8, ctx, 8)
    vc = t.zeros(n, dtype=t.float16, device="cuda").view(nslots, kv, hd, ctx)
    a = Attention(24, [5], [300], 4, kv, hd, max_nodes=max_nodes)
    k, v = a.k[0, :, :300], a.v[0, :, :300]
    kc[-1, :, :, :300] = t.from_numpy(k.reshape(kv, 300, hd // 8, 8).transpose(0, 2, 1, 3).copy()).cuda()
    vc[-1, :, :, :300] = t.from_numpy(v.transpose(0, 2, 1).copy()).cuda()
    kd = dev.put(a.kd.reshape(kv, a.dctx, hd // 8, 8).transpose(0, 2, 1, 3).copy().view(np.int16))
    vd = dev.put(a.vd.transpose(0, 2, 1).copy().view(np.int16))
    first, mask, prefix, slot, q = (dev.put(x) for x in (a.first, a.mask.view(np.int32), a.prefix,
                                                         np.array([nslots - 1], np.int32), a.q.view(np.int16)))
    out = dev.full((5, 4 * hd), 0.0)
    size = capi.size_out("gx_qwen_attention_tree_workspace_bytes", 1, 5, max_nodes, 4, kv, hd, max_prefix)
    ws = dev.empty((size,), np.uint8)
    capi.call("gx_qwen_attention_tree", dev.ctx.ptr, vp(q), 1, 5, max_nodes, vp(first), vp(mask), vp(prefix), max_prefix, 4, kv,
              hd, vp(kc), vp(vc), ctx, vp(kd), vp(vd), a.dctx, vp(out), None, None, None, vp(ws), size, vp(slot), nslots)
    want, tol = a.reference()
    assert np.all(np.abs(dev.get(out).reshape(5, 4, hd) - want) <= tol[..., :1])


# ---- verification ----------------------------------------------------------------


def chances(x, temperature):
    x = x.astype(np.float64) / temperature
    with np.errstate(invalid="ignore"):
        e = np.exp(x - x.max())
        return e / e.sum()


def verify_reference(sizes, parents, tokens, logits, draft, temperature, draft_temperature, u, max_nodes):
    """The walk from the definition: after each child that is turned down, the
    target's residual against the drafts' distribution without the tokens tried."""
    first, V = offsets(sizes), logits.shape[1]
    path = np.full((len(sizes), max_nodes), -1, np.int32)
    counts, nxt = [], []
    for b, t in enumerate(sizes):
        t = min(t, max_nodes)
        if t == 0:
            counts.append(0)
            nxt.append(-1)
            continue
        kept, v = [0], first[b]
        while True:
            kids = [m for m in range(first[b] + 1, first[b] + t) if parents[m] == v - first[b]]
            go, tried = None, set()
            row = logits[v]
            if temperature == 0:
                pick = 0
                for i in range(1, V):
                    if row[i] > row[pick]:
                        pick = i
                go = next((m for m in kids if tokens[m] == pick), None)
            elif not np.any(row > -np.inf) or np.any(np.isnan(row)) or np.any(row == np.inf):
                pick = -1
            else:
                p = chances(row, temperature)
                left = p.copy()
                q = None if draft is None else chances(draft[v], draft_temperature)
                if q is not None and not np.all(np.isfinite(q)):
                    kids = []
                for m in kids:
                    x = int(tokens[m])
                    if not 0 <= x < V or x in tried:
                        continue
                    if q is None:
                        if float(u[m]) * left.sum() < left[x]:
                            go = m
                            break
                        left[x] = 0
                    else:
                        if q.sum() <= 0 or left.sum() <= 0:
                            break
                        qn = q / q.sum()
                        if float(u[m]) * qn[x] * left.sum() < left[x]:
                            go = m
                            break
                        left = np.maximum(left - left.sum() * qn, 0)
                        q[x] = 0
                    tried.add(x)
                if left.sum() <= 0:
                    left = p
                cum = np.cumsum(left)
                pick = int(np.searchsorted(cum, float(u[first[b]]) * cum[-1], side="right"))
                pick = min(pick, int(np.nonzero(left)[0][-1]))
            if go is None:
                break
            kept.append(go - first[b])
            v = go
        counts.append(len(kept))
        nxt.append(pick)
        path[b, :len(kept)] = kept
    return path, np.array(counts, np.int32), np.array(nxt, np.int32)


def run_verify(dev, sizes, parents, tokens, logits, draft, temperature, draft_temperature, u, max_nodes, ld=0):
    M, V = logits.shape
    ldl = max(V, ld)
    def put(x):
        if x is None:
            return None
        y = np.full((M, ldl), 1e30, np.float32)  # past the vocabulary: nothing to draw
        y[:, :V] = x
        return dev.put(y)
    n = len(sizes)
    held = [put(logits), put(draft)]
    first, par, tok, un = (dev.put(x) for x in (offsets(sizes), np.append(parents, 0).astype(np.int32),
                                                np.append(tokens, 0).astype(np.int32),
                                                np.append(u, 0).astype(np.float32)))
    path, counts, nxt = dev.full((n, max_nodes), 77, np.int32), dev.full((n,), 77, np.int32), dev.full((n,), 77, np.int32)
    size = capi.size_out("gx_tree_verify_workspace_bytes", n, M, V)
    ws = dev.full((max(size, 256),), 0xFF, np.uint8)
    capi.call("gx_tree_verify", dev.ctx.ptr, vp(held[0]), ldl, n, M, max_nodes, V, vp(first), vp(par), vp(tok),
              vp(held[1]), ldl, temperature, draft_temperature, vp(un), vp(path), vp(counts), vp(nxt), vp(ws), size)
    return dev.get(path), dev.get(counts), dev.get(nxt)


def make_verify(seed, sizes, fanout, V, draws, near=1.0, peak=6.0):
    g = synth.rng(seed)
    M = sum(sizes)
    parents = random_parents(g, sizes, fanout)
    logits = (peak * g.standard_normal((M, V)) * g.random((M, 1))).astype(np.float32)
    draft = (logits + near * g.standard_normal((M, V))).astype(np.float32)
    tokens, first = np.zeros(M, np.int32), offsets(sizes)
    order = draft + (g.gumbel(size=(M, V)) if draws else 0)
    for b, t in enumerate(sizes):
        used = {}
        for m in range(first[b], first[b] + t):
            p = parents[m]
            if p < 0:
                continue
            r = used.get(p, 0)
            used[p] = r + 1
            tokens[m] = np.argsort(-order[first[b] + p])[r % V]
    return parents, tokens, logits, draft, g.random(M).astype(np.float32)


VERIFY = [([1], 1, 1, 0), ([4], 1, 2, 0), ([6, 3], 2, 5, 3), ([9, 1, 5], 3, 255, 0), ([40, 17], 5, 1000, 1),
          ([12], 11, 2047, 0), ([12], 3, 2048, 0), ([12], 3, 2049, 7), ([7, 7], 2, 8191, 0), ([7, 7], 2, 8193, 0),
          ([5, 0, 4], 2, 151936, 0), ([512], 1, 64, 0), ([512], 9, 700, 0), ([3] * 60, 2, 130, 0)]


@pytest.mark.parametrize("sizes,fanout,V,pad", VERIFY)
@pytest.mark.parametrize("form", ["greedy", "given", "drawn"])
def test_verify(dev, sizes, fanout, V, pad, form):
    longest = 0
    for seed in range(3):
        parents, tokens, logits, draft, u = make_verify(30 + seed, sizes, fanout, V, form == "drawn")
        t = 0.0 if form == "greedy" else 0.9
        args = (sizes, parents, tokens, logits, draft if form == "drawn" else None, t, t, u, max(sizes))
        want = verify_reference(*args)
        got = run_verify(dev, *args, ld=V + pad)
        for x, y in zip(got, want):
            np.testing.assert_array_equal(x, y)
        longest = max(longest, int(want[1].max()))
    log(f"  {form}: the longest path keeps {longest}")


@pytest.mark.parametrize("trees,V", [(300, 6000), (40, 40000), (700, 2049)])
def test_verify_with_fewer_workgroups_than_parts(dev, trees, V):
    """More trees than leave each one a workgroup for every part of its sums."""
    sizes = [2] * trees
    parents, tokens, logits, draft, u = make_verify(39, sizes, 1, V, True)
    args = (sizes, parents, tokens, logits, draft, 1.0, 1.0, u, 2)
    for x, y in zip(run_verify(dev, *args), verify_reference(*args)):
        np.testing.assert_array_equal(x, y)


def test_verify_temperatures_apart(dev):
    """A draft temperature of its own, and temperatures that leave one token or all alike."""
    sizes = [20, 9]
    for t, td in ((0.05, 0.5), (1.7, 0.6), (40.0, 3.0), (1e-12, 1e-10), (1e30, 1e20)):
        parents, tokens, logits, draft, u = make_verify(40, sizes, 4, 300, True)
        args = (sizes, parents, tokens, logits, draft, t, td, u, 20)
        for x, y in zip(run_verify(dev, *args), verify_reference(*args)):
            np.testing.assert_array_equal(x, y)


def test_verify_tokens_repeated_and_foreign(dev):
    """Siblings with one token, tokens outside the vocabulary, parents that are none."""
    sizes = [10, 8]
    for form in (0.0, 0.8):
        for q in (False, True):
            parents, tokens, logits, draft, u = make_verify(41, sizes, 6, 12, True)
            parents[1:4], tokens[1:4] = 0, tokens[1]
            tokens[4], tokens[12] = -1, 12
            parents[6], parents[15] = 9, -1
            args = (sizes, parents, tokens, logits, draft if q else None, form, form or 1.0, u, 10)
            for x, y in zip(run_verify(dev, *args), verify_reference(*args)):
                np.testing.assert_array_equal(x, y)


def test_verify_rows_without_a_chance(dev):
    """-inf logits are never drawn; rows of NaN, +inf or nothing but -inf
    take no child and give no token; where the draft's row is one of those the
    walk takes no child and draws from the target's."""
    sizes = [3] * 7
    parents, tokens, logits, draft, u = make_verify(42, sizes, 1, 500, False)
    logits[0, ::2] = -np.inf
    tokens[1] = 4  # hidden by the line above
    logits[3, 77], logits[18, 12], logits[9] = np.nan, np.inf, -np.inf
    logits[12, :490] = -np.inf
    u[12] = 1.0 - 2.0 ** -24
    u[15] = 0.0
    logits[15, :100] = -np.inf
    draft[6], draft[12, 3], draft[15, 4] = -np.inf, np.nan, np.inf
    for q in (None, draft):
        args = (sizes, parents, tokens, logits, q, 0.7, 0.7, u, 3)
        got, want = run_verify(dev, *args), verify_reference(*args)
        for x, y in zip(got, want):
            np.testing.assert_array_equal(x, y)
        assert got[2][1] == got[2][3] == got[2][6] == -1 and got[2][2] >= 0
    # a NaN in the greedy row follows gx_argmax: it wins only at index 0
    logits[3, 77], logits[6, 0] = np.nan, np.nan
    got = run_verify(dev, sizes, parents, tokens, logits, None, 0.0, 0.0, u, 3)
    want = verify_reference(sizes, parents, tokens, logits, None, 0.0, 0.0, u, 3)
    for x, y in zip(got, want):
        np.testing.assert_array_equal(x, y)


def test_verify_draft_equal_to_target(dev):
    """p = q keeps every first child whatever the numbers, and a residual that rounds to nothing falls back to p."""
    sizes = [6] * 40
    parents, tokens, logits, draft, u = make_verify(43, sizes, 1, 50, True)
    tokens_ok = make_verify(43, sizes, 1, 50, True, near=0.0)
    parents, tokens, logits, draft, u = tokens_ok
    path, counts, _ = run_verify(dev, sizes, parents, tokens, logits, logits.copy(), 1.0, 1.0, u, 6)
    assert np.all(counts == 6) and np.all(path == np.arange(6))


@pytest.mark.parametrize("form", ["given", "drawn"])
def test_verify_keeps_the_targets_distribution(dev, form):
    """The first token after the root -- kept or drawn -- over 60,000 walks of
    a small vocabulary, whose trees hold three drafts each: its counts are the
    target's chances.  A count of N p (1 - p) variance is within 5 of its
    standard deviations (six tokens: a chance of 4e-6 to be off)."""
    V, trees, rounds = 6, 1000, 60
    g = synth.rng(44)
    p_row = g.standard_normal(V).astype(np.float32)
    q_row = (p_row + 1.2 * g.standard_normal(V)).astype(np.float32)
    sizes, parents = [4] * trees, np.tile([-1, 0, 0, 0], trees).astype(np.int32)
    logits = np.tile(p_row, (4 * trees, 1))
    draft = np.tile(q_row, (4 * trees, 1))
    count = np.zeros(V)
    for _ in range(rounds):
        order = np.argsort(-(q_row + g.gumbel(size=(trees, V))), 1)[:, :3] if form == "drawn" else np.tile(
            np.argsort(-q_row)[:3], (trees, 1))
        tokens = np.concatenate([np.zeros((trees, 1), int), order], 1).reshape(-1).astype(np.int32)
        u = g.random(4 * trees).astype(np.float32)
        path, counts, nxt = run_verify(dev, sizes, parents, tokens, logits, draft if form == "drawn" else None, 1.0,
                                       1.0, u, 4)
        kept = tokens.reshape(trees, 4)[np.arange(trees), np.maximum(path[:, 1], 0)]
        count += np.bincount(np.where(counts > 1, kept, nxt), minlength=V)
    p, n = chances(p_row, 1.0), trees * rounds
    off = np.abs(count - n * p) / np.sqrt(n * p * (1 - p))
    log(f"  {form}: off by {off.round(2)} standard deviations")
    assert np.all(off < 5)


# ---- cache commit and fork --------------------------------------------------------


def _layer_pointers(xs):
    return (ctypes.c_void_p * len(xs))(*[x.data_ptr() for x in xs])


@pytest.mark.parametrize("layers,kv,hd,sizes,nslots", [(1, 1, 8, [1], 1), (3, 2, 64, [5, 9, 2], 4), (65, 2, 32, [7], 2),
                                                       (2, 8, 128, [33, 12], 3), (2, 3, 96, [0, 4], 2)])
def test_commit(dev, layers, kv, hd, sizes, nslots):
    g = synth.rng(50)
    n, M, nodes, ctx, dctx = len(sizes), sum(sizes), max(sizes), 48, (sum(sizes) + 8) // 8 * 8
    def draw(*s):
        return g.integers(-30000, 30000, s).astype(np.int16)
    kc, vc = draw(layers, nslots, kv, hd // 8, ctx, 8), draw(layers, nslots, kv, hd, ctx)
    kd, vd = draw(layers, kv, hd // 8, dctx, 8), draw(layers, kv, hd, dctx)
    first, slots = offsets(sizes), g.permutation(nslots)[:n].astype(np.int32)
    prefix = g.integers(0, 14, n).astype(np.int32)
    path, counts = np.full((n, nodes), -1, np.int32), np.zeros(n, np.int32)
    for b, t in enumerate(sizes):
        counts[b] = g.integers(1, t + 1) if t else 0
        path[b, :counts[b]] = np.sort(g.permutation(t)[:counts[b]])
    held = [dev.put(x) for x in (kc, vc, kd, vd)]
    small = [dev.put(x) for x in (first, path, counts, prefix)]
    sl = dev.put(slots)
    capi.call("gx_qwen_cache_commit", dev.ctx.ptr, layers, *[_layer_pointers(x) for x in held], n, M, nodes,
              *map(vp, small), kv, hd, ctx, dctx, vp(sl), nslots)
    for b in range(n):
        for j in range(counts[b]):
            kc[:, slots[b], :, :, prefix[b] + j] = kd[:, :, :, first[b] + path[b, j]]
            vc[:, slots[b], :, :, prefix[b] + j] = vd[:, :, :, first[b] + path[b, j]]
    np.testing.assert_array_equal(dev.get(held[0]), kc)
    np.testing.assert_array_equal(dev.get(held[1]), vc)


def test_commit_stores_nothing_out_of_range(dev):
    """Positions past the context, nodes that are none, slots and prefixes out of range, counts past the tree."""
    layers, kv, hd, ctx, dctx = 2, 2, 16, 16, 24
    g = synth.rng(51)
    def draw(*s):
        return g.integers(-30000, 30000, s).astype(np.int16)
    kc, vc = draw(layers, 3, kv, hd // 8, ctx, 8), draw(layers, 3, kv, hd, ctx)
    kd, vd = draw(layers, kv, hd // 8, dctx, 8), draw(layers, kv, hd, dctx)
    sizes = [4, 4, 4, 4, 4]
    path = np.tile(np.arange(4, dtype=np.int32), (5, 1))
    path[1] = [0, -1, 9, 2]
    prefix, slots = np.array([14, 2, -1, 16, 5], np.int32), np.array([0, 1, 2, 2, 3], np.int32)
    counts = np.array([4, 1 << 30, 4, 4, 4], np.int32)
    held = [dev.put(x) for x in (kc, vc, kd, vd)]
    small = [dev.put(x) for x in (offsets(sizes), path, counts, prefix)]
    sl = dev.put(slots)
    capi.call("gx_qwen_cache_commit", dev.ctx.ptr, layers, *[_layer_pointers(x) for x in held], 5, 20, 4,
              *map(vp, small), kv, hd, ctx, dctx, vp(sl), 3)
    for slot, pos, row in ((0, 14, 0), (0, 15, 1), (1, 2, 4), (1, 5, 6)):
        kc[:, slot, :, :, pos] = kd[:, :, :, row]
        vc[:, slot, :, :, pos] = vd[:, :, :, row]
    np.testing.assert_array_equal(dev.get(held[0]), kc)
    np.testing.assert_array_equal(dev.get(held[1]), vc)


@pytest.mark.parametrize("layers,kv,hd,ctx,nslots,src,dsts,length", [
    (1, 1, 8, 8, 2, 0, [1], 1), (2, 2, 64, 40, 4, 2, [3, 0], 7), (3, 2, 96, 64, 3, 1, [0, 2], 64),
    (66, 2, 32, 16, 3, 0, [2], 9), (2, 8, 128, 520, 5, 4, [1, 3], 513), (1, 1, 8, 16, 70, 3, [i for i in range(70) if i != 3], 11),
    (2, 2, 16, 24, 3, 1, [0], 0), (2, 2, 16, 24, 3, 1, [], 8)])
def test_fork(dev, layers, kv, hd, ctx, nslots, src, dsts, length):
    g = synth.rng(52)
    kc = g.integers(-30000, 30000, (layers, nslots, kv, hd // 8, ctx, 8)).astype(np.int16)
    vc = g.integers(-30000, 30000, (layers, nslots, kv, hd, ctx)).astype(np.int16)
    dk, dv = dev.put(kc), dev.put(vc)
    capi.call("gx_qwen_cache_fork", dev.ctx.ptr, layers, _layer_pointers(dk), _layer_pointers(dv), nslots, kv, hd, ctx,
              src, (ctypes.c_int32 * len(dsts))(*dsts), len(dsts), length)
    for d in dsts:
        kc[:, d, :, :, :length] = kc[:, src, :, :, :length]
        vc[:, d, :, :, :length] = vc[:, src, :, :, :length]
    np.testing.assert_array_equal(dev.get(dk), kc)
    np.testing.assert_array_equal(dev.get(dv), vc)


# ---- together ----------------------------------------------------------------------

CFG = synth.QwenConfig(256, 512, 2, 4, 2, 64, 1024, 96)


def _model(dev, seed=81, cfg=CFG, max_batch=32):
    return QwenModel(dev.ctx, cfg, synth.qwen_weights(cfg, seed, symmetric=True), max_batch=max_batch)


def _close(got, want):
    """Two orders of the attention's sums, each held to 5e-2 of RMS of golem's
    engine by the model tests (a head's Q8_0 moves by a step where its sum
    does by an ulp): |a - b| <= |a - o| + |b - o| <= 1e-1 of RMS."""
    rms = float(np.sqrt((want.astype(np.float64) ** 2).mean()))
    off = float(np.abs(got - want).max()) / rms
    assert off <= 1e-1, off
    return off


def test_a_tree_gives_each_path_its_own_pass(dev):
    """Every node's hidden state is what its path gives run as tokens after
    the same prompt; a kept path continues as if it had been decoded."""
    g = synth.rng(60)
    prompts = [[int(t) for t in g.integers(0, CFG.vocab, k)] for k in (11, 4)]
    parents = [[-1, 0, 0, 1, 1, 2, 5, 3], [-1, 0, 1, 1, 0]]
    tokens = [[int(t) for t in g.integers(0, CFG.vocab, len(p))] for p in parents]
    m = _model(dev)
    m.set_slots(3)
    slots = [2, 0]
    for p, s in zip(prompts, slots):
        m.use_slot(s)
        m.forward(p, 0)
    before = [x.clone() for x in m.kc + m.vc]
    m.set_drafts(16)
    got = m.forward_tree(tokens, parents, [len(p) for p in prompts], slots).cpu().numpy()
    for x, y in zip(before, m.kc + m.vc):
        assert torch.equal(x, y), "a pass over drafts changed a cache"
    solo, at, worst = _model(dev), 0, 0.0
    for b in range(2):
        for i in range(len(parents[b])):
            path, x = [], i
            while x >= 0:
                path.insert(0, tokens[b][x])
                x = parents[b][x]
            solo.reset()
            solo.forward(prompts[b], 0)
            for k, tok in enumerate(path):
                h = solo.forward([tok], len(prompts[b]) + k)[0].cpu().numpy()
            worst = max(worst, _close(got[at + i], h))
        at += len(parents[b])
    log(f"  nodes off their paths' passes by at most {worst:.2e} of RMS")
    # keep 0 -> 2 -> 5 of the first tree and the root of the second
    t = m.tree
    t["path"].fill_(-1)
    t["path"][0, :3] = torch.tensor([0, 2, 5], dtype=torch.int32)
    t["path"][1, 0] = 0
    t["counts"].copy_(torch.tensor([3, 1], dtype=torch.int32))
    m.commit_tree()
    for b, path in enumerate(([0, 2, 5], [0])):
        m.use_slot(slots[b])
        h = m.forward([7], len(prompts[b]) + len(path))[0].cpu().numpy()
        solo.reset()
        solo.forward(prompts[b] + [tokens[b][i] for i in path], 0)
        _close(h, solo.forward([7], len(prompts[b]) + len(path))[0].cpu().numpy())
    solo.free()
    m.free()


def test_a_tree_in_the_products_epilogue(dev):
    """More than sixteen drafted tokens: the Q|K|V product stores the drafts'
    heads itself.  Each node's hidden state is that of a smaller pass of its
    path alone."""
    g = synth.rng(64)
    prompt = [int(t) for t in g.integers(0, CFG.vocab, 10)]
    parents = [-1] + [int(g.integers(max(0, i - 6), i)) for i in range(1, 27)]
    tokens = [int(t) for t in g.integers(0, CFG.vocab, 27)]
    m = _model(dev)
    m.set_drafts(27)
    m.forward(prompt, 0)
    got = m.forward_tree([tokens], [parents], [len(prompt)]).cpu().numpy().copy()
    for i in range(27):
        path, x = [], i
        while x >= 0:
            path.insert(0, tokens[x])
            x = parents[x]
        assert len(path) <= 16
        h = m.forward_tree([path], [[-1] + list(range(len(path) - 1))], [len(prompt)])[-1].cpu().numpy()
        _close(got[i], h)
    m.free()


def _oracle_draft(ids, sequence, width):
    """Three tokens along the sequence with a wrong one in some places, and `width` - 1 wrong siblings of each."""
    tokens, parents, up = [], [], 0
    for k in range(3):
        at = len(ids) + k
        right = sequence[at] if at < len(sequence) else 1
        if at % 5 == 4:
            right = (right + 1) % CFG.vocab
        for w in range(width - 1):
            tokens.append((right + 2 + w) % CFG.vocab)
            parents.append(up)
        tokens.append(right)
        parents.append(up)
        up = len(tokens)
    return tokens, parents


@pytest.mark.parametrize("width", [1, 3])
def test_speculation_draws_greedys_tokens(dev, width):
    m = _model(dev)
    prompt, steps = [int(t) for t in synth.rng(61).integers(0, CFG.vocab, 9)], 40
    want = m.greedy(prompt, steps)
    m.reset()
    got, passes = m.speculate(prompt, steps, lambda ids: _oracle_draft(ids, prompt + want, width))
    log(f"  {steps} tokens in {passes} passes")
    assert got == want and passes < steps // 2
    m.reset()
    got, passes = m.speculate(prompt, steps, lambda ids: ([], []))
    assert got == want and passes == steps
    # to the context's last position, drafts cut off there
    m.reset()
    steps = CFG.max_context - len(prompt) + 1
    want = m.greedy(prompt, steps)
    m.reset()
    got, _ = m.speculate(prompt, steps, lambda ids: _oracle_draft(ids, prompt + want, width))
    assert got == want
    m.free()


def test_speculation_in_a_slot(dev):
    """In one conversation of several, beside another whose caches stay as they are."""
    m = _model(dev)
    prompt, steps = [int(t) for t in synth.rng(66).integers(0, CFG.vocab, 7)], 24
    want = m.greedy(prompt, steps)
    m.set_slots(3)
    m.use_slot(0)
    m.forward([9, 8, 7], 0)
    beside = [x[0].clone() for x in m.kc + m.vc]
    m.use_slot(2)
    got, passes = m.speculate(prompt, steps, lambda ids: _oracle_draft(ids, prompt + want, 2))
    assert got == want and passes < steps // 2
    for x, y in zip(beside, m.kc + m.vc):
        assert torch.equal(x, y[0])
    with pytest.raises(ValueError, match="exceed the context"):
        m.speculate(prompt, m.slot_context, lambda ids: ([], []))
    m.free()


def test_sampled_speculation_runs_and_repeats(dev):
    m = _model(dev)
    prompt = [5, 9, 400]

    def draft(ids):
        lg = torch.randn((4, CFG.vocab), generator=torch.Generator("cuda").manual_seed(len(ids)), device="cuda")
        pick = torch.softmax(lg[0] / 0.8, 0).argsort(descending=True)[:3].tolist()
        return pick, [0, 0, 0], lg

    runs = []
    for _ in range(2):
        m.reset()
        gen = torch.Generator("cuda").manual_seed(5)
        runs.append(m.speculate(prompt, 12, draft, temperature=0.8, generator=gen)[0])
    assert runs[0] == runs[1] and all(0 <= t < CFG.vocab for t in runs[0])
    m.free()


def test_forked_conversations_go_on_alone(dev):
    m = _model(dev)
    m.set_slots(3)
    prompt = [int(t) for t in synth.rng(62).integers(0, CFG.vocab, 13)]
    m.use_slot(1)
    m.forward(prompt, 0)
    m.fork_slot(1, [0, 2], len(prompt))
    want = None
    for s in (1, 0, 2):
        m.use_slot(s)
        h = m.forward([3], len(prompt))[0].cpu().numpy().copy()
        want = h if want is None else want
        np.testing.assert_array_equal(h.view(np.uint32), want.view(np.uint32))
    with pytest.raises(capi.GxError, match="into itself"):
        m.fork_slot(1, [1], 3)
    with pytest.raises(ValueError, match="positions of a slot"):
        m.fork_slot(1, [0], m.slot_context + 1)
    m.free()


def test_model_refusals(dev):
    m = _model(dev)
    with pytest.raises(ValueError, match="no pass over drafted"):
        m.verify_tree()
    with pytest.raises(ValueError, match="set_drafts"):
        m.forward_tree([[1]], [[-1]], [0])
    with pytest.raises(ValueError, match="for a batch of"):
        m.set_drafts(33)
    m.set_drafts(8)
    for args, message in ((([[1, 2]], [[-1, 1]], [0]), "no earlier node"), (([[1, 2]], [[-1]], [0]), "no earlier|needs"),
                          (([[1]], [[-1]], [CFG.max_context]), "past the context"), (([[1]], [[-1]], [-1]), "past the context"),
                          (([[1], [2]], [[-1], [-1]], [0, 0], [0, 0]), "two trees"), (([], [], []), "needs tokens"),
                          (([[1] * 9], [[-1] + list(range(8))], [0]), "for buffers of 8")):
        with pytest.raises(ValueError, match=message):
            m.forward_tree(*args)
    with pytest.raises(IndexError):
        m.forward_tree([[1]], [[-1]], [0], [1])
    m.forward_tree([[1, 2]], [[-1, 0]], [0])
    with pytest.raises(ValueError, match="random numbers"):
        m.verify_tree(0.5, uniforms=torch.rand(3, device="cuda"))
    with pytest.raises(ValueError, match="draft logits"):
        m.verify_tree(0.5, draft_logits=torch.zeros((2, 5), device="cuda"))
    m.set_slots(2)
    with pytest.raises(ValueError, match="no pass over drafted"):
        m.commit_tree()
    m.free()


def test_passes_in_between(dev):
    """A pass between forward_tree and verify_tree takes the states away; one
    after verify_tree does not keep its path from being committed, and before
    it there is none to commit."""
    m = _model(dev)
    m.set_drafts(8)
    m.forward([4, 5, 6], 0)
    saved = [x.clone() for x in m.kc + m.vc]
    m.forward_tree([[1, 2]], [[-1, 0]], [3])
    m.commit_tree()
    for x, y in zip(saved, m.kc + m.vc):
        assert torch.equal(x, y)
    m.forward([7], 3)
    with pytest.raises(ValueError, match="another pass"):
        m.verify_tree()
    m.forward_tree([[1, 2]], [[-1, 0]], [3])
    path, counts, _ = m.verify_tree()
    want = [x.clone() for x in m.kd]
    m.forward([8], 20)
    m.commit_tree()
    for i in range(int(counts[0])):
        node = int(path[0, i])
        for x, y in zip(want, m.kc):
            assert torch.equal(x[:, :, node], y.reshape(x.shape[0], x.shape[1], -1, 8)[:, :, 3 + i])
    m.capture_decode()
    m.forward_tree([[1, 2]], [[-1, 0]], [3])
    m.start_decode(torch.tensor([3], dtype=torch.int32, device="cuda"), 5)
    with pytest.raises(ValueError, match="another pass"):
        m.verify_tree()
    m.free()


def test_speculation_with_foreign_drafts(dev):
    """Drafted tokens outside the vocabulary are passed over: their rows are
    NaN, and nothing of them reaches the others."""
    m = _model(dev)
    prompt, steps = [int(t) for t in synth.rng(65).integers(0, CFG.vocab, 6)], 12
    want = m.greedy(prompt, steps)

    def draft(ids):
        right = (prompt + want + [1])[len(ids)]
        return [CFG.vocab + 3, -7, right, right], [0, 1, 0, 1], None

    m.reset()
    got, passes = m.speculate(prompt, steps, draft)
    assert got == want and passes <= (steps + 1) // 2
    m.free()


def test_captured_pass_equals_eager(dev):
    """A pass -- forward, verification, commit -- captured once and replayed
    for other tokens and prefixes, with eager work between the replays."""
    t = torch
    m = _model(dev)
    m.set_drafts(8)
    prompt = [int(x) for x in synth.rng(63).integers(0, CFG.vocab, 20)]
    m.forward(prompt, 0)
    parents = [[-1, 0, 0, 1, 2]]
    u = t.rand(5, device="cuda")
    m.forward_tree([[1, 2, 3, 4, 5]], parents, [40])  # prefixes to 40
    m.verify_tree(0.8, uniforms=u)
    m.commit_tree()
    tree, stream, graph = m.tree, t.cuda.Stream(), t.cuda.CUDAGraph()
    saved = [x.clone() for x in m.kc + m.vc]
    t.cuda.synchronize()
    capi.call("gx_set_stream", dev.ctx.ptr, ctypes.c_void_p(stream.cuda_stream))
    try:
        with t.cuda.graph(graph, stream=stream):
            m._tree_blocks(tree)
            m.verify_tree(0.8, uniforms=u)
            m.commit_tree()
    finally:
        capi.call("gx_set_stream", dev.ctx.ptr, ctypes.c_void_p(t.cuda.current_stream().cuda_stream))
    t.cuda.synchronize()
    for k in range(4):
        tokens = [int(x) for x in synth.rng(70 + k).integers(0, CFG.vocab, 5)]
        new = t.rand(5, device="cuda")
        results = []
        for way in ("eager", "replay"):
            m.tree = tree
            tree["prefix"].fill_(20 + k)
            m.tokens[:5].copy_(t.tensor(tokens, dtype=t.int32))
            u.copy_(new)
            for x, y in zip(m.kc + m.vc, saved):
                x.copy_(y)
            if way == "eager":
                m._tree_blocks(tree)
                m.verify_tree(0.8, uniforms=u)
                m.commit_tree()
            else:
                graph.replay()
            t.cuda.synchronize()
            results.append([x.clone() for x in (m.hidden[:5], tree["path"], tree["counts"], tree["next"], *m.kc, *m.vc)])
        for a, b in zip(*results):
            assert t.equal(a, b)
    m.free()


def test_two_verifications_at_once(dev):
    """Walks of two contexts on two streams together, more workgroups than the
    GPU holds: neither waits for the other's."""
    t = torch
    ctxs, cases, held = [], [], []
    for k in range(2):
        sizes = [6] * 8
        parents, tokens, logits, draft, u = make_verify(90 + k, sizes, 2, 151936, True)
        args = (sizes, parents, tokens, logits, draft, 1.0, 1.0, u, 6)
        cases.append((args, verify_reference(*args)))
        s = t.cuda.Stream()
        ctxs.append((capi.Context(0, stream=s.cuda_stream), s))
        M = sum(sizes)
        size = capi.size_out("gx_tree_verify_workspace_bytes", 8, M, 151936)
        held.append([dev.put(x) for x in (logits, draft, offsets(sizes), parents, tokens, u)]
                    + [dev.empty((8, 6), np.int32), dev.empty((8,), np.int32), dev.empty((8,), np.int32),
                       dev.empty((size,), np.uint8)])
    t.cuda.synchronize()
    for _ in range(20):
        for (ctx, s), x in zip(ctxs, held):
            lg, dr, first, par, tok, u, path, counts, nxt, ws = x
            capi.call("gx_tree_verify", ctx.ptr, vp(lg), 151936, 8, 48, 6, 151936, vp(first), vp(par), vp(tok), vp(dr),
                      151936, 1.0, 1.0, vp(u), vp(path), vp(counts), vp(nxt), vp(ws), ws.numel())
    t.cuda.synchronize()
    for (_, want), x in zip(cases, held):
        for got, w in zip(x[6:9], want):
            np.testing.assert_array_equal(got.cpu().numpy(), w)
    for ctx, _ in ctxs:
        ctx.close()


def test_two_contexts_on_their_own_streams(dev):
    """The same call from two contexts at once, each on a stream and workspace of its own."""
    t = torch
    a, b = Attention(80, [30], [900], 8, 2, 128), Attention(81, [9, 40], [500, 700], 8, 2, 128)
    want = [a.run(dev), b.run(dev)]
    streams = [t.cuda.Stream() for _ in range(2)]
    ctxs = [capi.Context(0, stream=s.cuda_stream) for s in streams]

    class On:
        def __init__(self, ctx):
            self.ctx = ctx
        put, full, empty = staticmethod(dev.put), staticmethod(dev.full), staticmethod(dev.empty)

        def get(self, x):
            return x

    outs = []
    t.cuda.synchronize()
    for x, c, s in zip((a, b), ctxs, streams):
        with t.cuda.stream(s):
            outs.append(x.run(On(c)))
    t.cuda.synchronize()
    for x, w in zip(outs, want):
        np.testing.assert_array_equal(x.cpu().numpy(), w)
    for c in ctxs:
        c.close()
