"""The attention of drafted trees where a workgroup takes several steps of keys
in a row: whole ones and partial ones, prefix and drafts, maxima that rise from
one to the next; what lies behind a tree's rows; and the precision that the
probabilities' second part gives."""
import math

import numpy as np
import pytest

from golem_amd import capi, synth
from tests.gpu_util import log
from tests.test_gpu_tree import Attention, long_context, offsets

gpu = pytest.mark.gpu


def ceil_div(a, b):
    return -(-a // b)


class Steps(Attention):
    """A case whose calls have `trees` trees, all but the first few empty, and are
    launched for `most` positions: as many trees leave each a few shares of its
    keys alone, however short the reference's work.  Scores rise by `ramp` over the
    positions."""

    def __init__(self, seed, sizes, prefix, heads, kv, hd, trees=1, most=0, ramp=0.0, **kw):
        super().__init__(seed, sizes, prefix, heads, kv, hd, **kw)
        g = synth.rng(seed + 1000)
        if ramp:
            # a direction that every query has 16 of, and the keys more and more of
            d = g.standard_normal(hd)
            d /= np.sqrt((d * d).sum())
            self.q = (self.q + 16 * d).astype(np.float16)
            at = np.arange(self.context) / max(int(max(prefix)), 1) - 0.5
            self.k = (self.k + (ramp * math.sqrt(hd) / 16 * at)[:, None] * d).astype(np.float16)
        more = trees - self.n
        if more > 0:
            self.sizes, self.n = self.sizes + [0] * more, trees
            self.prefix = np.concatenate([self.prefix, g.integers(0, 60, more)]).astype(np.int32)
            self.slots = np.concatenate([self.slots, np.zeros(more)]).astype(np.int32)
            self.first = offsets(self.sizes)
        self.most = max(most, int(self.prefix.max()))
        longer = max((self.most + 7) // 8 * 8 - self.context, 0)
        pad = ((0, 0), (0, 0), (0, longer), (0, 0))
        self.k, self.v = (np.pad(x, pad, constant_values=np.nan) for x in (self.k, self.v))
        self.context += longer

    def behind(self, value):
        """Every row behind a prefix, and behind the last token, set to `value`."""
        for s in range(self.nslots):
            at = list(self.slots[:len(self.sizes) - self.sizes.count(0)])
            p = int(self.prefix[at.index(s)]) if s in at else 0
            self.k[s, :, p:], self.v[s, :, p:] = value, value
        self.kd[:, self.tokens:], self.vd[:, self.tokens:] = value, value
        return self

    def launch(self):
        """(the kernel of several tiles a workgroup is chosen, the steps of a share
        of the first tree's keys), by the library's rules."""
        heads, kv, most, nodes = self.heads, self.kv, self.most, self.max_nodes
        tiles = ceil_div(nodes * (heads // kv), 32)
        every = self.n * kv * tiles
        few = ceil_div(most, 32) + ceil_div(nodes + 7, 32)
        one = 1 if few <= 16 else max(1, min((few + 1) // 2, 64, 256 // every))
        narrow = tiles == 1 or (every * one + 255) // 256 * few <= 7 * 8 * one
        size = capi.size_out("gx_qwen_attention_tree_workspace_bytes", self.n, self.M, nodes, heads, kv, self.hd, most)
        S = size // (self.M * heads * (self.hd + 2) * 4)
        total = ceil_div(int(self.prefix[0]), 64) + ceil_div(self.sizes[0] + self.first[0] % 8, 64)
        return not narrow, ceil_div(total, S)

    def run(self, dev, **kw):
        return super().run(dev, **{"max_prefix": self.most, **kw})


# (heads, kv, hd, sizes, prefix, trees, most): three tiles of rows; five and six, the
# last of them in halves; eight; nine in two groups, with three steps of drafts in
# one share; two tiles and one share
MANY = {"three": (4, 2, 64, [37, 16], [700, 333], 128, 704),
        "five": (4, 2, 64, [80, 3], [651, 70], 64, 720),
        "six": (8, 2, 128, [47, 40], [1001, 640], 40, 1008),
        "eight": (8, 2, 128, [64, 9], [1000, 131], 32, 1024),
        "nine": (2, 1, 32, [130, 5], [517, 64], 64, 640),
        "two": (6, 2, 96, [17, 6], [461, 100], 256, 600)}


def many(name, seed, **kw):
    heads, kv, hd, sizes, prefix, trees, most = MANY[name]
    a = Steps(seed, sizes, prefix, heads, kv, hd, trees=trees, most=most, **kw)
    assert a.launch()[0] and a.launch()[1] >= 3, a.launch()
    return a


@gpu
@pytest.mark.parametrize("ramp", [0.0, 14.0, 120.0, -120.0])
@pytest.mark.parametrize("name", MANY)
def test_many_steps_a_share(dev, name, ramp):
    """Whole and partial steps of the prefix and the drafts in one share; with a
    ramp the maximum rises past the reference at some steps, or at every one, or
    is the first one's."""
    many(name, 300, ramp=ramp, pad=3).behind(0.25).check(dev)


@gpu
@pytest.mark.parametrize("name", ["three", "five", "eight"])
@pytest.mark.parametrize("prefix", [576, 577, 583, 584, 607, 608, 609, 639, 640])
def test_many_steps_and_prefixes(dev, name, prefix):
    """The prefix's last step of every kind: whole, one key, and ends on and off a
    chunk of eight and a half of the step."""
    heads, kv, hd, sizes, _, trees, _ = MANY[name]
    a = Steps(301, [sizes[0] - 1, 11], [prefix, prefix - 5], heads, kv, hd, trees=2 * trees, most=1600)
    assert a.launch()[0] and a.launch()[1] >= 3, a.launch()
    a.check(dev)


def bits(x):
    return np.ascontiguousarray(x).view(np.uint32)


# (a tile a workgroup, the keys over several and several tiles a workgroup, of one and of many steps)
BEHIND = [("short", (4, 2, 64, [9, 5], [75, 13], 2, 0)), ("shared", (4, 2, 64, [9, 5], [1101, 70], 2, 0)),
          ("long", (4, 2, 64, [21, 12], [77, 101], 2, long_context(2, 21, 4, 2)))] + list(MANY.items())


@gpu
@pytest.mark.parametrize("name,case", BEHIND, ids=[n for n, _ in BEHIND])
def test_rows_behind_leave_no_trace(dev, name, case):
    """What a cache holds behind a prefix, and the draft buffers behind the last
    token, are of no matter: the same bits with zeros, numbers, NaN and infinities
    there, and they are the float64 result's within its tolerance."""
    heads, kv, hd, sizes, prefix, trees, most = case
    a = Steps(302, sizes, prefix, heads, kv, hd, trees=trees, most=most)
    want = a.behind(0.0).check(dev)
    for value in (3.0, np.inf, -np.inf, np.nan):
        np.testing.assert_array_equal(bits(a.behind(value).run(dev)[:a.tokens]), bits(want))


@gpu
@pytest.mark.parametrize("name", ["short", "shared", "long", "three", "nine"])
def test_another_trees_rows_leave_no_trace(dev, name):
    """Rows of the next tree's nodes in a chunk with the last of this one's."""
    heads, kv, hd, sizes, prefix, trees, most = dict(BEHIND)[name]
    a = Steps(303, sizes, prefix, heads, kv, hd, trees=trees, most=most)
    t = sizes[0]
    assert t % 8
    want = a.behind(0.0).run(dev)
    for value in (np.inf, np.nan):
        a.kd[:, t:], a.vd[:, t:] = value, value
        np.testing.assert_array_equal(bits(a.run(dev)[:t]), bits(want[:t]))


# ---- the probabilities' precision ---------------------------------------------------


def value_bound(count):
    """How far o / v may be from 1 where every key has the value v.  The scores'
    errors are in numerator and denominator alike and cancel.  A probability's
    two parts, each cut off after eleven bits, are it but for less than 2^-21 of
    it, or 2^-24 where the second is below fp16's normal numbers; the row's sum is
    2^8 at least.  Every float32 addition is off by half a step, 2^-24, of a sum
    that is never above the last: one a term in the denominator and two (a part
    each) in the numerator, and 64 more each for rescalings, wavefronts and
    shares; four for the weights' products, the quotient and the output."""
    return 3 * (count + 64) * 2.0 ** -24 + 2.0 ** -21 + count * 2.0 ** -32 + 4 * 2.0 ** -24


def cut(p, least):
    """p with its leading eleven bits, or down to `least`."""
    e = np.floor(np.log2(np.maximum(p, 1e-300)))
    step = np.maximum(2.0 ** (e - 10), least)
    return np.floor(p / step) * step


@pytest.mark.parametrize("count", [300, 520, 720])
def test_the_bound_tells_one_part_from_two(count):
    """The bound below holds for two parts and for one part does not (the sums
    exact here: their roundings are what the bound has besides)."""
    g = synth.rng(310)
    for _ in range(20):
        p = 256.0 * np.exp2(np.minimum(g.standard_normal(count) * 0.7 - 2, 0)).astype(np.float32).astype(np.float64)
        p[0] = 256.0
        one = cut(p, 2.0 ** -24)
        two = one + cut(p - one, 2.0 ** -24)
        assert abs(two.sum() / p.sum() - 1) < 2.0 ** -21 + count * 2.0 ** -32
        assert abs(one.sum() / p.sum() - 1) > 1.5 * value_bound(count)


@gpu
@pytest.mark.parametrize("heads,kv,hd,sizes,prefix,trees,most", [
    (4, 2, 64, [9], [300], 1, 0), (8, 2, 128, [6, 4], [511, 300], 2, 0), (4, 2, 64, [40], [520], 1, long_context(1, 40, 4, 2)),
    MANY["three"], MANY["five"], MANY["nine"], MANY["two"]])
def test_values_all_alike_come_back(dev, heads, kv, hd, sizes, prefix, trees, most):
    """Every key of a head with one value an element: that value is the result.  A
    probability that lost its second part on the way to the values would leave
    3.5e-4 of it behind."""
    a = Steps(311, sizes, prefix, heads, kv, hd, trees=trees, most=most, spread=0.5)
    v = (1.0 + np.arange(kv * hd).reshape(kv, 1, hd) % 61 / 64).astype(np.float16)
    a.v[:], a.vd[:] = v, v
    got = a.run(dev)[:a.tokens].astype(np.float64).reshape(a.tokens, kv, heads // kv, hd)
    off = np.abs(got / v.astype(np.float64).reshape(kv, 1, hd) - 1)
    worst = 0.0
    for b, t in enumerate(sizes):
        rows = slice(a.first[b], a.first[b] + t)
        worst = max(worst, off[rows].max() / value_bound(prefix[b] + t))
    log(f"  worst {off.max():.2e}, {worst:.3f} of the bound")
    assert worst <= 1
