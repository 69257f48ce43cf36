"""The attention of drafted trees where a workgroup takes several steps of keys
in a row, and what lies behind a tree's rows."""
import math

import numpy as np
import pytest

from golem_amd import capi, synth
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
