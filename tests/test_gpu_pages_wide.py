"""The attention over pages by the kernel for many rows, whole and in shares: what
the other forms are held to, launched for bounds by which this one is chosen
(the tests' own rows are few enough for the 16-row tiles)."""
import numpy as np
import pytest

from tests import test_gpu_pages as base

pytestmark = pytest.mark.gpu


class Whole(base.Attention):
    """Launched for 16000 tokens a conversation: a tile's keys by one workgroup."""

    tokens_bound, length_bound = 16000, 0

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.max_tokens, pool = max(self.max_tokens, self.tokens_bound), self.pool
        pool.width = max(pool.width, (self.length_bound + pool.size - 1) // pool.size)
        table, pool.table = pool.table, np.full((self.n, pool.width), -1, np.int32)
        pool.table[:, :table.shape[1]] = table

    def run(self, dev, max_length=None, **kw):
        return super().run(dev, self.length_bound or max_length, **kw)


class Shares(Whole):
    """Launched for few tokens over a long context: a tile's keys by several."""

    tokens_bound, length_bound = 33, 32768


@pytest.fixture(params=[Whole, Shares], ids=["whole", "shares"])
def wide(request, monkeypatch):
    monkeypatch.setattr(base, "Attention", request.param)
    return request.param


BITS = pytest.mark.parametrize("bits", [16, 8])
# a few rows, tiles of 128 rows and parts of one, steps of 64 keys and parts of one
FORMS = pytest.mark.parametrize("counts,lengths", [([1], [200]), ([9], [200]), ([9], [2300]), ([150], [300]), ([70], [1100])])


@BITS
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (32, 8, 128), (3, 3, 64), (16, 1, 128), (40, 2, 64)])
@pytest.mark.parametrize("counts,lengths", [([1, 1, 1], [45, 1, 300]), ([7, 1, 12], [64, 200, 12]), ([70], [133])])
def test_heads(dev, wide, heads, kv, hd, counts, lengths, bits):
    base.test_attention_heads(dev, heads, kv, hd, counts, lengths, bits)


@BITS
@pytest.mark.parametrize("length", [1, 2, 8, 16, 31, 63, 64, 65, 127, 128, 129, 500, 2050])
def test_lengths(dev, wide, length, bits):
    base.test_attention_lengths(dev, length, bits)


@BITS
@pytest.mark.parametrize("size", [16, 64, 128, 1024])
def test_page_sizes(dev, wide, size, bits):
    base.test_attention_page_sizes(dev, size, bits)


@BITS
@pytest.mark.parametrize("counts", [[31], [33], [64, 2], [3, 64, 30], [129, 5], [1] * 11, [0, 4, 0, 3], [257]])
def test_pieces(dev, wide, counts, bits):
    base.test_attention_pieces(dev, counts, bits)


@pytest.mark.parametrize("counts,lengths", [([20], [700]), ([150], [400])])
def test_large_scores(dev, wide, counts, lengths):
    base.test_attention_large_scores(dev, counts, lengths)


@FORMS
def test_outputs_of_any_alignment(dev, wide, counts, lengths):
    base.test_attention_outputs_of_any_alignment(dev, counts, lengths)


@BITS
def test_rows_that_see_nothing(dev, wide, bits):
    base.test_attention_rows_that_see_nothing(dev, bits)


@FORMS
@pytest.mark.parametrize("page", [-1, 1 << 30])
def test_pages_that_are_not_there(dev, wide, counts, lengths, page):
    base.test_attention_pages_that_are_not_there(dev, counts, lengths, page)


@BITS
@pytest.mark.parametrize("counts,lengths", [([6, 5], [200, 14]), ([6, 5], [2300, 14]), ([150, 5], [300, 14])])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_hidden_values_stay_hidden(dev, wide, counts, lengths, bad, bits):
    base.test_attention_hidden_values_stay_hidden(dev, counts, lengths, bad, bits)


@FORMS
def test_infinite_cached_values(dev, wide, counts, lengths):
    base.test_attention_infinite_cached_values(dev, counts, lengths)


@pytest.mark.parametrize("counts,lengths", [([9], [200]), ([9], [2300]), ([150], [300])])
def test_nan_query_is_its_own(dev, wide, counts, lengths):
    base.test_attention_nan_query_is_its_own(dev, counts, lengths)


@FORMS
def test_scales_of_any_size(dev, wide, counts, lengths):
    base.test_attention_scales_of_any_size(dev, counts, lengths)


@FORMS
def test_scales_of_any_sign(dev, wide, counts, lengths):
    base.test_attention_scales_of_any_sign(dev, counts, lengths)


def test_shared_pages(dev, wide):
    base.test_attention_shared_pages(dev)


def test_none(dev, wide):
    base.test_attention_none(dev)


@BITS
@pytest.mark.parametrize("counts,lengths", [([9], [200]), ([150], [300]), ([40], [1500]), ([3, 35], [2300, 2100])])
def test_large_hidden_scores_leave_no_trace(dev, wide, counts, lengths, bits):
    base.test_attention_large_hidden_scores_leave_no_trace(dev, counts, lengths, bits)


@FORMS
@pytest.mark.parametrize("near", [0, 1])
@pytest.mark.parametrize("grow", [20, 60, 110])
def test_large_scales_of_small_weight(dev, wide, counts, lengths, near, grow):
    base.test_attention_large_scales_of_small_weight(dev, counts, lengths, near, grow)
