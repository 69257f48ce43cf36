"""Conversations in pages through QwenModel: the append and the attention run
together with the rest of the model, next to the slots' caches; common
beginnings, pages that come back, steps in lock step and their captured form;
rotations of long contexts."""
import math

import numpy as np
import pytest
import torch

from golem_amd import capi, synth
from golem_amd.qwen import QwenModel
from tests.gpu_util import log
from tests.test_gpu_tree import _close

pytestmark = pytest.mark.gpu
CFG = synth.QwenConfig(256, 512, 2, 4, 2, 64, 1024, 160)


def model(dev, seed=81, cfg=CFG, max_batch=96):
    return QwenModel(dev.ctx, cfg, synth.qwen_weights(cfg, seed, symmetric=True), max_batch=max_batch)


def prompt(seed, k):
    return [int(t) for t in synth.rng(seed).integers(0, CFG.vocab, k)]


def bits(x):
    return x.cpu().numpy().view(np.uint32).copy()


@pytest.mark.parametrize("hd,heads,kv", [(64, 4, 2), (32, 8, 2), (128, 2, 1)])
@pytest.mark.parametrize("size", [16, 64])
def test_pages_give_what_the_slots_give(dev, hd, heads, kv, size):
    """A prompt in one pass, in pieces and a token at a time: the states that the slots' caches give."""
    cfg = synth.QwenConfig(256, 512, 2, heads, kv, hd, 1024, 160)
    m = model(dev, 90, cfg)
    p = prompt(91, 75)
    m.reset()
    want = m.forward(p, 0).cpu().numpy().copy()
    m.set_pages(24, size)
    whole, pieces = m.open_conversation(), m.open_conversation()
    _close(m.forward_pages([p], [whole]).cpu().numpy(), want)
    at, got = 0, []
    for k in (1, 20, 3, 1, 50):
        got.append(m.forward_pages([p[at:at + k]], [pieces]).cpu().numpy().copy())
        at += k
    off = _close(np.concatenate(got), want)
    log(f"  off by {off:.3g} of RMS")
    assert m.conversation_length(whole) == m.conversation_length(pieces) == 75
    # 8-bit entries are within half a step of 1/127 of a head's largest: far from the fp16 states, yet near
    m.set_pages(24, size, "int8")
    got = m.forward_pages([p], [m.open_conversation()]).cpu().numpy()
    rms = np.sqrt((want.astype(np.float64) ** 2).mean())
    assert np.sqrt(((got - want).astype(np.float64) ** 2).mean()) < 0.1 * rms
    m.free()


@pytest.mark.parametrize("kind", ["fp16", "int8"])
def test_pages_of_a_batch_decode_greedily(dev, kind):
    """Five conversations read together and decoded in lock step draw what each
    draws alone; with fp16 pages, what greedy() draws."""
    prompts = [prompt(92 + i, k) for i, k in enumerate((9, 30, 1, 17, 33))]
    steps, m = 12, model(dev)
    m.set_pages(40, 16, kind)
    cs = [m.open_conversation() for _ in prompts]
    h = m.forward_pages(prompts, cs)
    last = np.cumsum([len(p) for p in prompts]) - 1
    ids = [m.next_tokens(list(last)).cpu().numpy().copy()]
    m.start_pages(torch.from_numpy(ids[0]).cuda(), cs)
    for _ in range(steps - 1):
        ids.append(m.pages_step().cpu().numpy().copy())
    ids = np.array(ids).T
    for i, p in enumerate(prompts):
        c = m.open_conversation()
        m.forward_pages([p], [c])
        alone = [int(m.next_tokens([len(p) - 1])[0])]
        while len(alone) < steps:
            m.forward_pages([[alone[-1]]], [c])
            alone.append(int(m.next_tokens([0])[0]))
        m.close_conversation(c)
        assert list(ids[i]) == alone
        if kind == "fp16":
            assert list(ids[i]) == m.greedy(p, steps)
    m.free()


@pytest.mark.parametrize("kind", ["fp16", "int8"])
def test_captured_steps_are_the_steps(dev, kind):
    """Replays of the captured step, with eager passes and other steps between,
    leave the eager steps' states bit for bit; past a page's end, and past a
    capture's bound into the next one's."""
    cfg = synth.QwenConfig(256, 512, 2, 4, 2, 64, 1024, 600)
    prompts, runs = [prompt(97, 250), prompt(98, 40), prompt(99, 31)], []
    for graph in (False, True):
        m = model(dev, 81, cfg, 256)
        m.set_pages(80, 16, kind)
        cs = [m.open_conversation() for _ in prompts]
        for p, c in zip(prompts, cs):
            m.forward_pages([p], [c])
        m.start_pages([3, 5, 7], cs)
        seen = []
        for step in range(14):
            ids = m.pages_step(graph).cpu().numpy().copy()
            seen.append((ids, bits(m.hidden[:3]), bits(m.logit[:3])))
            if step in (3, 9):  # another conversation in between
                other = m.open_conversation()
                m.forward_pages([prompt(5, 20)], [other])
                m.close_conversation(other)
                with pytest.raises(ValueError, match="no conversations in lock step"):
                    m.pages_step(graph)
                m.start_pages(torch.from_numpy(ids).cuda(), cs)
        if graph:
            assert sorted(k for k in m.page_graphs) == [(3, 256), (3, 512)]
        runs.append(seen)
        m.free()
    for x, y in zip(*runs):
        for a, b in zip(x, y):
            np.testing.assert_array_equal(a, b)


def test_a_common_beginning_is_shared(dev):
    """A conversation that takes another's first pages goes on as one that read
    them itself, bit for bit, and neither changes the other."""
    m = model(dev)
    start, a, b = prompt(100, 48), prompt(101, 20), prompt(102, 9)
    m.set_pages(16, 16)
    first = m.open_conversation()
    m.forward_pages([start + a[:7]], [first])
    used = 16 - len(m.pool["free"])
    second = m.share_conversation(first, 48)
    assert 16 - len(m.pool["free"]) == used
    own = m.open_conversation()
    m.forward_pages([start], [own])
    want = bits(m.forward_pages([b], [own]))
    np.testing.assert_array_equal(bits(m.forward_pages([b], [second])), want)
    m.close_conversation(own)
    alone = m.open_conversation()
    m.forward_pages([start + a[:7]], [alone])
    want = bits(m.forward_pages([a[7:]], [alone]))
    m.close_conversation(alone)
    np.testing.assert_array_equal(bits(m.forward_pages([a[7:]], [first])), want)
    # a shared page goes back with the last that holds it
    m.close_conversation(first)
    assert 16 - len(m.pool["free"]) == 4
    np.testing.assert_array_equal(m.pool["held"].count(1), 4)
    m.close_conversation(second)
    assert sorted(m.pool["free"]) == list(range(16))
    m.free()


def test_pages_that_come_back(dev):
    """Stale entries of a page's last conversation leave no trace in the next one's."""
    m = model(dev)
    p = prompt(103, 23)
    for kind in ("fp16", "int8"):
        m.set_pages(4, 16, kind)
        c = m.open_conversation()
        want = bits(m.forward_pages([p], [c]))
        m.close_conversation(c)
        for x in m.pool["k"] + m.pool["v"]:
            x.fill_(0x7E00 if kind == "fp16" else 77)  # NaN
        for x in m.pool["ks"] + m.pool["vs"]:
            if x is not None:
                x.fill_(float("nan"))
        c = m.open_conversation()
        np.testing.assert_array_equal(bits(m.forward_pages([p], [c])), want)
    m.free()


def test_pages_leave_the_slots_alone(dev):
    m = model(dev)
    p, q = prompt(104, 21), prompt(105, 18)
    m.reset()
    m.forward(p, 0)
    caches = [x.clone() for x in m.kc + m.vc]
    m.set_pages(8, 16)
    m.forward_pages([q], [m.open_conversation()])
    for x, y in zip(caches, m.kc + m.vc):
        assert torch.equal(x, y)
    assert m.greedy(p, 8) == model(dev).greedy(p, 8)
    m.free()


def test_pages_refusals(dev):
    m = model(dev)
    with pytest.raises(ValueError, match="no pages"):
        m.open_conversation()
    for bad in ((0, 16), (4, 24), (4, 8), (4, 2048)):
        with pytest.raises(ValueError, match="pages of"):
            m.set_pages(*bad)
    with pytest.raises(ValueError, match="pages of 'fp8'"):
        m.set_pages(4, 16, "fp8")
    m.set_pages(3, 16)
    c, d = m.open_conversation(), m.open_conversation()
    with pytest.raises(ValueError, match="twice"):
        m.forward_pages([[1], [2]], [c, c])
    with pytest.raises(IndexError, match="no conversation 9"):
        m.forward_pages([[1]], [9])
    with pytest.raises(ValueError, match="0 tokens"):
        m.forward_pages([[]], [c])
    with pytest.raises(ValueError, match="for a batch of 96"):
        m.forward_pages([[1] * 97], [c])
    m.forward_pages([[1] * 17], [c])
    with pytest.raises(ValueError, match="2 pages wanted, 1 free"):
        m.forward_pages([[1] * 17], [d])
    assert m.conversation_length(d) == 0 and len(m.pool["free"]) == 1
    with pytest.raises(ValueError, match="no whole pages"):
        m.share_conversation(c, 17)
    with pytest.raises(ValueError, match="no whole pages"):
        m.share_conversation(c, 32)
    with pytest.raises(ValueError, match="no conversations in lock step"):
        m.pages_step()
    m.start_pages([1], [c])
    m.forward([1, 2], 0)
    with pytest.raises(ValueError, match="no conversations in lock step"):
        m.pages_step()
    m.close_conversation(c)
    with pytest.raises(IndexError):
        m.conversation_length(c)
    m.set_pages(40, 16)
    c = m.open_conversation()
    for _ in range(5):
        m.forward_pages([[1] * 32], [c])
    with pytest.raises(ValueError, match="exceed the context 160"):
        m.forward_pages([[1]], [c])
    m.start_pages([1], [c])
    with pytest.raises(ValueError, match="exceed the context 160"):
        m.pages_step()
    m.free()


def test_lock_step_tokens_are_one_a_conversation(dev):
    """A single id in a tensor would reach every conversation, a longer one none."""
    m = model(dev)
    m.set_pages(8, 16)
    c, d = m.open_conversation(), m.open_conversation()
    for tokens in (dev.put(np.array([5], np.int32)), [5], [5, 6, 7], 5):
        with pytest.raises(ValueError, match="2 conversations for tokens of shape"):
            m.start_pages(tokens, [c, d])
    m.start_pages([5, 6], [c, d])
    m.pages_step()
    m.free()


def test_rope_scaling(dev):
    """Scaled tables reach every kind of pass, and plain ones are the model's again."""
    m = model(dev)
    p = prompt(106, 40)
    plain = bits(m.forward(p, 0))
    tables = bits(m.rope_cos), bits(m.rope_sin)
    m.set_rope_scaling("linear", 1.0)
    assert np.mean(bits(m.rope_cos) != tables[0]) < 1e-3
    m.set_rope_scaling("ramp", 4.0, original=64)
    theta = np.arange(m.rope_cos.shape[0])[:, None] * 1e6 ** (-2.0 * np.arange(32) / 64)
    lo, hi = (64 * math.log(64 / (2 * math.pi * t)) / (2 * math.log(1e6)) for t in (32.0, 1.0))
    u = np.clip((np.arange(32) - max(math.floor(lo), 0)) / (min(math.ceil(hi), 63) - max(math.floor(lo), 0)), 0, 1)
    want = (0.1 * math.log(4.0) + 1) * np.cos(theta * (1 - u) + theta / 4 * u)
    np.testing.assert_allclose(m.rope_cos.cpu().numpy(), want, rtol=0, atol=2.0 ** -23)
    slots = m.forward(p, 0).cpu().numpy().copy()
    assert not np.array_equal(slots.view(np.uint32), plain)
    m.set_pages(8, 16)
    _close(m.forward_pages([p], [m.open_conversation()]).cpu().numpy(), slots)
    with pytest.raises(ValueError, match="scaled by"):
        m.set_rope_scaling("yes")
    with pytest.raises(ValueError, match="original context"):
        m.set_rope_scaling("turns", 2.0)
    with pytest.raises(capi.GxError, match="factor of 0"):
        m.set_rope_scaling("linear", 0.0)
    m.set_rope_scaling("plain")
    np.testing.assert_array_equal(bits(m.rope_cos), tables[0])
    np.testing.assert_array_equal(bits(m.forward(p, 0)), plain)
    m.free()


def test_workspaces_of_passes_over_pages_go_back(dev):
    """Passes of rising sizes leave no more behind than a few times the largest
    one's workspace, and a new pool leaves none."""
    cfg = synth.QwenConfig(256, 512, 2, 16, 1, 64, 1024, 2048)
    m = model(dev, 110, cfg, 400)
    m.set_pages(64, 64)
    m.forward_pages([prompt(111, 8)], [m.open_conversation()])
    before, largest = torch.cuda.memory_allocated(), 0
    for k in range(40, 400, 8):
        c = m.open_conversation()
        for piece in range(3):
            m.forward_pages([prompt(112 + piece, k)], [c])
            largest = max(largest, capi.size_out("gx_qwen_attention_paged_workspace_bytes", 1, k, k, 16, 1, 64, (piece + 1) * k))
        m.close_conversation(c)
    log(f"  {torch.cuda.memory_allocated() - before} bytes more, the largest workspace {largest}")
    assert largest > 4 << 20 and torch.cuda.memory_allocated() - before <= 4 * largest
    m.set_pages(1, 16)
    m.pool = None
    assert torch.cuda.memory_allocated() < before
    m.free()


def test_captured_steps_keep_their_workspace(dev):
    """A captured step replayed after a pass whose workspace outgrew its own, and
    after what that freed has been written over, gives the eager step's bits."""
    cfg = synth.QwenConfig(256, 512, 2, 16, 1, 64, 1024, 4096)
    runs = []
    for graph in (False, True):
        m = model(dev, 113, cfg, 400)
        m.set_pages(128, 64)
        c = m.open_conversation()
        for piece in range(6):
            m.forward_pages([prompt(114 + piece, 400)], [c])
        m.page_ws = None  # (the captured step's own is then a small one)
        m.start_pages([3], [c])
        seen = []
        for step in range(6):
            ids = m.pages_step(graph).cpu().numpy().copy()
            seen.append((ids, bits(m.hidden[:1]), bits(m.logit[:1])))
            if step in (1, 3):
                other = m.open_conversation()
                for piece in range(3):
                    m.forward_pages([prompt(5 + piece, 390)], [other])
                m.close_conversation(other)
                held = [torch.full((1 << k,), 0xFF, dtype=torch.uint8, device="cuda") for k in range(12, 26) for _ in range(3)]
                torch.cuda.synchronize()
                del held
                m.start_pages(torch.from_numpy(ids).cuda(), [c])
        runs.append(seen)
        m.free()
    for x, y in zip(*runs):
        for a, b in zip(x, y):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("where", ["tokens", "workspace", "blocks"])
def test_a_pass_that_fails_takes_no_pages(dev, where):
    """Pages, lengths and later steps as if the failed pass had not been asked for."""
    cfg = synth.QwenConfig(256, 512, 2, 4, 2, 64, 1024, 1024)
    m = model(dev, 115, cfg, 400)
    m.set_pages(60, 16)
    c, d = m.open_conversation(), m.open_conversation()
    m.forward_pages([prompt(116, 20), prompt(117, 9)], [c, d])
    free, lists = list(m.pool["free"]), {k: list(v) for k, v in m.pool["lists"].items()}

    def fail(*a, **kw):
        raise RuntimeError("out of memory")

    if where == "tokens":
        with pytest.raises((TypeError, ValueError)):
            m.forward_pages([["x"] * 350, [1]], [c, d])
    else:
        name = {"workspace": "_page_workspace", "blocks": "_blocks"}[where]
        setattr(m, name, fail)
        with pytest.raises(RuntimeError, match="out of memory"):
            m.forward_pages([prompt(118, 350), [1]], [c, d])
        m.start_pages([1, 2], [c, d])
        for _ in range(2):
            with pytest.raises(RuntimeError, match="out of memory"):
                m.pages_step()
        delattr(m, name)
    assert m.pool["free"] == free and m.pool["lists"] == lists
    assert m.pool["held"] == [sum(p in x for x in lists.values()) for p in range(60)]
    assert m.conversation_length(c) == 20 and m.conversation_length(d) == 9
    other = model(dev, 115, cfg, 400)
    other.set_pages(60, 16)
    cs = [other.open_conversation() for _ in range(2)]
    other.forward_pages([prompt(116, 20), prompt(117, 9)], cs)
    for x, y in ((m, [c, d]), (other, cs)):
        x.start_pages([1, 2], y)
    for _ in range(14):
        np.testing.assert_array_equal(m.pages_step().cpu().numpy(), other.pages_step().cpu().numpy())
        np.testing.assert_array_equal(bits(m.hidden[:2]), bits(other.hidden[:2]))
    other.free()
    m.free()


def test_conversations_of_a_replaced_pool_are_gone(dev):
    """A number from before set_pages names no conversation of the new pool."""
    m = model(dev)
    m.set_pages(4, 16)
    old = m.open_conversation()
    m.set_pages(4, 16)
    new = m.open_conversation()
    assert new != old
    for call in (lambda: m.forward_pages([[1]], [old]), lambda: m.start_pages([1], [old]),
                 lambda: m.share_conversation(old, 0), lambda: m.close_conversation(old)):
        with pytest.raises(IndexError, match=f"no conversation {old} "):
            call()
    m.free()


def test_captures_leave_the_stream_as_it_was(dev):
    """A model whose context works on a stream of its own: after a capture its
    passes are on that stream again."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = capi.Context(0, stream=stream.cuda_stream)
        m = QwenModel(ctx, CFG, synth.qwen_weights(CFG, 81, symmetric=True), max_batch=96)
        stream.synchronize()
        seen, call = [], m._call

        def watched(name, *args):
            if name == "gx_set_stream":
                seen.append(args[1].value if hasattr(args[1], "value") else args[1])
            return call(name, *args)

        m._call = watched
        m.set_pages(8, 16)
        c = m.open_conversation()
        m.forward_pages([prompt(119, 20)], [c])
        m.start_pages([5], [c])
        m.pages_step(graph=True)
        m.capture_decode()
        m.set_slots(2)
        m.capture_slots(2)
        assert len(seen) == 6 and seen[1::2] == [stream.cuda_stream] * 3
        stream.synchronize()
        m.free()
        ctx.close()
