"""Misuse of the entry points for drafted trees is named before anything
else, without a GPU: every argument check runs ahead of the context's."""
import ctypes

import pytest

from golem_amd import capi

A = 0x10000  # an aligned address that no call here reads


def refused(name, args, message):
    with pytest.raises(capi.GxError, match=message):
        capi.call(name, *args)


def _change(base, changes):
    args = dict(base)
    args.update(changes)
    return list(args.values())


PLAN = dict(ctx=None, n=1, M=4, max_nodes=4, first=A, parents=A, prefix=A, cos=A, sin=A, half=32, context=64, rows=A,
            positions=A, mask=A, oc=A, os=A)


@pytest.mark.parametrize("changes,message", [
    ({}, "no context"), ({"n": -1}, "trees"), ({"n": 1025}, "at most 1024"), ({"M": -1}, "tokens"),
    ({"M": 65536}, "at most 65535"), ({"max_nodes": 0}, "trees of 0 nodes"), ({"max_nodes": 513}, "1 to 512"),
    ({"half": 0}, "rotation tables"),
    ({"half": 513}, "at most 512"), ({"context": 0}, "rotation tables"), ({"parents": None}, "missing"),
    ({"os": None}, "missing"),
])
def test_plan(changes, message):
    refused("gx_qwen_tree_plan", _change(PLAN, changes), message)


ATTENTION = dict(ctx=None, qh=A, n=1, M=4, max_nodes=4, first=A, mask=A, prefix=A, max_prefix=10, heads=4, kv_heads=2,
                 head_dim=64, kc=A, vc=A, context=64, kd=A, vd=A, draft_context=8, out=A, q=None, scales=None,
                 qsum=None, ws=A, size=1 << 30, slots=None, nslots=0)


@pytest.mark.parametrize("changes,message", [
    ({}, "no context"), ({"heads": 5}, "5 query heads over 2"), ({"kv_heads": 0}, "query heads"),
    ({"heads": 4098}, "at most 4096"), ({"head_dim": 80}, "32, 64, 96 and 128"), ({"max_prefix": -1}, "prefix of -1"),
    ({"max_prefix": 65}, "cannot hold 65"), ({"context": 60}, "multiple of 8"), ({"draft_context": 4}, "draft buffers"),
    ({"M": 9}, "cannot hold 9"), ({"context": 1 << 26}, "too long"), ({"out": None}, "missing"),
    ({"q": A}, "missing"), ({"qh": A + 2}, "16-byte"), ({"vd": A + 8}, "16-byte"), ({"ws": A + 64}, "256-byte"),
    ({"ws": None}, "missing"), ({"slots": A}, "0 slots"), ({"size": 100}, "the workspace holds 100 bytes"),
    ({"mask": None}, "missing"),
])
def test_attention(changes, message):
    refused("gx_qwen_attention_tree", _change(ATTENTION, changes), message)


def test_attention_workspace():
    size = ("gx_qwen_attention_tree_workspace_bytes",)
    one = capi.size_out(*size, 1, 4, 4, 4, 2, 64, 10)
    assert one % 256 == 0 and one >= 4 * 4 * 66 * 4
    # the largest there is neither overflows nor shrinks
    assert capi.size_out(*size, 1024, 65535, 512, 32, 8, 128, 1 << 20) >= 65535 * 32 * 130 * 4
    assert capi.size_out(*size, 0, 0, 1, 4, 2, 64, 0) == 0
    refused(size[0], [1, 4, 4, 4, 2, 64, 10, None], "no place")


VERIFY = dict(ctx=None, logits=A, ldl=100, n=1, M=4, max_nodes=4, vocab=100, first=A, parents=A, tokens=A, draft=None,
              ldd=0, temperature=0.7, draft_temperature=0.7, uniforms=A, path=A, counts=A, next=A, ws=A, size=1 << 30)


@pytest.mark.parametrize("changes,message", [
    ({}, "no context"), ({"vocab": 0}, "vocabulary of 0"), ({"vocab": (1 << 20) + 1, "ldl": 1 << 21}, "vocabulary"),
    ({"ldl": 99}, "bad shape"), ({"draft": A, "ldd": 99}, "bad shape"), ({"temperature": -0.5}, "temperature of -0.5"),
    ({"temperature": float("nan")}, "temperature"), ({"temperature": float("inf")}, "temperature"),
    ({"draft": A, "ldd": 100, "draft_temperature": 0.0}, "draft temperature"), ({"uniforms": None}, "missing"),
    ({"uniforms": None, "temperature": 0.0}, "no context"), ({"tokens": None}, "missing"),
    ({"ws": A + 8}, "256-byte"), ({"size": 0}, "the workspace holds 0 bytes"),
])
def test_verify(changes, message):
    refused("gx_tree_verify", _change(VERIFY, changes), message)


def _layers(*addresses):
    return (ctypes.c_void_p * len(addresses))(*addresses)


COMMIT = dict(ctx=None, layers=2, kc=_layers(A, A), vc=_layers(A, A), kd=_layers(A, A), vd=_layers(A, A), n=1, M=4,
              max_nodes=4, first=A, path=A, counts=A, prefix=A, kv_heads=2, head_dim=64, context=64, draft_context=8,
              slots=None, nslots=0)


@pytest.mark.parametrize("changes,message", [
    ({}, "no context"), ({"layers": 0}, "0 layers"), ({"kc": _layers(A, None)}, "layer 1"),
    ({"vc": _layers(A + 2, A)}, "layer 0"), ({"kd": _layers(A, A + 4)}, "layer 1"), ({"vd": _layers(None, A)}, "layer 0"),
    ({"head_dim": 60}, "key-value heads of 60"), ({"context": 12}, "multiple of 8"), ({"draft_context": 2}, "draft buffers"),
    ({"context": 1 << 25}, "too long"), ({"path": None}, "missing"), ({"slots": A}, "0 slots"), ({"kd": None}, "missing"),
])
def test_commit(changes, message):
    refused("gx_qwen_cache_commit", _change(COMMIT, changes), message)


def _slots(*s):
    return (ctypes.c_int32 * len(s))(*s)


FORK = dict(ctx=None, layers=2, kc=_layers(A, A), vc=_layers(A, A), nslots=4, kv_heads=2, head_dim=64, context=64, src=1,
            dsts=_slots(0, 3), n=2, len=10)


@pytest.mark.parametrize("changes,message", [
    ({}, "no context"), ({"src": 4}, "slot 4 of 4"), ({"src": -1}, "slot -1"), ({"dsts": _slots(0, 4)}, "slot 4 of 4"),
    ({"dsts": _slots(1, 0)}, "into itself"), ({"dsts": _slots(2, 2)}, "named twice"), ({"n": 4}, "4 forks"),
    ({"n": -1}, "-1 forks"), ({"len": 65}, "65 positions"), ({"len": -1}, "-1 positions"), ({"kc": None}, "missing"),
    ({"dsts": None}, "forks among"), ({"context": 1 << 25}, "too long"),
])
def test_fork(changes, message):
    refused("gx_qwen_cache_fork", _change(FORK, changes), message)
