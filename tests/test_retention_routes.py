"""How a call of the linear attention chooses to run its sequences, on the host."""

import os
import re

import pytest

from mamba4_amd import _lib

DATA = 1 << 20  # stands for device memory: nothing here is launched
SOURCE = os.path.join(os.path.dirname(_lib.LIBRARY), "csrc", "api_retention.hip")


def _qkv(heads, n, p):
    return _lib.pack_qkv(*[x for w in (n, n, p) for x in (DATA, 0, heads * w, w, heads, w)])


def _sizes(T, H=2, n=64, p=64, decays=0):
    lib, rows = _lib.load(), _qkv(H, n, p)
    return (lib.m4rt_attention_workspace_bytes(rows, 0, 1, T, H),
            lib.m4rt_attention_backward_workspace_bytes(rows, DATA, 0, 1, T, H, decays))


def test_the_override_sets_the_workspace(monkeypatch):
    """A walk keeps no segments' states, a split one slot a segment (4 chunks of 64
    tokens) and tile: 64 x 64 floats and the decay."""
    monkeypatch.setenv("M4RT_ATTENTION", "walk")
    assert _sizes(600) == (0, 0)
    monkeypatch.setenv("M4RT_ATTENTION", "split")
    slots = 2 * 3
    one = slots * 64 * 64 * 4 + 256
    assert _sizes(600) == (one, 3 * one)


def test_a_call_makes_its_choice_once():
    """The environment may change between two looks at it (another thread's setenv):
    the workspace would be carved for one route and the other one launched.  So each
    entry point settles the route in one place and passes it on."""
    text = open(SOURCE).read()
    body = text[text.index('extern "C" {\n\nsize_t m4rt_attention_workspace_bytes'):]
    entries = re.split(r"\n(?=(?:size_t|int) m4rt_)", body)
    looks = {e.split("(")[0].split()[-1]: e.count("attention_route(") for e in entries
             if " m4rt_attention" in e.split("(")[0]}
    assert looks == {"m4rt_attention_workspace_bytes": 1, "m4rt_attention_forward": 1,
                     "m4rt_attention_backward_workspace_bytes": 1, "m4rt_attention_backward": 1,
                     "m4rt_attention_step": 0}
    assert len(re.findall(r"\battention_splits\(", text)) == 2  # its definition, the route's
    assert text.count("getenv") == 1


def test_segments_of_the_longest_sequences_fit_a_launch(monkeypatch):
    """65,535 blocks along y at most: 16-chunk segments reach that at 67M tokens."""
    monkeypatch.setenv("M4RT_ATTENTION", "split")
    slot = 64 * 64 * 4
    for T, chunks in ((65535 * 1024, 16), (65535 * 1024 + 1, 32), (2**27 - 16, 64)):
        count = -(-T // (64 * chunks))
        assert count <= 65535
        assert _sizes(T, H=1)[0] == count * slot + -(-4 * count // 256) * 256
