"""What a net that reads tokens holds for its callers' graphs (CPU only, a library that is not there)."""
import gc

import numpy as np
import pytest

from test_operator_refusals import Fake


class Library:
    """Memory that is given and taken back; everything else does nothing."""

    def __init__(self, real):
        self.real, self.at, self.freed, self.calls = real, 0, [], []

    def call(self, name, *args):
        if name == "sb_malloc":
            self.at += 1 << 32
            args[0]._obj.value = self.at
        elif name == "sb_free":
            self.freed.append(args[0])
        elif name.endswith("_bytes") or name.endswith("_offsets") or name.endswith("_offset"):
            self.real(name, *args)
        else:
            self.calls.append((name, args))


@pytest.fixture
def net(sb, monkeypatch):
    from spiral_b200 import _lib, device
    lib = Library(_lib.call)
    monkeypatch.setattr(_lib, "call", lib.call)
    monkeypatch.setattr(device, "_WORKSPACES", type(device._WORKSPACES)())
    policy = sb.TokenPolicy(16, 4, 8, [64], 8, 32, gated=24, training=True)
    gc.collect()
    lib.freed.clear()
    yield lib, policy
    gc.collect()


def places(lib, name, *which):
    args = [a for n, a in lib.calls if n == name][-1]
    return [args[i] for i in which]


def test_evaluations_of_other_alternatives_free_nothing(net):
    lib, policy = net
    tokens, actions = Fake((32, 4), "int32"), Fake((32,), "int32")
    held = {}
    for top in (2, 0, 5, 2, 0, 5):
        got = policy.evaluate(tokens, actions, top=top)
        assert set(got) == {"log_probs", "entropy"} | ({"top_log_probs", "top_actions"} if top else set())
        if top:
            assert got["top_actions"].shape == got["top_log_probs"].shape == (32, top)
        del got
        at = places(lib, "sb_log_probs", 10, 11, 12, 13, 14, 15)                   # out, entropy, stats, top and the alternatives
        assert held.setdefault(top, at) == at and at[3] == top
    gc.collect()
    assert not lib.freed
    policy.policy_gradients(tokens, actions, Fake((32,)))
    assert places(lib, "sb_log_probs_grad", 10, 12) == [held[5][2], held[5][1]]          # the statistics and entropies that evaluate() left


def test_codes_of_other_groups_free_nothing(net):
    lib, policy = net
    tokens = Fake((32, 4), "int32")
    held = {}
    for group in (128, 32, 128, 32):
        policy.quantize_4bit(group).forward_4bit(tokens)
        at = places(lib, "sb_matmul_int4", 3, 5, 12)                               # codes, scales, group
        assert held.setdefault(group, at) == at and at[2] == group
    gc.collect()
    assert not lib.freed and held[128] != held[32]
    policy.optimizer.calls += 1                                                    # weights have changed: the codes of this group are made anew
    before = len(lib.calls)
    policy.forward_4bit(tokens)
    assert [n for n, _ in lib.calls[before:]].count("sb_quantize_int4") == 2
    policy.quantize_4bit(128)
    before = len(lib.calls)
    policy.forward_4bit(tokens)
    assert "sb_quantize_int4" not in [n for n, _ in lib.calls[before:]]
