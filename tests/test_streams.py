"""runtime.branch_stream: the streams that a capture forks into are never one hardware stream, whatever else draws from torch's pool."""
import os
import re

import pytest
import torch

from efficientvlm_amd import runtime

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROLES = ["capture", "text", "teacher", "warm", "prefetch", "exchange", "loop", "l0"]


class Ring:
    """torch's pool: a stream is one of `size` handles, in turn"""

    def __init__(self, size=32, offset=0):
        self.size, self.next = size, offset

    def __call__(self, device):
        handle = 1000 * (device + 1) + self.next % self.size
        self.next += 1
        return type("Stream", (), {"cuda_stream": handle})()


@pytest.fixture
def fresh(monkeypatch):
    monkeypatch.setattr(runtime, "_BRANCHES", {})


@pytest.mark.parametrize("offset", range(32))
def test_roles_never_share_a_stream(fresh, offset, monkeypatch):
    for gap in range(33):                                     # streams that the program draws for itself between two roles
        monkeypatch.setattr(runtime, "_BRANCHES", {})
        ring = Ring(offset=offset)
        got = {}
        for role in ROLES:
            got[role] = runtime.branch_stream(role, torch.device("cuda", 0), ring)
            for _ in range(gap):
                ring(0)
        assert len({s.cuda_stream for s in got.values()}) == len(ROLES)
        for role in reversed(ROLES):                          # the same ones ever after
            assert runtime.branch_stream(role, 0, ring) is got[role]


def test_streams_drawn_on_their_own_coincide():
    """what branch_stream is there for: of 33 numbers of foreign draws between two siblings, one puts them onto one stream"""
    same = 0
    for gap in range(33):
        ring = Ring()
        first = ring(0).cuda_stream
        for _ in range(gap):
            ring(0)
        same += ring(0).cuda_stream == first
    assert same == 1


def test_devices_are_apart_and_a_small_pool_is_refused(fresh):
    ring = Ring(size=3)
    for role in ROLES[:3]:
        runtime.branch_stream(role, 0, ring)
    with pytest.raises(RuntimeError, match="of its own"):
        runtime.branch_stream(ROLES[3], 0, ring)
    assert runtime.branch_stream(ROLES[3], 1, ring).cuda_stream >= 2000      # another device has a pool of its own


def test_the_package_draws_no_stream_elsewhere():
    """every other torch.cuda.Stream() of the package could coincide with one of these (a stream of another priority is of another pool)"""
    found = []
    for folder, _, names in os.walk(os.path.join(ROOT, "efficientvlm_amd")):
        for name in names:
            if name.endswith(".py"):
                text = open(os.path.join(folder, name)).read()
                found += [(name, m) for m in re.findall(r"cuda\.Stream\(([^)]*)\)", re.sub(r'""".*?"""|#[^\n]*', "", text, flags=re.S))]
    assert sorted(set(found)) == [("runtime.py", "device=index"), ("trainer.py", "priority=-1")]
    trainer = open(os.path.join(ROOT, "efficientvlm_amd", "trainer.py")).read()
    for call in re.findall(r"torch\.cuda\.graph\((?:[^()]|\([^()]*\))*\)", trainer):
        assert "stream=" in call, call                        # (torch's own capture stream is drawn from the same pool)
