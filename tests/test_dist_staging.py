"""What the gloo path hands to the collective (no GPU needed: the tensors are fake ones, with a device and without data).

gloo gets host memory only: ranks that share one GPU have hung in its collectives on device tensors.  RCCL gets the device tensor itself."""
import os
import sys

import pytest
import torch
import torch.distributed as dist
from torch._subclasses.fake_tensor import FakeTensorMode

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)


@pytest.fixture
def mod():
    import __graft_entry__ as ge
    return ge.load_package().dist


@pytest.fixture
def two_ranks(monkeypatch):
    """a group of two ranks whose collective only notes what it was given"""
    seen = []
    config = ["cpu:gloo,cuda:gloo"]
    monkeypatch.setattr(dist, "is_initialized", lambda: True)
    monkeypatch.setattr(dist, "get_world_size", lambda group=None: 2)
    monkeypatch.setattr(dist, "get_backend_config", lambda group=None: config[0])
    monkeypatch.setattr(dist, "get_backend", lambda group=None: "gloo" if config[0].endswith("gloo") else "nccl")
    monkeypatch.setattr(dist, "all_reduce", lambda t, op=None, group=None: seen.append((t.device.type, tuple(t.shape), op)))
    return seen, config


@pytest.mark.parametrize("config,device,expected", [("cpu:gloo,cuda:gloo", "cuda", "cpu"), ("cpu:gloo,cuda:gloo", "cpu", "cpu"), ("cuda:nccl", "cuda", "cuda"),
                                                    ("cpu:gloo,cuda:nccl", "cuda", "cuda"), ("cpu:gloo,cuda:nccl", "cpu", "cpu")])
def test_combine_means_gives_gloo_host_memory_only(mod, two_ranks, config, device, expected):
    seen, cfg = two_ranks
    cfg[0] = config
    with FakeTensorMode():
        acc = torch.empty(7, 3, device=device)
        assert mod.combine_means(acc, 4) is acc
    assert acc.device.type == device
    assert seen == [(expected, (7 * 3 + 1,), dist.ReduceOp.SUM)]


@pytest.mark.parametrize("host_only", [True, False])
def test_all_reduce_writes_the_result_back(mod, two_ranks, monkeypatch, host_only):
    """the staged and the direct form leave the reduced values in the caller's tensor"""
    monkeypatch.setattr(mod, "_host_only", lambda t, group=None: host_only)
    monkeypatch.setattr(dist, "all_reduce", lambda t, op=None, group=None: t.add_(1.0))
    t = torch.zeros(5, dtype=torch.float64)
    assert mod.all_reduce(t, dist.ReduceOp.MAX) is t
    assert t.tolist() == [1.0] * 5


def test_bench_calls_no_collective_on_its_own():
    """bench.py reduces through the package, which stages; a barrier carries no tensor"""
    with open(os.path.join(ROOT, "bench.py")) as f:
        calls = [l.strip() for l in f if "dist." in l and any(c in l for c in ("all_reduce", "broadcast", "all_gather", "reduce_scatter", "all_to_all"))]
    assert all(".dist.all_reduce(" in c for c in calls), calls
