"""Env workers are forked from a process that may own GPU objects: nothing that a worker inherits may be finalised in it."""
import gc
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

_after_fork = []  # called in every child of this process, before anything else runs in it
os.register_at_fork(after_in_child=lambda: [f() for f in _after_fork])


class _Owned:
    """Stands for an object whose finaliser calls a runtime that does not survive a fork; in a reference cycle, so that only a collection ends it."""

    def __init__(self, pipe):
        self.pipe, self.me = pipe, self

    def __del__(self):
        os.write(self.pipe, b"%d\n" % os.getpid())


def _many_containers():
    return [[i] for i in range(20000)]  # enough for the collector to run by itself, old generations too


class _CollectingEnv:
    """Two agents; a worker that resets it collects."""
    n_agents = 2

    def __init__(self):
        import numpy as np
        self.obs, self.state, self.avail = np.zeros((2, 3), np.float32), np.zeros(4, np.float32), np.ones((2, 5), np.uint8)

    def reset(self, seed=None):
        _many_containers()
        gc.collect()
        return self.obs, {}

    def get_state(self):
        return self.state

    def get_avail_actions(self):
        return self.avail

    def get_obs_size(self):
        return 3

    def get_state_size(self):
        return 4

    def get_action_size(self):
        return 5

    def close(self):
        pass


@pytest.mark.parametrize("kind", ["pipe", "shm"])
@pytest.mark.parametrize("collecting", [True, False])
def test_nothing_inherited_is_finalised_in_a_worker(kind, collecting, monkeypatch):
    """A dropped cycle with a finaliser is there at the fork; the child makes enough objects for a collection at once, and its env collects on reset.
    A worker collects again afterwards if its parent does."""
    from cleanmarl_amd.env import shm_vector, vector
    monkeypatch.setattr(shm_vector, "environment", lambda **kw: _CollectingEnv())
    monkeypatch.setattr(vector, "environment", lambda **kw: _CollectingEnv())
    got, put = os.pipe()
    states, report = os.pipe()
    was, threshold = gc.isenabled(), gc.get_threshold()
    real_reset = _CollectingEnv.reset

    def reset(self, seed=None):
        os.write(report, b"1" if gc.isenabled() else b"0")
        return real_reset(self, seed)
    monkeypatch.setattr(_CollectingEnv, "reset", reset)
    _after_fork.append(_many_containers)
    v = None
    try:
        (gc.enable if collecting else gc.disable)()
        gc.collect()
        gc.set_threshold(10 ** 6, *threshold[1:])  # the parent itself does not collect it before the fork; its workers have ordinary thresholds
        _after_fork.append(lambda: gc.set_threshold(*threshold))
        _after_fork.reverse()
        for _ in range(20):
            _Owned(put)
        fac = dict(env_type="pz", env_name="x", env_family="mpe", agent_ids=True)
        v = vector.PipeVectorEnv(2, fac) if kind == "pipe" else shm_vector.ShmVectorEnv(2, fac, n_workers=2)
        assert gc.isenabled() == collecting  # the parent is as it was
        if kind == "pipe":
            v.reset_all()
        else:
            v._all("reset")
        assert os.read(states, 16) == (b"11" if collecting else b"00")
    finally:
        _after_fork.clear()
        gc.set_threshold(*threshold)
        if v is not None:
            v.close()
        (gc.enable if was else gc.disable)()
    gc.collect()
    os.close(put)
    with os.fdopen(got) as f:
        pids = [int(line) for line in f.read().split()]
    os.close(states); os.close(report)
    assert pids == [os.getpid()] * 20, f"{sum(p != os.getpid() for p in pids)} finalisers ran in workers"


def test_a_closed_host_rollout_keeps_no_page_locked_memory(monkeypatch):
    """Whoever still refers to it (a reference cycle, a frame that a forked worker inherits): close() itself lets go of the twins, behind the copies that use them."""
    import weakref

    import torch
    from cleanmarl_amd import host_rollout
    from cleanmarl_amd.env.shm_vector import ShmVectorEnv

    class Stream:
        def synchronize(self):
            order.append(len([w for w in twins if w() is not None]))

    order, real = [], torch.empty
    monkeypatch.setattr(host_rollout.torch, "empty", lambda *a, pin_memory=False, **kw: real(*a, **kw))  # ordinary memory stands in for page-locked
    monkeypatch.setattr(host_rollout.N, "load", lambda: None)
    fac = dict(env_type="synthetic_cpu", env_name="x", env_family="mpe", agent_ids=True, kwargs={}, seed=3, synthetic=dict(agents=2, steps=3))
    v = ShmVectorEnv(3, fac, n_workers=1)
    roll = host_rollout.PinnedHostRollout(v, None, False, torch.device("cpu"), t_cap=3)
    roll.myself = roll
    try:
        twins = [weakref.ref(t) for t in (roll.h_obs, roll.h_state, roll.h_avail, roll.h_act)]
        roll.stream = Stream()
        roll.close()
        assert order == [4] and [w() for w in twins] == [None] * 4
        roll.close()  # closing twice is closing once
        assert order == [4]
    finally:
        v.close()


@pytest.mark.gpu
@pytest.mark.parametrize("recurrent", [False, True])
def test_a_host_rollout_leaves_torchs_host_threads_alone(recurrent):
    """The env workers need the cores: no step of an episode runs a torch operation between host tensors (one of this size would wake every thread of torch's
    pool, and they spin)."""
    import torch
    from torch.utils._python_dispatch import TorchDispatchMode
    from cleanmarl_amd.env.shm_vector import ShmVectorEnv
    from cleanmarl_amd.gru import GRUPPOLearner
    from cleanmarl_amd.host_rollout import PinnedHostRollout
    from cleanmarl_amd.learner import HParams, NetSpec, PPOLearner

    class OnTheHost(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            there = [t for t in (*args, out) if isinstance(t, torch.Tensor)]
            if len(there) > 1 and all(t.device.type == "cpu" for t in there) and max(t.numel() for t in there) > 10000:
                seen.append(str(func))
            return out

    seen, E, A, T = [], 64, 8, 6
    dev = torch.device("cuda:0")
    fac = dict(env_type="synthetic_cpu", env_name="x", env_family="mpe", agent_ids=True, kwargs={}, seed=3, synthetic=dict(agents=A, steps=T))
    kind = GRUPPOLearner if recurrent else PPOLearner
    v = ShmVectorEnv(E, fac, n_workers=2)
    actor = NetSpec(7 * A, 64, 0, 5, "gru") if recurrent else NetSpec(7 * A, 64, 1, 5)
    roll = PinnedHostRollout(v, kind("mappo", actor, NetSpec(6 * A * A, 64, 1, 1), A, HParams(), dev), recurrent, dev, t_cap=T)
    try:
        assert min(a.size for a in (v.arr["obs"], v.arr["state"])) > 10000  # blocks that count
        roll.collect(1)
        with OnTheHost():
            roll.collect(2)
    finally:
        roll.close()
        v.close()
    assert seen == []
