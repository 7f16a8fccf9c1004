"""When captured graphs may be freed: a trainer that nobody holds goes at once (with its graph, streams and arenas), not whenever the cyclic
collector runs.  On the CPU: the objects are built as on the GPU, nothing is launched."""
import gc
import weakref

import pytest
import torch


class _Store:
    def __init__(self):
        self.root_frames = torch.zeros(1)


@pytest.fixture
def trainer(monkeypatch):
    from diffuser.diffusion_policy.get_dp import build_policy, DEFAULT_CONF
    from v2a_hip.policy_engine import PolicyEngine
    from v2a_hip.trainer import PolicyTrainer

    def engine(self):                       # the policy's own property refuses a CPU device
        if self.__dict__.get("_engine") is None:
            self.__dict__["_engine"] = PolicyEngine(self._cfg, dict(self.named_parameters()))
        return self.__dict__["_engine"]

    def build(**kw):
        pol = build_policy(DEFAULT_CONF)
        monkeypatch.setattr(type(pol), "engine", property(engine))
        return PolicyTrainer(pol, _Store(), batch_size=2, **kw)
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t, *a, **k: t)
    return build


@pytest.mark.parametrize("presum", [False, True])
def test_a_dropped_trainer_is_freed_without_the_cyclic_collector(trainer, presum):
    tr = trainer(presum=presum)
    assert (tr._presum_range[1] > 0) == presum
    eng, ref = tr.eng, weakref.ref(tr)
    gc.collect()
    gc.disable()
    try:
        del tr
        assert ref() is None
    finally:
        gc.enable()
    if presum:
        eng.on_unet_wgrads_done()           # a backward through the engine that outlives its trainer: nothing to arm


def test_the_weight_gradient_hook_reaches_a_live_trainer(trainer, monkeypatch):
    tr = trainer(presum=True)
    calls = []
    monkeypatch.setattr(tr.opt, "presum", lambda *a: calls.append(a))
    tr.eng.on_unet_wgrads_done()            # outside the trainer's own step
    assert calls == [] and not tr._presummed
    tr._in_step = True
    tr.eng.on_unet_wgrads_done()
    assert calls == [tr._presum_range] and tr._presummed


class _Noted:
    """Finalizer that says whether a capture was under way."""

    def __init__(self, log, state):
        self.me, self.log, self.state = self, log, state

    def __del__(self):
        self.log.append(self.state["capturing"])


@pytest.fixture
def fake_graph(monkeypatch):
    """torch.cuda.graph without a GPU: only whether a capture is under way, and with which arguments it began."""
    import contextlib
    state = {"capturing": 0, "kw": []}

    @contextlib.contextmanager
    def graph(g, **kw):
        state["capturing"] += 1
        state["kw"].append((g, kw))
        try:
            yield
        finally:
            state["capturing"] -= 1
    monkeypatch.setattr(torch.cuda, "graph", graph)
    return state


def _allocate():
    """More container objects than any threshold of the collector's youngest generation, all alive, so that older generations are due too."""
    return [[i] for i in range(200000)]


def test_no_cyclic_collection_inside_a_capture(fake_graph):
    from v2a_hip import ops
    log = []
    gc.collect()
    _Noted(log, fake_graph)                  # a dropped cycle: the collector's to free
    with ops.capture_graph("g", pool=3):
        keep = _allocate()
        assert log == []
        with ops.capture_graph("h"):         # two captures at once (two threads): the first end does not let the collector back in
            pass
        assert not gc.isenabled()
    assert gc.isenabled() and fake_graph["kw"] == [("g", {"pool": 3}), ("h", {})]
    gc.collect()
    assert log == [0] and len(keep) == 200000


def test_a_capture_that_fails_lets_the_collector_go_on(fake_graph):
    from v2a_hip import ops
    with pytest.raises(ZeroDivisionError):
        with ops.capture_graph("g"):
            1 / 0
    assert gc.isenabled()
    gc.disable()
    try:
        with ops.capture_graph("g"):
            pass
        assert not gc.isenabled()            # the caller's own setting stays
    finally:
        gc.enable()


def test_every_capture_of_the_framework_goes_through_it(trainer, fake_graph, monkeypatch):
    """The trainer's graphs, with the step's pieces and the device replaced by notes of whether the collector was held off."""
    held = []
    tr = trainer(presum=True)
    note = lambda *a, **k: held.append((fake_graph["capturing"], gc.isenabled()))
    for name in ("_fwd_bwd", "_bwd_encoders", "_opt", "_draw_indices"):
        monkeypatch.setattr(tr, name, note)

    class Graph:
        def replay(self):
            note()
    monkeypatch.setattr(torch.cuda, "CUDAGraph", Graph)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    tr._warm = 2
    tr.step()
    assert held == [(0, True), (1, False), (1, False), (1, False), (0, True)]
    import os
    import re
    from v2a_hip import ops
    root = os.path.dirname(os.path.dirname(os.path.abspath(ops.__file__)))
    direct = []
    for d, _, files in os.walk(root):
        for f in files:
            if f.endswith(".py"):
                with open(os.path.join(d, f)) as fh:
                    direct += [f"{f}: {ln.strip()}" for ln in fh if re.search(r"with torch\.cuda\.graph\(", ln)]
    assert direct == ["ops.py: with torch.cuda.graph(graph, **kw):"]
