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
