"""Engines and loops that share one model's weights: each runs on the caches that it allocated, and they live as long
as it does (its captured graphs hold their addresses)."""
import types

import pytest
import torch

from r9700_stack_b200.engine import device_loop
from r9700_stack_b200.engine.llm import LLM
from r9700_stack_b200.engine.scheduler import SamplingParams
from r9700_stack_b200.models.config import EngineConfig, tiny_hybrid
from r9700_stack_b200.models.dsv4 import DSV4LM, tiny_dsv4
from r9700_stack_b200.models.hybrid import HybridLM, NoComm
from r9700_stack_b200.models.mla_moe import MLAMoELM, tiny_mla


class Ran(Exception):
    pass


class Model(HybridLM):
    def __init__(self):
        self.cfg, self.device, self.comm = tiny_hybrid(attn_window=96, attn_sinks=4), torch.device("cpu"), NoComm()
        self.attn_dims, self.gdn_dims = dict(hkv=2), dict(hv=2, conv_ch=6)
        self._rope_cache(1024)

    def alloc_workspace(self, *a):
        return types.SimpleNamespace()

    def forward(self, *a):
        raise Ran


def _ids(caches):
    return {n: {i: [id(t) for t in (v if isinstance(v, tuple) else (v,))] for i, v in d.items()} for n, d in caches.items()
            if isinstance(d, dict)}


def _now(m):
    return _ids({n: getattr(m, n) for n in m.CACHES})


class _Pages:
    def __init__(self, *a):
        self.block_table = torch.zeros(1, 1)

    def plan(self, *a, **kw):
        return types.SimpleNamespace(**{n: torch.zeros(1) for n in ("positions", "slots", "tok_seq", "tok_ctx", "seq_start", "seq_len")})


def test_a_loop_runs_on_its_own_caches(monkeypatch):
    monkeypatch.setattr(device_loop, "PagedState", _Pages)
    m = Model()
    a = device_loop.DeviceLoop(m, 1, 200, 64)
    first = _now(m)
    assert any(first["kv"].values()) and any(first["ssm"].values())
    b = device_loop.DeviceLoop(m, 3, 900, 64)
    assert _now(m) != first
    for loop in (a, b, a):
        loop.ctx = []
        with pytest.raises(Ran):
            loop.prefill([[1, 2]] * loop.seqs, [SamplingParams()] * loop.seqs)
        assert (_now(m) == first) == (loop is a)
    with pytest.raises(Ran):
        b.prefill([[1]] * 3)
    a.ctx, a.seeds, a.params, a.drawn = [2], [0], (), 1
    with pytest.raises(Ran):
        a.decode(2)
    assert _now(m) == first


def test_an_engine_runs_on_its_own_caches(monkeypatch):
    from r9700_stack_b200.engine import llm as module

    class Runner:
        def __init__(self, *a):
            self.ws = None

        def execute(self, out):
            raise Ran

    monkeypatch.setattr(module, "ModelRunner", Runner)
    m = Model()
    ec = EngineConfig(max_batch=1, max_model_len=128, max_prefill_tokens=64, cuda_graphs=False)
    a = LLM(m.cfg, ec, model=m, device="cpu")
    first = _now(m)
    b = LLM(m.cfg, EngineConfig(max_batch=4, max_model_len=500, max_prefill_tokens=64, cuda_graphs=False), model=m, device="cpu")
    for e in (a, b, a):
        e.add_request([1, 2], SamplingParams(max_tokens=2))
        with pytest.raises(Ran):
            e.step()
        assert (_now(m) == first) == (e is a)


@pytest.mark.parametrize("cls,cfg", [(MLAMoELM, tiny_mla), (DSV4LM, tiny_dsv4)])
def test_every_family_names_all_its_caches(cls, cfg):
    m = object.__new__(cls)
    m.cfg, m.device = cfg(), torch.device("cpu")
    before = set(m.__dict__)
    m.alloc_caches(3, 2, 64)
    assert set(m.__dict__) - before == set(m.CACHES)
    held = m.held_caches()
    m.alloc_caches(5, 2, 64)
    assert all(getattr(m, n) is not held[n] for n in m.CACHES)
    m.use_caches(held)
    assert all(getattr(m, n) is held[n] for n in m.CACHES)


def test_the_hybrid_family_names_all_its_caches():
    m = Model()
    before = set(m.__dict__)
    m.alloc_caches(3, 2)
    assert set(m.__dict__) - before == set(m.CACHES)
