"""Sequences longer than the rotary table that a model is built with: everything that runs a model up to some length
has the table cover it first (the kernels read it by position, without a bound)."""
import pytest
import torch

from r9700_stack_b200.engine.device_loop import DeviceLoop
from r9700_stack_b200.engine.llm import LLM
from r9700_stack_b200.models.config import EngineConfig, tiny_hybrid
from r9700_stack_b200.models.hybrid import HybridLM, NoComm
from r9700_stack_b200.models.mla_moe import MLAMoELM


class Enough(Exception):
    """The caches are the next thing a user of the model asks for."""


def _model(rows):
    class Model(HybridLM):
        def __init__(self):
            self.cfg, self.device, self.comm = tiny_hybrid(attn_window=96, attn_sinks=4), torch.device("cpu"), NoComm()
            self._rope_cache(rows)

        def alloc_caches(self, *a, **kw):
            raise Enough

    return Model()


def test_the_table_grows_and_the_old_one_stays():
    m = _model(100)
    old, values = m.cos_sin, m.cos_sin.clone()
    m.ensure_positions(100)
    assert m.cos_sin is old
    m.ensure_positions(1000)
    assert m.cos_sin.shape[0] >= 1000 and torch.equal(m.cos_sin[:100], values)
    # a graph captured before goes on reading where the old table is
    assert any(t is old for t in m.outgrown) and torch.equal(old, values)
    c = m.cfg
    inv = 1.0 / (c.rope_theta ** (torch.arange(0, c.rotary_dim, 2, dtype=torch.float64) / c.rotary_dim))
    want = torch.cat([torch.cos(999 * inv), torch.sin(999 * inv)]).float()
    assert torch.equal(m.cos_sin[999], want)


@pytest.mark.parametrize("max_len", [64, 1000, 5000])
def test_the_loop_and_the_engine_cover_their_lengths(max_len):
    m = _model(200)
    with pytest.raises(Enough):
        DeviceLoop(m, 1, max_len, 64)
    assert m.cos_sin.shape[0] >= max_len
    m = _model(200)
    with pytest.raises(Enough):
        LLM(m.cfg, EngineConfig(max_model_len=max_len), model=m, device="cpu")
    assert m.cos_sin.shape[0] >= max_len + 64  # drafts may reach this far past the last token


def test_a_drafter_covers_its_lengths(monkeypatch):
    from r9700_stack_b200.spec import draft_model, drafters

    m = _model(200)
    monkeypatch.setattr(draft_model, "build_draft_model", lambda *a, **kw: m)
    with pytest.raises(Enough):
        drafters.ModelDrafter(m, "mtp", 3, EngineConfig(max_model_len=900), 10, 2)
    assert m.cos_sin.shape[0] >= 964


def test_a_model_of_fixed_length_refuses_more():
    m = object.__new__(MLAMoELM)
    m.max_ctx, m.cos_sin = 512, torch.zeros(576, 64)
    m.ensure_positions(576)
    with pytest.raises(ValueError, match="512"):
        m.ensure_positions(577)
    with pytest.raises(ValueError):
        LLM(None, EngineConfig(max_model_len=513), model=m, device="cpu")
