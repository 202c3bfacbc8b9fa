"""Host side of the device loop: what it refuses before anything is launched."""
import types

import pytest
import torch

from r9700_stack_b200.engine import device_loop
from r9700_stack_b200.models.config import tiny_hybrid
from r9700_stack_b200.models.hybrid import HybridLM, NoComm


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


class _Pages:
    def __init__(self, *a):
        self.block_table = torch.zeros(1, 1)

    def plan(self, *a, **kw):
        return types.SimpleNamespace(**{n: torch.zeros(1) for n in ("positions", "slots", "tok_seq", "tok_ctx", "seq_start", "seq_len")})


@pytest.mark.parametrize("bad", [-1, 512, 2**31, 2**40])
def test_token_ids_outside_the_vocabulary_are_refused(monkeypatch, bad):
    """The embedding is gathered by these numbers on the device."""
    monkeypatch.setattr(device_loop, "PagedState", _Pages)
    loop = device_loop.DeviceLoop(Model(), 2, 200, 64)
    with pytest.raises(ValueError, match="vocabulary"):
        loop.prefill([[1, 2], [3, bad, 4]])
    with pytest.raises(Ran):
        loop.prefill([[0, 511], [3]])
