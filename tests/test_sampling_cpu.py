"""Host side of the device sampling and the step plan: the uniform numbers, min-p on the host sampler, the
sampling restatement on CPU tensors, launcher options."""
import pytest
import torch

from r9700_stack_b200.engine.sampler import device_params, sample_rows, uniform
from r9700_stack_b200.engine.scheduler import SamplingParams
from r9700_stack_b200.ops.sampling import sample_ref


def test_uniform_is_reproducible_and_spread():
    x = [uniform(seed, step) for seed in range(40) for step in range(100)]
    assert x == [uniform(seed, step) for seed in range(40) for step in range(100)]
    assert all(0.0 <= v < 1.0 for v in x) and len(set(x)) > 3990
    # 4000 draws: mean within 5 standard deviations (0.2887 / sqrt(4000) = 0.0046), ten bins within 5 of 20
    assert abs(sum(x) / len(x) - 0.5) < 0.023
    bins = [sum(1 for v in x if int(v * 10) == b) for b in range(10)]
    assert all(abs(b - 400) < 100 for b in bins)
    assert uniform(-1, 0) != uniform(1, 0) and uniform(2**70 + 3, 1) == uniform(2**70 % 2**64 + 3, 1)


def test_min_p_on_the_host_sampler():
    x = torch.log(torch.tensor([[0.5, 0.3, 0.15, 0.05]]))
    for step in range(40):
        t = sample_rows(x, [SamplingParams(temperature=1.0, min_p=0.4, seed=3)], [step])[0]
        assert t in (0, 1)
    assert sample_rows(x, [SamplingParams(temperature=1.0, min_p=1.0)], [0]) == [0]


def test_device_params():
    t, k, p, m = device_params([SamplingParams(), SamplingParams(temperature=0.5, top_k=7, top_p=0.9, min_p=0.1)], "cpu")
    assert t.tolist() == [0.0, 0.5] and k.dtype == torch.int32 and k.tolist() == [0, 7]
    assert p.dtype == torch.float32 and abs(float(m[1]) - 0.1) < 1e-7


def test_device_params_take_any_top_k():
    """A number past int32 keeps everything, as in the host sampler; it must not end the step that all requests share."""
    ks = [2**40, -2**40, 2**31, 2**31 - 1, -1, 0, None, 7]
    _, k, _, _ = device_params([SamplingParams(temperature=1.0, top_k=v) for v in ks], "cpu")
    assert k.dtype == torch.int32 and k.tolist() == [0, 0, 0, 2**31 - 1, 0, 0, 0, 7]
    x = torch.log(torch.tensor([[0.5, 0.3, 0.15, 0.05]])).expand(len(ks), 4)
    params = [SamplingParams(temperature=1.0, top_k=v, seed=1) for v in ks]
    assert len(sample_rows(x, params, [0] * len(ks))) == len(ks)


def test_sample_ref_on_cpu():
    f = lambda v: torch.tensor(v, dtype=torch.float32)
    x = torch.log(torch.tensor([[0.1, 0.4, 0.2, 0.3]])).expand(5, 4)
    one = f([1.0] * 5)
    u = f([0.0, 0.09, 0.11, 0.49, 0.99])
    assert sample_ref(x, u, one)[0].tolist() == [0, 0, 1, 1, 3]
    k = torch.tensor([1, 2, 2, 2, 3], dtype=torch.int32)
    assert sample_ref(x, u, one, k)[0].tolist() == [1, 1, 1, 1, 3]
    assert sample_ref(x, u, one, None, f([0.3] * 5))[0].tolist() == [1] * 5
    tok, lp = sample_ref(x, u, one, None, None, f([0.7] * 5))
    assert tok.tolist() == [1, 1, 1, 1, 3] and abs(float(lp[4]) - float(torch.log(torch.tensor(3 / 7)))) < 1e-6
    tok, lp = sample_ref(torch.full((2, 3), float("-inf")), u[:2], one[:2])
    assert tok.tolist() == [-1, -1] and lp.tolist() == [float("-inf")] * 2
    tok, lp = sample_ref(x[:1], u[:1], f([0.0]))
    assert tok.tolist() == [1] and lp.tolist() == [0.0]


def test_launcher_window_options():
    from r9700_stack_b200.serve import launch

    a = launch.parse(["--model", "tiny-hybrid", "--attn-window", "128", "--attn-sinks", "4", "--device-sampling"])
    assert launch.plan(a) is not None
    from r9700_stack_b200.models.config import model_config

    c = launch.windowed(model_config("tiny-hybrid"), a)
    assert (c.attn_window, c.attn_sinks) == (128, 4)
    a = launch.parse(["--model", "tiny-hybrid", "--attn-sinks", "4"])
    with pytest.raises(SystemExit):
        launch.windowed(model_config("tiny-hybrid"), a)
    a = launch.parse(["--model", "tiny-mla", "--attn-window", "64"])
    with pytest.raises(SystemExit):
        launch.windowed(model_config("tiny-mla"), a)
