"""The device-resident decode loop (plan, windowed attention, sampling in one graph) and the engine's use of
the same operators."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _cfg(**kw):
    from r9700_stack_b200.models.config import tiny_hybrid

    return tiny_hybrid(**{**dict(attn_window=96, attn_sinks=4), **kw})


def _prompt(n, vocab, seed=5):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("sinks", [0, 70])
def test_windowed_model_matches_reference(graphs, sinks):
    from r9700_stack_b200.engine.llm import LLM
    from r9700_stack_b200.engine.scheduler import SamplingParams
    from r9700_stack_b200.models.config import EngineConfig
    from r9700_stack_b200.models.reference import ReferenceState, reference_forward
    from r9700_stack_b200.utils import status

    cfg = _cfg(gdn_state_dtype="fp32", attn_sinks=sinks)
    llm = LLM(cfg, EngineConfig(max_batch=2, max_model_len=512, max_prefill_tokens=256, cuda_graphs=graphs,
                                graph_batch_sizes=[1, 2]), seed=3)
    prompt = _prompt(210, cfg.vocab)
    seq = llm.add_request(prompt, SamplingParams(max_tokens=5))
    st = ReferenceState(llm.model)
    cos = lambda a, b: float(torch.nn.functional.cosine_similarity(a.double().flatten(), b.double().flatten(), dim=0))
    llm.step()
    ref = reference_forward(llm.model, prompt, st)[-1]
    assert cos(llm.runner.ws.logits[0], ref) > 0.995
    for _ in range(4):
        llm.step()
        torch.cuda.synchronize()
        status.check()
        ref = reference_forward(llm.model, [seq.output[-2]], st)[-1]
        assert cos(llm.runner.ws.logits[0], ref) > 0.99


def test_loop_gives_the_engines_tokens():
    """One greedy request: the same kernels on the same shapes, so the same tokens; far past the window."""
    from r9700_stack_b200.engine.device_loop import DeviceLoop
    from r9700_stack_b200.engine.llm import LLM
    from r9700_stack_b200.engine.scheduler import SamplingParams
    from r9700_stack_b200.models.config import EngineConfig
    from r9700_stack_b200.models.hybrid import HybridLM
    from r9700_stack_b200.utils import status

    cfg = _cfg()
    prompt = _prompt(150, cfg.vocab)
    llm = LLM(cfg, EngineConfig(max_batch=1, max_model_len=1024, max_prefill_tokens=100, graph_batch_sizes=[1]), seed=7)
    want = llm.generate([prompt], SamplingParams(max_tokens=300))[0]
    loop = DeviceLoop(HybridLM(cfg, device="cuda", seed=7), 1, 1024, max_prefill_tokens=100)
    got = loop.prefill([prompt])
    for n in (1, 140, 158):
        toks, lp = loop.decode(n)
        got += toks[:, 0].tolist()
        assert bool((lp == 0).all())
    torch.cuda.synchronize()
    status.check()
    assert got == want
    # 449 tokens passed through a pool that holds fewer
    assert loop.pages.ring.numel() * 64 < 449 + 64 and int(loop.pages.state[1]) > 0
    assert loop.pages.ctx_len.tolist() == [449]


def test_loop_past_the_length_the_model_was_built_for():
    """The rotary table ends within the prompt; the loop grows it, and a loop captured before keeps its own."""
    from r9700_stack_b200.engine.device_loop import DeviceLoop
    from r9700_stack_b200.models.hybrid import HybridLM

    cfg = _cfg()
    prompt = _prompt(150, cfg.vocab)
    runs = []
    for rows in (65536, 100):
        model = HybridLM(cfg, device="cuda", seed=7)
        model._rope_cache(rows)
        loop = DeviceLoop(model, 1, 600, max_prefill_tokens=64)
        runs.append(loop.prefill([prompt]) + loop.decode(20)[0][:, 0].tolist())
        model.ensure_positions(100000)
        runs[-1] += loop.decode(100)[0][:, 0].tolist()
    assert runs[0] == runs[1]


def test_loops_and_an_engine_share_a_model():
    """Taking turns on one model's weights, each gives the tokens that it gives alone."""
    from r9700_stack_b200.engine.device_loop import DeviceLoop
    from r9700_stack_b200.engine.llm import LLM
    from r9700_stack_b200.engine.scheduler import SamplingParams
    from r9700_stack_b200.models.config import EngineConfig
    from r9700_stack_b200.models.hybrid import HybridLM
    from r9700_stack_b200.utils import status

    cfg = _cfg()
    prompts = [_prompt(n, cfg.vocab, n) for n in (150, 40, 70)]
    loop = lambda m, i: DeviceLoop(m, 1 + i, 600 - 100 * i, max_prefill_tokens=64)  # noqa: E731
    engine = lambda m: LLM(cfg, EngineConfig(max_batch=2, max_model_len=300, max_prefill_tokens=64, graph_batch_sizes=[1, 2]), model=m)  # noqa: E731
    alone = []
    for i in range(2):
        lp = loop(HybridLM(cfg, device="cuda", seed=7), i)
        alone.append([lp.prefill(prompts[: 1 + i])] + lp.decode(60)[0].tolist())
    alone.append(engine(HybridLM(cfg, device="cuda", seed=7)).generate([prompts[2]], SamplingParams(max_tokens=60))[0])
    model = HybridLM(cfg, device="cuda", seed=7)
    loops = [loop(model, 0)]
    got = [[loops[0].prefill(prompts[:1])] + loops[0].decode(10)[0].tolist()]
    eng = engine(model)
    req = eng.add_request(prompts[2], SamplingParams(max_tokens=60))
    for _ in range(12):
        eng.step()
    loops.append(loop(model, 1))
    got.append([loops[1].prefill(prompts[:2])])
    for _ in range(5):
        for lp, out in zip(loops, got):
            out += lp.decode(10)[0].tolist()
        for _ in range(10):
            eng.step()
    got[1] += loops[1].decode(10)[0].tolist()
    while eng.has_unfinished():
        eng.step()
    torch.cuda.synchronize()
    status.check()
    assert got[0] == alone[0] and got[1] == alone[1] and req.output == alone[2]


def test_loop_samples_and_repeats():
    from r9700_stack_b200.engine.device_loop import DeviceLoop
    from r9700_stack_b200.engine.scheduler import SamplingParams
    from r9700_stack_b200.models.hybrid import HybridLM

    cfg = _cfg()
    prompts = [_prompt(n, cfg.vocab, n) for n in (40, 130, 7)]
    params = [SamplingParams(temperature=0.9, top_k=20, top_p=0.95, seed=1), SamplingParams(),
              SamplingParams(temperature=1.2, min_p=0.05, seed=2)]
    runs = []
    for _ in range(2):
        loop = DeviceLoop(HybridLM(cfg, device="cuda", seed=7), 3, 512, max_prefill_tokens=64)
        first = loop.prefill(prompts, params)
        toks, lp = loop.decode(60)
        runs.append((first, toks.tolist(), lp.tolist()))
        assert bool((toks >= 0).all() and (toks < cfg.vocab).all() and (lp <= 0).all())
        assert bool((lp[:, 1] == 0).all()) and bool((lp[:, 0] < 0).any())
    assert runs[0] == runs[1]


def test_loop_refusals():
    from r9700_stack_b200.engine.device_loop import DeviceLoop
    from r9700_stack_b200.models.hybrid import HybridLM

    cfg = _cfg()
    model = HybridLM(cfg, device="cuda", seed=7)
    for bad in ((0, 64, 8), (1, 1, 8), (1, 64, 0)):
        with pytest.raises(ValueError):
            DeviceLoop(model, *bad)
    with pytest.raises(ValueError):
        DeviceLoop(object(), 1, 64, 8)
    loop = DeviceLoop(model, 2, 64, 16)
    with pytest.raises(RuntimeError):
        loop.decode(1)
    for bad in ([[1]], [[1], []], [[1], [1] * 64]):
        with pytest.raises(ValueError):
            loop.prefill(bad)
    loop.prefill([[1, 2], [3]])
    for bad in (0, 63):
        with pytest.raises(ValueError):
            loop.decode(bad)
    with pytest.raises(RuntimeError):
        loop.prefill([[1, 2], [3]])
    with pytest.raises(ValueError):
        HybridLM(_cfg(qsa_topk=4), device="cuda")


def _agree(a, b):
    """Length of the common prefix: other shapes add in other orders, so a rare near-tie may flip."""
    return next((i for i, (x, y) in enumerate(zip(a, b)) if x != y), min(len(a), len(b)))


@pytest.mark.parametrize("kind", ["moe", "heads of 128", "no window"])
def test_loop_on_other_models(kind):
    """One greedy request at a time, far past the window: the engine's kernels on the engine's shapes, so its tokens."""
    from r9700_stack_b200.engine.device_loop import DeviceLoop
    from r9700_stack_b200.engine.llm import LLM, build_model
    from r9700_stack_b200.engine.scheduler import SamplingParams
    from r9700_stack_b200.models.config import EngineConfig, ParallelConfig, tiny_moe
    from r9700_stack_b200.utils import status

    cfg = {"moe": tiny_moe(attn_window=50, attn_sinks=4), "heads of 128": _cfg(head_dim=128, attn_window=70),
           "no window": _cfg(attn_window=0, attn_sinks=0)}[kind]
    model = build_model(cfg, ParallelConfig(), torch.device("cuda"), seed=7)
    for prompt in (_prompt(90, cfg.vocab), _prompt(33, cfg.vocab, 6)):
        llm = LLM(cfg, EngineConfig(max_batch=1, max_model_len=512, max_prefill_tokens=64, graph_batch_sizes=[1]), model=model)
        want = llm.generate([prompt], SamplingParams(max_tokens=100))[0]
        loop = DeviceLoop(model, 1, 512, max_prefill_tokens=64)
        got = loop.prefill([prompt]) + loop.decode(99)[0][:, 0].tolist()
        torch.cuda.synchronize()
        status.check()
        assert got == want


@pytest.mark.parametrize("method", ["ngram", "mtp", "block", "dspark"])
def test_windowed_model_with_speculation(method):
    """Verification of drafts under a window that most of the sequence has left, captured graphs and ragged steps."""
    from r9700_stack_b200.engine.llm import LLM
    from r9700_stack_b200.engine.scheduler import SamplingParams
    from r9700_stack_b200.models.config import EngineConfig
    from r9700_stack_b200.utils import status

    cfg = _cfg(gdn_state_dtype="fp32", attn_window=40)
    prompts = [_prompt(n, cfg.vocab, n) for n in (37, 80, 12)]
    run = lambda **kw: LLM(cfg, EngineConfig(max_batch=3, max_model_len=256, max_prefill_tokens=64,  # noqa: E731
                                             graph_batch_sizes=[1, 2, 4], **kw), seed=7)
    want = run().generate(prompts, SamplingParams(max_tokens=20))
    llm = run(spec_tokens=3, spec_method=method)
    got = llm.generate(prompts, SamplingParams(max_tokens=20))
    torch.cuda.synchronize()
    status.check()
    for a, b in zip(got, want):
        assert len(a) == 20 and _agree(a, b) >= 16, (a, b)
    assert llm.spec_stats["steps"] > 0


def test_windowed_model_on_scripted_drafts():
    """Right and wrong drafts: rejected tokens leave no trace in what the window sees later."""
    from r9700_stack_b200.engine.llm import LLM
    from r9700_stack_b200.engine.scheduler import SamplingParams
    from r9700_stack_b200.models.config import EngineConfig
    from r9700_stack_b200.spec.drafters import ScriptedDrafter
    from r9700_stack_b200.utils import status

    cfg = _cfg(gdn_state_dtype="fp32", attn_window=40)
    prompts = [_prompt(n, cfg.vocab, n) for n in (37, 80, 12)]
    ec = dict(max_batch=3, max_model_len=256, max_prefill_tokens=64, graph_batch_sizes=[1, 2, 4])
    want = LLM(cfg, EngineConfig(**ec), seed=7).generate(prompts, SamplingParams(max_tokens=60))
    drafter = ScriptedDrafter(4, {}, pad=0, corrupt_every=3)
    llm = LLM(cfg, EngineConfig(spec_tokens=4, **ec), seed=7, drafter=drafter)
    seqs = [llm.add_request(p, SamplingParams(max_tokens=60)) for p in prompts]
    for s, ref in zip(seqs, want):
        drafter.script[s.seq_id] = ref
    while llm.has_unfinished():
        llm.step()
    torch.cuda.synchronize()
    status.check()
    for s, ref in zip(seqs, want):
        assert _agree(s.output, ref) >= 16, (s.output, ref)
    assert 0 < llm.spec_stats["accepted"] < llm.spec_stats["drafted"]


def test_engine_device_sampling():
    from r9700_stack_b200.engine.llm import LLM
    from r9700_stack_b200.engine.scheduler import SamplingParams
    from r9700_stack_b200.models.config import EngineConfig, tiny_hybrid

    cfg = tiny_hybrid()
    ec = EngineConfig(max_batch=4, max_model_len=256, max_prefill_tokens=128, graph_batch_sizes=[1, 2, 4],
                      device_sampling=True)
    prompts = [_prompt(20, cfg.vocab, s) for s in range(3)]
    outs = []
    for _ in range(2):
        llm = LLM(cfg, ec, seed=1)
        llm.runner.logit_log = []
        seqs = [llm.add_request(p, SamplingParams(max_tokens=12, temperature=t, top_k=5, min_p=0.01, seed=9))
                for p, t in zip(prompts, (0.8, 0.0, 1.5))]
        while llm.has_unfinished():
            llm.step()
        outs.append([s.output for s in seqs])
        for s in seqs:
            rows = [x for i, x in llm.runner.logit_log if i == s.seq_id]
            for x, t in zip(rows, s.output):
                assert t in torch.topk(x, 5).indices.tolist()
                assert s.params.temperature > 0 or t == int(x.argmax())
    assert outs[0] == outs[1]
