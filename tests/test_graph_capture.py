"""A sampler's plan and a user's own graphs side by side.

torch keeps one pair of RNG tensors for all live graphs of a device and makes it with the first of them; made inside
inference_mode it refuses every capture outside that mode for as long as one of those graphs lives."""
import contextlib

import pytest
import torch

import echo_tts_amd as E
from echo_tts_amd import engine, ops


def test_plan_registers_outside_inference_mode(monkeypatch):
    """Without a device: the plan's graph meets the generator outside inference mode and before its capture, which runs in
    the caller's mode."""
    seen = []

    class Graph:
        def register_generator_state(self, generator):
            seen.append(("register", generator, torch.is_inference_mode_enabled()))

        def replay(self):
            seen.append(("replay",))

    @contextlib.contextmanager
    def graph(g):
        seen.append(("capture", type(g), torch.is_inference_mode_enabled()))
        yield

    monkeypatch.setattr(torch.cuda, "CUDAGraph", Graph)
    monkeypatch.setattr(torch.cuda, "graph", graph)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    monkeypatch.setattr(torch.cuda, "default_generators", ("gen0", "gen1"))
    plan = engine.CFGPlan.__new__(engine.CFGPlan)
    plan.graph, plan.runs, plan.sync, plan.x = None, 0, None, torch.zeros(1)
    plan.loop = lambda: seen.append(("loop", torch.is_inference_mode_enabled()))
    with torch.inference_mode():
        plan.run(True)
        plan.run(True)
    assert seen == [("loop", True), ("register", "gen1", False), ("capture", Graph, True), ("loop", True), ("replay",)]


@pytest.fixture(scope="module")
def sampler():
    """A call of the public sampler that runs as a captured plan (its second call on replays it)."""
    from conftest import load_golden
    from echo_tts_amd import weights as W
    from echo_tts_amd.inference import sample_with_noise
    from echo_tts_amd.model import EchoDiTHip
    cfg = E.tiny()
    m = EchoDiTHip(cfg, W.synthetic_state_dict(cfg, dtype=torch.bfloat16), device="cuda", dtype=torch.bfloat16)
    g = {k: v.to("cuda") for k, v in load_golden("tiny_bf16").items()}

    def call(**kw):
        return sample_with_noise(m, g["speaker_latent"], g["speaker_mask"], g["text_ids"], g["text_mask"], g["caseA.noise"],
                                 **{**dict(num_steps=4, cfg_scale_text=3.0, cfg_scale_speaker=8.0, cfg_min_t=0.5, cfg_max_t=1.0,
                                           use_graph=True), **kw})
    return m, call


def replays(seeds=(1, 2, 3)):
    """Capture an operator in the caller's mode, and compare replays on new inputs with eager calls."""
    x = torch.randn(33, 256, device="cuda")
    ops.quantize_fp8(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q, s = ops.quantize_fp8(x)
    for seed in seeds:
        torch.manual_seed(seed)
        x.copy_(torch.randn(33, 256, device="cuda"))
        g.replay()
        want = ops.quantize_fp8(x)
        assert torch.equal(q.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(s.view(torch.uint8), want[1].view(torch.uint8))
    return g


@pytest.mark.gpu
def test_capture_beside_a_live_plan(sampler):
    m, call = sampler
    first, again = call(), call()
    assert any(p.graph is not None for p in m.__dict__["_plans"].values()) and torch.equal(first, again)
    g = replays()
    assert torch.equal(call(), first)
    with torch.inference_mode():
        replays()
    del g
    assert torch.equal(call(), first)


@pytest.mark.gpu
def test_plan_beside_a_graph_of_inference_mode(sampler):
    """A user's graph captured inside the mode, with no other alive, makes the pair an inference one: the plan's capture
    still goes through, as it runs in the mode itself."""
    m, call = sampler
    m.__dict__["_plans"].clear()
    with torch.inference_mode():
        g = replays()
    first = call(num_steps=3)
    assert torch.equal(call(num_steps=3), first)
    del g
