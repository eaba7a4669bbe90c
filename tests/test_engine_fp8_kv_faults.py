"""Rollout engine on the 8-bit KV cache where something goes wrong or changes under it: waits of the decode attention that gave
up, weights that change while cached prefixes exist."""

import asyncio

import pytest
import torch

from axrl_b200.ops import paged_fp8

CUDA = pytest.param("cuda", marks=pytest.mark.gpu)


def _model(dev, seed=0):
    from axrl_b200.models.qwen3 import Qwen3Config, Qwen3Model

    cfg = Qwen3Config(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                      head_dim=128)
    m = Qwen3Model(cfg)
    m.init_weights(seed)
    m = m.to(dev, torch.bfloat16 if dev == "cuda" else torch.float32)
    m.inv_freq = m.inv_freq.float()
    return m


def _engine(m, dev, **kw):
    from axrl_b200.rollout.engine import RolloutEngine

    args = dict(max_batch=8, kv_tokens=4096, max_context=512, page_size=16, seed=3, burst=8, kv_format="fp8_block", use_cuda_graph=dev == "cuda") | kw
    return RolloutEngine(m, **args)


def _greedy(rid, prompt, n=12, **kw):
    from axrl_b200.rollout.engine import GenRequest

    return GenRequest(rid=rid, prompt=prompt, max_new_tokens=n, temperature=0.0, seed_stream=1, **kw)


def _prompt(n, seed=0):
    return torch.randint(1, 512, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("dev", ["cpu", CUDA])
def test_a_decode_wait_that_gave_up_ends_generation(dev, monkeypatch):
    """No token of the burst is used; the bf16 engine does not ask."""
    m = _model(dev)
    eng = _engine(m, dev)
    assert len(eng.generate([_greedy("a", _prompt(20))])[0].output_ids) == 12
    assert paged_fp8.decode_wait_error(torch.device(dev)) == 0
    monkeypatch.setattr(paged_fp8, "decode_wait_error", lambda device: 1)
    eng.add_requests([_greedy("b", _prompt(20))])
    with pytest.raises(RuntimeError, match="wait"):
        eng.step()
    assert len(eng.running) == 1 and len(eng.running[0].out_ids) == 1  # the prefill's
    assert len(_engine(m, dev, kv_format="bf16").generate([_greedy("c", _prompt(20))])[0].output_ids) == 12


def test_calls_of_a_worker_fail_when_a_decode_wait_gave_up(monkeypatch):
    import numpy as np

    from axrl_b200.configs import SamplingConfig
    from axrl_b200.data.conversation import GenerationInput
    from axrl_b200.worker.rollout_worker import RolloutWorker

    monkeypatch.setattr(paged_fp8, "decode_wait_error", lambda device: 1)
    worker = RolloutWorker(_engine(_model("cpu"), "cpu"), SamplingConfig())
    try:
        inp = GenerationInput(session_id="s", input_ids=np.asarray(_prompt(20)), sampling_config=SamplingConfig(max_new_tokens=5))
        with pytest.raises(RuntimeError, match="rollout engine failed"):
            asyncio.run(asyncio.wait_for(worker.generate(inp), 60))
    finally:
        worker.shutdown()


# ----------------------------------------------------------------------------- weights that change
def test_a_prefill_that_a_reset_overtakes_registers_nothing():
    """The reset comes from another thread while the engine's is inside the forward pass: its rows are of the weights before."""
    m = _model("cpu")
    eng = _engine(m, "cpu")
    p = _prompt(50)
    assert eng.generate([_greedy("a", p)])[0].cached_tokens == 0
    layers = eng._layers

    def interrupted(*a, **k):
        h = layers(*a, **k)
        eng.reset_prefix_cache()
        return h

    eng._layers = interrupted
    eng.generate([_greedy("b", p + _prompt(30, 1), n=1)])
    eng._layers = layers
    assert eng.bm.num_cached() == 0 and eng.bm.num_available() == eng.num_pages - 1
    assert eng.generate([_greedy("c", p)])[0].cached_tokens == 0
    assert eng.generate([_greedy("d", p)])[0].cached_tokens == 48
    eng.release_kv()
    assert eng.generate([_greedy("e", p)])[0].cached_tokens == 0


def test_weights_quantised_again_leave_no_cached_prefix():
    m = _model("cpu")
    eng = _engine(m, "cpu")
    p = _prompt(50)
    eng.generate([_greedy("a", p)])
    with torch.no_grad():
        for w in m.parameters():
            w.mul_(1.01)
    eng.quantize_weights()
    assert eng.bm.num_cached() == 0


def test_a_loaded_checkpoint_leaves_no_cached_prefix(monkeypatch, tmp_path):
    """The controller's engine runs on the trainer's weights: what was generated before they are loaded is of other weights."""
    from types import SimpleNamespace

    from axrl_b200.pipeline.controller import PipelineController
    from axrl_b200.train import checkpoint

    eng = _engine(_model("cpu"), "cpu")
    eng.generate([_greedy("a", _prompt(50))])
    assert eng.bm.num_cached() == 3
    monkeypatch.setattr(checkpoint, "latest_iteration", lambda root: 7)
    monkeypatch.setattr(checkpoint, "load_dist_checkpoint", lambda *a: {"iteration": 7})
    ctl = SimpleNamespace(checkpoint_root=lambda: tmp_path, train=SimpleNamespace(model=eng.model, optim=None), engine=eng, train_dataset=None)
    assert PipelineController.load_checkpoint_if_existed(ctl)
    assert ctl.global_step == 7 and eng.bm.num_cached() == 0
