"""Rollout engine on the 8-bit KV cache: cached prefixes, shared and copied pages, preemption, decode against prefill."""

import dataclasses

import pytest
import torch

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


def _prompt(n, seed):
    return torch.randint(1, 512, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _greedy(rid, prompt, n=12, **kw):
    from axrl_b200.rollout.engine import GenRequest

    return GenRequest(rid=rid, prompt=prompt, max_new_tokens=n, temperature=0.0, seed_stream=1, **kw)


def _same(a, b, atol):
    """Greedy runs of the same computation.  Where logits differ by at most d, the largest one differs by at most d too, so the
    log-probs agree up to and at the first token that differs, and from there on the texts are not the same any more."""
    n = next((i for i, (x, y) in enumerate(zip(a.output_ids, b.output_ids)) if x != y), len(a.output_ids) - 1) + 1
    assert len(a.output_ids) == len(b.output_ids)
    torch.testing.assert_close(torch.tensor(a.output_logprobs[:n]), torch.tensor(b.output_logprobs[:n]), atol=atol, rtol=0)


# A product's rounding depends on the number of rows it is computed with, in the last bit on the CPU (fp32); a key next to the
# border between two codes then moves by a code, 2^-3 of it, and a score by 2^-3 |q_i k_i| / sqrt(128) < 0.02 of products below
# 2: fewer than one in 10^5 do.  On the GPU the products' order, and so the rounding, depends on the number of rows: logits of this model
# stay below 4 in size and are rounded to bf16, 2^-8 x 4 in each of two runs, and as much again from the hidden states.
ATOL = {"cpu": 0.02, "cuda": 4 * 2.0 ** -8 * 4}


@pytest.mark.parametrize("dev", ["cpu", CUDA])
@pytest.mark.parametrize("n,suffix", [(40, 7), (48, 1), (16, 30), (100, 16)])
def test_cached_prefix_gives_what_a_full_prefill_gives(dev, n, suffix):
    m = _model(dev)
    head = _prompt(n, 1)
    long = head + _prompt(suffix, 2)
    fresh = _engine(m, dev).generate([_greedy("a", long)])[0]
    assert fresh.cached_tokens == 0
    eng = _engine(m, dev)
    eng.generate([_greedy("h", head)])
    before = eng.stats["prefill_tokens"]
    again = eng.generate([_greedy("b", long)])[0]
    full = n // 16 * 16
    assert again.cached_tokens == full and eng.stats["prefill_tokens"] - before == len(long) - full
    _same(again, fresh, ATOL[dev])
    # the whole prompt cached: its last page is computed again (its logits are needed)
    third = eng.generate([_greedy("c", long)])[0]
    assert third.cached_tokens == (len(long) - 1) // 16 * 16
    _same(third, fresh, ATOL[dev])
    assert eng.bm.num_available() == eng.num_pages - 1
    # new weights: nothing cached may be used
    eng.update_weights_from_model(_model(dev, 1))
    other = eng.generate([_greedy("d", long)])[0]
    assert other.cached_tokens == 0
    _same(other, _engine(_model(dev, 1), dev).generate([_greedy("e", long)])[0], ATOL[dev])


@pytest.mark.parametrize("dev", ["cpu", CUDA])
def test_mixed_batch_of_cached_and_new_prompts(dev):
    m = _model(dev)
    head = _prompt(64, 5)
    prompts = [head + _prompt(9, 6), _prompt(21, 7), head[:32] + _prompt(3, 8), _prompt(1, 9), head]
    alone = [_engine(m, dev).generate([_greedy("x", p)])[0] for p in prompts]
    eng = _engine(m, dev)
    eng.generate([_greedy("h", head)])
    res = eng.generate([_greedy(f"r{i}", p) for i, p in enumerate(prompts)])
    assert [r.cached_tokens for r in res] == [64, 0, 32, 0, 48]
    for r, a in zip(res, alone):
        _same(r, a, ATOL[dev])


@pytest.mark.parametrize("dev", ["cpu", CUDA])
def test_group_members_share_and_copy_pages(dev):
    m = _model(dev)
    p = _prompt(37, 3)
    eng = _engine(m, dev)
    res = eng.generate([_greedy(f"g{i}", p, n=5 + 3 * i) for i in range(4)])
    ref = _engine(m, dev).generate([_greedy("one", p, n=14)])[0]
    for i, r in enumerate(res):
        n = 5 + 3 * i
        _same(r, dataclasses.replace(ref, output_ids=ref.output_ids[:n], output_logprobs=ref.output_logprobs[:n]), ATOL[dev])
    assert eng.bm.num_available() == eng.num_pages - 1


@pytest.mark.parametrize("dev", ["cpu", CUDA])
def test_preempted_sequences_resume_on_their_cached_prompt(dev):
    m = _model(dev)
    prompts = [_prompt(40, 20 + i) for i in range(4)]
    want = [_engine(m, dev).generate([_greedy("x", p, n=60)])[0] for p in prompts]
    eng = _engine(m, dev, kv_tokens=340)
    res = eng.generate([_greedy(f"r{i}", p, n=60) for i, p in enumerate(prompts)])
    assert eng.stats.get("preempted", 0) > 0
    for r, a in zip(res, want):
        _same(r, a, ATOL[dev])
    assert eng.bm.num_available() == eng.num_pages - 1


@pytest.mark.parametrize("dev", ["cpu", CUDA])
def test_close_to_the_bf16_cache(dev):
    """Log-probs of the same continuation on both cache formats: a row is off by at most 2^-4 of its values, so the
    scores and outputs move by a few percent, not in kind."""
    m = _model(dev)
    p = _prompt(90, 4)
    a = _engine(m, dev, kv_format="bf16").generate([_greedy("a", p, n=1)])[0]
    b = _engine(m, dev).generate([_greedy("b", p, n=1)])[0]
    assert abs(a.output_logprobs[0] - b.output_logprobs[0]) < 0.25


@pytest.mark.gpu
def test_graph_replay_matches_eager_and_memory_is_released():
    m = _model("cuda")
    reqs = lambda: [_greedy(f"r{i}", _prompt(30 + 11 * i, i), n=40) for i in range(6)]  # noqa: E731
    a = _engine(m, "cuda", page_size=64, kv_memory_saver=True)
    b = _engine(m, "cuda", page_size=64, use_cuda_graph=False)
    for x, y in zip(a.generate(reqs()), b.generate(reqs())):
        _same(x, y, ATOL["cuda"])
    first = a.generate(reqs())
    a.release_kv()
    free0 = torch.cuda.mem_get_info()[0]
    a.acquire_kv()
    assert torch.cuda.mem_get_info()[0] < free0
    for x, y in zip(a.generate(reqs()), first):
        _same(x, y, ATOL["cuda"])
    a.release_graphs()


def test_format_is_checked():
    from pydantic import ValidationError

    from axrl_b200.configs import RolloutWorkerConfig

    assert RolloutWorkerConfig(kv_cache_dtype="fp8_block").kv_cache_dtype == "fp8_block"
    with pytest.raises(ValidationError):
        RolloutWorkerConfig(kv_cache_dtype="fp8_e5m2")
    with pytest.raises(ValueError, match="kv_format"):
        _engine(_model("cpu"), "cpu", kv_format="int4")


@pytest.mark.gpu
def test_shapes_without_kernels_are_refused():
    m = _model("cuda")
    with pytest.raises(ValueError, match="fp8_block"):
        _engine(m, "cuda", page_size=24)
    with pytest.raises(ValueError, match="fp8_block"):
        _engine(m, "cuda", max_batch=4096)


def test_token_bytes():
    from axrl_b200.rollout.engine import kv_token_bytes

    cfg = _model("cpu").cfg
    codes, scales = _engine(_model("cpu"), "cpu").kv_fp8
    rows = codes.numel() // 128
    assert kv_token_bytes(cfg, "fp8_block") * (codes.shape[2] * codes.shape[4]) == codes.numel() + scales.numel() == rows * 129
    assert kv_token_bytes(cfg) == 2 * 2 * 2 * 128 * 2


def test_agentic_turns_continue_cached_prefixes():
    """Each turn of a trajectory begins with the context of the one before: on the 8-bit cache it prefills less."""
    from axrl_b200.configs import GrpoTrainerConfig, MegatronWorkerConfig
    from axrl_b200.models.qwen3 import resolve_preset
    from axrl_b200.pipeline.agentic_step import AgenticConfig, SyntheticAgentic

    done = {}
    for kv in ("bf16", "fp8_block"):
        torch.manual_seed(0)
        ac = AgenticConfig(group_size=2, inflight_groups=1, prefix_len=80, min_turns=3, max_turns=3, action_min=4, action_max=4, obs_min=70, obs_max=70,
                           max_context=400, pack_len=1024, seed=1, kv_format=kv, kv_gb=0.01)
        pipe = SyntheticAgentic(resolve_preset("tiny"), MegatronWorkerConfig(), GrpoTrainerConfig(loss_type="grpo"), ac, "cpu")
        m = pipe.run_step()
        assert m["trajectories"] == 2 and m["turns"] == 6
        done[kv] = pipe.rollout.stats["prefill_tokens"]
    assert done["fp8_block"] < done["bf16"]


@pytest.mark.gpu
def test_grpo_step_on_the_8_bit_cache():
    from axrl_b200.configs import GrpoTrainerConfig, MegatronWorkerConfig
    from axrl_b200.pipeline.grpo_step import SyntheticGRPO, SyntheticGRPOConfig

    wc = MegatronWorkerConfig()
    wc.lr_scheduler.lr_warmup_steps = 0
    sc = SyntheticGRPOConfig(num_prompts=2, prompt_len=64, group_size=4, max_new_tokens=24, reward_token=5, kv_format="fp8_block")
    g = SyntheticGRPO(_model("cpu").cfg, wc, GrpoTrainerConfig(loss_type="grpo"), sc, "cuda")
    for _ in range(2):
        m = g.run_step()
        assert m["trained_tokens"] > 0 and m["loss"] == m["loss"]
    g.rollout.release_graphs()
