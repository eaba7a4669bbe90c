"""Rollout engine on the 8-bit KV cache against a forward pass of its own, teacher-forced on the tokens that the engine gave: the log-probs
of prefilled, continued and decoded tokens.

The forward pass is plain torch in 64 bits, with K and V rounded as the cache holds them.  Its model makes attention matter: peaked
scores (norm weights of 1.6) and an output projection twenty times the usual.  Tolerance: what the same forward pass moves by when
every activation is rounded to bf16 (as on the GPU; products summed in 64 bits), times three: the kernels round in as many places, in
another order, so that the two errors are of one size but not alike, and the largest of a few dozen draws of one distribution stays within
three times another's.  Mistakes planted in the oracle (decoded tokens without attention, a prefix of zeros, another layer's rows, a
context that is a token short) must move some token of a batch by more than 1.5 times that."""

import pytest
import torch

from axrl_b200.ops import paged_fp8 as pf

CUDA = pytest.param("cuda", marks=pytest.mark.gpu)
NQ, NKV, D, H = 4, 2, 128, 256


def _model(dev):
    from axrl_b200.models.qwen3 import Qwen3Config, Qwen3Model

    cfg = Qwen3Config(vocab_size=512, hidden_size=H, intermediate_size=512, num_hidden_layers=2, num_attention_heads=NQ, num_key_value_heads=NKV,
                      head_dim=D)
    m = Qwen3Model(cfg)
    m.init_weights(4)
    with torch.no_grad():
        for name, p in m.named_parameters():
            if name.endswith("o_proj"):
                p.mul_(20)
            if name.endswith(("q_norm", "k_norm")):
                p.fill_(1.6)
            p.copy_(p.bfloat16())  # the same weights on both devices
    inv = m.inv_freq.clone()
    m = m.to(dev, torch.bfloat16 if dev == "cuda" else torch.float32)
    m.inv_freq = inv.float().to(dev)
    return m


def _oracle(m, ids, n, c0=0, rounded=False, plant=None):
    """log-softmax (64 bits) of the logits behind every token of `ids`; `n`: tokens of the prompt, `c0` of them from the cache."""
    r = (lambda x: x.bfloat16().double()) if rounded else (lambda x: x)
    W = lambda w: w.detach().cpu().double()  # noqa: E731
    eps = m.cfg.rms_norm_eps

    def rms(x, w):
        return r(x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * W(w))

    def held(x):  # as the cache holds it
        c, s = pf.quantize_rows_e8m0(x.float())
        return c.double() * s.float().double()[..., None]

    T = len(ids)
    pos = torch.arange(T)
    ang = pos.double()[:, None, None] * W(m.inv_freq)
    cos, sin = ang.cos(), ang.sin()

    def turned(x, w):
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * W(w)
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    seen = pos[None, :] <= pos[:, None]
    if plant == "short":
        seen &= (pos[:, None] < n) | (pos[None, :] < pos[:, None])
    h = W(m.embed_tokens)[torch.tensor(ids)]
    first = None
    for layer in m.layers:
        a = layer.self_attn
        x = rms(h, layer.input_layernorm.weight)
        q, k, v = r(x @ W(a.qkv_proj).t()).view(T, -1, D).split([NQ, NKV, NKV], 1)
        q, k, v = r(turned(q, a.q_norm)), held(turned(k, a.k_norm)), held(v)
        if plant == "layer" and first is not None:
            k, v = first
        first = (k, v)
        kk, vv = k.repeat_interleave(NQ // NKV, 1), v.repeat_interleave(NQ // NKV, 1)
        s = torch.einsum("qhd,khd->hqk", q, kk) * D ** -0.5
        if plant == "prefix":  # rows of zeros for what continues it
            s[:, c0:, :c0] = 0
        p = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
        if plant == "prefix":
            p[:, c0:, :c0] = 0
        o = torch.einsum("hqk,khd->qhd", p, vv).reshape(T, -1)
        if plant == "decode":
            o[n:] = 0
        h = r(h + r(o) @ W(a.o_proj).t())
        x = rms(h, layer.post_attention_layernorm.weight)
        g, u = r(x @ W(layer.mlp.gate_up_proj).t()).chunk(2, -1)
        h = r(h + r(torch.nn.functional.silu(g) * u) @ W(layer.mlp.down_proj).t())
    return torch.log_softmax(r(rms(h, m.norm.weight) @ W(m.lm_weight).t()), -1)


def _given(lp, ids, n):
    """Log-probs of the tokens behind the prompt."""
    return torch.tensor([float(lp[t - 1, ids[t]]) for t in range(n, len(ids))])


def _prompt(n, seed):
    return torch.randint(1, 512, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _engine(m, dev, **kw):
    from axrl_b200.rollout.engine import RolloutEngine

    args = dict(max_batch=8, kv_tokens=4096, max_context=512, page_size=16, seed=3, burst=8, kv_format="fp8_block", use_cuda_graph=dev == "cuda", eos_token_id=0)
    return RolloutEngine(m, **(args | kw))


def _req(rid, prompt, n):
    from axrl_b200.rollout.engine import GenRequest

    return GenRequest(rid=rid, prompt=prompt, max_new_tokens=n, temperature=1.0, seed_stream=len(prompt))


def _check(m, batch, plants):
    """`batch`: (result, prompt) of the requests that ran together."""
    moved = dict.fromkeys(plants, 0.0)
    for res, prompt in batch:
        ids, n, c0 = list(prompt) + res.output_ids, len(prompt), res.cached_tokens
        want = _given(_oracle(m, ids, n), ids, n)
        tol = 3 * (_given(_oracle(m, ids, n, rounded=True), ids, n) - want).abs().max()
        assert ((torch.tensor(res.output_logprobs) - want).abs() <= tol).all(), (res.output_logprobs, want.tolist(), float(tol))
        for plant in plants:
            moved[plant] = max(moved[plant], float((_given(_oracle(m, ids, n, c0, plant=plant), ids, n) - want).abs().max() / tol))
    assert all(x > 1.5 for x in moved.values()), moved


@pytest.mark.parametrize("dev", ["cpu", CUDA])
@pytest.mark.parametrize("page_size,max_context", [(16, 512), (16, 128), (64, 256)])
def test_decoded_tokens(dev, page_size, max_context):
    """A batch of lengths on both sides of page borders; with contexts of up to 448 tokens a CTA of the decode takes a whole sequence and head."""
    m = _model(dev)
    prompts = [_prompt(n, n) for n in (1, 15, 16, 17, 40, 64, 65, 90)]
    eng = _engine(m, dev, page_size=page_size, max_context=max_context)
    if dev == "cuda":
        from axrl_b200.ops import _ext

        direct = _ext.ext().paged_decode_attn_fp8_launches(8, eng.num_pages, NKV, page_size, eng.max_pages) == 1
        assert direct == (max_context == 128 or page_size == 64)
    results = eng.generate([_req(f"r{i}", p, 24) for i, p in enumerate(prompts)])
    assert all(len(r.output_ids) == 24 for r in results)
    _check(m, list(zip(results, prompts)), ["decode", "layer", "short"])


@pytest.mark.parametrize("dev", ["cpu", CUDA])
@pytest.mark.parametrize("n,suffix", [(48, 1), (16, 30), (100, 16)])
def test_continued_prefix(dev, n, suffix):
    m = _model(dev)
    head = _prompt(n, 1)
    eng = _engine(m, dev)
    eng.generate([_req("h", head, 3)])
    long = head + _prompt(suffix, 2)
    res = eng.generate([_req("c", long, 12)])[0]
    assert res.cached_tokens == n // 16 * 16
    _check(m, [(res, long)], ["prefix", "decode"])
