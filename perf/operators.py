"""Measured cases of the 8-bit paged KV cache: appending to it, decoding over it, loading rows back from it.

Cache of one layer: ``k``, ``v`` e4m3 codes [pages, Hkv, P, 128] and ``k_scale``, ``v_scale`` e8m0 powers of two
[pages, Hkv, P], one per token and head.  Slot = page * P + offset.
"""

import math
import random

import torch

own = False

D = 128
THETA = 1e6
EPS = 1e-6


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # a single request decoding: one token appended
        {"name": "append-1", "op": "append", "T": 1, "nq": 32, "nkv": 8, "P": 64, "far": 4096, "kv": False},
        # a decode step of 64 sequences, far into their contexts
        {"name": "append-64", "op": "append", "T": 64, "nq": 32, "nkv": 8, "P": 64, "far": 16384, "kv": False},
        # an odd-sized prefill on small pages, whose attention takes the rows as the cache holds them
        {"name": "append-2049", "op": "append", "T": 2049, "nq": 16, "nkv": 8, "P": 16, "far": 2049, "kv": True},
        # the largest prefill micro-batch of the rollout engine
        {"name": "append-16384", "op": "append", "T": 16384, "nq": 32, "nkv": 8, "P": 64, "far": 16384, "kv": True},
        # the smallest decode call: one short sequence
        {"name": "decode-1x300", "op": "decode", "B": 1, "L": 300, "shape": "even", "nq": 32, "nkv": 8, "P": 64},
        # a small batch at 2k contexts
        {"name": "decode-8x2048", "op": "decode", "B": 8, "L": 2048, "shape": "near", "nq": 32, "nkv": 8, "P": 64},
        # many short sequences, some rows idle; four kv heads
        {"name": "decode-256-short", "op": "decode", "B": 256, "L": 1024, "shape": "ragged", "nq": 32, "nkv": 4, "P": 64},
        # a rollout batch whose responses have long tails
        {"name": "decode-64-tail", "op": "decode", "B": 64, "L": 8704, "shape": "tail", "nq": 32, "nkv": 8, "P": 64},
        # two very long contexts
        {"name": "decode-2x100k", "op": "decode", "B": 2, "L": 100001, "shape": "near", "nq": 16, "nkv": 8, "P": 128},
        # one page of a shared prompt
        {"name": "load-64", "op": "load", "T": 64, "nkv": 8, "P": 64},
        # the prefixes of 32 conversations that go on
        {"name": "load-131072", "op": "load", "T": 131072, "nkv": 8, "P": 64},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "load"])
    nq, nkv = rng.choice([(32, 8), (32, 4), (16, 8), (8, 1), (32, 2), (20, 4)])
    P = rng.choice([16, 32, 64, 64, 128])
    if op == "append":
        T = _log(rng, 1, 16000)
        return {"op": op, "T": T, "nq": nq, "nkv": nkv, "P": P, "far": max(T, _log(rng, 64, 100000)), "kv": rng.random() < 0.5}
    if op == "load":
        return {"op": op, "T": _log(rng, 1, 130000), "nkv": nkv, "P": P}
    B = _log(rng, 1, 256)
    return {"op": op, "B": B, "L": _log(rng, 1, max(64, min(100000, 180000 // B))), "shape": rng.choice(["even", "near", "ragged", "tail"]),
            "nq": nq, "nkv": nkv, "P": P}


def _lens(case):
    """Context lengths of a decode case (the same for every seed)."""
    B, L = case["B"], case["L"]
    r = random.Random(B * 1000003 + L)
    if case["shape"] == "even":
        return [L] * B
    if case["shape"] == "near":  # all within a tenth of L
        return [max(1, L - r.randrange(1 + L // 10)) for _ in range(B)]
    if case["shape"] == "ragged":  # anything up to L; one in sixteen rows is idle
        return [0 if r.random() < 1 / 16 else r.randint(1, L) for _ in range(B)]
    return [min(L, max(1, L // 17 + int(L / 8 * math.exp(r.gauss(0, 1))))) for _ in range(B)]  # log-normal responses after a prompt


def work(case):
    nkv = case["nkv"]
    if case["op"] == "append":
        T, nq = case["T"], case["nq"]
        return {"bytes": T * ((nq + 2 * nkv) * 256 + nq * 256 + (nkv * 512 if case["kv"] else 0) + nkv * 258 + 12), "flops": T * (nq + nkv) * D * 9}
    if case["op"] == "load":
        T = case["T"]
        return {"bytes": T * (nkv * 2 * (129 + 256) + 8), "flops": T * nkv * 2 * D}
    total = sum(_lens(case))
    return {"bytes": total * nkv * 258 + case["B"] * case["nq"] * 512, "flops": 4 * total * case["nq"] * D}


# ----------------------------------------------------------------------------- inputs
def _quantise(x):
    """(codes, scales) of rows (..., 128) in fp32: the least power of two with amax <= 448 * scale."""
    m, e = torch.frexp(x.abs().amax(-1))
    e = e - 9 + (m > 0.875).to(e.dtype)
    e = torch.where(m == 0, torch.zeros_like(e), e)
    codes = torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _cache(pages, nkv, P, gen):
    """A cache full of rows such as normalised keys and values: values of a token share a size that varies from token to token."""
    dev = gen.device
    out = {}
    for name in ("k", "v"):
        codes = torch.empty(pages, nkv, P, D, dtype=torch.float8_e4m3fn, device=dev)
        scales = torch.empty(pages, nkv, P, dtype=torch.uint8, device=dev).view(torch.float8_e8m0fnu)
        step = max(1, (1 << 27) // (nkv * P * D))
        for a in range(0, pages, step):
            n = min(step, pages - a)
            x = torch.randn(n, nkv, P, D, generator=gen, device=dev)
            if name == "v":
                x *= torch.exp(torch.randn(n, nkv, P, 1, generator=gen, device=dev) * 0.7) * 0.3
            c, s = _quantise(x)
            codes[a:a + n], scales.view(torch.uint8)[a:a + n] = c, s.view(torch.uint8)
        out[name], out[name + "_scale"] = codes, scales
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(dev).manual_seed(seed * 7919 + 13)
    nkv, P = case["nkv"], case["P"]
    st = {"case": case, "dev": dev}
    if case["op"] == "decode":
        nq, lens = case["nq"], _lens(case)
        need = [-(-n // P) for n in lens]
        pages = sum(need) + 3
        st["cache"] = _cache(pages, nkv, P, gen)
        order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
        bt = torch.zeros(len(lens), max(1, max(need)), dtype=torch.int32, device=dev)
        at = 0
        for b, n in enumerate(need):
            bt[b, :n] = order[at:at + n]
            at += n
        st["block_table"], st["lens"] = bt, torch.tensor(lens, dtype=torch.int32, device=dev)
        st["q"] = (torch.randn(len(lens), nq, D, generator=gen, device=dev) * 2).bfloat16()
        return st
    T = case["T"]
    pages = -(-T // P) + 3
    st["cache"] = _cache(pages, nkv, P, gen)
    # runs of consecutive slots on pages in any order, as the engine hands them out
    order = torch.randperm(pages, generator=gen, device=dev)
    t = torch.arange(T, device=dev)
    st["slots"] = order[t // P] * P + t % P
    if case["op"] == "load":
        return st
    nq = case["nq"]
    qkv = torch.randn(T, (nq + 2 * nkv) * D, generator=gen, device=dev)
    st["qkv"] = (qkv * torch.exp(torch.randn(T, 1, generator=gen, device=dev) * 0.5)).bfloat16()
    st["qw"] = (1 + 0.2 * torch.randn(D, generator=gen, device=dev)).bfloat16()
    st["kw"] = (1 + 0.2 * torch.randn(D, generator=gen, device=dev)).bfloat16()
    st["pos"] = (t if T == case["far"] else torch.randint(0, case["far"], (T,), generator=gen, device=dev)).to(torch.int32)
    st["inv_freq"] = 1.0 / (THETA ** (torch.arange(0, D, 2, dtype=torch.float32, device=dev) / D))
    return st


# ----------------------------------------------------------------------------- the operators
def _values(codes, scales):
    return codes.float() * scales.float()[..., None]


def _plain_append(st):
    case, c = st["case"], st["cache"]
    T, nq, nkv, P = case["T"], case["nq"], case["nkv"], case["P"]
    x = st["qkv"].float().view(T, nq + 2 * nkv, D)
    ang = st["pos"].double()[:, None] * st["inv_freq"].double()  # far positions: 32 bits lose the angle
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]

    def turned(x, w):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    q = turned(x[:, :nq], st["qw"]).bfloat16()
    page, off = st["slots"] // P, st["slots"] % P
    out = {"q": q}
    for name, rows in (("k", turned(x[:, nq:nq + nkv], st["kw"])), ("v", x[:, nq + nkv:])):
        codes, scales = _quantise(rows)
        c[name].view(torch.uint8)[page, :, off] = codes.view(torch.uint8)
        c[name + "_scale"].view(torch.uint8)[page, :, off] = scales.view(torch.uint8)
        if case["kv"]:
            out[name] = _values(codes, scales).bfloat16()
    return out | {"cache": c}


def _plain_decode(st):
    case, c, bt, lens, q = st["case"], st["cache"], st["block_table"], st["lens"], st["q"]
    B, nq, nkv, P = case["B"], case["nq"], case["nkv"], case["P"]
    L = bt.shape[1] * P
    at = bt.long()
    k, v = (_values(c[n].view(torch.uint8)[at].view(torch.float8_e4m3fn), c[n + "_scale"].view(torch.uint8)[at].view(torch.float8_e8m0fnu))
            .permute(0, 2, 1, 3, 4).reshape(B, nkv, L, D) for n in ("k", "v"))
    s = q.float().view(B, nkv, nq // nkv, D) @ k.transpose(-1, -2) / math.sqrt(D)
    seen = torch.arange(L, device=q.device) < lens[:, None]
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e30))
    o = (p @ v) / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return {"o": o.view(B, nq, D).bfloat16()}


def _plain_load(st):
    c, P = st["cache"], st["case"]["P"]
    page, off = st["slots"] // P, st["slots"] % P
    return {n: _values(c[n].view(torch.uint8)[page, :, off].view(torch.float8_e4m3fn),
                       c[n + "_scale"].view(torch.uint8)[page, :, off].view(torch.float8_e8m0fnu)).bfloat16() for n in ("k", "v")}


def run(state):
    case = state["case"]
    if own:
        from axrl_b200.ops import paged_fp8

        c = state["cache"]
        cache = paged_fp8.Fp8KV(c["k"], c["v"], c["k_scale"], c["v_scale"])
        if case["op"] == "append":
            q, k, v = paged_fp8.qk_norm_rope_cache_fp8(state["qkv"], state["qw"], state["kw"], state["pos"], state["inv_freq"], case["nq"],
                                                       case["nkv"], EPS, cache, state["slots"], want_kv=case["kv"])
            return {"q": q, "cache": c} | ({"k": k, "v": v} if case["kv"] else {})
        if case["op"] == "decode":
            return {"o": paged_fp8.paged_decode_attention_fp8(state["q"], cache, state["block_table"], state["lens"])}
        k, v = paged_fp8.gather_kv_fp8(cache, state["slots"])
        return {"k": k, "v": v}
    return {"append": _plain_append, "decode": _plain_decode, "load": _plain_load}[case["op"]](state)


# ----------------------------------------------------------------------------- 64 bits
def _e4m3(x):
    """x (64 bits, |x| <= 448) rounded to e4m3: 3 bits after the leading one, exponents from -6, ties to even."""
    _, e = torch.frexp(x)
    quantum = torch.exp2((e - 1).clamp_min(-6).double() - 3)
    return torch.round(x / quantum) * quantum


def _split(x):
    """Codes and scales (64-bit values) of rows."""
    amax = x.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(torch.where(amax > 0, amax, torch.ones_like(amax)) / 448)))
    scale = torch.where(amax > scale * 448, scale * 2, scale)
    scale = torch.where(amax <= scale * 224, scale / 2, scale)  # log2 is not exact next to a power of two
    scale = torch.where(amax > 0, scale, torch.ones_like(scale))
    return _e4m3(x / scale), scale[..., 0]


def exact(case, seed):
    st = prepare(case, seed)
    c, P, nkv = st["cache"], case["P"], case["nkv"]
    if case["op"] == "load":
        rows = lambda x: x.double().transpose(1, 2).reshape(-1, nkv, *x.shape[3:])[st["slots"]]  # noqa: E731
        return {n: rows(c[n]) * rows(c[n + "_scale"])[..., None] for n in ("k", "v")}
    if case["op"] == "decode":
        G = case["nq"] // nkv
        o = torch.zeros(case["B"], case["nq"], D, dtype=torch.float64, device=st["dev"])
        for b, n in enumerate(_lens(case)):
            if n == 0:
                continue
            pages = st["block_table"][b, :-(-n // P)].long()
            for h in range(nkv):
                k, v = (c[x][pages, h].double().reshape(-1, D)[:n] * c[x + "_scale"][pages, h].double().reshape(-1)[:n, None] for x in ("k", "v"))
                o[b, h * G:(h + 1) * G] = torch.softmax(st["q"][b, h * G:(h + 1) * G].double() @ k.t() * D ** -0.5, -1) @ v
        return {"o": o}
    T, nq = case["T"], case["nq"]
    x = st["qkv"].double().reshape(T, -1, D)
    phase = torch.polar(torch.ones((), dtype=torch.float64, device=st["dev"]), st["pos"].double()[:, None, None] * st["inv_freq"].double())

    def turned(x, w):
        x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / D + EPS) * w.double()
        z = torch.complex(x[..., :D // 2], x[..., D // 2:]) * phase
        return torch.cat([z.real, z.imag], -1)

    out, cache = {"q": turned(x[:, :nq], st["qw"])}, {}
    for name, rows in (("k", turned(x[:, nq:nq + nkv], st["kw"])), ("v", x[:, nq + nkv:])):
        codes, scales = _split(rows)
        for key, was, now in ((name, c[name], codes), (name + "_scale", c[name + "_scale"], scales)):
            flat = was.double().transpose(1, 2).reshape(-1, nkv, *was.shape[3:])
            flat[st["slots"]] = now
            cache[key] = flat.reshape(was.shape[0], P, nkv, *was.shape[3:]).transpose(1, 2).contiguous()
        if case["kv"]:
            out[name] = codes * scales[..., None]
    return out | {"cache": cache}
