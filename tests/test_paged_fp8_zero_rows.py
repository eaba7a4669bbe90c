"""Decode over an 8-bit cache whose value rows differ in what they can add: rows of zeros that take a large share of the
weights, rows whose codes are far below their scale, outliers.

Tolerance, from the roundings (weights w_t = p_t 2^{e_t} on the codes c_t of row t, W the largest of them; a row of zeros adds
nothing whatever its weight, and counts in W as if its scale were 2^-60):
  a score is off by at most 2^-18 sum|q k| scale (32-bit sums of 128 products) and 2^-28 max|q| sum|k| scale (q in 16 bits);
  a weight is rounded to 16 bits, 2^-11 of itself (2^-10 with its exponential), and a small one by 2^-25 of 2^-15 W;
  the output is rounded to bf16, 2^-8."""

import math

import pytest
import torch

from axrl_b200.ops import paged_fp8 as pf

D = 128
CUDA = pytest.param("cuda", marks=pytest.mark.gpu)


def _check(q, cache, bt, lens):
    got = pf.paged_decode_attention_fp8(q, cache, bt, lens)
    if q.is_cuda:
        from axrl_b200.ops import _ext

        assert _ext.ext().kv_fp8_error() == 0
    B, Hq, _ = q.shape
    Hkv, P = cache.k.shape[1:3]
    G, scale = Hq // Hkv, D ** -0.5
    for b in range(B):
        n = int(lens[b])
        pages = bt[b, :-(-n // P)].long()
        for h in range(Hkv):
            rows = lambda t: t.view(torch.uint8)[pages, h].flatten(0, 1)[:n].view(t.dtype).double()  # noqa: E731,B023
            k, c, s = rows(cache.k) * rows(cache.k_scale)[:, None], rows(cache.v), rows(cache.v_scale)
            qq = q[b, h * G:(h + 1) * G].double()
            p = torch.softmax(qq @ k.t() * scale, -1)
            off = (2.0 ** -18 * (qq.abs() @ k.abs().t()).amax(-1) + 2.0 ** -28 * qq.abs().amax(-1) * k.abs().sum(-1).amax()) * scale
            want, a = p @ (c * s[:, None]), p @ (c.abs() * s[:, None])
            unit = torch.where((c == 0).all(-1), s.clamp_max(2.0 ** -60), s)
            W = (p * unit).amax(-1)
            tol = 2.0 ** -8 * want.abs() + a * (2.0 ** -10 + 2 * off[:, None]) + 2.0 ** -40 * W[:, None] * c.abs().sum(0)
            err = (got[b, h * G:(h + 1) * G].double() - want).abs()
            assert (err <= tol).all(), (b, h, float(err.max()), float(want.abs().max()), float(p.amax()))
    return got


def _case(lens, hq, hkv, P, dev, size, delta, zero, seed=0):
    """Sequences of values of about `size`, their scores within about 1 of 0; the tokens that `zero(n)` names have values of zero
    and scores of about `delta`."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // P) for n in lens]
    pages, G = sum(need) + 1, hq // hkv
    q = torch.randn(len(lens), hkv, 1, D, generator=g) + 0.1 * torch.randn(len(lens), hkv, G, D, generator=g)
    k = torch.randn(pages, hkv, P, D, generator=g) * 0.3
    v = torch.randn(pages, hkv, P, D, generator=g) * size
    order = torch.randperm(pages, generator=g)
    bt = torch.zeros(len(lens), max(need) + 1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = order[at:at + n].to(torch.int32)
        at += n
        top = q[b, :, 0] * (delta * math.sqrt(D) / q[b, :, 0].pow(2).sum(-1, keepdim=True))
        for t in zero(lens[b]):
            page = int(bt[b, t // P])
            k[page, :, t % P], v[page, :, t % P] = top, 0.0
    (kc, ks), (vc, vs) = pf.quantize_rows_e8m0(k), pf.quantize_rows_e8m0(v)
    cache = pf.Fp8KV(kc, vc, ks, vs)
    return q.reshape(len(lens), hq, D).bfloat16().to(dev), pf.Fp8KV(*(t.to(dev) for t in cache)), bt.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)


FIRST = {"first": lambda n: [0], "middle": lambda n: [n // 2], "last": lambda n: [n - 1], "unit": lambda n: range(min(64, n - 1)),
         "some": lambda n: range(0, n, 37)}


@pytest.mark.parametrize("dev", ["cpu", CUDA])
@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-6])
@pytest.mark.parametrize("delta", [0.0, 4.0, 8.0])
@pytest.mark.parametrize("n,where", [(300, "first"), (300, "middle"), (300, "unit"), (4096, "first"), (4096, "last")])
def test_zero_rows(dev, size, delta, n, where):
    _check(*_case([n, n - 7], 8, 2, 64, dev, size, delta, FIRST[where]))


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-6])
@pytest.mark.parametrize("delta", [0.0, 4.0, 8.0])
@pytest.mark.parametrize("hq,hkv", [(4, 1), (16, 1)])
def test_zero_rows_long_context(size, delta, hq, hkv):
    _check(*_case([100000], hq, hkv, 64, "cuda", size, delta, FIRST["first"]))


@pytest.mark.gpu
@pytest.mark.parametrize("where", list(FIRST))
@pytest.mark.parametrize("hq,hkv,P", [(32, 8, 64), (16, 1, 16), (4, 4, 128)])
def test_zero_rows_of_a_batch(where, hq, hkv, P):
    """Warps that walk whole sequences, and ranges that begin or end in them."""
    lens = [1000 + 97 * (i % 23) for i in range(40)]
    for size, delta in ((1.0, 8.0), (1e-3, 4.0), (1e-6, 0.0)):
        _check(*_case(lens, hq, hkv, P, "cuda", size, delta, FIRST[where], seed=len(where)))


@pytest.mark.parametrize("dev", ["cpu", CUDA])
@pytest.mark.parametrize("byte", [0, 66, 67, 127, 200, 254])
def test_zero_rows_of_any_scale(dev, byte):
    """A row of zeros adds nothing whatever scale it has, zeros with a sign among them."""
    q, cache, bt, lens = _case([300, 700], 8, 2, 64, dev, 0.05, 3.0, FIRST["some"])
    zero = (cache.v.float() == 0).all(-1)
    assert zero.any()
    cache.v_scale.view(torch.uint8)[zero] = byte
    cache.v.view(torch.uint8)[zero] = (torch.arange(D, device=dev) % 2 * 128).to(torch.uint8)
    _check(q, cache, bt, lens)


@pytest.mark.parametrize("dev", ["cpu", CUDA])
def test_appended_and_unwritten_zero_rows(dev):
    """Rows of zeros as append writes them, and slots that nothing was written to."""
    nq, nkv, P, T = 8, 2, 16, 90
    g = torch.Generator().manual_seed(5)
    cache = pf.layer_cache(*pf.empty_cache((), 8, nkv, P, dev))
    qkv = torch.randn(T, nq + 2 * nkv, D, generator=g)
    qkv[:, nq + nkv:] *= 1e-3
    qkv[[3, 40, 41, 89], nq + nkv:] = 0
    qkv = qkv.bfloat16().to(dev).view(T, -1)
    w = torch.ones(D, dtype=torch.bfloat16, device=dev)
    inv = (1e6 ** (-torch.arange(0, D, 2, dtype=torch.float32) / D)).to(dev)
    t = torch.arange(T, device=dev)
    order = torch.tensor([5, 1, 6, 2, 7, 3], dtype=torch.int32, device=dev)
    q, _, v = pf.qk_norm_rope_cache_fp8(qkv, w, w, t.to(torch.int32), inv, nq, nkv, 1e-6, cache, order.long()[t // P] * P + t % P)
    assert (v[40] == 0).all()
    for n in (45, 90, 96):  # 96: six rows behind the last one that was appended
        _check(q[-1:], cache, order[None], torch.tensor([n], dtype=torch.int32, device=dev))
    empty = pf.layer_cache(*pf.empty_cache((), 8, nkv, P, dev))
    assert (_check(q[-1:], empty, order[None], torch.tensor([90], dtype=torch.int32, device=dev)) == 0).all()


@pytest.mark.parametrize("dev", ["cpu", CUDA])
def test_codes_far_below_their_scale_and_outliers(dev):
    """A row that is not zero but small next to its scale, with most of the weight; a row with one large channel."""
    q, cache, bt, lens = _case([900, 4096], 8, 2, 64, dev, 0.02, 6.0, FIRST["middle"])
    zero = (cache.v.float() == 0).all(-1)
    codes = cache.v.view(torch.uint8)
    codes[zero] = 1  # 2^-9
    _check(q, cache, bt, lens)
    codes[zero] = 0
    one = torch.zeros(D, dtype=torch.uint8, device=dev)
    one[100] = 0x81
    codes[zero] = one  # a single code of -2^-9, the other 127 are zeros
    _check(q, cache, bt, lens)
    one[100], one[3] = 0x7E, 0x08  # 448 in one channel
    codes[zero] = one
    _check(q, cache, bt, lens)
    # what is not seen decides nothing
    cache.v.view(torch.uint8)[int(bt[0, 900 // 64]), :, 900 % 64:] = 0
    cache.v_scale.view(torch.uint8)[int(bt[0, 900 // 64]), :, 900 % 64:] = 255
    _check(q, cache, bt, lens)


@pytest.mark.parametrize("dev", ["cpu", CUDA])
def test_large_scores(dev):
    """Scores past the integers that 32 bits hold (where one is a multiple of 2 or more): one token takes everything."""
    q, cache, bt, lens = _case([300], 4, 1, 64, dev, 1.0, 0.0, FIRST["first"])
    for up in (130, 137, 143):  # keys of about 2^3, 2^10, 2^16
        cache.k_scale.view(torch.uint8)[:] = up
        big = (q.float() * 2.0 ** 6).bfloat16()
        got = pf.paged_decode_attention_fp8(big, cache, bt, lens).double()
        assert got.isfinite().all() and got.abs().max() < 10
