"""8-bit paged KV cache (append, decode attention, load) against plain implementations in 64 bits.

Tolerances, from the roundings: bf16 rounds by at most 2^-8 of a value, e4m3 by at most 2^-4 of it (or half of its
smallest step, 2^-10 of the row's scale).  A rotated value x c - y s carries a few 32-bit roundings of terms no larger
than the row's largest: 2^-18 of that covers them."""

import math

import pytest
import torch

from axrl_b200.ops import paged_fp8 as pf

D = 128
EPS = 1e-6
CUDA = pytest.param("cuda", marks=pytest.mark.gpu)


def _cache(pages, hkv, P, dev, seed=0, fill=True):
    codes, scales = pf.empty_cache((), pages, hkv, P, "cpu")
    if fill:
        g = torch.Generator().manual_seed(seed)
        x = torch.randn(2, pages, hkv, P, D, generator=g)
        x[1] *= torch.exp(torch.randn(pages, hkv, P, 1, generator=g))
        codes, scales = pf.quantize_rows_e8m0(x)
    return pf.layer_cache(codes.to(dev), scales.to(dev))


def _inputs(T, nq, nkv, dev, seed=0, far=1000):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(T, (nq + 2 * nkv) * D, generator=g) * torch.exp(torch.randn(T, 1, generator=g))).bfloat16().to(dev)
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=g)).bfloat16().to(dev) for _ in range(2))
    pos = torch.randint(0, far, (T,), generator=g).to(torch.int32).to(dev)
    inv = (1e6 ** (-torch.arange(0, D, 2, dtype=torch.float32) / D)).to(dev)
    return qkv, qw, kw, pos, inv


def _exact_rows(qkv, qw, kw, pos, inv, nq, nkv, eps=EPS):
    """q, k, v rows in 64 bits."""
    x = qkv.double().view(qkv.shape[0], -1, D)
    ang = pos.double()[:, None, None] * inv.double()
    c, s = ang.cos(), ang.sin()

    def turned(x, w):
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
        a, b = x.chunk(2, -1)
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    return turned(x[:, :nq], qw), turned(x[:, nq:nq + nkv], kw), x[:, nq + nkv:]


def _values(codes, scales):
    return codes.float().double() * scales.float().double()[..., None]


def _at(t, slots):
    P = t.shape[2]
    return t.view(torch.uint8)[slots // P, :, slots % P].view(t.dtype)


# ----------------------------------------------------------------------------- quantisation
def test_quantize_rows_scale_is_the_least_power_of_two():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4000, D, generator=g) * torch.exp2(torch.randint(-45, 60, (4000, 1), generator=g).float())
    x[0] = 0
    x[1, 0], x[1, 1:] = 448.0, 1.0  # on the border: scale 1
    x[2, 0], x[2, 1:] = 448.5, 1.0  # past it: scale 2
    codes, scales = pf.quantize_rows_e8m0(x)
    s = scales.float().double()
    amax = x.double().abs().amax(-1)
    assert torch.equal(torch.log2(s), torch.round(torch.log2(s)))
    assert s[0] == 1 and s[1] == 1 and s[2] == 2 and (codes[0].float() == 0).all()
    live = amax > 0
    assert (amax <= 448 * s).all() and (amax > 224 * s)[live].all()
    err = (_values(codes, scales) - x.double()).abs()
    assert (err <= torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * s[:, None])).all()


def test_quantize_rows_not_finite_stands_for_nan():
    x = torch.ones(3, D)
    x[0, 5], x[1, 7] = float("nan"), float("-inf")
    codes, scales = pf.quantize_rows_e8m0(x)
    v = pf.dequantize_rows_e8m0(codes, scales)
    assert v[:2].isnan().all() and (v[2] == 1).all()
    assert scales.view(torch.uint8).tolist()[:2] == [255, 255] and (codes.view(torch.uint8)[:2] == 0).all()


# ----------------------------------------------------------------------------- append
def _check_append(dev, T, nq, nkv, P, far, seed=0, want_kv=True):
    pages = -(-T // P) + 2
    cache = _cache(pages, nkv, P, dev, seed)
    before = [t.view(torch.uint8).clone() for t in cache]
    qkv, qw, kw, pos, inv = _inputs(T, nq, nkv, dev, seed, far)
    slots = torch.randperm(pages * P, generator=torch.Generator().manual_seed(seed))[:T].to(dev)
    q, k, v = pf.qk_norm_rope_cache_fp8(qkv, qw, kw, pos, inv, nq, nkv, EPS, cache, slots, want_kv=want_kv)
    xq, xk, xv = _exact_rows(qkv, qw, kw, pos, inv, nq, nkv)
    assert q.dtype == torch.bfloat16 and q.shape == (T, nq, D)
    top = xq.abs().amax(-1, keepdim=True) if nq else 0
    assert ((q.double() - xq).abs() <= 2.0 ** -8 * xq.abs() + 2.0 ** -18 * top).all()
    for x, codes, scales, back in ((xk, cache.k, cache.k_scale, k), (xv, cache.v, cache.v_scale, v)):
        c, s = _at(codes, slots), _at(scales, slots)
        sv, top = s.float().double(), x.abs().amax(-1)
        assert (top <= 448 * sv * (1 + 2.0 ** -18)).all() and (top >= 224 * sv * (1 - 2.0 ** -18)).all()
        err = (_values(c, s) - x).abs()
        assert (err <= torch.maximum(2.0 ** -4 * x.abs(), 2.0 ** -10 * sv[..., None]) + 2.0 ** -18 * top[..., None]).all()
        if want_kv:  # what is returned is what the cache stands for
            assert torch.equal(back.double(), _values(c, s))
        else:
            assert back is None
    # values are quantised from the input as it is
    cv, sv = pf.quantize_rows_e8m0(xv.float())
    assert torch.equal(_at(cache.v, slots).view(torch.uint8), cv.view(torch.uint8)) and torch.equal(_at(cache.v_scale, slots).view(torch.uint8), sv.view(torch.uint8))
    # nothing else in the cache moved
    rest = torch.ones(pages * P, dtype=torch.bool, device=dev)
    rest[slots] = False
    rest = rest.nonzero().squeeze(1)
    for t, was in zip(cache, before):
        assert torch.equal(_at(t.view(torch.uint8), rest), _at(was, rest))


@pytest.mark.parametrize("dev", ["cpu", CUDA])
@pytest.mark.parametrize("T,nq,nkv,P,far", [(1, 32, 8, 64, 5), (5, 4, 2, 64, 40), (33, 16, 8, 16, 100_000), (257, 20, 4, 32, 4096), (70, 1, 1, 128, 70),
                                            (19, 8, 1, 7, 300), (9, 6, 3, 64, 50), (3, 0, 2, 16, 9)])
@pytest.mark.parametrize("want_kv", [True, False])
def test_append(dev, T, nq, nkv, P, far, want_kv):
    _check_append(dev, T, nq, nkv, P, far, want_kv=want_kv)


@pytest.mark.gpu
@pytest.mark.parametrize("T,nq,nkv", [(700, 16, 8), (2048, 32, 8), (5003, 32, 8), (5003, 8, 1)])
def test_append_many_tokens(T, nq, nkv):
    _check_append("cuda", T, nq, nkv, 64, 20000)


@pytest.mark.parametrize("dev", ["cpu", CUDA])
def test_append_skips_slots_outside_the_cache_and_takes_no_tokens(dev):
    cache = _cache(2, 2, 16, dev)
    before = [t.view(torch.uint8).clone() for t in cache]
    qkv, qw, kw, pos, inv = _inputs(4, 4, 2, dev)
    slots = torch.tensor([-1, 2 * 16, 3, 1 << 40], device=dev)
    q, k, v = pf.qk_norm_rope_cache_fp8(qkv, qw, kw, pos, inv, 4, 2, EPS, cache, slots)
    xq, xk, xv = _exact_rows(qkv, qw, kw, pos, inv, 4, 2)
    assert (q.double() - xq).abs().max() < 2.0 ** -8 * xq.abs().max() * 1.01
    assert (k.double() - xk).abs().max() <= 2.0 ** -4 * xk.abs().max() * 1.01
    for t, was in zip(cache, before):
        now = t.view(torch.uint8).transpose(1, 2).flatten(0, 1)
        was = was.transpose(1, 2).flatten(0, 1)
        assert t.dim() == 3 or (now[3] != was[3]).any()
        keep = torch.arange(32, device=dev) != 3
        assert torch.equal(now[keep], was[keep])
    q, k, v = pf.qk_norm_rope_cache_fp8(qkv[:0], qw, kw, pos[:0], inv, 4, 2, EPS, cache, slots[:0])
    assert q.shape == (0, 4, D) and k.shape == (0, 2, D) and v.shape == (0, 2, D)


@pytest.mark.parametrize("dev", ["cpu", CUDA])
def test_append_tiny_values(dev):
    """No scale is below 2^-60; a row next to ones of ordinary size still takes its share of the weights when it is nearly zero."""
    cache = _cache(1, 1, 16, dev)
    qkv, qw, kw, pos, inv = _inputs(6, 1, 1, dev)
    x = qkv.view(6, 3, D)
    x[1, 2] *= 2.0 ** -55
    x[2, 2] *= 2.0 ** -120
    x[3, 2, 1:] = 0
    x[3, 2, 0] = 2.0 ** -133  # the smallest bf16
    q, _, v = pf.qk_norm_rope_cache_fp8(qkv, qw, kw, pos, inv, 1, 1, EPS, cache, torch.arange(6, device=dev))
    assert cache.v_scale.view(torch.uint8)[0, 0, :6].min() == 127 - 60
    err = (v.double() - x[:, 2:].double()).abs()
    assert (err <= torch.maximum(2.0 ** -4 * x[:, 2:].double().abs(), torch.full_like(err, 2.0 ** -70))).all()
    _check_decode(q[:1], cache, torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.tensor([6], dtype=torch.int32, device=dev))


@pytest.mark.parametrize("dev", ["cpu", CUDA])
def test_append_rows_that_are_not_finite(dev):
    cache = _cache(1, 1, 16, dev)
    qkv, qw, kw, pos, inv = _inputs(4, 1, 1, dev)
    x = qkv.view(4, 3, D)
    x[0, 1, 3], x[1, 2, 9], x[2, 2] = float("nan"), float("inf"), 0.0
    _, k, v = pf.qk_norm_rope_cache_fp8(qkv, qw, kw, pos, inv, 1, 1, EPS, cache, torch.arange(4, device=dev))
    assert k[0].isnan().all() and k[1:].isfinite().all()
    assert v[1].isnan().all() and (v[2] == 0).all() and v[0].isfinite().all() and v[3].isfinite().all()
    assert cache.k_scale.view(torch.uint8)[0, 0, 0] == 255 and cache.v_scale.view(torch.uint8)[0, 0, :4].tolist()[1:3] == [255, 127]
    gk, gv = pf.gather_kv_fp8(cache, torch.arange(4, device=dev))
    torch.testing.assert_close(gk, k, rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(gv, v, rtol=0, atol=0, equal_nan=True)


# ----------------------------------------------------------------------------- load
@pytest.mark.parametrize("dev", ["cpu", CUDA])
@pytest.mark.parametrize("T,hkv,P", [(1, 1, 16), (7, 8, 64), (300, 4, 32), (1000, 3, 7)])
def test_gather(dev, T, hkv, P):
    cache = _cache(9, hkv, P, dev)
    cache.v_scale.view(torch.uint8)[2, 0, 1] = 255
    g = torch.Generator().manual_seed(T)
    slots = torch.randint(0, 9 * P, (T,), generator=g).to(dev)  # repeats are fine
    slots[0] = 2 * P + 1
    bad = [] if T < 7 else [(3, -1), (4, 9 * P), (5, 1 << 35)]
    for i, s in bad:
        slots[i] = s
    k, v = pf.gather_kv_fp8(cache, slots)
    ok = torch.ones(T, dtype=torch.bool, device=dev)
    for i, _ in bad:
        ok[i] = False
    for x, codes, scales in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        want = _values(_at(codes, slots[ok]), _at(scales, slots[ok]))
        torch.testing.assert_close(x[ok].double(), want, rtol=0, atol=0, equal_nan=True)
        assert (x[~ok] == 0).all()
    # into given tensors, with rows behind them left as they were
    buf = torch.full((2, T + 3, hkv, D), 7.0, dtype=torch.bfloat16, device=dev)
    a, b = pf.gather_kv_fp8(cache, slots, buf[0, :T], buf[1, :T])
    assert a.data_ptr() == buf[0].data_ptr() and b.data_ptr() == buf[1].data_ptr()
    torch.testing.assert_close(buf[0, :T], k, rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(buf[1, :T], v, rtol=0, atol=0, equal_nan=True)
    assert (buf[:, T:] == 7).all()
    k, v = pf.gather_kv_fp8(cache, slots[:0])
    assert k.shape == (0, hkv, D) and v.shape == (0, hkv, D)


# ----------------------------------------------------------------------------- decode
def _exact_decode(q, cache, bt, lens, scale):
    """o in 64 bits and its tolerance.  A score is off by at most 2^-18 sum|q k| scale (32-bit sums of 128 products) and
    2^-28 max|q| sum|k| scale (what q drops in 16 bits).  A probability is rounded to 16 bits, at most 2^-11 of its value
    (2^-10 leaves room for its exponential), and a small one by 2^-24 of the largest weight.  The output is rounded to bf16."""
    B, Hq, _ = q.shape
    pages, Hkv, P, _ = cache.k.shape
    G = Hq // Hkv
    o, tol = (torch.zeros(B, Hq, D, dtype=torch.float64, device=q.device) for _ in range(2))
    for b in range(B):
        n = max(0, min(int(lens[b]), bt.shape[1] * P))
        t = torch.arange(n, device=q.device)
        page = bt[b, t // P].long()
        slots = (page * P + t % P)[(page >= 0) & (page < pages)]
        if not slots.numel():
            continue
        for h in range(Hkv):
            k, v = _values(_at(cache.k, slots)[:, h], _at(cache.k_scale, slots)[:, h]), _values(_at(cache.v, slots)[:, h], _at(cache.v_scale, slots)[:, h])
            qq = q[b, h * G:(h + 1) * G].double()
            p = torch.softmax(qq @ k.t() * scale, -1)
            off = 2.0 ** -18 * (qq.abs() @ k.abs().t() * abs(scale)).amax(-1, keepdim=True)
            off = off + 2.0 ** -28 * qq.abs().amax(-1, keepdim=True) * k.abs().sum(-1).amax() * abs(scale)
            a = p @ v.abs()
            o[b, h * G:(h + 1) * G] = p @ v
            tol[b, h * G:(h + 1) * G] = 2.0 ** -8 * (p @ v).abs() + a * (2.0 ** -10 + 2 * off) + 2.0 ** -24 * slots.numel() * a.amax(-1, keepdim=True)
    return o, tol


def _decode_case(lens, hq, hkv, P, dev, seed=0, spread=0, extra=1):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // P) for n in lens]
    pages = sum(need) + 4
    cache = _cache(pages, hkv, P, "cpu", seed)
    order = torch.randperm(pages, generator=g)
    bt = torch.zeros(len(lens), max(need + [0]) + extra, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    # whatever lies behind a sequence's last token must not be read as a number
    for b, n in enumerate(lens):
        if n % P:
            pg = int(bt[b, n // P])
            for t in (cache.k, cache.v):
                t.view(torch.uint8)[pg, :, n % P:] = 0x7F
            for t in (cache.k_scale, cache.v_scale):
                t.view(torch.uint8)[pg, :, n % P:] = 255
    bt[bt == 0] = int(order[0])
    q = (torch.randn(len(lens), hq, D, generator=g) * 2).bfloat16()
    return q.to(dev), pf.Fp8KV(*(t.to(dev) for t in cache)), bt.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)


def _check_decode(q, cache, bt, lens, scale=None):
    got = pf.paged_decode_attention_fp8(q, cache, bt, lens, scale)
    assert got.dtype == q.dtype and got.shape == q.shape
    want, tol = _exact_decode(q, cache, bt, lens, D ** -0.5 if scale is None else scale)
    if q.is_cuda:
        from axrl_b200.ops import _ext

        assert _ext.ext().kv_fp8_error() == 0
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (bad.nonzero()[:5].tolist(), float((got.double() - want).abs().max()))
    return got


@pytest.mark.parametrize("dev", ["cpu", CUDA])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 8), (16, 8), (32, 8), (20, 4), (16, 2), (9, 1), (32, 2)])
@pytest.mark.parametrize("P", [16, 64])
def test_decode_lengths(dev, hq, hkv, P):
    _check_decode(*_decode_case([0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 200, 0], hq, hkv, P, dev))


@pytest.mark.gpu
@pytest.mark.parametrize("P", [16, 32, 48, 64, 96, 128, 256, 1024])
@pytest.mark.parametrize("lens", [[1], [1000], [777, 3, 0, 2500], [64] * 40, [9000, 1, 5000]])
def test_decode_page_sizes(P, lens):
    _check_decode(*_decode_case(lens, 8, 2, P, "cuda", seed=P))


@pytest.mark.gpu
@pytest.mark.parametrize("B", [3, 150, 700, 1500])
def test_decode_many_short_sequences(B):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 90, (B,), generator=g).tolist()
    _check_decode(*_decode_case(lens, 8, 4, 16, "cuda", seed=B))


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv", [(16, 1), (11, 1), (16, 2), (3, 1)])
def test_decode_ragged_batches(hq, hkv):
    """Ranges that hold the end of one pair and the start of the next, several short ones, or the middle of a long one."""
    g = torch.Generator().manual_seed(hq)
    lens = (torch.rand(120, generator=g) ** 3 * 4000).int().tolist()
    _check_decode(*_decode_case(lens, hq, hkv, 64, "cuda", seed=hq))


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv", [(8, 2), (16, 1), (24, 2)])
def test_decode_long_context(hq, hkv):
    _check_decode(*_decode_case([70001, 33000], hq, hkv, 64, "cuda"))


@pytest.mark.parametrize("dev", ["cpu", CUDA])
def test_decode_scales_far_apart(dev):
    """Tokens whose values are far larger or smaller than the others', some of them hardly seen; scores far apart; scale given."""
    q, cache, bt, lens = _decode_case([300, 300, 300], 8, 2, 64, dev)
    for b, (page, byte) in enumerate(((0, 127 + 30), (1, 127 - 40), (2, 127 + 60))):
        cache.v_scale.view(torch.uint8)[int(bt[b, page]), :, 5:9] = byte
    cache.k_scale.view(torch.uint8)[int(bt[0, 2]), :, 7] = 127 - 20
    cache.v.view(torch.uint8)[int(bt[1, 3])] = 0
    _check_decode(q, cache, bt, lens)
    _check_decode(q, cache, bt, lens, scale=0.0)
    _check_decode(q * 4, cache, bt, lens, scale=0.25)
    # one token takes nearly everything, and it is not the one with the large values
    kq = q.clone()
    kq[:] = 0
    got = _check_decode(kq, cache, bt, lens)
    assert got.isfinite().all()


@pytest.mark.parametrize("dev", ["cpu", CUDA])
def test_decode_bad_pages_are_not_seen(dev):
    q, cache, bt, lens = _decode_case([200, 130, 64, 500], 8, 2, 64, dev)
    bt[0, 1], bt[1, 0], bt[2, 0], bt[3, 7] = -1, cache.k.shape[0], -(1 << 31), (1 << 31) - 1
    got = _check_decode(q, cache, bt, lens)
    assert (got[2] == 0).all()
    # lengths beyond the block table are cut to it, negative ones are empty
    lens2 = torch.tensor([1 << 30, 130, -5, (1 << 31) - 1], dtype=torch.int32, device=dev)
    bt[2, 0] = 0
    got = _check_decode(q, cache, bt, lens2)
    assert (got[2] == 0).all()


@pytest.mark.parametrize("dev", ["cpu", CUDA])
def test_decode_row_that_is_not_finite(dev):
    q, cache, bt, lens = _decode_case([100, 100], 4, 2, 64, dev)
    cache.v_scale.view(torch.uint8)[int(bt[0, 0]), 0, 3] = 255
    got = pf.paged_decode_attention_fp8(q, cache, bt, lens)
    assert got[0, :2].isnan().all() and got[0, 2:].isfinite().all() and got[1].isfinite().all()


# ----------------------------------------------------------------------------- together
@pytest.mark.parametrize("dev", ["cpu", CUDA])
def test_append_decode_load_together(dev):
    """Prefill by appending, then token by token: each step's attention is that over everything appended so far, and the rows
    load back as the append returned them."""
    nq, nkv, P, T = 8, 2, 16, 45
    cache = pf.layer_cache(*pf.empty_cache((), 8, nkv, P, dev))
    order = torch.tensor([5, 1, 6, 2], dtype=torch.int32, device=dev)
    qkv, qw, kw, pos, inv = _inputs(T, nq, nkv, dev)
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    slots = order.long()[torch.arange(T, device=dev) // P] * P + torch.arange(T, device=dev) % P
    _, k, v = pf.qk_norm_rope_cache_fp8(qkv[:30], qw, kw, pos[:30], inv, nq, nkv, EPS, cache, slots[:30])
    _, xk, xv = _exact_rows(qkv, qw, kw, pos, inv, nq, nkv)
    for t in range(30, T):
        q, _, _ = pf.qk_norm_rope_cache_fp8(qkv[t:t + 1], qw, kw, pos[t:t + 1], inv, nq, nkv, EPS, cache, slots[t:t + 1], want_kv=False)
        _check_decode(q, cache, order[None], torch.tensor([t + 1], dtype=torch.int32, device=dev))
    gk, gv = pf.gather_kv_fp8(cache, slots)
    assert torch.equal(gk[:30], k) and torch.equal(gv[:30], v)
    assert ((gk.double() - xk).abs() <= 2.0 ** -4 * xk.abs() + 2.0 ** -10 * xk.abs().amax(-1, keepdim=True)).all()
    assert ((gv.double() - xv).abs() <= 2.0 ** -4 * xv.abs() + 2.0 ** -10 * xv.abs().amax(-1, keepdim=True)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[100, 1, 64, 65, 300, 20], [5000, 0, 900, 1, 2000, 777]])
def test_captured_steps_replay_on_a_side_stream(lens):
    """Append + decode captured into two graphs that are replayed in turn on another stream, with new inputs in place."""
    nq, nkv, P, B = 8, 2, 64, 6
    q0, cache, bt, L = _decode_case(lens, nq, nkv, P, "cuda")
    qkv, qw, kw, pos, inv = _inputs(B, nq, nkv, "cuda")
    pos.copy_(L - 1)
    slots = bt.long().gather(1, ((L - 1).clamp_min(0) // P).long()[:, None])[:, 0] * P + (L - 1).long() % P
    slots = torch.where(L > 0, slots, torch.full_like(slots, -1))

    def step():
        q, _, _ = pf.qk_norm_rope_cache_fp8(qkv, qw, kw, pos, inv, nq, nkv, EPS, cache, slots, want_kv=False)
        return q, pf.paged_decode_attention_fp8(q, cache, bt, L)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(s):
        step()
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(step())
            graphs.append(g)
        for i in range(4):
            qkv.copy_(_inputs(B, nq, nkv, "cuda", seed=10 + i)[0])
            graphs[i % 2].replay()
            graphs[1 - i % 2].replay()
            want, tol = _exact_decode(outs[i % 2][0], cache, bt, L, D ** -0.5)
            for q, o in outs:
                assert ((o.double() - want).abs() <= tol).all()
    torch.cuda.current_stream().wait_stream(s)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A cache of 4.9 GB of codes each for K and V; rows in its last pages."""
    pages, nkv, P = 75000, 8, 64
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    codes = [torch.empty(pages, nkv, P, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.empty(pages, nkv, P, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2)]
    cache = pf.Fp8KV(*codes, *scales)
    T = 150
    order = torch.tensor([pages - 1, 3, pages - 2], dtype=torch.int32, device="cuda")
    t = torch.arange(T, device="cuda")
    slots = order.long()[t // P] * P + t % P
    qkv, qw, kw, _, inv = _inputs(T, 16, nkv, "cuda")
    q, k, v = pf.qk_norm_rope_cache_fp8(qkv, qw, kw, t.to(torch.int32), inv, 16, nkv, EPS, cache, slots)
    gk, gv = pf.gather_kv_fp8(cache, slots)
    assert torch.equal(gk, k) and torch.equal(gv, v)
    assert torch.equal(k.double(), _values(_at(cache.k, slots), _at(cache.k_scale, slots)))
    _check_decode(q[-1:], cache, order[None], torch.tensor([T], dtype=torch.int32, device="cuda"))
    wide = torch.zeros(1, 40, dtype=torch.int32, device="cuda")
    wide[0, :3] = order
    _check_decode(q[-1:], cache, wide, torch.tensor([T], dtype=torch.int32, device="cuda"))


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls on two streams, each with its own inputs, in flight together."""
    cases = [_decode_case([4000, 77, 900, 64], 8, 2, 64, "cuda", seed=1), _decode_case([300, 2500, 1, 8000, 40], 16, 1, 16, "cuda", seed=2)]
    want = [_exact_decode(*c, D ** -0.5) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i].append(pf.paged_decode_attention_fp8(*c))
    torch.cuda.synchronize()
    for outs, (o, tol) in zip(got, want):
        for x in outs:
            assert torch.equal(x, outs[0])  # the same order of sums every time
            assert ((x.double() - o).abs() <= tol).all()


# ----------------------------------------------------------------------------- refusals
def _refused(fn, *a, **k):
    with pytest.raises((RuntimeError, ValueError, NotImplementedError, TypeError)):
        fn(*a, **k)


@pytest.mark.gpu
def test_refusals():
    dev = "cuda"
    cache = _cache(3, 2, 16, dev)
    qkv, qw, kw, pos, inv = _inputs(4, 4, 2, dev)
    slots = torch.arange(4, device=dev)

    def app(qkv=qkv, qw=qw, pos=pos, inv=inv, nq=4, nkv=2, cache=cache, slots=slots):
        return pf.qk_norm_rope_cache_fp8(qkv, qw, kw, pos, inv, nq, nkv, EPS, cache, slots)

    app()
    _refused(app, qkv=qkv.float())
    _refused(app, qkv=qkv[:, :-D])
    _refused(app, nq=2, nkv=3)
    _refused(app, pos=pos[:3])
    _refused(app, slots=slots[:3])
    _refused(app, slots=slots.cpu())
    _refused(app, inv=inv[:32])  # a partial rotation has no kernel
    _refused(app, cache=cache._replace(k=cache.k.view(torch.uint8)))
    _refused(app, cache=cache._replace(v_scale=cache.v_scale[:2]))
    _refused(app, cache=cache._replace(k=cache.k[:, :, :, :64]))
    _refused(pf.gather_kv_fp8, cache, slots.view(2, 2))
    _refused(pf.gather_kv_fp8, cache, slots, torch.empty(3, 2, D, dtype=torch.bfloat16, device=dev))
    _refused(pf.gather_kv_fp8, cache, slots, torch.empty(4, 2, D, device=dev))
    q, bt, lens = torch.zeros(2, 4, D, dtype=torch.bfloat16, device=dev), torch.zeros(2, 3, dtype=torch.int32, device=dev), torch.ones(2, dtype=torch.int32, device=dev)

    def dec(q=q, cache=cache, bt=bt, lens=lens):
        return pf.paged_decode_attention_fp8(q, cache, bt, lens)

    dec()
    _refused(dec, q=q.half())
    _refused(dec, q=q[:, :3])
    _refused(dec, q=q.repeat(1, 10, 1))  # 20 heads a kv head
    _refused(dec, bt=bt.long())
    _refused(dec, bt=bt[:1])
    _refused(dec, lens=lens.long())
    _refused(dec, lens=lens.cpu())
    _refused(dec, cache=cache._replace(v=cache.v[:, :, :8]))
    _refused(dec, cache=_cache(3, 2, 24, dev))  # pages are multiples of 16 tokens
    many = (torch.zeros(2049, 4, D, dtype=torch.bfloat16, device=dev), torch.zeros(2049, 3, dtype=torch.int32, device=dev), torch.ones(2049, dtype=torch.int32, device=dev))
    _refused(dec, *many[:1], cache, *many[1:])
    assert dec(many[0][1:], cache, many[1][1:], many[2][1:]).shape == (2048, 4, D)
    assert dec(q=q[:0], bt=bt[:0], lens=lens[:0]).shape == (0, 4, D)
    assert (dec(bt=bt[:, :0]) == 0).all()
