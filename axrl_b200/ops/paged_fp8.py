"""Inference-side ops over a paged KV cache held in 8 bits (rollout engine, ``kv_format="fp8_block"``).

Cache layout per layer (:class:`Fp8KV`): e4m3 codes ``k, v: [num_pages, Hkv, page_size, 128]`` and e8m0
scales ``k_scale, v_scale: [num_pages, Hkv, page_size]``, one power of two per (token, head); a token's slot
is ``page * page_size + offset``.  A row stands for ``code * scale``, which is exact in bf16.  With one scale
per token and head an append writes no byte of another token, so the pages of a shared prefix stay as they
are.  258 bytes per token and head instead of 512.

A row whose values are not all finite is held as NaN (scale byte 255).  None of the ops is differentiable.
CUDA tensors use the kernels in ``csrc/kernels/kv_fp8.cu``; CPU tensors use the PyTorch definitions here
(oracle + CPU plumbing runs).
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from axrl_b200.ops import _ext
from axrl_b200.ops.core import _rms_ref, check_full_rotary


class Fp8KV(NamedTuple):
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def empty_cache(lead: tuple, pages: int, hkv: int, page_size: int, device, dim: int = 128) -> tuple[torch.Tensor, torch.Tensor]:  # noqa: ANN001
    """Zeroed storage ``codes [*lead, 2, pages, Hkv, P, dim]`` (e4m3) and ``scales [*lead, 2, pages, Hkv, P]`` (e8m0)
    of one cache per index of ``lead``; :func:`layer_cache` views one of them."""
    codes = torch.zeros(*lead, 2, pages, hkv, page_size, dim, dtype=torch.uint8, device=device)
    scales = torch.full((*lead, 2, pages, hkv, page_size), 127, dtype=torch.uint8, device=device)
    return codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)


def layer_cache(codes: torch.Tensor, scales: torch.Tensor) -> Fp8KV:
    """The cache of ``codes [2, ...]``, ``scales [2, ...]`` (one layer of :func:`empty_cache`)."""
    return Fp8KV(codes[0], codes[1], scales[0], scales[1])


def quantize_rows_e8m0(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows ``(..., D)`` to e4m3 codes and their e8m0 scales ``(...)``: the least power of two, 2^-60 or more, with
    ``amax <= 448 * scale`` (1 for a row of zeros, NaN with codes 0 for a row that is not finite)."""
    xf = x.float()
    amax = xf.abs().amax(-1)
    ok = amax.isfinite() & xf.isfinite().all(-1)
    m, e = torch.frexp(torch.where(ok, amax, torch.ones_like(amax)))
    e = (e - 9 + (m > 0.875).to(e.dtype)).clamp_min(-60)
    e = torch.where(amax == 0, torch.zeros_like(e), e)
    codes = torch.where(ok[..., None], torch.ldexp(xf, -e[..., None]), torch.zeros_like(xf)).to(torch.float8_e4m3fn)
    byte = torch.where(ok, e + 127, torch.full_like(e, 255)).to(torch.uint8)
    return codes, byte.view(torch.float8_e8m0fnu)


def dequantize_rows_e8m0(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """``codes * scales`` in fp32 (exact)."""
    return codes.float() * scales.float()[..., None]


def _rows(cache: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
    """Rows of a cache tensor at valid ``slots``: (T, Hkv, ...)."""
    P = cache.shape[2]
    return cache.view(torch.uint8)[slots // P, :, slots % P].view(cache.dtype)


def _live(cache: Fp8KV, slots: torch.Tensor) -> torch.Tensor:
    return (slots >= 0) & (slots < cache.k.shape[0] * cache.k.shape[2])


def _rope64(x: torch.Tensor, pos: torch.Tensor, inv_freq: torch.Tensor) -> torch.Tensor:
    """Rotation of (T, H, D) fp32 rows with the angles in 64 bits, as the kernel has them (far positions)."""
    ang = pos.double()[:, None, None] * inv_freq.double()
    c, s = ang.cos().float(), ang.sin().float()
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _append_ref(cache: Fp8KV, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    P, live = cache.k.shape[2], _live(cache, slots)
    at = slots[live]
    out = []
    for rows, codes_to, scales_to in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        codes, scales = quantize_rows_e8m0(rows)
        codes_to.view(torch.uint8)[at // P, :, at % P] = codes.view(torch.uint8)[live]
        scales_to.view(torch.uint8)[at // P, :, at % P] = scales.view(torch.uint8)[live]
        out.append(dequantize_rows_e8m0(codes, scales).to(torch.bfloat16))
    return out[0], out[1]


def qk_norm_rope_cache_fp8(qkv: torch.Tensor, qw: torch.Tensor, kw: torch.Tensor, pos: torch.Tensor, inv_freq: torch.Tensor, nq: int, nkv: int,
                           eps: float, cache: Fp8KV, slots: torch.Tensor, want_kv: bool = True
                           ) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor | None]:
    """q/k norm + RoPE, and append k/v to the 8-bit cache at ``slots`` (int64; a slot outside the cache, such as -1,
    is not written; slots that are read later must be distinct).  K is quantised from its fp32 value.

    Returns q and, with ``want_kv``, k and v as the cache stands for them (bf16, exact): a prefill that attends to
    these sees what later decode steps and :func:`gather_kv_fp8` see.  Without it both are None (decode)."""
    if not qkv.is_cuda:
        check_full_rotary(qw, inv_freq)
        T, dim = qkv.shape[0], qw.numel()
        q, k, v = qkv.view(T, nq + 2 * nkv, dim).float().split([nq, nkv, nkv], 1)
        q = _rope64(_rms_ref(q, qw, eps), pos, inv_freq).to(qkv.dtype)
        k = _rope64(_rms_ref(k, kw, eps), pos, inv_freq)
        k, v = _append_ref(cache, k, v, slots.long())
        return (q, k.to(qkv.dtype), v.to(qkv.dtype)) if want_kv else (q, None, None)
    return _ext.ext().qknorm_rope_cache_fp8(qkv, qw, kw, pos, inv_freq, nq, nkv, eps, *cache, slots, want_kv)


def gather_kv_fp8(cache: Fp8KV, slots: torch.Tensor, out_k: torch.Tensor | None = None, out_v: torch.Tensor | None = None
                  ) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of the cache at ``slots`` (T,) as bf16 ``k, v (T, Hkv, 128)`` (exact; zeros for a slot outside the cache), for a
    prefill that continues a cached prefix.  ``out_k`` / ``out_v``: contiguous tensors to write to instead of new ones."""
    if not cache.k.is_cuda:
        live = _live(cache, slots)
        at = torch.where(live, slots, torch.zeros_like(slots)).long()
        res = []
        for codes, scales, out in ((cache.k, cache.k_scale, out_k), (cache.v, cache.v_scale, out_v)):
            x = dequantize_rows_e8m0(_rows(codes, at), _rows(scales, at)).to(torch.bfloat16)
            x = torch.where(live[:, None, None], x, torch.zeros_like(x))
            res.append(x if out is None else out.copy_(x))
        return res[0], res[1]
    return _ext.ext().gather_kv_fp8(*cache, slots, out_k, out_v)


def decode_attention_fp8_ref(q: torch.Tensor, cache: Fp8KV, block_table: torch.Tensor, seq_lens: torch.Tensor, scale: float) -> torch.Tensor:
    B, Hq, dim = q.shape
    pages, Hkv, P, _ = cache.k.shape
    out = torch.zeros_like(q)
    for b in range(B):
        n = max(0, min(int(seq_lens[b]), block_table.shape[1] * P))
        t = torch.arange(n, device=q.device)
        page = block_table[b, t // P].long()
        ok = (page >= 0) & (page < pages)
        slots = (page * P + t % P)[ok]
        if slots.numel() == 0:
            continue
        k = dequantize_rows_e8m0(_rows(cache.k, slots), _rows(cache.k_scale, slots)).to(q.device)
        v = dequantize_rows_e8m0(_rows(cache.v, slots), _rows(cache.v_scale, slots)).to(q.device)
        rep = Hq // Hkv
        s = torch.einsum("hd,thd->ht", q[b].float(), k.repeat_interleave(rep, 1)) * scale
        out[b] = torch.einsum("ht,thd->hd", torch.softmax(s, -1), v.repeat_interleave(rep, 1)).to(q.dtype)
    return out


def paged_decode_attention_fp8(q: torch.Tensor, cache: Fp8KV, block_table: torch.Tensor, seq_lens: torch.Tensor, scale: float | None = None) -> torch.Tensor:
    """One query token per sequence, ``q (B, Hq, 128)``, over the first ``seq_lens[b]`` tokens of its pages
    ``block_table[b]`` (int32).  GQA groups up to 16, up to 2048 sequences, pages of a multiple of 16 tokens.  A length of 0 gives zeros; lengths beyond the block table are cut to
    it; tokens of a page id outside the cache are not seen.  A value row of zeros may have any scale; the scales of the others are at
    least 2^-90 (append writes none below 2^-60).  Needs no plan and no workspace of the caller's.  After a
    wait inside the kernel that gave up, rows may be undefined: :func:`check_decode_waits` tells."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    if not q.is_cuda:
        return decode_attention_fp8_ref(q, cache, block_table, seq_lens, scale)
    return _ext.ext().paged_decode_attn_fp8(q, *cache, block_table, seq_lens, scale)


def decode_wait_error(device: torch.device) -> int:
    """0, or the code of the first wait inside :func:`paged_decode_attention_fp8` that gave up on ``device`` since the process
    started.  Waits for the current stream."""
    if device.type != "cuda":
        return 0
    with torch.cuda.device(device):
        return int(_ext.ext().kv_fp8_error())


def check_decode_waits(device: torch.device) -> None:
    """Raise if a wait inside the decode attention gave up on ``device``: its outputs are then incomplete."""
    code = decode_wait_error(device)
    if code:
        raise RuntimeError(f"decode attention over the 8-bit KV cache: a wait inside the kernel timed out (code {code}) on {device}")
