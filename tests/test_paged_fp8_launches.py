"""Launches that the counter books for decode over the 8-bit cache: one where a CTA takes a whole (sequence, kv head), two where
a merge follows, none where there is nothing to launch."""

import pytest
import torch

from axrl_b200.ops import _ext
from axrl_b200.ops import paged_fp8 as pf


def _call(B, hq, hkv, P, width):
    cache = pf.layer_cache(*pf.empty_cache((), 40, hkv, P, "cuda"))
    q = torch.zeros(B, hq, 128, dtype=torch.bfloat16, device="cuda")
    bt, lens = torch.zeros(B, width, dtype=torch.int32, device="cuda"), torch.ones(B, dtype=torch.int32, device="cuda")
    return lambda: pf.paged_decode_attention_fp8(q, cache, bt, lens)


def _launched(fn):
    from torch.profiler import ProfilerActivity, profile

    fn()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        fn()
        torch.cuda.synchronize()
    return sum(e.count for e in p.key_averages() if "decode_k" in e.key or "merge_k" in e.key)


@pytest.mark.gpu
@pytest.mark.parametrize("B,hq,hkv,P,width", [(1, 32, 8, 64, 8), (1, 32, 8, 64, 9), (18, 8, 8, 16, 32), (19, 8, 8, 16, 32), (4, 16, 1, 128, 4),
                                              (4, 16, 1, 128, 5), (0, 8, 8, 16, 4), (3, 8, 8, 16, 0)])
def test_counted_launches_are_the_launched_ones(B, hq, hkv, P, width):
    fn = _call(B, hq, hkv, P, width)
    was = _ext._COUNT["enabled"]
    before = _ext.count_launches(True)
    fn()
    booked = _ext.count_launches(was) - before
    _ext._COUNT["launches"] = before
    assert booked == _launched(fn)
