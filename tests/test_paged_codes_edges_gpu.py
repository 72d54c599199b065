"""Attention over a cache of 8-bit codes whose scales are extreme, and what the results are promised to be there."""
import math

import pytest
import torch

from codes_util import CODES, CodesBatch, attend_codes64

pytestmark = pytest.mark.gpu

FP16, BF16, INT8, E4M3 = torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn


def _paged():
    from eet_b200 import paged
    return paged


def _mha(batch, **given):
    given = {w: (x.cuda() if torch.is_tensor(x) else x) for w, x in given.items()}
    return _paged().paged_mha(batch.q.cuda(), *batch.gpu(), **batch.scales(), **given)


def _within(got, ref, tol):
    off = (got.double().cpu() - ref).abs() - tol
    assert not torch.isnan(off).any()
    assert (off <= 0).all(), f"{off.max().item():.3g} beyond the tolerance at {int(off.argmax())}"


@pytest.mark.parametrize("down", [0, 40, 60, 80, 95])
@pytest.mark.parametrize("new,heads,kv_heads", [([1, 1], 8, 2), ([3, 1], 16, 4), ([40, 1], 8, 2)])
@pytest.mark.parametrize("kind", CODES)
def test_mha_of_small_values(kind, new, heads, kv_heads, down):
    """The result is linear in the values: with all their scales 2^down smaller it is 2^down smaller, and as good.  (bf16 reaches as far; the
    numbers are those of the batch itself, so the tolerance is, too.)"""
    batch = CodesBatch(new, [900, 40], heads, kv_heads, 128, 16, BF16, kind)
    ref, tol = attend_codes64(batch, tiles=max(new) > 8)
    batch.v_scale *= 2.0 ** -down
    _within(_mha(batch, max_tokens=max(new)).double() * 2.0 ** down, ref, tol)
