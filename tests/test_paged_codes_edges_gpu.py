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


@pytest.mark.parametrize("new,length,at", [(2, 300, 299), (3, 300, 299), (90, 300, 299), (2, 300, 7), (90, 300, 7), (1, 9000, 4321), (3, 9000, 8999),
                                           (90, 9000, 4321), (90, 9000, 8999)])
@pytest.mark.parametrize("kind,dtype", [(INT8, FP16), (E4M3, FP16), (INT8, BF16), (E4M3, BF16)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_mha_a_scale_of_nan_reaches_all_rows_that_see_it(which, kind, dtype, new, length, at):
    """That of a key as that of a value, every dim, also where a tile is cut and its parts are added up; the rows in front do not change."""
    batch = CodesBatch([new], [length], 4, 2, 128, 16, dtype, kind)
    clean = _mha(batch, max_tokens=new, max_len=length)
    getattr(batch, which + "_scale")[batch.pages[0, at // 16].long(), :, at % 16] = math.nan
    out = _mha(batch, max_tokens=new, max_len=length)
    blind = max(0, at - (length - new))                       # rows in front of that position
    assert torch.equal(out[:blind], clean[:blind]) and not torch.isnan(clean).any()
    assert torch.isnan(out[blind:]).all()


@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 64), (8, 8, 128)])
@pytest.mark.parametrize("max_len", [3000, 100])
def test_mha_rows_beside_a_chunk_are_as_good_as_alone(kind, heads, kv_heads, head_dim, max_len):
    """bf16, sequences of few tokens beside a chunk.  Where they are many and long enough (by max_len) they go to the kernel of few rows, whose
    weights are fp16: the tolerance is that of a call of their own.  Otherwise they go to the chunk's tiles, and so is the tolerance."""
    new, lens = [1] * 20 + [150] + [2] + [1] * 10, [100 + 41 * i for i in range(20)] + [700, 900] + [1 + 300 * i for i in range(10)]
    batch = CodesBatch(new, lens, heads, kv_heads, head_dim, 32, BF16, kind)
    batch.poison()
    got = _mha(batch, max_tokens=150, max_len=max_len)
    assert ((len(new) - 1) * kv_heads * (max_len // 128 + 1) >= 1024) == (max_len == 3000)
    ref, tight = attend_codes64(batch)
    wide = attend_codes64(batch, tiles=True)[1]
    tol = tight.clone() if max_len == 3000 else wide
    tol[20:170] = wide[20:170]
    _within(got, ref, tol)
