"""Attention over a cache of 8-bit codes with work that is cut up and laid out in every way: many sequences, shares of many short pieces."""
import pytest
import torch

from codes_util import CODES, CodesBatch, attend_codes64

pytestmark = pytest.mark.gpu

FP16, BF16, INT8, E4M3 = torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn


def _paged():
    from eet_b200 import paged
    return paged


def _check(batch, tiles=True, **given):
    out = torch.full_like(batch.q, 7.0).cuda()
    got = _paged().paged_mha(batch.q.cuda(), *batch.gpu(), out=out, **batch.scales(), **given)
    ref, tol = attend_codes64(batch, tiles=tiles)
    total = sum(batch.new)
    off = (got[:total].double().cpu() - ref).abs() - tol
    assert not torch.isnan(off).any()
    assert (off <= 0).all(), f"{off.max().item():.3g} beyond the tolerance at {int(off.argmax())}"
    assert (out[total:] == 7.0).all(), "rows behind the last sequence"
    from eet_b200 import _lib
    assert _lib.device_status() == 0
    return got


@pytest.mark.parametrize("max_len", [80, 9000])                       # whole tiles, cut ones
@pytest.mark.parametrize("kind,dtype", [(INT8, FP16), (E4M3, BF16)])
@pytest.mark.parametrize("seqs", [33, 385, 450, 512, 513, 1100])
def test_tiles_of_many_sequences(seqs, kind, dtype, max_len):
    """More sequences than a warp has lanes, and than a block has threads; 32 rows a kv head, so that all of them take tiles of 128 rows."""
    gen = torch.Generator().manual_seed(seqs)
    lens = torch.randint(1, 80, (seqs,), generator=gen).tolist()
    batch = CodesBatch([1] * seqs, lens, 32, 1, 64, 16, dtype, kind, behind=2)
    batch.poison()
    first = _check(batch, max_tokens=1, max_len=max_len)
    again = _paged().paged_mha(batch.q.cuda(), *batch.gpu(), **batch.scales(), max_tokens=1, max_len=max_len)
    assert torch.equal(first[:seqs], again[:seqs])


@pytest.mark.parametrize("kind,dtype", [(INT8, BF16), (E4M3, FP16)])
@pytest.mark.parametrize("seqs", [40, 420, 700])
def test_a_chunk_beside_many_single_tokens(seqs, kind, dtype):
    """Both kinds of tiles in one call, and slots without a sequence."""
    gen = torch.Generator().manual_seed(seqs)
    lens = torch.randint(1, 300, (seqs,), generator=gen).tolist()
    new = [1] * seqs
    new[seqs // 2], lens[seqs // 2] = 70, 400
    for empty in range(3, seqs, 7):
        new[empty], lens[empty] = 0, 0
    batch = CodesBatch(new, lens, 8, 4, 64, 16, dtype, kind)
    batch.poison()
    _check(batch, max_tokens=70, max_len=4000)


@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("new,before,heads,kv_heads,head_dim", [(5, (55, 255), 32, 8, 64), (17, (20, 250), 32, 32, 128), (60, (1, 150), 16, 4, 64)])
def test_shares_of_many_pieces_of_one_block(new, before, heads, kv_heads, head_dim, kind, dtype):
    """In a piece of one block the second tile of a pair has no turn, and its warps come to the next longer piece from far ahead of the
    copies; whatever lies in shared memory then, and the scales of the sequences in front, must not be taken for its own."""
    from eet_b200 import EET
    seqs = 256 if new == 5 else 64
    gen = torch.Generator().manual_seed(new)
    lens = [new + int(n) for n in torch.randint(*before, (seqs,), generator=gen)]
    batch = CodesBatch([new] * seqs, lens, heads, kv_heads, head_dim, 16, dtype, kind)
    for b, n in enumerate(lens):                                      # those of neighbours are 2^12 apart
        batch.v_scale[batch.pages[b, :-(-n // 16)].long()] *= 2.0 ** (6 if b % 2 else -6)
    batch.poison()
    ref, tol = attend_codes64(batch, tiles=True)
    # numbers of another kernel in shared memory
    weights = EET.quant_weights((torch.randn(512, 512, generator=gen) * 0.05).half().cuda(), torch.int8, False)[-2:]
    x = (100 * torch.randn(300, 512, generator=gen)).half().cuda()
    for max_len in (max(lens), 9000):                                 # whole tiles, cut ones
        runs = []
        for _ in range(4):
            EET.gemm_w8a16(x, weights[0], weights[1].half())
            runs.append(_paged().paged_mha(batch.q.cuda(), *batch.gpu(), **batch.scales(), max_tokens=new, max_len=max_len))
        off = (runs[0].double().cpu() - ref).abs() - tol
        assert not torch.isnan(off).any()
        assert (off <= 0).all(), f"{off.max().item():.3g} beyond the tolerance at {int(off.argmax())}"
        assert all(torch.equal(r, runs[0]) for r in runs)
