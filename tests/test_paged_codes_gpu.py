"""A paged cache of 8-bit codes against a plain restatement in 64 bits (codes_util), through the Python calls."""
import math

import pytest
import torch

from codes_util import CODES, MOST, CodesBatch, attend_codes64, half_step, quantize64
from paged_util import HALF_STEP, Batch, rotate64, rotate_tolerance

pytestmark = pytest.mark.gpu

FP16, BF16, INT8, E4M3 = torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn


def _paged():
    from eet_b200 import paged
    return paged


def _status():
    from eet_b200 import _lib
    return _lib.device_status()


def _within(got, ref, tol, what=""):
    off = (got.double().cpu() - ref).abs() - tol
    assert not torch.isnan(off).any(), what
    assert (off <= 0).all(), f"{what} {off.max().item():.3g} beyond the tolerance at {int(off.argmax())}"


def _slots(batch, b, t):
    p = torch.arange(batch.lens_list[b] - t, batch.lens_list[b])
    return batch.pages[b].long()[p // batch.page], p % batch.page


# ---------------------------------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("new,lens,page", [
    ([1], [1], 16), ([1, 1, 1], [5, 16, 17], 16), ([3, 0, 20, 1], [3, 40, 33, 64], 32), ([130], [257], 64), ([0, 0], [3, 0], 16),
    ([5, 2], [300, 2], 256), ([1] * 300, [1 + i % 50 for i in range(300)], 16)])
@pytest.mark.parametrize("dtype,head_dim,interleaved,rotary_dim", [(FP16, 128, False, 128), (BF16, 64, True, 32), (BF16, 128, False, 64),
                                                                   (FP16, 64, False, 0)])
@pytest.mark.parametrize("kind", CODES)
def test_store(new, lens, page, dtype, head_dim, interleaved, rotary_dim, kind):
    batch = CodesBatch(new, lens, 6, 2, head_dim, page, dtype, kind, behind=2)
    kc, vc, pages, starts, n = batch.gpu()
    scales = batch.scales()
    freqs = _paged().rotary_frequencies(rotary_dim, device="cpu")[0] if rotary_dim else None
    out = torch.full_like(batch.q, 7.0).cuda()
    got = _paged().paged_store(batch.k.cuda(), batch.v.cuda(), kc, vc, pages, starts, n, q=batch.q.cuda(), interleaved=interleaved,
                               freqs=None if freqs is None else freqs.cuda(), q_out=out, **scales)
    assert got is out
    total, positions = sum(new), batch.positions()
    k64, k_off = batch.k[:total].double(), torch.zeros(total, 2, head_dim, dtype=torch.float64)
    q64, q_off = batch.q[:total].double(), torch.zeros_like(batch.q[:total], dtype=torch.float64)
    if rotary_dim:
        q64, k64 = (rotate64(x[:total], positions, freqs, interleaved) for x in (batch.q, batch.k))
        q_off, k_off = (rotate_tolerance(x[:total], freqs, interleaved, dtype) for x in (batch.q, batch.k))
        q_off += HALF_STEP[dtype] * q64.abs() + 2.0 ** -25
    _within(out[:total], q64, q_off)
    assert (out[total:] == 7.0).all(), "rows behind the last sequence"
    kc, vc, ks, vs = kc.cpu(), vc.cpu(), scales["k_scale"].cpu(), scales["v_scale"].cpu()
    v_codes, v_scale = quantize64(batch.v[:total], kind)
    at = 0
    for b, t in enumerate(new):
        page_of, slot = _slots(batch, b, t)
        rows = slice(at, at + t)
        # v goes in as it is: its scale and codes are known to the bit
        assert torch.equal(vs[page_of, :, slot], v_scale[rows])
        assert torch.equal(vc.view(torch.uint8)[page_of, :, slot], v_codes[rows].view(torch.uint8))
        # k: the scale is that of the rotated values, which are off by k_off; the codes stand for them to half a step of the scale used
        scale = ks[page_of, :, slot]
        if t:
            top = k64[rows].abs().amax(-1)
            assert ((scale.double() * MOST[kind] - top).abs() <= k_off[rows].amax(-1) + 2.0 ** -23 * top).all()
        value = kc.float()[page_of, :, slot].double() * scale.double()[..., None]
        _within(value, k64[rows], half_step(k64[rows], scale, kind) * (1 + 2.0 ** -20) + 2 * k_off[rows])
        for held, was in ((kc, batch.k_cache), (vc, batch.v_cache), (ks, batch.k_scale), (vs, batch.v_scale)):
            held.view(torch.uint8 if held.dtype in CODES else held.dtype)[page_of, :, slot] = \
                was.view(torch.uint8 if was.dtype in CODES else was.dtype)[page_of, :, slot]
        at += t
    # every other slot holds what it held
    assert torch.equal(kc.view(torch.uint8), batch.k_cache.view(torch.uint8)) and torch.equal(ks, batch.k_scale)
    assert torch.equal(vc.view(torch.uint8), batch.v_cache.view(torch.uint8)) and torch.equal(vs, batch.v_scale)
    assert _status() == 0


@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_store_of_rows_on_the_border_of_two_codes(kind, dtype):
    """Small whole numbers under a scale made from one of them: many quotients lie on a border, and must go to the even code, many beside it."""
    gen = torch.Generator().manual_seed(3)
    batch = CodesBatch([400], [400], 2, 2, 128, 16, dtype, kind)
    v = torch.randint(-254, 255, (400, 2, 128), generator=gen).float()
    v[:, :, 5] = 254.0 if kind == INT8 else 448.0
    v[:100] *= 2.0 ** -12
    v[100:150, 1] = 0.0
    v[150:200] = torch.randint(-3, 4, (50, 2, 128), generator=gen).float() * 2.0 ** -24
    batch.v = v.to(dtype)
    kc, vc, *table = batch.gpu()
    scales = batch.scales()
    _paged().paged_store(batch.v.cuda(), batch.v.cuda(), kc, vc, *table, **scales)
    codes, scale = quantize64(batch.v, kind)
    page_of, slot = _slots(batch, 0, 400)
    for cache, s in ((kc, scales["k_scale"]), (vc, scales["v_scale"])):
        assert torch.equal(s.cpu()[page_of, :, slot], scale)
        assert torch.equal(cache.cpu().view(torch.uint8)[page_of, :, slot] & 127, codes.view(torch.uint8) & 127)
        assert torch.equal(cache.cpu().float()[page_of, :, slot], codes.float())


@pytest.mark.parametrize("kind", CODES)
def test_store_of_what_has_no_codes(kind):
    """A row with a NaN or an infinity reads back as NaN, its neighbours are kept; the largest and smallest values are, too."""
    batch = CodesBatch([7], [7], 2, 2, 128, 16, BF16, kind)
    v = batch.v.clone()
    v[0, 0, 3], v[1, 1, 127], v[2, 0, 0] = math.nan, math.inf, -math.inf
    v[3], v[4] = 3.3e38, 1e-38
    v[5, 0, 1:] = 0.0
    kc, vc, *table = batch.gpu()
    scales = batch.scales()
    _paged().paged_store(v.cuda(), v.cuda(), kc, vc, *table, **scales)
    k, back = _paged().paged_load(kc, vc, *table, 7, dtype=BF16, **scales)
    assert torch.equal(k.isnan(), back.isnan())
    lost = torch.zeros(7, 2, dtype=torch.bool)
    lost[0, 0] = lost[1, 1] = lost[2, 0] = True
    assert back.isnan().cpu().all(-1).equal(lost) and back.isnan().cpu().any(-1).equal(lost)
    ok = ~lost
    scale = scales["v_scale"].cpu()[_slots(batch, 0, 7)[0], :, _slots(batch, 0, 7)[1]]
    tol = half_step(v, scale, kind) + 2.0 ** -8 * v.double().abs()
    _within(back.cpu()[ok], v.double()[ok], tol[ok] * (1 + 2.0 ** -20))


# ---------------------------------------------------------------------------------------------------------------------
# reading back
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("new,lens,page", [
    ([1], [1], 16), ([300], [300], 16), ([3, 0, 20, 1], [3, 40, 33, 64], 32), ([7, 600, 0, 1], [7, 601, 5, 900], 64), ([0, 0], [3, 0], 16),
    ([255, 2], [700, 2], 256), ([2] * 100, [2 + i % 50 for i in range(100)], 128)])
@pytest.mark.parametrize("kind", CODES + (None,))
@pytest.mark.parametrize("dtype,head_dim,kv_heads", [(FP16, 128, 2), (BF16, 64, 3)])
def test_load(new, lens, page, kind, dtype, head_dim, kv_heads):
    batch = Batch(new, lens, kv_heads, kv_heads, head_dim, page, dtype) if kind is None else \
        CodesBatch(new, lens, kv_heads, kv_heads, head_dim, page, dtype, kind)
    total = sum(new)
    cache = [t.cuda() for t in (batch.k_cache, batch.v_cache, batch.pages, batch.starts, batch.lens)]
    scales = {} if kind is None else batch.scales()
    outs = [torch.full((total + 2, kv_heads, head_dim), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
    got = _paged().paged_load(*cache, k_out=outs[0], v_out=outs[1], **scales)
    assert got[0] is outs[0] and got[1] is outs[1]
    for w, y in zip("kv", outs):
        at = 0
        for b, t in enumerate(new):
            if kind is None:
                want = batch.history(getattr(batch, w + "_cache"), b)[lens[b] - t:]
                assert torch.equal(y[at:at + t].cpu(), want)
            else:
                want = batch.values(w, b)[lens[b] - t:]
                # (code times scale in fp32 and one rounding)
                _within(y[at:at + t], want, (HALF_STEP[dtype] + 2.0 ** -23) * want.abs() + 2.0 ** -25)
            at += t
        assert (y[total:] == 7.0).all(), "rows behind the last sequence"
    fresh = _paged().paged_load(*cache, total, dtype=dtype, **scales)
    assert all(torch.equal(x, y[:total]) for x, y in zip(fresh, outs))
    assert _status() == 0


def test_load_of_missing_pages_and_positions():
    batch = CodesBatch([4, 6], [40, 3], 2, 2)
    batch.pages[0, 2] = 10 ** 6
    cache, scales = batch.gpu(), batch.scales()
    out = [torch.full((10, 2, 128), 7.0, dtype=FP16, device="cuda") for _ in range(2)]
    _paged().paged_load(*cache, k_out=out[0], v_out=out[1], **scales)
    assert _status() == 6
    for w, y in zip("kv", out):
        assert (y[:4] == 0).all(), "a page outside the cache"
        assert (y[4:7] == 7.0).all(), "in front of the first position"
        _within(y[7:], batch.values(w, 1), 2.0 ** -11 * batch.values(w, 1).abs() * 1.01 + 2.0 ** -25)


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------
def _check(batch, what="", tiles=False, **options):
    given = {w: (x.cuda() if torch.is_tensor(x) else x) for w, x in options.items()}
    total = sum(batch.new)
    out = torch.full_like(batch.q, 7.0).cuda()
    got = _paged().paged_mha(batch.q.cuda(), *batch.gpu(), out=out, **batch.scales(), **given)
    assert got is out
    plain = {w: x for w, x in options.items() if w in ("scale", "window", "first_key", "alibi_slopes")}
    ref, tol = attend_codes64(batch, tiles=tiles, **plain)
    _within(out[:total], ref, tol, what)
    assert (out[total:] == 7.0).all(), "rows behind the last sequence"
    assert _status() == 0


ROWS = [([1], [1]), ([1], [300]), ([1, 1, 1], [5, 128, 129]), ([1] * 40, [1 + 37 * i % 400 for i in range(40)]), ([2, 0, 1], [2, 50, 1000]),
        ([1], [5000]), ([4, 3], [700, 1300])]


@pytest.mark.parametrize("new,lens", ROWS)
@pytest.mark.parametrize("heads,kv_heads,head_dim,page", [(4, 4, 128, 16), (8, 2, 128, 64), (8, 1, 64, 16), (16, 1, 128, 32), (6, 2, 64, 256)])
@pytest.mark.parametrize("kind,dtype", [(INT8, FP16), (INT8, BF16), (E4M3, FP16), (E4M3, BF16)])
def test_mha_few_rows(new, lens, heads, kv_heads, head_dim, page, kind, dtype):
    batch = CodesBatch(new, lens, heads, kv_heads, head_dim, page, dtype, kind, behind=1)
    batch.poison()
    _check(batch, max_tokens=max(new), tiles=max(new) * heads // kv_heads > 16)


@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("options", [dict(window=1), dict(window=100), dict(first=True), dict(alibi=True), dict(window=33, first=True, alibi=True),
                                     dict(scale=0.3), dict(scale=-0.1), dict(scale=0.0)])
def test_mha_few_rows_options(kind, options):
    lens = [3, 200, 517, 1]
    batch = CodesBatch([1, 2, 1, 1], lens, 8, 4, 128, 16, FP16, kind)
    batch.poison()
    options = dict(options)
    if options.pop("first", False):
        options["first_key"] = torch.tensor([3, 150, 0, 1], dtype=torch.int32)      # the first and last sequences see nothing
    if options.pop("alibi", False):
        options["alibi_slopes"] = torch.tensor([2.0 ** -i for i in range(1, 9)])
    _check(batch, max_tokens=2, **options)


TILES = [([17], [17]), ([200], [300]), ([129], [2000]), ([300, 260], [300, 700]), ([40, 0, 70], [40, 5, 1000]), ([513], [1300])]


@pytest.mark.parametrize("new,lens", TILES)
@pytest.mark.parametrize("heads,kv_heads,head_dim,page", [(4, 4, 128, 16), (8, 2, 128, 64), (8, 1, 64, 16), (32, 1, 128, 32), (6, 2, 64, 256),
                                                          (7, 1, 128, 128)])
@pytest.mark.parametrize("kind,dtype", [(INT8, FP16), (INT8, BF16), (E4M3, FP16), (E4M3, BF16)])
def test_mha_tiles(new, lens, heads, kv_heads, head_dim, page, kind, dtype):
    batch = CodesBatch(new, lens, heads, kv_heads, head_dim, page, dtype, kind, behind=1)
    batch.poison()
    _check(batch, max_tokens=max(new), tiles=True)


@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (64, 1), (128, 1)])
@pytest.mark.parametrize("options", [dict(window=1), dict(window=100), dict(first=True), dict(alibi=True), dict(window=33, first=True, alibi=True),
                                     dict(scale=0.3), dict(scale=-0.1), dict(scale=0.0)])
def test_mha_tiles_options(kind, heads, kv_heads, options):
    lens = [30, 200, 617, 50]
    batch = CodesBatch([30, 120, 200, 1], lens, heads, kv_heads, 128, 16, FP16, kind)
    batch.poison()
    options = dict(options)
    if options.pop("first", False):
        options["first_key"] = torch.tensor([30, 150, 0, 49], dtype=torch.int32)     # the first sequence sees nothing
    if options.pop("alibi", False):
        options["alibi_slopes"] = torch.tensor([2.0 ** -(i % 8 + 1) for i in range(heads)])
    _check(batch, max_tokens=200, tiles=True, **options)


@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("dtype,heads,kv_heads,head_dim,page", [(FP16, 8, 8, 128, 16), (BF16, 8, 2, 64, 64), (FP16, 32, 4, 128, 32)])
@pytest.mark.parametrize("alibi", [False, True])
def test_mha_a_chunk_beside_single_tokens(kind, dtype, heads, kv_heads, head_dim, page, alibi):
    """Both kinds of tiles in one call."""
    new, lens = [1] * 20 + [150] + [2] + [1] * 10, [100 + 41 * i for i in range(20)] + [700, 900] + [1 + 300 * i for i in range(10)]
    batch = CodesBatch(new, lens, heads, kv_heads, head_dim, page, dtype, kind, behind=3)
    batch.poison()
    more = dict(alibi_slopes=torch.tensor([2.0 ** -(i % 8 + 1) for i in range(heads)])) if alibi else {}
    _check(batch, max_tokens=150, max_len=3000, tiles=True, **more)


@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("spread", [0.0, 6.0, 13.0])
def test_mha_scales_of_very_different_sizes(kind, spread):
    """Rows of the cache that differ by up to 2^26 in size; q so small that all keys count."""
    batch = CodesBatch([1, 1], [900, 40], 4, 4, 128, 16, BF16, kind, spread=spread, q_scale=0.01)
    _check(batch, max_tokens=1)


@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("spread", [6.0, 13.0])
def test_mha_tiles_scales_of_very_different_sizes(kind, dtype, spread):
    batch = CodesBatch([150, 40], [900, 40], 4, 2, 128, 16, dtype, kind, spread=spread, q_scale=0.01)
    _check(batch, max_tokens=150, tiles=True)


@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("least", [1e-39, 1e-37, 1e-20, 0.0])
def test_mha_scales_next_to_nothing_in_the_newest_blocks(kind, dtype, new, least):
    """Positions 0 to 39 weigh, what is behind them hardly does or not at all."""
    batch = CodesBatch([new], [300], 4, 2, 128, 16, dtype, kind)
    batch.v_scale[:] = least
    for position in range(40):
        batch.v_scale[batch.pages[0, position // 16], :, position % 16] = 0.01
    total = sum(batch.new)
    out = _paged().paged_mha(batch.q.cuda(), *batch.gpu(), **batch.scales(), max_tokens=new)
    batch.v_scale.clamp_(min=1e-30)       # (the tolerance divides by it; 1e-30 times 448 is nothing beside the step of the result)
    ref, tol = attend_codes64(batch, tiles=new > 8)
    _within(out[:total], ref, tol)


@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("new", [2, 3, 90])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_mha_scales_that_are_not_finite_reach_the_rows_that_see_them(kind, new, bad):
    """(Such a scale stands for a row of k or v that was not finite.)"""
    batch = CodesBatch([new], [300], 4, 2, 128, 16, FP16, kind)
    clean = _paged().paged_mha(batch.q.cuda(), *batch.gpu(), **batch.scales(), max_tokens=new)
    page, slot = int(batch.gpu()[2][0, 299 // 16]), 299 % 16
    for which in ("k", "v"):
        scales = {w: x.clone() for w, x in batch.scales().items()}
        scales[which + "_scale"][page, :, slot] = bad
        out = _paged().paged_mha(batch.q.cuda(), *batch.gpu(), **scales, max_tokens=new)
        assert torch.equal(out[:-1], clean[:-1]), which
        assert not torch.isfinite(out[-1]).any() or which == "k" or bad == math.inf


def test_mha_is_the_same_whatever_the_hints():
    batch = CodesBatch([1, 3, 1], [700, 1500, 90], 8, 4, 128, 32)
    runs = [_paged().paged_mha(batch.q.cuda(), *batch.gpu(), **batch.scales(), **hint)
            for hint in (dict(max_tokens=3, max_len=1500), dict(max_tokens=3, max_len=1500), dict(), dict(max_tokens=1, max_len=1))]
    assert torch.equal(runs[0], runs[1])
    ref, tol = attend_codes64(batch)
    for r in runs:
        _within(r, ref, tol)


# ---------------------------------------------------------------------------------------------------------------------
# refusals, pages outside the cache, streams, graphs
# ---------------------------------------------------------------------------------------------------------------------
def test_refuses():
    paged = _paged()
    batch = CodesBatch([1, 2], [20, 40], 4, 2)
    kc, vc, *table = batch.gpu()
    scales = batch.scales()
    q, k, v = batch.q.cuda(), batch.k.cuda(), batch.v.cuda()
    ks, vs = scales["k_scale"], scales["v_scale"]
    for bad in (dict(k_scale=ks), dict(v_scale=vs), dict(k_scale=ks.half(), v_scale=vs), dict(k_scale=ks[1:], v_scale=vs),
                dict(k_scale=ks.cpu(), v_scale=vs), dict(k_scale=ks, v_scale=vs.transpose(1, 2).contiguous().transpose(1, 2)),
                dict(k_scale=ks[..., 0], v_scale=vs[..., 0])):
        with pytest.raises(RuntimeError):
            paged.paged_mha(q, kc, vc, *table, **bad)
        with pytest.raises(RuntimeError):
            paged.paged_store(k, v, kc, vc, *table, **bad)
        with pytest.raises(RuntimeError):
            paged.paged_load(kc, vc, *table, 3, **bad)
    for call in (lambda **s: paged.paged_mha(q, kc, vc, *table, **s), lambda **s: paged.paged_store(k, v, kc, vc, *table, **s),
                 lambda **s: paged.paged_load(kc, vc, *table, 3, **s)):
        with pytest.raises(RuntimeError):
            call()                                                              # codes without scales
    with pytest.raises(RuntimeError, match="scales belong"):
        paged.paged_mha(q, kc.half(), vc.half(), *table, **scales)             # scales without codes
    with pytest.raises(RuntimeError, match="scales belong"):
        paged.paged_load(kc.half(), vc.half(), *table, 3, **scales)
    with pytest.raises(RuntimeError):
        paged.paged_mha(q, kc, vc.view(E4M3), *table, **scales)                # two kinds of codes
    with pytest.raises(RuntimeError):
        paged.paged_load(kc, vc, *table, **scales)                             # how many rows?
    with pytest.raises(RuntimeError, match="read back as"):
        paged.paged_load(kc, vc, *table, 3, dtype=torch.float32, **scales)
    with pytest.raises(RuntimeError):
        paged.paged_load(kc, vc, *table, k_out=k, v_out=v[1:], **scales)
    wide = torch.zeros(kc.shape[0], 2, 16, 136, dtype=INT8, device="cuda")[..., :128]   # rows 136 bytes apart
    with pytest.raises(RuntimeError, match="multiples of 16"):
        paged.paged_mha(q, wide, wide, *table, **scales)


@pytest.mark.parametrize("new,most", [([1, 2], 2), ([30, 1], 30)])
@pytest.mark.parametrize("kind", CODES)
def test_mha_over_missing_pages(new, most, kind):
    """Keys of a page outside the cache count as zeros, and the status says so."""
    batch = CodesBatch(new, [70, 45], 4, 2, 128, 16, FP16, kind)
    batch.pages[0, 1] = 10 ** 6
    batch.pages[1, 0] = -7
    got = _paged().paged_mha(batch.q.cuda(), *batch.gpu(), max_tokens=most, **batch.scales())
    assert _status() == 6
    spare = batch.unused[0]
    for cache, scale in ((batch.k_cache, batch.k_scale), (batch.v_cache, batch.v_scale)):
        cache.view(torch.uint8)[spare] = 0
        scale[spare] = 1.0
    batch.pages[0, 1] = batch.pages[1, 0] = spare
    ref, tol = attend_codes64(batch, tiles=most > 8)
    _within(got, ref, tol)


def test_mha_of_strided_caches():
    """[page][slot][head][dim] codes and scales that are views of larger tensors."""
    batch = CodesBatch([1, 20, 1], [300, 50, 77], 8, 4, 64, 32, BF16, INT8)
    total = batch.k_cache.shape[0]
    kc, vc = (c.transpose(1, 2).contiguous().cuda().transpose(1, 2) for c in (batch.k_cache, batch.v_cache))
    both = torch.stack((batch.k_scale, batch.v_scale), 1).cuda()               # [page][k, v][head][slot]
    for most in (1, 20):
        got = _paged().paged_mha(batch.q.cuda(), kc, vc, *(t.cuda() for t in (batch.pages, batch.starts, batch.lens)), max_tokens=most,
                                 k_scale=both[:, 0], v_scale=both[:, 1])
        ref, tol = attend_codes64(batch, tiles=True)
        _within(got, ref, tol)
    k, v = _paged().paged_load(kc, vc, *(t.cuda() for t in (batch.pages, batch.starts, batch.lens)), 22, dtype=BF16, k_scale=both[:, 0],
                               v_scale=both[:, 1])
    assert total and torch.equal(k, _paged().paged_load(*batch.gpu(), 22, dtype=BF16, **batch.scales())[0])


def test_empty_calls():
    batch = CodesBatch([1], [20], 4, 2)
    kc, vc, pages, starts, lens = batch.gpu()
    scales = batch.scales()
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert _paged().paged_mha(batch.q[:0].cuda(), kc, vc, pages[:0], none, lens[:0], **scales).shape == (0, 4, 128)
    assert _paged().paged_load(kc, vc, pages[:0], none, lens[:0], 0, **scales)[0].shape == (0, 2, 128)
    zero = CodesBatch([0, 0], [0, 5], 4, 2)
    for most in (1, 40):
        out = torch.full((3, 4, 128), 7.0, dtype=FP16, device="cuda")
        _paged().paged_mha(out, *zero.gpu(), out=out, max_tokens=most, **zero.scales())
        assert (out == 7.0).all()


@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("new,most", [([1] * 6, 1), ([3, 1, 2, 1, 1, 2], 3), ([90, 1, 1, 1, 1, 1], 90)])
def test_a_captured_call_serves_other_lengths(kind, new, most):
    lens = [200, 7, 3000, 90, 1, 1000]
    batch = CodesBatch(new, [max(a, b) for a, b in zip(lens, new)], 8, 2, 128, 16, FP16, kind)
    cache, scales, q = batch.gpu(), batch.scales(), batch.q.cuda()
    run = lambda: _paged().paged_mha(q, *cache, max_tokens=most, max_len=3000, **scales)  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for other in (batch.lens_list, [max(n, x // 2) for n, x in zip(new, batch.lens_list)], list(new)):
        batch.lens_list = list(other)
        cache[4].copy_(torch.tensor(other, dtype=torch.int32))
        out.fill_(9.0)
        graph.replay()
        ref, tol = attend_codes64(batch, tiles=True)
        _within(out, ref, tol, str(other))
    assert _status() == 0


def test_calls_behind_one_another_without_a_pause():
    """Append and attention in turn, in place, many times over and captured: what one writes the next one reads, and the programmatic launches
    may overlap only as far as that allows."""
    paged = _paged()
    for new, most in (([1] * 5, 1), ([100, 1, 1, 1, 1], 100), ([2, 3, 1, 0, 4], 4)):
        batch = CodesBatch(new, [700 + 3 * n for n in new], 8, 2, 128, 16, FP16, INT8)
        freqs = paged.rotary_frequencies(128)[0]
        q, k, v = (t.cuda() for t in (batch.q, batch.k, batch.v))

        def steps(cache, scales, pause):
            out, x = [], q
            for i in range(12):
                turned = paged.paged_store((k * (1 + i)).half(), (v - i).half(), *cache, q=x, freqs=freqs, **scales)
                if pause:
                    torch.cuda.synchronize()
                x = paged.paged_mha(turned, *cache, max_tokens=most, **scales) * 3
                if pause:
                    torch.cuda.synchronize()
                out.append(x)
            return torch.stack(out)

        want = steps(batch.gpu(), batch.scales(), True)
        cache, scales = batch.gpu(), batch.scales()
        assert torch.equal(steps(cache, scales, False), want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = steps(cache, scales, False)
        for t, s in zip(cache, batch.gpu()):
            t.copy_(s)
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    assert _status() == 0


def test_two_streams_at_once():
    batches = [CodesBatch(new, lens, 8, 2, seed=i) for i, (new, lens) in enumerate((([1] * 9, [900] * 9), ([120, 1], [500, 3000])))]
    inputs = [(b.q.cuda(), b.gpu(), b.scales()) for b in batches]
    most = [1, 120]
    want = [_paged().paged_mha(q, *c, max_tokens=m, **s) for (q, c, s), m in zip(inputs, most)]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                q, c, s = inputs[i]
                got[i].append(_paged().paged_mha(q, *c, max_tokens=most[i], **s))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


# ---------------------------------------------------------------------------------------------------------------------
# serving: prompt and decode steps of the block, to the next token
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("kv_heads", [2, 1])
def test_serving_to_the_next_token(kind, kv_heads):
    """PagedMmha over a cache of codes is its parts called by hand, for a prompt of chunks and steps of single tokens behind it; a captured step
    draws the tokens that the calls by hand draw."""
    from eet_b200 import EET
    paged, heads, hidden, page = _paged(), 2, 256, 16
    gen = torch.Generator().manual_seed(3)
    desc = EET.MetaDesc(FP16, 4, heads, hidden, 1, 64, 128, "silu", 128, 512, "cuda:0", False, 1e-6, True)
    make = lambda k, n: EET.quant_weights((torch.randn(k, n, generator=gen) * 0.05).half().cuda(), torch.int8, False)  # noqa: E731
    qkv_w, qkv_s = make(hidden, 128 * (heads + 2 * kv_heads))[-2:]
    out_w, out_s = make(128 * heads, hidden)[-2:]
    qkv_s, out_s = qkv_s.half(), out_s.half()
    norm = torch.ones(hidden, dtype=FP16, device="cuda")
    head = (torch.randn(hidden, 1000, generator=gen) * 0.3).half().cuda()
    block = paged.PagedMmha(desc, qkv_w, qkv_s, out_w, out_s, norm, kv_head_num=kv_heads)
    freqs, _ = paged.rotary_frequencies(128)

    def cache():
        codes = [torch.zeros(24, kv_heads, page, 128, dtype=kind, device="cuda") for _ in "kv"]
        return codes, dict(k_scale=torch.zeros(24, kv_heads, page, device="cuda"), v_scale=torch.zeros(24, kv_heads, page, device="cuda"))

    def by_hand(x, codes, scales, table, most):
        xn = torch.empty_like(x)
        EET.check(EET.lib.eet_rmsnorm(x.data_ptr(), norm.data_ptr(), xn.data_ptr(), x.shape[0], hidden, 1e-6, EET._stream()))
        qkv = EET.gemm_w8a16(xn, qkv_w, qkv_s).view(x.shape[0], -1, 128)
        q, k, v = qkv.split((heads, kv_heads, kv_heads), 1)
        q = paged.paged_store(k, v, *codes, *table, q=q, freqs=freqs, **scales)
        ctx = paged.paged_mha(q, *codes, *table, max_tokens=most, **scales)
        return EET.gemm_w8a16(ctx.view(x.shape[0], -1), out_w, out_s, residual=x)

    pages = torch.randperm(24, generator=gen)[:16].view(2, 8).int().cuda()
    lens = torch.tensor([20, 33], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 20, 53], dtype=torch.int32, device="cuda")
    x = torch.randn(53, hidden, generator=gen).half().cuda()
    mine, other = cache(), cache()
    got, want = block(x, *mine[0], pages, starts, lens, max_tokens=33, **mine[1]).clone(), by_hand(x, *other, (pages, starts, lens), 33)
    # (the two go through the same kernels, the projections maybe with sums in another order: fp16 values of a few units)
    assert torch.allclose(got.float(), want.float(), atol=2e-2, rtol=1e-2)
    embed = torch.randn(1000, hidden, generator=gen).half().cuda()
    step = torch.arange(3, dtype=torch.int32, device="cuda")
    uniform = torch.rand(2, generator=gen).cuda()
    token = torch.tensor([5, 7], device="cuda")

    def one(token, attend):
        hidden_states = attend(embed[token])
        return EET.sample_rows((hidden_states @ head).float(), uniform, temperature=0.8, top_k=100, top_p=0.95)[0]

    def captured(token):
        return one(token, lambda y: block(y, *mine[0], pages, step, lens, max_tokens=1, max_len=128, **mine[1]))

    def hand(token):
        return one(token, lambda y: by_hand(y, *other, (pages, step, lens), 1))

    # the same cache for both from here on
    for a, b in zip((*mine[0], *mine[1].values()), (*other[0], *other[1].values())):
        b.copy_(a)
    held = token.clone()
    lens += 1
    captured(held)                      # (sizes the pooled buffers; the same rows are appended again below)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        drawn = captured(held)
    for t in range(6):
        if t:
            lens += 1
        graph.replay()
        by = hand(held)
        assert torch.equal(drawn, by), f"step {t}"
        uniform.copy_((uniform + 0.37) % 1.0)
        held.copy_(drawn)
    EET.check_device_status()
