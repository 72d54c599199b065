"""Serving from a paged cache against a plain restatement in 64 bits (paged_util), through the Python calls."""
import itertools
import math

import pytest
import torch

from paged_util import HALF_STEP, Batch, attend64, rotate64, rotate_tolerance

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16


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


# ---------------------------------------------------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tokens,heads,kv_heads,head_dim,rotary_dim", [
    (1, 1, 1, 128, 128), (3, 5, 2, 128, 64), (7, 32, 8, 64, 64), (130, 40, 40, 128, 32), (5, 2, 1, 256, 256), (2, 3, 1, 96, 48),
    (9, 4, 4, 16, 16), (1000, 8, 2, 128, 96)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_rotary(tokens, heads, kv_heads, head_dim, rotary_dim, interleaved, dtype):
    gen = torch.Generator().manual_seed(tokens)
    q, k = (torch.randn(tokens, h, head_dim, generator=gen).to(dtype) for h in (heads, kv_heads))
    positions = torch.randint(0, 1 << 20, (tokens,), generator=gen)
    freqs, magnitude = _paged().rotary_frequencies(rotary_dim, scaling={"type": "yarn", "factor": 4.0, "original": 4096}, device="cpu")
    got = _paged().apply_rotary(q.cuda(), k.cuda(), positions.cuda(), freqs.cuda(), interleaved=interleaved, magnitude=magnitude)
    for x, y in zip((q, k), got):
        ref = rotate64(x, positions, freqs, interleaved, magnitude)
        tol = HALF_STEP[dtype] * ref.abs() + rotate_tolerance(x, freqs, interleaved, dtype, magnitude) + 2.0 ** -25
        _within(y, ref, tol)
        assert torch.equal(y[..., rotary_dim:].cpu(), x[..., rotary_dim:])


def test_rotary_in_place_on_views_of_a_projection():
    gen = torch.Generator().manual_seed(5)
    qkv = torch.randn(33, (6 + 2 + 2) * 128, generator=gen).half().cuda()
    before = qkv.clone()
    q, k = qkv[:, :768].view(33, 6, 128), qkv[:, 768:1024].view(33, 2, 128)
    positions = torch.arange(100, 133).cuda()
    freqs, _ = _paged().rotary_frequencies(128)
    fresh = _paged().apply_rotary(q, k, positions, freqs)
    out = _paged().apply_rotary(q, k, positions, freqs, q_out=q, k_out=k)
    assert out[0] is q and out[1] is k
    assert torch.equal(q, fresh[0]) and torch.equal(k, fresh[1])
    assert torch.equal(qkv[:, 1024:], before[:, 1024:])


def test_rotary_of_one_of_the_two_and_of_nothing():
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(4, 3, 64, generator=gen).half().cuda()
    positions = torch.tensor([0, 1, -5, 2 ** 30]).cuda()
    freqs, _ = _paged().rotary_frequencies(64)
    a, none = _paged().apply_rotary(x, None, positions, freqs)
    assert none is None
    none, b = _paged().apply_rotary(None, x, positions, freqs)
    assert none is None and torch.equal(a, b)
    ref = rotate64(x.cpu(), positions.cpu(), freqs.cpu(), False)
    _within(a, ref, 2.0 ** -11 * ref.abs() + rotate_tolerance(x.cpu(), freqs.cpu(), False, FP16) + 2.0 ** -25)
    empty = _paged().apply_rotary(x[:0], x[:0], positions[:0], freqs)
    assert empty[0].shape == (0, 3, 64)


def test_rotary_refuses():
    paged = _paged()
    x = torch.zeros(4, 3, 64, dtype=FP16, device="cuda")
    positions = torch.zeros(4, dtype=torch.int64, device="cuda")
    freqs, _ = paged.rotary_frequencies(64)
    for bad in (dict(positions=positions.int()), dict(positions=positions[:3]), dict(positions=positions.cpu()), dict(freqs=freqs.float()),
                dict(k=x.bfloat16()), dict(k=x[:3]), dict(q_out=x[:, :2]), dict(k=x.transpose(1, 2)), dict(k_out=x.float()),
                dict(freqs=torch.zeros(40, dtype=torch.float64, device="cuda")),
                dict(q=torch.zeros(4, 3, 65, dtype=FP16, device="cuda")[..., :64]),
                dict(q=torch.zeros(800, dtype=FP16, device="cuda")[1:769].view(4, 3, 64))):
        args = dict(q=x, k=x, positions=positions, freqs=freqs)
        args.update(bad)
        with pytest.raises(RuntimeError):
            paged.apply_rotary(args.pop("q"), args.pop("k"), args.pop("positions"), args.pop("freqs"), **args)


# ---------------------------------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------------------------------
def _gpu(batch):
    return [t.cuda() for t in (batch.k_cache, batch.v_cache, batch.pages, batch.starts, batch.lens)]


@pytest.mark.parametrize("new,lens,page", [
    ([1], [1], 16), ([1, 1, 1], [5, 16, 17], 16), ([3, 0, 20, 1], [3, 40, 33, 64], 32), ([130], [257], 64), ([0, 0], [3, 0], 16),
    ([5, 2], [300, 2], 256), ([1] * 300, [1 + i % 50 for i in range(300)], 16)])
@pytest.mark.parametrize("dtype,head_dim,interleaved,rotary_dim", [(FP16, 128, False, 128), (BF16, 64, True, 32), (FP16, 64, False, 0)])
def test_store(new, lens, page, dtype, head_dim, interleaved, rotary_dim):
    batch = Batch(new, lens, 6, 2, head_dim, page, dtype, behind=2)
    kc, vc, pages, starts, n = _gpu(batch)
    freqs = _paged().rotary_frequencies(rotary_dim, device="cpu")[0] if rotary_dim else None
    out = torch.full_like(batch.q, 7.0).cuda()
    got = _paged().paged_store(batch.k.cuda(), batch.v.cuda(), kc, vc, pages, starts, n, q=batch.q.cuda(), interleaved=interleaved,
                               freqs=None if freqs is None else freqs.cuda(), q_out=out)
    assert got is out
    total, positions = sum(new), batch.positions()
    if rotary_dim:
        q64, k64 = (rotate64(x[:total], positions, freqs, interleaved) for x in (batch.q, batch.k))
        tols = [HALF_STEP[dtype] * y.abs() + rotate_tolerance(x[:total], freqs, interleaved, dtype) + 2.0 ** -25
                for x, y in ((batch.q, q64), (batch.k, k64))]
    else:
        q64, k64 = batch.q[:total].double(), batch.k[:total].double()
        tols = [torch.zeros_like(q64), torch.zeros_like(k64)]
    _within(out[:total], q64, tols[0])
    assert (out[total:] == 7.0).all(), "rows behind the last sequence"
    # every slot of the new tokens holds its row, every other slot what it held
    kc, vc = kc.cpu(), vc.cpu()
    at = 0
    for b, t in enumerate(new):
        p = torch.arange(lens[b] - t, lens[b])
        page_of, slot = batch.pages[b].long()[p // page], p % page
        _within(kc[page_of, :, slot], k64[at:at + t], tols[1][at:at + t])
        assert torch.equal(vc[page_of, :, slot], batch.v[at:at + t])
        kc[page_of, :, slot] = batch.k_cache[page_of, :, slot]
        vc[page_of, :, slot] = batch.v_cache[page_of, :, slot]
        at += t
    assert torch.equal(kc, batch.k_cache) and torch.equal(vc, batch.v_cache)
    assert _status() == 0


def test_store_with_positions_of_its_own_and_caches_in_another_order():
    """The cache as [pages][page][heads][dim] with k and v in one tensor, positions from the caller, q in place."""
    batch = Batch([4, 2], [20, 18], 4, 2)
    both = torch.zeros(batch.k_cache.shape[0], 2, 16, 2, 128, dtype=FP16, device="cuda")
    kc, vc = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    positions = torch.tensor([3, 1, 4, 1, 5, 9])
    freqs, _ = _paged().rotary_frequencies(128)
    q = batch.q.cuda()
    assert _paged().paged_store(batch.k.cuda(), batch.v.cuda(), kc, vc, batch.pages.cuda(), batch.starts.cuda(), batch.lens.cuda(), q=q,
                                freqs=freqs, positions=positions.cuda(), q_out=q) is q
    want, _ = _paged().apply_rotary(batch.q.cuda(), None, positions.cuda(), freqs)
    assert torch.equal(q, want)
    want, _ = _paged().apply_rotary(batch.k.cuda(), None, positions.cuda(), freqs)
    stored = torch.cat([batch.history(kc.cpu(), b)[n - t:] for b, (t, n) in enumerate(zip([4, 2], [20, 18]))])
    assert torch.equal(stored, want.cpu())
    assert int((both != 0).any(-1).sum()) == 2 * 6 * 2


def test_store_does_not_follow_bad_pages_or_positions():
    batch = Batch([2, 2, 3, 2], [17, 33, 1, 40], 4, 2)      # the third has two tokens in front of its first position
    batch.pages[0, 1] = batch.k_cache.shape[0]              # the page behind the last
    batch.pages[1, 2] = -1
    kc, vc, pages, starts, lens = _gpu(batch)
    lens[3] = 1 << 20                                       # positions behind its row of the table
    q = _paged().paged_store(batch.k.cuda(), batch.v.cuda(), kc, vc, pages, starts, lens, q=batch.q.cuda())
    assert _status() == 6
    assert torch.equal(q.cpu(), batch.q)
    changed = (kc.cpu() != batch.k_cache).any(-1).any(1).nonzero().tolist()
    assert changed == sorted([[int(batch.pages[0, 0]), 15], [int(batch.pages[1, 1]), 15], [int(batch.pages[2, 0]), 0]])


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------
def _mha(batch, out=None, **kw):
    kc, vc, pages, starts, lens = _gpu(batch)
    kw = {k: v.cuda() if torch.is_tensor(v) else v for k, v in kw.items()}
    return _paged().paged_mha(batch.q.cuda(), kc, vc, pages, starts, lens, out=out, **kw)


def _check(batch, hints=True, **kw):
    batch.poison()
    out = torch.full_like(batch.q, 7.0).cuda()
    if hints:
        kw = dict(kw, max_tokens=max(batch.new), max_len=max(batch.lens_list))
    got = _mha(batch, out, **kw)
    assert got is out and _status() == 0
    for k in ("max_tokens", "max_len"):
        kw.pop(k, None)
    ref, tol = attend64(batch, **kw)
    n = sum(batch.new)
    _within(out[:n], ref, tol)
    assert (out[n:] == 7.0).all(), "rows behind the last sequence"
    return out


LENGTHS = [
    ([1], [1]), ([1], [129]), ([1, 1, 1], [16, 127, 300]), ([1, 0, 1], [64, 5, 1000]), ([5, 3, 1, 2], [5, 70, 128, 131]),
    ([17], [17]), ([40, 1], [640, 33]), ([130, 1, 129], [130, 900, 700]), ([300], [333]),
]
HEADS = [(1, 1), (4, 4), (8, 2), (5, 1), (12, 2), (16, 1), (17, 1), (28, 4), (32, 1), (100, 1), (128, 1)]


@pytest.mark.parametrize("new,lens", LENGTHS)
@pytest.mark.parametrize("heads,kv_heads", HEADS)
def test_mha(new, lens, heads, kv_heads):
    n = len(new) * 10 + heads
    dtype, head_dim, page = (FP16, BF16)[n % 2], (128, 64, 128)[n % 3], (16, 32, 64, 128, 256)[n % 5]
    _check(Batch(new, lens, heads, kv_heads, head_dim, page, dtype, seed=n, behind=1))


@pytest.mark.parametrize("page,head_dim,dtype", list(itertools.product((16, 32, 64, 128, 256), (64, 128), (FP16, BF16))))
@pytest.mark.parametrize("new", [[1, 1], [4, 3], [200, 70]])
def test_mha_pages_types_and_head_sizes(page, head_dim, dtype, new):
    _check(Batch(new, [405, 258], 8, 4, head_dim, page, dtype, seed=page))


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 128, 200, 100000])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 2], [150, 1, 33]])
def test_mha_window(window, new):
    _check(Batch(new, [150, 700, 333], 4, 2, seed=window), window=window)


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [3, 1, 2, 4], [150, 1, 33, 140]])
def test_mha_left_padding_and_rows_that_see_nothing(new):
    first = torch.tensor([100, 0, 333, 500], dtype=torch.int32)    # the third sees its last position only if that is 332: nothing
    batch = Batch(new, [150, 700, 333, 501], 4, 2)
    out = _check(batch, first_key=first)
    at = sum(new[:2])
    assert (out[at:at + new[2]] == 0).all()
    _check(Batch(new, [150, 700, 333, 501], 4, 2, seed=9), first_key=first, window=70)


@pytest.mark.parametrize("new", [[5, 2], [1, 1], [40, 30], [200, 3]])
def test_mha_tokens_in_front_of_the_first_position(new):
    """A sequence shorter than its new tokens: the first ones stand at positions below zero, see nothing and get zeros."""
    lens = [3 if new[0] > 3 else 0, 2]
    batch = Batch(new, lens, 4, 2)
    out = torch.full_like(batch.q, 7.0).cuda()
    _mha(batch, out)
    ref, tol = attend64(batch)
    _within(out, ref, tol)
    assert (out[:new[0] - lens[0]] == 0).all()


@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (40, 8)])
@pytest.mark.parametrize("new", [[1, 1], [6, 2], [140, 1]])
def test_mha_alibi(heads, kv_heads, new):
    from eet_b200.EET import alibi_slopes
    slopes = torch.tensor(alibi_slopes(heads), dtype=torch.float32)
    _check(Batch(new, [141, 900], heads, kv_heads), alibi_slopes=slopes)
    _check(Batch(new, [141, 900], heads, kv_heads, dtype=BF16), alibi_slopes=slopes, window=100,
           first_key=torch.tensor([30, 0], dtype=torch.int32))


@pytest.mark.parametrize("new", [[1], [200]])
def test_mha_scale_and_large_scores(new):
    _check(Batch(new, [500], 4, 2, q_scale=30.0))
    _check(Batch(new, [500], 4, 2), scale=0.0)
    _check(Batch(new, [500], 4, 2), scale=-0.2)


@pytest.mark.parametrize("new", [[1, 1], [6, 1], [140, 20]])
def test_mha_without_hints_and_with_wrong_ones(new):
    """The hints choose how the work is cut up; what is computed does not depend on them."""
    _check(Batch(new, [400, 333], 8, 2), hints=False)
    _check(Batch(new, [400, 333], 8, 2), hints=False, max_tokens=1, max_len=1)
    _check(Batch(new, [400, 333], 8, 2), hints=False, max_tokens=10 ** 6, max_len=10 ** 9)


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan, 65504.0])
@pytest.mark.parametrize("new", [[1, 1], [7, 1], [100, 150]])
def test_mha_of_slots_behind_the_end_and_before_the_window(value, new):
    batch = Batch(new, [333, 190], 4, 2)
    batch.poison(value)
    # what lies before the window of the first new token, too
    for b, (t, n) in enumerate(zip(new, batch.lens_list)):
        p = torch.arange(max(0, n - t - 20 + 1))
        for cache in (batch.k_cache, batch.v_cache):
            cache[batch.pages[b].long()[p // 16], :, p % 16] = value
    got = _mha(batch, window=20)
    for b, (t, n) in enumerate(zip(new, batch.lens_list)):
        p = torch.arange(max(0, n - t - 20 + 1))
        for cache in (batch.k_cache, batch.v_cache):
            cache[batch.pages[b].long()[p // 16], :, p % 16] = 0.0
    ref, tol = attend64(batch, window=20)
    _within(got, ref, tol)


def test_mha_strides():
    """q and out as parts of wider rows, the caches as [pages][page][heads][dim] in one tensor, rows of the table far apart."""
    for new in ([1, 1], [5, 2], [150, 3]):
        batch = Batch(new, [222, 300], 6, 2)
        n = sum(new)
        wide = torch.zeros(n, 10, 128, dtype=FP16, device="cuda")
        wide[:, 2:8] = batch.q.cuda()
        both = torch.stack((batch.k_cache, batch.v_cache), 1).transpose(2, 3).contiguous().cuda()     # [pages][2][page][heads][dim]
        table = torch.full((2, 50), -1, dtype=torch.int32, device="cuda")
        table[:, :batch.pages.shape[1]] = batch.pages.cuda()
        out = torch.full((n, 8, 256), 7.0, dtype=FP16, device="cuda")
        _paged().paged_mha(wide[:, 2:8], both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2), table[:, :batch.pages.shape[1]],
                           batch.starts.cuda(), batch.lens.cuda(), out=out[:, 1:7, 128:])
        ref, tol = attend64(batch)
        _within(out[:, 1:7, 128:], ref, tol)
        assert (out[..., :128] == 7.0).all() and (out[:, 0] == 7.0).all() and (out[:, 7] == 7.0).all()
    assert _status() == 0


def test_mha_shared_pages():
    """Two sequences with a common beginning, held once; the same sequence twice in a batch."""
    for new in ([1, 1, 1], [2, 3, 2], [60, 70, 60]):
        batch = Batch(new, [160, 200, 160], 8, 2)
        batch.pages[1, :5] = batch.pages[0, :5]
        batch.pages[2] = batch.pages[0]
        _check(batch)


@pytest.mark.parametrize("new", [[1, 1, 1], [5, 1, 6], [140, 1, 60]])
def test_mha_does_not_follow_bad_pages(new):
    """The other sequences are served, the status names the fault."""
    batch = Batch(new, [160, 333, 160], 8, 2)
    ref, tol = attend64(batch)
    batch.pages[1, 3] = batch.k_cache.shape[0] + 5
    batch.pages[1, 4] = -7
    got = _mha(batch)
    assert _status() == 6
    a, b = new[0], new[0] + new[1]
    _within(got[:a], ref[:a], tol[:a])
    _within(got[b:], ref[b:], tol[b:])


def test_a_bad_page_is_named():
    from eet_b200 import EET
    batch = Batch([1], [20], 4, 2)
    batch.pages[0, 0] = 1 << 30
    _mha(batch)
    with pytest.raises(EET.EETError, match="paged cache"):
        EET.check_device_status()


@pytest.mark.parametrize("new", [[1, 1, 1], [4, 2, 3], [100, 40, 200]])
def test_mha_of_starts_and_lengths_that_go_too_far(new):
    """Fewer rows than starts say, lengths behind the table and below zero: nothing out of range, the others are served."""
    n = sum(new)
    batch = Batch(new, [260, 300, 280], 8, 2)
    ref, tol = attend64(batch)
    kc, vc, pages, starts, lens = _gpu(batch)
    q = batch.q.cuda()
    cut = n - 1 if new[2] == 1 else n - 2       # the last sequence loses its last rows, the rows that are there keep their positions
    got = _paged().paged_mha(q[:cut], kc, vc, pages, starts, lens)
    _within(got, ref[:cut], tol[:cut])
    assert _status() == 0
    for bad in (2 ** 31 - 1, 10 ** 6, -1, -2 ** 31):
        lens[1] = bad
        got = _paged().paged_mha(q, kc, vc, pages, starts, lens)
        a, b = new[0], new[0] + new[1]
        _within(got[:a], ref[:a], tol[:a])
        _within(got[b:], ref[b:], tol[b:])
        assert _status() == (6 if bad > 0 else 0)
        if bad < 0:
            assert (got[a:b] == 0).all()
    lens[1] = 300
    for bad in ([0, n + 5, new[0] + new[1], n], [-3, -1, 2 ** 31 - 1, n], [5, 3, 1, 0], [0, -2 ** 31, n, 2 ** 31 - 1]):
        _paged().paged_mha(q, kc, vc, pages, torch.tensor(bad, dtype=torch.int32).cuda(), lens)
        _paged().paged_store(batch.k.cuda(), batch.v.cuda(), kc, vc, pages, torch.tensor(bad, dtype=torch.int32).cuda(), lens, q=q)
        _status()


@pytest.mark.parametrize("heads, kv_heads", [(32, 1), (34, 2), (128, 1), (16, 1), (8, 4)])
@pytest.mark.parametrize("new", [[5] + [0] * 63, [0] * 40 + [7], [2] + [1] * 3 + [0] * 60])
def test_mha_one_chunk_beside_sequences_without_tokens(heads, kv_heads, new):
    """Long histories of sequences that ask nothing, with any number of query heads to a kv head."""
    batch = Batch(new, [max(n, 40 + 3 * i % 70) for i, n in enumerate(new)], heads, kv_heads)
    ref, tol = attend64(batch)
    kc, vc, pages, starts, lens = _gpu(batch)
    for kw in ({}, {"max_len": 10 ** 6}, {"max_tokens": 1}, {"max_tokens": 1, "max_len": 1}):
        wide = torch.zeros(len(new), 4096, dtype=torch.int32, device="cuda")
        wide[:, :pages.shape[1]] = pages
        _within(_paged().paged_mha(batch.q.cuda(), kc, vc, wide, starts, lens, **kw), ref, tol)
    assert _status() == 0


@pytest.mark.parametrize("tokens,heads", [(1, 4), (5, 1), (5, 4), (1, 1)])
@pytest.mark.parametrize("view", ["plain", "fused", "heads first", "expanded heads", "expanded tokens", "wide rows"])
def test_results_are_contiguous_whatever_the_strides(tokens, heads, view):
    batch = Batch([tokens], [tokens + 40], heads, 1)
    q = batch.q[:tokens].cuda()
    if view == "fused":
        q = torch.cat((q, q, q), 1)[:, heads:2 * heads]
    elif view == "heads first":
        q = q.transpose(0, 1).contiguous().transpose(0, 1)
    elif view == "expanded heads":
        q = q[:, :1].expand(tokens, heads, 128)
    elif view == "expanded tokens":
        q = q[:1].expand(tokens, heads, 128)
    elif view == "wide rows":
        q = torch.cat((q, q), 2)[..., :128]
    kc, vc, pages, starts, lens = _gpu(batch)
    freqs, at = _paged().rotary_frequencies(128, device="cuda")[0], torch.arange(tokens, device="cuda")
    same = q.contiguous()
    for get in (lambda x: _paged().paged_mha(x, kc, vc, pages, starts, lens),
                lambda x: _paged().apply_rotary(x, None, at, freqs)[0],
                lambda x: _paged().apply_rotary(None, x, at, freqs)[1],
                lambda x: _paged().paged_store(batch.k.cuda()[:tokens], batch.v.cuda()[:tokens], kc, vc, pages, starts, lens, q=x,
                                               freqs=freqs)):
        got, want = get(q), get(same)
        assert got.is_contiguous() and got.shape == q.shape and torch.equal(got, want)


@pytest.mark.parametrize("tokens", [1, 30])
def test_mha_slots_without_a_sequence(tokens):
    """Gaps of every length up to 19 between the sequences that ask something, many of them in one CTA's share."""
    new = []
    for gap in range(20):
        new += [0] * gap + [tokens]
    _check(Batch(new + [0] * 9, [tokens + 20 * i % 90 if n else 7 * i % 30 for i, n in enumerate(new + [0] * 9)], 2, 1, 64))


@pytest.mark.parametrize("new", [[1] * 40, [5, 7, 1], [70, 3, 200], [300]])
@pytest.mark.parametrize("length", [400, 5000])
def test_a_nan_in_q_stays_a_nan(new, length):
    """Whole and cut tiles of both kinds: the token whose q holds it, no other."""
    batch = Batch(new, [length + i for i in range(len(new))], 8, 2)
    ref, tol = attend64(batch)
    kc, vc, pages, starts, lens = _gpu(batch)
    q, bad = batch.q.cuda(), sum(new) // 2
    q[bad, 3, 17] = float("nan")
    got = _paged().paged_mha(q, kc, vc, pages, starts, lens, max_tokens=max(new))
    assert got[bad, 3].isnan().all()
    got[bad, 3] = ref[bad, 3].to(got)
    _within(got, ref, tol)


def test_mha_of_nothing():
    batch = Batch([0, 0], [5, 0], 4, 2)
    assert _mha(batch).shape == (0, 4, 128)
    none = Batch([1], [4], 4, 2)
    empty = torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    out = torch.full_like(none.q, 7.0).cuda()
    _paged().paged_mha(none.q.cuda(), none.k_cache.cuda(), none.v_cache.cuda(), empty, torch.zeros(1, dtype=torch.int32, device="cuda"),
                       torch.zeros(0, dtype=torch.int32, device="cuda"), out=out)
    assert (out == 7.0).all()


def test_mha_many_sequences():
    lens = [1 + (37 * i) % 400 for i in range(700)]
    _check(Batch([1] * 700, lens, 4, 1))
    _check(Batch([min(n, 1 + i % 3) for i, n in enumerate(lens)], lens, 20, 1, head_dim=64))


def test_mha_long():
    """Split over many CTAs: a long history, for one token and for a few."""
    _check(Batch([1, 1], [20000, 300], 8, 1))
    _check(Batch([1], [9000], 32, 1, dtype=BF16))
    _check(Batch([30], [9000], 8, 1))


def test_mha_twice_is_the_same():
    for new in ([1, 1], [3, 1], [130, 9]):
        batch = Batch(new, [3000, 333], 8, 2)
        assert torch.equal(_mha(batch), _mha(batch))


def test_mha_refuses():
    paged = _paged()
    batch = Batch([1, 2], [20, 30], 4, 2)
    q = batch.q.cuda()
    kc, vc, pages, starts, lens = _gpu(batch)
    names = ("q", "k_cache", "v_cache", "pages", "starts", "lens")
    for bad in (dict(q=q.float()), dict(q=q[0]), dict(q=q.bfloat16()), dict(k_cache=kc[0]), dict(v_cache=vc[:1]), dict(v_cache=vc.bfloat16()),
                dict(pages=pages.long()), dict(pages=pages.cpu()), dict(pages=pages[:1]), dict(starts=starts[:2]), dict(starts=starts.long()),
                dict(lens=lens[:1]), dict(lens=lens.cpu()), dict(out=q[:, :2]), dict(out=q.float()), dict(first_key=lens.long()),
                dict(first_key=lens[:1]), dict(alibi_slopes=torch.ones(3, device="cuda")), dict(alibi_slopes=torch.ones(4)),
                dict(window=-1), dict(q=torch.zeros(3, 3, 128, dtype=FP16, device="cuda")),
                dict(q=torch.zeros(3, 4, 64, dtype=FP16, device="cuda")), dict(k_cache=kc[:, :, :8], v_cache=vc[:, :, :8]),
                dict(q=torch.zeros(3 * 512 + 8, dtype=FP16, device="cuda")[1:1537].view(3, 4, 128)),
                dict(q=torch.zeros(3, 4, 129, dtype=FP16, device="cuda")[..., :128])):
        args = dict(zip(names, (q, kc, vc, pages, starts, lens)))
        args.update(bad)
        with pytest.raises(RuntimeError):
            paged.paged_mha(*[args.pop(n) for n in names], **args)


def test_mha_captured_and_replayed_with_other_lengths():
    batch = Batch([1, 1, 2], [100, 300, 200], 8, 2)
    later = Batch([1, 1, 2], [140, 3, 310], 8, 2, seed=4)
    width, total = 20, max(batch.k_cache.shape[0], later.k_cache.shape[0])
    q = batch.q.cuda()
    kc, vc = (torch.zeros(total, 2, 16, 128, dtype=FP16, device="cuda") for _ in range(2))
    pages, starts, lens = (torch.zeros(3, width, dtype=torch.int32, device="cuda"), batch.starts.cuda(),
                           torch.zeros(3, dtype=torch.int32, device="cuda"))

    def fill(b):
        q.copy_(b.q)
        kc[:b.k_cache.shape[0]].copy_(b.k_cache)
        vc[:b.v_cache.shape[0]].copy_(b.v_cache)
        pages.fill_(-1)
        pages[:, :b.pages.shape[1]].copy_(b.pages)
        starts.copy_(b.starts)
        lens.copy_(b.lens)

    fill(batch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _paged().paged_mha(q, kc, vc, pages, starts, lens, max_tokens=2)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _paged().paged_mha(q, kc, vc, pages, starts, lens, max_tokens=2)
    for b in (batch, later, batch):
        fill(b)
        graph.replay()
        ref, tol = attend64(b)
        _within(out, ref, tol)


def test_two_captured_graphs_and_two_streams_do_not_share_scratch():
    batches = [Batch([1, 3], [3000, 500], 8, 2, seed=s) for s in (1, 2)]
    refs = [attend64(b) for b in batches]
    inputs = [(b.q.cuda(), *_gpu(b)) for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    graphs, outs = [], []
    for args, s in zip(inputs, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            _paged().paged_mha(*args)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(_paged().paged_mha(*args))
        graphs.append(g)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for out, (ref, tol) in zip(outs, refs):
        _within(out, ref, tol)
    eager = []
    for _ in range(10):
        for args, s in zip(inputs, streams):
            with torch.cuda.stream(s):
                eager.append(_paged().paged_mha(*args))
    torch.cuda.synchronize()
    for i, out in enumerate(eager):
        _within(out, *refs[i % 2])


def test_store_and_attention_of_a_prompt_in_chunks_and_then_token_by_token():
    """As they are used: the sequence grows by chunks of 50, 1, 128 and single tokens; each step's context is that of the whole
    sequence so far."""
    H, K, D, page = 8, 2, 128, 32
    gen = torch.Generator().manual_seed(0)
    total = [183, 90]
    qkv = [torch.randn(n, H + 2 * K, D, generator=gen).half() for n in total]
    kc, vc = (torch.full((12, K, page, D), math.nan, dtype=FP16, device="cuda") for _ in range(2))
    pages = torch.tensor([[3, 9, 0, 5, 11, 1], [2, 10, 4, -1, -1, -1]], dtype=torch.int32)
    freqs, _ = _paged().rotary_frequencies(D)
    done = [0, 0]
    for step in ([50, 0], [1, 30], [128, 1], [1, 57], [1, 1], [1, 1], [1, 0]):
        new = [qkv[b][done[b]:done[b] + n] for b, n in enumerate(step)]
        done = [a + n for a, n in zip(done, step)]
        rows = torch.cat(new).cuda()
        starts = torch.tensor([0, step[0], sum(step)], dtype=torch.int32).cuda()
        lens = torch.tensor(done, dtype=torch.int32).cuda()
        q = _paged().paged_store(rows[:, H:H + K], rows[:, H + K:], kc, vc, pages.cuda(), starts, lens, q=rows[:, :H], freqs=freqs)
        ctx = _paged().paged_mha(q, kc, vc, pages.cuda(), starts, lens, max_tokens=max(step))
        # the same from what the cache holds now
        view = Batch.__new__(Batch)
        view.new, view.lens_list, view.page, view.dtype = step, done, page, FP16
        view.k_cache, view.v_cache, view.pages, view.q = kc.cpu(), vc.cpu(), pages, q.cpu()
        ref, tol = attend64(view)
        _within(ctx, ref, tol, f"step {step}")
    # and the cache holds every rotated key
    for b in range(2):
        want = rotate64(qkv[b][:done[b], H:H + K], torch.arange(done[b]), freqs.cpu(), False)
        got = kc.cpu()[pages[b].long()[torch.arange(done[b]) // page], :, torch.arange(done[b]) % page]
        x = qkv[b][:done[b], H:H + K]
        _within(got, want, 2.0 ** -11 * want.abs() + rotate_tolerance(x, freqs.cpu(), False, FP16) + 2.0 ** -25)
    assert _status() == 0


@pytest.mark.parametrize("new", [[1, 1], [5, 3], [150, 40], [700, 1]])
def test_mha_out_in_the_place_of_q(new):
    """A tile's rows are written by who has read them, or by the second launch."""
    batch = Batch(new, [3000, 710 if new[0] < 700 else 900], 8, 2)
    kc, vc, *table = _gpu(batch)
    want = _paged().paged_mha(batch.q.cuda(), kc, vc, *table)
    q = batch.q.cuda()
    assert _paged().paged_mha(q, kc, vc, *table, out=q) is q
    assert torch.equal(q, want)


def test_pages_far_behind_the_2_to_the_31st_value():
    """Caches of 2.6e9 values each: the pages at their end and the same rows at their beginning."""
    pages, K, P, D = 20000, 8, 128, 128
    kc, vc = (torch.zeros(pages, K, P, D, dtype=FP16, device="cuda") for _ in range(2))
    assert kc.numel() > 2 ** 31
    gen = torch.Generator().manual_seed(1)
    lens = torch.tensor([200, 131], dtype=torch.int32).cuda()
    for new in ([200, 131], [3, 1]):
        n = sum(new)
        k, v = (torch.randn(n, K, D, generator=gen).half().cuda() for _ in range(2))
        q = torch.randn(n, 16, D, generator=gen).half().cuda()
        starts = torch.tensor([0, new[0], n], dtype=torch.int32).cuda()
        got = []
        for table in ([[0, 1], [2, 3]], [[pages - 1, pages - 7], [16384 + 1, pages - 2]]):
            table = torch.tensor(table, dtype=torch.int32).cuda()
            _paged().paged_store(k, v, kc, vc, table, starts, lens)
            got.append(_paged().paged_mha(q, kc, vc, table, starts, lens))
        assert torch.equal(*got)
        for a, b, t in ((0, pages - 1, 128), (1, pages - 7, 72), (2, 16385, 128), (3, pages - 2, 3)):
            assert torch.equal(kc[a, :, :t], kc[b, :, :t]) and torch.equal(vc[a, :, :t], vc[b, :, :t])
    assert _status() == 0


def test_calls_on_streams_of_their_own_in_turn():
    """Work of one call behind another's on two streams that wait for each other; each call takes scratch of its own."""
    batch = Batch([1, 1, 1], [4000, 50, 900], 8, 2)
    args = (batch.q.cuda(), *_gpu(batch))
    want = _paged().paged_mha(*args)
    chunk = Batch([300, 2], [2000, 900], 8, 2, seed=3)
    chunk_args = (chunk.q.cuda(), *_gpu(chunk))
    chunk_want = _paged().paged_mha(*chunk_args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for i in range(30):
        with torch.cuda.stream(streams[i % 3]):
            outs.append((_paged().paged_mha(*args), want) if i % 2 else (_paged().paged_mha(*chunk_args), chunk_want))
    torch.cuda.synchronize()
    assert all(torch.equal(got, ref) for got, ref in outs)
    assert _status() == 0


def test_mha_both_kernels_in_one_call():
    """One chunk beside so many single tokens that they get the kernel of their own."""
    new, lens = [200] + [1] * 40, [1100] + [3000 + 37 * i for i in range(40)]
    assert 40 * 32 * (max(lens) // 128 + 1) >= 16384
    for dtype in (FP16, BF16):
        batch = Batch(new, lens, 32, 32, 64, 64, dtype, behind=2)
        _check(batch)
    some = Batch([1, 300, 0] + [1] * 30, [0, 300, 5] + [4000] * 30, 64, 32, 64, 32, seed=2)
    _check(some, window=700, first_key=torch.tensor([0, 10, 0] + [3700 + i for i in range(30)], dtype=torch.int32))

# ---------------------------------------------------------------------------------------------------------------------
# the attention block
# ---------------------------------------------------------------------------------------------------------------------
def _block(heads, kv_heads, hidden, is_int8, seed=0, **kw):
    """(PagedMmha, its weights as they were quantized)."""
    from eet_b200 import EET
    gen = torch.Generator().manual_seed(seed)
    desc = EET.MetaDesc(FP16, 4, heads, hidden, 1, 128, 512, d_kv=128, is_int8=is_int8)
    qkv = (torch.randn(hidden, 128 * (heads + 2 * kv_heads), generator=gen) * hidden ** -0.5).half()
    out = (torch.randn(128 * heads, hidden, generator=gen) * (128 * heads) ** -0.5).half()
    norm = (1 + 0.1 * torch.randn(hidden, generator=gen)).half().cuda()
    if is_int8:
        (qkv, qkv_s), (out, out_s) = (EET.quant_weights(w) for w in (qkv, out))
        args = qkv.cuda(), qkv_s.cuda(), out.cuda(), out_s.cuda(), norm
    else:
        args = qkv.cuda(), None, out.cuda(), None, norm
    return _paged().PagedMmha(desc, *args, kv_head_num=kv_heads, **kw), args


@pytest.mark.parametrize("heads,kv_heads,is_int8,alibi", [(4, 2, True, False), (2, 2, False, False), (6, 1, True, True)])
def test_block_is_the_calls_behind_one_another(heads, kv_heads, is_int8, alibi):
    """At most 16 rows, where the projections add in one order: the same bits."""
    from eet_b200 import EET
    hidden = 256
    slopes = torch.tensor(EET.alibi_slopes(heads), dtype=torch.float32).cuda() if alibi else None
    block, (qkv_w, qkv_s, out_w, out_s, norm) = _block(heads, kv_heads, hidden, is_int8, alibi_slopes=slopes)
    batch = Batch([3, 1, 6], [20, 300, 150], heads, kv_heads)
    x = torch.randn(10, hidden, generator=torch.Generator().manual_seed(1)).half().cuda()
    kc, vc, *table = _gpu(batch)
    got = block(x, kc, vc, *table, max_tokens=6, window=100).clone()
    kc2, vc2, *_ = _gpu(batch)
    xn = EET.LayerNorm(block.desc, norm, torch.empty(0)).layer_norm(x.view(1, 10, hidden)).view(10, hidden)
    qkv = EET.gemm_w8a16(xn, qkv_w, qkv_s) if is_int8 else xn @ qkv_w
    qkv = qkv.view(10, -1, 128)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    freqs = None if alibi else _paged().rotary_frequencies(128)[0]
    q = _paged().paged_store(k, v, kc2, vc2, *table, q=q, freqs=freqs)
    ctx = _paged().paged_mha(q, kc2, vc2, *table, max_tokens=6, window=100, alibi_slopes=slopes).view(10, -1)
    want = EET.gemm_w8a16(ctx, out_w, out_s, residual=x) if is_int8 else (ctx @ out_w) + x
    assert torch.equal(got, want) and torch.equal(kc, kc2) and torch.equal(vc, vc2)


def test_block_beside_llama_mmha():
    """Two prompts of one length and three steps, the paged block against EET.LlamaMmha with its own caches.

    Both round q, k, v and the context to fp16 once, so with |w| the weights: the outputs differ by at most the rounding of the
    context and of the probabilities in both (4 half steps of the mean of |v|, times |w|), by that of q and k where their angles
    differ in the last bit (2 half steps of each score's magnitude, as a relative error of the probabilities, twice), LlamaMmha's
    scores in fp16 (one more half step of the score), and two roundings of the result and of the sum with the residual."""
    from eet_b200 import EET
    heads, hidden, S, B = 4, 256, 130, 2
    block, (qkv_w, qkv_s, out_w, out_s, norm) = _block(heads, heads, hidden, True, seed=3)
    desc = EET.MetaDesc(FP16, B, heads, hidden, 1, S, S + 4, d_kv=128, is_int8=True)
    none = torch.empty(0)
    llama = EET.LlamaMmha(desc, qkv_w, qkv_s, none, none, none, out_w, out_s, none, norm, none)
    x = torch.randn(B, S + 3, hidden, generator=torch.Generator().manual_seed(2)).half().cuda()
    kc, vc = (torch.full((20, heads, 16, 128), math.nan, dtype=FP16, device="cuda") for _ in range(2))
    pages = torch.arange(20, dtype=torch.int32, device="cuda").view(2, 10)
    weights = (EET.unpack_weights(out_w).double() * out_s.double()).abs()
    u = 2.0 ** -11
    for first, last in ((0, S), (S, S + 1), (S + 1, S + 2), (S + 2, S + 3)):
        part = x[:, first:last].contiguous()
        want = llama(part, none, none, True, True, first == 0).clone().view(-1, hidden)
        n = last - first
        starts = torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda")
        lens = torch.tensor([last, last], dtype=torch.int32, device="cuda")
        got = block(part.view(-1, hidden), kc, vc, pages, starts, lens, max_tokens=n).clone()
        k, v = (c[pages[:, :(last + 15) // 16].long()].transpose(2, 3).reshape(B, -1, heads, 128)[:, :last].abs().double().amax((1, 3))
                for c in (kc, vc))                                                                 # [B][heads]
        q = EET._pool.rows("qkv_paged", 2 * n, 3 * 512, 1, FP16, x.device).view(B, n, 3 * heads, 128)[:, :, :heads].abs().double()
        score = q.sum(-1) * k[:, None] / math.sqrt(128)                                           # [B][n][heads], at least the largest
        context = (4 * u + 2 * (4 + 1) * u * score) * v[:, None]
        tol = context.repeat_interleave(128, -1).view(-1, 512) @ weights + 1e-5
        tol += 2 * u * (want.double().abs() + part.view(-1, hidden).double().abs())
        off = (got.double() - want.double()).abs()
        assert (off <= tol).all() and off.max() < 0.02
    assert _status() == 0


def test_block_refuses():
    from eet_b200 import EET
    block, args = _block(4, 2, 256, True)
    x = torch.zeros(3, 256, dtype=FP16, device="cuda")
    batch = Batch([1, 2], [4, 5], 4, 2)
    for bad in (x.float(), x[:, :128], x.cpu(), x.view(1, 3, 256), torch.zeros(513, 256, dtype=FP16, device="cuda")):
        with pytest.raises(RuntimeError):
            block(bad, *_gpu(batch))
    assert block(x[:0], *_gpu(Batch([0], [3], 4, 2))).shape == (0, 256)
    with pytest.raises(RuntimeError, match="kv heads"):
        _paged().PagedMmha(block.desc, *args, kv_head_num=3)
    with pytest.raises(RuntimeError, match="QKV_weights"):
        _paged().PagedMmha(block.desc, *args, kv_head_num=4)
    with pytest.raises(RuntimeError, match="exclude"):
        _paged().PagedMmha(block.desc, *args, kv_head_num=2, freqs=_paged().rotary_frequencies(128)[0],
                           alibi_slopes=torch.ones(4, device="cuda"))
    wide = EET.MetaDesc(FP16, 4, 4, 256, 1, 128, 512, is_int8=True)
    with pytest.raises(RuntimeError, match="head size 128"):
        _paged().PagedMmha(wide, *args, kv_head_num=2)


def test_a_layer_of_a_model_step_captured():
    """Block and FFN op of one decoder layer in a captured step, replayed while lengths and pages change: as in eager calls."""
    from eet_b200 import EET
    hidden, heads, kv_heads = 256, 4, 2
    block, _ = _block(heads, kv_heads, hidden, True, seed=5)
    desc = EET.MetaDesc(FP16, 4, heads, hidden, 1, 128, 512, activation_fn="silu", d_kv=128, d_ff=512, is_int8=True)
    gen = torch.Generator().manual_seed(8)
    w = [EET.quant_weights((torch.randn(*s, generator=gen) * 0.05).half()) for s in ((hidden, 512), (hidden, 512), (512, hidden))]
    none = torch.empty(0)
    ffn = EET.GatedFeedForwardNetworkInt8(desc, w[0][0].cuda(), w[0][1].cuda(), none, w[1][0].cuda(), w[1][1].cuda(), none,
                                          w[2][0].cuda(), w[2][1].cuda(), none, torch.ones(hidden, dtype=FP16, device="cuda"), none)
    kc, vc = (torch.randn(12, kv_heads, 16, 128, generator=gen).half().cuda() for _ in range(2))
    pages = torch.tensor([[0, 3, 6, 9], [1, 4, 7, 10], [2, 5, 8, 11]], dtype=torch.int32, device="cuda")
    starts = torch.arange(4, dtype=torch.int32, device="cuda")
    lens = torch.tensor([5, 17, 30], dtype=torch.int32, device="cuda")
    x = torch.randn(3, hidden, generator=gen).half().cuda()

    def step():
        y = block(x, kc, vc, pages, starts, lens, max_tokens=1, max_len=64)
        return ffn(y.view(1, 3, hidden)).view(3, hidden)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(6):
        lens += 5
        x.copy_(torch.randn(3, hidden, generator=gen).half())
        before = kc.clone(), vc.clone()
        graph.replay()
        got = out.clone()
        kc.copy_(before[0])
        vc.copy_(before[1])
        assert torch.equal(step(), got)
    assert _status() == 0


@pytest.mark.parametrize("rows,is_int8", [(3, False), (20, False), (70, False), (3, True), (16, True)])
def test_block_and_llama_mmha_behind_one_another(rows, is_int8):
    """The output of an attention op handed to the next: input and output of that one are the same buffer."""
    from eet_b200 import EET
    hidden, none = 256, torch.empty(0)
    block, (qkv_w, qkv_s, out_w, out_s, norm) = _block(2, 2, hidden, is_int8, seed=7)
    llama = EET.LlamaMmha(EET.MetaDesc(FP16, 4, 2, hidden, 1, 128, 512, d_kv=128, is_int8=is_int8), qkv_w, qkv_s, none, none, none, out_w,
                          out_s, none, norm, none)
    x = torch.randn(rows, hidden, generator=torch.Generator().manual_seed(rows)).half().cuda()
    batch = Batch([rows], [rows], 2, 2)

    def paged(y):
        return block(y.view(rows, hidden), *_gpu(batch))

    def own(y):
        return llama(y.view(1, rows, hidden), none, none, True, True, True).view(rows, hidden)

    for first in (paged, own):
        for second in (paged, own):
            want = second(first(x).clone()).clone()
            assert torch.equal(second(first(x)), want)


def _deferred_chain(rows, seed=11):
    """A decode step of LlamaMmha (its input, behind a prompt of two), and a PagedMmha of fp16 weights that shows what it was given: its
    queries, keys and values are channels of the norm, the output projection is zero, so that its output is its input."""
    from eet_b200 import EET
    hidden, none = 256, torch.empty(0)
    gen = torch.Generator().manual_seed(seed)
    desc = EET.MetaDesc(FP16, rows, 2, hidden, 1, 2, 4, d_kv=128, is_int8=True)
    (qkv, qkv_s), (out, out_s) = (EET.quant_weights((torch.randn(hidden, n, generator=gen) / 16).half()) for n in (3 * hidden, hidden))
    norm = (1 + 0.1 * torch.randn(hidden, generator=gen)).half().cuda()
    llama = EET.LlamaMmha(desc, qkv.cuda(), qkv_s.cuda(), none, none, none, out.cuda(), out_s.cuda(), none, norm, none)
    plain = EET.MetaDesc(FP16, rows, 2, hidden, 1, 2, 4, d_kv=128, is_int8=False)
    eye = torch.eye(hidden, dtype=FP16)
    block = _paged().PagedMmha(plain, torch.cat((eye, eye), 1).cuda(), None, torch.zeros(hidden, hidden, dtype=FP16).cuda(), None, norm,
                               kv_head_num=1, alibi_slopes=torch.zeros(2, device="cuda"))
    llama(torch.randn(rows, 2, hidden, generator=gen).half().cuda(), none, none, True, True, True)
    x = torch.randn(rows, 1, hidden, generator=gen).half().cuda()

    def step():
        llama.step_ = 2
        return llama(x, none, none, True, True, False).view(rows, hidden)

    return step, block, norm


@pytest.mark.parametrize("n", [17, 20, 64])
def test_block_behind_an_attention_op_that_left_its_output_unfinished(n):
    """17 to 64 rows inside deferred_epilogue(): the block finishes its input, which lies in the buffer that its own output takes.

    Input and output are y, LlamaMmha's result, rounded to fp16 from sums that may be added in another order than outside: two roundings
    of half a step u and 512 additions of terms that make at most 16 in magnitude (2^-24 each).  The keys and values are rounded norms of
    it: two more roundings, and the factor of the norm, which moves by no more than its rows do."""
    from eet_b200 import EET
    step, block, norm = _deferred_chain(n)
    want = step().clone()
    batch = Batch([n], [n], 2, 1)
    _, _, *table = _gpu(batch)
    u, order = 2.0 ** -11, 512 * 16 * 2.0 ** -24
    for _ in range(2):     # twice: the first leaves nothing behind
        kc, vc = (torch.zeros(batch.k_cache.shape, dtype=FP16, device="cuda") for _ in range(2))
        step().fill_(7.0)                 # what the buffer holds before
        with EET.deferred_epilogue():
            got = block(step(), kc, vc, *table).clone()
        ref = want.double().cpu()
        _within(got, ref, 2 * u * ref.abs() + order)
        xn = ref * torch.rsqrt(ref.square().mean(-1, keepdim=True) + 1e-6) * norm.double().cpu()
        tol = 6 * u * xn.abs() + 4 * order
        for cache, part in ((kc, slice(0, 128)), (vc, slice(128, 256))):
            _within(batch.history(cache.cpu(), 0)[:, 0], xn[:, part], tol[:, part])
    with EET.deferred_epilogue():
        again = step()
    _within(again, want.double().cpu(), 2 * u * want.double().cpu().abs() + order)
    assert _status() == 0


def test_an_unfinished_output_that_nobody_reads_leaves_nothing_behind():
    """Inside deferred_epilogue(): the sums of a projection whose output is overwritten, by this block or by an op of the same kind, are
    zero for the next one.  The tolerance is that of the test above."""
    from eet_b200 import EET
    step, block, _ = _deferred_chain(20)
    want = step().clone().double().cpu()
    tol = 2 * 2.0 ** -11 * want.abs() + 512 * 16 * 2.0 ** -24
    batch = Batch([20], [20], 2, 1)
    other = torch.randn(20, 256, generator=torch.Generator().manual_seed(1)).half().cuda()
    for write in (lambda: block(other, *_gpu(batch)), step):
        with EET.deferred_epilogue():
            step()
            write()
            got = step()
        _within(got, want, tol)


@pytest.mark.parametrize("new", [[3, 1, 1], [3, 40, 200]])
def test_mha_of_starts_that_end_far_below_their_beginning(new):
    """The sequence whose rows would end at -2^31 has none; the rows of the others, and what lies behind q's, stay as they are to be."""
    n = sum(new)
    batch = Batch(new, [260, 300, 280], 8, 2)
    ref, tol = attend64(batch)
    kc, vc, pages, starts, lens = _gpu(batch)
    starts[2] = -2 ** 31
    out = torch.full((n + 400, 8, 128), 7.0, dtype=FP16, device="cuda")
    _paged().paged_mha(batch.q.cuda(), kc, vc, pages, starts, lens, out=out[:n])
    _within(out[:3], ref[:3], tol[:3])
    assert (out[3:] == 7.0).all() and _status() == 0


@pytest.mark.parametrize("new", [1, 20])
def test_mha_fp16_counts_keys_far_below_the_largest(new):
    """One key holds nearly all of the weight and 20000 others e^-18 = 2^-26 of it each: 3.0e-4 of the result, half a step of fp16 being
    2.4e-4.  148 sequences that share one history, so that a CTA walks the whole of it under one reference.

    The largest probability enters the product as 2^7 or more, so what is below the type's normal values is off by at most 2^-25 / 2^7 of it,
    20000 times; the others and the result by half a step; the scores are exact."""
    H, page, n = 1, 128, 20000
    total = n + new
    pages = -(-total // page)
    kc, vc = torch.zeros(pages, H, page, 64, dtype=FP16), torch.ones(pages, H, page, 64, dtype=FP16)
    kc[(n - 1) // page, 0, (n - 1) % page, 0] = 18.0
    vc[(n - 1) // page, 0, (n - 1) % page] = 0.0
    q = torch.zeros(148 * new, H, 64, dtype=FP16)
    q[:, :, 0] = 1.0
    table = torch.arange(pages, dtype=torch.int32).expand(148, pages).contiguous()
    starts, lens = torch.arange(149, dtype=torch.int32) * new, torch.full((148,), total, dtype=torch.int32)
    got = _paged().paged_mha(*(t.cuda() for t in (q, kc, vc, table, starts, lens)), scale=1.0, max_tokens=new).double().cpu()
    w = math.exp(-18.0)
    others = n - 1 + 1.0 + torch.arange(new, dtype=torch.float64).repeat(148)[:, None, None]     # the token itself and those before it
    exact = others * w / (1.0 + others * w)
    _within(got, exact.expand_as(got), (20100 * 2.0 ** -32 + 2 * 2.0 ** -11 * exact + 2.0 ** -25).expand_as(got))


@pytest.mark.parametrize("slopes,sign", [(False, 1), (True, 1), (False, -1)])
@pytest.mark.parametrize("new,length", [(1, 300), (1, 6000), (5, 300), (200, 300), (200, 6000), (20, 300)])
def test_mha_scores_far_below_zero(new, length, slopes, sign):
    """All scores at -8e25, far within fp32: the mean of the values that a token sees.  All weights are the same number, so the result is
    off by half a step of the probabilities and of its own, and by fp32 sums (2^-19)."""
    batch = Batch([new], [length], 2, 1, 64, dtype=BF16)
    batch.q[:] = 1e13
    batch.k_cache[:] = -1e12 * sign
    batch.poison()
    got = _mha(batch, scale=sign / 8.0, alibi_slopes=torch.zeros(2) if slopes else None).double().cpu()
    v = batch.history(batch.v_cache, 0).double()[:, 0]
    seen = torch.arange(length - new, length)[:, None, None] + 1.0
    mean, size = (x.cumsum(0)[length - new:, None] / seen for x in (v, v.abs()))
    _within(got, mean.expand_as(got), (2 * 2.0 ** -8 * size + 2.0 ** -8 * mean.abs() + 2.0 ** -19).expand_as(got))
    assert _status() == 0


@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("new,length", [(1, 300), (5, 6000), (200, 300), (200, 6000), (20, 300)])
@pytest.mark.parametrize("dtype,large", [(FP16, 20000.0), (BF16, 20000.0), (BF16, 1e8)])
def test_mha_scores_far_above_zero(new, length, slopes, dtype, large):
    """All scores 64 large^2 / 8, where one unit in the last place of fp32 is 2^8 and more: the mean of the values, as above."""
    batch = Batch([new], [length], 2, 1, 64, dtype=dtype)
    batch.q[:] = large
    batch.k_cache[:] = large
    batch.poison()
    got = _mha(batch, alibi_slopes=torch.zeros(2) if slopes else None).double().cpu()
    u, v = HALF_STEP[dtype], batch.history(batch.v_cache, 0).double()[:, 0]
    seen = torch.arange(length - new, length)[:, None, None] + 1.0
    mean, size = (x.cumsum(0)[length - new:, None] / seen for x in (v, v.abs()))
    _within(got, mean.expand_as(got), (2 * u * size + u * mean.abs() + 2.0 ** -19).expand_as(got))
    assert _status() == 0


@pytest.mark.parametrize("new,length,slopes", [([1], 400, False), ([5], 5000, False), ([200], 1000, False), ([200], 1000, True),
                                               ([30, 300], 3000, False)])
@pytest.mark.parametrize("dtype,size", [(FP16, 100.0), (FP16, 3000.0), (BF16, 1e6), (BF16, 1e15)])
def test_mha_of_large_scores_takes_the_largest(new, length, slopes, dtype, size):
    """Scores of 10^4 to 10^30, both signs, some references near and some far: where the largest leads by more than what fp32 can lose of
    both (D + 8 half steps of their sums of magnitudes each) and 40 units, its value alone is the result, to two roundings."""
    heads = 4
    batch = Batch(new, [length] * len(new), heads, 2, 64, dtype=dtype, q_scale=size)
    batch.k_cache = (batch.k_cache * size).clamp(-6e4, 6e4) if dtype == FP16 else batch.k_cache * size
    batch.q = batch.q.clamp(-6e4, 6e4) if dtype == FP16 else batch.q
    batch.poison()
    bias = torch.tensor([0.5, 0.25, 0.125, 0.0625]) if slopes else None
    got = _mha(batch, alibi_slopes=bias).double().cpu()
    at, rows = 0, 0
    for b, t in enumerate(new):
        k, v = (batch.history(c, b).double().repeat_interleave(2, 1).transpose(0, 1) for c in (batch.k_cache, batch.v_cache))
        q = batch.q[at:at + t].double().transpose(0, 1)
        s, lost = q @ k.transpose(1, 2) / 8.0, q.abs() @ k.abs().transpose(1, 2) / 8.0 * (64 + 8) * 2.0 ** -24
        p, j = torch.arange(length - t, length)[:, None], torch.arange(length)[None, :]
        if slopes:
            s, lost = s + bias.double()[:, None, None] * (j - p), lost + bias.double()[:, None, None] * (p - j) * 2.0 ** -22
        s, lost = s.masked_fill(j > p, -math.inf), lost.masked_fill(j > p, 0.0)
        two = s.topk(2, -1).values
        clear = two[..., 0] - two[..., 1] > 40 + 2 * lost.amax(-1)
        want = torch.gather(v, 1, s.argmax(-1, keepdim=True).expand(-1, -1, 64))
        off = (got[at:at + t].transpose(0, 1) - want).abs() - 2 * HALF_STEP[dtype] * want.abs() - 1e-7
        assert not got[at:at + t].isnan().any() and (off[clear] <= 0).all()
        rows += int(clear.sum())
        at += t
    assert rows >= 0.9 * sum(new) * heads and _status() == 0


def _scratch(batch, max_tokens, max_len, window=0):
    """What the host plans: the scratch of the call, in bytes."""
    from eet_b200._lib import lib
    from test_paged_cpu import _mha as args
    H, D = batch.q.shape[1:]
    K, P = batch.k_cache.shape[1:3]
    return lib.eet_paged_mha_workspace_bytes(args(
        heads=H, kv_heads=K, head_dim=D, tokens=batch.q.shape[0], seqs=len(batch.new), page_size=P, max_pages=batch.pages.shape[1],
        pages_stride=batch.pages.shape[1], num_pages=batch.k_cache.shape[0], max_tokens=max_tokens, max_len=max_len, window=window))


def _scratch_of_both(head_dim):
    """Two parts of 16 and of 256 rows - a maximum, a sum and head_dim values each - and a header, twice for every CTA."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    return sum(sms * (32 + 2 * 4 * rows * (2 + head_dim)) for rows in (16, 256))


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("dtype,head_dim", [(FP16, 64), (FP16, 128), (BF16, 64), (BF16, 128)])
@pytest.mark.parametrize("kind", ["plain", "slopes", "negative scale", "whole"])
def test_mha_both_kernels_with_every_kind_of_scores(kind, dtype, head_dim, page):
    """A chunk and an empty sequence among 40 single tokens behind histories of up to 900, where the plan has few-row CTAs and tiles in one
    launch: tiles of both kinds cut, or ("whole", behind a window) neither, then without a second launch."""
    from eet_b200.EET import alibi_slopes
    new = [1] * 15 + [200, 0] + [1] * 25
    lens = [800 + 5 * i % 100 if n else 77 for i, n in enumerate(new)]
    heads, kv_heads = ((12, 6), (8, 8))[page % 3 % 2]
    batch = Batch(new, lens, heads, kv_heads, head_dim, page, dtype, seed=page, behind=2)
    slopes = torch.tensor(alibi_slopes(heads), dtype=torch.float32)
    kw = {"plain": {}, "slopes": dict(alibi_slopes=slopes, first_key=torch.arange(42, dtype=torch.int32) * 7),
          "negative scale": dict(scale=-0.1), "whole": dict(alibi_slopes=slopes, window=100)}[kind]
    both = _scratch_of_both(head_dim)
    assert _scratch(batch, 200, max(lens), kw.get("window", 0)) == (0 if kind == "whole" else both)
    if kind == "whole":   # beside a plan that cuts, for the same sizes: both kinds are there
        assert _scratch(batch, 200, max(lens)) == both
    _check(batch, **kw)


def test_mha_both_kernels_where_there_is_work_for_one_only():
    """The plan goes by the hints; what the sequences turn out to be may leave either kind without work."""
    for new in ([1] * 41, [0] * 10 + [3] + [0] * 30, [30] * 3 + [0] * 38, [0] * 40 + [200], [0] * 41):
        batch = Batch(new, [900 - i for i in range(41)], 8, 8, 128, 32, behind=40)
        assert _scratch(batch, 200, 900) == _scratch_of_both(128)
        for kw in ({}, {"alibi_slopes": torch.full((8,), 0.1)}):
            _check(batch, hints=False, max_tokens=200, max_len=900, **kw)


@pytest.mark.parametrize("new", [[200] + [1] * 40, [24] + [1] * 40, [1] * 40])
@pytest.mark.parametrize("window", [0, 100])
def test_block_over_both_kernels_and_projections_without_a_pause(new, window):
    """The projections take tensor memory while the attention in front of them runs, and the other way round: thirty blocks behind one
    another against one call at a time.

    Rotation, append and attention give the same bits, as does the projection in front of them.  That behind adds 1024 products in any
    order (2^-24 of their magnitudes each time, on either side) and rounds the sum and its sum with the residual (half a step each)."""
    heads, kv_heads, hidden = 8, 8, 256
    from eet_b200 import EET
    gen = torch.Generator().manual_seed(0)
    desc = EET.MetaDesc(FP16, 4, heads, hidden, 1, 128, 512, d_kv=128, is_int8=True)
    qkv, out = (EET.quant_weights((torch.randn(*s, generator=gen) / 16).half()) for s in ((hidden, 3 * 1024), (1024, hidden)))
    norm = torch.ones(hidden, dtype=FP16).cuda()
    block = _paged().PagedMmha(desc, qkv[0].cuda(), qkv[1].cuda(), out[0].cuda(), out[1].cuda(), norm)
    batch = Batch(new, [900 - i for i in range(len(new))], heads, kv_heads)
    kc, vc, *table = _gpu(batch)
    x = torch.randn(sum(new), hidden, generator=gen).half().cuda()
    kw = dict(max_tokens=max(new), max_len=900, window=window)
    xn = EET.LayerNorm(desc, norm, torch.empty(0)).layer_norm(x.view(1, -1, hidden)).view(-1, hidden).clone()
    rows = EET.gemm_w8a16(xn, qkv[0].cuda(), qkv[1].cuda()).view(-1, 3 * heads, 128).clone()
    torch.cuda.synchronize()
    q = _paged().paged_store(rows[:, 8:16], rows[:, 16:], kc, vc, *table, q=rows[:, :8], freqs=block.freqs)
    torch.cuda.synchronize()
    ctx = _paged().paged_mha(q, kc, vc, *table, **kw)
    torch.cuda.synchronize()
    want = EET.gemm_w8a16(ctx.view(-1, 1024), out[0].cuda(), out[1].cuda(), residual=x).clone()
    torch.cuda.synchronize()
    weights = EET.unpack_weights(out[0]).double().cuda() * out[1].double().cuda()
    ctx, want = ctx.view(-1, 1024).double(), want.double()
    tol = 2 * 1024 * 2.0 ** -24 * (ctx.abs() @ weights.abs()) + 2 * 2.0 ** -11 * ((ctx @ weights).abs() + want.abs())
    stored = kc.clone(), vc.clone()
    got = [block(x, kc, vc, *table, **kw).clone() for _ in range(30)]
    for y in got:
        _within(y, want.cpu(), tol.cpu())
    assert torch.equal(kc, stored[0]) and torch.equal(vc, stored[1])
    assert _status() == 0


@pytest.mark.parametrize("which", ["QKV_scale", "Output_scale", "layernorm_weights"])
def test_block_refuses_scales_and_norms_that_the_kernels_would_read_past(which):
    block, args = _block(4, 2, 256, True)
    at = {"QKV_scale": 1, "Output_scale": 3, "layernorm_weights": 4}[which]
    good = args[at]
    for bad in (good[:-1].contiguous(), good[::2], good.float(), good.cpu(), None, torch.empty(0)):
        with pytest.raises(RuntimeError, match=which):
            _paged().PagedMmha(block.desc, *args[:at], bad, *args[at + 1:], kv_head_num=2)
