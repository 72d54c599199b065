"""A paged cache of 8-bit codes and the choice of tokens: what the calls refuse on the host, without a GPU, and the oracle's rounding."""
import math
import os
import re

import pytest
import torch

from codes_util import MOST, half_step, quantize64
from eet_b200 import EET, paged
from eet_b200._lib import lib
from test_paged_cpu import _mha, _store

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _codes(**kw):
    f = dict(k_scale=16, v_scale=16, codes=1, ks_page=32, ks_head=16, vs_page=32, vs_head=16)
    f.update(kw)
    return paged._pack_codes(*f.values())


# (addresses that no call may follow: these calls end on the host)
_MHA = dict(q=16, k_cache=16, v_cache=16, out=16, pages=4, starts=4, lens=4, ws=0, ws_bytes=0)


@pytest.mark.parametrize("change,codes,message", [
    ({}, {}, b"NULL"), (_MHA, {"k_scale": 0}, b"NULL scales"), (_MHA, {"codes": 0}, b"kind of codes 0"), (_MHA, {"codes": 3}, b"kind of codes 3"),
    (_MHA, {"v_scale": 18}, b"4-byte aligned"), (dict(_MHA, kc_slot=136), {}, b"multiples of 16"), (dict(_MHA, q=24), {}, b"16-byte aligned"),
    (dict(_MHA, heads=7), {}, b"7 heads"), (dict(_MHA, head_dim=96), {}, b"head size 96"), (dict(_MHA, page_size=8), {}, b"page size 8"),
    (dict(_MHA, window=-1), {}, b"window"), (dict(_MHA, max_pages=4000, pages_stride=4000, max_len=64000), {}, b"workspace too small")])
def test_mha_refuses(change, codes, message):
    assert lib.eet_paged_mha_codes(_mha(**change) + _codes(**codes), None) != 0
    assert message in lib.eet_last_error()


def test_mha_of_nothing_is_no_error():
    for empty in (dict(tokens=0), dict(seqs=0)):
        assert lib.eet_paged_mha_codes(_mha(**empty) + _codes(), None) == 0
        assert lib.eet_paged_mha_codes_workspace_bytes(_mha(**empty) + _codes()) == 0
    assert lib.eet_paged_mha_codes(None, None) != 0 and b"NULL" in lib.eet_last_error()


@pytest.mark.parametrize("group", [1, 3, 8, 9, 16, 17, 32, 128])
def test_scratch_is_bounded_whatever_the_sizes(group):
    most = 148 * 2 * (256 + 3 * 16) * (128 + 2) * 4 + (1 << 16)     # two parts a CTA, of both kinds of tiles
    for tokens in (1, 2, 5, 64, 65, 777, 10 ** 6):
        for seqs in (1, 2, 33, 64, 3000):
            for max_tokens in (0, 1, 2, 17, tokens):
                for pages, max_len in ((0, 0), (1, 0), (4, 1), (4096, 0), (1 << 26, 0)):
                    need = lib.eet_paged_mha_codes_workspace_bytes(_mha(
                        heads=4 * group, kv_heads=4, tokens=tokens, seqs=seqs, max_tokens=max_tokens, max_pages=pages, pages_stride=pages,
                        max_len=max_len) + _codes())
                    assert 0 <= need <= most


_STORE = dict(k=16, v=16, k_cache=16, v_cache=16, pages=4, starts=4, lens=4, q=16, q_out=16, freqs=8)


@pytest.mark.parametrize("change,codes,message", [
    ({}, {}, b"NULL"), (_STORE, {"v_scale": 0}, b"NULL scales"), (_STORE, {"codes": -1}, b"kind of codes -1"),
    (dict(_STORE, vc_page=4104), {}, b"multiples of 16"), (dict(_STORE, rotary_dim=24), {}, b"rotary_dim 24")])
def test_store_refuses(change, codes, message):
    assert lib.eet_paged_store_codes(_store(**change) + _codes(**codes), None) != 0
    assert message in lib.eet_last_error()
    assert lib.eet_paged_store_codes(_store(tokens=0) + _codes(), None) == 0


def _load(**kw):
    f = dict(k_cache=16, v_cache=16, k_scale=16, v_scale=16, k_out=16, v_out=16, pages=4, starts=4, lens=4, tokens=3, seqs=2, kv_heads=2, head_dim=128,
             codes=1, bf16=0, num_pages=10, page_size=16, max_pages=4, pages_stride=4, ko_tok=256, ko_head=128, vo_tok=256, vo_head=128,
             kc_page=4096, kc_head=2048, kc_slot=128, vc_page=4096, vc_head=2048, vc_slot=128, ks_page=32, ks_head=16, vs_page=32, vs_head=16)
    f.update(kw)
    values = list(f.values())
    return paged._pack_load(*values[:29]) + paged._pack_codes(0, 0, 0, *values[29:])[24:]


@pytest.mark.parametrize("change,message", [
    ({"k_out": 0}, b"NULL"), ({"k_scale": 0}, b"NULL scales"), ({"codes": 5}, b"kind of codes 5"), ({"v_out": 8}, b"16-byte aligned"),
    ({"ko_tok": 257}, b"multiples of 8"), ({"kc_head": 2056}, b"multiples of 16"), ({"page_size": 24}, b"page size 24"), ({"head_dim": 80}, b"head size 80"),
    ({"tokens": -1}, b"tokens"), ({"codes": 0, "kc_slot": 132}, b"multiples of 8")])
def test_load_refuses(change, message):
    assert lib.eet_paged_load(_load(**change), None) != 0
    assert message in lib.eet_last_error()
    assert lib.eet_paged_load(_load(tokens=0), None) == 0


def _sample(**kw):
    f = dict(logits=16, uniform=4, temperatures=0, top_ps=0, min_ps=0, top_ks=0, tokens=8, logprobs=4, rows=2, vocab=100, type=0, row_stride=100,
             top_k=0, temperature=1.0, top_p=1.0, min_p=0.0)
    f.update(kw)
    return EET._pack_sample(*f.values())


@pytest.mark.parametrize("change,message", [
    ({"logits": 0}, b"NULL"), ({"uniform": 0}, b"NULL"), ({"vocab": 0}, b"0 tokens"), ({"vocab": (1 << 18) + 1, "row_stride": 1 << 20}, b"only 1 to 262144"),
    ({"type": 3}, b"type 3"), ({"row_stride": 99}, b"overlap"), ({"rows": -1}, b"rows"), ({"top_k": -1}, b"top_k"),
    ({"logits": 18, "type": 2}, b"aligned")])
def test_sample_refuses(change, message):
    assert lib.eet_sample_rows(_sample(**change), None) != 0
    assert message in lib.eet_last_error()
    assert lib.eet_sample_rows(_sample(rows=0), None) == 0


def test_tensors_of_the_wrong_kind_are_refused():
    codes, scale = torch.zeros(4, 2, 16, 128, dtype=torch.int8), torch.ones(4, 2, 16)
    with pytest.raises(RuntimeError, match="paged_load"):
        paged.paged_load(codes, codes, None, None, None, 3, k_scale=scale, v_scale=scale)
    with pytest.raises(RuntimeError, match="sample_rows"):
        EET.sample_rows(torch.zeros(2, 8), torch.zeros(2))


def test_structures_have_the_sizes_that_python_packs():
    text = open(os.path.join(ROOT, "include", "eet_b200.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    sizes = {"eet_paged_store_args": len(_store()), "eet_paged_mha_args": len(_mha())}
    for name, pack in (("paged_store_codes", _store() + _codes()), ("paged_mha_codes", _mha() + _codes()), ("paged_load", _load()),
                       ("sample_rows", _sample())):
        body = re.search(r"typedef struct \{([^}]*)\} eet_%s_args;" % name, text).group(1)
        total = 0
        for decl in filter(str.strip, body.split(";")):
            kind = decl.split()[0]
            total += sizes[kind] if kind in sizes else 8 * len(decl.split(","))
        assert total == len(pack), name


# ---- the oracle
def test_every_code_is_the_nearest():
    """Half the distance of two codes is never passed, and a value halfway goes to the even one."""
    gen = torch.Generator().manual_seed(0)
    for kind in MOST:
        y = torch.randn(500, 64, generator=gen).double() * torch.logspace(-6, 6, 500, dtype=torch.float64)[:, None]
        codes, scale = quantize64(y, kind)
        assert ((codes.double() * scale.double()[:, None] - y).abs() <= half_step(y, scale, kind) * (1 + 1e-12)).all()
    halves = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -3.5, 63.5, 126.5]])
    assert quantize64(halves, torch.int8)[0].tolist() == [[127, 0, 2, 2, 0, -4, 64, 126]]
    halves = torch.tensor([[448.0, 17.0, 19.0, 416.0 + 16, 1 + 1 / 16, 2.0 ** -10, 3 * 2.0 ** -10, -17.0]])
    assert quantize64(halves, torch.float8_e4m3fn)[0].double().tolist() == [[448, 16, 20, 448, 1, 0, 2 * 2.0 ** -9, -16]]
    assert quantize64(torch.zeros(2, 8), torch.int8)[1].tolist() == [1.0, 1.0]
    assert math.isfinite(quantize64(torch.full((1, 8), 3e-38), torch.int8)[1].item())
