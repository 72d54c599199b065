"""Serving from a paged cache: what the calls refuse, and the frequencies of rotary positions, without a GPU."""
import ctypes
import math

import pytest
import torch

from eet_b200 import paged
from eet_b200._lib import lib


def _base(i, dim):
    return 10000.0 ** (-2.0 * i / dim)


def test_frequencies_without_scaling():
    freqs, magnitude = paged.rotary_frequencies(64, device="cpu")
    assert freqs.dtype == torch.float64 and magnitude == 1.0
    assert freqs.tolist() == [_base(i, 64) for i in range(32)]


def test_frequencies_linear_and_ntk():
    freqs, _ = paged.rotary_frequencies(32, scaling={"type": "linear", "factor": 4.0}, device="cpu")
    assert freqs.tolist() == [_base(i, 32) / 4.0 for i in range(16)]
    freqs, magnitude = paged.rotary_frequencies(32, scaling={"type": "ntk", "factor": 4.0}, device="cpu")
    # the fastest pair stays, the slowest is stretched by the factor
    assert freqs[0] == 1.0 and magnitude == 1.0
    assert math.isclose(freqs[15].item(), _base(15, 32) / 4.0, rel_tol=1e-14)


def test_frequencies_in_bands():
    length, low, high, factor = 4096.0, 1.0, 4.0, 8.0
    freqs, magnitude = paged.rotary_frequencies(
        128, scaling={"type": "bands", "factor": factor, "original": length, "low": low, "high": high}, device="cpu")
    assert magnitude == 1.0
    kinds = set()
    for i, f in enumerate(freqs.tolist()):
        wave = 2 * math.pi / _base(i, 128)
        if wave < length / high:
            kinds.add("stays")
            assert f == _base(i, 128)
        elif wave > length / low:
            kinds.add("stretched")
            assert math.isclose(f, _base(i, 128) / factor, rel_tol=1e-15)
        else:
            kinds.add("blend")
            s = (length / wave - low) / (high - low)
            assert math.isclose(f, (1 - s) * _base(i, 128) / factor + s * _base(i, 128), rel_tol=1e-13)
    assert kinds == {"stays", "stretched", "blend"}


def test_frequencies_yarn():
    factor, length = 16.0, 4096.0
    freqs, magnitude = paged.rotary_frequencies(128, scaling={"type": "yarn", "factor": factor, "original": length}, device="cpu")
    assert math.isclose(magnitude, 0.1 * math.log(factor) + 1)
    ratio = [f / _base(i, 128) for i, f in enumerate(freqs.tolist())]
    index = lambda turns: 128 * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(10000.0))  # noqa: E731
    low, high = math.floor(index(32.0)), math.ceil(index(1.0))
    assert all(r == 1.0 for r in ratio[:low + 1])
    assert all(math.isclose(r, 1 / factor, rel_tol=1e-14) for r in ratio[high:])
    assert all(a > b for a, b in zip(ratio[low:high], ratio[low + 1:high + 1]))
    _, magnitude = paged.rotary_frequencies(128, scaling={"type": "yarn", "factor": 16.0, "original": 4096, "magnitude": 1.5},
                                            device="cpu")
    assert magnitude == 1.5


@pytest.mark.parametrize("dim,base,scaling", [
    (20, 1e4, None), (0, 1e4, None), (64, 1.0, None), (64, 1e4, {"type": "linear", "factor": 0.0}),
    (64, 1e4, {"type": "stretch", "factor": 2.0}), (64, 1e4, {"type": "linear", "factor": 2.0, "original": 4096}),
    (64, 1e4, {"type": "bands", "factor": 2.0, "original": 4096, "low": 4.0, "high": 4.0})])
def test_frequencies_refuse(dim, base, scaling):
    with pytest.raises(RuntimeError, match="rotary_frequencies"):
        paged.rotary_frequencies(dim, base, scaling, device="cpu")


def test_tensors_of_the_wrong_kind_are_refused():
    q = torch.zeros(2, 4, 128, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA fp16 or bf16"):
        paged.apply_rotary(q, None, None, None)
    with pytest.raises(RuntimeError, match="neither"):
        paged.apply_rotary(None, None, None, None)
    with pytest.raises(RuntimeError, match="CUDA fp16 or bf16"):
        paged.paged_mha(q, None, None, None, None, None)
    with pytest.raises(RuntimeError, match="CUDA fp16 or bf16"):
        paged.paged_store(q.float(), None, None, None, None, None, None)


# The C entry points refuse on the host, before anything is launched.  The defaults below pass every check but that for NULL
# pointers, which comes last.
def _mha(**kw):
    f = dict(q=0, k_cache=0, v_cache=0, out=0, pages=0, starts=0, lens=0, first_key=0, slopes=0, tokens=3, seqs=2, heads=8,
             kv_heads=2, head_dim=128, bf16=0, num_pages=10, page_size=16, max_pages=4, pages_stride=4, q_tok=1024, q_head=128,
             o_tok=1024, o_head=128, kc_page=4096, kc_head=2048, kc_slot=128, vc_page=4096, vc_head=2048, vc_slot=128, window=0,
             max_tokens=2, max_len=64, scale=0.1, ws=0, ws_bytes=0)
    f.update(kw)
    *fields, ws, ws_bytes = f.values()
    return paged._pack_mha(*fields) + paged._pack_scratch(ws, ws_bytes)


@pytest.mark.parametrize("change,message", [
    ({}, b"NULL"), ({"head_dim": 80}, b"head size 80"), ({"page_size": 48}, b"page size 48"), ({"page_size": 8}, b"page size 8"),
    ({"heads": 7}, b"7 heads"), ({"heads": 0}, b"0 heads"), ({"heads": 512}, b"512 heads"), ({"kv_heads": 0}, b"number of heads"),
    ({"window": -1}, b"window"), ({"q_tok": 1028}, b"multiples of 8"), ({"vc_slot": 132}, b"multiples of 8"),
    ({"tokens": -1}, b"tokens"), ({"seqs": -1}, b"sequences"), ({"pages_stride": 3}, b"overlap"),
    ({"max_pages": 1 << 28, "pages_stride": 1 << 28}, b"2^31"),
    ({"max_pages": (1 << 27) - 1, "pages_stride": 1 << 28}, b"2^31"), ({"num_pages": -1}, b"pages")])
def test_mha_refuses(change, message):
    assert lib.eet_paged_mha(_mha(**change), None) != 0
    assert message in lib.eet_last_error()


def test_nothing_to_do_is_no_error():
    assert lib.eet_paged_mha(_mha(tokens=0), None) == 0
    assert lib.eet_paged_mha(_mha(seqs=0), None) == 0
    assert lib.eet_paged_mha_workspace_bytes(_mha(tokens=0)) == 0
    assert lib.eet_paged_mha(None, None) != 0 and b"NULL" in lib.eet_last_error()


@pytest.mark.parametrize("group", [1, 3, 16, 17, 32, 128])
def test_scratch_is_bounded_whatever_the_sizes(group):
    """Any mix of chunks, single tokens and sequences that ask nothing; the work is planned before anything is launched."""
    most = 148 * 2 * (256 + 16) * (128 + 2) * 4 + (1 << 16)     # two parts a CTA, of both kinds of tiles
    for tokens in (1, 2, 5, 64, 65, 777, 10 ** 6):
        for seqs in (1, 2, 33, 64, 3000):
            for max_tokens in (0, 1, 2, 17, tokens):
                for pages, max_len in ((0, 0), (1, 0), (4, 1), (4096, 0), (1 << 26, 0)):
                    for window in (0, 1, 1000):
                        need = lib.eet_paged_mha_workspace_bytes(_mha(
                            heads=4 * group, kv_heads=4, tokens=tokens, seqs=seqs, max_tokens=max_tokens, max_pages=pages,
                            pages_stride=pages, max_len=max_len, window=window))
                        assert 0 <= need <= most


def _store(**kw):
    f = dict(q=0, k=0, v=0, q_out=0, k_cache=0, v_cache=0, pages=0, starts=0, lens=0, positions=0, freqs=0, tokens=3, seqs=2,
             heads=8, kv_heads=2, head_dim=128, rotary_dim=128, interleaved=0, bf16=0, num_pages=10, page_size=16, max_pages=4,
             pages_stride=4, q_tok=1024, q_head=128, k_tok=256, k_head=128, v_tok=256, v_head=128, qo_tok=1024, qo_head=128,
             kc_page=4096, kc_head=2048, kc_slot=128, vc_page=4096, vc_head=2048, vc_slot=128, magnitude=1.0)
    f.update(kw)
    return paged._pack_store(*f.values())


@pytest.mark.parametrize("change,message", [
    ({}, b"NULL"), ({"rotary_dim": 136}, b"rotary_dim 136"), ({"rotary_dim": 24}, b"rotary_dim 24"), ({"head_dim": 96}, b"head size 96"),
    ({"page_size": 512}, b"page size 512"), ({"k_tok": 257}, b"multiples of 8"), ({"k": 8, "v": 16, "k_cache": 16, "v_cache": 16,
     "pages": 4, "starts": 4, "lens": 4, "q": 16, "q_out": 16, "freqs": 8}, b"16-byte aligned")])
def test_store_refuses(change, message):
    if "k" not in change:
        change = dict(change, k=16, v=16, k_cache=16, v_cache=16, pages=4, starts=4, lens=4, q=16, q_out=16, freqs=8) if change else change
    assert lib.eet_paged_store(_store(**change), None) != 0
    assert message in lib.eet_last_error()


def _rotary(**kw):
    f = dict(q=0, k=0, q_out=0, k_out=0, positions=0, freqs=0, tokens=3, heads=8, kv_heads=2, head_dim=128, rotary_dim=64,
             interleaved=0, bf16=0, q_tok=1024, q_head=128, k_tok=256, k_head=128, qo_tok=1024, qo_head=128, ko_tok=256,
             ko_head=128, magnitude=1.0)
    f.update(kw)
    return paged._pack_rotary(*f.values())


@pytest.mark.parametrize("change,message", [
    ({}, b"NULL"), ({"head_dim": 264}, b"head size 264"), ({"head_dim": 24}, b"head size 24"), ({"rotary_dim": 0}, b"rotary_dim 0"),
    ({"rotary_dim": 144}, b"rotary_dim 144"), ({"tokens": -1}, b"tokens"), ({"heads": -1}, b"heads")])
def test_rotary_refuses(change, message):
    assert lib.eet_rotary(_rotary(**change), None) != 0
    assert message in lib.eet_last_error()


def test_structures_have_the_sizes_that_python_packs():
    """Fields of 8 bytes each, in the order of the header."""
    import os
    import re
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "eet_b200.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name, pack in (("rotary", _rotary()), ("paged_store", _store()), ("paged_mha", _mha())):
        body = re.search(r"typedef struct \{([^}]*)\} eet_%s_args;" % name, text).group(1)
        fields = [f for decl in body.split(";") if decl.strip() for f in decl.split(",")]
        assert 8 * len(fields) == len(pack)
    assert ctypes.sizeof(ctypes.c_void_p) == 8


def test_rows_of_a_sequence_whatever_starts_holds(tmp_path):
    """How many rows of q a sequence has, by the kernels' own expression compiled for the host: never one outside q, also where the
    difference of two bad starts would not fit 32 bits (which the compiler's check for that turns into an abort)."""
    import os
    import re
    import subprocess
    share = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "eet_b200", "csrc", "paged_share.cuh")
    text = open(share).read()
    seq = re.search(r"PgSeq pg_seq\([^)]*\)\s*\{(.*?)\n\}", text, re.S).group(1)
    tokens = re.search(r"s\.tokens = (.*?);", seq).group(1).replace("s.row0", "row0").replace("a.tokens", "tokens")
    helper = re.search(r"constexpr __host__ __device__ int pg_rows_of\(.*?\n\}", text, re.S)
    source = (helper.group(0).replace("__host__ __device__", "") if helper else "") + """
        #include <algorithm>
        #include <cstdio>
        #include <cstdlib>
        using std::max;
        using std::min;
        int main(int, char** v)
        {
            const int row0 = (int)std::atoll(v[1]), end = (int)std::atoll(v[2]), tokens = (int)std::atoll(v[3]);
            std::printf("%%d", %s);
        }
        """ % tokens
    source = source.replace("max(", "max<int>(").replace("min(", "min<int>(")
    (tmp_path / "rows.cc").write_text(source)
    program = str(tmp_path / "rows")
    subprocess.run(["g++", "-std=c++17", "-fsanitize=signed-integer-overflow", "-fsanitize-undefined-trap-on-error", "-o", program,
                    str(tmp_path / "rows.cc")], check=True)
    low, high = -2 ** 31, 2 ** 31 - 1
    for tokens in (1, 100, high):
        for row0 in (low, -1, 0, 1, 50, 100, high):
            for end in (low, low + 1, -1, 0, 1, 50, 51, 100, high):
                got = subprocess.run([program, str(row0), str(end), str(tokens)], check=True, capture_output=True, text=True).stdout
                assert int(got) == (max(0, min(end, tokens) - row0) if row0 >= 0 else 0), (row0, end, tokens)
