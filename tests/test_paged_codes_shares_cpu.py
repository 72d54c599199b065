"""How the warps of a block find their share of the work of the attention over codes: what the kernels' source promises."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "eet_b200", "csrc")


def _source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def _constant(text, name):
    value = re.search(r"constexpr int %s = (\w+);" % name, text).group(1)
    return int(value) if value.isdigit() else _constant(text, value)


def test_every_warp_has_a_place_for_its_sum():
    """With more than 32 sequences each warp of a block leaves a sum in PgFound::warp_sum, and all of them read all sums while one
    already writes what it has found behind them: a block of more warps than places would overwrite that, and warps would go on with
    different shares of the work."""
    share, rows, tiles, codes = (_source(n) for n in ("paged_share.cuh", "paged_rows.cu", "paged_tc.cu", "paged_codes.cu"))
    assert "f.warp_sum[warp]" in share and "warp = tid >> 5" in share
    length = re.search(r"long long warp_sum\[(\w+)\]", share).group(1)
    places = int(length) if length.isdigit() else _constant(share, length)
    threads = [_constant(rows, "kPwThreads"), _constant(tiles, "kPgThreads"), _constant(tiles, "kPgCodesThreads"),
               32 * int(re.search(r"static constexpr int kWarps = (\d+);", codes).group(1))]
    bounds = set(re.findall(r"__launch_bounds__\((kP\w+Threads|32 \* PcShape[^,]*, kRows>::kWarps)", rows + tiles + codes))
    assert bounds == {"kPwThreads", "kPgThreads", "kPgCodesThreads", "32 * PcShape<D, kRows>::kWarps"}
    assert max(threads) <= 32 * places
