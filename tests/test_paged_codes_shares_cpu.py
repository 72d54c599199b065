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


def _body(text, head):
    """The braces behind `head`, and what they hold."""
    start = text.index("{", text.index(head))
    depth = 0
    for i in range(start, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[start:i + 1]
    raise AssertionError(head)


def _passed_by_b(new, lens, heads, kv_heads, whole, ctas=148, extra=3, keys=128):
    """For each first block that tile b of a pair has in a piece: how many blocks it has passed without a wait in front of that, since its
    last turn.  The walk of PgShare: tiles of 2 (128 / group) tokens, each `extra` blocks more than it has, the shares equal."""
    tokens = 2 * (128 // (heads // kv_heads))
    tiles = []                                       # (blocks, blocks of which b has a turn)
    for t, n in zip(new, lens):
        for _ in range(kv_heads):
            for at in range(0, t, tokens):
                blocks = -(-(n - t + min(at + tokens, t)) // keys)
                tiles.append((blocks, t - at <= tokens // 2))
    total = sum(b + extra for b, _ in tiles)
    pieces, place = [[] for _ in range(ctas)], 0
    begin = [total // ctas * c + min(c, total % ctas) for c in range(ctas + 1)]
    for blocks, split in tiles:
        for c in range(ctas):
            if whole:
                n = blocks if begin[c] <= place < begin[c + 1] else 0
            else:
                low, high = (min(max(begin[c + i] - place - extra, 0), blocks) for i in (0, 1))
                n = high - low
            if n:
                pieces[c].append((n, split))
        place += blocks + extra
    passed = []
    for share in pieces:
        ahead = 0
        for n, split in share:
            if split and n == 1:
                ahead += 1
                continue
            passed.append(ahead)
            ahead = 0
    return passed


def test_the_warps_of_tile_b_come_to_their_first_block_from_far_ahead():
    """Ordinary loads of few new tokens: in some shares tile b has passed six blocks and more, a turn of the ring of scales, without a wait.
    A wait by parity would then end before its data is there, so the softmax waits for the scores of a piece's first block first, in front
    of everything that it reads of the scales."""
    tiles = _source("paged_tc.cu")
    ring = int(re.search(r"kPlaces = 3, kScales = (\d+);", tiles).group(1))
    import random
    rng = random.Random(1)
    loads = [([5] * 256, [rng.randint(60, 260) for _ in range(256)], 32, 8),
             ([17] * 64, [17 + rng.randint(20, 250) for _ in range(64)], 32, 32)]
    for new, lens, heads, kv_heads in loads:
        assert any(max(_passed_by_b(new, lens, heads, kv_heads, whole)) >= ring for whole in (False, True))
    assert max(_passed_by_b([512], [8704], 32, 8, False)) < ring      # (a chunk's pieces are long)
    # s_full of a piece's first block is waited for in front of the loop over its blocks, which looks at the scales.
    softmax = tiles[tiles.index("PgReference ref = {1.0f, -kPgNone};"):]
    loop = _body(softmax, "for (int j = turns.first;")
    front = softmax[:softmax.index(loop)]
    guard = re.search(r"if \(kCodes && turns\.any\(\)\) ok = tc_wait_warp\(&sm\.s_full\[x\], \(uint32_t\)\(used & 1\), &sm\.abort\);\s*"
                      r"for \(int j = turns\.first; j < turns\.end && ok; j \+= turns\.stride\) $", front)
    assert guard, "the scores of the first block"
    assert "scales_full" in loop and "scales" not in front
