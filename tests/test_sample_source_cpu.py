"""Rules of the sampling kernel's source that no run can show without a race: read from the text."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "eet_b200", "csrc")


def _body(text, head):
    """The braces behind `head`, and what they hold."""
    start = text.index("{", text.index(head))
    depth = 0
    for i in range(start, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[start:i + 1]
    raise AssertionError(head)


def test_a_bracket_is_read_by_all_before_the_next_is_written():
    """narrow() ends with a read of shared memory that its next call writes, also into the other CTAs' memory: between two of them every way
    goes through a barrier of the cluster.  gather() and cut_list() have one, and so has the second histogram."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "sample.cu")).read())
    narrow = _body(text, "SaBracket narrow(")
    assert re.search(r"barrier\(\);\s*return sm\.bracket;\s*\}$", narrow)
    assert "barrier()" in _body(text, "Sums exchange(") and "return exchange(" in _body(text, "Sums gather(")
    assert "barrier();" in _body(text, "SaCut cut_list(")
    find = _body(text, "SaCut find(")
    assert find.count("narrow(") == 3
    first, second, third = (m.start() for m in re.finditer(r"narrow\(", find))
    # by mass: a list, whose calls have barriers, or a barrier of its own
    between = find[first:second]
    lists = _body(between, "if (b.count <= kSaList)")
    assert "gather(" in lists and "cut_list(" in lists
    otherwise = between[between.index(lists) + len(lists):]
    assert re.match(r"\s*else \{\s*barrier\(\);\s*\}", otherwise)
    # the second histogram lies behind the list's return, and has barriers that every way passes
    way = find[second:third]
    assert re.search(r"\n        barrier\(\);", way[way.index("return cut_list("):])
