"""The calls of tests/products_plans.py take the ways through the library that they stand for (CPU): a changed figure in the
model's tables can not silently leave a kernel without a test."""

import pytest
from products_plans import CUTS, DW, INT8, ROWS, ROWS_TURNED, Plans, counts


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    return Plans(str(tmp_path_factory.mktemp("plans")))


def last_round(tiles):
    left = tiles % 256
    return 0 if left == 0 else 4 if left <= 64 else 2 if left <= 128 else 1


def up(a, b):
    return -(-a // b)


def test_calls_take_the_ways_they_are_listed_for(plans):
    for turned, cases in ((False, ROWS), (True, ROWS_TURNED)):
        for size, t, n, k, g, cut, split, pack, parts in cases:
            assert plans.rows(size, t, n, k, g, turned) == (cut, split, pack), (size, t, n, k, g, turned)
            if cut == "PIPE256":
                assert last_round(sum(up(c, 256) for c in counts(t, g)) * up(n, 256)) == parts
    for size, t, n, k, g, cut, split, pack, parts in DW:
        assert plans.dw(size, t, n, k, g) == (cut, split, pack), (size, t, n, k, g)
        if cut == "PIPE256":
            assert last_round(g * up(n, 256) * up(k, 256)) == parts
    for out_bytes, m, n, k, cut, split, pack, parts in INT8:
        assert plans.int8(out_bytes, m, n, k) == (cut, split, pack), (out_bytes, m, n, k)
        if cut == "PIPE256":
            assert last_round(up(m, 256) * up(n, 256)) == parts


def test_every_way_is_listed():
    """all cuts of each product and type, whole and split, of operands as they are and copied"""

    def ways(cases, size):
        return {(c[-4], c[-3] > 1, c[-2]) for c in cases if c[0] == size}

    direct, plain = {"DIRECT16", "DIRECT32"}, {"PLAIN64", "PLAIN128"}
    for cases, small in ((ROWS, (2, 4, 8)), (ROWS_TURNED, (4, 8)), (DW, (4, 8))):
        for size in (2, 4, 8):
            got = ways(cases, size)
            pipes = {2: {"PIPE64", "PIPE128", "PIPE256", "TWIN64"}, 4: {"PIPE64", "PIPE128"}, 8: {"PIPE64"}}[size]
            assert {c for c, _, _ in got} == (direct if size in small else set()) | plain | pipes
            assert plain <= {c for c, split, _ in got if split} and pipes <= {c for c, _, pack in got if pack}
            assert {c for c, split, _ in got if split} & pipes  # a split of k, joined
    assert {c for c, _, _ in {(c[-4], c[-3], c[-2]) for c in INT8}} == set(CUTS)
    assert {c[-4] for c in INT8 if c[-2]} == {"PIPE64", "PIPE128", "PIPE256", "TWIN64"}
    for cases in (ROWS, ROWS_TURNED, DW, INT8):
        assert {c[-1] for c in cases if c[-4] == "PIPE256"} >= {1, 2, 4}
