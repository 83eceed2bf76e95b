"""Which way the gradient of an embedding takes (csrc/lf_rules.h, compiled for the host).  Its sort: loads that a thread makes one after the other stay few, whatever the
number of digits.  Its sums in float32: both sides of each line.  The times behind the lines stand at the rules."""
import ctypes

import pytest

from helpers import host_library

SOURCE = """
#include "lf_rules.h"
extern "C" int adds_counts(long long groups, int bits) { return lf::sort_adds_counts(groups, bits); }
extern "C" int by_slice(long long ids, long long rows, long long dim) { return lf::sums_by_slice(ids, rows, dim); }
"""


def rules(tmp_path_factory):
    lib, size = host_library(tmp_path_factory.mktemp("rule"), SOURCE), ctypes.c_longlong
    return lambda groups, bits: bool(lib.adds_counts(size(groups), bits)), lambda *sizes: bool(lib.by_slice(*map(size, sizes)))


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    return rules(tmp_path_factory)[0]


@pytest.fixture(scope="module")
def by_slice(tmp_path_factory):
    return rules(tmp_path_factory)[1]


def test_loads_of_a_thread_are_few(rule):
    for bits in range(1, 12):
        spared = [groups for groups in range(1, 1025) if rule(groups, bits)]
        assert spared == list(range(1, len(spared) + 1)) and 8 <= len(spared)
        # four digits of all groups: fewer digits than threads make them no fewer
        assert 4 * len(spared) <= 64


@pytest.mark.parametrize("bits,most", [(4, 16), (7, 16), (8, 16), (9, 8), (10, 8), (11, 8)])
def test_both_sides_of_the_line(rule, bits, most):
    assert rule(most, bits) and not rule(most + 1, bits)


@pytest.mark.parametrize("ids,rows,dim,slices", [
    (1, 65_104, 576, True), (130_208, 65_104, 576, True), (130_209, 65_104, 576, False), (0, 10, 513, True), (100, 1000, 512, False), (937, 60_000, 640, True), (48_828, 48_828, 768, True),
    (48_828, 48_828, 769, True), (1500, 48_828, 769, False),
    (19_908, 24_964, 1792, True), (18_723, 24_964, 1792, True), (18_722, 24_964, 1792, False), (37_446, 24_964, 1792, True), (37_447, 24_964, 1792, False), (6250, 25_000, 1792, False),
    (2663, 2663, 2816, False), (5461, 5461, 3584, True), (4682, 4682, 3584, True), (4681, 4681, 3584, False),
    (30_000, 30_000, 1024, False), (18_310, 18_310, 2048, False), (8000, 8000, 4096, False), (17, 28_215, 3824, False)])
def test_slices_one_after_the_other(by_slice, ids, rows, dim, slices):
    assert by_slice(ids, rows, dim) == slices
