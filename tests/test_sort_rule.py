"""Which way the sort of an embedding's ids takes (csrc/lf_rules.h, compiled for the host): loads that a thread makes one after the other stay few, whatever the
number of digits, and both sides of each line."""
import ctypes

import pytest

from helpers import host_library

SOURCE = """
#include "lf_rules.h"
extern "C" int adds_counts(long long groups, int bits) { return lf::sort_adds_counts(groups, bits); }
"""


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    lib = host_library(tmp_path_factory.mktemp("rule"), SOURCE)
    return lambda groups, bits: bool(lib.adds_counts(ctypes.c_longlong(groups), bits))


def test_loads_of_a_thread_are_few(rule):
    for bits in range(1, 12):
        spared = [groups for groups in range(1, 1025) if rule(groups, bits)]
        assert spared == list(range(1, len(spared) + 1)) and 8 <= len(spared)
        # four digits of all groups: fewer digits than threads make them no fewer
        assert 4 * len(spared) <= 64


@pytest.mark.parametrize("bits,most", [(4, 16), (7, 16), (8, 16), (9, 8), (10, 8), (11, 8)])
def test_both_sides_of_the_line(rule, bits, most):
    assert rule(most, bits) and not rule(most + 1, bits)
