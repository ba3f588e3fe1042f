"""Which sequences of a batched step read their common pages once (csrc/shared_group.h, compiled for the host) against trying all sets."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from conftest import PKG


@pytest.fixture(scope="module")
def find(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("host") / "libhost.so")
    subprocess.run(["g++", "-O2", "-ffp-contract=off", "-fPIC", "-shared", os.path.join(PKG, "csrc", "host_selftest.cpp"), "-o", out], check=True)
    lib = ctypes.CDLL(out)

    def call(tables, bt, heads, width=1024):
        """the members and the pages that they share"""
        n, stride = len(tables), max(1, max(len(t) for t in tables))
        flat = np.full((n, stride), -1, dtype=np.int32)
        for i, t in enumerate(tables):
            flat[i, :len(t)] = t
        lens = np.array([len(t) for t in tables], dtype=np.int32)
        members, tokens = ctypes.c_uint64(), ctypes.c_int32()
        p = lambda a: a.ctypes.data_as(ctypes.c_void_p)
        got = lib.b2_host_shared_group(p(flat), stride, p(lens), n, bt, heads, width, ctypes.byref(members), ctypes.byref(tokens))
        who = [i for i in range(n) if members.value >> i & 1]
        assert got == len(who) and tokens.value % bt == 0
        return who, tokens.value // bt
    return call


def pays(n, n_all, tokens, heads, width):
    if n < 2:
        return False
    if n < n_all:
        return n * tokens >= max(32768, 6144 * heads)
    if n * heads <= 16:
        return tokens >= 128
    return n * tokens >= (20480 if n > 16 and heads >= 4 and width >= 1024 else 16384)


def most(tables, bt, heads, width):
    """members times tokens of the best set: sequences with the same first d pages, for every d"""
    best = 0
    for d in range(1, max(len(t) for t in tables) + 1):
        sets = {}
        for t in tables:
            if len(t) >= d:
                sets[tuple(t[:d])] = sets.get(tuple(t[:d]), 0) + 1
        best = max([best] + [n * d * bt for n in sets.values() if pays(n, len(tables), d * bt, heads, width)])
    return best


def check(find, tables, bt, heads, width=1024):
    who, depth = find(tables, bt, heads, width)
    assert len(who) * depth * bt == most(tables, bt, heads, width)
    assert len({tuple(tables[i][:depth]) for i in who}) <= 1 and all(len(tables[i]) >= depth for i in who)
    assert not who or pays(len(who), len(tables), depth * bt, heads, width)
    return who, depth


def test_one_sequence_with_a_short_common_part_leaves_the_others_their_group(find):
    """32 behind 4096 common tokens, one that shares the first page of them alone"""
    for bt in (16, 64):
        doc = list(range(4096 // bt))
        tables = [doc + [1000 + i] for i in range(32)] + [[0, 5000, 5001]]
        assert check(find, tables, bt, 4) == (list(range(32)), 4096 // bt)
        assert check(find, tables[::-1], bt, 4)[0] == list(range(1, 33))


def test_groups_behind_a_common_header(find):
    """30 with one document beside 30 with the same header and another, shorter one; and the header alone for both where that is more"""
    header, a, b = [0], list(range(100, 163)), list(range(200, 232))
    tables = [header + (a if i % 2 else b) + [1000 + i] for i in range(60)]
    assert check(find, tables, 64, 4) == ([i for i in range(60) if i % 2], 64)
    long_header = list(range(500, 560))
    tables = [long_header + (a[:2] if i % 2 else b[:9]) + [1000 + i] for i in range(60)]
    assert check(find, tables, 64, 4) == (list(range(60)), 60)


def test_a_group_within_a_group(find):
    """chats that share more with some than with others, and end at different pages"""
    tables = [list(range(n)) for n in [3] * 30 + [50] * 20 + [70] * 10]
    assert check(find, tables, 64, 4) == (list(range(30, 60)), 50)
    tables = [list(range(2 * (i + 1))) for i in range(64)]                     # a chain: the best cut is in the middle
    check(find, tables, 64, 4)


@pytest.mark.parametrize("heads,width", [(1, 4096), (4, 1024), (4, 128), (7, 512), (8, 256), (8, 1024)])
def test_edges_of_the_rule(find, heads, width):
    common = list(range(5000))
    for n in (1, 2, 3, 4, 5, 16, 17, 63, 64):
        for others in (0, 1):
            for tokens in (64, 128, 192, 256, 512, *(t // n + more for t in (16384, 20480, 32768, 43008, 49152) for more in (0, 63, 64))):
                depth = tokens // 64
                if n + others <= 64:
                    check(find, [common[:depth] + [6000 + i] for i in range(n)] + [[9000]] * others, 64, heads, width)
    assert find([[], []], 64, heads, width) == ([], 0)


def test_where_every_sequence_for_itself_was_faster(find):
    """the measured points next to the edges, us a layer won or lost by reading common pages once"""
    for n, others, tokens, heads, width, won in [(32, 0, 512, 4, 1024, -2.5), (64, 0, 256, 4, 1024, -2.3), (32, 0, 512, 8, 1024, -2.7), (32, 0, 1024, 4, 1024, 9), (64, 0, 512, 4, 1024, 10),
                                                 (16, 0, 1024, 4, 1024, 2.5), (8, 0, 2048, 8, 1024, 5.3), (32, 0, 512, 8, 256, 21), (64, 0, 256, 8, 256, 16), (32, 0, 512, 1, 4096, 68),
                                                 (32, 1, 1024, 8, 256, -6), (16, 1, 2048, 8, 256, -6.9), (32, 1, 1024, 8, 1024, -8.2), (16, 1, 2048, 8, 1024, -5.3), (32, 1, 1024, 7, 512, -8.3),
                                                 (32, 1, 2048, 8, 256, 3.5), (57, 7, 1024, 8, 1024, 12.5), (26, 7, 2048, 8, 256, 2.8), (32, 1, 2048, 4, 1024, 19.5), (32, 1, 1024, 1, 4096, 74)]:
        common = list(range(tokens // 64))
        who, _ = find([common + [6000 + i] for i in range(n)] + [[9000 + i] for i in range(others)], 64, heads, width)
        assert (len(who) == n) == (won > 0), (n, others, tokens, heads, width)


def test_random_trees(find):
    rng = np.random.default_rng(5)
    for _ in range(1500):
        n, bt = int(rng.integers(1, 65)), int(rng.choice([16, 64, 512, 2048]))
        tables, fresh = [], 1000
        for i in range(n):
            t = list(tables[rng.integers(len(tables))]) if tables and rng.random() < 0.9 else []
            t = t[:int(rng.integers(0, len(t) + 1))] if rng.random() < 0.6 else t
            k = int(rng.integers(0, 30))
            tables.append(t + list(range(fresh, fresh + k)))
            fresh += k
        order = rng.permutation(n)
        check(find, [tables[i] for i in order], bt, int(rng.choice([1, 2, 4, 8])), int(rng.choice([128, 1024])))
