"""The rule by which tree attention's running maximum moves
(``csrc/running_max.cuh``), compiled for the host: whether a score asks for a
rise and whether its row rises are one question, so a tile that has risen once
asks no more."""
from __future__ import annotations

import ctypes
import os
import subprocess

import numpy as np
import pytest

import running_max as M

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F = np.float32
SRC = """
#include "running_max.cuh"
using namespace halo::tree;
extern "C" float no_max() { return kNoMax; }
extern "C" float headroom(float scale_log2) { return raw_headroom(scale_log2); }
extern "C" float excess_of(float s, float m) { return excess(s, m); }
extern "C" int rises_over(float s, float m, float h) { return rises(s, m, h); }
"""


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    d = tmp_path_factory.mktemp("rule")
    src, lib = d / "rule.cpp", d / "rule.so"
    src.write_text(SRC)
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC",
                    "-I" + os.path.join(ROOT, "halo_b200", "csrc"), str(src), "-o", str(lib)],
                   check=True)
    so = ctypes.CDLL(str(lib))
    f = ctypes.c_float
    for name, res, n in (("no_max", f, 0), ("headroom", f, 1), ("excess_of", f, 2),
                         ("rises_over", ctypes.c_int, 3)):
        getattr(so, name).restype = res
        getattr(so, name).argtypes = [f] * n
    return so


def _tile(rule, scores, m, h, first):
    """A tile as the kernel takes it: the maximum after it, and how often a
    score asked for a rise.  Ends by the rule alone, without a bound."""
    asked = 0
    while first or any(rule.rises_over(s, m, h) for s in scores):
        asked += not first
        assert asked <= 3, "the tile asks for a rise again and again"
        top = max(scores)
        if rule.rises_over(top, rule.no_max() if first else m, h):
            m = top
        elif first:
            m = rule.no_max()
        first = False
    return m, asked


@pytest.mark.parametrize("D", [64, 128])
def test_a_tile_rises_at_most_once(rule, D):
    scale = F(F(1 / np.sqrt(D)) * M.LOG2E)
    h = rule.headroom(scale)
    rng = np.random.default_rng(D)
    windows = 0
    for _ in range(3000):
        s0 = F(rng.uniform(1, 10) * 10.0 ** rng.integers(0, 9) * rng.choice([-1, 1]))
        later = [M.at_headroom(s0, scale, n) for n in (-2, -1, 0, 1, 2)]
        c = M.split_window(s0, scale)
        if c is not None:
            windows += 1
            later.append(c)
        for s in later:
            m, asked = _tile(rule, [float(s0)], 0.0, h, True)
            assert m == s0 and asked == 0
            m2, asked = _tile(rule, [float(s), float(s0)], m, h, False)
            assert asked <= 1 and m2 == (s if asked else s0)
            # what is left of the tile's excess is within the headroom
            assert rule.excess_of(s, m2) <= h
    assert windows > 500          # such scores are common, not made up


def test_the_instance_of_128_columns(rule):
    """Scores whose two roundings disagree: 35.494537, then 98.231064."""
    s0, s1 = F(35.494537), F(98.231064)
    scale = F(F(1 / np.sqrt(128)) * M.LOG2E)
    m = F(s0 * scale)
    assert F(np.longdouble(s1) * np.longdouble(scale) - np.longdouble(m)) > 8
    assert not F(s1 * scale) > F(m + F(8))
    m, asked = _tile(rule, [float(s1)], s0, rule.headroom(scale), False)
    assert asked <= 1


@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e-3, 0.125, 1.0, 1e3, 1e30])
def test_scores_of_any_size_end(rule, scale):
    """Up to the largest numbers; rows that see nothing; infinities and NaN."""
    scale = F(F(scale) * M.LOG2E)
    h = rule.headroom(scale)
    big = float(np.finfo(np.float32).max)
    some = [0.0, 1.0, -1.0, 1.5e9, 3e9, -3e9, 1e20, -1e20, 1e30, -2e30, big, -big, np.inf, -np.inf,
            np.nan]
    for a in some:
        for b in some:
            m, asked = _tile(rule, [a], 0.0, h, True)
            assert asked <= 1
            if np.isfinite(a) and a > -big and h < big:
                assert m == F(a)
            if a == -np.inf:
                assert m == rule.no_max()
            if not np.isnan(b):
                m, asked = _tile(rule, [b], m, h, False)
                assert asked <= 1 and not rule.rises_over(b, m, h)


def test_rounding_keeps_the_order_of_excesses(rule):
    """The largest score has the largest excess, so the vote over all scores
    and the rise of a row's largest one agree."""
    rng = np.random.default_rng(3)
    for _ in range(300):
        m = F(rng.normal() * 10.0 ** rng.integers(-3, 12))
        s = np.sort((rng.normal(size=50) * 10.0 ** rng.integers(-3, 12)).astype(F))
        e = [rule.excess_of(x, m) for x in s]
        assert e == sorted(e)
        assert all(F(F(x) - m) == F(y) for x, y in zip(s, e))
