"""What the paged cache's C ABI refuses beyond test_cpu_paged.py, and the rule on overlapping caches against brute force."""
import ctypes
import itertools
import os
import random
import subprocess

import pytest

from conftest import ROOT
from b200_hpu_ops import abi
from test_cpu_paged import AT, BAD, UNSUPPORTED, _append, _attend, _plan

CSRC = os.path.join(ROOT, "gaudi-pytorch-bridge_b200", "csrc")


# ----------------------------------------------------------------------------- caches that overlap
@pytest.mark.parametrize("kw", [
    dict(k_cache_head_stride=4), dict(k_slot_stride=64), dict(v_page_stride=1024), dict(v_cache_head_stride=0), dict(k_slot_stride=0), dict(v_page_stride=0),
    dict(k_cache=AT, v_cache=AT), dict(k_cache=AT, v_cache=AT + 64), dict(k_cache=AT, v_cache=AT + 2048 * 7 + 128),
    dict(k_page_stride=4096, v_page_stride=4096, v_cache=AT + 2048 - 64), dict(k_page_stride=-2048, v_page_stride=-2048, v_cache=AT + 2048),
])
def test_append_refuses_caches_that_overlap(kw):
    """8 pages of 16 slots of two heads of 64 one-byte values; where a case names no v_cache it lies far behind k_cache."""
    assert _append(**{**dict(v_cache=AT << 4), **kw}) == BAD


@pytest.fixture(scope="module")
def layouts(tmp_path_factory):
    at = tmp_path_factory.mktemp("layout")
    (at / "layout.cpp").write_text("""
#include "paged_layout.h"
using b200q::CacheLayout;
static CacheLayout layout(long at, long elt, long dim, const long* n, const long* s) {
  return CacheLayout(reinterpret_cast<void*>(at), elt, dim, {n[0], n[1], n[2]}, {s[0], s[1], s[2]});
}
extern "C" int layout_apart(long at, long elt, long dim, const long* n, const long* s) { return layout(at, elt, dim, n, s).apart(); }
extern "C" int layouts_apart(long elt, long dim, long at0, const long* n0, const long* s0, long at1, const long* n1, const long* s1) {
  return layout(at0, elt, dim, n0, s0).apart_from(layout(at1, elt, dim, n1, s1));
}
""")
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-I", CSRC, str(at / "layout.cpp"), "-o", str(at / "layout.so")], check=True)
    lib = ctypes.CDLL(str(at / "layout.so"))
    three = ctypes.c_long * 3

    def one(at, elt, dim, n, s):
        return bool(lib.layout_apart(ctypes.c_long(at), ctypes.c_long(elt), ctypes.c_long(dim), three(*n), three(*s)))

    def two(elt, dim, a, b):
        (at0, n0, s0), (at1, n1, s1) = a, b
        return bool(lib.layouts_apart(ctypes.c_long(elt), ctypes.c_long(dim), ctypes.c_long(at0), three(*n0), three(*s0), ctypes.c_long(at1), three(*n1), three(*s1)))

    return one, two


def _places(at, elt, dim, n, s):
    """Every byte of a cache, once for each head of a slot that it belongs to."""
    for i in itertools.product(*map(range, n)):
        first = at + sum(x * y for x, y in zip(i, s)) * elt
        yield from range(first, first + dim * elt)


def test_layouts_against_brute_force(layouts):
    one, two = layouts
    rng, base = random.Random(5), 1 << 16
    shared = 0
    for _ in range(4000):
        elt, dim, n = rng.choice([1, 2]), rng.choice([4, 8]), [rng.randint(1, 3) for _ in range(3)]
        s = [rng.choice([-1, 1, 1, 1]) * 4 * rng.randint(0, 14) for _ in range(3)]
        places = list(_places(base, elt, dim, n, s))
        if one(base, elt, dim, n, s):
            assert len(set(places)) == len(places)
            shift = elt * rng.randint(-60, 60)
            other = (base + shift, n, s if rng.random() < 0.7 else [4 * rng.randint(0, 14) for _ in range(3)])
            if not one(other[0], elt, dim, *other[1:]):
                continue
            meet = bool(set(places) & set(_places(other[0], elt, dim, *other[1:])))
            said = two(elt, dim, (base, n, s), other)
            assert not (said and meet)
            if other[2] is s:
                assert said != meet  # (exact where the strides are the same)
                shared += meet
            assert said == two(elt, dim, other, (base, n, s))
    assert shared > 100


def test_layouts_that_are_taken(layouts):
    """Any order of the three, pitches between them, both caches as halves of one allocation at any depth, keys and values in different orders."""
    one, two = layouts
    n, dim = [5, 16, 3], 8
    for order in itertools.permutations(range(3)):
        for pitch in (0, 24):
            s, step = [0, 0, 0], dim
            for i in order:
                s[i] = step
                step = step * n[i] + pitch
            assert one(4096, 2, dim, n, s)
            assert two(2, dim, (4096, n, s), (4096 + 2 * step, n, s))
            for depth in range(3):  # the second cache behind the first one within dimension `depth` of the order
                t, step = [0, 0, 0], dim
                for at, i in enumerate(order):
                    if at == depth:
                        shift, step = step, 2 * step
                    t[i] = step
                    step *= n[i]
                assert one(4096, 2, dim, n, t) and two(2, dim, (4096, n, t), (4096 + 2 * shift, n, t))
                assert not two(2, dim, (4096, n, t), (4096 + 2 * shift - 2, n, t))
    page = 2 * 16 * 3 * dim
    assert two(2, dim, (4096, n, [page, 3 * dim, dim]), (4096 + page, n, [page, dim, 16 * dim]))
    assert two(2, dim, (4096, [0, 16, 3], [page, 24, 8]), (4096, [0, 16, 3], [page, 24, 8]))  # no pages


# ----------------------------------------------------------------------------- addresses between elements
@pytest.mark.parametrize("name", ["context", "new", "table", "free", "head", "start", "lens", "next", "slots", "positions"])
def test_plan_refuses_addresses_between_elements(name):
    assert _plan(**{name: AT + 2}) == UNSUPPORTED
    if name in ("slots", "positions"):
        assert _plan(**{name: AT + 4}) == UNSUPPORTED


@pytest.mark.parametrize("kw", [dict(slot_map=AT + 4), dict(cos_sin=AT, rotary_dim=64, positions=AT + 4), dict(k_scale=AT + 2), dict(v_scale=AT + 1),
                                dict(q_scale=AT + 2)])
def test_append_refuses_addresses_between_elements(kw):
    assert _append(**{**dict(v_cache=AT << 4), **kw}) == UNSUPPORTED


@pytest.mark.parametrize("kw", [dict(q=AT + 1), dict(out=AT + 1), dict(out=AT + 2, out_dtype=abi.F32), dict(k_cache=AT + 1, cache_dtype=abi.BF16),
                                dict(v_cache=AT + 1, cache_dtype=abi.BF16), dict(block_table=AT + 2), dict(kv_lens=AT + 1), dict(lse=AT + 2),
                                dict(k_scale_inv=AT + 2), dict(v_scale_inv=AT + 1), dict(out_scale=AT + 3)])
@pytest.mark.parametrize("plain", [0, 1])
def test_attention_refuses_addresses_between_elements(kw, plain):
    assert _attend(force_plain=plain, **kw) == UNSUPPORTED
