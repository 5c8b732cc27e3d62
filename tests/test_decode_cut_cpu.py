"""The cut of a decode attention call's work list, as the kernels have it
(velo-core_b200/csrc/kernels/decode_cut.cuh compiled for the host): every step of
every item in exactly one block, and for each cut item the states its join reads."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import velo_cuda

CSRC = os.path.join(os.path.dirname(velo_cuda.__file__), "csrc")
TOKENS = {velo_cuda.KV_F16: 16, velo_cuda.KV_INT8: 32, velo_cuda.KV_F32: 8}

HARNESS = """
#include <vector>
#include "kernels/decode_cut.cuh"
using namespace velo;
template <int kTok>
static void ranges(const Cut& k, const int* pre, const int* lens, int B, int join, int* first, int* item) {
    for (int c = 0; c <= k.blocks(); ++c) first[c] = cut_at<kTok>(pre, lens, B, k, join, c);
    for (int c = 0; c < k.blocks(); ++c) {
        if (first[c] >= k.total()) continue;
        const Item x = item_of<kTok>(pre, lens, B, first[c]);
        item[4 * c] = x.b, item[4 * c + 1] = x.it, item[4 * c + 2] = x.start, item[4 * c + 3] = x.units;
    }
}
struct Call { int kv, D, group, n_kv, B, max_pages, sms; };
extern "C" {
// the plan: main, blocks, tiles, join units, most units
void plan(const Call* c, int* out) {
    const Plan p = make_plan(c->kv, c->group, c->n_kv, c->B, c->max_pages, c->sms);
    out[0] = p.main, out[1] = p.blocks, out[2] = p.tiles, out[3] = join_units(c->kv, c->D), out[4] = most_units(c->kv, c->max_pages);
}
// per block its first unit (and the list's end) and the item that lies there; the number of blocks
int cut(const Call* c, const int* lens, const int* pre, int items, int longest, int* first, int* item) {
    const Plan p = make_plan(c->kv, c->group, c->n_kv, c->B, c->max_pages, c->sms);
    const int join = join_units(c->kv, c->D);
    const Cut k = cut_list(p, pre[c->B], items, longest, join);
    if (c->kv == VELO_KV_F16) ranges<16>(k, pre, lens, c->B, join, first, item);
    else if (c->kv == VELO_KV_INT8) ranges<32>(k, pre, lens, c->B, join, first, item);
    else ranges<8>(k, pre, lens, c->B, join, first, item);
    return k.blocks();
}
int block_of(const Call* c, const int* pre, int items, int longest, int u) {
    const Plan p = make_plan(c->kv, c->group, c->n_kv, c->B, c->max_pages, c->sms);
    return cut_list(p, pre[c->B], items, longest, join_units(c->kv, c->D)).block_of(u);
}
}
"""


class Call(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("kv", "D", "group", "n_kv", "B", "max_pages", "sms")]


@pytest.fixture(scope="module")
def cut(tmp_path_factory):
    d = tmp_path_factory.mktemp("cut")
    src, lib = str(d / "cut.cpp"), str(d / "cut.so")
    with open(src, "w") as f:
        f.write(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-ftrapv", "-shared", "-fPIC", "-I" + CSRC,
                    "-I" + os.path.join(os.path.dirname(CSRC), "..", "include"), src, "-o", lib], check=True)
    return ctypes.CDLL(lib)


def _check(lib, kv, D, group, n_kv, lens, max_pages, sms=148):
    lens = np.asarray(lens, np.int32)
    B, tok = len(lens), TOKENS[kv]
    call = Call(kv, D, group, n_kv, B, max_pages, sms)
    p = (ctypes.c_int * 5)()
    lib.plan(ctypes.byref(call), p)
    main, grid, tiles, join, most = p
    per_seq = n_kv * tiles
    units = -(-lens.astype(np.int64) // tok)
    assert units.max(initial=0) <= most
    pre64 = np.concatenate(([0], np.cumsum(units * per_seq)))
    assert pre64[-1] <= 1 << 30
    pre = pre64.astype(np.int32)
    first, item = np.full(grid + 1, -1, np.int32), np.zeros((grid, 4), np.int32)
    ptr = lambda a: a.ctypes.data_as(ctypes.c_void_p)
    items, longest = int((lens > 0).sum()) * per_seq, int(units.max(initial=0))
    n = lib.cut(ctypes.byref(call), ptr(lens), ptr(pre), items, longest, ptr(first), ptr(item))
    assert n <= grid
    total = int(pre[-1])
    if total == 0:
        return n
    assert first[0] == 0 and first[n] == total and (np.diff(first[:n + 1]) >= 0).all()
    written, read, cut_items = {}, [], 0
    for c in range(n):
        seg, end = int(first[c]), int(first[c + 1])
        open_ = None
        while seg < end:  # as a block walks its range
            b = int(np.searchsorted(pre, seg, "right")) - 1
            it = (seg - int(pre[b])) // int(units[b])
            start = int(pre[b]) + it * int(units[b])
            if seg == first[c]:
                assert tuple(item[c]) == (b, it, start, units[b])
            stop = min(start + int(units[b]), end)
            whole = seg == start and stop == start + units[b]
            if not whole:
                assert units[b] > join  # short items are never cut, so tables of short rows need no join
                slot = 2 * c + (seg == start)
                assert slot not in written
                written[slot] = (b, it, seg)
                if seg == start:
                    assert open_ is None
                    open_ = (b, it, start, lib.block_of(ctypes.byref(call), ptr(pre), items, longest, start + int(units[b]) - 1))
            seg = stop
        if open_:
            b, it, start, last = open_
            states = [2 * c + 1] + [2 * i for i in range(c + 1, last + 1)]
            read.append((b, it, start, states))
    got = []
    for b, it, start, states in read:  # every state of the item, in order, and no other's
        cut_items += 1
        at = [written[s] for s in states]
        assert all(w[:2] == (b, it) for w in at)
        assert at[0][2] == start and [w[2] for w in at] == sorted(w[2] for w in at)
        got += states
    assert sorted(got) == sorted(written) and len(set(got)) == len(got)
    return cut_items


@pytest.mark.parametrize("seed", range(80))
def test_every_step_once_and_every_state_joined(cut, seed):
    rng = np.random.default_rng(seed)
    kv = int(rng.choice([velo_cuda.KV_F16, velo_cuda.KV_INT8, velo_cuda.KV_F32]))
    B = int(rng.choice([1, 2, 7, 30, 120, 500]))
    hi = int(rng.choice([20, 300, 3000, 40000]))
    lens = rng.integers(0, hi + 1, B) if seed % 3 else np.full(B, hi)
    if seed % 7 == 0:
        lens[rng.integers(0, B)] = 60 * hi
    if not lens.any():
        lens[0] = 1
    width = -(-int(lens.max()) // 16) + int(rng.choice([0, 0, 5, 8192]))
    _check(cut, kv, int(rng.choice([64, 128])), int(rng.choice([1, 4, 5, 8, 9, 24])), int(rng.choice([1, 2, 8, 32])), lens, width,
           int(rng.choice([148, 148, 3, 16])))


def test_some_lists_are_cut_with_a_tail(cut):
    """The property above is not empty: such calls have items joined over many blocks."""
    assert _check(cut, velo_cuda.KV_F16, 128, 8, 8, [100003], 6251) == 8
    assert _check(cut, velo_cuda.KV_F16, 128, 8, 8, 3900 + 61 * np.arange(64) % 390, 270) > 100
    assert _check(cut, velo_cuda.KV_INT8, 128, 4, 8, 512 + 777 * np.arange(128) % 7680, 512) > 100
    assert _check(cut, velo_cuda.KV_F16, 128, 4, 8, [32] * 256, 2) == 0


@pytest.mark.parametrize("kv,n_kv,lens,width", [
    (velo_cuda.KV_F16, 8, [(1 << 19)] * 4096, 1 << 15),     # 2^30 steps
    (velo_cuda.KV_F16, 1, [1 << 30], 1 << 26),              # one item of 2^26
    (velo_cuda.KV_F32, 8, [(1 << 18) - 5 * (i % 7) for i in range(4096)], 1 << 14),
    (velo_cuda.KV_INT8, 2, [1 << 30, 17, 0, 1 << 30], 1 << 26)])
def test_lists_of_the_largest_size(cut, kv, n_kv, lens, width):
    _check(cut, kv, 128, 8, n_kv, lens, width)


def test_empty_lists_have_no_blocks(cut):
    for B in (1, 5):
        assert _check(cut, velo_cuda.KV_F16, 128, 4, 2, [0] * B, 4) == 0
