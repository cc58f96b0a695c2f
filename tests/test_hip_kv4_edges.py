"""Attention over a 4-bit cache at the ends of what its arguments allow: scores far above the exponent's usual
range, blocks that are not numbers far below the maximum, offsets of a chunk's rows, sizes of a launch."""
import ctypes as C

import numpy as np
import pytest

import axon_hip as H
import kv4
from test_hip_kv4 import Attention, addr, put

gpu = pytest.mark.gpu

# Heads and rows that take each kernel: single rows (whole and split), single rows of large groups or heads, chunks.
FORMS = [dict(lengths=[300], n_head=8, n_kv=2, dim=64), dict(lengths=[3000], n_head=8, n_kv=1, dim=128),
         dict(lengths=[2500, 40], n_head=17, n_kv=1, dim=64), dict(lengths=[300, 9], n_head=4, n_kv=2, dim=256),
         dict(lengths=[33], n_head=8, n_kv=2, dim=64, chunk=(30, 270)), dict(lengths=[], n_head=8, n_kv=2, dim=64, chunk=(4, 3000)),
         dict(lengths=[], n_head=256, n_kv=64, dim=32, chunk=(130, 0)), dict(lengths=[], n_head=8, n_kv=2, dim=192, chunk=(30, 70))]


# ---------------------------------------------------------------------------------------------
# Scores whose size leaves 32 bits no fraction

@gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("power", [20, 24, 25, 26, 27, 28, 30, 33, 60, 100])
@pytest.mark.parametrize("sign", [1, -1])
def test_equal_scores_of_any_size(form, power, sign):
    """Every position has the same key, so every weight is the same, and 32 bits give every position the same
    score, however large: the mean of the values, to the rounding of a sum of that many products (2^-20
    of the products' magnitudes and the joins' share besides)."""
    def change(a, rng):
        a.q[:] = np.float32(2.0 ** power) * rng.choice([1, 1.25, 1.5], a.q.shape) * sign
        for (k, kd), _ in a.caches:
            k[:] = 13
            kd[:] = np.float16(1)
    a = Attention(**form, seed=power, change=change)
    out = a.run()
    for r in range(a.rows):
        n = a.vis[r]
        v = kv4.dequantize(*a.caches[a.of[r]][1])[:n]
        group = a.n_head // a.n_kv
        want = np.repeat(v.mean(0), group, 0)
        bound = np.repeat(np.abs(v).mean(0), group, 0) * (2.0 ** -20 + (n / 32 + 64) * 2.0 ** -24) + n * 8 * 2.0 ** -34
        assert np.all(np.abs(out[r] - want) <= bound), (r, n)


@gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("power", [10, 20, 25, 26, 27, 28, 30, 33, 60, 100])
def test_the_largest_score_of_any_size(form, power):
    """One position's score is twice the largest of the others, and then some hundred above: its values alone
    are the output. It is neither first nor last, so that some waves begin with others."""
    def change(a, rng):
        a.q[:] = np.float32(2.0 ** power) * rng.choice([1, 1.25, 1.5], a.q.shape)
        for (k, kd), _ in a.caches:
            kd[:] = np.float16(1)
            k[:] = rng.integers(8, 11, (len(k), a.n_kv, 1))
            k[len(k) // 3] = 15
    a = Attention(**form, seed=power, change=change)
    out = a.run()
    for r in range(a.rows):
        n, seq = a.vis[r], a.of[r]
        at = len(a.caches[seq][0][0]) // 3
        if at >= n:
            continue
        want = np.repeat(kv4.dequantize(*a.caches[seq][1])[at], a.n_head // a.n_kv, 0)
        assert np.all(np.abs(out[r] - want) <= np.abs(want) * 2.0 ** -20), (r, n)


# ---------------------------------------------------------------------------------------------
# Blocks held as NaN, far below the maximum

@gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("which", ["key", "value"])
def test_a_block_that_is_not_a_number_is_felt_at_any_weight(form, which):
    """One position outweighs the rest by more than 32 bits can say, and a block of another, in a tile far from
    it, is held as NaN: the rows that see it give NaN (a key's in its head's outputs, a value's in its
    block's), whether the positions are split over workgroups or not, and everything else is a number."""
    def change(a, rng):
        a.q[:] = 4
        for i, ((k, kd), (v, vd)) in enumerate(a.caches):
            kd[:] = np.float16(1)
            k[:] = rng.integers(6, 9, k.shape)
            k[0] = 15
            bad = kd if which == "key" else vd
            bad[2 * len(bad) // 3, -1, 0] = np.nan
    a = Attention(**form, seed=1, change=change)
    out = a.run()
    group, felt = a.n_head // a.n_kv, 0
    for r in range(a.rows):
        sees = a.vis[r] > 2 * len(a.caches[a.of[r]][0][0]) // 3
        felt += sees
        want = np.zeros(out[r].shape, bool)
        want[-group:, :a.dim if which == "key" else 32] = sees
        assert np.array_equal(np.isnan(out[r]), want), (r, a.vis[r])
    assert felt != 0


# ---------------------------------------------------------------------------------------------
# A chunk's sequence

@gpu
@pytest.mark.parametrize("form", [dict(n_head=8, n_kv=2, dim=64, chunk=(300, 20)), dict(n_head=8, n_kv=2, dim=64, chunk=(6, 3000)),
                                  dict(n_head=40, n_kv=1, dim=32, chunk=(20, 5)), dict(n_head=256, n_kv=64, dim=32, chunk=(130, 0))])
def test_a_chunk_goes_by_the_first_rows_offset(form):
    """Entries 1 to chunk_rows - 1 of cache_off are not read: they name another sequence here. The rows behind
    the chunk go by their own."""
    a = Attention([50, 7], seed=12, **form)
    args = a.args()
    off = np.array([i * a.slot for i in a.of], np.int64)
    off[1:a.chunk_rows] = a.slot
    entries = put(off)
    args.cache_off = entries.ptr
    H.call("attention_kv4", addr(args), a.rows)
    a.check(a.got())


# ---------------------------------------------------------------------------------------------
# Sizes that no launch can take are refused as arguments, before any device is asked for

def test_sizes_past_a_launch_are_refused():
    def refuse(name, a, *rest):
        with pytest.raises(H.HipError, match="workgroups"):
            H.call(name, addr(a), *rest)

    for n_kv, n_head, dim, rows in ((65536, 0, 256, 2), (32768, 0, 256, 1), (2, 65536, 256, 1 << 24), (32767, 512, 256, 3), (2, 4, 64, 1 << 24)):
        a = H.RopeRowsArgs()
        a.k = a.v = a.cache = a.table = a.pos = 4096
        a.q = 4096 if n_head else None
        a.n_head, a.n_kv, a.head_dim, a.rotary_dim = n_head, n_kv, dim, 32
        a.q_stride, a.k_stride = n_head * dim, n_kv * dim
        refuse("rope_rows_kv4", a, 64, rows)
    for n_kv, dim, rows in ((65536, 256, 2), (32768, 256, 1), (2, 64, 1 << 24), (1, 32, (1 << 31) - 1)):
        b = H.Kv4ReadArgs()
        b.cache = b.k = b.v = b.pos = 4096
        b.n_kv, b.head_dim, b.max_ctx, b.stride = n_kv, dim, 64, n_kv * dim
        refuse("kv4_read_rows", b, rows)
    for n_head, n_kv, rows, chunk in ((8, 8, 1 << 20, 0), (64, 1, 1 << 21, 0), (65536, 65536, 200, 0), (1, 1, 1 << 23, 0), (64, 64, 1 << 30, 1 << 30),
                                      (8, 8, (1 << 20) + 16, 16), (8, 8, (1 << 27) + 1, 1 << 27)):
        c = H.AttentionKv4Args()
        c.q = c.out = c.cache = c.n_vis = c.scratch = 4096
        c.n_head, c.n_kv, c.head_dim, c.max_ctx, c.max_vis, c.scale, c.chunk_rows = n_head, n_kv, 32, 64, 64, 0.125, chunk
        c.q_stride = c.out_stride = n_head * 32
        refuse("attention_kv4", c, rows)


# ---------------------------------------------------------------------------------------------
# Nothing to see, and factors at their ends

@gpu
@pytest.mark.parametrize("form", FORMS)
def test_no_row_sees_anything(form):
    """max_vis 0 and every n_vis 0: zeros, and the cache is not read (its address is that of a buffer of one tile)."""
    a = Attention(**form, seed=2)
    args = a.args()
    none, small = put(np.zeros(a.rows), np.int32), put(np.full(kv4.tile_bytes(a.dim), 255, np.uint8))
    args.n_vis, args.max_vis, args.cache, args.cache_off = none.ptr, 0, small.ptr, None
    H.call("attention_kv4", addr(args), a.rows)
    assert np.all(a.got() == 0)


@gpu
@pytest.mark.parametrize("form", FORMS[:5])
@pytest.mark.parametrize("scale,queries", [(0.0, 1.0), (-0.0, 1.0), (1e30, 1e-31), (-1e-30, 1e30), (1e-38, 1e37)])
def test_scales_at_their_ends(form, scale, queries):
    """A scale of zero weighs every position alike; one that only a query at the other end makes ordinary."""
    def change(a, rng):
        a.q *= np.float32(queries)
    Attention(**form, seed=3, change=change, scale=float(np.float32(scale))).check()
