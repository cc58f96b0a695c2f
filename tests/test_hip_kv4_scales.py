"""Attention over a 4-bit cache whose value scales differ widely: a block's outputs are as exact as its own
scales allow, whatever the scales of other blocks, positions and rows are."""
import numpy as np
import pytest

import kv4
from test_hip_kv4 import Attention

pytestmark = pytest.mark.gpu

# ln(2) / 8 in 32 bits, whose product with log2(e) in 32 bits is 1 / 8.
SCALE = float(np.float32(np.log(2) / 8))


def bounded(q, k, v, v_scales, scale):
    """One row's heads in 64 bits and how far the kernel's may be off, for queries that fp16 holds exactly,
    key scales that are powers of two and SCALE: the products' sums of a block are then exact, and a score is off
    by the roundings of its blocks' sums (up to 8), of SCALE and of the exponent's argument: within 2^-21 of
    the largest. A score off by e makes a probability off by e, in the numerator and in the sum. The
    exponential and the two fp16 terms of each product cost 2^-20, the 32-bit sums a rounding per step of 32
    positions and of the waves' and parts' joins (a quarter of the tiles at most falls to one wave, 64 for
    the rest). Below fp16's normal range a term is rounded to a multiple of 2^-24 instead. A tile whose
    scales are below 2 holds its products as multiples of 2^-11 of the largest weight: 8 2^-34 a position, the
    code counting 8 at most. Any other tile holds a block's products with their largest at 2^14 or more: 2^-39 of it."""
    n, n_kv, dim = k.shape
    qq = q.astype(np.float64).reshape(n_kv, -1, dim)
    s = qq @ k.transpose(1, 2, 0) * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    vt = v.transpose(1, 0, 2)
    e = np.abs(s).max(-1, keepdims=True) * 2.0 ** -21
    largest = np.stack([(p * np.abs(v_scales[:, :, b].astype(np.float64)).T[:, None]).max(-1) for b in range(dim // 32)], -1)
    floor = n * 8 * (2.0 ** -34 + np.repeat(largest, 32, -1) * 2.0 ** -39)
    bound = (p @ np.abs(vt)) * (2 * e + 2.0 ** -20 + (n / 128 + 64) * 2.0 ** -24) + floor
    return (p @ vt).reshape(-1, dim), bound.reshape(-1, dim)


def check(a, out=None, rows=None):
    out = a.run() if out is None else out
    for r in range(a.rows) if rows is None else rows:
        n = a.vis[r]
        (kc, kd), (vc, vd) = a.caches[a.of[r]]
        want, bound = bounded(a.q[r], kv4.dequantize(kc[:n], kd[:n]), kv4.dequantize(vc[:n], vd[:n]), vd[:n], a.scale)
        off = np.abs(out[r] - want)
        assert np.all(off <= bound), f"row {r} of {n} positions: {np.max(off / bound):.2f} of its bound"


def exact_queries(a, rng):
    a.q[:] = rng.choice([-1.0, -0.5, 0.5, 1.0], a.q.shape)
    for (k, kd), _ in a.caches:
        kd[:] = rng.choice([-0.25, 0.25], kd.shape)


def peak(a, cache, at, nats):
    """Two positions' scores some nats above the others' mean (every head's: they share one query), the second's a
    little lower, so that its weight is no number of few bits."""
    a.q[:] = a.q[0, 0]
    (k, kd), _ = a.caches[cache]
    kd[at] = kd[at + 21] = 0.5
    steps = int(np.clip(round(nats / (0.5 * a.scale * np.abs(a.q[0, 0]).sum())), -6, 6))
    k[at] = k[at + 21] = np.where(a.q[0, 0] > 0, 8 + steps, 8 - steps)
    k[at + 21, :, :3] -= np.where(a.q[0, 0, :3] > 0, 1, -1).astype(np.int8).view(np.uint8)


SHAPES = [(8, 2, 64), (8, 1, 128), (9, 3, 96), (4, 2, 256), (17, 1, 64), (6, 2, 192)]


@pytest.mark.parametrize("n_head,n_kv,dim", SHAPES)
@pytest.mark.parametrize("large", [2.0, 300.0, 60000.0])
@pytest.mark.parametrize("where", ["every", "first", "last", "some"])
def test_small_scales_beside_a_large_one(n_head, n_kv, dim, large, where):
    """Two positions have most of the weight and 4000 others share the rest; block 0 has a large scale at
    every position, the first, the last or some, the others' are near 0.01. Rows of their own (split over
    workgroups, and not) and a chunk, of which only the last row sees the last position."""
    def change(a, rng):
        exact_queries(a, rng)
        for i, (_, (v, vd)) in enumerate(a.caches):
            vd[:, :, 1:] = (rng.uniform(0.01, 0.02, vd[:, :, 1:].shape)).astype(np.float16)
            vd[:, :, 0] = (rng.uniform(0.01, 0.02, vd[:, :, 0].shape)).astype(np.float16)
            at = {"every": slice(None), "first": 0, "last": -1, "some": slice(7, None, 190)}[where]
            vd[at, :, 0] = np.float16(large)
            peak(a, i, len(vd) // 3, 10)
    check(Attention([4001], n_head, n_kv, dim, seed=dim, scale=SCALE, change=change))
    check(Attention([500, 70], n_head, n_kv, dim, seed=dim, scale=SCALE, change=change))
    check(Attention([], n_head, n_kv, dim, chunk=(3, 3000), seed=dim, scale=SCALE, change=change))
    check(Attention([], n_head, n_kv, dim, chunk=(40, 500), seed=dim, scale=SCALE, change=change))


@pytest.mark.parametrize("large", [2.0, 60000.0])
def test_large_scales_beside_small_ones_in_a_block(large):
    """Blocks whose large scales belong to positions of little weight, or of nearly all."""
    for nats in (-10, 10):
        def change(a, rng):
            exact_queries(a, rng)
            for i, (_, (v, vd)) in enumerate(a.caches):
                vd[:] = (rng.uniform(0.01, 0.02, vd.shape)).astype(np.float16)
                vd[len(vd) // 2] = np.float16(large)
                peak(a, i, len(vd) // 2, nats)
        check(Attention([3000], 8, 2, 64, seed=3, scale=SCALE, change=change))
        check(Attention([], 8, 2, 64, chunk=(20, 2000), seed=4, scale=SCALE, change=change))


def test_earlier_rows_do_not_feel_a_later_rows_scale():
    """A chunk's rows that do not see the position whose scale is large, against the cache without it."""
    def change(a, rng):
        exact_queries(a, rng)
        for i, (_, (v, vd)) in enumerate(a.caches):
            vd[:] = (rng.uniform(0.01, 0.02, vd.shape)).astype(np.float16)
            peak(a, i, 100, 10)
    plain = Attention([], 8, 2, 64, chunk=(16, 600), seed=5, scale=SCALE, change=change)

    def larger(a, rng):
        change(a, rng)
        a.caches[0][1][1][-1] = np.float16(60000)
    mixed = Attention([], 8, 2, 64, chunk=(16, 600), seed=5, scale=SCALE, change=larger)
    out = mixed.run()
    check(mixed, out)
    check(plain, out, rows=range(15))
