"""Attention over a 4-bit cache in every form that a launch can choose: head sizes by group sizes by how many rows,
positions and workgroups there are, each against its definition in 64 bits."""
import numpy as np
import pytest

import kv4
from test_hip_kv4 import DIMS, Attention

pytestmark = pytest.mark.gpu


def all_heads(q, k, v, scale):
    """kv4.attention and its bound, for all heads of a row at once (value scales below 2)."""
    n, n_kv, dim = k.shape
    qq, kt, vt = q.astype(np.float64).reshape(n_kv, -1, dim), k.transpose(1, 2, 0), v.transpose(1, 0, 2)
    s = qq @ kt * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    e = abs(scale) * (np.abs(k).sum(2).max(0)[:, None, None] * np.abs(qq).max(-1, keepdims=True) * 2.0 ** -21 +
                      (np.abs(qq) @ np.abs(kt)).max(-1, keepdims=True) * (dim + 8) * 2.0 ** -24)
    e += np.abs(s).max(-1, keepdims=True) * 2.0 ** -22 + np.abs(s - s.max(-1, keepdims=True)).max(-1, keepdims=True) * 2.0 ** -23
    bound = (p @ np.abs(vt)) * (2 * e + 2.0 ** -20 + (n / 32 + 64) * 2.0 ** -24) + n * 8 * 2.0 ** -34
    return (p @ vt).reshape(-1, dim), bound.reshape(-1, dim)


def check(a):
    out = a.run()
    held = [[kv4.dequantize(*x) for x in c] for c in a.caches]
    for r in range(a.rows):
        n, (k, v) = a.vis[r], held[a.of[r]]
        if n == 0:
            assert np.all(out[r] == 0)
            continue
        want, bound = all_heads(a.q[r], k[:n], v[:n], a.scale)
        off = np.abs(out[r] - want)
        assert np.all(off <= bound), f"row {r} of {n} positions: {np.max(off / bound):.2f} of its bound"


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("group", [1, 3, 4, 5, 8, 18])
@pytest.mark.parametrize("what", ["short", "long", "split"])
def test_rows(dim, group, what):
    """Rows of their own: one to four heads a group, five to eight and more; up to 512 positions (four waves),
    more of them in one workgroup, and split over several. A row that ends inside its first tile, one at a
    tile's border and an empty one are with them."""
    rng = np.random.default_rng(dim + group)
    if what == "short":
        a = Attention([512, 1, 77, 0, 256, 257], group * 2, 2, dim, seed=dim)
    elif what == "long":
        a = Attention([1000, 0, 5, 544, 513] + [int(x) for x in rng.integers(500, 1000, 15)], group * 8, 8, dim, seed=dim)
        a.args()
        assert a.scratch_floats == 0
    else:
        a = Attention([3001, 2100, 0, 33], group * 2, 2, dim, seed=dim)
        a.args()
        assert a.scratch_floats > 0
    check(a)


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("rows,past", [(130, 300), (112, 320), (70, 350), (130, 0), (33, 5)])
def test_chunks_of_many_heads(dim, rows, past):
    """64 KV heads of four: with 130 rows two tiles of columns a wave, two waves a set (heads up to 128), with 112
    two tiles and four waves, with 70 one tile and two waves, with 33 one and four. The chunk's end is not
    a whole workgroup's, nor a whole tile's."""
    check(Attention([40], 256, 64, dim, chunk=(rows, past), seed=rows + dim))


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("n_head,n_kv", [(350, 50), (96, 96), (160, 8)])
def test_chunks_of_odd_groups(dim, n_head, n_kv):
    """Groups of 7 (no whole number of rows a set of columns), 1 and 20 (more heads than a wave's columns)."""
    check(Attention([], n_head, n_kv, dim, chunk=(101, 60), seed=dim))


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("n_head,n_kv", [(8, 2), (7, 1), (20, 1)])
def test_chunks_split_over_positions(dim, n_head, n_kv):
    """Parts of 256 positions (20 heads over one: 640), with a border among the chunk's rows, the earlier of which see a
    part less; and a chunk behind nothing that is not split."""
    a = Attention([300, 0], n_head, n_kv, dim, chunk=(37, 1775), seed=dim)
    a.args()
    assert a.scratch_floats > 0
    check(a)
    b = Attention([], n_head, n_kv, dim, chunk=(600, 0), seed=dim)
    check(b)
