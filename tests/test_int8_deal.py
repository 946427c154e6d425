"""How the 8-bit product deals its work, restated on the CPU: every tile once, every stage of K once, every
column of a shared tile by one warp pair of one CTA pair of the cluster."""

import random

import pytest


def place(m_tiles, n_tiles, tile, group=8):
    per = group * n_tiles
    g, inside = divmod(tile, per)
    width = min(group, m_tiles - g * group)
    return g * group + inside % width, inside // width


@pytest.mark.parametrize("m_tiles,n_tiles", [(1, 1), (1, 40), (8, 3), (9, 3), (16, 1), (112, 32), (501, 2), (7, 7)])
def test_every_tile_has_its_place(m_tiles, n_tiles):
    got = sorted(place(m_tiles, n_tiles, t) for t in range(m_tiles * n_tiles))
    assert got == [(a, b) for a in range(m_tiles) for b in range(n_tiles)]


def test_pairs_take_every_tile_in_turn():
    for units in (1, 3, 74):
        for tiles in (1, 2, 73, 74, 75, 1000):
            taken = sorted(t for u in range(units) for t in range(u, tiles, units))
            assert taken == list(range(tiles))


@pytest.mark.parametrize("split", [1, 2, 3, 4])
def test_the_pairs_of_a_cluster_share_k(split):
    rng = random.Random(split)
    for nk in [2 * split, 2 * split + 1, 31, 32, 112, 1024] + [rng.randrange(2 * split, 2000) for _ in range(50)]:
        cuts = [(nk * p // split, nk * (p + 1) // split) for p in range(split)]
        assert cuts[0][0] == 0 and cuts[-1][1] == nk
        assert all(a < b for a, b in cuts) and all(x[1] == y[0] for x, y in zip(cuts, cuts[1:]))


@pytest.mark.parametrize("split", [2, 3, 4])
@pytest.mark.parametrize("tile_n", range(32, 257, 32))
def test_every_column_of_a_shared_tile_is_added_up_once(split, tile_n):
    cols = []
    for p in range(split):
        for half in range(2):
            for c in range(8 * (2 * p + half), tile_n, 16 * split):
                cols += range(c, c + 8)
    assert sorted(cols) == list(range(tile_n))


@pytest.mark.parametrize("tile_n", range(32, 257, 32))
def test_stages_and_sums_fit_in_shared_memory(tile_n):
    budget, sub = 227 * 1024 - 1024 - 512, 2 if tile_n <= 128 else 1
    block = 128 * 128 + tile_n * 64
    stages = min(12, budget // (sub * block))
    assert stages >= 3 and block % 1024 == 0  # (a tile of the 128-byte swizzle starts on 1024)
    assert 128 * tile_n * 4 <= stages * sub * block
    assert 8 * (2 * 12 + 2 + 2 + 1) + 4 <= 512  # barriers and the tensor memory's address
