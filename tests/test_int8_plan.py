"""How the 8-bit product deals its work, by the library's own code (compiled for the host)."""

import random

import pytest

from int8_plan import CLUSTERS, SHAPES, lib, place, plan


def sizes():
    rng = random.Random(3)
    yield from [(9, 1, 1), (17, 64, 131071), (24, 4096, 14336), (512, 6144, 4096), (8191, 28672, 4096), (2**31 - 4096, 1, 64)]
    for _ in range(400):
        yield tuple(int(2 ** rng.uniform(a, b)) for a, b in ((4, 14), (0, 17), (0, 16.9)))


@pytest.mark.parametrize("clusters", CLUSTERS + [(1, 0, 0, 0), (148, 74, 49, 37), (10, 5, 0, 0)])
def test_plans_hold_what_the_kernel_takes(clusters):
    for rows, m, k in sizes():
        p = plan(rows, m, k, clusters)
        n, split, tiles = p["tile_n"], p["split"], p["m_tiles"] * p["n_tiles"]
        assert n in range(32, 257, 32) and p["sub"] == (2 if n <= 128 else 1) and 1 <= split <= 4
        assert (p["m_tiles"] - 1) * 256 < m <= p["m_tiles"] * 256 and (p["n_tiles"] - 1) * n < rows <= p["n_tiles"] * n
        assert (p["nk"] - 1) * 128 * p["sub"] < k <= p["nk"] * 128 * p["sub"]
        # one tile for each cluster of pairs, all at once, with two stages or more a pair; or the pairs in turn
        assert p["ctas"] == 2 * split * (tiles if split > 1 else min(tiles, clusters[0]))
        assert split == 1 or (tiles <= clusters[split - 1] and p["nk"] >= 2 * split)


def test_too_many_tiles_have_no_plan():
    assert plan(2**31 - 4096, 2**31 - 4096, 64, CLUSTERS[0])["ctas"] == 0


@pytest.mark.parametrize("m_tiles,n_tiles", [(1, 1), (1, 40), (8, 3), (9, 3), (16, 1), (112, 32), (501, 2), (7, 7)])
def test_every_tile_has_its_place(m_tiles, n_tiles):
    got = sorted(place(m_tiles, n_tiles, t) for t in range(m_tiles * n_tiles))
    assert got == [(a, b) for a in range(m_tiles) for b in range(n_tiles)]


@pytest.mark.parametrize("split", [1, 2, 3, 4])
def test_pairs_share_k(split):
    rng = random.Random(split)
    for nk in [2 * split, 2 * split + 1, 31, 32, 112, 1024] + [rng.randrange(2 * split, 2000) for _ in range(50)]:
        cuts = [lib().cut(nk, split, p) for p in range(split + 1)]
        assert cuts[0] == 0 and cuts[-1] == nk and all(a < b for a, b in zip(cuts, cuts[1:]))


@pytest.mark.parametrize("n", range(32, 257, 32))
def test_stages_and_sums_fit_in_shared_memory(n):
    sub = 2 if n <= 128 else 1
    stages, block = lib().stages(n, sub), lib().block_bytes(n)
    assert 3 <= stages <= 12 and block % 1024 == 0  # (a tile of the 128-byte swizzle starts on 1024)
    assert 1024 + stages * sub * block + 512 <= 227 * 1024
    assert 128 * n * 4 <= stages * sub * block  # a shared tile's sums take the stages' place
    assert 8 * (2 * 12 + 2 + 2 + 1) + 4 <= 512  # barriers and the tensor memory's address


def test_the_shapes_that_run_on_a_gpu_are_dealt_as_they_say():
    for (n, split, rounds), (rows, m, k) in SHAPES.items():
        for c in CLUSTERS:
            p = plan(rows, m, k, c)
            assert (p["tile_n"], p["split"]) == (n, split)
        assert min(3, -(-p["m_tiles"] * p["n_tiles"] // 74)) == rounds if split == 1 else rounds == 1
    assert {(n, s) for n, s, _ in SHAPES} >= {(n, s) for n in range(32, 257, 32) for s in (1, 2, 4)} | {(n, 3) for n in range(32, 161, 32)}
    assert {(n, 3) for n in range(32, 257, 32)} <= {(n, r) for n, s, r in SHAPES if s == 1}
