"""How the 8-bit product deals its tiles to pairs of CTAs, restated on the CPU: every stage of every tile is
done once, no two parts of cut tiles share a place, and every pair that shares a tile finds the others."""

import random

import pytest

from opac1ty_b200 import _lib

COUNT_BYTES = 16384


def clocks(n):
    return max(2 * n, 256 + n)


def plan(rows, m, k, sms):
    pairs = min(max(sms // 2, 1), 256)
    tile_n = min(range(256, 31, -32), key=lambda n: -(-rows // n) * clocks(n))
    sub = 2 if tile_n <= 64 else 1
    nk = -(-k // (128 * sub))
    m_tiles, n_tiles = -(-m // 256), -(-rows // tile_n)
    tiles = m_tiles * n_tiles
    full = tiles // pairs * pairs
    rest = tiles - full
    stages, least, sharers = rest * nk, 0, rest
    for s in range(rest, min(pairs, stages) + 1) if rest else ():
        share = -(-s // rest) + (1 if s % rest else 0)
        t = -(-stages // s) * clocks(tile_n) * sub + (2000 + share * tile_n * 13 if s > rest else 0)
        if not least or t < least:
            least, sharers = t, s
    if not full:
        pairs = sharers
    size = COUNT_BYTES + (sharers * 4 * 128 * tile_n * 4 if sharers > rest else 0)
    return dict(tile_n=tile_n, m_tiles=m_tiles, n_tiles=n_tiles, nk=nk, full=full, rest=rest, sharers=sharers, pairs=pairs, bytes=size)


def items(d, p):
    for t in range(p, d["full"], d["pairs"]):
        yield t, 0, d["nk"]
    if p < d["sharers"]:
        every = d["rest"] * d["nk"]
        u, u1 = every * p // d["sharers"], every * (p + 1) // d["sharers"]
        while u < u1:
            j = u // d["nk"]
            k0 = u - j * d["nk"]
            k1 = min(d["nk"], k0 + u1 - u)
            yield d["full"] + j, k0, k1
            u += k1 - k0


def place(d, tile, group=8):
    per = group * d["n_tiles"]
    g, inside = divmod(tile, per)
    width = min(group, d["m_tiles"] - g * group)
    return g * group + inside % width, inside // width


def slot(d, tile, p):
    begin = d["rest"] * d["nk"] * p // d["sharers"]
    return 2 * p + (begin // d["nk"] != tile - d["full"])


def check(rows, m, k, sms):
    d = plan(rows, m, k, sms)
    assert d["tile_n"] % 32 == 0 and d["rest"] <= 255 and d["rest"] * 16 * 4 <= COUNT_BYTES
    assert d["rest"] == 0 or d["rest"] <= d["sharers"] <= d["pairs"]
    assert sorted(place(d, t) for t in range(d["full"] + d["rest"])) == \
        [(a, b) for a in range(d["m_tiles"]) for b in range(d["n_tiles"])]
    done, who = {}, {}
    for p in range(d["pairs"]):
        for tile, k0, k1 in items(d, p):
            assert 0 <= k0 < k1 <= d["nk"]
            done.setdefault(tile, []).append((k0, k1))
            if k0 > 0 or k1 < d["nk"]:
                who.setdefault(tile, []).append(p)
    assert len(done) == d["full"] + d["rest"]
    for parts in done.values():
        parts.sort()
        assert parts[0][0] == 0 and parts[-1][1] == d["nk"]
        assert all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
    taken = set()
    for tile, ps in who.items():
        every = d["rest"] * d["nk"]
        a = (tile - d["full"]) * d["nk"]
        first, last = (((u + 1) * d["sharers"] - 1) // every for u in (a, a + d["nk"] - 1))
        assert ps == list(range(first, last + 1)) and len(ps) > 1
        for p in ps:
            s = slot(d, tile, p)
            assert s not in taken and s < 2 * d["sharers"]
            taken.add(s)
    if who:
        assert d["bytes"] >= COUNT_BYTES + (max(taken) + 1) * 2 * 128 * d["tile_n"] * 4
    return d


@pytest.mark.parametrize("rows,m,k", [(9, 1, 1), (9, 256, 128), (24, 4096, 14336), (512, 6144, 4096), (333, 1011, 1000),
                                      (8191, 28672, 4096), (17, 128256, 4096), (300, 28672, 4096), (4097, 4096, 131071)])
def test_layers(rows, m, k):
    check(rows, m, k, 148)


def test_random_products():
    rng = random.Random(1)
    for _ in range(400):
        rows = max(9, int(2 ** rng.uniform(3, 12)))
        check(rows, int(2 ** rng.uniform(0, 14)), int(2 ** rng.uniform(0, 17)) or 1, rng.choice([148, 148, 148, 2, 3, 132, 17]))


def test_the_workspace_of_the_library_is_the_plans():
    """(Without a device the library knows no number of SMs and gives 0.)"""
    for rows, m, k in ((1, 4096, 4096), (24, 4096, 14336), (512, 6144, 4096)):
        size = _lib.load().opc_i8_gemm_workspace_bytes(rows, m, k, 0)
        if size:
            assert size == (COUNT_BYTES if rows <= 8 else plan(rows, m, k, 148)["bytes"])
