"""The library's own rules for dealing the 8-bit product's work (csrc/opc_i8_plan.h), compiled for the host."""

import ctypes
import functools
import subprocess
import tempfile
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "opac1ty_b200" / "csrc"
SHIM = """
#include "opc_i8_plan.h"
extern "C" {
void plan(int rows, int M, int K, const int* clusters, int* out) {
  int c[5];
  for (int i = 0; i < 5; ++i) c[i] = clusters[i];
  const opc::I8Plan p = opc::i8_plan(rows, M, K, c);
  const int v[7] = {p.deal.tile_n, p.deal.m_tiles, p.deal.n_tiles, p.deal.sub, p.deal.nk, p.deal.split, p.ctas};
  for (int i = 0; i < 7; ++i) out[i] = v[i];
}
void place(int m_tiles, int n_tiles, int tile, int* out) {
  opc::I8Deal d = {};
  d.m_tiles = m_tiles;
  d.n_tiles = n_tiles;
  opc::i8_place(d, tile, out, out + 1);
}
int cut(int nk, int split, int part) {
  opc::I8Deal d = {};
  d.nk = nk;
  d.split = split;
  return opc::i8_cut(d, part);
}
int stages(int n, int sub) { return opc::i8_stages(n, sub); }
int block_bytes(int n) { return opc::i8_block_bytes(n); }
}
"""
FIELDS = ("tile_n", "m_tiles", "n_tiles", "sub", "nk", "split", "ctas")

# clusters of 1 to 4 pairs that run at once, on parts whose groups of processors are cut in different ways
CLUSTERS = [(74, 37, 24, 18), (74, 36, 22, 16), (74, 36, 24, 16), (74, 35, 20, 14), (74, 36, 21, 15), (72, 32, 16, 16), (66, 32, 20, 14)]


# Products (tokens, channels, width) whose tiles are dealt alike under each of these: by the tokens of a tile, the pairs that
# share one, and the rounds of tiles that 74 pairs take (3: at least).  Every pair of a width and a split that they can
# agree on.
SHAPES = {
    (32, 1, 1): (17, 64, 74), (32, 1, 2): (2244, 307, 76), (32, 1, 3): (2870, 277, 73),
    (32, 2, 1): (17, 3594, 2420), (32, 3, 1): (353, 65, 2069), (32, 4, 1): (17, 71, 1845),
    (64, 1, 1): (2635, 73, 67), (64, 1, 2): (3853, 291, 80), (64, 1, 3): (3529, 526, 79),
    (64, 2, 1): (41, 4987, 3962), (64, 3, 1): (454, 305, 2106), (64, 4, 1): (298, 321, 1845),
    (96, 1, 1): (2413, 302, 266), (96, 1, 2): (3855, 555, 257), (96, 1, 3): (644, 6696, 144),
    (96, 2, 1): (89, 4677, 3898), (96, 3, 1): (87, 3094, 3278), (96, 4, 1): (626, 275, 1842),
    (128, 1, 1): (3703, 264, 277), (128, 1, 2): (1757, 1801, 387), (128, 1, 3): (2319, 2374, 411),
    (128, 2, 1): (108, 5076, 3895), (128, 3, 1): (99, 3254, 4252), (128, 4, 1): (867, 306, 2386),
    (160, 1, 1): (3506, 518, 257), (160, 1, 2): (2026, 1558, 73), (160, 1, 3): (210, 19147, 64),
    (160, 2, 1): (306, 3787, 3317), (160, 3, 1): (137, 4031, 2582), (160, 4, 1): (302, 1697, 2476),
    (192, 1, 1): (2493, 1043, 554), (192, 1, 2): (1810, 3094, 259), (192, 1, 3): (2244, 3772, 262),
    (192, 2, 1): (1139, 1150, 4368), (192, 4, 1): (336, 1739, 2384), (224, 1, 1): (2408, 1384, 558),
    (224, 1, 2): (1282, 5605, 416), (224, 1, 3): (643, 15863, 311), (224, 2, 1): (1778, 795, 4111),
    (224, 4, 1): (399, 1606, 3486), (256, 1, 1): (706, 4846, 549), (256, 1, 2): (989, 8016, 599),
    (256, 1, 3): (1455, 8027, 546), (256, 2, 1): (951, 1937, 4453), (256, 4, 1): (484, 1644, 3567),
}


@functools.lru_cache(None)
def lib():
    with tempfile.TemporaryDirectory() as d:
        src, so = Path(d) / "plan.cpp", Path(d) / "plan.so"
        src.write_text(SHIM)
        subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(CSRC), "-o", str(so), str(src)], check=True)
        return ctypes.CDLL(str(so))


def plan(rows, m, k, clusters):
    out = (ctypes.c_int * 7)()
    lib().plan(rows, m, k, (ctypes.c_int * 5)(0, *clusters), out)
    return dict(zip(FIELDS, out))


def place(m_tiles, n_tiles, tile):
    out = (ctypes.c_int * 2)()
    lib().place(m_tiles, n_tiles, tile, out)
    return tuple(out)
