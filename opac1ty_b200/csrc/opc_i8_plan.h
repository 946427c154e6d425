// opc_i8_plan.h -- how the 8-bit product on the tensor cores (opc_i8_gemm.cuh) deals its work: the width of its
// tiles, the pairs of CTAs that share one, each pair's tiles and stages.  Plain C++ besides, so that a test can
// compile it for the host.
#pragma once

#include <algorithm>
#include <cstdint>

#ifdef __CUDACC__
#define OPC_I8_HD __host__ __device__
#else
#define OPC_I8_HD
#endif

namespace opc {

constexpr int kI8Block = 128;                 // values of K per stage (one 128-byte swizzled row)
constexpr int kI8ABytes = 128 * kI8Block;     // a CTA's channels of a stage
constexpr int kI8Group = 8;                   // channel tiles taken together
constexpr int kI8MaxStages = 12;
constexpr int kI8SmemBudget = 227 * 1024 - 1024 - 512;  // less alignment slack and barriers

// A stage holds `sub` blocks of 128 values of K: the channels' block, then half of the tokens'.
OPC_I8_HD constexpr int i8_block_bytes(int n) { return kI8ABytes + n * (kI8Block / 2); }
OPC_I8_HD constexpr int i8_stages(int n, int sub) {
  return kI8SmemBudget / (sub * i8_block_bytes(n)) > kI8MaxStages ? kI8MaxStages : kI8SmemBudget / (sub * i8_block_bytes(n));
}

// How the tiles are dealt to the pairs of CTAs.
struct I8Deal {
  int32_t tile_n;              // tokens of a tile
  int32_t m_tiles, n_tiles;    // tiles of 256 channels, of tile_n tokens
  int32_t sub;                 // blocks of 128 values of K in a stage
  int32_t nk;                  // stages of a tile
  int32_t split;               // 1: a pair does whole tiles in turn; 2 .. 4: so many pairs (a cluster) do one
};

// First stage of the `part`-th of the pairs that share a tile (part = split: the end).
OPC_I8_HD inline int32_t i8_cut(const I8Deal& d, int32_t part) { return d.nk * part / d.split; }

// Channel and token tile of a tile: groups of kI8Group channel tiles, channels first.
OPC_I8_HD inline void i8_place(const I8Deal& d, int32_t tile, int32_t* mi, int32_t* ni) {
  const int32_t per = kI8Group * d.n_tiles, g = tile / per, in = tile - g * per;
  const int32_t left = d.m_tiles - g * kI8Group, width = left < kI8Group ? left : kI8Group;
  *mi = g * kI8Group + in % width;
  *ni = in / width;
}

struct I8Plan {
  I8Deal deal;
  int ctas;  // 0: too many tiles
};

// clusters[s]: how many clusters of s pairs run at once.  The choice is by a model of the time in clocks,
// fitted to 5 widths and 3 splits of 14 products (in the comments: what was measured, at 1.9 GHz).
inline I8Plan i8_plan(int32_t rows, int32_t M, int32_t K, const int (&clusters)[5]) {
  I8Plan p = {};
  const int64_t m_tiles = (static_cast<int64_t>(M) + 255) / 256;
  int64_t best = 0;
  for (int n = 256; n >= 32; n -= 32) {
    // Narrow tiles: two blocks a stage, since the barriers of a stage outlast its small MMAs (96 tokens,
    // 14336 -> 4096: 25.1 -> 21.5 us; 512 tokens, 4096 -> 6144 with tiles of 128: 18.5 -> 17.3; four blocks,
    // or two in wide tiles, no better).
    const int sub = n <= 128 ? 2 : 1;
    const int nk = (K + kI8Block * sub - 1) / (kI8Block * sub);
    const int64_t n_tiles = (static_cast<int64_t>(rows) + n - 1) / n, tiles = m_tiles * n_tiles;
    if (tiles > INT32_MAX / 2) continue;
    for (int split = 1; split <= 4; ++split) {
      if (split > 1 && (tiles > clusters[split] || nk < 2 * split)) continue;
      const int64_t rounds = (tiles + clusters[1] - 1) / clusters[1];
      const int64_t busy = 2 * split * std::min<int64_t>(tiles, clusters[1]);  // CTAs
      // One block: its MMAs at 2 clocks a token, its loads at 75 bytes a clock into an SM (57 when every SM
      // loads), the weights' part of them at 3580 a clock from memory.
      const int64_t rate = 75 - 18 * busy / (2 * clusters[1]);
      const int64_t block = std::max<int64_t>(std::max<int64_t>(2 * n + 12, (16384 + 64 * n) / rate),
                                              16384 * busy / (3580 * std::min<int64_t>(n_tiles, 8)));
      // Then the results of a tile, and for a split tile the exchange of sums (1.2 us for 32 tokens, 2.4 for 256).
      const int64_t t = rounds * ((nk + split - 1) / split) * sub * block + 19 * n / split + (split > 1 ? 2200 + 10 * n : 0);
      if (!best || t < best) {
        best = t;
        p.deal = {n, static_cast<int32_t>(m_tiles), static_cast<int32_t>(n_tiles), sub, nk, split};
        p.ctas = static_cast<int>(2 * split * (split > 1 ? tiles : std::min<int64_t>(tiles, clusters[1])));
      }
    }
  }
  return p;
}

}  // namespace opc
