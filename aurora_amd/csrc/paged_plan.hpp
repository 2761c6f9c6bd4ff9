// How a call of the paged attention is cut into items, and which kernel takes them: host arithmetic alone,
// so that it can be looked at without a device.
#pragma once

#include <algorithm>
#include <cmath>

namespace aurpaged {

// What the host knows of a call.
struct Sizes {
  int b, n_tok, max_tok, max_own, prefix_len;  // of the batch (max_tok up to n_tok)
  int Hkv, G, dh;                              // K/V heads, query heads of each, columns
  bool f32;
  bool e4m3 = false;
};
// How it is cut; the scratch's size follows from it.  Tiles are an item's rows, splits the ranges of an
// axis, of so many keys each; p_ the prefix's items (pooled: 0 of them otherwise), o_ a sequence's own.
struct Plan {
  int pooled, p_tile, o_tile, p_tiles, p_splits, p_keys, o_tiles, o_splits, o_keys;
  int parts() const { return p_splits + o_splits; }
  // One launch serves both kinds of items, unless the prefix has the larger tiles.
  bool together() const { return p_tile <= 64; }
};

// Rows of an item: 16 keep their keys in registers, more lay them down in LDS.
inline int tile_of(long long rows, int dh) { return rows <= 16 ? 16 : rows <= 64 ? 64 : rows <= 128 || dh > 64 ? 128 : 256; }

// Items that a launch aims at, measured at 128 to 4096 of them: with 16-row own items 3 of a CU (64
// sequences on a prefix of 32768 in bf16: 86 µs, with 256 items 140, with 2048 97), with larger ones 4
// (tails of 66 to 122 on 2048: 113 µs, with 768 items 120), of 8 waves one (512 sequences on a prefix of 16384:
// 240 µs, with 1024 items 303).
// fp32 keys of more than 64 columns fill the registers, and keys without a prefix's items beside them the
// memory, with 2 a CU (64 sequences of 512 to 1024 keys, 8 heads of 128, 4 rows each: 77 µs, with 768 items
// 85; one sequence of 16757 keys, 16 heads of 64: 28, with 768 items 30).
constexpr int kItems16 = 768, kItemsWide = 512, kItems = 1024, kItems8 = 256;
// An axis up to so many keys is one range: a join costs 4 µs, 128 keys of a 16-row item (a round of its
// waves) 1.5 µs.  Longer ones are cut into ranges of 128 keys or more, 48 at most.  Larger items of so many
// axes that they fill the chip uncut are not cut up to twice that length (23 sequences of 72 rows on 506
// keys, 15 heads of 48, bf16: 31 µs, cut 40; uncut with fewer than 256 axes cost a batch's block its chain
// of tiles: 6 of 185 rows on 465, one head, 36 µs against 20).
constexpr int kWhole16 = 384, kWhole = 256, kWholeFull = 512, kFill = 256;
constexpr int kLeastKeys = 128, kMostRanges = 48;
// e4m3 keys: a CU holds two of their larger items, which take their keys faster (tails of 66 to 122 on 2048, 16
// heads of 64: 71 µs with 512 items, 78 with 1024), and ranges of 256 keys (48 sequences of 16 heads on 4 of
// 128, prefix 4999, own 500: 26.7 µs, with 192 keys 30.5, with 384 27.6; d_head 64 20.5, 22.6 and 21.1; 36 of them
// on 1500 17.4, 15.8 and 20.1).
constexpr int kItemsE4m3 = 512, kLeastKeysE4m3 = 256;
// With little work the time is a block's chain of tiles, not the products: smaller items then.  16 rows up
// to so many items of 16 rows by 128 keys (5 sequences of 74 rows on 434 keys, 3 heads of 48, bf16, 300 of
// them: 9.9 µs, in 128 rows 14, in 64 rows 11.7; at 1024 a batch took 15 instead of 11), 64 rows where items
// times ranges of 128 keys come to less than kSmall (10 sequences of 315 rows on 763, 2 heads of 64, 1440:
// 19 µs, in 256 rows 25; 30 of 85 rows on 721, 2160: 27 against 25; 6 of 355 rows on 392, 14 heads, 2688:
// 43 against 30).
constexpr int kSmall16 = 512, kSmall = 1536;
// Keys times heads that pooling saves, from where it pays its records and its join (8 sequences of 12 heads
// on a prefix of 1294, 108,000: 13 against 33 µs; 53 sequences of 5 heads on 139, 35,000: 22 against 10).
constexpr int kPoolFrom = 65536;
// Rows of all sequences up to which the prefix's items have 64, in the own ones' launch, instead of 256 (128
// from d_head 65 on) in one of their own.  d_head 128 on a prefix of 4999, 16 heads on 4, µs with 64 and 128
// rows: 144 rows of the batch fp32 43 and 53, 192 46 and 57, 256 56 and 63; bf16 32 and 43, 32 and 46, 40 and
// 50.  d_head 64, with 64 and 256: 144 rows 27 and 35, 192 31 and 41, 256 36 and 45; bf16 20 and 28, 20 and 31,
// 24 and 35: there too 64 rows are the faster up to 256, and its bound of 128 is short of that.
constexpr int kPool64 = 128, kPool64Wide = 256;
// For e4m3 keys, whose launches are shorter, 64 rows up to so many rows times prefix keys times K/V columns too: on 4
// heads of 64, µs with 64 and 256 rows: 192 rows on 4999 20 and 32, on 16384 34 and 39, on 30000 49 and 48, on 65536
// 85 and 74; 384 rows on 4999 30 and 36; 2 heads of 128, with 64 and 128: 512 rows on 6000 32 and 38, on 24000 70
// and 57; 1024 rows on 1500 24 and 35, on 6000 50 and 42.
constexpr double kPoolWorkE4m3 = 1.1e9;

inline Plan make_plan(const Sizes& b) {
  Plan p{};
  const int P = b.prefix_len, Hkv = b.Hkv, G = b.G, dh = b.dh;
  const long long o_rows = (long long)b.max_tok * G, p_rows = (long long)b.n_tok * G;
  p.o_tile = tile_of(o_rows, dh);
  p.o_tiles = (int)((o_rows + p.o_tile - 1) / p.o_tile);
  const bool light = b.e4m3 && (double)p_rows * P * Hkv * dh <= kPoolWorkE4m3;
  p.p_tile = p_rows <= 32 ? 16 : light || p_rows <= (dh > 64 ? kPool64Wide : kPool64) ? 64 : dh > 64 ? 128 : 256;
  const int p_tiles = (int)((p_rows + p.p_tile - 1) / p.p_tile);
  p.pooled = o_rows < 64 && ((double)b.b * p.o_tiles - p_tiles) * Hkv * P >= kPoolFrom;
  if (p.pooled && p.p_tile == 16 && p.o_tile > 16) p.p_tile = 64;
  if (!p.pooled && p.o_tile > 16) {
    const double ranges = (P + b.max_own + kLeastKeys - 1) / kLeastKeys;
    auto items = [&](int tile) { return (double)Hkv * b.b * ((o_rows + tile - 1) / tile) * ranges; };
    if (items(16) <= kSmall16)
      p.o_tile = 16;
    else if (items(p.o_tile) * ranges <= kSmall)
      p.o_tile = 64;
    p.o_tiles = (int)((o_rows + p.o_tile - 1) / p.o_tile);
  }
  p.p_tiles = p.pooled ? (int)((p_rows + p.p_tile - 1) / p.p_tile) : 0;
  const int axis = b.max_own + (p.pooled ? 0 : P);
  // Ranges of one length, so that no item is left with a few keys.
  // (A CU holds one block of 8 waves: more of them than CUs would be a second round.)
  auto eight = [dh](int tile) { return tile == 256 || (tile == 128 && dh > 64); };
  const int items16 = b.f32 && (dh > 64 || !p.pooled) ? kItemsWide : kItems16;
  const int four = b.e4m3 ? kItemsE4m3 : kItems, least = b.e4m3 ? kLeastKeysE4m3 : kLeastKeys;
  auto items = [&](int tile) { return eight(tile) ? kItems8 : tile > 16 ? four : items16; };
  auto cut = [&](int n, double axes, double want, int tile, int* keys) {
    int splits = 1;
    if (n > (tile == 16 ? kWhole16 : axes >= kFill ? kWholeFull : kWhole)) {
      const int most = std::min(kMostRanges, (n + least - 1) / least);
      const double parts = n / want;
      splits = (int)std::min((double)most, std::max(1.0, eight(tile) ? parts : std::ceil(parts)));
    }
    *keys = n > 0 ? ((n + splits - 1) / splits + 31) / 32 * 32 : 32;
    return n > 0 ? (n + *keys - 1) / *keys : 1;
  };
  const double p_axes = (double)Hkv * p.p_tiles, o_axes = (double)Hkv * b.b * p.o_tiles;
  const double p_work = p_axes * P, o_work = o_axes * axis;
  const bool one = !p.pooled || p.together();
  const double o_want = (one ? p_work + o_work : o_work) / items(p.o_tile);
  p.o_splits = cut(axis, o_axes, o_want, p.o_tile, &p.o_keys);
  p.p_splits = p.pooled ? cut(P, p_axes, one ? o_want : p_work / items(p.p_tile), p.p_tile, &p.p_keys) : 0;
  return p;
}

// Rows of the step kernels' own items where the plan says 16: those of a single token by vector
// instructions, up to 4 of fp32 keys and 2 of bf16 ones.
inline int step_rows(const Sizes& z) {
  const int rows = z.max_tok == 1 ? z.G : 16;
  return rows <= 2 ? rows : z.f32 && rows <= 4 ? 4 : 16;
}
// 16-column tiles of a head that the kernels are made for.
inline int head_tiles(int dh) {
  const int dt = (dh + 15) / 16;
  return dt <= 4 ? dt : dt <= 6 ? 6 : 8;
}

}  // namespace aurpaged
