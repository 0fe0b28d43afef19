// Products in tiles of 256 rows (group_tile.h), and the plans of them all.
#include "group_tile.h"

namespace tri {

// Workgroups that a CU holds side by side (by their LDS): two of the small tiles, and they hide each other's waits; one of 256 x 256.
static int tile_slots(int bm) { return bm == 256 ? 256 : 512; }
static int tile_cols(int bm) { return bm == 32 || bm == 256 ? 256 : 128; }

// parts of K for `tiles` tiles: so many that all slots are taken, of at least 512 values
static int parts_of(int tiles, int K, int slots) {
  const int deep = (K + 255) / 256;
  int parts = tiles >= slots ? 1 : slots / tiles;
  if (parts > deep / 2) parts = deep / 2 > 0 ? deep / 2 : 1;
  const int per = (deep + parts - 1) / parts;
  return (deep + per - 1) / per;  // (no part is empty)
}

// Rows of a tile by the mean rows of an expert.  us of both products of 8 experts of [4096, 14336], by 32, 64, 128, 256 rows:
//   16-bit weights, 32 rows each 555, 501, 574, 499; 42 of 32 experts of [4544, 2272] -, 401, -, 435; 64 818, 669, 588, 507; 150 1395,
//     1116, 740, 591; 500 3800, 2710, 1990, 1540
//   4-bit weights, 32 rows 228, 281, 371, 312; 64 373, 387, 384, 361; 100 479, 459, 404, 383
// From there on 4-bit weights go by whole tiles: 256 rows while an expert has one of them, 128 where a second one would be half empty, and
// 256 beyond.  Time of a call with 256 over that with 128 rows, of 8 experts of [4096, 14336], 64 of [4096, 1792], 32 of [4544, 2272], 16 of
// [2048, 8192] and 128 of [2048, 1024] - their mean; without the last from 700 on, and the second at 2000 -, first with the same rows for
// each, then as a router's random choices fall:
//   150 0.83, 1.03; 190 0.84, 1.05; 225 0.98, 1.03; 256 0.98, 1.02; 270 1.07, 1.02; 350 1.08, 0.98; 400 0.90, 1.00; 700 0.92, 0.96;
//   1000 0.90, 0.96; 2000 0.90, 0.93.  (One call of random choices is off from its neighbours by up to 20 % either way.)
GroupPlan experts_plan(int choices, int top_k, int experts, int N, int F, bool w4) {
  GroupPlan p;
  const int mean = (choices + experts - 1) / experts, groups = choices < experts ? choices : experts;
  const int rows = choices / top_k < 16 ? choices / top_k : 16;  // (of an expert, at most, if a token chooses it once)
  // (few rows stream past the weights at once: 8 each of 8 experts of [4096, 14336] 165 us, 183 by tiles of 32 rows; where an expert is
  // likely to have more than 16, twice: 9.4 each of 64 of [4096, 1792] 247, 193)
  // Rows wider than LDS holds as many as an expert may have (16 of up to 4608 values, 4 of 19968, one of 81408) go by tiles: four rows at a
  // time would have the experts of more than four stream their weights again.  That and tiles, us: 8, 16 and 32 tokens x 2 of 8 of [5120,
  // 14336] 252 for 198, 279 for 214, 470 for 227; 8, 32 and 64 x 6 of 64 of [5120, 1792] 177 for 129, 297 for 224, 405 for 234; of
  // [7168, 2048] 237 for 220, 413 for 301, 606 for 320; x 8 of 256 of [7168, 2048] 274 for 299, 673 for 704, 1026 for 1009 and,
  // 128 tokens, 1589 for 1185.  (At [4096, 14336] 16 rows in LDS 145, 158 and 164 for 170, 176 and 178.)
  if (w4 && mean <= 8 && group_stream_takes(rows, N, false) && group_stream_takes(rows, F, true)) {
    p.bm = 16;
    p.ksplit = group_stream_parts(rows, F, N, groups);
    return p;
  }
  p.bm = w4 ? (mean <= 48 ? 32 : (mean <= 256 || mean > 384 ? 256 : 128)) : (mean <= 48 ? 64 : 256);
  const int tiles = ((mean + p.bm - 1) / p.bm) * groups * ((N + tile_cols(p.bm) - 1) / tile_cols(p.bm));
  p.ksplit = parts_of(tiles, F, tile_slots(p.bm));
  return p;
}

int experts_parts(int choices, int top_k, int experts, int N, int F) {
  const int a = experts_plan(choices, top_k, experts, N, F, false).ksplit, b = experts_plan(choices, top_k, experts, N, F, true).ksplit;
  return a > b ? a : b;
}

// The cheapest tile and number of parts, by what a round of workgroups takes for a k tile (us; measured over [4544, 18176] and
// [14336, 4096] at 24 to 4096 rows): with every slot taken, and with one workgroup a CU at most; 3 us to begin and end a round; the parts'
// sums cost their trip to memory and the launch that joins them.
GroupPlan group_rows_plan(int M, int K, int N, bool x4) {
  struct Cost {
    int bm;
    float full, half;
  };
  static const Cost k164[4] = {{32, 0.68f, 0.33f}, {64, 0.64f, 0.46f}, {128, 0.90f, 0.57f}, {256, 1.40f, 1.40f}};
  static const Cost k44[4] = {{32, 2.4f, 1.3f}, {64, 1.7f, 1.05f}, {128, 1.85f, 1.3f}, {256, 2.6f, 2.6f}};
  GroupPlan best = {256, 1};
  float least = 1e30f;
  const int deep = (K + 255) / 256;
  for (const Cost& c : x4 ? k44 : k164) {
    const int row_tiles = (M - 1) / c.bm + 1, col_tiles = (N - 1) / tile_cols(c.bm) + 1, slots = tile_slots(c.bm);
    const int64_t tiles = (int64_t)row_tiles * col_tiles;
    const int most = parts_of(tiles < slots ? (int)tiles : slots, K, slots);
    // (a 256-row tile of fewer rows, the only one in a column, costs less)
    const float share = c.bm == 256 && row_tiles == 1 && !x4 ? 0.22f + 0.08f * (float)((M + 63) / 64) : 1.0f;
    for (int want = 1; want <= most; ++want) {
      const int per = (deep + want - 1) / want, parts = (deep + per - 1) / per;  // (no part is empty)
      const int64_t units = tiles * parts, rounds = (units - 1) / slots, last = (units - 1) % slots + 1;
      const float round = (float)rounds * c.full + (last > 256 || slots == 256 ? c.full : c.half);
      float us = round * share * (float)per * (x4 ? 1.0f : 4.0f) + 3.0f * (float)(rounds + 1);
      if (parts > 1) us += 4.0f + (float)parts * (float)M * (float)N * 2.5e-6f;
      if (us < least) {
        least = us;
        best = {c.bm, parts};
      }
    }
  }
  return best;
}

int64_t fp4_matmul_workspace(int M, int K, int N, bool x4) {
  const int parts = !x4 && group_stream_takes(M, K, true) ? group_stream_parts(M, K, N, 1) : group_rows_plan(M, K, N, x4).ksplit;
  return parts > 1 ? (int64_t)parts * M * N * 4 : 0;
}

template <GroupMul MUL, GroupKind KIND>
static int launch_tile_kind(const GroupArgs& a, int, hipStream_t stream) {
  return launch_tile_t<GroupTile<256, 256, 2, MUL == kMul164 ? 4 : 2, 2, MUL == kMul16 ? 3 : 2, MUL>, KIND>(a, stream);
}

int launch_group_tile(const GroupArgs& a, GroupKind kind, int bm, hipStream_t stream) {
  if (bm < 256) return launch_group_tile_small(a, kind, bm, stream);
  const bool w4 = a.ws[0] != nullptr;
  switch (kind) {
    case kGroupRows: return a.xs != nullptr ? launch_tile_kind<kMul44, kGroupRows>(a, bm, stream) : launch_tile_kind<kMul164, kGroupRows>(a, bm, stream);
    case kGroupParts: return a.xs != nullptr ? launch_tile_kind<kMul44, kGroupParts>(a, bm, stream) : launch_tile_kind<kMul164, kGroupParts>(a, bm, stream);
    case kGroupGate: return w4 ? launch_tile_kind<kMul164, kGroupGate>(a, bm, stream) : launch_tile_kind<kMul16, kGroupGate>(a, bm, stream);
    default: return w4 ? launch_tile_kind<kMul164, kGroupDown>(a, bm, stream) : launch_tile_kind<kMul16, kGroupDown>(a, bm, stream);
  }
}

}  // namespace tri
