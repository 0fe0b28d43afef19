// Products in tiles of 256 rows (group_tile.h), and the plans of them all.
#include "group_tile.h"

namespace tri {

#ifndef STREAMMEAN
#define STREAMMEAN 10
#endif
// parts of K for `tiles` tiles: so many that every CU has one, of at least 512 values
static int parts_of(int tiles, int K) {
  const int deep = (K + 255) / 256;
  int parts = tiles >= 256 ? 1 : 256 / tiles;
  if (parts > deep / 2) parts = deep / 2 > 0 ? deep / 2 : 1;
  const int per = (deep + parts - 1) / parts;
  return (deep + per - 1) / per;  // (no part is empty)
}

GroupPlan experts_plan(int choices, int top_k, int experts, int N, int F, bool w4) {
  GroupPlan p;
  const int mean = (choices + experts - 1) / experts;
  const int rows = choices / top_k < 16 ? choices / top_k : 16;  // (of an expert, at most, if a token chooses it once)
  if (w4 && mean <= STREAMMEAN && group_stream_takes(rows, N, false) && group_stream_takes(rows, F, true)) {
    p.bm = 16;
    p.ksplit = group_stream_parts(rows, F, N, choices < experts ? choices : experts);
    return p;
  }
  p.bm = mean <= 24 ? 32 : (mean <= 64 ? 64 : (mean <= 256 ? 128 : 256));
  const int bn = p.bm == 32 || p.bm == 256 ? 256 : 128;
  const int groups = choices < experts ? choices : experts;
  p.ksplit = parts_of(((mean + p.bm - 1) / p.bm) * groups * ((N + bn - 1) / bn), F);
  return p;
}

int experts_parts(int choices, int top_k, int experts, int N, int F) {
  const int a = experts_plan(choices, top_k, experts, N, F, false).ksplit, b = experts_plan(choices, top_k, experts, N, F, true).ksplit;
  return a > b ? a : b;
}

GroupPlan group_rows_plan(int M, int K, int N, bool x4) {
  GroupPlan p;
  p.bm = M <= 32 ? 32 : (M <= 64 ? 64 : (M <= 256 ? 128 : 256));
  const int bn = p.bm == 32 || p.bm == 256 ? 256 : 128;
  p.ksplit = parts_of(((M + p.bm - 1) / p.bm) * ((N + bn - 1) / bn), K);
  return p;
}

int64_t fp4_matmul_workspace(int M, int K, int N, bool x4) {
  const int parts = !x4 && group_stream_takes(M, K, true) ? group_stream_parts(M, K, N, 1) : group_rows_plan(M, K, N, x4).ksplit;
  return parts > 1 ? (int64_t)parts * M * N * 4 : 0;
}

template <GroupMul MUL, GroupKind KIND>
static int launch_tile_kind(const GroupArgs& a, int, hipStream_t stream) {
  return launch_tile_t<GroupTile<256, 256, 2, 2, 2, MUL == kMul16 ? 3 : 2, MUL>, KIND>(a, stream);
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
