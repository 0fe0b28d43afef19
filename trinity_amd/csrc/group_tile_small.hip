// Products in tiles of 32, 64 and 128 rows (group_tile.h).  Compiled with accumulators in ordinary registers: these kernels have room,
// and two copies of a loop body would move accumulators between the two files of registers.
#include "group_tile.h"

namespace tri {

template <GroupMul MUL, GroupKind KIND>
static int launch_tile_kind(const GroupArgs& a, int bm, hipStream_t stream) {
  // (k tiles in LDS: as many as leave room for two workgroups a CU)
  constexpr int D = MUL == kMul164 ? 2 : 3;
  constexpr bool EXPERTS = KIND == kGroupGate || KIND == kGroupDown;  // (experts_plan: 64 rows for 16-bit weights, 32 and 128 for 4-bit ones)
  switch (bm) {
    case 32:
      if constexpr (MUL == kMul16) return -1;
      else return launch_tile_t<GroupTile<32, 256, 1, 4, 3, D, MUL>, KIND>(a, stream);
    case 64:
      if constexpr (EXPERTS && MUL == kMul164) return -1;
      else return launch_tile_t<GroupTile<64, 128, 2, 2, 3, D, MUL>, KIND>(a, stream);
    default:
      if constexpr (MUL == kMul16) return -1;
      else return launch_tile_t<GroupTile<128, 128, 2, 2, 2, 2, MUL>, KIND>(a, stream);
  }
}

int launch_group_tile_small(const GroupArgs& a, GroupKind kind, int bm, hipStream_t stream) {
  const bool w4 = a.ws[0] != nullptr;
  switch (kind) {
    case kGroupRows: return a.xs != nullptr ? launch_tile_kind<kMul44, kGroupRows>(a, bm, stream) : launch_tile_kind<kMul164, kGroupRows>(a, bm, stream);
    case kGroupParts: return a.xs != nullptr ? launch_tile_kind<kMul44, kGroupParts>(a, bm, stream) : launch_tile_kind<kMul164, kGroupParts>(a, bm, stream);
    case kGroupGate: return w4 ? launch_tile_kind<kMul164, kGroupGate>(a, bm, stream) : launch_tile_kind<kMul16, kGroupGate>(a, bm, stream);
    default: return w4 ? launch_tile_kind<kMul164, kGroupDown>(a, bm, stream) : launch_tile_kind<kMul16, kGroupDown>(a, bm, stream);
  }
}

}  // namespace tri
