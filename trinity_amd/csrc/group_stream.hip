// Products of up to 16 rows (of a group) over 4-bit weights: weights go from memory to registers, 16 bytes - a block - per lane,
// a segment of 512 values of K (or two) ahead, and meet rows that wait in LDS.
//
// What bounds them: streaming the weights once, 4.25 bits a value.  At that width the rows are what costs: a wave that reads them
// from the cache beside its weights moves four bytes of each row pair for every byte of weights (16 rows x [4096, 14336]: 43 us),
// so a workgroup fetches its part of K of all rows once and takes several column tiles over it: 14 us; one row 25 -> 10.5, [14336,
// 4096] 10.2, 16 rows 16.7; 32 tokens over 8 experts of [4096, 14336 x 2] 99 us, 5.0 TB/s.  (Two segments ahead
// cost registers and give nothing elsewhere - one row 10.6 -> 11.8 us, gate and up 101 -> 120 -, but 2 to 10 % in the down projection,
// whose parts of K are short: 64 experts of [1792, 4096] 104 -> 94.)
//
// A workgroup has eight waves, `kw` of which share a tile of 16 columns (of gate and of up: 16 each) and take a part of K each -
// short sums are then spread over many waves, and they add up through LDS - and runs `tpw` tiles with every such set.  A 16x16x32
// MFMA multiplies the same eighth of four blocks: lane group g holds block 4 s + g of the columns, its values 8 j .. 8 j + 7 in
// MFMA j, and reads the rows at the same values.
#include "fp4.h"
#include "gemm_core.h"
#include "launch.h"

namespace tri {

constexpr int kStreamWaves = 8, kSegment = 512;

// RB: rows that LDS has room for (a.row_block are in use at a time)
template <GroupKind KIND, int RB>
__global__ __launch_bounds__(kStreamWaves * 64, 2) void group_stream_kernel(GroupArgs a) {
  extern __shared__ __attribute__((aligned(16))) half_t lds[];
  constexpr bool GATE = KIND == kGroupGate, ALL = KIND == kGroupRows || KIND == kGroupParts;
  constexpr int NM = GATE ? 2 : 1, NST = KIND == kGroupDown ? 3 : 2;  // (segments in registers, one of them in use)
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int kw = a.kw, cw = kStreamWaves / kw;  // ways of K, column tiles side by side
  const int way = wave % kw, col_way = wave / kw;

  // ---- which columns, part of K, group (column blocks are padded to a multiple of eight: every group's go to all XCDs)
  int id = blockIdx.x;
  const int cb = id % a.col_blocks;
  id /= a.col_blocks;
  const int part = id % a.ksplit, group = id / a.ksplit;
  const int tiles = (a.N + 15) / 16, tile0 = cb * cw * a.tpw;
  if (tile0 >= tiles) return;

  float4v* const sums = reinterpret_cast<float4v*>(lds);  // [waves][NM][64]
  int* const list = reinterpret_cast<int*>(sums + (kw > 1 ? kStreamWaves * NM * 64 : 0));
  half_t* const xs = reinterpret_cast<half_t*>(list + kStripChoices);
  int rows = a.M, expert = 0, place0 = 0;
  if constexpr (!ALL) {
    if (a.tiles != nullptr) {
      if (group >= a.tiles[0].x) return;  // (counted on the device)
      const int4 tile = a.tiles[1 + group];
      expert = tile.x;
      place0 = tile.y;
      rows = tile.z;
    } else {  // the choices of the expert of choice `group`, if that is the first of them
      const int mine = lane < a.n ? a.ids[lane] : -1;
      expert = __builtin_amdgcn_readlane(mine, group);
      const uint64_t same = __ballot(mine == expert);
      if (expert < 0 || expert >= a.E || __builtin_ctzll(same) != group) return;
      if (mine == expert) list[__popcll(same & ((1ull << lane) - 1))] = lane;  // (every wave the same values)
      rows = __popcll(same);
      __syncthreads();
    }
  }
  // place of row r: among the choices themselves, or in the order that expert_rows_kernel made
  auto choice_of = [&](int r) { return ALL ? r : (a.tiles != nullptr ? a.rows[place0 + r] : list[r]); };
  auto place_of = [&](int r) { return ALL ? r : (a.tiles != nullptr ? place0 + r : list[r]); };

  // ---- K: the workgroup's part, and this wave's segments of it
  const int segs = (a.K + kSegment - 1) / kSegment, seg_part = (segs + a.ksplit - 1) / a.ksplit;
  const int seg0 = part * seg_part, nseg = min(seg_part, segs - seg0);
  const int k0 = seg0 * kSegment, deep = min(nseg * kSegment, a.K - k0);
  const int per = (nseg + kw - 1) / kw;  // segments of a way (the last ones may have fewer)
  const int s0 = way * per, mine = max(0, min(per, nseg - s0));
  const int nb = a.K / 32;
  const int tpw = min(a.tpw, (tiles - tile0 + cw - 1) / cw);  // tiles of the workgroup's busiest set
  const int steps = tpw * mine;                               // segments of this wave

  const uint8_t *const w1 = a.w[0] + expert * a.w_se[0], *const w2 = GATE ? a.w[1] + expert * a.w_se[1] : w1;
  const uint8_t *const x1 = a.ws[0] + expert * a.ws_se[0], *const x2 = GATE ? a.ws[1] + expert * a.ws_se[1] : x1;
  const int last16 = a.K / 2 - 16;
  uint4v wq[NST][NM][4], sc[NST][NM];
  // what is loaded next: tile of the workgroup, segment of this wave; past the end one line over and over (a number of loads on their
  // way that the compiler knows lets it wait for the oldest alone)
  int to_tile = 0, to_seg = 0;
  auto load = [&](int st) __attribute__((always_inline)) {
    const int sg = seg0 + s0 + to_seg;
    const uint32_t live = to_tile < tpw ? ~0u : 0u;
    const uint32_t col = (uint32_t)min(min(tile0 + to_tile * cw + col_way, tiles - 1) * 16 + c, a.N - 1);
    const int at = min(sg * 16, nb - 16);  // its scales: sixteen bytes of the row
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      const uint8_t* const w = m ? w2 : w1;
      const uint32_t row = col * (uint32_t)a.w_ld[m];
#pragma unroll
      for (int s = 0; s < 4; ++s)
        wq[st][m][s] = *reinterpret_cast<const uint4v*>(w + ((row + (uint32_t)min(sg * 256 + s * 64 + g * 16, last16)) & live));
      __builtin_memcpy(&sc[st][m], (m ? x2 : x1) + ((col * (uint32_t)a.ws_ld[m] + (uint32_t)at) & live), 16);
    }
    if (++to_seg == mine) {
      to_seg = 0;
      ++to_tile;
    }
  };

  for (int r0 = 0; r0 < rows; r0 += a.row_block) {
    const int nr = min(a.row_block, rows - r0);
    to_tile = to_seg = 0;
    if (mine > 0) {
#pragma unroll
      for (int s = 0; s < NST - 1; ++s) load(s);
    }
    // ---- the rows' part of K to LDS, zeros behind K
    // (LDS: [chunk of eight values][row], so that a fragment read - one chunk of 16 rows - falls on different banks.  A wave fetches
    // 64 / rows chunks of all rows, four times at a time.)
    constexpr int lanes = 64 / RB;
    const int fr = lane % RB, chunks = nseg * (kSegment / 8);
    const int64_t from = (GATE ? choice_of(r0 + min(fr, nr - 1)) / a.top_k : place_of(r0 + min(fr, nr - 1))) * a.ldx;
    for (int q0 = wave * lanes + lane / RB; q0 < chunks; q0 += kStreamWaves * lanes * 4) {
      half8v v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int k = min(q0 + u * kStreamWaves * lanes, chunks - 1) * 8;
        v[u] = *reinterpret_cast<const half8v*>(a.x + from + (int64_t)(k0 + min(k, deep - 8)) * 2);
        if (k >= deep) v[u] = half8v{};
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int q = q0 + u * kStreamWaves * lanes;
        if (q < chunks && fr < nr) *reinterpret_cast<half8v*>(xs + (q * RB + fr) * 8) = v[u];
      }
    }
    __syncthreads();
    const half_t* const xr = xs + (g * 4 * RB + min(c, nr - 1)) * 8;
    float4v acc[NM];
#pragma unroll
    for (int m = 0; m < NM; ++m) acc[m] = float4v{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](int in_tile, int st) __attribute__((always_inline)) {
      const int sl = s0 + in_tile, sg = seg0 + sl;  // segment of the part, and of K
      const half_t* const x = xr + sl * kSegment * RB;
      const int off = sg * 16 - min(sg * 16, nb - 16);  // bytes that the scales were fetched too early
      if (off != 0) {
#pragma unroll
        for (int m = 0; m < NM; ++m) {
          uint4v v = sc[st][m];
          for (int b = 0; b < off; ++b) {  // (at most fifteen, in the last segment only; what comes in stands for no block)
            v[0] = (v[0] >> 8) | (v[1] << 24);
            v[1] = (v[1] >> 8) | (v[2] << 24);
            v[2] = (v[2] >> 8) | (v[3] << 24);
            v[3] >>= 8;
          }
          sc[st][m] = v;
        }
      }
      // (the rows' fragments of the next four MFMAs are on their way while these are multiplied)
      half8v xf[2][4];
      auto rows_of = [&](int s, int set) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) xf[set][j] = *reinterpret_cast<const half8v*>(x + (s * 16 + j) * 8 * RB);
      };
      rows_of(0, 0);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if (s < 3) rows_of(s + 1, (s + 1) & 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int m = 0; m < NM; ++m) {
          const float scale = fp4_scale((sc[st][m][s] >> (g * 8)) & 255);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[m] = mfma16(fp4x8_to_half8(wq[st][m][s][j], scale), xf[s & 1][j], acc[m]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto store = [&](int tl) __attribute__((always_inline)) {  // lane: row c, columns 16 tl + 4 g .. + 3
      const int n = tl * 16 + g * 4;
      if (c >= nr || tl >= tiles || n >= a.N) return;
      if constexpr (KIND == kGroupParts || KIND == kGroupDown) {
        const int64_t at = KIND == kGroupParts ? (int64_t)part * a.M + r0 + c : (int64_t)part * a.n + choice_of(r0 + c);
        *reinterpret_cast<float4v*>(a.y + at * a.N + n) = acc[0];
      } else {
        half4v h;
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = (half_t)(GATE ? silu(acc[0][e]) * acc[NM - 1][e] : acc[0][e]);
        *reinterpret_cast<half4v*>(a.out + (int64_t)place_of(r0 + c) * a.ldo + n) = h;
      }
    };
    int tile_i = 0;  // tiles done
    // a tile is over: the ways of K add up, in order
    auto finish = [&]() __attribute__((always_inline)) {
      const int tl = tile0 + tile_i * cw + col_way;
      const bool adds = way == tile_i % kw;  // (in turn)
      if (kw > 1) {
        __syncthreads();  // (the sums of the tile before have been read)
#pragma unroll
        for (int m = 0; m < NM; ++m) sums[(wave * NM + m) * 64 + lane] = acc[m];
        __syncthreads();
        if (adds) {
#pragma unroll
          for (int m = 0; m < NM; ++m) {
            acc[m] = sums[(wave - way) * NM * 64 + m * 64 + lane];
            for (int w = 1; w < kw; ++w) acc[m] += sums[((wave - way + w) * NM + m) * 64 + lane];
          }
        }
      }
      if (adds) store(tl);
      ++tile_i;
#pragma unroll
      for (int m = 0; m < NM; ++m) acc[m] = float4v{0.f, 0.f, 0.f, 0.f};
    };
    if (mine > 0) {
      int in_tile = 0;
      for (int i0 = 0; i0 < steps; i0 += NST) {
#pragma unroll
        for (int st = 0; st < NST; ++st) {
          load((st + NST - 1) % NST);
          if (i0 + st < steps) {
            multiply(in_tile, st);
            if (++in_tile == mine) {
              in_tile = 0;
              finish();
            }
          }
        }
      }
    } else {
      for (int i = 0; i < tpw; ++i) finish();  // (a way without segments: zeros)
    }
    __syncthreads();  // (the rows' place is filled again)
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct StreamPlan {
  int kw, tpw, ksplit, row_block, col_blocks, lds, room_rows;
};
// groups: how many have rows; at most `rows` rows each
static StreamPlan stream_plan(int rows, int K, int N, int groups, bool gate, bool may_split) {
  StreamPlan p;
  const int segs = (K + kSegment - 1) / kSegment, tiles = (N + 15) / 16;
  const int list = kStripChoices * 4, sums = kStreamWaves * (gate ? 2 : 1) * 1024;
  const int room = 160 * 1024 - list;
  auto row_bytes = [&](int parts) { return (segs + parts - 1) / parts * kSegment * 2; };
  p.room_rows = rows <= 1 ? 1 : (rows <= 4 ? 4 : 16);
  p.ksplit = 1;
  while (may_split && p.room_rows * row_bytes(p.ksplit) > room) ++p.ksplit;
  while (p.room_rows > 1 && p.room_rows * row_bytes(p.ksplit) > room) p.room_rows /= 4;
  p.row_block = rows < p.room_rows ? rows : p.room_rows;
  const int per = (segs + p.ksplit - 1) / p.ksplit;
  p.ksplit = (segs + per - 1) / per;  // (no part is empty)
  // ways of K, where their sums fit beside the rows: for waves that would have no tile otherwise, and two at least - neighbours then
  // read the same rows of weights one behind the other (32 tokens, 8 experts of [4096, 14336 x 2]: 107 -> 102 us)
  const int64_t waves = (int64_t)groups * p.ksplit * tiles;
  const int bytes = p.room_rows * row_bytes(p.ksplit);
  p.kw = 1;
  while (p.kw < kStreamWaves && bytes + sums <= room && (waves * p.kw < 256 * kStreamWaves || p.kw < 2) && p.kw * 2 <= per) p.kw *= 2;
  p.lds = list + (p.kw > 1 ? sums : 0) + bytes;
  const int cw = kStreamWaves / p.kw, most = (tiles + cw - 1) / cw;
  // a workgroup a CU, and eight of a group at least, which go to the XCDs in turn: with a workgroup a CU alone, four of each of 64 experts
  // ran on four XCDs (64 tokens x 6 of 64 experts of [4096, 1792]: 166 + 96 -> 106 + 61 us; of 128 experts 593 + 336 -> 204 + 115)
  const int units = groups * p.ksplit, share = (255 + units) / units, blocks = share > 8 ? share : 8;
  p.tpw = (most + blocks - 1) / blocks;
  p.col_blocks = ((most + p.tpw - 1) / p.tpw + 7) / 8 * 8;
  return p;
}
// rows of this length fit the LDS all together
static bool stream_fits(int rows, int K) {
  const int deep = (K + kSegment - 1) / kSegment * kSegment;
  return (int64_t)(rows <= 1 ? 1 : (rows <= 4 ? 4 : 16)) * deep * 2 <= 160 * 1024 - kStripChoices * 4;
}

template <GroupKind KIND, int RB>
static int launch_stream_rows(const GroupArgs& a, const StreamPlan& p, int groups, hipStream_t stream) {
  constexpr auto kern = group_stream_kernel<KIND, RB>;
  if (set_max_lds<kern, 160 * 1024>() != 0) return -1;
  hipLaunchKernelGGL(kern, dim3(p.col_blocks * p.ksplit * groups), dim3(kStreamWaves * 64), p.lds, stream, a);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
template <GroupKind KIND>
static int launch_stream_kind(GroupArgs a, const StreamPlan& p, int groups, hipStream_t stream) {
  a.ksplit = p.ksplit;
  a.kw = p.kw;
  a.tpw = p.tpw;
  a.row_block = p.row_block;
  a.col_blocks = p.col_blocks;
  if (p.room_rows == 1) return launch_stream_rows<KIND, 1>(a, p, groups, stream);
  return p.room_rows == 4 ? launch_stream_rows<KIND, 4>(a, p, groups, stream) : launch_stream_rows<KIND, 16>(a, p, groups, stream);
}

// (by tiles of 32 rows instead, us, [4096, 14336], [14336, 4096], [4544, 4544]: one row 17.3, 17.6, 15.6 for 10.8, 10.4, 6.6; 16 rows 18.4,
// 18.6, 16.2 for 14.0, 16.8, 10.8)
bool group_stream_takes(int rows, int K, bool may_split) { return rows <= 16 && K >= kSegment && (may_split || stream_fits(rows, K)); }
int group_stream_parts(int rows, int K, int N, int groups) { return stream_plan(rows, K, N, groups, false, true).ksplit; }

int launch_group_stream(const GroupArgs& a, GroupKind kind, int rows, int groups, int grid_groups, hipStream_t stream) {
  const StreamPlan p = stream_plan(rows, a.K, a.N, groups, kind == kGroupGate, kind != kGroupGate && kind != kGroupRows);
  switch (kind) {
    case kGroupRows: return launch_stream_kind<kGroupRows>(a, p, grid_groups, stream);
    case kGroupParts: return launch_stream_kind<kGroupParts>(a, p, grid_groups, stream);
    case kGroupGate: return launch_stream_kind<kGroupGate>(a, p, grid_groups, stream);
    default: return launch_stream_kind<kGroupDown>(a, p, grid_groups, stream);
  }
}

}  // namespace tri
