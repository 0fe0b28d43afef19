// Products over K-contiguous weights in tiles of rows: of all rows (4-bit weights), or of the rows of every expert, which
// expert_rows_kernel has put next to each other.  Three kinds of multiplication, one loop:
//   kMul16   16-bit rows and weights:   32x32x16 MFMAs
//   kMul164  16-bit rows, 4-bit weights: the same, weights converted on their way from LDS
//   kMul44   4-bit rows and weights:    32x32x64 MFMAs that take the blocks' scales
//
// A k tile is 128 bytes of a row: 64 values, or 256 in 4 bits.  (kMul164: the weights' 128 bytes last for four k tiles of the
// rows.)  Both operands go global -> LDS without passing through registers, whole 128-byte lines, chunk c (of 16 bytes) of row r
// at slot c ^ ((r >> 1) & 7), so that fragment reads are free of bank conflicts.  A lane's 16 bytes are its share of an MFMA
// either way: eight values of 16 bits, or a whole block of 32 in 4 bits.  K ends within a k tile: addresses stop at the row's last
// 16 bytes, and what they fetch in place of values behind it is not multiplied (16-bit rows: two of the four steps are left out),
// or by the scale 2^-127 on either side (4-bit rows: its products vanish, and codes are finite).
//
// Scales (a byte per block, rows of any alignment): a thread keeps the next 32 bytes of one or two rows - a trip to memory for 1024
// values of K, as a row's bytes for 256 would have each cost a whole line again - and hands the eight of a 256-deep tile over through LDS.
// kMul44: lane group g takes the chunks 4 g to 4 g + 3 of a k tile, whose four scales are one word (which values of K meet in an
// MFMA is free as long as both operands agree).
//
// One barrier per k tile, in front of the last of its four steps, when the next tile must have landed; that step then requests
// the tile that takes its place.
//
// What bounds them and what they take:
//   kMul16   4096 tokens x 2 of 8 experts of [4096, 14336], 256 x 256 tiles, fp16: gate and up 1.68 to 1.87 ms, down 1.16 to 1.24, 1.03
//            and 0.83 PFLOP/s: the power limit (a library product of 8192 cubed 1.16).  333 tokens x 4 of 32 experts of [4544, 2272], 64 x
//            128 tiles: 250 + 152 us, the weights' bytes at 4.9 TB/s
//   kMul164  333 rows x [4544, 18176], 128 x 128 tiles: 68 us, 0.81 PFLOP/s, conversions between MFMAs; 256 x 256 tiles, eight waves:
//            2048 tokens x 6 of 64 experts of [4096, 1792] 417 + 232 us
//   kMul44   4096 rows x [4096, 14336], 256 x 256 tiles: 153 to 160 us, 3.1 PFLOP/s; [14336, 4096] 125, 3.8.  MFMAs are busy 37 % of that
//            time (a k tile takes 2.5 us, they 1.0).  Not the L2's rate: 64 KB a CU and k tile are 13 bytes a clock, a read's
//            latency 340 clocks.  A k tile's loads are asked for in the step before it begins and waited for three steps later,
//            and a SIMD has one wave: a quarter of the waves' time waits for loads and barriers, a third for an instruction to issue.
//            LDS has room for two k tiles (four of half a line each: 177 and 145 us)
#if (defined(TRI_BF16) && !defined(TRI_GROUP_TILE_H_BF16)) || (!defined(TRI_BF16) && !defined(TRI_GROUP_TILE_H_F16))
#ifdef TRI_BF16
#define TRI_GROUP_TILE_H_BF16
#else
#define TRI_GROUP_TILE_H_F16
#endif
#include <type_traits>

#include "fp4.h"
#include "gemm_core.h"
#include "launch.h"

namespace tri {

enum GroupMul { kMul16, kMul164, kMul44 };

typedef int int8x __attribute__((ext_vector_type(8)));

// NA, NB: k tiles of rows and of weights (kMul164: 256 deep) in LDS
template <int BM_, int BN_, int WM_, int WN_, int NA_, int NB_, GroupMul MUL_>
struct GroupTile {
  static constexpr GroupMul MUL = MUL_;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NA = NA_, NB = NB_;
  static constexpr int NW = WM * WN, NT = NW * 64;
  static constexpr int TM = BM / WM, TN = BN / WN, MI = TM / 32, NI = TN / 32;
  static constexpr int XI = BM / 8 / NW, WI = BN / 8 / NW;  // 1 KB load instructions per wave and tile
  static constexpr bool XS = MUL == kMul44, WS = MUL != kMul16;
  static constexpr int SROWS = (WS ? BN : 0) + (XS ? BM : 0), SR = (SROWS + NT - 1) / NT;  // rows of scales, per thread
  static constexpr int SUB = MUL == kMul164 ? 4 : 1;  // k tiles of rows per tile of weights
  static constexpr int KX = MUL == kMul44 ? 256 : 64, KW = MUL == kMul16 ? 64 : 256;
  static constexpr int W_BYTES = BN * 128, S_BYTES = SROWS * 8;
  // a tile whose waves have `live` row blocks: bytes of a k tile's rows, and how many k tiles of them LDS holds
  static constexpr int x_bytes(int live) { return live * WM * 32 * 128; }
  static constexpr int na(int live) { return MUL == kMul164 && MI == 4 && live < 4 ? (live == 3 ? 3 : 4) : NA; }
  static constexpr int x_room() {
    int most = 0;
    for (int l = 1; l <= MI; ++l) most = most > na(l) * x_bytes(l) ? most : na(l) * x_bytes(l);
    return most;
  }
  static constexpr int X_OFF = 0, W_OFF = x_room(), S_OFF = W_OFF + NB * W_BYTES;
  static constexpr int LOOP_BYTES = S_OFF + 2 * S_BYTES, STAGED_BYTES = NW * TM * (TN + 8) * 2;  // (STAGED: of the epilogue)
  static constexpr int LDS_BYTES = LOOP_BYTES > STAGED_BYTES ? LOOP_BYTES : STAGED_BYTES;
  static constexpr bool DEEP = MI * NI <= 4;  // fragments are read a whole k tile ahead (see there)
  static constexpr bool LATE = NB > NA && SUB == 1;  // weights are requested in the first step of a tile
  static_assert((NW == 4 || NW == 8) && BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && TM % 32 == 0 && TN % 32 == 0, "four or eight waves");
  static_assert(WM * 4 % NW == 0, "whole load instructions for a row block of every wave");
  static_assert(NA >= 2 && NB >= 2 && LDS_BYTES <= 160 * 1024, "LDS budget");
  static_assert(NA == NB || LATE || SUB == 4, "waits below");
  static_assert(!LATE || (NA == 2 && NB == 3), "waits below");
  static_assert(SUB == 1 || NA <= 4, "waits below");
  // loads that may be on their way at the barrier of a tile; xi: those of rows per wave and tile
  static constexpr int inflight(int na, int xi) { return SUB == 4 ? (na - 2) * xi : (LATE ? WI : (na - 2) * (xi + WI)); }
  static_assert(inflight(NA, XI) + WI < 64, "vmcnt");
};

__device__ __forceinline__ void dma16(const void* g, void* l) {
  load_to_lds16(static_cast<const half_t*>(g), static_cast<half_t*>(l));
}

template <class T, GroupKind KIND>
__global__ __launch_bounds__(T::NT) void group_tile_kernel(GroupArgs a) {
  extern __shared__ __attribute__((aligned(16))) half_t lds_h[];
  char* const lds = reinterpret_cast<char*>(lds_h);
  constexpr bool GATE = KIND == kGroupGate, ALL = KIND == kGroupRows || KIND == kGroupParts;
  constexpr int OUT_BN = GATE ? T::BN / 2 : T::BN, OUT_TN = GATE ? T::TN / 2 : T::TN;
  constexpr GroupMul MUL = T::MUL;
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = wave % T::WM, wn = wave / T::WM;
  const int l32 = lane & 31, g = lane >> 5;

  // ---- which tile
  const int tiles_m = ALL ? (a.M + T::BM - 1) / T::BM : a.tiles[0].x;
  const int tiles_n = (a.N + OUT_BN - 1) / OUT_BN;
  if ((int)blockIdx.x >= tiles_m * tiles_n * a.ksplit) return;  // (the experts' tiles are counted on the device)
  int tm, tn;
  tile_coords(blockIdx.x, tiles_m, tiles_n * a.ksplit, T::BN >= 256 ? 8 : 4, tm, tn);
  const int split = tn / tiles_n;
  tn -= split * tiles_n;
  const int n0 = tn * OUT_BN;
  int expert = 0, place0 = tm * T::BM, rows = min(T::BM, a.M - tm * T::BM);
  if constexpr (!ALL) {
    const int4 tile = a.tiles[1 + tm];
    expert = tile.x;
    place0 = tile.y;
    rows = tile.z;
  }
  // k tiles of this part: whole 256-deep ones
  const int deep = (a.K + 255) / 256, per = (deep + a.ksplit - 1) / a.ksplit;
  const int k0 = split * per * 256, k1 = min(a.K, k0 + per * 256);
  const int KT = (k1 - k0 + T::KX - 1) / T::KX, MT = (k1 - k0 + T::KW - 1) / T::KW;
  const int x0 = MUL == kMul44 ? k0 / 2 : k0 * 2, w0 = MUL == kMul16 ? k0 * 2 : k0 / 2;  // bytes

  // ---- load sources: a base that all lanes share and 32 bits of distance from it
  const int chunk = (lane & 7) ^ ((wave * 4 + (lane >> 4)) & 7);  // (the same for all of a lane's loads)
  const uint8_t* const xbase = a.x + (GATE ? 0 : place0 * a.ldx) + x0;
  const uint8_t* const xsbase = T::XS ? a.xs + (GATE ? 0 : place0 * a.ldxs) + k0 / 32 : nullptr;
  // (variables, no arrays: an index that is not known to the compiler would put those into memory)
  const uint8_t *const wbase = a.w[0] + expert * a.w_se[0] + w0, *const wbase2 = GATE ? a.w[1] + expert * a.w_se[1] + w0 : wbase;
  const uint8_t* const sbase = T::WS ? a.ws[0] + expert * a.ws_se[0] + k0 / 32 : nullptr;
  const uint8_t* const sbase2 = T::WS && GATE ? a.ws[1] + expert * a.ws_se[1] + k0 / 32 : sbase;
  const uint32_t ldw = (uint32_t)a.w_ld[0], ldw2 = GATE ? (uint32_t)a.w_ld[1] : ldw, ld_s = (uint32_t)a.ws_ld[0], ld_s2 = GATE ? (uint32_t)a.ws_ld[1] : ld_s;
  auto input_row = [&](int rloc) -> int {  // from xbase
    const int r = min(rloc, rows - 1);
    if constexpr (GATE) return a.rows[place0 + r] / a.top_k;
    return r;
  };
  // LDS row of the weight tile -> weight matrix (the same for 32 rows) and its column
  auto column = [&](int nloc, int& m) {
    m = 0;
    int col = n0 + nloc;
    if constexpr (GATE) {  // a wave has its gate columns, then the up columns of the same outputs
      const int within = nloc % T::TN;
      m = within / OUT_TN;
      col = n0 + nloc / T::TN * OUT_TN + within % OUT_TN;
    }
    return col < a.N ? col : n0;
  };
  uint32_t xofs[T::XI], wofs[T::WI];
#pragma unroll
  for (int i = 0; i < T::XI; ++i) xofs[i] = (uint32_t)input_row((i * T::NW + wave) * 8 + (lane >> 3)) * (uint32_t)a.ldx;
#pragma unroll
  for (int i = 0; i < T::WI; ++i) {
    int m;
    const int col = column((i * T::NW + wave) * 8 + (lane >> 3), m);
    wofs[i] = (uint32_t)col * (m ? ldw2 : ldw);
  }
  const int nb = (k1 - k0) / 32;  // blocks of this part
  const int xend = (MUL == kMul44 ? (k1 - k0) / 2 : (k1 - k0) * 2) - 16, wend = (MUL == kMul16 ? (k1 - k0) * 2 : (k1 - k0) / 2) - 16;
  // (past the end the loop keeps its load count, which the waits assume)
  auto load_x = [&](int kt, int buf, int i, int live) __attribute__((always_inline)) {
    const uint32_t k = (uint32_t)min(kt * 128 + chunk * 16, xend);
    dma16(xbase + (xofs[i] + k), lds + T::X_OFF + buf * T::x_bytes(live) + (i * T::NW + wave) * 1024);
  };
  auto load_w = [&](int mt, int buf, int i) {
    const uint32_t k = (uint32_t)min(mt * 128 + chunk * 16, wend);
    int m = 0;
    if constexpr (GATE) m = (i * T::NW + wave) * 8 % T::TN / OUT_TN;
    dma16((m ? wbase2 : wbase) + (wofs[i] + k), lds + T::W_OFF + buf * T::W_BYTES + (i * T::NW + wave) * 1024);
  };
  // scales of a thread's rows (the weights', then the rows')
  constexpr int SR = T::SR > 0 ? T::SR : 1;
  const uint8_t* ssrc[SR];
  uint4v skept[SR][2];
  if constexpr (T::WS) {
#pragma unroll
    for (int j = 0; j < T::SR; ++j) {
      const int r = min(t + j * T::NT, T::SROWS - 1);
      int m;
      const int col = column(min(r, T::BN - 1), m);
      ssrc[j] = T::XS && r >= T::BN ? xsbase + (uint32_t)input_row(r - T::BN) * (uint32_t)a.ldxs
                                    : (m ? sbase2 + (uint32_t)col * ld_s2 : sbase + (uint32_t)col * ld_s);
    }
  }
  auto fetch_scales = [&](int at) {  // 32 blocks from `at` on; zeros (2^-127) behind K
    const int left = nb - at;
    if (left <= 0) return;
#pragma unroll
    for (int j = 0; j < T::SR; ++j) {
      if (left >= 32) {
        __builtin_memcpy(&skept[j][0], ssrc[j] + at, 16);
        __builtin_memcpy(&skept[j][1], ssrc[j] + at + 16, 16);
      } else {
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          uint32_t w = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if (d * 4 + b < left) w |= (uint32_t)ssrc[j][at + d * 4 + b] << (8 * b);
          skept[j][d / 4][d % 4] = w;
        }
      }
    }
  };
  auto store_scales = [&](int mt) {
    const int q = mt & 3;
#pragma unroll
    for (int j = 0; j < T::SR; ++j) {
      const int r = t + j * T::NT;
      uint2v v;
#pragma unroll
      for (int e = 0; e < 2; ++e) v[e] = q == 0 ? skept[j][0][e] : (q == 1 ? skept[j][0][2 + e] : (q == 2 ? skept[j][1][e] : skept[j][1][2 + e]));
      if (r < T::SROWS) *reinterpret_cast<uint2v*>(lds + T::S_OFF + (mt & 1) * T::S_BYTES + r * 8) = v;
    }
  };
  // hands over the scales of 256-deep tile mt (before the barrier that its first fragments are read behind)
  auto pass_scales = [&](int mt) {
    if constexpr (T::WS) {
      if (mt < MT) store_scales(mt);
      if ((mt & 3) == 3) fetch_scales((mt + 1) * 8);
    }
  };
  constexpr int WL = T::WI;

  // ---- fragments
  const int sx = (l32 >> 1) & 7;
  const int xrow = (wm * 32 + l32) * 128, wrow = (wn * T::TN + l32) * 128;
  const char* const scales = lds + T::S_OFF;  // of a tile: [rows][8]
  const int s_row = (wn * T::TN + l32) * 8, xs_row = (T::BN + wm * 32 + l32) * 8;
  // Fragments: two sets of a step's, or (DEEP) of a k tile's four steps'.  kMul164 keeps codes and converts them for their MFMAs.
  constexpr int FS = T::DEEP ? 8 : 2;
  half8v xf[FS][T::MI], wf[MUL == kMul164 && T::DEEP ? 1 : FS][T::NI];
  uint32_t codes[MUL == kMul164 ? (T::DEEP ? FS : 1) : 1][T::NI];
  // scales of the fragments: kMul164 of the block that they are in, kMul44 of the k tile's four steps, for this one and the next
  uint32_t wsc[T::WS ? (MUL == kMul164 ? (T::DEEP ? FS / 2 : 1) : 2) : 1][T::NI], xsc[T::XS ? 2 : 1][T::MI];
  // fragment i of step kk of k tile kt in buffers (xb, wb), into set `buf`: the weights' first, then the rows'
  auto read_one = [&](int kt, int xb, int wb, int kk, int buf, int i, int live) __attribute__((always_inline)) {
    const int c = MUL == kMul44 ? g * 4 + kk : kk * 2 + g;  // chunk
    const int next = T::DEEP ? buf / 4 : 1;
    if (i < T::NI) {
      const char* const w = lds + T::W_OFF + wb * T::W_BYTES + wrow + i * 32 * 128;
      if constexpr (MUL == kMul164) {
        const int b = (kt & 3) * 2 + kk / 2;
        codes[T::DEEP ? buf : 0][i] = *reinterpret_cast<const uint32_t*>(w + ((b ^ sx) << 4) + (kk & 1) * 8 + g * 4);
        if ((kk & 1) == 0) wsc[T::DEEP ? buf / 2 : 0][i] = (uint32_t)(uint8_t)scales[((kt >> 2) & 1) * T::S_BYTES + s_row + i * 256 + b] << 23;
      } else {
        wf[buf][i] = *reinterpret_cast<const half8v*>(w + ((c ^ sx) << 4));
        if constexpr (MUL == kMul44)
          if (kk == 0) wsc[next][i] = *reinterpret_cast<const uint32_t*>(scales + (kt & 1) * T::S_BYTES + s_row + i * 256 + g * 4);
      }
    } else {
      const int mi = i - T::NI;
      xf[buf][mi] = *reinterpret_cast<const half8v*>(lds + T::X_OFF + xb * T::x_bytes(live) + xrow + mi * T::WM * 32 * 128 + ((c ^ sx) << 4));
      if constexpr (MUL == kMul44)
        if (kk == 0) xsc[next][mi] = *reinterpret_cast<const uint32_t*>(scales + (kt & 1) * T::S_BYTES + xs_row + mi * T::WM * 256 + g * 4);
    }
  };
  auto convert_one = [&](int buf, int i) __attribute__((always_inline)) {
    if constexpr (MUL == kMul164) {
      if constexpr (T::DEEP) wf[0][i] = fp4x8_to_half8(codes[buf][i], __uint_as_float(wsc[buf / 2][i]));
      else wf[buf][i] = fp4x8_to_half8(codes[0][i], __uint_as_float(wsc[0][i]));
    }
  };
  float16v acc[T::NI][T::MI];
#pragma unroll
  for (int ni = 0; ni < T::NI; ++ni)
#pragma unroll
    for (int mi = 0; mi < T::MI; ++mi)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[ni][mi][r] = 0.f;
  // MFMA i of step kk, on set `buf`; `live` row blocks
  auto mfma_one = [&](int buf, int kk, int i, int live) __attribute__((always_inline)) {
    const int ni = i / live, mq = i % live;
    const int mi = (ni & 1) ? live - 1 - mq : mq;  // serpentine: consecutive MFMAs share a source operand
    if constexpr (MUL == kMul44) {
      const uint4v w = __builtin_bit_cast(uint4v, wf[buf][ni]), x = __builtin_bit_cast(uint4v, xf[buf][mi]);
      const int8x w8 = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0}, x8 = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
      const int sw = (int)wsc[T::DEEP ? buf / 4 : 0][ni], sx_ = (int)xsc[T::DEEP ? buf / 4 : 0][mi];
#define TRI_MFMA44(k) acc[ni][mi] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w8, x8, acc[ni][mi], 4, 4, k, sw, k, sx_)
      if (kk == 0) TRI_MFMA44(0);
      else if (kk == 1) TRI_MFMA44(1);
      else if (kk == 2) TRI_MFMA44(2);
      else TRI_MFMA44(3);
#undef TRI_MFMA44
    } else {
      acc[ni][mi] = mfma32(wf[MUL == kMul164 && T::DEEP ? 0 : buf][ni], xf[buf][mi], acc[ni][mi]);
    }
  };
  auto turn_scales = [&]() __attribute__((always_inline)) {  // the next k tile's are this one's
    if constexpr (MUL == kMul44 && !T::DEEP) {
#pragma unroll
      for (int i = 0; i < T::NI; ++i) wsc[0][i] = wsc[1][i];
#pragma unroll
      for (int i = 0; i < T::MI; ++i) xsc[0][i] = xsc[1][i];
    }
  };
  auto none = [](int) {};

  // ---- prologue: the first tile, then the others (live: row blocks of a wave)
  auto prologue = [&](auto LIVEC) __attribute__((always_inline)) {
    constexpr int live = decltype(LIVEC)::value, xi = live * T::WM * 4 / T::NW, NA = T::na(live);
    if constexpr (T::WS) fetch_scales(0);
#pragma unroll
    for (int i = 0; i < WL; ++i) load_w(0, 0, i);
#pragma unroll
    for (int s = 0; s < NA; ++s) {
#pragma unroll
      for (int i = 0; i < xi; ++i) load_x(s, s, i, live);
      if (T::SUB == 1 && s + 1 < NA) {
#pragma unroll
        for (int i = 0; i < WL; ++i) load_w(s + 1, s + 1, i);
      }
    }
    constexpr int V0 = T::SUB == 4 ? (NA - 1) * xi + (T::NB - 1) * WL : (NA - 1) * (xi + WL);
    if constexpr (T::SUB == 4) {
#pragma unroll
      for (int s = 1; s < T::NB; ++s)
#pragma unroll
        for (int i = 0; i < WL; ++i) load_w(s, s, i);
    }
    pass_scales(0);
    __builtin_amdgcn_s_waitcnt(((V0 < 63 ? V0 : 63) & 15) | (((V0 < 63 ? V0 : 63) >> 4) << 14) | 0x0070);  // vmcnt, lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
  };
  int kt = 0, xb = 0, wb = 0;  // k tile and its buffers
  int xb1 = 0, wb1 = 0;        // the next one's
  bool wnext = false;          // whether its weights are another tile
  auto next_buffers = [&](int kt, int na) {
    xb1 = xb == na - 1 ? 0 : xb + 1;
    wnext = T::SUB == 1 || (kt & 3) == 3;
    wb1 = !wnext ? wb : (wb == T::NB - 1 ? 0 : wb + 1);
  };
  // this wave's reads of tile kt are in its registers and its share of tile kt + 1 has landed; everybody's, behind the barrier
  auto landed = [&](int kt, auto LIVEC) {
    constexpr int live = decltype(LIVEC)::value, xi = live * T::WM * 4 / T::NW, NA = T::na(live);
    if (wnext) pass_scales((T::SUB == 4 ? kt >> 2 : kt) + 1);
    constexpr int V = T::inflight(NA, xi), V2 = T::SUB == 4 ? V + WL : V;
    if (T::SUB == 4 && (kt & 3) <= NA - 2) {  // (weights requested after the rows of tile kt + 1 may be on their way, too)
      __builtin_amdgcn_s_waitcnt((V2 & 15) | ((V2 >> 4) << 14) | 0x0070);  // vmcnt, lgkmcnt(0)
    } else {
      __builtin_amdgcn_s_waitcnt((V & 15) | ((V >> 4) << 14) | 0x0070);
    }
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  const bool half = MUL != kMul44 && (k1 - k0) % 64 != 0;  // the last tile's second half lies behind K
  typedef std::integral_constant<int, T::MI> AllRows;
  if constexpr (T::DEEP) {
    constexpr int NM = T::NI * T::MI, NF = T::NI + T::MI;
    prologue(AllRows{});
    // Waves of few MFMAs per step read the fragments of all four steps of the next k tile while they multiply this one's: step by
    // step each waits for an LDS read, its conversion and two or four MFMAs in a row, with nothing beside them (32 x 256 tiles,
    // 4-bit weights: 2500 clocks a k tile of 32 MFMAs).
    constexpr int NS = 4 * NM, NR = 4 * NF;
    auto multiply = [&](int set, int i) __attribute__((always_inline)) {
      const int kk = i / NM, j = i % NM;
      if (MUL == kMul164 && j == 0) {
#pragma unroll
        for (int ni = 0; ni < T::NI; ++ni) convert_one(set + kk, ni);
      }
      mfma_one(set + kk, kk, j, T::MI);
    };
    auto tile = [&](auto SET) __attribute__((always_inline)) {
      constexpr int set = decltype(SET)::value;
      next_buffers(kt, T::NA);
      landed(kt, AllRows{});
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        multiply(set, i);
        constexpr int NL = T::XI + WL;
#pragma unroll
        for (int j = i * NL / NS; j < (i + 1) * NL / NS; ++j) {
          if (j < T::XI) load_x(kt + T::NA, xb, j, T::MI);
          else if (wnext) load_w((T::SUB == 4 ? kt >> 2 : kt) + T::NB, wb, j - T::XI);
        }
#pragma unroll
        for (int j = i * NR / NS; j < (i + 1) * NR / NS; ++j) read_one(kt + 1, xb1, wb1, j / NF, (4 - set) + j / NF, j % NF, T::MI);
        __builtin_amdgcn_sched_barrier(0);
      }
      xb = xb1;
      wb = wb1;
      ++kt;
    };
    auto last = [&](auto SET) __attribute__((always_inline)) {
      constexpr int set = decltype(SET)::value;
#pragma unroll
      for (int i = 0; i < NS; ++i)
        if (i < NS / 2 || !half) multiply(set, i);
    };
    typedef std::integral_constant<int, 0> Set0;
    typedef std::integral_constant<int, 4> Set1;
#pragma unroll
    for (int j = 0; j < NR; ++j) read_one(0, 0, 0, j / NF, j / NF, j % NF, T::MI);
    while (kt + 2 < KT) {
      tile(Set0{});
      tile(Set1{});
    }
    if (kt + 1 < KT) {
      tile(Set0{});
      last(Set1{});
    } else {
      last(Set0{});
    }
  } else {
    // LIVE: blocks of 32 rows that a wave has; the row blocks of a tile go to its waves in turn, so that a tile of fewer rows costs
    // less whole steps' MFMAs, loads and fragments - not time alone, the large products run at the power limit.
    auto run = [&](auto LIVEC) __attribute__((always_inline)) {
      constexpr int LIVE = decltype(LIVEC)::value, NM = T::NI * LIVE, NF = T::NI + LIVE, XL = LIVE * T::WM * 4 / T::NW, NA = T::na(LIVE);
      typedef std::integral_constant<int, LIVE> Rows;
      // step kk, slot by slot (a schedule fence after each): MFMA i, its share of `n` loads, and of the fragments of
      // step rkk of tile rkt into the other set (rkk < 0: none)
      auto step = [&](int kk, int n, auto load, int rkt, int rxb, int rwb, int rkk) __attribute__((always_inline)) {
        const int buf = kk & 1;
#pragma unroll
        for (int i = 0; i < NM; ++i) {
          mfma_one(buf, kk, i, LIVE);
#pragma unroll
          for (int j = i * n / NM; j < (i + 1) * n / NM; ++j) load(j);
          if (rkk >= 0) {
            // (reads in the first half of the step, so that none is waited for; conversions in the last slots)
            constexpr int RPS = (2 * NF + NM - 1) / NM;
#pragma unroll
            for (int j = i * RPS; j < (i + 1) * RPS && j < NF; ++j) read_one(rkt, rxb, rwb, rkk, buf ^ 1, j, LIVE);
            constexpr int C0 = NM * 5 / 8, CS = NM - C0;
            if (i >= C0) {
#pragma unroll
              for (int j = (i - C0) * T::NI / CS; j < (i - C0 + 1) * T::NI / CS; ++j) convert_one(buf ^ 1, j);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      prologue(Rows{});
#pragma unroll
      for (int i = 0; i < NF; ++i) read_one(0, 0, 0, 0, 0, i, LIVE);
#pragma unroll
      for (int i = 0; i < T::NI; ++i) convert_one(0, i);
      turn_scales();

      for (; kt < KT - 1; ++kt) {
        next_buffers(kt, NA);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (T::LATE) {
          const int wb2 = wb == 0 ? T::NB - 1 : wb - 1;  // tile kt - 1 has left it
          step(0, WL, [&](int j) { load_w(kt + 2, wb2, j); }, kt, xb, wb, 1);
        } else {
          step(0, 0, none, kt, xb, wb, 1);
        }
        step(1, 0, none, kt, xb, wb, 2);
        step(2, 0, none, kt, xb, wb, 3);
        landed(kt, Rows{});
        // rows of tile kt + NA, and weights where a tile of them is over
        step(3, T::LATE ? XL : XL + WL, [&](int j) {
          if (j < XL) load_x(kt + NA, xb, j, LIVE);
          else if (wnext) load_w((T::SUB == 4 ? kt >> 2 : kt) + T::NB, wb, j - XL);
        }, kt + 1, xb1, wb1, 0);
        xb = xb1;
        wb = wb1;
        turn_scales();
      }
      // the last tile, whole or half
      step(0, 0, none, kt, xb, wb, 1);
      if (!half) {
        step(1, 0, none, kt, xb, wb, 2);
        step(2, 0, none, kt, xb, wb, 3);
      }
      step(3, 0, none, kt, xb, wb, -1);
    };
    static_assert(T::MI == 2 || T::MI == 4, "row blocks of a wave");
    const int live = MUL == kMul44 ? T::MI : (rows + 32 * T::WM - 1) / (32 * T::WM);  // (kMul44: there is one such tile a column at most)
    if (MUL == kMul44 || live == T::MI) run(std::integral_constant<int, T::MI>{});
    else if (live == 1) run(std::integral_constant<int, 1>{});
    else if (live == 2) run(std::integral_constant<int, 2>{});
    else run(std::integral_constant<int, T::MI == 4 ? 3 : 1>{});
  }
  TRI_WAIT_VMCNT(0);
  __syncthreads();  // every wave is done with the tiles in LDS, and every load into them has landed

  // ---- epilogue: a lane owns one row and four consecutive columns per register quad; tiles are turned around in LDS (a
  // wave's own region) and leave as 16-byte pieces of rows.
  if constexpr (KIND == kGroupDown || KIND == kGroupParts) {
    constexpr int RS = T::TN + 4;  // floats per staged row
    static_assert(T::NW * 32 * RS * 4 <= T::LDS_BYTES, "the staged rows fit");
    float* const stg = reinterpret_cast<float*>(lds) + wave * 32 * RS;
#pragma unroll
    for (int mi = 0; mi < T::MI; ++mi) {
#pragma unroll
      for (int ni = 0; ni < T::NI; ++ni)
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
          const float4v v = {acc[ni][mi][rq * 4], acc[ni][mi][rq * 4 + 1], acc[ni][mi][rq * 4 + 2], acc[ni][mi][rq * 4 + 3]};
          *reinterpret_cast<float4v*>(stg + l32 * RS + ni * 32 + rq * 8 + g * 4) = v;
        }
      constexpr int LPR = T::TN / 4;  // 16-byte pieces per staged row
#pragma unroll 4
      for (int idx = lane; idx < 32 * LPR; idx += 64) {
        const int row = idx / LPR, ch = idx % LPR;
        const int r = (mi * T::WM + wm) * 32 + row, n = n0 + wn * T::TN + ch * 4;
        const float4v v = *reinterpret_cast<const float4v*>(stg + row * RS + ch * 4);
        if (r < rows && n < a.N) {
          const int64_t at = KIND == kGroupDown ? (int64_t)split * a.n + a.rows[place0 + r] : (int64_t)split * a.M + place0 + r;
          *reinterpret_cast<float4v*>(a.y + at * a.N + n) = v;
        }
      }
    }
  } else {
    constexpr int ONI = GATE ? T::NI / 2 : T::NI;
    constexpr int RS = OUT_TN + 8;  // halfs per staged row
    static_assert(T::NW * T::TM * RS * 2 <= T::LDS_BYTES, "the staged output tile fits");
    half_t* const stg = lds_h + wave * (T::TM * RS);
  #pragma unroll
    for (int mi = 0; mi < T::MI; ++mi)
  #pragma unroll
      for (int ni = 0; ni < ONI; ++ni)
  #pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
          half4v h;
  #pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = acc[ni][mi][rq * 4 + e];
            h[e] = (half_t)(GATE ? silu(v) * acc[(ni + ONI) % T::NI][mi][rq * 4 + e] : v);
          }
          *reinterpret_cast<half4v*>(stg + (mi * 32 + l32) * RS + ni * 32 + rq * 8 + g * 4) = h;
        }
    constexpr int LPR = OUT_TN / 8;
  #pragma unroll 4
    for (int idx = lane; idx < T::TM * LPR; idx += 64) {
      const int row = idx / LPR, ch = idx % LPR;
      const int r = (row / 32 * T::WM + wm) * 32 + row % 32, n = n0 + wn * OUT_TN + ch * 8;
      const half8v v = *reinterpret_cast<const half8v*>(stg + row * RS + ch * 8);
      if (r < rows && n < a.N) *reinterpret_cast<half8v*>(a.out + (int64_t)(place0 + r) * a.ldo + n) = v;
    }
  }
}

template <class T, GroupKind KIND>
int launch_tile_t(const GroupArgs& a, hipStream_t stream) {
  constexpr int OUT_BN = KIND == kGroupGate ? T::BN / 2 : T::BN;
  constexpr bool ALL = KIND == kGroupRows || KIND == kGroupParts;
  constexpr auto kern = group_tile_kernel<T, KIND>;
  if (set_max_lds<kern, T::LDS_BYTES>() != 0) return -1;
  // (experts: as many tiles as there can be)
  const int64_t tiles_m = ALL ? (a.M + T::BM - 1) / T::BM : (a.n + T::BM - 1) / T::BM + (a.E < a.n ? a.E : a.n);
  const int64_t tiles = tiles_m * ((a.N + OUT_BN - 1) / OUT_BN) * a.ksplit;
  hipLaunchKernelGGL(kern, dim3((unsigned)tiles), dim3(T::NT), T::LDS_BYTES, stream, a);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tri

#endif  // once per element type
