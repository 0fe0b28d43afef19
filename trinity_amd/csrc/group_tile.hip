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
// Scales (a byte per block, rows of any alignment) come the same way: the one or two aligned 16-byte pieces of memory that hold
// a row's eight bytes of a 256-deep tile.  Every such piece holds a byte that is wanted, so none lies outside the tensor's pages.
//
// One barrier per k tile, in front of the last of its four steps, when the next tile must have landed; that step then requests
// the tile that takes its place.
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
  static constexpr int TM = BM / WM, TN = BN / WN, MI = TM / 32, NI = TN / 32;
  static constexpr int XI = BM / 32, WI = BN / 32;  // 1 KB load instructions per wave and tile
  static constexpr bool XS = MUL == kMul44, WS = MUL != kMul16;
  // scales: two 16-byte pieces a row; load instructions per wave (a wave without any repeats another's)
  static constexpr int SROWS = (WS ? BN : 0) + (XS ? BM : 0), SI = (SROWS * 2 + 255) / 256;
  static constexpr int SUB = MUL == kMul164 ? 4 : 1;  // k tiles of rows per tile of weights
  static constexpr int KX = MUL == kMul44 ? 256 : 64, KW = MUL == kMul16 ? 64 : 256;
  static constexpr int X_BYTES = BM * 128, W_BYTES = BN * 128, S_BYTES = SI * 4096;
  static constexpr int X_OFF = 0, W_OFF = NA * X_BYTES, S_OFF = W_OFF + NB * W_BYTES;
  static constexpr int LDS_BYTES = S_OFF + NB * S_BYTES;
  static constexpr bool LATE = NB > NA && SUB == 1;  // weights are requested in the first step of a tile
  static_assert(WM * WN == 4 && BM % 32 == 0 && BN % 32 == 0 && TM % 32 == 0 && TN % 32 == 0, "four waves");
  static_assert(NA >= 2 && NB >= 2 && LDS_BYTES <= 160 * 1024, "LDS budget");
  static_assert(NA == NB || LATE || SUB == 4, "waits below");
  static_assert(!LATE || (NA == 2 && NB == 3), "waits below");
  static_assert(SUB == 1 || NA <= 4, "waits below");
  // loads that may be on their way at the barrier of a tile
  static constexpr int INFLIGHT = SUB == 4 ? (NA - 2) * XI : (LATE ? WI + SI : (NA - 2) * (XI + WI + SI));
  static_assert(INFLIGHT + WI + SI < 64, "vmcnt");
};

__device__ __forceinline__ void dma16(const void* g, void* l) {
  load_to_lds16(static_cast<const half_t*>(g), static_cast<half_t*>(l));
}

template <class T, GroupKind KIND>
__global__ __launch_bounds__(256) void group_tile_kernel(GroupArgs a) {
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
  const uint8_t* wbase[2];
  const uint8_t* sbase[2];
#pragma unroll
  for (int m = 0; m < (GATE ? 2 : 1); ++m) {
    wbase[m] = a.w[m] + expert * a.w_se[m] + w0;
    sbase[m] = T::WS ? a.ws[m] + expert * a.ws_se[m] + k0 / 32 : nullptr;
  }
  if constexpr (!GATE) {
    wbase[1] = wbase[0];
    sbase[1] = sbase[0];
  }
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
  uint32_t xofs[T::XI], wofs[T::WI], sofs[T::SI > 0 ? T::SI : 1];
#pragma unroll
  for (int i = 0; i < T::XI; ++i) xofs[i] = (uint32_t)input_row((i * 4 + wave) * 8 + (lane >> 3)) * (uint32_t)a.ldx;
#pragma unroll
  for (int i = 0; i < T::WI; ++i) {
    int m;
    const int col = column((i * 4 + wave) * 8 + (lane >> 3), m);
    wofs[i] = (uint32_t)col * (uint32_t)a.w_ld[GATE ? m : 0];
  }
  // scales: a row's first byte, from its base rounded down to 16
  auto scale_base = [&](int r, int& m) -> const uint8_t* {
    m = 0;
    if (T::XS && r >= T::BN) return xsbase;
    if constexpr (GATE) m = r % T::TN / OUT_TN;
    return sbase[m];
  };
  auto scale_ofs = [&](int r) -> uint32_t {
    int m;
    const uint32_t low = (uint32_t)((uintptr_t)scale_base(r, m) & 15);
    if (T::XS && r >= T::BN) return low + (uint32_t)input_row(r - T::BN) * (uint32_t)a.ldxs;
    const int col = column(r, m);
    return low + (uint32_t)col * (uint32_t)a.ws_ld[m];
  };
  auto scale_row = [&](int i) { return min(((i * 4 + wave) * 64 + lane) >> 1, T::SROWS - 1); };
  if constexpr (T::WS) {
#pragma unroll
    for (int i = 0; i < T::SI; ++i) sofs[i] = scale_ofs(scale_row(i));
  }
  const int nb = (k1 - k0) / 32;  // blocks of this part
  const int xend = (MUL == kMul44 ? (k1 - k0) / 2 : (k1 - k0) * 2) - 16, wend = (MUL == kMul16 ? (k1 - k0) * 2 : (k1 - k0) / 2) - 16;
  // (past the end the loop keeps its load count, which the waits assume)
  auto load_x = [&](int kt, int buf, int i) {
    const uint32_t k = (uint32_t)min(kt * 128 + chunk * 16, xend);
    dma16(xbase + (xofs[i] + k), lds + T::X_OFF + buf * T::X_BYTES + (i * 4 + wave) * 1024);
  };
  auto load_w = [&](int mt, int buf, int i) {
    if (i < T::WI) {
      const uint32_t k = (uint32_t)min(mt * 128 + chunk * 16, wend);
      int m = 0;
      if constexpr (GATE) m = (i * 4 + wave) * 8 % T::TN / OUT_TN;
      dma16((m ? wbase[1] : wbase[0]) + (wofs[i] + k), lds + T::W_OFF + buf * T::W_BYTES + (i * 4 + wave) * 1024);
    } else if constexpr (T::SI > 0) {
      const int j = i - T::WI, k = min(mt, MT - 1) * 8;
      int m;
      const uint8_t* const base = reinterpret_cast<const uint8_t*>((uintptr_t)scale_base(min((j * 4 + wave) * 32, T::SROWS - 1), m) & ~(uintptr_t)15);
      const uint32_t first = sofs[j] + (uint32_t)k, o = (lane & 1) ? first + (uint32_t)min(8, nb - k) - 1 : first;
      dma16(base + (o & ~15u), lds + T::S_OFF + buf * T::S_BYTES + (j * 4 + wave) * 1024);
    }
  };
  constexpr int WL = T::WI + T::SI;

  // ---- fragments
  const int sx = (l32 >> 1) & 7;
  const int xrow = (wm * T::TM + l32) * 128, wrow = (wn * T::TN + l32) * 128;
  // where in its two pieces a row's scales begin
  int s_at[T::WS ? T::NI : 1], xs_at[T::XS ? T::MI : 1];
  if constexpr (T::WS) {
#pragma unroll
    for (int ni = 0; ni < T::NI; ++ni) {
      const int r = wn * T::TN + ni * 32 + l32;
      s_at[ni] = (int)(scale_ofs(r) & 15) + r * 32;
    }
  }
  if constexpr (T::XS) {
#pragma unroll
    for (int mi = 0; mi < T::MI; ++mi) {
      const int r = T::BN + wm * T::TM + mi * 32 + l32;
      xs_at[mi] = (int)(scale_ofs(r) & 15) + r * 32;
    }
  }
  // the scale of block b (0 to 7) of 256-deep tile mt; 2^-127 behind K
  auto read_scale = [&](int mt, int buf, int at, int b) -> uint32_t {
    const int o = (at & ~15) + ((at + mt * 8) & 15) + b;
    const uint32_t s = *reinterpret_cast<const uint8_t*>(lds + T::S_OFF + buf * T::S_BYTES + o);
    return mt * 8 + b < nb ? s : 0u;
  };
  half8v xf[2][T::MI], wf[2][T::NI];
  uint32_t codes[MUL == kMul164 ? T::NI : 1];  // eight values on their way from LDS to a fragment
  uint32_t wsc[2][T::WS ? T::NI : 1], xsc[2][T::XS ? T::MI : 1];
  // fragment i of step kk of k tile kt in buffers (xb, wb), into set `buf`: the weights' first, then the rows'
  auto read_one = [&](int kt, int xb, int wb, int kk, int buf, int i) {
    if (i < T::NI) {
      const char* const w = lds + T::W_OFF + wb * T::W_BYTES + wrow + i * 32 * 128;
      if constexpr (MUL == kMul164) {
        const int b = (kt & 3) * 2 + kk / 2;
        codes[i] = *reinterpret_cast<const uint32_t*>(w + ((b ^ sx) << 4) + (kk & 1) * 8 + g * 4);
        if ((kk & 1) == 0) wsc[0][i] = read_scale(kt >> 2, wb, s_at[i], b) << 23;
      } else {
        wf[buf][i] = *reinterpret_cast<const half8v*>(w + (((kk * 2 + g) ^ sx) << 4));
        if constexpr (MUL == kMul44) wsc[buf][i] = read_scale(kt, wb, s_at[i], kk * 2 + g);
      }
    } else {
      const int mi = i - T::NI;
      xf[buf][mi] = *reinterpret_cast<const half8v*>(lds + T::X_OFF + xb * T::X_BYTES + xrow + mi * 32 * 128 + (((kk * 2 + g) ^ sx) << 4));
      if constexpr (MUL == kMul44) xsc[buf][mi] = read_scale(kt, wb, xs_at[mi], kk * 2 + g);
    }
  };
  auto convert_one = [&](int buf, int i) {
    if constexpr (MUL == kMul164) wf[buf][i] = fp4x8_to_half8(codes[i], __uint_as_float(wsc[0][i]));
  };
  float16v acc[T::NI][T::MI];
#pragma unroll
  for (int ni = 0; ni < T::NI; ++ni)
#pragma unroll
    for (int mi = 0; mi < T::MI; ++mi)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[ni][mi][r] = 0.f;
  auto mfma_one = [&](int buf, int i) {
    const int ni = i / T::MI, mq = i % T::MI;
    const int mi = (ni & 1) ? T::MI - 1 - mq : mq;  // serpentine: consecutive MFMAs share a source operand
    if constexpr (MUL == kMul44) {
      const uint4v w = __builtin_bit_cast(uint4v, wf[buf][ni]), x = __builtin_bit_cast(uint4v, xf[buf][mi]);
      const int8x w8 = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0}, x8 = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
      acc[ni][mi] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w8, x8, acc[ni][mi], 4, 4, 0, (int)wsc[buf][ni], 0, (int)xsc[buf][mi]);
    } else {
      acc[ni][mi] = mfma32(wf[buf][ni], xf[buf][mi], acc[ni][mi]);
    }
  };
  constexpr int NM = T::NI * T::MI, NF = T::NI + T::MI;
  // one step, slot by slot (a schedule fence after each): MFMA i on set `buf`, its share of `n` loads, and of the fragments of
  // step rkk of tile rkt into the other set (rkk < 0: none)
  auto step = [&](int buf, int n, auto load, int rkt, int rxb, int rwb, int rkk) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      mfma_one(buf, i);
#pragma unroll
      for (int j = i * n / NM; j < (i + 1) * n / NM; ++j) load(j);
      if (rkk >= 0) {
        if (NM >= 2 * NF) {
          if (i < NF) read_one(rkt, rxb, rwb, rkk, buf ^ 1, i);
          if (i >= NM - T::NI) convert_one(buf ^ 1, i - (NM - T::NI));
        } else {
#pragma unroll
          for (int j = i * NF / NM; j < (i + 1) * NF / NM; ++j) read_one(rkt, rxb, rwb, rkk, buf ^ 1, j);
          if (i == NM - 1) {
#pragma unroll
            for (int j = 0; j < T::NI; ++j) convert_one(buf ^ 1, j);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto none = [](int) {};

  // ---- prologue: the first tile, then the others
#pragma unroll
  for (int i = 0; i < WL; ++i) load_w(0, 0, i);
#pragma unroll
  for (int s = 0; s < T::NA; ++s) {
#pragma unroll
    for (int i = 0; i < T::XI; ++i) load_x(s, s, i);
    if (T::SUB == 1 && s + 1 < T::NA) {
#pragma unroll
      for (int i = 0; i < WL; ++i) load_w(s + 1, s + 1, i);
    }
  }
  constexpr int V0 = T::SUB == 4 ? (T::NA - 1) * T::XI + (T::NB - 1) * WL : (T::NA - 1) * (T::XI + WL);
  if constexpr (T::SUB == 4) {
#pragma unroll
    for (int s = 1; s < T::NB; ++s)
#pragma unroll
      for (int i = 0; i < WL; ++i) load_w(s, s, i);
  }
  TRI_WAIT_VMCNT(V0 < 63 ? V0 : 63);
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int i = 0; i < NF; ++i) read_one(0, 0, 0, 0, 0, i);
#pragma unroll
  for (int i = 0; i < T::NI; ++i) convert_one(0, i);

  int xb = 0, wb = 0;  // buffers of tile kt
  int kt = 0;
  for (; kt < KT - 1; ++kt) {
    const int xb1 = xb == T::NA - 1 ? 0 : xb + 1;
    const bool wnext = T::SUB == 1 || (kt & 3) == 3;
    const int wb1 = !wnext ? wb : (wb == T::NB - 1 ? 0 : wb + 1);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (T::LATE) {
      const int wb2 = wb == 0 ? T::NB - 1 : wb - 1;  // tile kt - 1 has left it
      step(0, WL, [&](int j) { load_w(kt + 2, wb2, j); }, kt, xb, wb, 1);
    } else {
      step(0, 0, none, kt, xb, wb, 1);
    }
    step(1, 0, none, kt, xb, wb, 2);
    step(0, 0, none, kt, xb, wb, 3);
    // this wave's reads of tile kt are in its registers and its share of tile kt + 1 has landed
    constexpr int V = T::INFLIGHT, V2 = T::SUB == 4 ? V + WL : V;
    if (T::SUB == 4 && (kt & 3) <= T::NA - 2) {  // (weights requested after the rows of tile kt + 1 may be on their way, too)
      __builtin_amdgcn_s_waitcnt((V2 & 15) | ((V2 >> 4) << 14) | 0x0070);  // vmcnt, lgkmcnt(0)
    } else {
      __builtin_amdgcn_s_waitcnt((V & 15) | ((V >> 4) << 14) | 0x0070);
    }
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    // rows of tile kt + NA, and weights where a tile of them is over
    step(1, T::LATE ? T::XI : T::XI + WL, [&](int j) {
      if (j < T::XI) load_x(kt + T::NA, xb, j);
      else if (wnext) load_w((T::SUB == 4 ? kt >> 2 : kt) + T::NB, wb, j - T::XI);
    }, kt + 1, xb1, wb1, 0);
    xb = xb1;
    wb = wb1;
  }
  // the last tile, whole or half
  step(0, 0, none, kt, xb, wb, 1);
  if (MUL == kMul44 || (k1 - k0) % 64 == 0) {
    step(1, 0, none, kt, xb, wb, 2);
    step(0, 0, none, kt, xb, wb, 3);
  }
  step(1, 0, none, kt, xb, wb, -1);
  TRI_WAIT_VMCNT(0);
  __syncthreads();  // every wave is done with the tiles in LDS, and every load into them has landed

  // ---- epilogue: a lane owns one row and four consecutive columns per register quad; tiles are turned around in LDS (a
  // wave's own region) and leave as 16-byte pieces of rows.
  if constexpr (KIND == kGroupDown || KIND == kGroupParts) {
    constexpr int RS = T::TN + 4;  // floats per staged row
    static_assert(4 * 32 * RS * 4 <= T::LDS_BYTES, "the staged rows fit");
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
        const int r = wm * T::TM + mi * 32 + row, n = n0 + wn * T::TN + ch * 4;
        const float4v v = *reinterpret_cast<const float4v*>(stg + row * RS + ch * 4);
        if (r < rows && n < a.N) {
          const int64_t at = KIND == kGroupDown ? (int64_t)a.rows[place0 + r] : (int64_t)split * a.M + place0 + r;
          *reinterpret_cast<float4v*>(a.y + at * a.N + n) = v;
        }
      }
    }
  } else {
    constexpr int ONI = GATE ? T::NI / 2 : T::NI;
    constexpr int RS = OUT_TN + 8;  // halfs per staged row
    static_assert(4 * T::TM * RS * 2 <= T::LDS_BYTES, "the staged output tile fits");
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
      const int r = wm * T::TM + row, n = n0 + wn * OUT_TN + ch * 8;
      const half8v v = *reinterpret_cast<const half8v*>(stg + row * RS + ch * 8);
      if (r < rows && n < a.N) *reinterpret_cast<half8v*>(a.out + (int64_t)(place0 + r) * a.ldo + n) = v;
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
int group_tile_rows(int choices, int experts) {
  const int mean = (choices + experts - 1) / experts;
  return mean <= 24 ? 32 : (mean <= 64 ? 64 : (mean <= 256 ? 128 : 256));
}

GroupPlan group_rows_plan(int M, int K, int N, bool x4) {
  GroupPlan p;
  p.bm = M <= 32 ? 32 : (M <= 64 ? 64 : (M <= 256 ? 128 : 256));
  const int bn = p.bm == 32 || p.bm == 256 ? 256 : 128;
  const int tiles = ((M + p.bm - 1) / p.bm) * ((N + bn - 1) / bn), deep = (K + 255) / 256;
  int parts = tiles >= 256 ? 1 : 256 / tiles;
  if (parts > deep / 2) parts = deep / 2 > 0 ? deep / 2 : 1;
  const int per = (deep + parts - 1) / parts;
  p.ksplit = (deep + per - 1) / per;  // (no part is empty)
  return p;
}

int64_t fp4_matmul_workspace(int M, int K, int N, bool x4) {
  GroupArgs a{};
  a.M = M;
  a.K = K;
  const uint8_t any = 0;
  a.ws[0] = &any;
  a.xs = x4 ? &any : nullptr;
  if (group_strip_takes(a, kGroupRows)) return 0;
  const GroupPlan p = group_rows_plan(M, K, N, x4);
  return p.ksplit > 1 ? (int64_t)p.ksplit * M * N * 4 : 0;
}

template <class T, GroupKind KIND>
static int launch_tile_t(const GroupArgs& a, hipStream_t stream) {
  constexpr int OUT_BN = KIND == kGroupGate ? T::BN / 2 : T::BN;
  constexpr bool ALL = KIND == kGroupRows || KIND == kGroupParts;
  constexpr auto kern = group_tile_kernel<T, KIND>;
  if (set_max_lds<kern, T::LDS_BYTES>() != 0) return -1;
  // (experts: as many tiles as there can be)
  const int64_t tiles_m = ALL ? (a.M + T::BM - 1) / T::BM : (a.n + T::BM - 1) / T::BM + (a.E < a.n ? a.E : a.n);
  const int64_t tiles = tiles_m * ((a.N + OUT_BN - 1) / OUT_BN) * a.ksplit;
  hipLaunchKernelGGL(kern, dim3((unsigned)tiles), dim3(256), T::LDS_BYTES, stream, a);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <GroupMul MUL, GroupKind KIND>
static int launch_tile_kind(const GroupArgs& a, int bm, hipStream_t stream) {
  constexpr int D = MUL == kMul164 ? 2 : 3;
  switch (bm) {
    case 32: return launch_tile_t<GroupTile<32, 256, 1, 4, 3, D, MUL>, KIND>(a, stream);
    case 64: return launch_tile_t<GroupTile<64, 128, 2, 2, 3, D, MUL>, KIND>(a, stream);
    case 128: return launch_tile_t<GroupTile<128, 128, 2, 2, 3, D, MUL>, KIND>(a, stream);
    default: return launch_tile_t<GroupTile<256, 256, 2, 2, 2, MUL == kMul16 ? 3 : 2, MUL>, KIND>(a, stream);
  }
}

int launch_group_tile(const GroupArgs& a, GroupKind kind, int bm, hipStream_t stream) {
  const bool w4 = a.ws[0] != nullptr;
  switch (kind) {
    case kGroupRows: return a.xs != nullptr ? launch_tile_kind<kMul44, kGroupRows>(a, bm, stream) : launch_tile_kind<kMul164, kGroupRows>(a, bm, stream);
    case kGroupParts: return a.xs != nullptr ? launch_tile_kind<kMul44, kGroupParts>(a, bm, stream) : launch_tile_kind<kMul164, kGroupParts>(a, bm, stream);
    case kGroupGate: return w4 ? launch_tile_kind<kMul164, kGroupGate>(a, bm, stream) : launch_tile_kind<kMul16, kGroupGate>(a, bm, stream);
    default: return w4 ? launch_tile_kind<kMul164, kGroupDown>(a, bm, stream) : launch_tile_kind<kMul16, kGroupDown>(a, bm, stream);
  }
}

}  // namespace tri
