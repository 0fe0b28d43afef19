// Products of few rows over K-contiguous weights, 16-bit or in 4-bit blocks: of up to 16 rows, or of the few rows that each
// expert of a decode step has.  A workgroup owns 16 columns (of gate and of up: 16 each) over the whole of K; its four waves take
// the pieces of K - 128 bytes of a column: 64 values, or 256 in 4 bits - in turn, each through an LDS ring of its own, and add
// up through LDS at the end.
//
// What bounds them: streaming the weights once.  Weights go global -> LDS without passing through registers; the rows' fragments
// come straight from the cache, which they stay in.
//
// The experts' rows are found without a launch that sorts them: the workgroups of choice s look for its expert among all
// choices (at most 64: one load, one ballot) and work only if s is the first to have it.
#include "fp4.h"
#include "gemm_core.h"
#include "launch.h"

namespace tri {

constexpr int kGsCols = 16, kGsPieceBytes = 128;

// LDS piece [16 columns][128 bytes]: 16-byte chunk j (of 8) of column c at slot j ^ ((c >> 1) & 7) - the lanes of a fragment
// read (16 columns, one chunk) then fall on different banks.  A load instruction fetches 128 bytes of eight columns.
template <bool W4, GroupKind KIND, int NW, int NST>
__global__ __launch_bounds__(NW * 64) void group_strip_kernel(GroupArgs a) {
  extern __shared__ __attribute__((aligned(16))) half_t lds[];
  __shared__ int list[kStripChoices];
  constexpr int NM = KIND == kGroupGate ? 2 : 1;       // weight matrices
  constexpr int PK = kGsPieceBytes * (W4 ? 2 : 1) / (W4 ? 1 : 2);  // values of a piece
  constexpr int STEPS = PK / 32;
  constexpr int PIECE = NM * kGsCols * kGsPieceBytes;  // bytes
  constexpr int L = 2 * NM + STEPS + (W4 ? NM : 0);    // loads of a piece
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  // neighbouring columns on one XCD, every choice's on all of them
  const int per = (a.N + 8 * kGsCols - 1) / (8 * kGsCols);  // strips per XCD
  const int choice = (int)blockIdx.x / (8 * per), at8 = (int)blockIdx.x - choice * 8 * per;
  const int n0 = ((at8 & 7) * per + (at8 >> 3)) * kGsCols;
  if (n0 >= a.N) return;

  int rows = a.M, expert = 0;
  if constexpr (KIND == kGroupGate || KIND == kGroupDown) {
    const int mine = lane < a.n ? a.ids[lane] : -1;
    expert = __builtin_amdgcn_readlane(mine, choice);
    const uint64_t same = __ballot(mine == expert);
    if (expert < 0 || expert >= a.E || __builtin_ctzll(same) != choice) return;
    if (mine == expert) list[__popcll(same & ((1ull << lane) - 1))] = lane;
    rows = __popcll(same);
    __syncthreads();
  }
  const int np = (a.K + PK - 1) / PK;
  const int pieces = KIND == kGroupDownOne ? np * a.n : np;  // (of all choices of the token, one after the other)
  const int mine = (pieces - wave + NW - 1) / NW;  // pieces wave, wave + 4, ...

  char* const ring = reinterpret_cast<char*>(lds) + wave * NST * PIECE;
  int64_t wofs[NM][2], sofs[NM];
#pragma unroll
  for (int m = 0; m < NM; ++m) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int col = i * 8 + (lane >> 3);
      wofs[m][i] = (int64_t)min(n0 + col, a.N - 1) * a.w_ld[m] + ((lane & 7) ^ ((col >> 1) & 7)) * 16;
    }
    sofs[m] = (int64_t)min(n0 + c, a.N - 1) * a.ws_ld[m];
  }

  for (int r0 = 0; r0 < rows; r0 += kStripRows) {
    const int r = min(r0 + c, rows - 1);
    const int choice_r = (KIND == kGroupGate || KIND == kGroupDown) ? list[r] : r;
    const int xrow = KIND == kGroupGate ? choice_r / a.top_k : choice_r;
    const half_t* const xsrc = reinterpret_cast<const half_t*>(a.x + (KIND == kGroupDownOne ? 0 : xrow) * a.ldx) + g * 8;
    half8v xf[NST][STEPS];
    uint2v sc[NST][NM];
    struct At {
      int k, seg, skip;
    };
    // piece i of this wave: its first value (the last piece is moved back where K ends within it; its first `skip` steps were
    // those of the piece before), past the end the last one again (the waits count on every load)
    auto at = [&](int i) __attribute__((always_inline)) {
      const int q = wave + min(i, mine - 1) * NW;
      At p;
      p.seg = KIND == kGroupDownOne ? q / np : 0;
      const int k = (q - p.seg * np) * PK;
      p.k = min(k, a.K - PK);
      p.skip = (k - p.k) / 32;
      return p;
    };
    auto expert_of = [&](int seg) __attribute__((always_inline)) {
      if constexpr (KIND != kGroupDownOne) return expert;
      const int e = a.ids[seg];
      return e < 0 || e >= a.E ? 0 : e;
    };
    auto load = [&](int i, int st) __attribute__((always_inline)) {
      const At p = at(i);
      const int e = expert_of(p.seg);
#pragma unroll
      for (int m = 0; m < NM; ++m) {
        const uint8_t* const w = a.w[m] + e * a.w_se[m] + (W4 ? p.k / 2 : p.k * 2);
#pragma unroll
        for (int j = 0; j < 2; ++j)
          load_to_lds16<true>(reinterpret_cast<const half_t*>(w + wofs[m][j]), reinterpret_cast<half_t*>(ring + st * PIECE + m * (kGsCols * kGsPieceBytes) + j * 1024));
        if constexpr (W4) __builtin_memcpy(&sc[st][m], a.ws[m] + e * a.ws_se[m] + sofs[m] + p.k / 32, 8);
      }
      const half_t* const x = xsrc + p.k + (KIND == kGroupDownOne ? p.seg * (a.ldx / 2) : 0);
#pragma unroll
      for (int j = 0; j < STEPS; ++j) xf[st][j] = *reinterpret_cast<const half8v*>(x + j * 32);
    };
    // the weights' fragment of step j
    auto frag = [&](int st, int m, int j) __attribute__((always_inline)) {
      const char* const p = ring + st * PIECE + m * (kGsCols * kGsPieceBytes) + c * kGsPieceBytes;
      if constexpr (W4) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(p + ((j ^ ((c >> 1) & 7)) << 4) + g * 4);
        return fp4x8_to_half8(w, fp4_scale((sc[st][m][j / 4] >> (j % 4 * 8)) & 255));
      } else {
        return *reinterpret_cast<const half8v*>(p + (((j * 4 + g) ^ ((c >> 1) & 7)) << 4));
      }
    };
    float4v acc[NM], sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int m = 0; m < NM; ++m) acc[m] = float4v{0.f, 0.f, 0.f, 0.f};
    // (DownOne) the piece's share of the token's sum
    auto weigh = [&](int i) __attribute__((always_inline)) {
      if constexpr (KIND == kGroupDownOne) {
        const int seg = at(i).seg, e = a.ids[seg];
        if (e >= 0 && e < a.E) {
          const float w = a.weights[seg];
#pragma unroll
          for (int q = 0; q < 4; ++q) sum[q] = fmaf(w, acc[0][q], sum[q]);
        }
        acc[0] = float4v{0.f, 0.f, 0.f, 0.f};
      }
    };
    auto multiply = [&](int st, int skip) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        if (j < skip) continue;
#pragma unroll
        for (int m = 0; m < NM; ++m) acc[m] = mfma16(frag(st, m, j), xf[st][j], acc[m]);
      }
    };
    if (mine > 0) {
#pragma unroll
      for (int s = 0; s < NST - 1; ++s) load(s, s);
      int i0 = 0;
      for (; i0 + NST < mine; i0 += NST) {
#pragma unroll
        for (int st = 0; st < NST; ++st) {
          load(i0 + st + NST - 1, (st + NST - 1) % NST);
          TRI_WAIT_VMCNT((NST - 1) * L);
          __builtin_amdgcn_sched_barrier(0);
          const int skip = KIND == kGroupDownOne ? at(i0 + st).skip : 0;
          if (KIND == kGroupDownOne && skip != 0) multiply(st, skip);
          else multiply(st, 0);
          weigh(i0 + st);
          __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the stage is loaded again next
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      // the last one to NST pieces
      load(i0 + NST - 1, NST - 1);
      TRI_WAIT_VMCNT(0);
#pragma unroll
      for (int st = 0; st < NST; ++st) {
        if (i0 + st < mine) {
          multiply(st, at(i0 + st).skip);
          weigh(i0 + st);
        }
      }
    }
    if constexpr (KIND == kGroupDownOne) acc[0] = sum;
    TRI_WAIT_VMCNT(0);
    __syncthreads();
    float4v* part = reinterpret_cast<float4v*>(lds);
    if (wave > 0) {
#pragma unroll
      for (int m = 0; m < NM; ++m) part[((wave - 1) * NM + m) * 64 + lane] = acc[m];
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int w = 0; w < NW - 1; ++w)
#pragma unroll
        for (int m = 0; m < NM; ++m) acc[m] += part[(w * NM + m) * 64 + lane];
      // lane: row c, columns n0 + 4 g .. + 3
      const int n = n0 + g * 4;
      if (r0 + c < rows && n < a.N) {
        if constexpr (KIND == kGroupDown) {
          *reinterpret_cast<float4v*>(a.y + (int64_t)choice_r * a.N + n) = acc[0];
        } else {
          half4v h;
#pragma unroll
          for (int e = 0; e < 4; ++e) h[e] = (half_t)(NM == 2 ? silu(acc[0][e]) * acc[NM - 1][e] : acc[0][e]);
          *reinterpret_cast<half4v*>(a.out + (int64_t)choice_r * a.ldo + n) = h;
        }
      }
    }
    __syncthreads();  // (the ring is loaded again for the next rows)
  }
}

#ifndef STRIPN
#define STRIPN kStripChoices
#endif
bool group_strip_takes(const GroupArgs& a, GroupKind kind) {
  if (a.xs != nullptr || a.K < (a.ws[0] != nullptr ? 256 : 64) || a.K % 32 != 0) return false;
  return kind == kGroupRows ? a.M <= kStripRows : a.n <= STRIPN;
}

template <bool W4, GroupKind KIND>
static int launch_strip_kind(const GroupArgs& a, hipStream_t stream) {
#ifndef SNW
#define SNW 4
#define SNST 3
#define SNW1 8
#define SNST1 4
#endif
  constexpr bool ONE = KIND == kGroupDownOne || KIND == kGroupRows;
  constexpr int NW = ONE ? SNW1 : SNW, NST = ONE ? SNST1 : SNST, NM = KIND == kGroupGate ? 2 : 1;
  constexpr int LDS = NW * NST * NM * kGsCols * kGsPieceBytes;
  constexpr auto kern = group_strip_kernel<W4, KIND, NW, NST>;
  if (set_max_lds<kern, LDS>() != 0) return -1;
  const int groups = KIND == kGroupGate || KIND == kGroupDown ? a.n : 1;
  hipLaunchKernelGGL(kern, dim3((a.N + 8 * kGsCols - 1) / (8 * kGsCols) * 8 * groups), dim3(NW * 64), LDS, stream, a);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
template <bool W4>
static int launch_strip_w(const GroupArgs& a, GroupKind kind, hipStream_t stream) {
  switch (kind) {
    case kGroupRows: return launch_strip_kind<W4, kGroupRows>(a, stream);
    case kGroupGate: return launch_strip_kind<W4, kGroupGate>(a, stream);
    case kGroupDown: return launch_strip_kind<W4, kGroupDown>(a, stream);
    default: return launch_strip_kind<W4, kGroupDownOne>(a, stream);
  }
}
int launch_group_strip(const GroupArgs& a, GroupKind kind, hipStream_t stream) {
  return a.ws[0] != nullptr ? launch_strip_w<true>(a, kind, stream) : launch_strip_w<false>(a, kind, stream);
}

}  // namespace tri
