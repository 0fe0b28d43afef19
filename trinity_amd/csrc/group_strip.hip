// Products of the few rows that each expert of a decode step has over K-contiguous 16-bit weights.  A workgroup owns 16 columns (of gate
// and of up: 16 each) over the whole of K; its four waves take the pieces of K - 128 bytes of a column, 64 values - in turn, each
// through an LDS ring of its own, and add up through LDS at the end.
//
// What bounds them: streaming the weights once.  Weights go global -> LDS without passing through registers; the rows' fragments
// come straight from the cache, which they stay in.  One token through two experts of [4096, 14336]: 470 MB of gate and up in 69
// to 72 us, 235 MB of down in 37, 6.4 to 6.8 TB/s.
//
// The experts' rows are found without a launch that sorts them: the workgroups of choice s look for its expert among all
// choices (at most 64: one load, one ballot) and work only if s is the first to have it.
#include "gemm_core.h"
#include "launch.h"

namespace tri {

constexpr int kGsCols = 16, kGsPieceBytes = 128;

// LDS piece [16 columns][128 bytes]: 16-byte chunk j (of 8) of column c at slot j ^ ((c >> 1) & 7) - the lanes of a fragment
// read (16 columns, one chunk) then fall on different banks.  A load instruction fetches 128 bytes of eight columns.
template <GroupKind KIND, int NW, int NST>
__global__ __launch_bounds__(NW * 64) void group_strip_kernel(GroupArgs a) {
  extern __shared__ __attribute__((aligned(16))) half_t lds[];
  __shared__ int list[kStripChoices];
  constexpr int NM = KIND == kGroupGate ? 2 : 1;       // weight matrices
  constexpr int PK = kGsPieceBytes / 2;                // values of a piece
  constexpr int STEPS = PK / 32;
  constexpr int PIECE = NM * kGsCols * kGsPieceBytes;  // bytes
  constexpr int L = 2 * NM + STEPS;                    // loads of a piece
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  // neighbouring columns on one XCD, every choice's on all of them
  const int per = (a.N + 8 * kGsCols - 1) / (8 * kGsCols);  // strips per XCD
  const int choice = (int)blockIdx.x / (8 * per), at8 = (int)blockIdx.x - choice * 8 * per;
  const int n0 = ((at8 & 7) * per + (at8 >> 3)) * kGsCols;
  if (n0 >= a.N) return;

  const int own = lane < a.n ? a.ids[lane] : -1;
  const int expert = __builtin_amdgcn_readlane(own, choice);
  const uint64_t same = __ballot(own == expert);
  if (expert < 0 || expert >= a.E || __builtin_ctzll(same) != choice) return;
  if (own == expert) list[__popcll(same & ((1ull << lane) - 1))] = lane;  // (every wave the same values)
  const int rows = __popcll(same);
  __syncthreads();
  const int np = (a.K + PK - 1) / PK;
  const int mine = (np - wave + NW - 1) / NW;  // pieces wave, wave + NW, ...

  char* const ring = reinterpret_cast<char*>(lds) + wave * NST * PIECE;
  int64_t wofs[NM][2];
#pragma unroll
  for (int m = 0; m < NM; ++m) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int col = i * 8 + (lane >> 3);
      wofs[m][i] = (int64_t)min(n0 + col, a.N - 1) * a.w_ld[m] + ((lane & 7) ^ ((col >> 1) & 7)) * 16;
    }
  }

  for (int r0 = 0; r0 < rows; r0 += kStripRows) {
    const int choice_r = list[min(r0 + c, rows - 1)];
    const half_t* const xsrc = reinterpret_cast<const half_t*>(a.x + (KIND == kGroupGate ? choice_r / a.top_k : choice_r) * a.ldx) + g * 8;
    half8v xf[NST][STEPS];
    // first value of piece i of this wave (the last piece is moved back where K ends within it), past the end the last one again
    // (the waits count on every load)
    auto at = [&](int i) __attribute__((always_inline)) { return min((wave + min(i, mine - 1) * NW) * PK, a.K - PK); };
    auto load = [&](int i, int st) __attribute__((always_inline)) {
      const int k = at(i);
#pragma unroll
      for (int m = 0; m < NM; ++m) {
        const uint8_t* const w = a.w[m] + expert * a.w_se[m] + k * 2;
#pragma unroll
        for (int j = 0; j < 2; ++j)
          load_to_lds16<true>(reinterpret_cast<const half_t*>(w + wofs[m][j]), reinterpret_cast<half_t*>(ring + st * PIECE + m * (kGsCols * kGsPieceBytes) + j * 1024));
      }
#pragma unroll
      for (int j = 0; j < STEPS; ++j) xf[st][j] = *reinterpret_cast<const half8v*>(xsrc + k + j * 32);
    };
    // the weights' fragment of step j
    auto frag = [&](int st, int m, int j) __attribute__((always_inline)) {
      const char* const p = ring + st * PIECE + m * (kGsCols * kGsPieceBytes) + c * kGsPieceBytes;
      return *reinterpret_cast<const half8v*>(p + (((j * 4 + g) ^ ((c >> 1) & 7)) << 4));
    };
    float4v acc[NM];
#pragma unroll
    for (int m = 0; m < NM; ++m) acc[m] = float4v{0.f, 0.f, 0.f, 0.f};
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
          multiply(st, 0);
          __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the stage is loaded again next
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      // the last one to NST pieces; the very last may begin with a step that the piece before it has done already
      load(i0 + NST - 1, NST - 1);
      TRI_WAIT_VMCNT(0);
#pragma unroll
      for (int st = 0; st < NST; ++st) {
        if (i0 + st < mine) {
          multiply(st, ((wave + (i0 + st) * NW) * PK - at(i0 + st)) / 32);
        }
      }
    }
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

// (tiles of 64 rows, with their sort, in place of strips, us of both products: one token of 8 experts of [4096, 14336] 119 + 5 for 114, 8
// tokens 446 + 5 for 337, 32 tokens 496 + 5 for 474; 10 tokens x 6 of 64 experts of [4096, 1792] 317 + 7 for 240)
bool group_strip_takes(const GroupArgs& a) {
  return a.ws[0] == nullptr && a.K >= kGsPieceBytes / 2 && a.n <= kStripChoices;
}

template <GroupKind KIND>
static int launch_strip_kind(const GroupArgs& a, hipStream_t stream) {
  // (48 and 32 KB of LDS a workgroup: three and five of them a CU have about 96 KB of weights on their way)
  constexpr int NW = 4, NST = KIND == kGroupGate ? 3 : 4, NM = KIND == kGroupGate ? 2 : 1;
  constexpr int LDS = NW * NST * NM * kGsCols * kGsPieceBytes;
  constexpr auto kern = group_strip_kernel<KIND, NW, NST>;
  if (set_max_lds<kern, LDS>() != 0) return -1;
  hipLaunchKernelGGL(kern, dim3((a.N + 8 * kGsCols - 1) / (8 * kGsCols) * 8 * a.n), dim3(NW * 64), LDS, stream, a);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
int launch_group_strip(const GroupArgs& a, GroupKind kind, hipStream_t stream) {
  return kind == kGroupGate ? launch_strip_kind<kGroupGate>(a, stream) : launch_strip_kind<kGroupDown>(a, stream);
}

}  // namespace tri
