// Routing of tokens to experts (tri_route), and the order in which the experts' products take their rows.
//
// Routing: with s the softmax or sigmoid of a token's logits and c = s + bias, the top_k experts of the largest c in descending
// order (ties: the lowest index), out of the top_groups best groups (a group counts the sum of its group_top largest c); weights
// are s of the chosen, over their sum if renormalised, times a factor.
//
// Scores and choices are computed in 64 bits: which expert is chosen is a whole number, and two scores that 32 bits cannot tell
// apart are common among millions of them.  The arithmetic is small all the same (4096 x 256 exponentials: the matrix would take
// as long to read as they to compute).
//
// A token has LPT lanes of a wave, each with EPL experts next to each other.  What bounds it is a chain of trips in a row: top_k searches, each a
// reduction over the lanes by operand exchanges (21 us with exchanges through LDS) and three reads of the winner's values through
// LDS, and before them, where there are groups, a lane's loop over the E / groups scores of its group in LDS.  4096 tokens x 256 experts in
// 8 groups, 8 chosen: 12.6 us, where a launch takes 2.2.
#include "common.h"
#include "launch.h"

namespace tri {

constexpr int kRouteThreads = 256;

// a double's bits in an order that unsigned integers have; NaN (of either sign) below all numbers; none is 0
__device__ __forceinline__ uint64_t order_key(double x) {
  const uint64_t b = (uint64_t)__double_as_longlong(x);
  if (x != x) return 1;
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}

// Both halves of an exchange between lanes `O` apart, for a reduction that takes O = 1, 2, 4, ... in turn: within 16 lanes through
// the data path of an instruction's operand (a mirror serves for 4 and 8, smaller groups being alike by then), beyond by swaps of
// whole rows of lanes.  (An exchange through LDS takes about ten times as long, and every choice waits for six.)
template <int O>
__device__ __forceinline__ void exchange(uint32_t x, uint32_t& p, uint32_t& q) {
  if constexpr (O <= 8) {
    constexpr int kHow = O == 1 ? 0xB1 : (O == 2 ? 0x4E : (O == 4 ? 0x141 : 0x140));
    p = x;
    q = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kHow, 0xF, 0xF, true);
  } else {
    const uint2v r = O == 16 ? __builtin_amdgcn_permlane16_swap(x, x, false, false) : __builtin_amdgcn_permlane32_swap(x, x, false, false);
    p = r[0];
    q = r[1];
  }
}
template <int O>
__device__ __forceinline__ void exchange(double x, double& p, double& q) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  uint32_t pl, ql, ph, qh;
  exchange<O>((uint32_t)b, pl, ql);
  exchange<O>((uint32_t)(b >> 32), ph, qh);
  p = __builtin_bit_cast(double, (uint64_t)ph << 32 | pl);
  q = __builtin_bit_cast(double, (uint64_t)qh << 32 | ql);
}
template <int LPT, int O = 1>
__device__ __forceinline__ double lanes_sum(double x) {
  if constexpr (O < LPT) {
    double p, q;
    exchange<O>(x, p, q);
    return lanes_sum<LPT, O * 2>(p + q);
  } else {
    return x;
  }
}
template <int LPT, int O = 1>
__device__ __forceinline__ double lanes_max(double x) {
  if constexpr (O < LPT) {
    double p, q;
    exchange<O>(x, p, q);
    return lanes_max<LPT, O * 2>(fmax(p, q));
  } else {
    return x;
  }
}
template <int LPT, int O = 1>
__device__ __forceinline__ uint32_t lanes_max(uint32_t x) {
  if constexpr (O < LPT) {
    uint32_t p, q;
    exchange<O>(x, p, q);
    return lanes_max<LPT, O * 2>(p > q ? p : q);
  } else {
    return x;
  }
}

template <typename T>
__device__ __forceinline__ double logit_of(const void* p, int64_t i) { return (double)(float)static_cast<const T*>(p)[i]; }

template <int LPT, int EPL>
__global__ __launch_bounds__(kRouteThreads) void route_kernel(RouteArgs a) {
  constexpr int TPB = kRouteThreads / LPT;  // tokens per workgroup
  __shared__ double choice_s[LPT == 64 ? TPB * 64 * EPL : 1];  // (groups: a wave per token)
  const int lane = threadIdx.x & (LPT - 1), slot = threadIdx.x / LPT;
  const int64_t token = (int64_t)blockIdx.x * TPB + slot;
  const bool live = token < a.T;  // (lanes of other tokens take part in the exchanges below)
  const int64_t row = (live ? token : a.T - 1) * a.ldl;
  double s[EPL];
  bool in[EPL];
  double top = -__builtin_inf();
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = lane * EPL + j;
    in[j] = e < a.E;
    double z = -__builtin_inf();
    if (in[j]) {
      z = a.dtype == 2 ? logit_of<float>(a.logits, row + e)
                       : (a.dtype == 1 ? logit_of<__bf16>(a.logits, row + e) : logit_of<_Float16>(a.logits, row + e));
    }
    s[j] = z;
    top = fmax(top, z);
  }
  if (a.sigmoid) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) s[j] = in[j] ? 1.0 / (1.0 + exp(-s[j])) : 0.0;
  } else {
    top = lanes_max<LPT>(top);
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      s[j] = in[j] ? (s[j] == -__builtin_inf() ? 0.0 : exp(s[j] - top)) : 0.0;  // (no logit above -inf: zeros, not NaN)
      sum += s[j];
    }
    sum = lanes_sum<LPT>(sum);
#pragma unroll
    for (int j = 0; j < EPL; ++j) s[j] = sum == 0.0 ? 0.0 : s[j] / sum;
  }
  double c[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) c[j] = s[j] + (a.bias != nullptr && in[j] ? (double)a.bias[lane * EPL + j] : 0.0);
  constexpr uint64_t kMine = LPT == 64 ? ~0ull : (1ull << (LPT & 63)) - 1;
  const int first = (int)(threadIdx.x & 63) - lane;  // (of this token's lanes in the wave)
  // a NaN of the token's makes all its weights NaN: an expert that has one is the last to be chosen, and would not be seen
  bool nan = false;
#pragma unroll
  for (int j = 0; j < EPL; ++j) nan = nan || c[j] != c[j];
  nan = ((__ballot(nan) >> first) & kMine) != 0;
  if constexpr (LPT == 64) {
    if (a.groups > 1) {
      double* const mine = choice_s + slot * 64 * EPL;
#pragma unroll
      for (int j = 0; j < EPL; ++j) mine[lane * EPL + j] = c[j];
      __syncthreads();
      // lane g: the score of group g, and its place among all
      const int size = a.E / a.groups;
      uint64_t key = 0;
      if (lane < a.groups) {
        double m1 = -__builtin_inf(), m2 = -__builtin_inf();
        for (int i = 0; i < size; ++i) {
          const double v = mine[lane * size + i];
          if (v > m1) {
            m2 = m1;
            m1 = v;
          } else if (v > m2) {
            m2 = v;
          }
        }
        key = order_key(a.group_top == 2 ? m1 + m2 : m1);
      }
      int place = 0;
      for (int g = 0; g < a.groups; ++g) {
        const uint64_t other = __shfl(key, g);
        place += (other > key || (other == key && g < lane)) ? 1 : 0;
      }
      const uint64_t stays = __ballot(lane < a.groups && place < a.top_groups);
#pragma unroll
      for (int j = 0; j < EPL; ++j) in[j] = in[j] && ((stays >> ((lane * EPL + j) / size)) & 1);
    }
  }
  uint64_t key[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) key[j] = in[j] ? order_key(c[j]) : 0;
  double sum = 0.0, my_w = 0.0;
  int my_id = 0;
  for (int r = 0; r < a.k; ++r) {
    // this lane's best: largest key, lowest index
    uint64_t bk = key[0];
    int bj = 0;
    double bs = s[0];
#pragma unroll
    for (int j = 1; j < EPL; ++j) {
      const bool take = key[j] > bk;
      bk = take ? key[j] : bk;
      bj = take ? j : bj;
      bs = take ? s[j] : bs;
    }
    // of all lanes: by the upper 32 bits, and by the lower ones where those are not enough; then the first such lane
    const uint32_t hi = (uint32_t)(bk >> 32), lo = (uint32_t)bk;
    const bool near = hi == lanes_max<LPT>(hi);
    uint64_t who = (__ballot(near) >> first) & kMine;
    if (__ballot((who & (who - 1)) != 0) != 0) {  // (of any token of the wave)
      const uint32_t best = lanes_max<LPT>(near ? lo : 0u);
      who = (__ballot(near && lo == best) >> first) & kMine;
    }
    const int owner = __builtin_ctzll(who);
    const int be = __shfl(lane * EPL + bj, first + owner);
    bs = __shfl(bs, first + owner);
    if (lane == owner) {
#pragma unroll
      for (int j = 0; j < EPL; ++j) key[j] = j == bj ? 0 : key[j];
    }
    sum += bs;
    my_id = r == lane ? be : my_id;
    my_w = r == lane ? bs : my_w;
  }
  if (live && lane < a.k) {  // (top_k is at most LPT)
    a.ids[token * a.k + lane] = my_id;
    const double w = !a.renormalize ? my_w : (sum == 0.0 ? 0.0 : my_w / sum);
    a.weights[token * a.k + lane] = nan ? __builtin_nanf("") : (float)(w * (double)a.scale);
  }
}

template <int LPT, int EPL>
static int launch_route_t(const RouteArgs& a, hipStream_t stream) {
  constexpr int TPB = kRouteThreads / LPT;
  hipLaunchKernelGGL((route_kernel<LPT, EPL>), dim3((unsigned)((a.T + TPB - 1) / TPB)), dim3(kRouteThreads), 0, stream, a);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
int launch_route(const RouteArgs& a, hipStream_t stream) {
  // (lanes per token are at least the experts, up to 64, and so at least top_k; groups want a wave per token)
  if (a.E <= 8 && a.groups == 1) return launch_route_t<8, 1>(a, stream);
  if (a.E <= 16 && a.groups == 1) return launch_route_t<16, 1>(a, stream);
  if (a.E <= 32 && a.groups == 1) return launch_route_t<32, 1>(a, stream);
  if (a.E <= 64) return launch_route_t<64, 1>(a, stream);
  if (a.E <= 128) return launch_route_t<64, 2>(a, stream);
  if (a.E <= 256) return launch_route_t<64, 4>(a, stream);
  return launch_route_t<64, 8>(a, stream);
}


// ---------------------------------------------------------------------------
// The rows of every expert next to each other: places (row of a token's choice, token * top_k + i) in ascending order for each
// expert, and the row tiles of `bm` that the experts' products take.  One workgroup: a wave counts and places a contiguous
// sixteenth of the choices, 64 at a time, so that the order does not depend on timing.  Bound by trips to memory and LDS in a row:
// 5 us, 8192 choices of 8 experts 7 to 10, 12288 of 64 14.
// ---------------------------------------------------------------------------
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;

__global__ __launch_bounds__(kSortThreads) void expert_rows_kernel(ExpertRowsArgs a) {
  extern __shared__ int sort_lds[];
  int* const base = sort_lds;                  // [waves][E]: counts, then where a wave's rows of an expert begin
  int* const start = base + kSortWaves * a.E;  // [E]
  int* const tiles = start + a.E;              // [E]
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  for (int i = t; i < kSortWaves * a.E; i += kSortThreads) base[i] = 0;
  __syncthreads();
  const int rounds = (a.n + kSortThreads - 1) / kSortThreads;  // of 64 choices per wave
  const int s0 = wave * rounds * 64 + lane;
  int* const mine = base + wave * a.E;
  constexpr int B = 8;  // rounds whose choices are on their way at a time
  auto fetch = [&](int r, int (&e)[B]) {
#pragma unroll
    for (int u = 0; u < B; ++u) {
      const int s = s0 + (r + u) * 64;
      e[u] = r + u < rounds && s < a.n ? a.ids[s] : -1;
    }
  };
  int kept[B];
  for (int r = 0; r < rounds; r += B) {
    fetch(r, kept);
#pragma unroll
    for (int u = 0; u < B; ++u)
      if (kept[u] >= 0 && kept[u] < a.E) atomicAdd(&mine[kept[u]], 1);
  }
  __syncthreads();
  for (int e = t; e < a.E; e += kSortThreads) {
    int sum = 0;
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = base[w * a.E + e];
      base[w * a.E + e] = sum;
      sum += c;
    }
    start[e] = sum;
    tiles[e] = (sum + a.bm - 1) / a.bm;
  }
  __syncthreads();
  if (wave == 0) {  // exclusive sums over the experts
    int rows0 = 0, tiles0 = 0;
    for (int e0 = 0; e0 < a.E; e0 += 64) {
      const int e = e0 + lane;
      const int rc = e < a.E ? start[e] : 0, tc = e < a.E ? tiles[e] : 0;
      int ri = rc, ti = tc;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int ro = __shfl_up(ri, o), to = __shfl_up(ti, o);
        ri += lane >= o ? ro : 0;
        ti += lane >= o ? to : 0;
      }
      if (e < a.E) {
        const int rb = rows0 + ri - rc, tb = tiles0 + ti - tc;
        start[e] = rb;
        for (int i = 0; i < tc; ++i) a.tiles[1 + tb + i] = make_int4(e, rb + i * a.bm, min(a.bm, rc - i * a.bm), 0);
      }
      rows0 += __shfl(ri, 63);
      tiles0 += __shfl(ti, 63);
    }
    if (lane == 0) a.tiles[0] = make_int4(tiles0, rows0, 0, 0);
  }
  __syncthreads();
  for (int r0 = 0; r0 < rounds; r0 += B) {
    if (rounds > B) fetch(r0, kept);
#pragma unroll
    for (int u = 0; u < B; ++u) {
      const int s = s0 + (r0 + u) * 64, e = kept[u];
      const bool real = e >= 0 && e < a.E;
      uint64_t same = __ballot(real);  // lanes of this one's expert
      for (int b = 0; (1 << b) < a.E; ++b) {
        const uint64_t bit = __ballot((e >> b) & 1);
        same &= ((e >> b) & 1) ? bit : ~bit;
      }
      if (real) {
        const int rank = __popcll(same & ((1ull << lane) - 1)), at = mine[e];
        a.rows[start[e] + at + rank] = s;
        if (rank == 0) mine[e] = at + __popcll(same);  // (a wave's reads of LDS come before its later writes)
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
}

int launch_expert_rows(const ExpertRowsArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(expert_rows_kernel, dim3(1), dim3(kSortThreads), (kSortWaves + 2) * a.E * sizeof(int), stream, a);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}

// out[t] = sum of w[t, i] * y[t * k + i] over the choices i that are experts, in 32 bits, y being the sum of its parts; or
// (no weights, k = 1) that sum itself.
// Bound by the bytes of y, of which rows of four choices (or eight parts) are on their way at a time: 4096 tokens x 2 x 4096 in 43 us,
// 2048 x 6 x 4096 in 46, 4.7 TB/s.
template <bool PARTS>
__global__ __launch_bounds__(256) void join_rows_kernel(JoinRowsArgs a) {
  const int c = ((int)blockIdx.x * 256 + (int)threadIdx.x) * 4;
  if (c >= a.N) return;
  for (int64_t t = blockIdx.y; t < a.T; t += gridDim.y) {
    float4v s = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < a.k; i0 += 4) {
      float4v v[4];
      float w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t row = t * a.k + min(i0 + u, a.k - 1);
        w[u] = 1.0f;
        bool real = i0 + u < a.k;
        if (a.weights != nullptr) {
          const int e = a.ids[row];
          real = real && e >= 0 && e < a.E;
          w[u] = a.weights[row];
        }
        v[u] = float4v{0.f, 0.f, 0.f, 0.f};
        if (!real) w[u] = 0.0f;  // (rows without an expert are not there: their memory may hold anything)
        else if (PARTS) v[u] = sum_splits(a.y, a.parts, a.T * a.k * a.N, row * a.N + c);
        else v[u] = *reinterpret_cast<const float4v*>(a.y + row * a.N + c);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = fmaf(w[u], v[u][j], s[j]);
    }
    const half4v h = {(half_t)s[0], (half_t)s[1], (half_t)s[2], (half_t)s[3]};
    *reinterpret_cast<half4v*>(a.out + t * a.ldo + c) = h;
  }
}

int launch_join_rows(const JoinRowsArgs& a, hipStream_t stream) {
  const dim3 grid((a.N / 4 + 255) / 256, (unsigned)(a.T < 65535 ? a.T : 65535));
  if (a.parts > 1) hipLaunchKernelGGL((join_rows_kernel<true>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((join_rows_kernel<false>), grid, dim3(256), 0, stream, a);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tri
