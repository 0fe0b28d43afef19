// Attention of new tokens over caches of several sequences that hold them already, 16-bit or in 4-bit blocks (fp4.h), with
// a causal mask, and in a sliding window behind a few first keys that stay visible.
//
// Rows.  The query heads of a KV head are stacked along the query axis, tokens outermost: row r of (sequence, KV head) is
// head r % group of token r / group.  K and V are then read once for the whole group, and the rows of a block stand at few
// positions, so that its masks cost little.
//
// Keys.  The keys that some row of a block sees are [0, sinks) and [lo, end).  They are walked as ONE list, of which
// index l stands for key l where l < sinks, for key l + lo - sinks beyond: a handful of first keys shares its tile with the
// first keys of the window.  Where the gap between the two is empty (or there is no window) the list is [0, end).
//
// Scores are computed transposed, S^T[key, row] = K . Q^T, so that a lane owns one row and sixteen keys of a block of 32,
// the running maximum and sum are per-lane scalars, and the probabilities lie in the registers as O^T += V^T . P^T wants
// them.
#include "common.h"
#include "fp4.h"
#include "launch.h"

namespace tri {

constexpr int kCacheTile = 64;       // keys
constexpr int kCacheRows = 128;      // stacked rows per workgroup, 32 a wave
// the running maximum is raised when a score exceeds it by this many powers of two: probabilities stay below 2^8, and the
// sums are rescaled rarely
constexpr float kCacheLazyMax = 8.0f;

// what a row block of a sequence sees
struct KeyList {
  int len;        // keys of the sequence
  int n;          // ... in the list
  int sinks, gap; // list index l is key l + (l < sinks ? 0 : gap)
};

__device__ __forceinline__ KeyList key_list(const CacheAttnArgs& a, int b, int tok0, int tok1) {
  KeyList k;
  k.len = a.lens == nullptr ? a.kv_len : min(max(a.lens[b], 0), a.kv_len);
  const int first = max(k.len - a.S + tok0, 0), last = k.len - a.S + tok1;  // positions of the block's tokens
  const int end = last < 0 ? 0 : (a.causal ? last + 1 : k.len);
  const int lo = a.window > 0 ? max(0, first - a.window + 1) : 0;
  k.sinks = lo > a.sinks ? a.sinks : 0;
  k.gap = lo > a.sinks ? lo - a.sinks : 0;
  k.n = end - k.gap;
  return k;
}

template <int D>
struct CacheLds {
  static constexpr int CPR = D / 8;  // 16-byte chunks per row; chunk c of row r at slot c ^ fk(r) (K), c ^ fv(r) (V)
  static constexpr int HALFS = kCacheTile * D;
  __device__ static __forceinline__ int fk(int row) { return D == 128 ? (row & 15) : ((row >> 1) & 7); }
  __device__ static __forceinline__ int fv(int row) { return D == 128 ? ((row & 3) << 2) : (((row >> 1) & 1) << 2); }
};

// blockIdx.x: (run, row block, KV head, sequence), the last one outermost
template <int D, bool FP4>
__device__ __forceinline__ void cache_attn_body(const CacheAttnArgs& a, half_t* lds) {
  using L = CacheLds<D>;
  constexpr int KSTEPS = D / 16, DT = D / 32, CPR = D / 8;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int l32 = lane & 31, g = lane >> 5;
  const int group = a.Hq / a.Hkv, rows = a.S * group, nrb = (rows + kCacheRows - 1) / kCacheRows;
  int id = (int)blockIdx.x;
  const int run = id % a.runs; id /= a.runs;
  const int rb = nrb - 1 - id % nrb; id /= nrb;  // (the latest rows, which see most, first)
  const int hk = id % a.Hkv, b = id / a.Hkv;
  const int r0 = rb * kCacheRows;
  const KeyList kl = key_list(a, b, r0 / group, (min(r0 + kCacheRows, rows) - 1) / group);
  const int ntiles = (kl.n + kCacheTile - 1) / kCacheTile;
  const int per = (ntiles + a.runs - 1) / a.runs, tile0 = min(run * per, ntiles), tile1 = min(tile0 + per, ntiles);

  const int row = r0 + wave * 32 + l32, rowc = min(row, rows - 1);
  const int tok = rowc / group, head = hk * group + rowc % group;
  const int pos = kl.len - a.S + tok;
  half8v qf[KSTEPS];
  const half_t* qp = a.q + ((int64_t)b * a.S + tok) * a.ldq + (int64_t)head * D + g * 8;
#pragma unroll
  for (int ks = 0; ks < KSTEPS; ++ks) qf[ks] = *reinterpret_cast<const half8v*>(qp + ks * 16);

  half_t *const kt = lds, *const vt = lds + L::HALFS;
  const float c2 = a.scale * kLog2e;
  float m = -INFINITY, l = 0.f;
  float16v o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;

  const int j4 = (lane & 15) >> 2;
  for (int tile = tile0; tile < tile1; ++tile) {
    __syncthreads();
    // ---- K and V to LDS (past the last key: the last one again, whose scores are masked)
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const CacheView& c = kv ? a.vc : a.kc;
      half_t* const dst = kv ? vt : kt;
      for (int p = t; p < kCacheTile * CPR; p += 256) {
        const int r = p / CPR, ch = p % CPR;
        const int li = min(tile * kCacheTile + r, kl.n - 1);
        const int64_t key = li + (li < kl.sinks ? 0 : kl.gap);
        half8v x;
        if (FP4) {
          const uint8_t* src = static_cast<const uint8_t*>(c.p) + b * c.sb + hk * c.sh + key * c.sr + ch * 4;
          x = fp4x8_to_half8(*reinterpret_cast<const uint32_t*>(src), fp4_scale(c.scales[b * c.xb + hk * c.xh + key * c.xr + ch / 4]));
        } else {
          x = *reinterpret_cast<const half8v*>(static_cast<const half_t*>(c.p) + b * c.sb + hk * c.sh + key * c.sr + ch * 8);
        }
        *reinterpret_cast<half8v*>(dst + r * D + ((ch ^ (kv ? L::fv(r) : L::fk(r))) << 3)) = x;
      }
    }
    __syncthreads();
    // ---- S^T = K . Q^T
    float16v st[2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r) st[mt][r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
        st[mt] = mfma32(lds_read8(kt + (mt * 32 + l32) * D + (((ks * 2 + g) ^ L::fk(l32)) << 3)), qf[ks], st[mt]);
    // ---- mask, maximum
    float mx = -INFINITY;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int li = tile * kCacheTile + mt * 32 + (r >> 2) * 8 + g * 4 + (r & 3);
        const int key = li + (li < kl.sinks ? 0 : kl.gap);
        const bool hidden = li >= kl.n || pos < 0 || (a.causal && key > pos) ||
                            (a.window > 0 && key <= pos - a.window && key >= a.sinks);
        if (hidden) st[mt][r] = -INFINITY;
        mx = fmaxf(mx, st[mt][r]);
      }
    mx = pair_max(mx) * c2;
    if (__builtin_amdgcn_ballot_w64(mx > m + kCacheLazyMax) != 0) {
      const float mnew = fmaxf(m, mx);
      const float alpha = mnew == -INFINITY ? 1.0f : fast_exp2(m - mnew);
      m = mnew;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] = o[dt] * alpha;
    }
    const float nm = m == -INFINITY ? 0.f : -m;
    // ---- probabilities, rounded to nearest (half the error of cutting them off), their sum before that
    half8v pf[2][2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float p = fast_exp2(fmaf(st[mt][hh * 8 + e], c2, nm));
          l += p;
          pf[mt][hh][e] = (half_t)p;
        }
    // ---- O^T += V^T . P^T
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const int chunk = dt * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
          const half_t* vp = vt + (mt * 32 + hh * 16 + 4 * g + j4) * D + ((chunk ^ L::fv(j4)) << 3) + (lane & 1) * 4;
          o[dt] = mfma32(cat8(lds_read_tr16(vp), lds_read_tr16(vp + 8 * D)), pf[mt][hh], o[dt]);
        }
  }

  l = pair_sum(l);
  if (row >= rows) return;
  if (a.runs > 1) {
    // this run's unnormalised O [b][hk][row][run][D], then (max, sum) [b][hk][row][run][2]
    const int64_t at = (((int64_t)b * a.Hkv + hk) * rows + row) * a.runs + run;
    float* po = a.ws + at * D + g * 4;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq)
        *reinterpret_cast<float4v*>(po + dt * 32 + rq * 8) =
            float4v{o[dt][rq * 4], o[dt][rq * 4 + 1], o[dt][rq * 4 + 2], o[dt][rq * 4 + 3]};
    if (g == 0) {
      float* ps = a.ws + (int64_t)a.B * a.Hkv * rows * a.runs * D + at * 2;
      ps[0] = m;
      ps[1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;  // (no visible key: zeros)
  half_t* op = a.out + ((int64_t)b * a.S + tok) * a.ldo + (int64_t)head * D + g * 4;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) {
      half4v hv;
#pragma unroll
      for (int e = 0; e < 4; ++e) hv[e] = (half_t)(o[dt][rq * 4 + e] * inv);
      *reinterpret_cast<half4v*>(op + dt * 32 + rq * 8) = hv;
    }
  if (a.lse != nullptr && g == 0)
    a.lse[((int64_t)b * a.Hq + head) * a.S + tok] = l == 0.f ? -INFINITY : (m + fast_log2(l)) * kLn2;
}

template <int D, bool FP4>
__global__ __launch_bounds__(256) void cache_attn_kernel(CacheAttnArgs a) {
  __shared__ __attribute__((aligned(16))) half_t lds[2 * CacheLds<D>::HALFS];
  cache_attn_body<D, FP4>(a, lds);
}

// Merge of the runs: one thread per four channels of a row, in a fixed order.
template <int D>
__global__ __launch_bounds__(256) void cache_merge_kernel(CacheAttnArgs a) {
  constexpr int LPR = D / 4;
  const int group = a.Hq / a.Hkv, rows = a.S * group;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x, at = idx / LPR;
  const int d4 = (int)(idx % LPR);
  if (at >= (int64_t)a.B * a.Hkv * rows) return;
  const float* po = a.ws + at * a.runs * D + d4 * 4;
  const float* ps = a.ws + (int64_t)a.B * a.Hkv * rows * a.runs * D + at * a.runs * 2;
  float m = -INFINITY;
  for (int i = 0; i < a.runs; ++i) m = fmaxf(m, ps[i * 2]);
  float l = 0.f;
  float4v acc = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < a.runs; ++i) {
    const float w = ps[i * 2] == -INFINITY ? 0.f : fast_exp2(ps[i * 2] - m);
    const float4v v = *reinterpret_cast<const float4v*>(po + (int64_t)i * D);
    l = fmaf(ps[i * 2 + 1], w, l);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(v[e], w, acc[e]);
  }
  const int row = (int)(at % rows), hk = (int)(at / rows % a.Hkv), b = (int)(at / rows / a.Hkv);
  const int tok = row / group, head = hk * group + row % group;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  half4v hv;
#pragma unroll
  for (int e = 0; e < 4; ++e) hv[e] = (half_t)(acc[e] * inv);
  *reinterpret_cast<half4v*>(a.out + ((int64_t)b * a.S + tok) * a.ldo + (int64_t)head * D + d4 * 4) = hv;
  if (a.lse != nullptr && d4 == 0)
    a.lse[((int64_t)b * a.Hq + head) * a.S + tok] = l == 0.f ? -INFINITY : (m + fast_log2(l)) * kLn2;
}

// ---- how many runs
struct CachePlan {
  int runs;
  int64_t nwg;  // workgroups per run
};
static CachePlan cache_plan(int B, int S, int Hq, int Hkv, int kv_len, int window, int sinks) {
  const int rows = S * (Hq / Hkv);
  CachePlan p;
  p.nwg = (int64_t)((rows + kCacheRows - 1) / kCacheRows) * Hkv * B;
  // most keys of a row block, in tiles
  const int64_t toks = (kCacheRows + Hq / Hkv - 1) / (Hq / Hkv) + 1;
  int64_t keys = kv_len;
  if (window > 0 && toks + window + sinks < keys) keys = toks + window + sinks;
  const int64_t tiles = (keys + kCacheTile - 1) / kCacheTile;
  int64_t runs = 512 / p.nwg;
  if (runs > tiles / 4) runs = tiles / 4;
  if (runs > 64) runs = 64;
  p.runs = runs < 1 ? 1 : (int)runs;
  return p;
}

static int64_t run_bytes(int B, int S, int Hq, int D) { return (int64_t)B * S * Hq * (D + 2) * 4; }

int64_t cache_attn_workspace_bytes(int B, int S, int Hq, int Hkv, int D, int kv_len, int window, int sinks, bool /*four_bit*/) {
  const int runs = cache_plan(B, S, Hq, Hkv, kv_len, window, sinks).runs;
  return runs > 1 ? runs * run_bytes(B, S, Hq, D) : 0;
}

template <int D, bool FP4>
static void launch_t(const CacheAttnArgs& a, unsigned nwg, hipStream_t stream) {
  hipLaunchKernelGGL((cache_attn_kernel<D, FP4>), dim3(nwg), dim3(256), 0, stream, a);
}

int launch_cache_attention(const CacheAttnArgs& args, hipStream_t stream) {
  CacheAttnArgs a = args;
  const CachePlan p = cache_plan(a.B, a.S, a.Hq, a.Hkv, a.kv_len, a.window, a.sinks);
  const int64_t fit = a.ws != nullptr ? a.ws_bytes / run_bytes(a.B, a.S, a.Hq, a.D) : 0;
  a.runs = (int)(fit < p.runs ? (fit < 1 ? 1 : fit) : p.runs);
  const unsigned nwg = (unsigned)(p.nwg * a.runs);
  const bool fp4 = a.kc.scales != nullptr;
  if (a.D == 128) fp4 ? launch_t<128, true>(a, nwg, stream) : launch_t<128, false>(a, nwg, stream);
  else fp4 ? launch_t<64, true>(a, nwg, stream) : launch_t<64, false>(a, nwg, stream);
  if (hipGetLastError() != hipSuccess) return -1;
  if (a.runs == 1) return 0;
  const int64_t lanes = (int64_t)a.B * a.S * a.Hq * (a.D / 4);
  const dim3 grid((unsigned)((lanes + 255) / 256));
  if (a.D == 128) hipLaunchKernelGGL((cache_merge_kernel<128>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((cache_merge_kernel<64>), grid, dim3(256), 0, stream, a);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tri
