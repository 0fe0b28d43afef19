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

// result of a row: four channels d4 of the finished sum, divided by the softmax's, and its log-sum-exp (no visible key:
// zeros and -inf)
template <int D>
__device__ __forceinline__ void store_row(const CacheAttnArgs& a, int b, int hk, int row, int d4, float m, float l, float4v acc) {
  const int group = a.Hq / a.Hkv, tok = row / group, head = hk * group + row % group;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  half4v hv;
#pragma unroll
  for (int e = 0; e < 4; ++e) hv[e] = (half_t)(acc[e] * inv);
  *reinterpret_cast<half4v*>(a.out + ((int64_t)b * a.S + tok) * a.ldo + (int64_t)head * D + d4 * 4) = hv;
  if (a.lse != nullptr && d4 == 0)
    a.lse[((int64_t)b * a.Hq + head) * a.S + tok] = l == 0.f ? -INFINITY : (m + fast_log2(l)) * kLn2;
}

// ... or, of several runs, its partial result: unnormalised O [b][hk][row][run][D], then (max, sum) [b][hk][row][run][2]
template <int D>
__device__ __forceinline__ void finish_row(const CacheAttnArgs& a, int b, int hk, int row, int run, int d4, float m, float l, float4v acc) {
  if (a.runs == 1) {
    store_row<D>(a, b, hk, row, d4, m, l, acc);
    return;
  }
  const int64_t rows = (int64_t)a.S * (a.Hq / a.Hkv), at = (((int64_t)b * a.Hkv + hk) * rows + row) * a.runs + run;
  *reinterpret_cast<float4v*>(a.ws + at * D + d4 * 4) = acc;
  if (d4 == 0) {
    float* ps = a.ws + (int64_t)a.B * a.Hkv * rows * a.runs * D + at * 2;
    ps[0] = m;
    ps[1] = l;
  }
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
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq)
      finish_row<D>(a, b, hk, row, run, dt * 8 + rq * 2 + g, m, l,
                    float4v{o[dt][rq * 4], o[dt][rq * 4 + 1], o[dt][rq * 4 + 2], o[dt][rq * 4 + 3]});
}

template <int D, bool FP4>
__global__ __launch_bounds__(256) void cache_attn_kernel(CacheAttnArgs a) {
  __shared__ __attribute__((aligned(16))) half_t lds[2 * CacheLds<D>::HALFS];
  cache_attn_body<D, FP4>(a, lds);
}

// ---------------------------------------------------------------------------------------------------- few rows
// At most 16 * NT stacked rows of a KV head: a call is bound by reading the keys and values once.  Every wave walks tiles
// of 32 keys of its own - no barrier until the waves of a workgroup merge - with the next tile's loads in flight.  K goes
// from memory straight into the registers that the matrix instructions want: a lane holds D / 4 channels of one key, in
// 4 bits one block with one scale (the order of the channels in the product is free, as long as q has the same).  V goes
// through a tile of LDS that only its wave touches, for the transpose.
constexpr int kFewRowTile = 32;   // keys

template <int D>
__device__ __forceinline__ int few_row_swizzle(int row) { return D == 128 ? (row & 7) << 1 : ((row >> 1) & 3) << 1; }

// the 16-byte chunks (4-bit: blocks) of a row of n, to 64 lanes
template <int D, bool FP4>
struct FewRowTile {
  static constexpr int KB = kFewRowTile / 16, KS = D / 32, DB = D / 16;
  static constexpr int KP = FP4 ? 1 : KS;                          // 16-byte pieces (4-bit, D = 64: half ones) of a key per lane
  static constexpr int VPR = FP4 ? D / 32 : D / 8;                  // pieces of a row of V
  static constexpr int VP = kFewRowTile * VPR / 64;                 // ... per lane
  uint4v k[KB][KP], v[VP];
  uint32_t kx[KB], vx[VP];
};

template <int D, bool FP4, int NT>
__device__ __forceinline__ void cache_attn_few_body(const CacheAttnArgs& a, half_t* lds) {
  using T = FewRowTile<D, FP4>;
  constexpr int KB = T::KB, KS = T::KS, DB = T::DB;
  const int t = threadIdx.x, lane = t & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int group = a.Hq / a.Hkv, rows = a.S * group;
  int id = (int)blockIdx.x;
  const int run = id % a.runs; id /= a.runs;
  const int hk = id % a.Hkv, b = id / a.Hkv;
  const KeyList kl = key_list(a, b, 0, a.S - 1);
  const int ntiles = (kl.n + kFewRowTile - 1) / kFewRowTile;
  const int per = (ntiles + a.runs - 1) / a.runs, tile0 = min(run * per, ntiles), tile1 = min(tile0 + per, ntiles);

  half8v qf[NT][KS];
  int pos[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = min(nt * 16 + l16, rows - 1), tok = row / group;
    pos[nt] = kl.len - a.S + tok;
    const half_t* qp = a.q + ((int64_t)b * a.S + tok) * a.ldq + (int64_t)(hk * group + row % group) * D;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[nt][s] = *reinterpret_cast<const half8v*>(qp + (FP4 ? g * (D / 4) + s * 8 : s * 32 + g * 8));
  }
  const int pos0 = kl.len - a.S, pos1 = kl.len - 1;  // first and last token's

  // ---- loads of a tile
  constexpr int ES = FP4 ? 1 : 2;  // bytes per element of a CacheView
  const uint8_t* const kbase = static_cast<const uint8_t*>(a.kc.p) + (b * a.kc.sb + hk * a.kc.sh) * ES;
  const uint8_t* const vbase = static_cast<const uint8_t*>(a.vc.p) + (b * a.vc.sb + hk * a.vc.sh) * ES;
  const uint8_t* const kxbase = FP4 ? a.kc.scales + b * a.kc.xb + hk * a.kc.xh : nullptr;
  const uint8_t* const vxbase = FP4 ? a.vc.scales + b * a.vc.xb + hk * a.vc.xh : nullptr;
  const int64_t ksr = a.kc.sr * ES, vsr = a.vc.sr * ES;
  auto fetch = [&](int tile, T& x) __attribute__((always_inline)) {
    auto key_of = [&](int r) {  // (past the last key: the last one again, whose scores are masked)
      const int li = min(tile * kFewRowTile + r, kl.n - 1);
      return (int64_t)(li + (li < kl.sinks ? 0 : kl.gap));
    };
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int64_t key = key_of(kb * 16 + l16);
      const uint8_t* p = kbase + key * ksr;
      if constexpr (FP4) {
        if constexpr (D == 128) {
          x.k[kb][0] = *reinterpret_cast<const uint4v*>(p + g * 16);
        } else {
          const uint2v h = *reinterpret_cast<const uint2v*>(p + g * 8);
          x.k[kb][0] = uint4v{h[0], h[1], 0u, 0u};
        }
        x.kx[kb] = kxbase[key * a.kc.xr + (D == 128 ? g : g / 2)];
      } else {
#pragma unroll
        for (int s = 0; s < KS; ++s) x.k[kb][s] = *reinterpret_cast<const uint4v*>(p + s * 64 + g * 16);
      }
    }
#pragma unroll
    for (int i = 0; i < T::VP; ++i) {
      const int p = i * 64 + lane, r = p / T::VPR, c = p % T::VPR;
      const int64_t key = key_of(r);
      x.v[i] = *reinterpret_cast<const uint4v*>(vbase + key * vsr + c * 16);
      if constexpr (FP4) x.vx[i] = vxbase[key * a.vc.xr + c];
    }
  };

  half_t* const vt = lds + wave * kFewRowTile * D;
  const float c2 = a.scale * kLog2e;
  float m[NT], l[NT];
  float4v o[NT][DB];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt] = -INFINITY; l[nt] = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db) o[nt][db] = float4v{0.f, 0.f, 0.f, 0.f};
  }
  const int j4 = (lane & 15) >> 2;

  // A tile in two parts: V to LDS and the scores, which free the registers of the tile for the next one's loads ...
  float4v st[NT][KB];
  auto begin = [&](const T& x) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < T::VP; ++i) {
      const int p = i * 64 + lane, r = p / T::VPR, c = p % T::VPR;
      if constexpr (FP4) {
        const float sc = fp4_scale(x.vx[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<half8v*>(vt + r * D + (((c * 4 + j) ^ few_row_swizzle<D>(r)) << 3)) = fp4x8_to_half8(x.v[i][j], sc);
      } else {
        *reinterpret_cast<uint4v*>(vt + r * D + ((c ^ few_row_swizzle<D>(r)) << 3)) = x.v[i];
      }
    }
    // ---- S^T = K . Q^T
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const float sc = FP4 ? fp4_scale(x.kx[kb]) : 1.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) st[nt][kb] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        half8v kf;
        if constexpr (FP4) kf = fp4x8_to_half8(x.k[kb][0][s], sc);
        else kf = __builtin_bit_cast(half8v, x.k[kb][s]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) st[nt][kb] = mfma16(kf, qf[nt][s], st[nt][kb]);
      }
    }
  };
  // ... and the softmax and its product with V
  auto end = [&](int tile) __attribute__((always_inline)) {
    // ---- mask: needed where the list ends, a token's keys end, or the window of a later token has begun
    const int li0 = tile * kFewRowTile, li1 = li0 + kFewRowTile - 1;
    const bool masked = li1 >= kl.n || pos0 < 0 || (a.causal && li1 + kl.gap > pos0) ||
                        (a.window > 0 && li0 + (li0 < kl.sinks ? 0 : kl.gap) <= pos1 - a.window && li1 >= a.sinks);
    half8v pf[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (masked) {  // wave-uniform
        asm volatile("");
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int li = li0 + kb * 16 + g * 4 + r, key = li + (li < kl.sinks ? 0 : kl.gap);
            if (li >= kl.n || pos[nt] < 0 || (a.causal && key > pos[nt]) ||
                (a.window > 0 && key <= pos[nt] - a.window && key >= a.sinks))
              st[nt][kb][r] = -INFINITY;
          }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, st[nt][kb][r]);
      mx *= c2;
      if (__builtin_amdgcn_ballot_w64(mx > m[nt] + kCacheLazyMax) != 0) {  // wave-uniform; m is the same for a row's lanes
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float mnew = fmaxf(m[nt], mx);
        const float alpha = mnew == -INFINITY ? 1.0f : fast_exp2(m[nt] - mnew);
        m[nt] = mnew;
        l[nt] *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[nt][db] = o[nt][db] * alpha;
      }
      const float nm = m[nt] == -INFINITY ? 0.f : -m[nt];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = fast_exp2(fmaf(st[nt][kb][r], c2, nm));
          l[nt] += p;
          pf[nt][kb * 4 + r] = (half_t)p;
        }
    }
    // ---- O^T += V^T . P^T
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const int chunk = db * 2 + ((lane & 3) >> 1), r = 4 * g + j4;
      const half_t* vp = vt + r * D + ((chunk ^ few_row_swizzle<D>(r)) << 3) + (lane & 1) * 4;
      const half8v vf = cat8(lds_read_tr16(vp), lds_read_tr16(vp + 16 * D));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) o[nt][db] = mfma16(vf, pf[nt], o[nt][db]);
    }
  };

  // the wave's tiles tile0 + wave + 4 i; 4-bit tiles, a quarter the size, travel two at a time
  const int cnt = (tile1 - tile0 - wave + 3) / 4;
  auto at = [&](int i) { return tile0 + wave + 4 * i; };
  if (cnt > 0) {
    T x;
    fetch(at(0), x);
    if constexpr (FP4) {
      T y;
      fetch(at(min(1, cnt - 1)), y);
      int i = 0;
      for (; i + 3 < cnt; i += 2) {  // (no load under a condition: the waits can then count the loads behind the one they need)
        begin(x);
        fetch(at(i + 2), x);
        end(at(i));
        begin(y);
        fetch(at(i + 3), y);
        end(at(i + 1));
      }
      begin(x);
      if (i + 2 < cnt) fetch(at(i + 2), x);
      end(at(i));
      if (i + 1 < cnt) {
        begin(y);
        end(at(i + 1));
      }
      if (i + 2 < cnt) {
        begin(x);
        end(at(i + 2));
      }
    } else {
      for (int i = 0; i + 1 < cnt; ++i) {
        begin(x);
        fetch(at(i + 1), x);
        end(at(i));
      }
      begin(x);
      end(at(cnt - 1));
    }
  }

  // ---- the waves' states through LDS: O [wave][nt][d / 4][row] as float4, then (max, sum) [wave][nt][row]
  float4v* const ow = reinterpret_cast<float4v*>(lds);
  float* const sw = reinterpret_cast<float*>(ow + 4 * NT * (D / 4) * 16);
  __syncthreads();  // (every wave is done with its V tile)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float ls = l[nt];
    ls += __shfl_xor(ls, 16);
    ls += __shfl_xor(ls, 32);
#pragma unroll
    for (int db = 0; db < DB; ++db) ow[((wave * NT + nt) * (D / 4) + db * 4 + g) * 16 + l16] = o[nt][db];
    if (g == 0) {
      sw[((wave * NT + nt) * 16 + l16) * 2] = m[nt];
      sw[((wave * NT + nt) * 16 + l16) * 2 + 1] = ls;
    }
  }
  __syncthreads();
  for (int p = t; p < rows * (D / 4); p += 256) {
    const int row = p / (D / 4), d4 = p % (D / 4), nt = row / 16, r = row % 16;
    float M = -INFINITY, L = 0.f;
    float4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, sw[((w * NT + nt) * 16 + r) * 2]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = sw[((w * NT + nt) * 16 + r) * 2];
      const float sc = mw == -INFINITY ? 0.f : fast_exp2(mw - M);
      L = fmaf(sw[((w * NT + nt) * 16 + r) * 2 + 1], sc, L);
      const float4v v = ow[((w * NT + nt) * (D / 4) + d4) * 16 + r];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(v[e], sc, acc[e]);
    }
    finish_row<D>(a, b, hk, row, run, d4, M, L, acc);
  }
}

template <int D, bool FP4, int NT>
constexpr int kFewRowLds = 4 * (kFewRowTile * D * 2 > NT * 16 * D * 4 ? kFewRowTile * D * 2 : NT * 16 * D * 4) + 4 * NT * 16 * 8;

template <int D, bool FP4, int NT>
__global__ __launch_bounds__(256, 2) void cache_attn_few_kernel(CacheAttnArgs a) {
  __shared__ __attribute__((aligned(16))) half_t lds[kFewRowLds<D, FP4, NT> / 2];
  cache_attn_few_body<D, FP4, NT>(a, lds);
}

// Merge of the runs: four channels of a row per thread, WAYS threads for every WAYS-th run each, eight runs' loads in
// flight together, in a fixed order.  One way where the rows alone fill the chip.
template <int D, int WAYS>
__global__ __launch_bounds__(256) void cache_merge_kernel(CacheAttnArgs a) {
  constexpr int LPR = D / 4, LANES = 256 / WAYS, UNROLL = 8;
  const int group = a.Hq / a.Hkv, rows = a.S * group;
  const int64_t total = (int64_t)a.B * a.Hkv * rows;
  const int way = threadIdx.x / LANES, lane = threadIdx.x % LANES;
  const int64_t idx = (int64_t)blockIdx.x * LANES + lane;
  const int64_t at = min(idx / LPR, total - 1);
  const int d4 = (int)(idx % LPR);
  const float* po = a.ws + at * a.runs * D + d4 * 4;
  const float* ps = a.ws + total * a.runs * D + at * a.runs * 2;
  float m = -INFINITY, l = 0.f;
  float4v acc = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = way; i0 < a.runs; i0 += UNROLL * WAYS) {
    float mi[UNROLL], li[UNROLL];
    float4v v[UNROLL];
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const int i = min(i0 + j * WAYS, a.runs - 1);
      mi[j] = i0 + j * WAYS < a.runs ? ps[i * 2] : -INFINITY;
      li[j] = ps[i * 2 + 1];
      v[j] = *reinterpret_cast<const float4v*>(po + (int64_t)i * D);
    }
    float mn = m;
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) mn = fmaxf(mn, mi[j]);
    if (mn == -INFINITY) continue;  // (runs without a visible key)
    const float keep = fast_exp2(m - mn);
    l *= keep;
    acc = acc * keep;
    m = mn;
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      if (mi[j] == -INFINITY) continue;
      const float w = fast_exp2(mi[j] - m);
      l = fmaf(li[j], w, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(v[j][e], w, acc[e]);
    }
  }
  if (WAYS > 1) {
    __shared__ float4v so[256];
    __shared__ float sm[256], sl[256];
    so[threadIdx.x] = acc;
    sm[threadIdx.x] = m;
    sl[threadIdx.x] = l;
    __syncthreads();
    if (way != 0) return;
#pragma unroll
    for (int w = 1; w < WAYS; ++w) m = fmaxf(m, sm[w * LANES + lane]);
    acc = float4v{0.f, 0.f, 0.f, 0.f};
    l = 0.f;
#pragma unroll
    for (int w = 0; w < WAYS; ++w) {
      const float mw = sm[w * LANES + lane];
      const float sc = mw == -INFINITY ? 0.f : fast_exp2(mw - m);
      l = fmaf(sl[w * LANES + lane], sc, l);
      const float4v v = so[w * LANES + lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(v[e], sc, acc[e]);
    }
  }
  if (idx / LPR >= total) return;
  store_row<D>(a, (int)(at / rows / a.Hkv), (int)(at / rows % a.Hkv), (int)(at % rows), d4, m, l, acc);
}

// ---- which kernel, and in how many runs
constexpr int kFewRowsMost = 32;        // stacked rows of a KV head, up to which the kernel of few rows runs
struct CachePlan {
  int nt;       // few rows: column tiles of 16 rows (0: the tile kernel)
  int runs;
  int64_t nwg;  // workgroups per run
};
static CachePlan cache_plan(int B, int S, int Hq, int Hkv, int kv_len, int window, int sinks) {
  const int rows = S * (Hq / Hkv);
  CachePlan p;
  p.nt = rows <= kFewRowsMost ? (rows + 15) / 16 : 0;
  p.nwg = p.nt > 0 ? (int64_t)Hkv * B : (int64_t)((rows + kCacheRows - 1) / kCacheRows) * Hkv * B;
  // most keys of a row block
  const int64_t toks = p.nt > 0 ? S : (kCacheRows + Hq / Hkv - 1) / (Hq / Hkv) + 1;
  int64_t keys = kv_len;
  if (window > 0 && toks + window + sinks < keys) keys = toks + window + sinks;
  const int64_t least = p.nt > 0 ? 4 * kFewRowTile : 4 * kCacheTile;  // keys per run
  int64_t runs = 512 / p.nwg;
  if (runs > keys / least) runs = keys / least;
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
static void launch_t(const CacheAttnArgs& a, int nt, unsigned nwg, hipStream_t stream) {
  if (nt == 1) hipLaunchKernelGGL((cache_attn_few_kernel<D, FP4, 1>), dim3(nwg), dim3(256), 0, stream, a);
  else if (nt == 2) hipLaunchKernelGGL((cache_attn_few_kernel<D, FP4, 2>), dim3(nwg), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((cache_attn_kernel<D, FP4>), dim3(nwg), dim3(256), 0, stream, a);
}

template <int D>
static void launch_merge(const CacheAttnArgs& a, hipStream_t stream) {
  const int64_t lanes = (int64_t)a.B * a.S * a.Hq * (D / 4);
  if (a.runs > 8 && lanes < 256 * 256)
    hipLaunchKernelGGL((cache_merge_kernel<D, 8>), dim3((unsigned)((lanes + 31) / 32)), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((cache_merge_kernel<D, 1>), dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, stream, a);
}

int launch_cache_attention(const CacheAttnArgs& args, hipStream_t stream) {
  CacheAttnArgs a = args;
  const CachePlan p = cache_plan(a.B, a.S, a.Hq, a.Hkv, a.kv_len, a.window, a.sinks);
  const int64_t fit = a.ws != nullptr ? a.ws_bytes / run_bytes(a.B, a.S, a.Hq, a.D) : 0;
  a.runs = (int)(fit < p.runs ? (fit < 1 ? 1 : fit) : p.runs);
  const unsigned nwg = (unsigned)(p.nwg * a.runs);
  const bool fp4 = a.kc.scales != nullptr;
  if (a.D == 128) fp4 ? launch_t<128, true>(a, p.nt, nwg, stream) : launch_t<128, false>(a, p.nt, nwg, stream);
  else fp4 ? launch_t<64, true>(a, p.nt, nwg, stream) : launch_t<64, false>(a, p.nt, nwg, stream);
  if (hipGetLastError() != hipSuccess) return -1;
  if (a.runs == 1) return 0;
  if (a.D == 128) launch_merge<128>(a, stream);
  else launch_merge<64>(a, stream);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tri
