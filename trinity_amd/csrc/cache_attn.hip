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
#include <type_traits>

#include "common.h"
#include "fp4.h"
#include "launch.h"

namespace tri {

constexpr int kCacheTile = 64;       // keys
constexpr int kCacheRows = 128;      // stacked rows per workgroup, 32 a wave
// the running maximum is raised when a score exceeds it by this many powers of two: probabilities stay below 2^8, and the
// sums are rescaled rarely
constexpr float kCacheLazyMax = 8.0f;

// (divisions by what the launcher knows are multiplications: a division of integers takes forty instructions, one after the
// other, and the place of a workgroup takes four)
__device__ __forceinline__ int div_by(int n, CacheDiv d) { return (int)(__umulhi((uint32_t)n << 4, d.mul) >> d.sh); }
__device__ __forceinline__ int row_token(const CacheAttnArgs& a, int row) { return div_by(row, a.by_group); }

// offset of a key's row: row strides are less than 2^31 bytes, so that this is one product of 32 bits and not three
__device__ __forceinline__ uint64_t row_at(int key, int64_t stride) { return (uint64_t)(uint32_t)key * (uint32_t)stride; }

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

// result of a row: four channels d4 of the finished sum, divided by the softmax's, and its log-sum-exp.  Padding, the rows without
// a visible key, gets zeros and -inf, chosen and not multiplied: its sum is zero times the rows of V that others of the block see,
// NaN where one of these holds no number.  (A row whose scores are all -inf has a sum of zero, too: it is NaN.)
template <int D>
__device__ __forceinline__ void store_row(const CacheAttnArgs& a, int b, int hk, int row, bool padding, int d4, float m, float l, float4v acc) {
  const int tok = row_token(a, row), head = hk * a.group + row - tok * a.group;
  const float inv = 1.0f / l;
  half4v hv;
#pragma unroll
  for (int e = 0; e < 4; ++e) hv[e] = (half_t)(acc[e] * inv);
  *reinterpret_cast<half4v*>(a.out + ((int64_t)b * a.S + tok) * a.ldo + (int64_t)head * D + d4 * 4) = padding ? half4v{} : hv;
  if (a.lse != nullptr && d4 == 0)
    a.lse[((int64_t)b * a.Hq + head) * a.S + tok] = padding || l == 0.f ? -INFINITY : (m + fast_log2(l)) * kLn2;
}

// ... or, of several runs, its partial result: unnormalised O [b][hk][row][run][D], then (max, sum) [b][hk][row][run][2].  Padding
// has the sum -1, which the merge knows it by.
template <int D>
__device__ __forceinline__ void finish_row(const CacheAttnArgs& a, int b, int hk, int row, bool padding, int run, int d4, float m, float l, float4v acc) {
  if (a.runs == 1) {
    store_row<D>(a, b, hk, row, padding, d4, m, l, acc);
    return;
  }
  const int64_t rows = a.rows, at = (((int64_t)b * a.Hkv + hk) * rows + row) * a.runs + run;
  *reinterpret_cast<float4v*>(a.ws + at * D + d4 * 4) = acc;
  if (d4 == 0) {
    float* ps = a.ws + (int64_t)a.B * a.Hkv * rows * a.runs * D + at * 2;
    ps[0] = m;
    ps[1] = padding ? -1.f : l;
  }
}

template <int D>
struct CacheLds {
  static constexpr int CPR = D / 8;  // 16-byte chunks per row; chunk c of row r at slot c ^ fk(r) (K), c ^ fv(r) (V)
  static constexpr int HALFS = kCacheTile * D;
  __device__ static __forceinline__ int fk(int row) { return D == 128 ? (row & 15) : ((row >> 1) & 7); }
  __device__ static __forceinline__ int fv(int row) { return D == 128 ? ((row & 3) << 2) : (((row >> 1) & 1) << 2); }
};

// Workgroups go to the eight XCDs in turn, each with an L2 of its own: the row blocks of one KV head, which read the same
// keys, stay on one XCD.  Per XCD the latest row blocks, which see most, come first.
__device__ __forceinline__ void cache_wg_map(const CacheAttnArgs& a, int id, int& b, int& hk, int& rb, int& run) {
  const int heads = a.B * a.Hkv;
  int bh;
  if (heads % 8 == 0) {
    const int s = id >> 3, hx = heads >> 3;  // (by_heads: hx)
    id = div_by(s, a.by_heads);
    bh = (s - id * hx) * 8 + (int)(blockIdx.x & 7);  // (an XCD has heads of all sequences, the long ones and the short)
  } else {
    id = div_by(id, a.by_heads);
    bh = (int)blockIdx.x - id * heads;
  }
  const int back = a.runs == 1 ? id : div_by(id, a.by_runs);
  rb = a.nrb - 1 - back;
  run = id - back * a.runs;
  b = a.B == 1 ? 0 : div_by(bh, a.by_hkv);
  hk = bh - b * a.Hkv;
}

// ---------------------------------------------------------------------------------------------------- many rows, 128-wide heads
// Four waves of 32 rows walk tiles of 64 keys.  Inside each wave the matrix pipe works on S^T of tile t + 1 while the
// probabilities of tile t are computed, and on O^T of tile t while the maximum of tile t + 1 is found; a slot below holds
// the MFMAs of one K or V fragment, the LDS read of a fragment PD slots ahead, and its share of the vector arithmetic.
// Step t reads K(t + 1) and V(t), so K tiles travel two steps ahead and V tiles one; each has two buffers.  16-bit tiles go
// from memory to LDS directly.  4-bit tiles are a 16-byte block per thread: it travels through registers, a step longer,
// and is turned into 16 bits in the slots of O^T, which have little else to do.
//
// KW = 2: eight waves, the four row groups twice, on every other tile each with buffers of their own; they merge through
// LDS at the end.  For calls with one workgroup a CU at most, whose time is the chain of its tiles.
//
// For 128-wide heads.  What bounds it: the board's power limit, as the other attention kernels (a prompt of 4096 tokens over a
// 4-bit cache 133 us, 1.03 PFLOP/s, level with 16-bit rows: the conversion is hidden; matrix pipe busy 45 % of the time at the
// clock that the limit leaves), and beside it some 9 us a round of workgroups for their first loads, the first tile's scores and
// the stores (8192 tokens in a window of 1024, four rounds of 17 tiles, 160 us).  Measured and level: fixed offsets in place of
// an address per row, cheaper masks, workgroups that start apart.  Slower: a second copy of the step without the product after
// the last tile (the registers spill, 33 to 57 %), a branch around each of its instructions (level, 4-bit 2 to 11 %), three waves
// a SIMD on tiles of 32 keys as below for 64-wide heads (11 % to 30 %; 1.6 % faster for the window of 1024 in 16 bits).
struct TilePipe {
  static constexpr int D = 128;
  static constexpr int KSTEPS = D / 16, DT = D / 32;
  static constexpr int NKF = 2 * KSTEPS, NVF = 4 * DT;  // K / V fragments (MFMAs) per tile
  static constexpr int GPS = 16 / NKF, EPS = 32 / NVF;  // pairs of probabilities per S^T slot; scores per O^T slot
  static constexpr int PD = 3, RING = 4;
};

// The end of a workgroup's rows: the states of the key ways merged, and the result stored.
template <int D, int KW>
__device__ __forceinline__ void tile_finish(const CacheAttnArgs& a, half_t* lds_all, int b, int hk, int run, int w0, int pos, int wave, int lane,
                                            int kway, float m, float l, float16v (&o)[D / 32]) {
  constexpr int DT = D / 32, CPR = D / 8;
  const int l32 = lane & 31, g = lane >> 5, group = a.group, rows = a.rows;
  const int row = w0 + l32, rowc = min(row, rows - 1), tok = row_token(a, rowc), head = hk * group + rowc - tok * group;
  // ---- more ways: the others hand their state over, lane for lane, and leave
  constexpr int REG = DT * 16 + 2;
  float* const mg = reinterpret_cast<float*>(lds_all) + wave * REG * 64 + lane;
  if constexpr (KW == 2) {
    __syncthreads();  // (every wave is done with the tiles)
    if (kway == 1) {
      mg[0] = m;
      mg[64] = l;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) mg[(2 + dt * 16 + e) * 64] = o[dt][e];
    }
    __syncthreads();
    if (kway == 1) return;
    const float m1 = mg[0], mn = fmaxf(m, m1);
    const float a0 = m == -INFINITY ? 0.f : fast_exp2(m - mn), a1 = m1 == -INFINITY ? 0.f : fast_exp2(m1 - mn);
    m = mn;
    l = l * a0 + mg[64] * a1;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[dt][e] = o[dt][e] * a0 + mg[(2 + dt * 16 + e) * 64] * a1;
  }

  l = pair_sum(l);
  if (a.runs == 1) {
    // ---- a lane has sixteen pieces of 8 bytes of its row: stored as they are, every store instruction touches 32 lines, so
    // each wave turns its rows around in LDS and stores whole ones, 16 bytes a lane
    constexpr int LDO = D + 8;
    static_assert(32 * LDO * 2 <= REG * 64 * 4, "two ways: in the place of the state that only this wave has read");
    half_t* const stage = KW == 2 ? reinterpret_cast<half_t*>(mg - lane) : lds_all + wave * 32 * LDO;
    if (KW == 1) __syncthreads();  // (every wave is done with the tiles)
    float inv = 1.0f / l;
    if (__builtin_amdgcn_ballot_w64(pos < 0) != 0) {  // wave-uniform; padding (see store_row), which most calls have none of
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] = pos < 0 ? 0.f : o[dt][e];
      inv = pos < 0 ? 0.f : inv;
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        half4v hv;
#pragma unroll
        for (int e = 0; e < 4; ++e) hv[e] = (half_t)(o[dt][rq * 4 + e] * inv);
        *reinterpret_cast<half4v*>(stage + l32 * LDO + dt * 32 + rq * 8 + g * 4) = hv;
      }
    if (a.lse != nullptr && g == 0 && row < rows)
      a.lse[((int64_t)b * a.Hq + head) * a.S + tok] = l == 0.f ? -INFINITY : (m + fast_log2(l)) * kLn2;
    constexpr int RPI = 64 / CPR;  // rows per store instruction
#pragma unroll
    for (int i = 0; i < 32 / RPI; ++i) {
      const int r = i * RPI + lane / CPR, c = lane % CPR;
      const half8v v = *reinterpret_cast<const half8v*>(stage + r * LDO + c * 8);
      if (w0 + r < rows) {
        const int tk = row_token(a, w0 + r), hd = hk * group + w0 + r - tk * group;
        *reinterpret_cast<half8v*>(a.out + ((int64_t)b * a.S + tk) * a.ldo + (int64_t)hd * D + c * 8) = v;
      }
    }
    return;
  }
  if (row >= rows) return;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq)
      finish_row<D>(a, b, hk, row, pos < 0, run, dt * 8 + rq * 2 + g, m, l,
                    float4v{o[dt][rq * 4], o[dt][rq * 4 + 1], o[dt][rq * 4 + 2], o[dt][rq * 4 + 3]});
}

template <bool FP4, int KW>
__device__ __forceinline__ void cache_attn_tile_body(const CacheAttnArgs& a, half_t* lds_all, const half_t* __restrict__ qglob) {
  // (qglob = a.q.  Inlined, every LDS access of this function carries "does not alias q", and an LDS read with alias
  // information is not made to wait for the loads to LDS in flight; barriers and explicit waits order those here.)
  using P = TilePipe;
  constexpr int D = P::D;
  using L = CacheLds<D>;
  constexpr int KSTEPS = P::KSTEPS, DT = P::DT, NKF = P::NKF, NVF = P::NVF, GPS = P::GPS, EPS = P::EPS, PD = P::PD, RING = P::RING;
  constexpr int CPR = L::CPR;
  const int t = threadIdx.x & 255, lane = t & 63;  // of the way's four waves
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int kway = KW == 2 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0;
  half_t* const lds = lds_all + kway * 4 * L::HALFS;
  const int l32 = lane & 31, g = lane >> 5;
  const int group = a.group, rows = a.rows;
  int b, hk, rb, run;
  cache_wg_map(a, (int)blockIdx.x, b, hk, rb, run);
  const int r0 = rb * kCacheRows, w0 = r0 + wave * 32;
  const KeyList kl = key_list(a, b, row_token(a, r0), row_token(a, min(r0 + kCacheRows, rows) - 1));
  const int ntiles = (kl.n + kCacheTile - 1) / kCacheTile;
  const int per = div_by(ntiles + a.runs - 1, a.by_runs), tile0 = min(run * per, ntiles);
  const int tile1 = min(tile0 + per, ntiles), nsteps = (tile1 - tile0 + KW - 1) / KW;
  auto tile_of = [&](int step) { return tile0 + step * KW + kway; };  // (may lie past the last one)

  const int row = w0 + l32, rowc = min(row, rows - 1);
  const int tok = row_token(a, rowc), head = hk * group + rowc - tok * group;
  const int pos = kl.len - a.S + tok;
  // positions of the wave's rows (it may have none)
  const int pos0 = kl.len - a.S + row_token(a, min(w0, rows - 1)), pos1 = kl.len - a.S + row_token(a, min(w0 + 31, rows - 1));
  // the steps that hold a key some row of the wave sees are [0, nact)
  const int seen = a.causal ? min(kl.n, pos1 + 1 - kl.gap) : kl.n;  // ... of the list
  const int nact = w0 >= rows ? 0 : max(0, (min(tile1, (seen + kCacheTile - 1) / kCacheTile) - tile0 - kway + KW - 1) / KW);

  half8v qf[KSTEPS];
  const half_t* qp = qglob + ((int64_t)b * a.S + tok) * a.ldq + (int64_t)head * D + g * 8;
#pragma unroll
  for (int ks = 0; ks < KSTEPS; ++ks) qf[ks] = *reinterpret_cast<const half8v*>(qp + ks * 16);

  // ---- tiles: a thread's pieces of 16 bytes (16-bit: chunks, 4-bit: blocks) and the row of the tile each is of
  constexpr int PPR = FP4 ? D / 32 : CPR;              // pieces per row
  constexpr int NP = kCacheTile * PPR / 256;           // per thread
  constexpr int ES = FP4 ? 1 : 2;
  const uint8_t* const kbase = static_cast<const uint8_t*>(a.kc.p) + (b * a.kc.sb + hk * a.kc.sh) * ES;
  const uint8_t* const vbase = static_cast<const uint8_t*>(a.vc.p) + (b * a.vc.sb + hk * a.vc.sh) * ES;
  const uint8_t* const kxbase = FP4 ? a.kc.scales + b * a.kc.xb + hk * a.kc.xh : nullptr;
  const uint8_t* const vxbase = FP4 ? a.vc.scales + b * a.vc.xb + hk * a.vc.xh : nullptr;
  const int64_t ksr = a.kc.sr * ES, vsr = a.vc.sr * ES;
  half_t *const kt = lds, *const vt = lds + 2 * L::HALFS;
  // key of row r of a tile (past the last key: the last one again, whose scores are masked)
  auto key_of = [&](int step, int r) {
    const int li = min(tile_of(step) * kCacheTile + r, kl.n - 1);
    return li + (li < kl.sinks ? 0 : kl.gap);
  };
  auto load16 = [&](int step, bool isv, int buf) {  // 16-bit: to LDS, 1 KB an instruction
    half_t* const dst = (isv ? vt : kt) + buf * L::HALFS;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int p = i * 256 + t, r = p / CPR, slot = p % CPR;
      const uint8_t* src = (isv ? vbase : kbase) + row_at(key_of(step, r), isv ? vsr : ksr) + (slot ^ (isv ? L::fv(r) : L::fk(r))) * 16;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(uintptr_t)src,
                                       (TRI_LDS void*)(dst + (i * 4 + wave) * 512), 16, 0, 0);
    }
  };
  uint4v kraw, vraw;
  uint32_t kxraw = 0, vxraw = 0;
  const int pr = t / PPR, pc = t % PPR;  // 4-bit: the thread's row and block
  auto fetch4 = [&](int step, bool isv) {
    const int key = key_of(step, pr);
    if (isv) {
      vraw = *reinterpret_cast<const uint4v*>(vbase + row_at(key, vsr) + pc * 16);
      vxraw = vxbase[row_at(key, a.vc.xr) + pc];
    } else {
      kraw = *reinterpret_cast<const uint4v*>(kbase + row_at(key, ksr) + pc * 16);
      kxraw = kxbase[row_at(key, a.kc.xr) + pc];
    }
  };
  auto commit4 = [&](int step, bool isv, int j) {  // chunk j of the block
    half_t* const dst = (isv ? vt : kt) + (step & 1) * L::HALFS;
    *reinterpret_cast<half8v*>(dst + pr * D + (((pc * 4 + j) ^ (isv ? L::fv(pr) : L::fk(pr))) << 3)) =
        fp4x8_to_half8(isv ? vraw[j] : kraw[j], fp4_scale(isv ? vxraw : kxraw));
  };

  // ---- fragments: K fragment j = (16 channels j / 2, key half j % 2), V fragment v = (key half, key quarter, 32 channels)
  int kbyte[KSTEPS], vbyte[DT];
#pragma unroll
  for (int ks = 0; ks < KSTEPS; ++ks) {
    kbyte[ks] = (l32 * D + (((ks * 2 + g) ^ L::fk(l32)) << 3)) * 2;
    asm volatile("" : "+v"(kbyte[ks]));
  }
  const int j4 = (lane & 15) >> 2;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    const int chunk = dt * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    vbyte[dt] = (int)(uint32_t)(uintptr_t)lds + (2 * L::HALFS + (4 * g + j4) * D + ((chunk ^ L::fv(j4)) << 3) + (lane & 1) * 4) * 2;
    asm volatile("" : "+v"(vbyte[dt]));
  }
  const char* const ldsb = reinterpret_cast<const char*>(lds);
  auto read_kf = [&](int par, int j) {
    return *reinterpret_cast<const half8v*>(ldsb + kbyte[j / 2] + (par * L::HALFS + (j % 2) * 32 * D) * 2);
  };
  auto read_vf = [&](int par, int v) {
    TRI_LDS char* vp = (TRI_LDS char*)(uintptr_t)(uint32_t)vbyte[v % DT] +
                       (par * L::HALFS + ((v / (2 * DT)) * 32 + ((v / DT) % 2) * 16) * D) * 2;
    const short4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TRI_LDS short4s*)vp);
    const short4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TRI_LDS short4s*)(vp + 8 * D * 2));
    half4v hl, hh;
    __builtin_memcpy(&hl, &lo, 8);
    __builtin_memcpy(&hh, &hi, 8);
    return cat8(hl, hh);
  };

  const float c2 = a.scale * kLog2e;
  float m = -INFINITY, l = 0.f;
  float16v o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;

  // Masks in terms of list indices: visible are those up to `last`, and of them those from `from` on or below a.sinks (in
  // front of a gap all of these are sinks).  `last` differs between the wave's rows by less than 32, `from` as much.
  const int last = pos < 0 ? -1 : (a.causal ? pos - kl.gap : kl.n - 1), from = a.window > 0 ? pos - a.window + 1 - kl.gap : 0;
  auto need_mask = [&](int step) {
    const int li0 = tile_of(step) * kCacheTile, li1 = li0 + kCacheTile - 1;
    return li1 >= kl.n || pos0 < 0 || (a.causal && li1 + kl.gap > pos0) || (a.window > 0 && li0 + kl.gap <= pos1 - a.window && li1 >= a.sinks);
  };
  auto apply_mask = [&](float16v (&s)[2], int step) {
    const int base = tile_of(step) * kCacheTile + g * 4;  // the lane's scores are of indices base + (0 to 3) + 8 i
    const int end = min(last, kl.n - 1) - base;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (mt * 32 + (r >> 2) * 8 + (r & 3) > end) s[mt][r] = -INFINITY;
    const int li0 = tile_of(step) * kCacheTile;
    if (a.window > 0 && li0 + kl.gap <= pos1 - a.window) {  // wave-uniform: the window of some row begins in the tile, or behind it
      asm volatile("");
      const int begin = from - base, sinks = a.sinks - base;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int c = mt * 32 + (r >> 2) * 8 + (r & 3);
          if (c < begin && c >= sinks) s[mt][r] = -INFINITY;
        }
    }
  };
  auto tile_max = [&](const float16v (&s)[2]) {
    float mx = -INFINITY;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[mt][r]);
    return mx;
  };
  auto raise = [&](float mx) {  // mx: the lane's maximum of the raw scores
    mx = pair_max(mx) * c2;
    if (__builtin_amdgcn_ballot_w64(mx > m + kCacheLazyMax) != 0) {  // wave-uniform
      const float mnew = fmaxf(m, mx);
      const float alpha = mnew == -INFINITY ? 1.0f : fast_exp2(m - mnew);
      m = mnew;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] = o[dt] * alpha;
    }
  };
  auto zero = [&](float16v (&s)[2]) {
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[mt][r] = 0.f;
  };
  // probabilities (two keys) of group gi, rounded to nearest - half the error of cutting them off -, their sum before that
  half8v pf[2][2];
  float sum, nm;
  auto softmax_pair = [&](const float16v (&s)[2], int gi) {
    const int mt = gi / 8, hh = (gi / 4) % 2, e = (gi % 4) * 2;
    const float p0 = fast_exp2(fmaf(s[mt][hh * 8 + e], c2, nm));
    const float p1 = fast_exp2(fmaf(s[mt][hh * 8 + e + 1], c2, nm));
    sum += p0 + p1;
    pf[mt][hh][e] = (half_t)p0;
    pf[mt][hh][e + 1] = (half_t)p1;
  };

  // this wave's share of the tiles is in LDS - 4-bit: written, lgkmcnt(0); 16-bit: landed, vmcnt(0) - and everybody's
  auto meet = [&]() __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
    if constexpr (FP4) __builtin_amdgcn_s_waitcnt(0xC07F);
    else __builtin_amdgcn_s_waitcnt(0x0F70);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");  // (to the compiler the barrier is no memory access)
  };

  half8v fr[RING];
  // One step.  cur: S^T of its tile, masked, its maximum folded into m; next: receives S^T of the next tile.
  auto step = [&](int st, auto parc, float16v (&cur)[2], float16v (&next)[2]) __attribute__((always_inline)) {
    constexpr int PAR = decltype(parc)::value;
    meet();  // K(st + 1) and V(st) are there, K(st) and V(st - 1) retired
    if constexpr (!FP4) {
      if (st + 2 < nsteps) load16(st + 2, false, PAR);
      if (st + 1 < nsteps) load16(st + 1, true, PAR ^ 1);
    }
    auto commit_all = [&]() {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        commit4(st, false, j);      // K(st + 2): the buffer of K(st)
        commit4(st + 1, true, j);
      }
    };
    if (st < nact) {
      // ---- S^T(st + 1) = K . Q^T beside the probabilities of tile st (after the wave's last tile the product is not used)
#pragma unroll
      for (int j = 0; j < PD; ++j) fr[j] = read_kf(PAR ^ 1, j);
      zero(next);
      sum = 0.f;
      nm = m == -INFINITY ? 0.f : -m;
      __builtin_amdgcn_s_setprio(1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < NKF; ++j) {
        if (j + PD < NKF) fr[(j + PD) % RING] = read_kf(PAR ^ 1, j + PD);
        else fr[(j + PD) % RING] = read_vf(PAR, j + PD - NKF);
        next[j % 2] = mfma32(fr[j % RING], qf[j / 2], next[j % 2]);
#pragma unroll
        for (int x = 0; x < GPS; ++x) softmax_pair(cur, j * GPS + x);
        __builtin_amdgcn_sched_barrier(0);
      }
      // ---- O^T += V^T . P^T of tile st beside the maximum of tile st + 1
      float mx = -INFINITY;
      __builtin_amdgcn_s_setprio(0);
#pragma unroll
      for (int v = 0; v < NVF; ++v) {
        if (v + PD < NVF) fr[(NKF + v + PD) % RING] = read_vf(PAR, v + PD);
        o[v % DT] = mfma32(fr[(NKF + v) % RING], pf[v / (2 * DT)][(v / DT) % 2], o[v % DT]);
#pragma unroll
        for (int x = 0; x < EPS; ++x) {
          const int idx = v * EPS + x;
          mx = fmaxf(mx, next[idx / 16][idx % 16]);
        }
        if constexpr (FP4) {
          if (v % (NVF / 8) == 0) {
            const int j = v / (NVF / 8);
            commit4(st + (j % 2), j % 2 != 0, j / 2);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      l += sum;
      if (st + 1 < nact) {
        if (need_mask(st + 1)) {  // wave-uniform
          asm volatile("");
          apply_mask(next, st + 1);
          mx = tile_max(next);
        }
        raise(mx);
      }
    } else if constexpr (FP4) {
      commit_all();
    }
    if constexpr (FP4) {  // (past the last step: its last keys again)
      fetch4(st + 3, false);
      fetch4(st + 2, true);
    }
  };

  if (nsteps > 0) {
    // ---- prologue: K(0), K(1), V(0); S^T of tile 0
    if constexpr (FP4) {
      // (all five on their way at once: one trip to memory)
      fetch4(0, false);
      const uint4v k0 = kraw;
      const uint32_t kx0 = kxraw;
      fetch4(0, true);
      const uint4v v0 = vraw;
      const uint32_t vx0 = vxraw;
      fetch4(1, false);
      const uint4v k1 = kraw;
      const uint32_t kx1 = kxraw;
      fetch4(2, false);
      const uint4v k2 = kraw;
      const uint32_t kx2 = kxraw;
      fetch4(1, true);
      const uint4v v1 = vraw;
      const uint32_t vx1 = vxraw;
      kraw = k0; kxraw = kx0; vraw = v0; vxraw = vx0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        commit4(0, false, j);
        commit4(0, true, j);
      }
      kraw = k1; kxraw = kx1;
#pragma unroll
      for (int j = 0; j < 4; ++j) commit4(1, false, j);
      kraw = k2; kxraw = kx2; vraw = v1; vxraw = vx1;
    } else {
      load16(0, false, 0);
      load16(0, true, 0);
      load16(min(1, nsteps - 1), false, 1);  // (not under a condition: the wait below counts it)
    }
    if constexpr (FP4) {
      meet();
    } else {  // K(0) is there, V(0) and K(1) may still be on their way
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0x0F70 | (2 * NP));
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    }
    float16v sa[2], sb[2];
    if (0 < nact) {
      zero(sa);
      half8v kf[NKF];  // (all reads on their way before the first product waits for one)
#pragma unroll
      for (int j = 0; j < NKF; ++j) kf[j] = read_kf(0, j);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < NKF; ++j) sa[j % 2] = mfma32(kf[j], qf[j / 2], sa[j % 2]);
      if (need_mask(0)) {
        asm volatile("");
        apply_mask(sa, 0);
      }
      raise(tile_max(sa));
    }
    for (int st = 0; st < nsteps; st += 2) {
      step(st, std::integral_constant<int, 0>{}, sa, sb);
      if (st + 1 < nsteps) step(st + 1, std::integral_constant<int, 1>{}, sb, sa);
    }
  }

  tile_finish<D, KW>(a, lds_all, b, hk, run, w0, pos, wave, lane, kway, m, l, o);
}

template <bool FP4, int KW>
__global__ __launch_bounds__(256 * KW) __attribute__((amdgpu_waves_per_eu(2, 2))) void cache_attn_tile_kernel(CacheAttnArgs a) {
  __shared__ __attribute__((aligned(16))) half_t lds[KW * 4 * CacheLds<TilePipe::D>::HALFS];
  cache_attn_tile_body<FP4, KW>(a, lds, a.q);
}

// ---------------------------------------------------------------------------------------------------- many rows, 64-wide heads
// The same tiles, two buffers of each, K and V one step ahead, and a step without overlap inside a wave: scores of 32 keys, their
// probabilities, their product with V.  A 64-wide head has half the matrix work per probability, so that what a SIMD lacks is not a
// schedule but other waves: at 32 keys at a time a wave takes 114 registers (4-bit 122), and four of them, of four workgroups, share
// a SIMD.  Halves of a tile that no row of the wave sees are skipped.  Against the pipelined step above with two waves a SIMD: two
// prompts of 1000 tokens, 71 heads, in a window of 256 25.3 -> 20.0 us, 4096 in one of 1024 109.3 -> 95.8, one token against 8000 keys 9.6
// -> 8.9; 64 keys at a time (119 registers) 22.8; three waves a SIMD 24.5; five spill.  Level: the waves' priority raised for the
// products.  4-bit tiles: a thread has one block, of K or of V.
//
// KW = 2: as above.
template <bool FP4, int KW>
__device__ __forceinline__ void cache_attn_waves_body(const CacheAttnArgs& a, half_t* lds_all, const half_t* __restrict__ qglob) {
  constexpr int D = 64;
  using L = CacheLds<D>;  // (qglob = a.q, as above)
  constexpr int KSTEPS = D / 16, DT = D / 32, CPR = D / 8;
  constexpr int HALFS = L::HALFS;
  const int t = threadIdx.x & 255, lane = t & 63;  // of the way's four waves
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int kway = KW == 2 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0;
  half_t* const lds = lds_all + kway * 4 * HALFS;
  const int l32 = lane & 31, g = lane >> 5;
  const int group = a.group, rows = a.rows;
  int b, hk, rb, run;
  cache_wg_map(a, (int)blockIdx.x, b, hk, rb, run);
  const int r0 = rb * kCacheRows, w0 = r0 + wave * 32;
  const KeyList kl = key_list(a, b, row_token(a, r0), row_token(a, min(r0 + kCacheRows, rows) - 1));
  const int ntiles = (kl.n + kCacheTile - 1) / kCacheTile;
  const int per = div_by(ntiles + a.runs - 1, a.by_runs), tile0 = min(run * per, ntiles);
  const int tile1 = min(tile0 + per, ntiles), nsteps = (tile1 - tile0 + KW - 1) / KW;
  auto tile_of = [&](int step) { return tile0 + step * KW + kway; };  // (may lie past the last one)

  const int row = w0 + l32, rowc = min(row, rows - 1);
  const int tok = row_token(a, rowc), head = hk * group + rowc - tok * group;
  const int pos = kl.len - a.S + tok;
  // positions of the wave's rows (it may have none)
  const int pos0 = kl.len - a.S + row_token(a, min(w0, rows - 1)), pos1 = kl.len - a.S + row_token(a, min(w0 + 31, rows - 1));
  // the wave's rows see list indices below this
  const int seen = w0 >= rows ? 0 : min(tile1 * kCacheTile, a.causal ? min(kl.n, pos1 + 1 - kl.gap) : kl.n);

  half8v qf[KSTEPS];
  const half_t* qp = qglob + ((int64_t)b * a.S + tok) * a.ldq + (int64_t)head * D + g * 8;
#pragma unroll
  for (int ks = 0; ks < KSTEPS; ++ks) qf[ks] = *reinterpret_cast<const half8v*>(qp + ks * 16);

  constexpr int ES = FP4 ? 1 : 2;
  const uint8_t* const kbase = static_cast<const uint8_t*>(a.kc.p) + (b * a.kc.sb + hk * a.kc.sh) * ES;
  const uint8_t* const vbase = static_cast<const uint8_t*>(a.vc.p) + (b * a.vc.sb + hk * a.vc.sh) * ES;
  const int64_t ksr = a.kc.sr * ES, vsr = a.vc.sr * ES;
  half_t *const kt = lds, *const vt = lds + 2 * HALFS;
  // key of row r of a tile (past the last key: the last one again, whose scores are masked)
  auto key_of = [&](int step, int r) {
    const int li = min(tile_of(step) * kCacheTile + r, kl.n - 1);
    return li + (li < kl.sinks ? 0 : kl.gap);
  };
  auto load16 = [&](int step, bool isv, int buf) {  // 16-bit: to LDS, 1 KB an instruction
    half_t* const dst = (isv ? vt : kt) + buf * HALFS;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int p = i * 256 + t, r = p / CPR, slot = p % CPR;
      const uint8_t* src = (isv ? vbase : kbase) + row_at(key_of(step, r), isv ? vsr : ksr) + (slot ^ (isv ? L::fv(r) : L::fk(r))) * 16;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(uintptr_t)src,
                                       (TRI_LDS void*)(dst + (i * 4 + wave) * 512), 16, 0, 0);
    }
  };
  // 4-bit: a block per thread, of K in the first two waves, of V in the others
  constexpr int BPR = D / 32;
  const bool own_v = wave >= 2;
  const int pr = t % 128 / BPR, pc = t % BPR;
  const uint8_t* const own = own_v ? vbase : kbase;
  const uint8_t* const own_x = FP4 ? (own_v ? a.vc.scales + b * a.vc.xb + hk * a.vc.xh : a.kc.scales + b * a.kc.xb + hk * a.kc.xh) : nullptr;
  const int64_t own_sr = own_v ? vsr : ksr, own_xr = own_v ? a.vc.xr : a.kc.xr;
  const int own_at = (own_v ? 2 * HALFS : 0) + pr * D, own_f = own_v ? L::fv(pr) : L::fk(pr);
  uint4v raw;
  uint32_t xraw = 0;
  auto fetch4 = [&](int step) {
    const int key = key_of(step, pr);
    raw = *reinterpret_cast<const uint4v*>(own + row_at(key, own_sr) + pc * 16);
    xraw = own_x[row_at(key, own_xr) + pc];
  };
  auto commit4 = [&](int buf) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<half8v*>(lds + own_at + buf * HALFS + (((pc * 4 + j) ^ own_f) << 3)) = fp4x8_to_half8(raw[j], fp4_scale(xraw));
  };

  int kbyte[KSTEPS], vbyte[DT];
#pragma unroll
  for (int ks = 0; ks < KSTEPS; ++ks) {
    kbyte[ks] = (l32 * D + (((ks * 2 + g) ^ L::fk(l32)) << 3)) * 2;
    asm volatile("" : "+v"(kbyte[ks]));
  }
  const int j4 = (lane & 15) >> 2;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    const int chunk = dt * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    vbyte[dt] = (int)(uint32_t)(uintptr_t)lds + (2 * HALFS + (4 * g + j4) * D + ((chunk ^ L::fv(j4)) << 3) + (lane & 1) * 4) * 2;
    asm volatile("" : "+v"(vbyte[dt]));
  }
  const char* const ldsb = reinterpret_cast<const char*>(lds);
  auto read_kf = [&](int par, int hf, int ks) {
    return *reinterpret_cast<const half8v*>(ldsb + kbyte[ks] + (par * HALFS + hf * 32 * D) * 2);
  };
  auto read_vf = [&](int par, int hf, int v) {  // 16 keys v / DT, 32 channels v % DT
    TRI_LDS char* vp = (TRI_LDS char*)(uintptr_t)(uint32_t)vbyte[v % DT] + (par * HALFS + (hf * 32 + (v / DT) * 16) * D) * 2;
    const short4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TRI_LDS short4s*)vp);
    const short4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TRI_LDS short4s*)(vp + 8 * D * 2));
    half4v hl, hh;
    __builtin_memcpy(&hl, &lo, 8);
    __builtin_memcpy(&hh, &hi, 8);
    return cat8(hl, hh);
  };

  const float c2 = a.scale * kLog2e;
  float m = -INFINITY, l = 0.f;
  float16v o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
  // Masks in terms of list indices: visible are those up to `last`, and of them those from `from` on or below a.sinks (in
  // front of a gap all of these are sinks).
  const int last = pos < 0 ? -1 : (a.causal ? min(pos - kl.gap, kl.n - 1) : kl.n - 1), from = a.window > 0 ? pos - a.window + 1 - kl.gap : 0;

  auto step = [&](int st, auto parc) __attribute__((always_inline)) {
    constexpr int PAR = decltype(parc)::value;
    // this wave's share of the tiles is in LDS - 4-bit: written, lgkmcnt(0); 16-bit: landed, vmcnt(0) - and everybody's
    asm volatile("" ::: "memory");
    if constexpr (FP4) __builtin_amdgcn_s_waitcnt(0xC07F);
    else __builtin_amdgcn_s_waitcnt(0x0F70);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if constexpr (!FP4) {
      if (st + 1 < nsteps) {
        load16(st + 1, false, PAR ^ 1);
        load16(st + 1, true, PAR ^ 1);
      }
    }
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int li0 = tile_of(st) * kCacheTile + hf * 32, li1 = li0 + 31;
      if (li0 >= seen) break;  // wave-uniform
      float16v s;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.f;
      half8v kf[KSTEPS];
#pragma unroll
      for (int j = 0; j < KSTEPS; ++j) kf[j] = read_kf(PAR, hf, j);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < KSTEPS; ++j) s = mfma32(kf[j], qf[j], s);
      half8v vf[2 * DT];
#pragma unroll
      for (int v = 0; v < 2 * DT; ++v) vf[v] = read_vf(PAR, hf, v);
      __builtin_amdgcn_sched_barrier(0);
      const int base = li0 + g * 4;  // the lane's scores are of indices base + (0 to 3) + 8 i
      if (li1 >= kl.n || pos0 < 0 || (a.causal && li1 + kl.gap > pos0)) {  // wave-uniform
        asm volatile("");
        const int end = last - base;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if ((r >> 2) * 8 + (r & 3) > end) s[r] = -INFINITY;
      }
      if (a.window > 0 && li0 + kl.gap <= pos1 - a.window && li1 >= a.sinks) {  // ... the window of some row begins here, or behind it
        asm volatile("");
        const int begin = from - base, sinks = a.sinks - base;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int c = (r >> 2) * 8 + (r & 3);
          if (c < begin && c >= sinks) s[r] = -INFINITY;
        }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[r]);
      mx = pair_max(mx) * c2;
      if (__builtin_amdgcn_ballot_w64(mx > m + kCacheLazyMax) != 0) {  // wave-uniform
        const float mnew = fmaxf(m, mx);
        const float alpha = mnew == -INFINITY ? 1.0f : fast_exp2(m - mnew);
        m = mnew;
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = o[dt] * alpha;
      }
      const float nm = m == -INFINITY ? 0.f : -m;
      half8v pf[2];
      float sum = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = fast_exp2(fmaf(s[r], c2, nm));
        sum += p;
        pf[r / 8][r % 8] = (half_t)p;
      }
      l += sum;
#pragma unroll
      for (int v = 0; v < 2 * DT; ++v) o[v % DT] = mfma32(vf[v], pf[v / DT], o[v % DT]);
    }
    if constexpr (FP4) {
      commit4(PAR ^ 1);
      fetch4(st + 2);  // (past the last step: its last keys again)
    }
  };

  if (nsteps > 0) {
    if constexpr (FP4) {
      fetch4(0);
      const uint4v r0v = raw;
      const uint32_t x0 = xraw;
      fetch4(1);
      const uint4v r1v = raw;
      const uint32_t x1 = xraw;
      raw = r0v; xraw = x0;
      commit4(0);
      raw = r1v; xraw = x1;
    } else {
      load16(0, false, 0);
      load16(0, true, 0);
    }
    for (int st = 0; st < nsteps; st += 2) {
      step(st, std::integral_constant<int, 0>{});
      if (st + 1 < nsteps) step(st + 1, std::integral_constant<int, 1>{});
    }
  }
  tile_finish<D, KW>(a, lds_all, b, hk, run, w0, pos, wave, lane, kway, m, l, o);
}

template <bool FP4, int KW>
__global__ __launch_bounds__(256 * KW) __attribute__((amdgpu_waves_per_eu(4, 4))) void cache_attn_waves_kernel(CacheAttnArgs a) {
  __shared__ __attribute__((aligned(16))) half_t lds[KW * 4 * CacheLds<64>::HALFS];
  cache_attn_waves_body<FP4, KW>(a, lds, a.q);
}

// ---------------------------------------------------------------------------------------------------- few rows
// At most 16 * NT stacked rows of a KV head: a call is bound by reading the keys and values once.  Every wave walks tiles
// of 32 keys of its own - no barrier until the waves of a workgroup merge - with the next tile's loads in flight.  K goes
// from memory straight into the registers that the matrix instructions want: a lane holds D / 4 channels of one key, in
// 4 bits one block with one scale (the order of the channels in the product is free, as long as q has the same).  V goes
// through a tile of LDS that only its wave touches, for the transpose.
//
// Long lists run at the rate of memory: 32 sequences of up to 8192 keys in 4 bits 36 us of kernel for 217 MB (6.0 TB/s, half of
// it out of the last-level cache where the call is repeated), 16 in a window of 4096 in 16 bits 41 us for 268 MB (6.5).  Short
// ones are latency: one sequence of 4096 keys 5.2 us and 3.4 of merge.  48 and 64 rows this way, with four waves on a CU, are
// slower than the kernel of many rows (64 rows of 8 KV heads against 16000 keys 23.7 us, 21.9 there; 71 of 64-wide against 8000
// 10.8 and 9.0).
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
  const int group = a.group, rows = a.rows;
  const int bh = a.runs == 1 ? (int)blockIdx.x : div_by((int)blockIdx.x, a.by_runs), run = (int)blockIdx.x - bh * a.runs;
  const int b = a.B == 1 ? 0 : div_by(bh, a.by_hkv), hk = bh - b * a.Hkv;
  const KeyList kl = key_list(a, b, 0, a.S - 1);
  const int ntiles = (kl.n + kFewRowTile - 1) / kFewRowTile;
  const int per = div_by(ntiles + a.runs - 1, a.by_runs), tile0 = min(run * per, ntiles), tile1 = min(tile0 + per, ntiles);

  half8v qf[NT][KS];
  int pos[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = min(nt * 16 + l16, rows - 1), tok = row_token(a, row);
    pos[nt] = kl.len - a.S + tok;
    const half_t* qp = a.q + ((int64_t)b * a.S + tok) * a.ldq + (int64_t)(hk * group + row - tok * group) * D;
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
  // one row of K, one piece of V: the tile's place (kp, kxp, vp, vxp) and the offsets of a lane in it, of either width
  auto fetch_k = [&](T& x, int kb, const uint8_t* kp, const uint8_t* kxp, auto off, auto xoff) __attribute__((always_inline)) {
    if constexpr (FP4) {
      if constexpr (D == 128) {
        x.k[kb][0] = *reinterpret_cast<const uint4v*>(kp + off);
      } else {
        const uint2v h = *reinterpret_cast<const uint2v*>(kp + off);
        x.k[kb][0] = uint4v{h[0], h[1], 0u, 0u};
      }
      x.kx[kb] = kxp[xoff];
    } else {
#pragma unroll
      for (int s = 0; s < KS; ++s) x.k[kb][s] = *reinterpret_cast<const uint4v*>(kp + off + s * 64);
    }
  };
  auto fetch_v = [&](T& x, int i, const uint8_t* vp, const uint8_t* vxp, auto off, auto xoff) __attribute__((always_inline)) {
    x.v[i] = *reinterpret_cast<const uint4v*>(vp + off);
    if constexpr (FP4) x.vx[i] = vxp[xoff];
  };
  // 4 bits: tiles of neighbouring rows (all but the list's last one and that with the end of the sinks) are addressed by the
  // tile's place, the same for the wave, and fixed offsets in place of an address per row, eight of them a tile (32 sequences of
  // up to 8192 keys 41.2 -> 40.2 us; 16-bit tiles, four times the bytes, are 2 % slower so, and in the kernel of many rows it is
  // level, too: that one is bound elsewhere)
  const bool flat = FP4 && (uint64_t)ksr * kFewRowTile < (1u << 31) && (uint64_t)vsr * kFewRowTile < (1u << 31) &&
                    (uint64_t)a.kc.xr * kFewRowTile < (1u << 31) && (uint64_t)a.vc.xr * kFewRowTile < (1u << 31);
  constexpr int KPB = FP4 ? D / 8 : 16;  // bytes of a key that a lane takes at a time
  uint32_t koff[KB], kxoff[KB], voff[T::VP], vxoff[T::VP];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    koff[kb] = (uint32_t)(kb * 16 + l16) * (uint32_t)ksr + g * KPB;
    kxoff[kb] = FP4 ? (uint32_t)(kb * 16 + l16) * (uint32_t)a.kc.xr + (D == 128 ? g : g / 2) : 0;
  }
#pragma unroll
  for (int i = 0; i < T::VP; ++i) {
    const int p = i * 64 + lane, r = p / T::VPR, c = p % T::VPR;
    voff[i] = (uint32_t)r * (uint32_t)vsr + c * 16;
    vxoff[i] = FP4 ? (uint32_t)r * (uint32_t)a.vc.xr + c : 0;
  }
  auto fetch = [&](int tile, T& x) __attribute__((always_inline)) {
    const int li0 = tile * kFewRowTile;
    if (flat && li0 + kFewRowTile <= kl.n && (kl.gap == 0 || li0 >= kl.sinks)) {  // wave-uniform
      const int64_t key0 = li0 + kl.gap;
      const uint8_t *kp = kbase + key0 * ksr, *vp = vbase + key0 * vsr;
      const uint8_t *kxp = FP4 ? kxbase + key0 * a.kc.xr : nullptr, *vxp = FP4 ? vxbase + key0 * a.vc.xr : nullptr;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) fetch_k(x, kb, kp, kxp, koff[kb], kxoff[kb]);
#pragma unroll
      for (int i = 0; i < T::VP; ++i) fetch_v(x, i, vp, vxp, voff[i], vxoff[i]);
      return;
    }
    auto key_of = [&](int r) {  // (past the last key: the last one again, whose scores are masked)
      const int li = min(li0 + r, kl.n - 1);
      return li + (li < kl.sinks ? 0 : kl.gap);
    };
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int key = key_of(kb * 16 + l16);
      fetch_k(x, kb, kbase, kxbase, row_at(key, ksr) + g * KPB, FP4 ? row_at(key, a.kc.xr) + (D == 128 ? g : g / 2) : 0);
    }
#pragma unroll
    for (int i = 0; i < T::VP; ++i) {
      const int p = i * 64 + lane, r = p / T::VPR, c = p % T::VPR;
      const int key = key_of(r);
      fetch_v(x, i, vbase, vxbase, row_at(key, vsr) + c * 16, FP4 ? row_at(key, a.vc.xr) + c : 0);
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
                        (a.window > 0 && li0 + kl.gap <= pos1 - a.window && li1 >= a.sinks);
    half8v pf[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (masked) {  // wave-uniform
        asm volatile("");
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {  // (visible: see the kernel of many rows)
            const int li = li0 + kb * 16 + g * 4 + r;
            const int last = pos[nt] < 0 ? -1 : (a.causal ? pos[nt] - kl.gap : kl.n - 1);
            const int from = a.window > 0 ? pos[nt] - a.window + 1 - kl.gap : 0;
            if (li >= kl.n || li > last || (li < from && li >= a.sinks)) st[nt][kb][r] = -INFINITY;
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
    finish_row<D>(a, b, hk, row, kl.len - a.S + row_token(a, row) < 0, run, d4, M, L, acc);
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
  const int rows = a.rows;
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
      li[j] = i0 + j * WAYS < a.runs ? ps[i * 2 + 1] : 0.f;
      v[j] = *reinterpret_cast<const float4v*>(po + (int64_t)i * D);
    }
    float mn = m;
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) mn = fmaxf(mn, mi[j]);
    // (a run whose maximum is -inf sees no key, and its sum is 0, or it sees NaN alone, and its sum is one; that of padding is -1)
    if (mn == -INFINITY) {
#pragma unroll
      for (int j = 0; j < UNROLL; ++j) l += li[j];
      continue;
    }
    const float keep = fast_exp2(m - mn);
    l *= keep;
    acc = acc * keep;
    m = mn;
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      if (mi[j] == -INFINITY) {
        l += li[j];
        continue;
      }
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
      l = mw == -INFINITY ? l + sl[w * LANES + lane] : fmaf(sl[w * LANES + lane], sc, l);
      const float4v v = so[w * LANES + lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(v[e], sc, acc[e]);
    }
  }
  if (idx / LPR >= total) return;
  store_row<D>(a, (int)(at / rows / a.Hkv), (int)(at / rows % a.Hkv), (int)(at % rows), l < 0.f, d4, m, l, acc);
}

// ---- which kernel, and in how many runs
// The kernel of few rows runs up to 16 stacked rows of a KV head (16 rows, tile kernels / few rows: 8 KV heads of 128 against 16000
// keys in 4 bits 12.3 / 9.5 us, in 16 12.7 / 11.2), and up to 32 in 4 bits where there is enough to read that its rate counts, and not
// its latency, KV heads times keys (32 rows of 128 in 4 bits: 64 x 1024 12.7 / 15.2, 8 x 16000 17.8 / 18.9, 64 x 2048 17.8 / 18.9, 256 x
// 512 14.1 / 12.0, 128 x 1024 18.5 / 16.2, 32 x 8000 22.7 / 20.9, 256 x 2000 34.6 / 24.7; 64-wide 9.6 / 10.4, 12.2 / 11.9, 12.2 / 11.6, 10.1 / 8.5,
// 12.2 / 10.9, 16.2 / 14.2, 26.8 / 16.9; in 16 bits 64 x 1024 13.0 / 15.9, 64 x 4000 27.9 / 29.3, 256 x 2000 44.3 / 45.8).
constexpr int kFewRowsMost = 16, kFewRowsMost4 = 32;
constexpr int64_t kFewRowsMost4Keys = 1 << 17;
constexpr int kCacheMaxRuns = 64;
// Few rows: as many runs as give 512 workgroups (eight waves a CU), of at least four tiles, one a wave (8 KV heads in 4 bits,
// 512 / 256 / 1024 workgroups: 32 sequences of 8192 keys 41.0 / 54.6 / 41.1 us, 8 of 4000 11.7 / 13.1 / 14.5; one of 4096, 128 /
// 64 / 256 keys a run 7.5 / 8.9 / 7.9).
constexpr int kFewRowWorkgroups = 512, kFewRowKeys = 4 * kFewRowTile;
// ... but one run where it is so short that the merge takes longer than what the runs spare, and a launch: up to five tiles a
// wave in 4 bits, three in 16, or eight where the KV heads alone are half a round of workgroups (8 KV heads, one run / several,
// one sequence in 4 bits of 512 keys 6.5 / 7.0, 768 7.9 / 7.2, in 16 bits of 384 7.3 / 7.5, 512 8.5 / 7.3; sixteen of 768 8.7 / 9.0 and
// 11.9 / 12.2, of 1500 13.0 / 10.3 and 18.7 / 18.4; graph replays, eager calls gain another 2.7 us of host time).
constexpr int kFewRowAlone4 = 5, kFewRowAlone16 = 3, kFewRowAloneMany = 8, kFewRowManyHeads = 128;
// Many rows: what a call takes in us, fitted over sixteen calls of 71 to 65536 rows in 1 to 64 runs, for 64- and 128-wide heads:
// a tile alone on its CU, beside another workgroup's, and a pair of them in two key ways (128-wide in 4 bits a little more: there
// the conversion of both is in the chain); fixed costs with and without the merge, and of the two ways; the partial results'
// way to memory and back.  (8 KV heads of 128 in 4 bits: 64 tokens against 2000 keys in 4 / 8 / 16 / 32 runs 21.1 / 18.5 / 21.7 /
// 30.5 us, two ways in eight 19.4; 512 against 16512 in 2 / 4 / 8 202 / 164 / 175, two ways in two 165; 128 against 8000 in sixteen
// 39.6, two ways in eight 37.6; a prompt of 1024, one way / two 27.0 / 24.7, in 16 bits 28.3 / 23.6; two of 400 against 3000 keys 58.3
// in two runs / 53.7.  71 heads of 64 on one in 16 bits: one token against 8000 in 24 / 32 / 48 / 64 12.2 / 10.3 / 9.5 / 8.6, 33 in
// 24 22.7, two ways in twelve 20.3, 100 in eight 35.3, two ways in four 33.2.)
struct TileUs {
  float alone, beside, pair;
};
constexpr TileUs tile_us(int D, bool four_bit) {
  return D == 64 ? TileUs{0.9f, 1.25f, 1.3f} : TileUs{1.2f, 2.0f, four_bit ? 2.25f : 1.95f};
}
constexpr float kTileFixedUs = 5.0f, kTileMergeUs = 7.8f, kTilePairFixedUs = 1.0f, kTilePartBytesPerUs = 4.1e6f;
constexpr int kTileRound = 512;  // workgroups at a time, two a CU

CachePlan cache_plan(int B, int S, int Hq, int Hkv, int D, int kv_len, int window, int sinks, bool four_bit) {
  const int group = Hq / Hkv, rows = S * group;
  const int64_t heads = (int64_t)B * Hkv;
  CachePlan p{};
  p.ways = 1;
  const int64_t few_keys = window > 0 && (int64_t)S + window + sinks < kv_len ? (int64_t)S + window + sinks : kv_len;
  const bool most4 = four_bit && heads * few_keys >= kFewRowsMost4Keys;
  p.nt = rows <= (most4 ? kFewRowsMost4 : kFewRowsMost) ? (rows + 15) / 16 : 0;
  p.nwg = p.nt > 0 ? heads : (rows + kCacheRows - 1) / kCacheRows * heads;
  // most keys of a row block
  const int64_t toks = p.nt > 0 ? S : (kCacheRows + group - 1) / group + 1;
  int64_t keys = kv_len;
  if (window > 0 && toks + window + sinks < keys) keys = toks + window + sinks;
  if (p.nt > 0) {
    int64_t runs = kFewRowWorkgroups / p.nwg;
    if (runs > keys / kFewRowKeys) runs = keys / kFewRowKeys;
    const int alone = p.nwg >= kFewRowManyHeads ? kFewRowAloneMany : (four_bit ? kFewRowAlone4 : kFewRowAlone16);
    if (keys <= alone * kFewRowKeys) runs = 1;
    p.runs = (int)(runs < 1 ? 1 : (runs > kCacheMaxRuns ? kCacheMaxRuns : runs));
    return p;
  }
  const int64_t tiles = (keys + kCacheTile - 1) / kCacheTile;
  const int64_t most = tiles < kCacheMaxRuns ? tiles : kCacheMaxRuns;
  const float part_us = (float)(heads * rows) * (float)D * 8.f / kTilePartBytesPerUs;
  const TileUs tile = tile_us(D, four_bit);
  float best = 0.f;
  p.runs = 1;
  for (int r = 1; r <= most && (r == 1 || p.nwg * r <= 4 * kTileRound); ++r) {
    const int64_t wgs = p.nwg * r, per = (tiles + r - 1) / r;
    const float steps = wgs <= kTileRound / 2 ? tile.alone : tile.beside * (float)((wgs + kTileRound - 1) / kTileRound);
    const float us = (float)per * steps + (r == 1 ? kTileFixedUs : kTileMergeUs + (float)r * part_us);
    if (r == 1 || us < best) {
      best = us;
      p.runs = r;
      p.ways = 1;
    }
    if (wgs > kTileRound / 2) continue;
    const float two_us = (float)((per + 1) / 2) * tile.pair + kTilePairFixedUs + (r == 1 ? kTileFixedUs : kTileMergeUs + (float)r * part_us);
    if (two_us < best) {
      best = two_us;
      p.runs = r;
      p.ways = 2;
    }
  }
  return p;
}

static int64_t run_bytes(int B, int S, int Hq, int D) { return (int64_t)B * S * Hq * (D + 2) * 4; }

int64_t cache_attn_workspace_bytes(int B, int S, int Hq, int Hkv, int D, int kv_len, int window, int sinks, bool four_bit) {
  const int runs = cache_plan(B, S, Hq, Hkv, D, kv_len, window, sinks, four_bit).runs;
  return runs > 1 ? runs * run_bytes(B, S, Hq, D) : 0;
}

template <int D, bool FP4>
static void launch_t(const CacheAttnArgs& a, int nt, int ways, unsigned nwg, hipStream_t stream) {
  if (nt == 1) {
    hipLaunchKernelGGL((cache_attn_few_kernel<D, FP4, 1>), dim3(nwg), dim3(256), 0, stream, a);
    return;
  }
  if constexpr (FP4) {
    if (nt == 2) {
      hipLaunchKernelGGL((cache_attn_few_kernel<D, FP4, 2>), dim3(nwg), dim3(256), 0, stream, a);
      return;
    }
  }
  if constexpr (D == 64) {
    if (ways == 2) hipLaunchKernelGGL((cache_attn_waves_kernel<FP4, 2>), dim3(nwg), dim3(512), 0, stream, a);
    else hipLaunchKernelGGL((cache_attn_waves_kernel<FP4, 1>), dim3(nwg), dim3(256), 0, stream, a);
  } else {
    if (ways == 2) hipLaunchKernelGGL((cache_attn_tile_kernel<FP4, 2>), dim3(nwg), dim3(512), 0, stream, a);
    else hipLaunchKernelGGL((cache_attn_tile_kernel<FP4, 1>), dim3(nwg), dim3(256), 0, stream, a);
  }
}

template <int D>
static void launch_merge(const CacheAttnArgs& a, hipStream_t stream) {
  const int64_t lanes = (int64_t)a.B * a.S * a.Hq * (D / 4);
  if (a.runs > 8 && lanes < 256 * 256)
    hipLaunchKernelGGL((cache_merge_kernel<D, 8>), dim3((unsigned)((lanes + 31) / 32)), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((cache_merge_kernel<D, 1>), dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, stream, a);
}

static CacheDiv cache_div(int d) {
  CacheDiv r{0, 0};
  while (((int64_t)1 << r.sh) < d) ++r.sh;
  r.mul = (uint32_t)((((uint64_t)1 << (28 + r.sh)) + d - 1) / d);
  return r;
}

int launch_cache_attention(const CacheAttnArgs& args, hipStream_t stream) {
  CacheAttnArgs a = args;
  const CachePlan p = cache_plan(a.B, a.S, a.Hq, a.Hkv, a.D, a.kv_len, a.window, a.sinks, a.kc.scales != nullptr);
  const int64_t fit = a.ws != nullptr ? a.ws_bytes / run_bytes(a.B, a.S, a.Hq, a.D) : 0;
  a.runs = (int)(fit < p.runs ? (fit < 1 ? 1 : fit) : p.runs);
  a.group = a.Hq / a.Hkv;
  a.rows = a.S * a.group;
  a.nrb = p.nt > 0 ? 1 : (a.rows + kCacheRows - 1) / kCacheRows;
  const int heads = a.B * a.Hkv;
  a.by_group = cache_div(a.group);
  a.by_runs = cache_div(a.runs);
  a.by_hkv = cache_div(a.Hkv);
  a.by_heads = cache_div(heads % 8 == 0 ? heads / 8 : heads);
  const unsigned nwg = (unsigned)(p.nwg * a.runs);
  const bool fp4 = a.kc.scales != nullptr;
  if (a.D == 128) fp4 ? launch_t<128, true>(a, p.nt, p.ways, nwg, stream) : launch_t<128, false>(a, p.nt, p.ways, nwg, stream);
  else fp4 ? launch_t<64, true>(a, p.nt, p.ways, nwg, stream) : launch_t<64, false>(a, p.nt, p.ways, nwg, stream);
  if (hipGetLastError() != hipSuccess) return -1;
  if (a.runs == 1) return 0;
  if (a.D == 128) launch_merge<128>(a, stream);
  else launch_merge<64>(a, stream);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tri
