// Rows of caches of several sequences: written (tri_cache_append) and read back (tri_cache_read), 16-bit or in 4-bit
// blocks (fp4.h).
//
// A thread has eight channels of a row; the four threads of a 4-bit block share its largest magnitude.  Both directions are
// bound by the bytes they move, 2.53 a value (single tokens by a launch and a trip to memory: 2.6 us).
#include "common.h"
#include "fp4.h"
#include "launch.h"

namespace tri {

// largest magnitude of eight elements as bits without the sign (infinities and NaN above all numbers)
__device__ __forceinline__ uint32_t amax_bits(half8v x) {
  typedef uint16_t ushort8v __attribute__((ext_vector_type(8)));
  const ushort8v u = __builtin_bit_cast(ushort8v, x) & (uint16_t)0x7FFF;
  uint16_t m = u[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) m = u[e] > m ? u[e] : m;
  return m;
}

// position n - S + i of token (or row) i; n: length of the sequence
__device__ __forceinline__ int seq_len(const int32_t* lens, int b, int kv_len) {
  return lens == nullptr ? kv_len : min(max(lens[b], 0), kv_len);
}

// blockIdx: (rows of a head, head of a sequence, K or V); U pieces of eight channels per thread, whose loads travel together
template <int D, bool FP4, bool READ, int U>
__device__ __forceinline__ void cache_rows_body(const CacheRowsArgs& a) {
  constexpr int CPR = D / 8;
  const bool isv = blockIdx.z != 0;
  const CacheView& c = isv ? a.vc : a.kc;
  half_t* const rows = isv ? a.v : a.k;
  const int64_t r_sb = isv ? a.v_sb : a.k_sb, r_sh = isv ? a.v_sh : a.k_sh, r_sr = isv ? a.v_sr : a.k_sr;
  const int rpb = (int)blockDim.x / CPR;  // rows per pass of the block
  const int i0 = (int)blockIdx.x * rpb * U + (int)threadIdx.x / CPR, ch = threadIdx.x % CPR;
  for (int bh = blockIdx.y; bh < a.B * a.Hkv; bh += gridDim.y) {
    const int b = bh / a.Hkv, h = bh - b * a.Hkv;
    const int pos0 = seq_len(a.lens, b, a.kv_len) - a.S;
    half_t* const r = rows + b * r_sb + h * r_sh + ch * 8;
    // the cache's row of position 0, and its scale
    uint8_t* const codes = static_cast<uint8_t*>(c.p) + (b * c.sb + h * c.sh) * (FP4 ? 1 : 2) + ch * (FP4 ? 4 : 16);
    uint8_t* const sc = c.scales + b * c.xb + h * c.xh + ch / 4;
    const int64_t sr = c.sr * (FP4 ? 1 : 2);
    half8v x[U];
    uint32_t w[U], e[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * rpb;
      const int64_t pos = (int64_t)pos0 + i;
      x[u] = half8v{};
      w[u] = 0;
      e[u] = 1;
      if (i >= a.S || pos < 0) continue;  // (the same for the threads of a row)
      if (!READ) {
        x[u] = *reinterpret_cast<const half8v*>(r + i * r_sr);
      } else if (FP4) {
        w[u] = *reinterpret_cast<const uint32_t*>(codes + pos * sr);
        e[u] = sc[pos * c.xr];
      } else {
        x[u] = *reinterpret_cast<const half8v*>(codes + pos * sr);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * rpb;
      const int64_t pos = (int64_t)pos0 + i;
      if (i >= a.S) continue;
      if (READ) {
        *reinterpret_cast<half8v*>(r + i * r_sr) = FP4 ? fp4x8_to_half8(w[u], fp4_scale(e[u])) : x[u];  // (padding: zeros)
        continue;
      }
      if (pos < 0) continue;
      if (FP4) {
        uint32_t m = amax_bits(x[u]);
        m = max(m, (uint32_t)__shfl_xor((int)m, 1));
        m = max(m, (uint32_t)__shfl_xor((int)m, 2));
        const uint32_t byte = fp4_scale_byte(m);
        *reinterpret_cast<uint32_t*>(codes + pos * sr) = byte == kFp4Nan ? 0u : half8_to_fp4x8(x[u], fp4_scale(byte));
        if (ch % 4 == 0) sc[pos * c.xr] = (uint8_t)byte;
      } else {
        *reinterpret_cast<half8v*>(codes + pos * sr) = x[u];
      }
    }
  }
}

template <int D, bool FP4, bool READ, int U>
__global__ __launch_bounds__(256) void cache_rows_kernel(CacheRowsArgs a) {
  cache_rows_body<D, FP4, READ, U>(a);
}

template <int D, bool READ, int U>
static void launch_rows_u(const CacheRowsArgs& a, dim3 grid, int block, hipStream_t stream) {
  if (a.kc.scales != nullptr) hipLaunchKernelGGL((cache_rows_kernel<D, true, READ, U>), grid, dim3(block), 0, stream, a);
  else hipLaunchKernelGGL((cache_rows_kernel<D, false, READ, U>), grid, dim3(block), 0, stream, a);
}

// Four rows per thread, from as many pieces on as keep every CU busy all the same: what bounds a call is then how much of it
// is on its way at a time (128-wide heads, four prompts of 4096 tokens written and read 39.3 us with one row per thread, 29.7
// with two, 28.4 with four, 30.0 with eight, 138 MB at 4.9 TB/s; 32752 rows read 36.0, 26.9, 26.6, 26.5, 170 MB at 6.4; 16 of
// 256 written and read 15.4 -> 11.8; one of 333 of 64 level).
constexpr int64_t kRowsManyThreads = 1 << 18;
constexpr int kRowsPerThread = 4;
template <bool READ>
static int launch_rows(const CacheRowsArgs& a, hipStream_t stream) {
  const int64_t threads = (int64_t)a.S * (a.D / 8), heads = (int64_t)a.B * a.Hkv;
  const int block = threads >= 256 ? 256 : 64;
  const bool many = 2 * heads * threads >= kRowsManyThreads;
  const int64_t per = (int64_t)block * (many ? kRowsPerThread : 1);
  const dim3 grid((unsigned)((threads + per - 1) / per), (unsigned)(heads < 65535 ? heads : 65535), 2);
  if (a.D == 128) many ? launch_rows_u<128, READ, kRowsPerThread>(a, grid, block, stream) : launch_rows_u<128, READ, 1>(a, grid, block, stream);
  else many ? launch_rows_u<64, READ, kRowsPerThread>(a, grid, block, stream) : launch_rows_u<64, READ, 1>(a, grid, block, stream);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}

int launch_cache_append(const CacheRowsArgs& a, hipStream_t stream) { return launch_rows<false>(a, stream); }
int launch_cache_read(const CacheRowsArgs& a, hipStream_t stream) { return launch_rows<true>(a, stream); }

}  // namespace tri
