// Rows of caches of several sequences: written (tri_cache_append) and read back (tri_cache_read), 16-bit or in 4-bit
// blocks (fp4.h).
//
// One thread per eight channels of a row; the four threads of a 4-bit block share its largest magnitude.  Both directions
// are bound by the bytes they move: 2.53 of 16-bit rows and codes per value.
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

// blockIdx: (rows of a head, head of a sequence, K or V)
template <int D, bool FP4, bool READ>
__device__ __forceinline__ void cache_rows_body(const CacheRowsArgs& a) {
  constexpr int CPR = D / 8;
  const bool isv = blockIdx.z != 0;
  const CacheView& c = isv ? a.vc : a.kc;
  half_t* const rows = isv ? a.v : a.k;
  const int64_t r_sb = isv ? a.v_sb : a.k_sb, r_sh = isv ? a.v_sh : a.k_sh, r_sr = isv ? a.v_sr : a.k_sr;
  const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int i = (int)(idx / CPR), ch = (int)(idx % CPR);
  if (i >= a.S) return;
  for (int bh = blockIdx.y; bh < a.B * a.Hkv; bh += gridDim.y) {
    const int b = bh / a.Hkv, h = bh % a.Hkv;
    const int pos = seq_len(a.lens, b, a.kv_len) - a.S + i;
    half_t* const r = rows + b * r_sb + h * r_sh + i * r_sr + ch * 8;
    if (!READ && pos < 0) continue;  // (the same for the threads of a row)
    if (FP4) {
      uint8_t* const codes = static_cast<uint8_t*>(c.p) + b * c.sb + h * c.sh + pos * c.sr + ch * 4;
      uint8_t* const sc = c.scales + b * c.xb + h * c.xh + pos * c.xr + ch / 4;
      if (READ) {
        half8v x = {};
        if (pos >= 0) x = fp4x8_to_half8(*reinterpret_cast<const uint32_t*>(codes), fp4_scale(*sc));
        *reinterpret_cast<half8v*>(r) = x;
      } else {
        const half8v x = *reinterpret_cast<const half8v*>(r);
        uint32_t m = amax_bits(x);
        m = max(m, (uint32_t)__shfl_xor((int)m, 1));
        m = max(m, (uint32_t)__shfl_xor((int)m, 2));
        const uint32_t byte = fp4_scale_byte(m);
        *reinterpret_cast<uint32_t*>(codes) = byte == kFp4Nan ? 0u : half8_to_fp4x8(x, fp4_scale(byte));
        if (ch % 4 == 0) *sc = (uint8_t)byte;
      }
    } else {
      half_t* const e = static_cast<half_t*>(c.p) + b * c.sb + h * c.sh + pos * c.sr + ch * 8;
      if (READ) *reinterpret_cast<half8v*>(r) = pos >= 0 ? *reinterpret_cast<const half8v*>(e) : half8v{};
      else *reinterpret_cast<half8v*>(e) = *reinterpret_cast<const half8v*>(r);
    }
  }
}

template <int D, bool FP4, bool READ>
__global__ __launch_bounds__(256) void cache_rows_kernel(CacheRowsArgs a) {
  cache_rows_body<D, FP4, READ>(a);
}

template <bool READ>
static int launch_rows(const CacheRowsArgs& a, hipStream_t stream) {
  const int64_t threads = (int64_t)a.S * (a.D / 8), heads = (int64_t)a.B * a.Hkv;
  const int block = threads >= 256 ? 256 : 64;
  const dim3 grid((unsigned)((threads + block - 1) / block), (unsigned)(heads < 65535 ? heads : 65535), 2);
  const bool fp4 = a.kc.scales != nullptr;
  if (a.D == 128) {
    if (fp4) hipLaunchKernelGGL((cache_rows_kernel<128, true, READ>), grid, dim3(block), 0, stream, a);
    else hipLaunchKernelGGL((cache_rows_kernel<128, false, READ>), grid, dim3(block), 0, stream, a);
  } else {
    if (fp4) hipLaunchKernelGGL((cache_rows_kernel<64, true, READ>), grid, dim3(block), 0, stream, a);
    else hipLaunchKernelGGL((cache_rows_kernel<64, false, READ>), grid, dim3(block), 0, stream, a);
  }
  return hipGetLastError() == hipSuccess ? 0 : -1;
}

int launch_cache_append(const CacheRowsArgs& a, hipStream_t stream) { return launch_rows<false>(a, stream); }
int launch_cache_read(const CacheRowsArgs& a, hipStream_t stream) { return launch_rows<true>(a, stream); }

}  // namespace tri
