// Rows of 16-bit values to 4-bit blocks of 32 (fp4.h) and back: tri_fp4_quantize, tri_fp4_dequantize.
//
// A thread has eight values; the four threads of a block share its largest magnitude.  Both directions are bound by the bytes
// they move, 2.53 a value: 4096 x 14336 in 27.4 us there (5.4 TB/s) and 20.9 back (7.1; most of it written).  Few rows take a launch
// and a trip to memory, 2.6 us.
#include "common.h"
#include "fp4.h"
#include "launch.h"

namespace tri {

// largest magnitude of eight elements as bits without the sign (infinities and NaN above all numbers)
__device__ __forceinline__ uint32_t amax_bits8(half8v x) {
  typedef uint16_t ushort8v __attribute__((ext_vector_type(8)));
  const ushort8v u = __builtin_bit_cast(ushort8v, x) & (uint16_t)0x7FFF;
  uint16_t m = u[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) m = u[e] > m ? u[e] : m;
  return m;
}

// blockIdx: (pieces of eight values of a row, rows); U pieces per thread, whose loads travel together
template <bool READ, int U>
__global__ __launch_bounds__(256) void fp4_rows_kernel(Fp4RowsArgs a) {
  const int pieces = a.K / 8, c0 = (int)blockIdx.x * 256 * U + (int)threadIdx.x;
  for (int64_t row = blockIdx.y; row < a.M; row += gridDim.y) {
    half_t* const x = a.x + row * a.ldx;
    uint8_t* const codes = a.codes + row * a.ldc;
    uint8_t* const scales = a.scales + row * a.lds;
    half8v v[U];
    uint32_t w[U], e[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * 256;
      v[u] = half8v{};
      w[u] = 0;
      e[u] = 1;
      if (c >= pieces) continue;  // (the same for the threads of a block: K is a multiple of 32)
      if (READ) {
        w[u] = *reinterpret_cast<const uint32_t*>(codes + c * 4);
        e[u] = scales[c >> 2];
      } else {
        v[u] = *reinterpret_cast<const half8v*>(x + c * 8);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * 256;
      if (c >= pieces) continue;
      if (READ) {
        *reinterpret_cast<half8v*>(x + c * 8) = fp4x8_to_half8(w[u], fp4_scale(e[u]));
        continue;
      }
      uint32_t m = amax_bits8(v[u]);
      m = max(m, (uint32_t)__shfl_xor((int)m, 1));
      m = max(m, (uint32_t)__shfl_xor((int)m, 2));
      const uint32_t byte = fp4_scale_byte(m);
      *reinterpret_cast<uint32_t*>(codes + c * 4) = byte == kFp4Nan ? 0u : half8_to_fp4x8(v[u], fp4_scale(byte));
      if ((c & 3) == 0) scales[c >> 2] = (uint8_t)byte;
    }
  }
}

template <bool READ>
static int launch_fp4_rows(const Fp4RowsArgs& a, hipStream_t stream) {
  const int pieces = a.K / 8;
  const bool many = (int64_t)a.M * pieces >= (1 << 18);
  const int per = 256 * (many ? 4 : 1);
  const dim3 grid((pieces + per - 1) / per, a.M < 65535 ? a.M : 65535);
  if (many) hipLaunchKernelGGL((fp4_rows_kernel<READ, 4>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((fp4_rows_kernel<READ, 1>), grid, dim3(256), 0, stream, a);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}

int launch_fp4_quantize(const Fp4RowsArgs& a, hipStream_t stream) { return launch_fp4_rows<false>(a, stream); }
int launch_fp4_dequantize(const Fp4RowsArgs& a, hipStream_t stream) { return launch_fp4_rows<true>(a, stream); }

}  // namespace tri
