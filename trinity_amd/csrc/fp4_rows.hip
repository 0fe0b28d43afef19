// Rows of 16-bit values to 4-bit blocks of 32 (fp4.h) and back: tri_fp4_quantize, tri_fp4_dequantize.
//
// A thread has eight values; the four threads of a block share its largest magnitude.  Both directions are bound by the bytes
// they move, 2.53 a value: 4096 x 14336 in 29.7 us there (5.0 TB/s) and 25.5 back (5.8).  Few rows take a launch and a trip to memory,
// 2.3 us.
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

// blockIdx: (256 pieces of eight values of a row, rows).  (Four pieces a thread, loads side by side: 4.5 for 3.7 us at 1024 x 4096, level
// at 4096 x 14336.)
template <bool READ>
__global__ __launch_bounds__(256) void fp4_rows_kernel(Fp4RowsArgs a) {
  const int c = (int)blockIdx.x * 256 + (int)threadIdx.x;
  if (c >= a.K / 8) return;  // (the same for the threads of a block: K is a multiple of 32)
  for (int64_t row = blockIdx.y; row < a.M; row += gridDim.y) {
    half_t* const x = a.x + row * a.ldx + c * 8;
    uint8_t* const codes = a.codes + row * a.ldc + c * 4;
    uint8_t* const scale = a.scales + row * a.lds + (c >> 2);
    if (READ) {
      *reinterpret_cast<half8v*>(x) = fp4x8_to_half8(*reinterpret_cast<const uint32_t*>(codes), fp4_scale(*scale));
    } else {
      const half8v v = *reinterpret_cast<const half8v*>(x);
      uint32_t m = amax_bits8(v);
      m = max(m, (uint32_t)__shfl_xor((int)m, 1));
      m = max(m, (uint32_t)__shfl_xor((int)m, 2));
      const uint32_t byte = fp4_scale_byte(m);
      *reinterpret_cast<uint32_t*>(codes) = byte == kFp4Nan ? 0u : half8_to_fp4x8(v, fp4_scale(byte));
      if ((c & 3) == 0) *scale = (uint8_t)byte;
    }
  }
}

template <bool READ>
static int launch_fp4_rows(const Fp4RowsArgs& a, hipStream_t stream) {
  const dim3 grid((a.K / 8 + 255) / 256, a.M < 65535 ? a.M : 65535);
  hipLaunchKernelGGL((fp4_rows_kernel<READ>), grid, dim3(256), 0, stream, a);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}

int launch_fp4_quantize(const Fp4RowsArgs& a, hipStream_t stream) { return launch_fp4_rows<false>(a, stream); }
int launch_fp4_dequantize(const Fp4RowsArgs& a, hipStream_t stream) { return launch_fp4_rows<true>(a, stream); }

}  // namespace tri
