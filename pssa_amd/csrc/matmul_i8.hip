// Products of 8-bit rows and weights with a scale for each row and channel:
//   y[i][j] = x_scale[i] w_scale[j] sum_l x[i][l] w[j][l].
//
// The sums are whole numbers in 32 bits, exact, so neither tiles nor the order
// of a sum change a result; each y has the rounding of its sum to fp32, two of
// the scales, and the last one to bf16 where y is.
#include <algorithm>

#include "operators.h"

namespace pssa {
namespace {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef i32x4_t i32x4_any_t __attribute__((aligned(1)));

struct Bf16 {
  uint16_t bits;
};
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(Bf16* p, float v) { p->bits = bf16_bits_dev(v); }

// 16 codes, zeros past `left`.
__device__ __forceinline__ i32x4_t load16(const int8_t* p, int left) {
  if (left >= 16) return *reinterpret_cast<const i32x4_any_t*>(p);
  i32x4_t v = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 15; ++i)
    if (i < left) v[i >> 2] |= (int)(uint8_t)p[i] << (8 * (i & 3));
  return v;
}

// Any widths and alignment, straight from memory: a wave computes 16 rows by
// 16 N channels.
template <class T, int N>
__global__ __launch_bounds__(256) void matmul_i8_any_kernel(I8Args a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
  const int row0 = blockIdx.y * 16, ch0 = (blockIdx.x * 4 + wave) * 16 * N;
  if (ch0 >= a.n) return;
  const int8_t* x = a.x + (size_t)min(row0 + col, a.m - 1) * a.ld_x;
  const int8_t* w[N];
#pragma unroll
  for (int c = 0; c < N; ++c) w[c] = a.w + (size_t)min(ch0 + 16 * c + col, a.n - 1) * a.ld_w;
  i32x4_t acc[N];
#pragma unroll
  for (int c = 0; c < N; ++c) acc[c] = i32x4_t{0, 0, 0, 0};
  for (int l = 16 * quad; l - 16 * quad < a.k; l += 64) {
    const i32x4_t xf = load16(x + l, a.k - l);
#pragma unroll
    for (int c = 0; c < N; ++c) acc[c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xf, load16(w[c] + l, a.k - l), acc[c], 0, 0, 0);
  }
#pragma unroll
  for (int c = 0; c < N; ++c)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = row0 + 4 * quad + r, j = ch0 + 16 * c + col;
      if (i < a.m && j < a.n)
        store1(static_cast<T*>(a.y) + (size_t)i * a.ld_y + j, (float)acc[c][r] * a.x_scales[i] * a.w_scales[j]);
    }
}

template <class T>
Status launch_any(hipStream_t stream, const I8Args& a) {
  const dim3 grid((a.n + 255) / 256, (a.m + 15) / 16);
  matmul_i8_any_kernel<T, 4><<<grid, 256, 0, stream>>>(a);
  PSSA_LAUNCH_CHECK("matmul_i8_any_kernel");
  return Status::Ok();
}

}  // namespace

int i8_splits(size_t m, size_t n, size_t k) { return 1; }
Status init_i8_attributes() { return Status::Ok(); }

Status launch_matmul_i8(hipStream_t stream, int y_dtype, const I8Args& a) {
  return y_dtype == PSSA_HIP_F32 ? launch_any<float>(stream, a) : launch_any<Bf16>(stream, a);
}

}  // namespace pssa
