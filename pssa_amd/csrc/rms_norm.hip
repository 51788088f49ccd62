// Root-mean-square norm of rows with the residual's addition, and rows in 8
// bits with a scale each:
//   h = x + residual,   inv = 1 / sqrt(mean h^2 + eps),   out = gamma h inv
//   codes = round(t 127 / max|t|),   scale = max|t| inv / 127,   t = gamma h.
//
// inv is a factor of the whole row, so the codes go by t alone: the maximum is
// taken beside the sum of squares and one pass over a row is enough.  A row
// stays in the registers of its workgroup (of one wave up to 4 KiB), as
// 16-byte pieces, so that every byte moves once.
#include <algorithm>

#include "operators.h"

namespace pssa {
namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef f32x4_t f32x4_any_t __attribute__((aligned(4)));
// Rows start at any element.
typedef u32x4_t u32x4_any_t __attribute__((aligned(2)));
typedef u32x2_t u32x2_any_t __attribute__((aligned(1)));
typedef uint32_t u32_any_t __attribute__((aligned(1)));

struct Bf16 {
  uint16_t bits;
};
template <class T>
constexpr int vec_n() { return 16 / (int)sizeof(T); }

__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(Bf16* p, float v) { p->bits = bf16_bits_dev(v); }

template <class T>
__device__ __forceinline__ void widen(u32x4_t u, float (&v)[vec_n<T>()]) {
#pragma unroll
  for (int j = 0; j < vec_n<T>(); ++j) {
    if constexpr (sizeof(T) == 4)
      v[j] = __uint_as_float(u[j]);
    else
      v[j] = __uint_as_float(j & 1 ? u[j >> 1] & 0xFFFF0000u : u[j >> 1] << 16);
  }
}
// Elements c .. of a row: a piece of them, or the `left` that there are, then zeros.
template <class T>
__device__ __forceinline__ u32x4_t load_piece(const T* row, int c, int left) {
  constexpr int N = vec_n<T>();
  if (left >= N) return *reinterpret_cast<const u32x4_any_t*>(row + c);
  u32x4_t u = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (j >= left) continue;
    if constexpr (sizeof(T) == 4)
      u[j] = __float_as_uint(row[c + j]);
    else
      u[j >> 1] |= (uint32_t)row[c + j].bits << (16 * (j & 1));
  }
  return u;
}
template <class T>
__device__ __forceinline__ void store_vec(T* row, int c, int left, const float (&v)[vec_n<T>()]) {
  constexpr int N = vec_n<T>();
  if (left >= N) {
    u32x4_t u;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (sizeof(T) == 4)
        u[e] = __float_as_uint(v[e]);
      else
        u[e] = bf16x2_bits(v[2 * e], v[2 * e + 1]);
    }
    *reinterpret_cast<u32x4_any_t*>(row + c) = u;
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < left) store1(row + c + j, v[j]);
  }
}
template <int N>
__device__ __forceinline__ void store_codes(int8_t* row, int c, int left, const int (&q)[N]) {
  if (left >= N) {
    uint32_t w[N / 4];
#pragma unroll
    for (int e = 0; e < N / 4; ++e)
      w[e] = (q[4 * e] & 255) | (q[4 * e + 1] & 255) << 8 | (q[4 * e + 2] & 255) << 16 | (uint32_t)q[4 * e + 3] << 24;
    if constexpr (N == 8)
      *reinterpret_cast<u32x2_any_t*>(row + c) = u32x2_t{w[0], w[1]};
    else
      *reinterpret_cast<u32_any_t*>(row + c) = w[0];
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < left) row[c + j] = (int8_t)q[j];
  }
}

// Sum and maximum over the threads of a row: W waves of one workgroup.
template <int W>
__device__ __forceinline__ void row_reduce(float& sum, float& most, float (*s_part)[2]) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    sum += __shfl_xor(sum, off, 64);
    most = fmaxf(most, __shfl_xor(most, off, 64));
  }
  if constexpr (W > 1) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      s_part[wave][0] = sum;
      s_part[wave][1] = most;
    }
    __syncthreads();
    sum = s_part[0][0];
    most = s_part[0][1];
#pragma unroll
    for (int w = 1; w < W; ++w) {
      sum += s_part[w][0];
      most = fmaxf(most, s_part[w][1]);
    }
    __syncthreads();
  }
}

// W waves hold a row, NV pieces a thread; where a row takes one wave, four of
// them share a workgroup.  A workgroup goes through several rows: gamma stays
// in its registers, and the next row is on its way while one is summed (8192 x
// 8192 bf16 with a residual, sum and norm stored: 100 us, 5.4 TB/s, where a row a
// workgroup took 155; 256 x 768 fp32: 5.7 us, a launch).
template <class T, int W, int NV>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void rms_norm_kernel(RmsNormArgs a, int rows) {
  constexpr int N = vec_n<T>(), PER = W == 1 ? 4 : 1;  // rows of a workgroup at a time
  constexpr bool kAhead = NV * N <= 32 && W < 16;      // registers for gamma and a second row
  __shared__ float s_part[W][2];
  int tid = W == 1 ? threadIdx.x & 63 : threadIdx.x;
  int r = W == 1 ? blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  float gamma[kAhead ? NV : 1][N];
  auto gamma_of = [&](int k, float (&g)[N]) {
    const int c = (tid + k * 64 * W) * N;
    if (a.gamma && c + N <= a.width) {
#pragma unroll
      for (int j4 = 0; j4 < N; j4 += 4) {
        const f32x4_t v = *reinterpret_cast<const f32x4_any_t*>(a.gamma + c + j4);
#pragma unroll
        for (int e = 0; e < 4; ++e) g[j4 + e] = v[e];
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) g[j] = c + j >= a.width ? 0.0f : a.gamma ? a.gamma[c + j] : 1.0f;
    }
  };
  u32x4_t next[kAhead ? NV : 1], next_res[kAhead ? NV : 1];
  auto fetch = [&](int row) {
    const T* x = static_cast<const T*>(a.x) + (size_t)row * a.ld_x;
    const T* res = static_cast<const T*>(a.residual) + (size_t)row * a.ld_residual;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (tid + k * 64 * W) * N;
      next[kAhead ? k : 0] = load_piece<T>(x, c, a.width - c);
    }
    if (a.residual) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (tid + k * 64 * W) * N;
        next_res[kAhead ? k : 0] = load_piece<T>(res, c, a.width - c);
      }
    }
  };
  if constexpr (kAhead) {
    if (r < rows) fetch(r);
#pragma unroll
    for (int k = 0; k < NV; ++k) gamma_of(k, gamma[k]);
  }
  for (; r < rows; r += PER * gridDim.x) {
    // New for the compiler with each row: addresses kept for all pieces would take more registers than the row.
    if constexpr (!kAhead) asm volatile("" : "+v"(tid));
    float h[NV][N];
    const T* x = static_cast<const T*>(a.x) + (size_t)r * a.ld_x;
    const T* res = static_cast<const T*>(a.residual) + (size_t)r * a.ld_residual;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (tid + k * 64 * W) * N;
      widen<T>(kAhead ? next[kAhead ? k : 0] : load_piece<T>(x, c, a.width - c), h[k]);
    }
    if (a.residual) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (tid + k * 64 * W) * N;
        float v[N];
        widen<T>(kAhead ? next_res[kAhead ? k : 0] : load_piece<T>(res, c, a.width - c), v);
#pragma unroll
        for (int j = 0; j < N; ++j) h[k][j] += v[j];
      }
    }
    if constexpr (kAhead) {
      const int r_next = r + PER * (int)gridDim.x;
      if (r_next < rows) fetch(r_next);
    }
    // The sum of squares; the largest |gamma h|, infinite where one is not a
    // number (a maximum passes over it).
    float ss = 0.0f, most = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int j = 0; j < N; ++j) ss = fmaf(h[k][j], h[k][j], ss);
      if (a.codes) {
        float g[N];
        if constexpr (!kAhead) gamma_of(k, g);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float t = fabsf(h[k][j] * (kAhead ? gamma[kAhead ? k : 0][j] : g[j]));
          most = fmaxf(most, t < INFINITY ? t : INFINITY);
        }
      }
    }
    row_reduce<W>(ss, most, s_part);
    // Squares past fp32's range: again with the row scaled down, by a power of
    // two that lets 65536 of the largest values in (an infinity in the row comes
    // out the same).  inv is then that of the scaled row.
    float inv = 1.0f / sqrtf(ss / (float)a.width + a.eps), half = 1.0f;
    if (ss == INFINITY) {
      half = 3.5527136788005009e-15f;  // 2^-48
      float low = 0.0f, none = 0.0f;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float v = h[k][j] * (half * half);
          low = fmaf(v, v, low);
        }
      row_reduce<W>(low, none, s_part);
      inv = 1.0f / sqrtf(low / (float)a.width);
    }
    const float down = a.normed ? half * half : 1.0f;
    if (!a.normed) inv = half = 1.0f;

    if (a.sum) {
      T* sum = static_cast<T*>(a.sum) + (size_t)r * a.ld_sum;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (tid + k * 64 * W) * N, left = a.width - c;
        if (left > 0) store_vec<T>(sum, c, left, h[k]);
      }
    }
    if (a.out) {
      T* out = static_cast<T*>(a.out) + (size_t)r * a.ld_out;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (tid + k * 64 * W) * N, left = a.width - c;
        if (left <= 0) continue;
        float v[N], g[N];
        if constexpr (!kAhead) gamma_of(k, g);
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = h[k][j] * down * inv * (kAhead ? gamma[kAhead ? k : 0][j] : g[j]);
        store_vec<T>(out, c, left, v);
      }
    }
    if (a.codes) {
      // A row that is not finite has the scale NaN, which its products take on.
      const bool fine = most < INFINITY;
      // Small maxima are scaled up, exactly: 127 / max would overflow, max / 127 have few bits left.
      const float up = most < 1.0f ? 18446744073709551616.0f : 1.0f;  // 2^64
      const float by = 127.0f / (most * up);
      int8_t* codes = a.codes + (size_t)r * a.ld_codes;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (tid + k * 64 * W) * N, left = a.width - c;
        if (left <= 0) continue;
        int q[N];
        float g[N];
        if constexpr (!kAhead) gamma_of(k, g);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float t = h[k][j] * (kAhead ? gamma[kAhead ? k : 0][j] : g[j]);
          q[j] = fine && most > 0.0f ? (int)fminf(fmaxf(rintf(t * up * by), -127.0f), 127.0f) : 0;
        }
        store_codes<N>(codes, c, left, q);
      }
      if (tid == 0) a.scales[r] = fine ? most * up / 127.0f * half * inv * half / up : NAN;  // halves: products inside the range
    }
  }
}

template <class T, int W, int NV>
Status launch_rows(hipStream_t stream, const RmsNormArgs& a, size_t rows) {
  constexpr int WAVES = W == 1 ? 4 : W;
  // As many workgroups as the machine holds at once, 16 waves a compute unit.
  constexpr size_t most = 256 * std::max(1, 16 / WAVES);
  static_assert((W == 1 ? 4 : 1) * most <= kRmsStep, "rows of a step");
  const size_t all = W == 1 ? (rows + 3) / 4 : rows;
  rms_norm_kernel<T, W, NV><<<(uint32_t)std::min(all, most), 64 * WAVES, 0, stream>>>(a, (int)rows);
  PSSA_LAUNCH_CHECK("rms_norm_kernel");
  return Status::Ok();
}

template <class T>
Status launch_typed(hipStream_t stream, const RmsNormArgs& a, size_t rows) {
  const int pieces = (a.width + vec_n<T>() - 1) / vec_n<T>();
  if (pieces <= 64) return launch_rows<T, 1, 1>(stream, a, rows);
  if (pieces <= 128) return launch_rows<T, 1, 2>(stream, a, rows);
  if (pieces <= 256) return launch_rows<T, 1, 4>(stream, a, rows);
  if (pieces <= 512) return launch_rows<T, 4, 2>(stream, a, rows);
  if (pieces <= 1024) return launch_rows<T, 4, 4>(stream, a, rows);
  if (pieces <= 2048) return launch_rows<T, 8, 4>(stream, a, rows);
  if (pieces <= 4096) return launch_rows<T, 16, 4>(stream, a, rows);
  if constexpr (sizeof(T) == 4) {
    if (pieces > 8192) return launch_rows<T, 16, 16>(stream, a, rows);
  }
  return launch_rows<T, 16, 8>(stream, a, rows);
}

}  // namespace

static_assert(kRmsWidth / 4 <= 16 * 64 * 16 && kRmsWidth / 8 <= 16 * 64 * 8, "the widest row's pieces");

Status launch_rms_norm(hipStream_t stream, int dtype, const RmsNormArgs& a, size_t rows) {
  return dtype == PSSA_HIP_F32 ? launch_typed<float>(stream, a, rows) : launch_typed<Bf16>(stream, a, rows);
}

}  // namespace pssa
