// Products of 8-bit rows and weights with a scale for each row and channel:
//   y[i][j] = x_scale[i] w_scale[j] sum_l x[i][l] w[j][l].
//
// The sums are whole numbers in 32 bits, exact, so neither tiles nor the order
// of a sum change a result; each y has the rounding of its sum to fp32, two of
// the scales, and the last one to bf16 where y is.
//
// Few rows read the weights straight into the matrix instructions' registers;
// many rows run in tiles whose slabs of 128 codes go from memory straight into
// one of two LDS buffers while the other one is multiplied.
#include <algorithm>

#include "operators.h"

namespace pssa {
namespace {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef i32x4_t i32x4_any_t __attribute__((aligned(1)));
typedef int i32x16_t __attribute__((ext_vector_type(16)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef f32x4_t f32x4_any_t __attribute__((aligned(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef u32x2_t u32x2_any_t __attribute__((aligned(2)));

constexpr size_t kComputeUnits = 256;

struct Bf16 {
  uint16_t bits;
};
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(Bf16* p, float v) { p->bits = bf16_bits_dev(v); }
// Four neighbouring elements, the `left` that there are.
template <class T>
__device__ __forceinline__ void store4(T* p, const f32x4_t& v, int left) {
  if (left >= 4) {
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<f32x4_any_t*>(p) = v;
    else
      *reinterpret_cast<u32x2_any_t*>(p) = u32x2_t{bf16x2_bits(v[0], v[1]), bf16x2_bits(v[2], v[3])};
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < left) store1(p + e, v[e]);
  }
}

// 16 codes, zeros past `left`.
__device__ __forceinline__ i32x4_t load16(const int8_t* p, int left) {
  if (left >= 16) return *reinterpret_cast<const i32x4_any_t*>(p);
  i32x4_t v = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 15; ++i)
    if (i < left) v[i >> 2] |= (int)(uint8_t)p[i] << (8 * (i & 3));
  return v;
}

// ---------------------------------------------------------------- few rows
// A wave multiplies 16 MT rows by 16 NC channels over its part of k: WK waves
// of a workgroup share the channels, 4 / WK... of them lie side by side, and
// the parts meet in LDS.  Rows at any byte.
template <class T, int MT, int NC, int WK>
__global__ __launch_bounds__(256) void matmul_i8_rows_kernel(I8Args a) {
  constexpr int WN = 4 / WK, DEEP = MT * NC >= 4 ? 2 : 4;  // steps of 64 codes whose loads are in flight together
  __shared__ i32x4_t s_acc[WK > 1 ? (WK - 1) * MT * NC * 64 : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4, wk = wave % WK;
  const int ch0 = (blockIdx.x * WN + wave / WK) * 16 * NC, row0 = blockIdx.y * 16 * MT;
  const int8_t *x[MT], *w[NC];
#pragma unroll
  for (int t = 0; t < MT; ++t) x[t] = a.x + (size_t)min(row0 + 16 * t + col, a.m - 1) * a.ld_x + 16 * quad;
#pragma unroll
  for (int c = 0; c < NC; ++c) w[c] = a.w + (size_t)min(ch0 + 16 * c + col, a.n - 1) * a.ld_w + 16 * quad;
  i32x4_t acc[NC][MT];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[c][t] = i32x4_t{0, 0, 0, 0};
  const int steps = a.k / 64, first = wk * steps / WK, last = (wk + 1) * steps / WK;
  auto some = [&](int s, auto n) {
    constexpr int N = decltype(n)::value;
    i32x4_t xf[N][MT], wf[N][NC];
#pragma unroll
    for (int d = 0; d < N; ++d) {
#pragma unroll
      for (int c = 0; c < NC; ++c) wf[d][c] = *reinterpret_cast<const i32x4_any_t*>(w[c] + 64 * (s + d));
#pragma unroll
      for (int t = 0; t < MT; ++t) xf[d][t] = *reinterpret_cast<const i32x4_any_t*>(x[t] + 64 * (s + d));
    }
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[c][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[d][c], xf[d][t], acc[c][t], 0, 0, 0);
  };
  int s = first;
  for (; s + DEEP <= last; s += DEEP) some(s, std::integral_constant<int, DEEP>{});
  for (; s < last; ++s) some(s, std::integral_constant<int, 1>{});
  if (wk == WK - 1 && a.k % 64) {
    const int left = a.k - 64 * steps - 16 * quad;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const i32x4_t wf = load16(w[c] + 64 * steps, left);
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[c][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf, load16(x[t] + 64 * steps, left), acc[c][t], 0, 0, 0);
    }
  }
  if constexpr (WK > 1) {
    if (wk) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int t = 0; t < MT; ++t) s_acc[(((wk - 1) * NC + c) * MT + t) * 64 + lane] = acc[c][t];
    }
    __syncthreads();
    if (wk) return;
#pragma unroll
    for (int p = 0; p < WK - 1; ++p)
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[c][t] += s_acc[((p * NC + c) * MT + t) * 64 + lane];
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int i = row0 + 16 * t + col;
    if (i >= a.m) continue;
    const float sx = a.x_scales[i];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int j = ch0 + 16 * c + 4 * quad;
      if (j >= a.n) continue;
      f32x4_t y;
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] = (float)acc[c][t][r] * sx * a.w_scales[min(j + r, a.n - 1)];
      store4(static_cast<T*>(a.y) + (size_t)i * a.ld_y + j, y, a.n - j);
    }
  }
}

// ----------------------------------------------------------------- many rows
__device__ uint32_t g_zeros[4];  // codes behind a row's end

// Consecutive workgroups lie on different XCDs: each of the eight gets
// neighbouring tiles, walked in bands of 8 rows of tiles, so that what runs at
// one time on an XCD shares its L2's rows and weights.
__device__ __forceinline__ void tile_of(int bid, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int all = tiles_m * tiles_n, per = all / 8, more = all % 8, xcd = bid % 8, at = bid / 8;
  const int tile = xcd * per + min(xcd, more) + at;
  constexpr int BAND = 8;
  const int band = tile / (BAND * tiles_n), in_band = tile - band * BAND * tiles_n;
  const int height = min(BAND, tiles_m - band * BAND);
  tm = band * BAND + in_band % height;
  tn = in_band / height;
}

// BM rows by BN channels, WM x WN waves; rows and weights at multiples of 16
// bytes, k a multiple of 16.
template <class T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void matmul_i8_tiles_kernel(I8Args a, int tiles_m, int tiles_n) {
  constexpr int WAVES = WM * WN, THREADS = 64 * WAVES, TM = BM / WM / 32, TN = BN / WN / 32;
  constexpr int UNITS = (BM + BN) * 8, PER = UNITS / THREADS;  // of 16 bytes; of a thread
  extern __shared__ __attribute__((aligned(256))) i32x4_t s_tile[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l32 = lane & 31, half = lane >> 5, wm = wave % WM, wn = wave / WM;
  int tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const int slabs = (a.k + 127) / 128, first = (int)((int64_t)blockIdx.y * slabs / a.splits),
            last = (int)((int64_t)(blockIdx.y + 1) * slabs / a.splits);

  // A slab row is 8 units of 16 codes; unit u of row r lies at u ^ (r & 7), so
  // that rows read at one unit hit different banks.
  const int8_t* src[PER];
  int unit_k;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int row = (i * THREADS + (int)threadIdx.x) / 8, u = (threadIdx.x & 7) ^ (row & 7);
    unit_k = 16 * u;  // THREADS / 8 is a multiple of 8: the same for all of a thread's rows
    src[i] = row < BM ? a.x + (size_t)min(m0 + row, a.m - 1) * a.ld_x + 16 * u
                      : a.w + (size_t)min(n0 + row - BM, a.n - 1) * a.ld_w + 16 * u;
  }
  auto issue = [&](int slab, i32x4_t* buffer) {
    const bool there = 128 * slab + unit_k < a.k;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const void* from = there ? static_cast<const void*>(src[i] + (size_t)slab * 128) : g_zeros;
      auto* to = (__attribute__((address_space(3))) void*)(buffer + i * THREADS + wave * 64);
      __builtin_amdgcn_global_load_lds(from, to, 16, 0, 0);
    }
  };
  i32x16_t acc[TN][TM];
#pragma unroll
  for (int b = 0; b < TN; ++b)
#pragma unroll
    for (int t = 0; t < TM; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[b][t][e] = 0;

  i32x4_t* buffer = s_tile;
  if (first < last) issue(first, buffer);
  for (int slab = first; slab < last; ++slab) {
    __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
    __syncthreads();  // the slab is there, and the one before is read
    i32x4_t* other = buffer == s_tile ? s_tile + UNITS : s_tile;
    if (slab + 1 < last) issue(slab + 1, other);
    const i32x4_t *sx = buffer + (wm * TM * 32 + l32) * 8, *sw = buffer + (BM + wn * TN * 32 + l32) * 8;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const int u = (2 * ks + half) ^ (l32 & 7);
      i32x4_t xf[TM], wf[TN];
#pragma unroll
      for (int b = 0; b < TN; ++b) wf[b] = sw[b * 256 + u];
#pragma unroll
      for (int t = 0; t < TM; ++t) xf[t] = sx[t * 256 + u];
#pragma unroll
      for (int b = 0; b < TN; ++b)
#pragma unroll
        for (int t = 0; t < TM; ++t) acc[b][t] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[b], xf[t], acc[b][t], 0, 0, 0);
    }
    buffer = other;
  }
  // A lane holds a row's channels 8 g + 4 half .. + 3 of each 32.
#pragma unroll
  for (int t = 0; t < TM; ++t) {
    const int i = m0 + (wm * TM + t) * 32 + l32;
    if (i >= a.m) continue;
    const float scale = a.x_scales[i];
#pragma unroll
    for (int b = 0; b < TN; ++b)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int j = n0 + (wn * TN + b) * 32 + 8 * g + 4 * half, left = a.n - j;
        if (left <= 0) continue;
        if (a.splits > 1) {
          int32_t* part = a.parts + ((size_t)blockIdx.y * a.m + i) * a.n + j;
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (r < left) part[r] = acc[b][t][4 * g + r];
          continue;
        }
        f32x4_t y;
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = (float)acc[b][t][4 * g + r] * scale * a.w_scales[min(j + r, a.n - 1)];
        store4(static_cast<T*>(a.y) + (size_t)i * a.ld_y + j, y, left);
      }
  }
}

// The parts of k summed, and scaled.
template <class T>
__global__ __launch_bounds__(256) void matmul_i8_join_kernel(I8Args a) {
  const size_t at = (size_t)blockIdx.x * 256 + threadIdx.x, all = (size_t)a.m * a.n;
  if (at >= all) return;
  int sum = 0;
  for (int s = 0; s < a.splits; ++s) sum += a.parts[s * all + at];
  const size_t i = at / a.n, j = at - i * a.n;
  store1(static_cast<T*>(a.y) + i * a.ld_y + j, (float)sum * a.x_scales[i] * a.w_scales[j]);
}

// Rows of k codes at any byte, copied to rows of whole units with zeros behind.
__global__ __launch_bounds__(256) void i8_pack_kernel(const int8_t* src, size_t ld, int k, int8_t* dst, size_t ld_dst, int rows) {
  const int units = (int)(ld_dst / 16);
  const size_t at = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= (size_t)rows * units) return;
  const size_t row = at / units;
  const int u = (int)(at - row * units);
  *reinterpret_cast<i32x4_t*>(dst + row * ld_dst + 16 * u) = load16(src + row * ld + 16 * u, k - 16 * u);
}

template <class T, int MT, int NC>
Status launch_rows_of(hipStream_t stream, const I8Args& a) {
  const int tiles = (a.n + 16 * NC - 1) / (16 * NC), rows = (a.m + 16 * MT - 1) / (16 * MT);
  // A workgroup's four waves share the channels of one tile where the tiles alone would not fill the machine.
  if (tiles * rows >= 2048)
    matmul_i8_rows_kernel<T, MT, NC, 1><<<dim3((tiles + 3) / 4, rows), 256, 0, stream>>>(a);
  else
    matmul_i8_rows_kernel<T, MT, NC, 4><<<dim3(tiles, rows), 256, 0, stream>>>(a);
  PSSA_LAUNCH_CHECK("matmul_i8_rows_kernel");
  return Status::Ok();
}
template <class T>
Status launch_few(hipStream_t stream, const I8Args& a) {
  if (a.m <= 16) return launch_rows_of<T, 1, 1>(stream, a);
  if (a.m <= 32) return launch_rows_of<T, 2, 2>(stream, a);
  return launch_rows_of<T, 4, 2>(stream, a);
}

template <class T, int BM, int BN, int WM, int WN>
struct Tiles {
  static constexpr size_t kLds = 2 * (size_t)(BM + BN) * 128;
  static constexpr int kRows = BM, kChannels = BN, kThreads = 64 * WM * WN;
  static constexpr auto kKernel = &matmul_i8_tiles_kernel<T, BM, BN, WM, WN>;
};
template <class T>
using Large = Tiles<T, 256, 256, 2, 4>;
template <class T>
using Small = Tiles<T, 128, 128, 2, 2>;

template <class C, class T>
Status launch_tiles(hipStream_t stream, const I8Args& a) {
  const int tiles_m = (a.m + C::kRows - 1) / C::kRows, tiles_n = (a.n + C::kChannels - 1) / C::kChannels;
  C::kKernel<<<dim3((uint32_t)tiles_m * tiles_n, a.splits), C::kThreads, C::kLds, stream>>>(a, tiles_m, tiles_n);
  PSSA_LAUNCH_CHECK("matmul_i8_tiles_kernel");
  if (a.splits > 1) {
    matmul_i8_join_kernel<T><<<(uint32_t)(((size_t)a.m * a.n + 255) / 256), 256, 0, stream>>>(a);
    PSSA_LAUNCH_CHECK("matmul_i8_join_kernel");
  }
  return Status::Ok();
}

size_t tiles_of(size_t m, size_t n, size_t side) { return ((m + side - 1) / side) * ((n + side - 1) / side); }
bool large_tiles(size_t m, size_t n) { return tiles_of(m, n, 256) >= 3 * kComputeUnits / 4; }

template <class T>
Status launch_typed(hipStream_t stream, const I8Args& a) {
  if (a.m <= kI8FewRows) return launch_few<T>(stream, a);
  return large_tiles(a.m, a.n) ? launch_tiles<Large<T>, T>(stream, a) : launch_tiles<Small<T>, T>(stream, a);
}

Status launch_pack(hipStream_t stream, const int8_t*& p, size_t& ld, int k, int rows, char*& scratch) {
  const size_t to = ((size_t)k + 15) / 16 * 16;
  i8_pack_kernel<<<(uint32_t)((rows * (to / 16) + 255) / 256), 256, 0, stream>>>(p, ld, k, reinterpret_cast<int8_t*>(scratch), to, rows);
  PSSA_LAUNCH_CHECK("i8_pack_kernel");
  p = reinterpret_cast<int8_t*>(scratch);
  ld = to;
  scratch += (rows * to + 255) & ~(size_t)255;
  return Status::Ok();
}
bool in_units(const void* p, size_t ld, size_t k) { return ((uintptr_t)p | ld | k) % 16 == 0; }

}  // namespace

I8Plan i8_plan(size_t m, size_t n, size_t k) {
  I8Plan p;
  if (m <= kI8FewRows) return p;
  const size_t rows = (k + 15) / 16 * 16;
  p.pack_bytes = ((m * rows + 255) & ~(size_t)255) + ((n * rows + 255) & ~(size_t)255);
  if (!large_tiles(m, n)) {
    // Two workgroups a compute unit, parts of four slabs or more.
    const size_t tiles = tiles_of(m, n, 128), slabs = (k + 127) / 128;
    p.splits = (int)std::max<size_t>(1, std::min(kComputeUnits * 2 / tiles, slabs / 4));
  }
  p.parts_bytes = p.splits > 1 ? (size_t)p.splits * m * n * 4 : 0;
  return p;
}

Status init_i8_attributes() {
  auto set = [](const void* f, size_t lds) -> Status {
    PSSA_HIP_TRY(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    return Status::Ok();
  };
  PSSA_RETURN_IF(set(reinterpret_cast<const void*>(Large<float>::kKernel), Large<float>::kLds));
  PSSA_RETURN_IF(set(reinterpret_cast<const void*>(Large<Bf16>::kKernel), Large<Bf16>::kLds));
  PSSA_RETURN_IF(set(reinterpret_cast<const void*>(Small<float>::kKernel), Small<float>::kLds));
  return set(reinterpret_cast<const void*>(Small<Bf16>::kKernel), Small<Bf16>::kLds);
}

Status launch_matmul_i8(hipStream_t stream, int y_dtype, I8Args a, const I8Plan& p, void* scratch) {
  if (a.m > kI8FewRows) {
    a.splits = p.splits;
    a.parts = static_cast<int32_t*>(scratch);
    char* at = static_cast<char*>(scratch) + ((p.parts_bytes + 255) & ~(size_t)255);
    if (!in_units(a.x, a.ld_x, (size_t)a.k)) PSSA_RETURN_IF(launch_pack(stream, a.x, a.ld_x, a.k, a.m, at));
    if (!in_units(a.w, a.ld_w, (size_t)a.k)) PSSA_RETURN_IF(launch_pack(stream, a.w, a.ld_w, a.k, a.n, at));
    a.k = (a.k + 15) / 16 * 16;
  }
  return y_dtype == PSSA_HIP_F32 ? launch_typed<float>(stream, a) : launch_typed<Bf16>(stream, a);
}

}  // namespace pssa
