// Products of 8-bit rows and weights with a scale for each row and channel:
//   y[i][j] = x_scale[i] w_scale[j] sum_l x[i][l] w[j][l].
//
// The sums are whole numbers in 32 bits, exact, so neither tiles nor the order
// of a sum change a result; each y has the rounding of its sum to fp32, two of
// the scales, and the last one to bf16 where y is.
//
// Few rows read the weights straight into the matrix instructions' registers;
// many rows run in tiles whose slabs of 128 codes go from memory straight into
// LDS while others are multiplied.
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

// 16 codes at any byte: the dwords that hold them, moved into place.  A load of
// 16 bytes that does not begin at a dword takes the L1 several times as long
// (28 x 183 x 5817: 34 us, so 18).
__device__ __forceinline__ i32x4_t load_odd(const int8_t* p) {
  const uintptr_t at = (uintptr_t)p;
  const i32x4_t v = *reinterpret_cast<const i32x4_any_t*>(at & ~(uintptr_t)3);
  const int e = *reinterpret_cast<const int*>((at + 15) & ~(uintptr_t)3);
  const uint32_t by = (uint32_t)at & 3;
  return i32x4_t{(int)__builtin_amdgcn_alignbyte(v[1], v[0], by), (int)__builtin_amdgcn_alignbyte(v[2], v[1], by),
                 (int)__builtin_amdgcn_alignbyte(v[3], v[2], by), (int)__builtin_amdgcn_alignbyte(e, v[3], by)};
}
// 16 codes of a row of k, zeros past the `left` that the row still has: its last
// 16 moved down, in one load (byte by byte a row's end took 6 us).
__device__ __forceinline__ i32x4_t load16(const int8_t* p, int left, int k) {
  if (k < 16) {  // uniform
    i32x4_t v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 15; ++i)
      if (i < left) v[i >> 2] |= (int)(uint8_t)p[i] << (8 * (i & 3));
    return v;
  }
  const i32x4_t v = load_odd(p + min(left - 16, 0));
  const int off = 8 * max(16 - left, 0);  // bits
  const uint64_t lo = (uint32_t)v[0] | (uint64_t)(uint32_t)v[1] << 32, hi = (uint32_t)v[2] | (uint64_t)(uint32_t)v[3] << 32;
  const uint64_t l = off >= 128 ? 0 : off >= 64 ? hi >> (off & 63) : off ? lo >> off | hi << (64 - off) : lo, h = off >= 64 ? 0 : hi >> off;
  return i32x4_t{(int)l, (int)(l >> 32), (int)h, (int)(h >> 32)};
}

// ---------------------------------------------------------------- few rows
// A wave multiplies 16 MT rows by 16 NC channels over its part of k: WK waves
// of a workgroup share the channels, 4 / WK such groups lie side by side, and
// the parts meet in LDS.  Rows at any dword, or (ODD) at any byte.  Bound by the
// weights' way from memory (24 x 8192 x 8192: 16 us, 4.2 TB/s) or by the launch (1 x
// 16384 x 768: 5.1 us).
template <class T, int MT, int NC, int WK, bool ODD>
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
  auto load = [&](const int8_t* p) { return ODD ? load_odd(p) : *reinterpret_cast<const i32x4_any_t*>(p); };
  auto some = [&](int s, auto n) {
    constexpr int N = decltype(n)::value;
    i32x4_t xf[N][MT], wf[N][NC];
#pragma unroll
    for (int d = 0; d < N; ++d) {
#pragma unroll
      for (int c = 0; c < NC; ++c) wf[d][c] = load(w[c] + 64 * (s + d));
#pragma unroll
      for (int t = 0; t < MT; ++t) xf[d][t] = load(x[t] + 64 * (s + d));
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
      const i32x4_t wf = load16(w[c] + 64 * steps, left, a.k);
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[c][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf, load16(x[t] + 64 * steps, left, a.k), acc[c][t], 0, 0, 0);
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
constexpr int kLdsDone = ~(0xF << 8);  // of an s_waitcnt: lgkmcnt(0)

// Bytes between packed rows.
__host__ __device__ __forceinline__ size_t packed_ld(size_t k) { return (k + 127) / 128 * 128; }
// Channels of a row of parts: whole units of 16 bytes.
__host__ __device__ __forceinline__ size_t parts_ld(size_t n) { return (n + 3) / 4 * 4; }

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
// bytes, k a multiple of 16.  Slabs of 128 codes, whole cache lines, pass
// through R LDS buffers, 2 or 4.  A step of 32 codes' fragments are read while
// the step before is multiplied, across the slabs' border too, and the loads of
// the slab R - 1 ahead go out over R steps between the products: the L1 takes
// 16 cycles for each, all at once they held the products up.  At the end a
// wave's 32 rows at a time turn in LDS, so that what it stores is whole lines.
// 8192 x 8192 x 8192: 455 to 550 us, by the card's clock, which falls to 1.7
// GHz under this load (2.0 to 2.4 POP/s; stores of 8 bytes a row took 70 us
// more, rows whose units lay two to a bank 20).
template <class T, int BM, int BN, int WM, int WN, int R>
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

  // A slab row is 8 units of 16 codes; unit u of row r lies at u ^ (r / 2 & 7),
  // so that rows read at one unit hit different banks.  What a slab has behind
  // k, and slabs behind the last, are other codes of the row.
  uint32_t from[PER];  // the row, of the tile's first
  const int unit_k = 16 * ((threadIdx.x & 7) ^ (threadIdx.x >> 4 & 7));  // THREADS / 8 rows further it is the same
  constexpr int OF_X = BM * 8 / THREADS;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int row = (i * THREADS + (int)threadIdx.x) / 8;
    from[i] = i < OF_X ? (uint32_t)min(row, a.m - 1 - m0) * (uint32_t)a.ld_x : (uint32_t)min(row - BM, a.n - 1 - n0) * (uint32_t)a.ld_w;
  }
  const int8_t *x = a.x + (size_t)m0 * a.ld_x, *w = a.w + (size_t)n0 * a.ld_w;
  // Loads begin .. end - 1 of a slab.
  auto issue = [&](int slab, int begin, int end) {
    const int k0 = 128 * min(slab, last - 1);
    const uint32_t at = k0 + unit_k < a.k ? k0 + unit_k : k0;
    i32x4_t* buffer = s_tile + (slab - first) % R * UNITS;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (i < begin || i >= end) continue;
      auto* to = (__attribute__((address_space(3))) void*)(buffer + i * THREADS + wave * 64);
      const void* codes = (i < OF_X ? x : w) + (from[i] + at);
      __builtin_amdgcn_global_load_lds(codes, to, 16, 0, 0);
    }
  };
  i32x16_t acc[TN][TM];
#pragma unroll
  for (int b = 0; b < TN; ++b)
#pragma unroll
    for (int t = 0; t < TM; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[b][t][e] = 0;
  // Slab s is there for all waves, and s - 1 read by them.  Slabs behind the last are the last again.
  auto meet = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(vmcnt_only((R - 2) * PER) & kLdsDone);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  i32x4_t xf[2][TM], wf[2][TN];
  auto read = [&](int slab, auto step) {
    constexpr int S = decltype(step)::value;
    const i32x4_t* buffer = s_tile + (slab - first) % R * UNITS;
    const i32x4_t *sx = buffer + (wm * TM * 32 + l32) * 8, *sw = buffer + (BM + wn * TN * 32 + l32) * 8;
    const int u = (2 * S + half) ^ (l32 >> 1 & 7);
#pragma unroll
    for (int b = 0; b < TN; ++b) wf[S & 1][b] = sw[b * 256 + u];
#pragma unroll
    for (int t = 0; t < TM; ++t) xf[S & 1][t] = sx[t * 256 + u];
  };
  auto multiply = [&](int slab, auto step, bool end) {
    constexpr int S = decltype(step)::value;
    if (end)  // the sums may end inside the slab
#pragma unroll
      for (int t = 0; t < TM; ++t)
        if (128 * slab + 32 * S + 16 * half >= a.k) xf[S & 1][t] = i32x4_t{0, 0, 0, 0};
#pragma unroll
    for (int b = 0; b < TN; ++b)
#pragma unroll
      for (int t = 0; t < TM; ++t) acc[b][t] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[S & 1][b], xf[S & 1][t], acc[b][t], 0, 0, 0);
    // Reads and loads between the products.
#pragma unroll
    for (int i = 0; i < TM * TN; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, TM + TN, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
  constexpr std::integral_constant<int, 0> zero;
  constexpr std::integral_constant<int, 1> one;
  constexpr std::integral_constant<int, 2> two;
  constexpr std::integral_constant<int, 3> three;
  constexpr int P = (PER + R - 1) / R;  // loads of a step
  for (int r = 0; r < R - 1; ++r) issue(first + r, 0, PER);
  issue(first + R - 1, 0, P);
  meet();
  read(first, zero);
  auto pass = [&](int slab, bool end) {
    read(slab, one);
    issue(slab + R - 1, P, 2 * P);
    multiply(slab, zero, end);
    read(slab, two);
    if constexpr (R > 2) issue(slab + R - 1, 2 * P, 3 * P);
    multiply(slab, one, end);
    read(slab, three);
    if constexpr (R > 2) issue(slab + R - 1, 3 * P, 4 * P);
    multiply(slab, two, end);
    meet();
    issue(slab + R, 0, P);
    read(slab + 1, zero);
    multiply(slab, three, end);
  };
  for (int slab = first; slab < last - 1; ++slab) pass(slab, false);
  pass(last - 1, true);
  __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
  meet();  // all have read the slabs, and none is on its way
  // A lane holds channels 8 g + 4 half .. + 3 of each 32 of a row; a unit is 4
  // channels, unit u of row r lies at u ^ (r & 15).
  constexpr int ROW = TN * 8;
  static_assert(ROW == 16);
  i32x4_t* s_out = s_tile + wave * 32 * ROW;
  const int row0 = m0 + wm * TM * 32, ch0 = n0 + wn * TN * 32;
  auto each = [&](auto units, auto out) {
    constexpr int U = decltype(units)::value, AT_ONCE = 64 / (ROW / U);  // a lane's units, an instruction's rows
    const int u = lane % (ROW / U) * U, j = ch0 + 4 * u;
    float scales[4 * U];
#pragma unroll
    for (int c = 0; c < 4 * U; ++c) scales[c] = a.w_scales[min(j + c, a.n - 1)];
#pragma unroll
    for (int t = 0; t < TM; ++t) {
#pragma unroll
      for (int b = 0; b < TN; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          s_out[l32 * ROW + ((8 * b + 2 * g + half) ^ (l32 & 15))] = i32x4_t{acc[b][t][4 * g], acc[b][t][4 * g + 1], acc[b][t][4 * g + 2], acc[b][t][4 * g + 3]};
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int r0 = 0; r0 < 32; r0 += AT_ONCE) {
        const int r = r0 + lane / (ROW / U), i = row0 + 32 * t + r;
        i32x4_t v[U];
#pragma unroll
        for (int e = 0; e < U; ++e) v[e] = s_out[r * ROW + ((u + e) ^ (r & 15))];
        if (i < a.m && j < a.n) out(i, j, v, scales);
      }
      __builtin_amdgcn_wave_barrier();
    }
  };
  if (a.splits > 1)
    each(one, [&](int i, int j, const i32x4_t* v, const float*) {
      *reinterpret_cast<i32x4_t*>(a.parts + ((size_t)blockIdx.y * a.m + i) * parts_ld(a.n) + j) = v[0];
    });
  else if constexpr (sizeof(T) == 2)
    each(two, [&](int i, int j, const i32x4_t* v, const float* scales) {
      const float scale = a.x_scales[i];
      T* y = static_cast<T*>(a.y) + (size_t)i * a.ld_y + j;
      f32x4_t f[2];
#pragma unroll
      for (int c = 0; c < 8; ++c) f[c / 4][c % 4] = (float)v[c / 4][c % 4] * scale * scales[c];
      if (a.n - j >= 8)
        *reinterpret_cast<i32x4_any_t*>(y) = i32x4_t{(int)bf16x2_bits(f[0][0], f[0][1]), (int)bf16x2_bits(f[0][2], f[0][3]),
                                                     (int)bf16x2_bits(f[1][0], f[1][1]), (int)bf16x2_bits(f[1][2], f[1][3])};
      else {
        store4(y, f[0], a.n - j);
        store4(y + 4, f[1], a.n - j - 4);
      }
    });
  else
    each(one, [&](int i, int j, const i32x4_t* v, const float* scales) {
      const float scale = a.x_scales[i];
      f32x4_t f;
#pragma unroll
      for (int c = 0; c < 4; ++c) f[c] = (float)v[0][c] * scale * scales[c];
      store4(static_cast<T*>(a.y) + (size_t)i * a.ld_y + j, f, a.n - j);
    });
}

// The parts of k summed, and scaled: four channels a thread, rows along y (two
// parts of 1024 x 4096: 11 us, 4 TB/s).
template <class T>
__global__ __launch_bounds__(256) void matmul_i8_join_kernel(I8Args a) {
  const size_t ld = parts_ld(a.n), all = a.m * ld, at = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= all) return;
  i32x4_t sum = {0, 0, 0, 0};
  for (int s = 0; s < a.splits; ++s) sum += *reinterpret_cast<const i32x4_t*>(a.parts + s * all + at);
  const size_t i = at / ld;
  const int j = (int)(at - i * ld);
  const float scale = a.x_scales[i];
  f32x4_t y;
#pragma unroll
  for (int c = 0; c < 4; ++c) y[c] = (float)sum[c] * scale * a.w_scales[min(j + c, a.n - 1)];
  store4(static_cast<T*>(a.y) + i * a.ld_y + j, y, a.n - j);
}

// Rows of k codes at any byte, copied to rows that begin at cache lines (at 16
// bytes their slabs would lie in two: 1021 x 5003 x 4100 7 us more), zeros up to a
// unit's end:
// x's and the weights' in one launch (25 MB: 9.6 us, 5 TB/s).
struct Packed {
  const int8_t* src;
  size_t ld;
  int8_t* dst;
  int rows;  // 0 where the rows are used as they are
};
__global__ __launch_bounds__(256) void i8_pack_kernel(Packed x, Packed w, int k, int units) {
  size_t at = (size_t)blockIdx.x * 256 + threadIdx.x;
  const size_t of_x = (size_t)x.rows * units;
  const Packed p = at < of_x ? x : w;
  if (at >= of_x) at -= of_x;
  if (at >= (size_t)p.rows * units) return;
  const size_t row = at / units;
  const int u = (int)(at - row * units);
  *reinterpret_cast<i32x4_t*>(p.dst + row * packed_ld(k) + 16 * u) = load16(p.src + row * p.ld + 16 * u, k - 16 * u, k);
}

template <class T, int MT, int NC, bool ODD>
Status launch_rows_of(hipStream_t stream, const I8Args& a) {
  const int tiles = (a.n + 16 * NC - 1) / (16 * NC), rows = (a.m + 16 * MT - 1) / (16 * MT);
  // A workgroup's four waves share the channels of one tile where the tiles alone would not fill the machine.
  if (tiles * rows >= 2048)
    matmul_i8_rows_kernel<T, MT, NC, 1, ODD><<<dim3((tiles + 3) / 4, rows), 256, 0, stream>>>(a);
  else
    matmul_i8_rows_kernel<T, MT, NC, 4, ODD><<<dim3(tiles, rows), 256, 0, stream>>>(a);
  PSSA_LAUNCH_CHECK("matmul_i8_rows_kernel");
  return Status::Ok();
}
template <class T, bool ODD>
Status launch_few_at(hipStream_t stream, const I8Args& a) {
  // 32 channels a workgroup leave most of the machine idle below some 2000 of
  // them: 16 by 16 rows read the codes more often, in more places at once (64 x
  // 2048 x 4096: 14.7 -> 9.1 us, 28 x 183 x 5817: 18 -> 9.5; 64 x 4096 x 4096 would
  // lose a tenth).
  if (a.m <= 16 || a.n <= 2048) return launch_rows_of<T, 1, 1, ODD>(stream, a);
  if (a.m <= 32) return launch_rows_of<T, 2, 2, ODD>(stream, a);
  return launch_rows_of<T, 4, 2, ODD>(stream, a);
}
template <class T>
Status launch_few(hipStream_t stream, const I8Args& a) {
  const bool odd = ((uintptr_t)a.x | a.ld_x | (uintptr_t)a.w | a.ld_w) % 4 != 0;
  return odd ? launch_few_at<T, true>(stream, a) : launch_few_at<T, false>(stream, a);
}

template <class T, int BM, int BN, int WM, int WN, int R>
struct Tiles {
  static constexpr size_t kLds = R * (size_t)(BM + BN) * 128;
  static constexpr int kRows = BM, kChannels = BN, kThreads = 64 * WM * WN;
  static constexpr auto kKernel = &matmul_i8_tiles_kernel<T, BM, BN, WM, WN, R>;
};
template <class T>
using Large = Tiles<T, 256, 256, 2, 4, 2>;
template <class T>
using Small = Tiles<T, 128, 128, 2, 2, 2>;
template <class T>
using Deep = Tiles<T, 128, 128, 2, 2, 4>;
template <class T>
using Tall = Tiles<T, 192, 128, 2, 2, 4>;

template <class C, class T>
Status launch_tiles(hipStream_t stream, const I8Args& a) {
  const int tiles_m = (a.m + C::kRows - 1) / C::kRows, tiles_n = (a.n + C::kChannels - 1) / C::kChannels;
  C::kKernel<<<dim3((uint32_t)tiles_m * tiles_n, a.splits), C::kThreads, C::kLds, stream>>>(a, tiles_m, tiles_n);
  PSSA_LAUNCH_CHECK("matmul_i8_tiles_kernel");
  if (a.splits > 1) {
    matmul_i8_join_kernel<T><<<(uint32_t)((a.m * parts_ld(a.n) / 4 + 255) / 256), 256, 0, stream>>>(a);
    PSSA_LAUNCH_CHECK("matmul_i8_join_kernel");
  }
  return Status::Ok();
}

size_t tiles_of(size_t m, size_t n, size_t side) { return ((m + side - 1) / side) * ((n + side - 1) / side); }
bool large_tiles(size_t m, size_t n) { return tiles_of(m, n, 256) >= 3 * kComputeUnits / 4; }

template <class T>
Status launch_typed(hipStream_t stream, const I8Args& a) {
  if (a.m <= kI8FewRows) return launch_few<T>(stream, a);
  if (large_tiles(a.m, a.n)) return launch_tiles<Large<T>, T>(stream, a);
  // 192 rows where these get by with a workgroup a compute unit and 128 do not
  // (1024 x 5120 x 4096: 31 us, 34 with 128 rows; 1500 x 4000 x 2048: 20 and 21,
  // x 512: 12 and 11).
  if (a.k >= 1024 && tiles_of(a.m, a.n, 128) > kComputeUnits && ((size_t)a.m + 191) / 192 * (((size_t)a.n + 127) / 128) <= kComputeUnits)
    return launch_tiles<Tall<T>, T>(stream, a);
  // A workgroup a compute unit has room for four buffers (1024 x 4096 x 4096:
  // 25 us, with two 28), more than that share it with two each (1024 x 5120 x
  // 4096: 34 us, one after the other 40).
  return tiles_of(a.m, a.n, 128) * a.splits <= kComputeUnits ? launch_tiles<Deep<T>, T>(stream, a) : launch_tiles<Small<T>, T>(stream, a);
}

}  // namespace

// Also offsets inside a tile's rows of 32 bits.
bool i8_in_units(const void* p, size_t ld, size_t k) { return ((uintptr_t)p | ld | k) % 16 == 0 && ld <= (size_t)1 << 24; }

I8Plan i8_plan(size_t m, size_t n, size_t k, bool copy_x, bool copy_w) {
  I8Plan p;
  if (m <= kI8FewRows) return p;
  p.pack_bytes = (copy_x ? (m * packed_ld(k) + 255) & ~(size_t)255 : 0) + (copy_w ? n * packed_ld(k) : 0);
  if (!large_tiles(m, n)) {
    // Parts of four slabs or more, for a workgroup a compute unit: two, of half
    // the slabs each, have twice the sums to join (1024 x 4096 x 4096 37 us, so 28).
    const size_t tiles = tiles_of(m, n, 128), slabs = (k + 127) / 128;
    p.splits = (int)std::max<size_t>(1, std::min(kComputeUnits / tiles, slabs / 4));
  }
  p.parts_bytes = p.splits > 1 ? p.splits * m * parts_ld(n) * 4 : 0;
  return p;
}

Status init_i8_attributes() {
  auto set = [](const void* f, size_t lds) -> Status {
    PSSA_HIP_TRY(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    return Status::Ok();
  };
  PSSA_RETURN_IF(set(reinterpret_cast<const void*>(Large<float>::kKernel), Large<float>::kLds));
  PSSA_RETURN_IF(set(reinterpret_cast<const void*>(Large<Bf16>::kKernel), Large<Bf16>::kLds));
  PSSA_RETURN_IF(set(reinterpret_cast<const void*>(Tall<float>::kKernel), Tall<float>::kLds));
  PSSA_RETURN_IF(set(reinterpret_cast<const void*>(Tall<Bf16>::kKernel), Tall<Bf16>::kLds));
  PSSA_RETURN_IF(set(reinterpret_cast<const void*>(Deep<float>::kKernel), Deep<float>::kLds));
  PSSA_RETURN_IF(set(reinterpret_cast<const void*>(Deep<Bf16>::kKernel), Deep<Bf16>::kLds));
  PSSA_RETURN_IF(set(reinterpret_cast<const void*>(Small<float>::kKernel), Small<float>::kLds));
  return set(reinterpret_cast<const void*>(Small<Bf16>::kKernel), Small<Bf16>::kLds);
}

Status launch_matmul_i8(hipStream_t stream, int y_dtype, I8Args a, const I8Plan& p, void* scratch) {
  if (a.m > kI8FewRows) {
    a.splits = p.splits;
    a.parts = static_cast<int32_t*>(scratch);
    char* at = static_cast<char*>(scratch) + ((p.parts_bytes + 255) & ~(size_t)255);
    const size_t units = ((size_t)a.k + 15) / 16;
    Packed x{a.x, a.ld_x, reinterpret_cast<int8_t*>(at), i8_in_units(a.x, a.ld_x, (size_t)a.k) ? 0 : a.m};
    Packed w{a.w, a.ld_w, reinterpret_cast<int8_t*>(at + ((x.rows * packed_ld((size_t)a.k) + 255) & ~(size_t)255)), i8_in_units(a.w, a.ld_w, (size_t)a.k) ? 0 : a.n};
    if (x.rows || w.rows) {
      i8_pack_kernel<<<(uint32_t)((((size_t)x.rows + w.rows) * units + 255) / 256), 256, 0, stream>>>(x, w, a.k, (int)units);
      PSSA_LAUNCH_CHECK("i8_pack_kernel");
    }
    if (x.rows) a.x = x.dst, a.ld_x = packed_ld((size_t)a.k);
    if (w.rows) a.w = w.dst, a.ld_w = packed_ld((size_t)a.k);
    a.k = (a.k + 15) / 16 * 16;
  }
  return y_dtype == PSSA_HIP_F32 ? launch_typed<float>(stream, a) : launch_typed<Bf16>(stream, a);
}

}  // namespace pssa
