// Token rows of linear attention and the delta rule: loads, bf16 parts, LDS
// tiles and the matrix instructions' operands.
#pragma once
#include "common.h"

namespace pssa {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef f32x4_t f32x4_any_t __attribute__((aligned(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef u32x2_t u32x2_any_t __attribute__((aligned(2)));

struct Bf16 {
  uint16_t bits;
};

// Four neighbouring elements in fp32, zeros past `left`.
template <class T>
__device__ __forceinline__ f32x4_t load4(const T* p, int left);
template <>
__device__ __forceinline__ f32x4_t load4<float>(const float* p, int left) {
  if (left >= 4) return *reinterpret_cast<const f32x4_any_t*>(p);
  f32x4_t v = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (i < left) v[i] = p[i];
  return v;
}
template <>
__device__ __forceinline__ f32x4_t load4<Bf16>(const Bf16* p, int left) {
  f32x4_t v = {0, 0, 0, 0};
  if (left >= 4) {
    const u32x2_t u = *reinterpret_cast<const u32x2_any_t*>(p);
    return f32x4_t{__uint_as_float(u[0] << 16), __uint_as_float(u[0] & 0xFFFF0000u), __uint_as_float(u[1] << 16),
                   __uint_as_float(u[1] & 0xFFFF0000u)};
  }
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (i < left) v[i] = __uint_as_float((uint32_t)p[i].bits << 16);
  return v;
}
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(Bf16* p, float v) { p->bits = bf16_bits_dev(v); }

// The arguments' tables are read from the kernel's argument segment.
typedef const __attribute__((address_space(4))) char* kernarg_t;

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef u32x4_t u32x4_any_t __attribute__((aligned(2)));

// Upper halves of two words side by side.
__device__ __forceinline__ uint32_t upper2(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
// Two fp32 values as bf16 parts: v = hi + lo to 2^-17 of it.
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = bf16x2_bits(a, b);
  lo = bf16x2_bits(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xFFFF0000u));
}
// As three parts of 8 bits each, exact.
__device__ __forceinline__ void split3(float a, float b, uint32_t& p0, uint32_t& p1, uint32_t& p2) {
  const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
  const float ra = a - __uint_as_float(ua & 0xFFFF0000u), rb = b - __uint_as_float(ub & 0xFFFF0000u);
  const uint32_t va = __float_as_uint(ra), vb = __float_as_uint(rb);
  p0 = upper2(ua, ub);
  p1 = upper2(va, vb);
  p2 = upper2(__float_as_uint(ra - __uint_as_float(va & 0xFFFF0000u)), __float_as_uint(rb - __uint_as_float(vb & 0xFFFF0000u)));
}
__device__ __forceinline__ f32x4_t mfma(const u32x4_t& a, const u32x4_t& b, const f32x4_t& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// Token rows of W columns lie in LDS as W / 8 units of 16 bytes, a row's units
// exchanged (twice is none) so that rows read at one unit hit different banks.
template <int W>
__device__ __forceinline__ int row_unit(int row, int u) {
  return W == 32 ? u ^ ((row >> 1) & 3) : u ^ (row & 7);
}
// Columns 8 u .. of a row: an operand in the rows' own order.
template <int W>
__device__ __forceinline__ u32x4_t row_frag(const u32x4_t* s, int row, int u) {
  return s[row * (W / 8) + row_unit<W>(row, u)];
}
// Columns c .. c + 3 (c in fours) of a row.
template <int W>
__device__ __forceinline__ u32x2_t four_of(const u32x4_t* s, int row, int c) {
  return reinterpret_cast<const u32x2_t*>(s + row * (W / 8) + row_unit<W>(row, c >> 3))[(c >> 2) & 1];
}
// Columns 32 kp + 4 quad .. + 3 and 16 more of a row: an operand in the accumulators' order.
template <int W>
__device__ __forceinline__ u32x4_t order_frag(const u32x4_t* s, int row, int kp, int quad) {
  const u32x2_t x = four_of<W>(s, row, 32 * kp + 4 * quad), y = four_of<W>(s, row, 32 * kp + 16 + 4 * quad);
  return u32x4_t{x[0], x[1], y[0], y[1]};
}
// Rows row0 + 4 quad .. + 3 and 16 more at column c0 + col (c0 in sixteens):
// 16 lanes read a 4 x 16 block, 4 columns each, and are handed its columns.
// The LDS address of the lane's part; the next sixteen columns are 32 bytes
// further but for the exchange, so theirs is an exclusive or.
template <int W>
__device__ __forceinline__ uint32_t turned_at(const u32x4_t* s, int row0, int c0, int lane) {
  const int row = row0 + 4 * (lane >> 4) + ((lane >> 2) & 3), c = c0 + 4 * (lane & 3);
  const u32x4_t* unit = s + row * (W / 8) + row_unit<W>(row, c >> 3);
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)unit + 8 * ((c >> 2) & 1);
}
// One fragment.  Written out, with their wait, because the compiler would let
// the builtin wait for the loads that are on their way into the other buffer.
template <int W>
__device__ __forceinline__ void turned_frag(uint32_t at, u32x4_t& v) {
  u32x2_t x, y;
  asm volatile("ds_read_b64_tr_b16 %0, %2\n\tds_read_b64_tr_b16 %1, %2 offset:%c3\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(x), "=&v"(y)
               : "v"(at), "i"(32 * W)
               : "memory");
  v = u32x4_t{x[0], x[1], y[0], y[1]};
}
// One of v and N neighbouring ones of k.
template <int WV, int WK, int N>
__device__ __forceinline__ void turned_frags(uint32_t av, u32x4_t& v, uint32_t ak, u32x4_t (&k)[N]) {
  static_assert(N == 2 || N == 4, "fragments of k");
  u32x2_t v0, v1, k0[N], k1[N];
  if constexpr (N == 4) {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %10\n\tds_read_b64_tr_b16 %1, %10 offset:%c15\n\t"
        "ds_read_b64_tr_b16 %2, %11\n\tds_read_b64_tr_b16 %3, %11 offset:%c16\n\t"
        "ds_read_b64_tr_b16 %4, %12\n\tds_read_b64_tr_b16 %5, %12 offset:%c16\n\t"
        "ds_read_b64_tr_b16 %6, %13\n\tds_read_b64_tr_b16 %7, %13 offset:%c16\n\t"
        "ds_read_b64_tr_b16 %8, %14\n\tds_read_b64_tr_b16 %9, %14 offset:%c16\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(v0), "=&v"(v1), "=&v"(k0[0]), "=&v"(k1[0]), "=&v"(k0[1]), "=&v"(k1[1]), "=&v"(k0[2]), "=&v"(k1[2]),
          "=&v"(k0[3]), "=&v"(k1[3])
        : "v"(av), "v"(ak), "v"(ak ^ 32), "v"(ak ^ 64), "v"(ak ^ 96), "i"(32 * WV), "i"(32 * WK)
        : "memory");
  } else {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %6\n\tds_read_b64_tr_b16 %1, %6 offset:%c9\n\t"
        "ds_read_b64_tr_b16 %2, %7\n\tds_read_b64_tr_b16 %3, %7 offset:%c10\n\t"
        "ds_read_b64_tr_b16 %4, %8\n\tds_read_b64_tr_b16 %5, %8 offset:%c10\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(v0), "=&v"(v1), "=&v"(k0[0]), "=&v"(k1[0]), "=&v"(k0[1]), "=&v"(k1[1])
        : "v"(av), "v"(ak), "v"(ak ^ 32), "i"(32 * WV), "i"(32 * WK)
        : "memory");
  }
  v = u32x4_t{v0[0], v0[1], v1[0], v1[1]};
#pragma unroll
  for (int i = 0; i < N; ++i) k[i] = u32x4_t{k0[i][0], k0[i][1], k1[i][0], k1[i][1]};
}

// Four more of k.
template <int WK>
__device__ __forceinline__ void turned_frags(uint32_t ak, u32x4_t (&k)[4]) {
  u32x2_t k0[4], k1[4];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%c12\n\t"
      "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%c12\n\t"
      "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:%c12\n\t"
      "ds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:%c12\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(k0[0]), "=&v"(k1[0]), "=&v"(k0[1]), "=&v"(k1[1]), "=&v"(k0[2]), "=&v"(k1[2]), "=&v"(k0[3]), "=&v"(k1[3])
      : "v"(ak), "v"(ak ^ 32), "v"(ak ^ 64), "v"(ak ^ 96), "i"(32 * WK)
      : "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i) k[i] = u32x4_t{k0[i][0], k0[i][1], k1[i][0], k1[i][1]};
}

constexpr int kLdsOnly = 0xF | (0x3 << 14) | (0x7 << 4);  // s_waitcnt lgkmcnt(0)

// Element i of bf16 values in a register or LDS.
template <class V>
__device__ __forceinline__ float bf16_at(const V* p, int i) {
  return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << 16);
}

// What stands in for rows and columns that are not there.
__device__ uint32_t g_nothing[4];

// Units of a row of W fp32 columns, exchanged like the bf16 ones.
__device__ __forceinline__ int row_unit32(int row, int u) { return u ^ (row & 7); }
template <int W>
__device__ __forceinline__ f32x4_t row_frag32(const f32x4_t* s, int row, int u) {
  return s[row * (W / 4) + row_unit32(row, u)];
}
template <int W>
__device__ __forceinline__ float element32(const f32x4_t* s, int row, int c) {
  return reinterpret_cast<const float*>(s + row * (W / 4) + row_unit32(row, c >> 2))[c & 3];
}
__device__ __forceinline__ f32x4_t mfma32(float a, float b, const f32x4_t& c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

}  // namespace
}  // namespace pssa
