// Products of a few rows with 4-bit weights: y[m, n] = x[m, k] W^T with
// W[n][k] = scale * (code - zero), scale and zero shared by a group of 32, 64
// or 128 neighbours in a row.
//
// The weights are laid out once, for the matrix cores' operand: a tile of 16
// rows x 128 columns is one 16-byte piece for each lane of a wave, so a
// wave's load is 1 KB in a row.  Lane l holds row l % 16; its word j carries
// columns 32 j + 8 (l / 16) .. + 7, one v_mfma_f32_16x16x32_bf16 operand.
//
// A code q is kept as the odd integer 2 q - 15 in sign and magnitude: eight
// magnitudes, which one byte permute looks up for four codes at a time, so the
// operand's bf16 values cost 14 instructions for 8 codes and are exact.  With
// X the group's sum of x (the same instruction on a row of ones)
//   sum (q - z) x = (sum (2 q - 15) x + (15 - 2 z) X) / 2,
// and since the integers are centred nothing large cancels.  fp32 rows enter
// as three bf16 parts (8 + 8 + 8 bits, together exact), each a column of its
// own: the products are exact in fp32 whatever the type.
#include <algorithm>
#include <type_traits>

#include "operators.h"

namespace pssa {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef u32x4_t u32x4_any_t __attribute__((aligned(2)));
typedef f32x4_t f32x4_any_t __attribute__((aligned(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef u32x2_t u32x2_any_t __attribute__((aligned(1)));

// The 8 codes of a word as bf16 odd integers: 1, 3 .. 15 by the low three
// bits, the sign in the fourth; codes 0..3 in the low nibbles, 4..7 above.
__device__ __forceinline__ bf16x8_t w4_operand(uint32_t w) {
  const uint32_t lo = w & 0x07070707u, hi = (w >> 4) & 0x07070707u;
  const uint32_t hl = __builtin_amdgcn_perm(0x41414141u, 0x4040403Fu, lo) | (w & 0x08080808u) << 4;
  const uint32_t ll = __builtin_amdgcn_perm(0x70503010u, 0xE0A04080u, lo);
  const uint32_t hh = __builtin_amdgcn_perm(0x41414141u, 0x4040403Fu, hi) | (w & 0x80808080u);
  const uint32_t lh = __builtin_amdgcn_perm(0x70503010u, 0xE0A04080u, hi);
  const u32x4_t v = {__builtin_amdgcn_perm(hl, ll, 0x05010400u), __builtin_amdgcn_perm(hl, ll, 0x07030602u),
                     __builtin_amdgcn_perm(hh, lh, 0x05010400u), __builtin_amdgcn_perm(hh, lh, 0x07030602u)};
  return __builtin_bit_cast(bf16x8_t, v);
}

// Four codes as held: |2 q - 15| / 2 in the low three bits (q ^ 15 below 8,
// q ^ 8 from there), the sign in the fourth.
__device__ __forceinline__ uint32_t held4(uint32_t q) {
  q &= 0x0F0F0F0Fu;
  return q ^ 0x08080808u ^ (((q >> 3 & 0x01010101u) ^ 0x01010101u) * 7u);
}
// Codes [n, k], one byte each, into the tiles: 8 codes to a load.  134 million
// of them (16384 x 8192) take 38 us, 5.3 TB/s; byte by byte they took 250.
__global__ __launch_bounds__(256) void w4_pack_kernel(const uint8_t* __restrict__ codes, int n, int k, int kblocks,
                                                      size_t pieces, u32x4_t* __restrict__ out) {
  const size_t piece = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (piece >= pieces) return;
  const int lane = (int)(piece & 63), kb = (int)((piece >> 6) % kblocks);
  const size_t row = (piece >> 6) / kblocks * 16 + (lane & 15);
  u32x4_t v;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int col = 128 * kb + 32 * j + 8 * (lane >> 4);
    const uint8_t* src = codes + row * k + col;
    uint32_t q[2] = {0x08080808u, 0x08080808u};
    if (row < (size_t)n && col + 8 <= k) {
      const u32x2_any_t u = *reinterpret_cast<const u32x2_any_t*>(src);
      q[0] = u[0];
      q[1] = u[1];
    } else if (row < (size_t)n) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < k) q[i >> 2] = (q[i >> 2] & ~(0xFFu << 8 * (i & 3))) | (uint32_t)src[i] << 8 * (i & 3);
    }
    v[j] = held4(q[0]) | held4(q[1]) << 4;
  }
  out[piece] = v;
}

// Half of each group's scale, and its zero point, as the accumulators' rows
// need them: [tile][group][16 rows]; 0 past the matrix.
__global__ __launch_bounds__(256) void w4_scales_kernel(const float* __restrict__ scales,
                                                        const uint8_t* __restrict__ zeros, int n, int groups,
                                                        int groups_held, size_t count, float* __restrict__ out_scale,
                                                        uint8_t* __restrict__ out_zero) {
  const size_t at = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= count) return;
  const int g = (int)((at >> 4) % groups_held);
  const size_t row = (at >> 4) / groups_held * 16 + (at & 15);
  const bool in = row < (size_t)n && g < groups;
  out_scale[at] = in ? 0.5f * scales[row * groups + g] : 0.0f;
  if (out_zero) out_zero[at] = in ? zeros[row * groups + g] : 8;
}

struct MatvecArgs {
  const void* x = nullptr;
  size_t ld_x = 0;
  const u32x4_t* w = nullptr;
  const float* scales = nullptr;
  const uint8_t* zeros = nullptr;
  float* y = nullptr;
  size_t ld_y = 0;
  int m = 0, n = 0, k = 0, kblocks = 0, tiles = 0;
};

// The bf16 parts of an fp32 value: 8 significant bits each, the rest exact.
__device__ __forceinline__ void split3(float v, uint32_t (&part)[3]) {
  const uint32_t u = __float_as_uint(v);
  const float r1 = v - __uint_as_float(u & 0xFFFF0000u);
  const uint32_t u1 = __float_as_uint(r1);
  const float r2 = r1 - __uint_as_float(u1 & 0xFFFF0000u);
  part[0] = u;
  part[1] = u1;
  part[2] = __float_as_uint(r2);
}
// The upper halves of two words side by side.
__device__ __forceinline__ uint32_t upper2(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// A workgroup of waves that share NT tiles of 16 weight rows and split k;
// CT column tiles of 16 hold the rows of x (three columns a row for fp32).
// GROUP: a scale's columns.  The order of a row's sums depends on n and k alone.
template <bool F32, int CT, int NT, int GROUP>
__global__ __launch_bounds__(512) void matvec_w4_kernel(MatvecArgs a) {
  constexpr int P = F32 ? 3 : 1, ROWS = 16 * CT / P, PIECES = F32 ? (ROWS * 16 + 63) / 64 : 0;
  constexpr int PER = GROUP / 32, NG = 4 / PER;  // words of a group, groups of a block
  extern __shared__ char lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int waves = blockDim.x >> 6, col = lane & 15, quad = lane >> 4;
  const int row0 = blockIdx.y * ROWS, rows = min(ROWS, a.m - row0), cols = rows * P;
  const int tile0 = blockIdx.x * NT;
  const int kb0 = (int)((long)a.kblocks * wave / waves), kb1 = (int)((long)a.kblocks * (wave + 1) / waves);

  u32x4_t* s_x = reinterpret_cast<u32x4_t*>(lds) + (F32 ? wave * 16 * cols : 0);  // fp32: [16 k pieces][cols]
  const u32x4_t ones_u = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
  const bf16x8_t ones = __builtin_bit_cast(bf16x8_t, ones_u);
  f32x4_t total[NT][CT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int c = 0; c < CT; ++c) total[t][c] = f32x4_t{0, 0, 0, 0};

  // What one block of 128 columns needs from memory, fetched one block ahead.
  // WHOLE: every column is there, and the loads are the same in every block:
  // behind a load that may not have been made the compiler waits for all.
  struct Block {
    u32x4_t w[NT];
    f32x4_t s[NT][NG];
    uint32_t z[NT][NG];
    u32x4_t xh[F32 ? 1 : 4][F32 ? 1 : CT];
    f32x4_t xf[F32 ? PIECES : 1][2];
  };
  const uint8_t* zeros = a.zeros ? a.zeros : reinterpret_cast<const uint8_t*>(a.scales);  // loaded, then not used
  auto fetch = [&](Block& b, int kb, auto whole) {
    constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const size_t tile = min(tile0 + t, a.tiles - 1);
      b.w[t] = a.w[(tile * a.kblocks + kb) * 64 + lane];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const size_t at = ((tile * a.kblocks + kb) * NG + g) * 16 + 4 * quad;
        b.s[t][g] = *reinterpret_cast<const f32x4_t*>(a.scales + at);
        b.z[t][g] = *reinterpret_cast<const uint32_t*>(zeros + at);
      }
    }
    if constexpr (F32) {
#pragma unroll
      for (int q = 0; q < PIECES; ++q) {
        const int piece = min(lane + 64 * q, rows * 16 - 1), r = piece >> 4, c = 128 * kb + 8 * (piece & 15);
        const float* src = static_cast<const float*>(a.x) + (size_t)(row0 + r) * a.ld_x + c;
        if (WHOLE || c + 8 <= a.k) {
          b.xf[q][0] = *reinterpret_cast<const f32x4_any_t*>(src);
          b.xf[q][1] = *reinterpret_cast<const f32x4_any_t*>(src + 4);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) b.xf[q][i >> 2][i & 3] = c + i < a.k ? src[i] : 0.0f;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const int c = 128 * kb + 32 * j + 8 * quad;
          const uint16_t* src =
              static_cast<const uint16_t*>(a.x) + (size_t)(row0 + min(16 * ct + col, rows - 1)) * a.ld_x + c;
          if (WHOLE || c + 8 <= a.k) {
            b.xh[j][ct] = *reinterpret_cast<const u32x4_any_t*>(src);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              b.xh[j][ct][i] = (c + 2 * i < a.k ? src[2 * i] : 0u) | (c + 2 * i + 1 < a.k ? (uint32_t)src[2 * i + 1] << 16 : 0u);
          }
        }
    }
  };
  auto compute = [&](const Block& b) {
    if constexpr (F32) {  // the wave's own part of LDS: columns 3 r + part
      wave_sync();
#pragma unroll
      for (int q = 0; q < PIECES; ++q) {
        const int piece = lane + 64 * q, r = piece >> 4;
        if (piece < rows * 16) {
          u32x4_t part[3];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t p0[3], p1[3];
            split3(b.xf[q][i >> 1][2 * (i & 1)], p0);
            split3(b.xf[q][i >> 1][2 * (i & 1) + 1], p1);
#pragma unroll
            for (int p = 0; p < 3; ++p) part[p][i] = upper2(p0[p], p1[p]);
          }
#pragma unroll
          for (int p = 0; p < 3; ++p) s_x[(piece & 15) * cols + 3 * r + p] = part[p];
        }
      }
      wave_sync();
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      f32x4_t acc[NT][CT], sum[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        sum[ct] = f32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t][ct] = f32x4_t{0, 0, 0, 0};
      }
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int j = g * PER + i;
        bf16x8_t xb[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          if constexpr (F32)
            xb[ct] = __builtin_bit_cast(bf16x8_t, s_x[(4 * j + quad) * cols + min(16 * ct + col, cols - 1)]);
          else
            xb[ct] = __builtin_bit_cast(bf16x8_t, b.xh[j][ct]);
          sum[ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, xb[ct], sum[ct], 0, 0, 0);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const bf16x8_t wb = w4_operand(b.w[t][j]);
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
            acc[t][ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb, xb[ct], acc[t][ct], 0, 0, 0);
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float zc = a.zeros ? 15.0f - 2.0f * (float)((b.z[t][g] >> (8 * r)) & 0xFFu) : -1.0f;
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
            total[t][ct][r] = fmaf(b.s[t][g][r], fmaf(zc, sum[ct][r], acc[t][ct][r]), total[t][ct][r]);
        }
    }
  };
  const int kb_whole = min(kb1, a.k / 128);
  Block cur;
  if (kb0 < kb_whole) fetch(cur, kb0, std::true_type{});
  for (int kb = kb0; kb < kb_whole; ++kb) {
    Block next;
    fetch(next, min(kb + 1, kb_whole - 1), std::true_type{});
    compute(cur);
    cur = next;
  }
  if (max(kb0, kb_whole) < kb1) {  // the last block, of fewer columns
    fetch(cur, kb1 - 1, std::false_type{});
    compute(cur);
  }

  // The waves' and the parts' sums, in order.
  __syncthreads();
  float* s_sum = reinterpret_cast<float*>(lds);  // [waves][NT][16 CT columns][16 rows]
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
      *reinterpret_cast<f32x4_t*>(s_sum + (((size_t)wave * NT + t) * 16 * CT + 16 * ct + col) * 16 + 4 * quad) = total[t][ct];
  __syncthreads();
  for (int o = tid; o < rows * NT * 16; o += blockDim.x) {
    const int r = o / (NT * 16), t = o / 16 % NT, row = (tile0 + t) * 16 + o % 16;
    if (row >= a.n) continue;
    float v = 0.0f;
    for (int w = 0; w < waves; ++w)
#pragma unroll
      for (int p = 0; p < P; ++p) v += s_sum[(((size_t)w * NT + t) * 16 * CT + r * P + p) * 16 + o % 16];
    a.y[(size_t)(row0 + r) * a.ld_y + row] = v;
  }
}

template <bool F32, int CT, int NT, int GROUP>
Status launch_one(hipStream_t stream, const MatvecArgs& a, int waves) {
  constexpr int ROWS = 16 * CT / (F32 ? 3 : 1);
  const size_t stage = F32 ? (size_t)waves * 16 * ROWS * 3 * 16 : 0, sums = (size_t)waves * NT * CT * 16 * 16 * 4;
  const dim3 grid((a.tiles + NT - 1) / NT, (a.m + ROWS - 1) / ROWS);
  matvec_w4_kernel<F32, CT, NT, GROUP><<<grid, 64 * waves, std::max(stage, sums), stream>>>(a);
  PSSA_LAUNCH_CHECK("matvec_w4_kernel");
  return Status::Ok();
}

template <bool F32, int CT, int NT>
Status launch_group(hipStream_t stream, const MatvecArgs& a, int group, int waves) {
  if (group == 32) return launch_one<F32, CT, NT, 32>(stream, a, waves);
  if (group == 64) return launch_one<F32, CT, NT, 64>(stream, a, waves);
  return launch_one<F32, CT, NT, 128>(stream, a, waves);
}

template <bool F32, int NT>
Status launch_columns(hipStream_t stream, const MatvecArgs& a, int group, int waves) {
  const int cols = F32 ? 3 * a.m : a.m;
  if (cols <= 16) return launch_group<F32, 1, NT>(stream, a, group, waves);
  if constexpr (F32)
    if (cols > 32) return launch_group<F32, 3, NT>(stream, a, group, waves);
  return launch_group<F32, 2, NT>(stream, a, group, waves);
}

// Waves that split k: enough for some thousands in all, a block of 128 for each.
int split_waves(int workgroups, int most, int kblocks) {
  int w = 1;
  while (w < 8 && w * workgroups < most && w * 2 <= kblocks) w *= 2;
  return w;
}

}  // namespace

namespace {
// Fp32 rows of two or three column tiles stage up to 96 KB.
template <int CT, int NT, int GROUP>
Status big_lds() {
  PSSA_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(&matvec_w4_kernel<true, CT, NT, GROUP>),
                                   hipFuncAttributeMaxDynamicSharedMemorySize, 8 * 16 * 48 * 16));
  return Status::Ok();
}
template <int NT, int GROUP>
Status big_lds() {
  PSSA_RETURN_IF((big_lds<2, NT, GROUP>()));
  return big_lds<3, NT, GROUP>();
}
}  // namespace

Status init_w4_attributes() {
  PSSA_RETURN_IF((big_lds<1, 32>()));
  PSSA_RETURN_IF((big_lds<1, 64>()));
  PSSA_RETURN_IF((big_lds<1, 128>()));
  PSSA_RETURN_IF((big_lds<2, 32>()));
  PSSA_RETURN_IF((big_lds<2, 64>()));
  return big_lds<2, 128>();
}

size_t w4_packed_bytes(size_t n, size_t k) { return (n + 15) / 16 * ((k + 127) / 128) * 1024; }
size_t w4_groups_held(size_t n, size_t k, size_t group) { return (n + 15) / 16 * ((k + 127) / 128) * (128 / group) * 16; }

Status launch_w4_pack(hipStream_t stream, const uint8_t* codes, const float* scales, const uint8_t* zeros, int n, int k,
                      int group, void* packed, float* out_scales, uint8_t* out_zeros) {
  const int kblocks = (k + 127) / 128;
  const size_t pieces = w4_packed_bytes(n, k) / 16, count = w4_groups_held(n, k, group);
  w4_pack_kernel<<<(uint32_t)((pieces + 255) / 256), 256, 0, stream>>>(codes, n, k, kblocks, pieces,
                                                                       static_cast<u32x4_t*>(packed));
  PSSA_LAUNCH_CHECK("w4_pack_kernel");
  w4_scales_kernel<<<(uint32_t)((count + 255) / 256), 256, 0, stream>>>(
      scales, zeros, n, (k + group - 1) / group, kblocks * (128 / group), count, out_scales, zeros ? out_zeros : nullptr);
  PSSA_LAUNCH_CHECK("w4_scales_kernel");
  return Status::Ok();
}

Status launch_matvec_w4(hipStream_t stream, int x_dtype, const void* x, size_t ld_x, int m, const W4View& w, float* y,
                        size_t ld_y) {
  MatvecArgs a;
  a.x = x;
  a.ld_x = ld_x;
  a.w = static_cast<const u32x4_t*>(w.packed);
  a.scales = w.scales;
  a.zeros = w.zeros;
  a.y = y;
  a.ld_y = ld_y;
  a.m = m;
  a.n = w.n;
  a.k = w.k;
  a.kblocks = (w.k + 127) / 128;
  a.tiles = (w.n + 15) / 16;
  // fp32 rows are split into their parts once for NT tiles: with 7 of them and
  // 16384 x 8192 weights the kernel took 35.7, 29.2 and 27.8 us at NT 1, 2 and
  // 4 under the profiler, of which the last spills with smaller groups (a call
  // in a stream takes 26 us).  bf16 rows come as they are: one of them with
  // 16384 x 768 took 4.8 us at NT 1 and 2.
  if (x_dtype != PSSA_HIP_F32) return launch_columns<false, 1>(stream, a, w.group, split_waves(a.tiles, 4096, a.kblocks));
  if (a.tiles < 512) return launch_columns<true, 1>(stream, a, w.group, split_waves(a.tiles, 4096, a.kblocks));
  return launch_columns<true, 2>(stream, a, w.group, split_waves((a.tiles + 1) / 2, 2048, a.kblocks));
}

}  // namespace pssa
