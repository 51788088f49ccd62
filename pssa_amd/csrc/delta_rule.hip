// The gated delta rule over packed sequences, from one token to long prompts:
//   S_t = a_t (1 - beta_t k_t k_t^T) S_{t-1} + beta_t k_t v_t^T,   o_t = scale q_t S_t,
// a_t = exp(log_decay_t).  With u_t = beta_t (v_t - a_t k_t S_{t-1}) that is
//   S_t = a_t S_{t-1} + k_t u_t^T,   o_t = scale (a_t q_t S_{t-1} + (q_t k_t) u_t).
//
// Prompts run in chunks of 64 tokens (32 in fp32).  With G_i the sum of the
// chunk's log decays up to token i, and S the state that the chunk is entered
// with, the tokens' u solve a triangular system:
//   (1 + A) U = beta (V - e^G K S),   A_ij = beta_i e^(G_i - G_j) k_i k_j for j < i,
//   O = scale e^G Q S + P U,          P_ij = scale e^(G_i - G_j) q_i k_j for j <= i,
//   S' = e^(G_n) S + K^T (e^(G_n - G) U).
// T = (1 + A)^-1 beta needs no state: a first kernel works it out for all
// chunks at once (delta_ahead), a second one walks the chunks of a sequence, a
// head and 64 value columns with S in its registers (delta_walk).
// There everything follows in registers: the accumulators' layout (lane l
// holds column l % 16, rows 4 (l / 16) + r) is the next product's operand
// layout once what meets it is read in the same order.
#include <algorithm>
#include <cstddef>
#include <type_traits>

#include "attention_tiles.h"
#include "operators.h"

namespace pssa {
namespace {

template <class T>
__device__ __forceinline__ float load1(const T* p);
template <>
__device__ __forceinline__ float load1<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float load1<Bf16>(const Bf16* p) { return __uint_as_float((uint32_t)p->bits << 16); }

// The arguments lie first in the kernel's argument segment; indexing the
// struct itself would copy it to scratch.
__device__ __forceinline__ uint32_t inline_word(size_t offset, int i) {
  return reinterpret_cast<const __attribute__((address_space(4))) uint32_t*>(
      (kernarg_t)__builtin_amdgcn_kernarg_segment_ptr() + offset)[i];
}
__device__ __forceinline__ uint32_t first_token(const DeltaArgs& a, int seq) {
  return a.table ? a.table[seq] : inline_word(offsetof(DeltaArgs, inline_tokens), seq);
}
__device__ __forceinline__ int first_chunk(const DeltaArgs& a, int seq) {
  return (int)(a.table ? a.table[a.n_seqs + 1 + seq] : inline_word(offsetof(DeltaArgs, inline_chunks), seq));
}
__device__ __forceinline__ int first_item(const DeltaArgs& a, int seq) {
  return (int)(a.table ? a.table[2 * (a.n_seqs + 1) + seq] : inline_word(offsetof(DeltaArgs, inline_items), seq));
}
// A sequence's tokens.
struct Span {
  size_t tok;
  int len;
};
__device__ __forceinline__ Span span_of(const DeltaArgs& a, int seq) {
  if (a.uniform_len >= 0) return Span{(size_t)seq * a.uniform_len, a.uniform_len};
  const uint32_t tok = first_token(a, seq);
  return Span{tok, (int)(first_token(a, seq + 1) - tok)};
}

// The recurrence itself, the state read and written once.  A workgroup's
// threads lie over 64 of the state's columns, four each, and its rows, 16
// apart: 16 x 16.  k S and q S of a token meet in LDS together.  Bound by the
// states' way through memory: 256 streams of one token, 12 heads of 64 x 64, 22.5
// us, 4.5 TB/s.
template <class T, int ROWS>
__global__ __launch_bounds__(256) void delta_steps_kernel(DeltaArgs a) {
  __shared__ float s_kq[2][2][kDeltaMaxKey];
  __shared__ f32x4_t s_part[2][4][2][16];
  const int tid = threadIdx.x, ct = tid & 15, rt = tid >> 4, wave = tid >> 6;
  const int j = 4 * (blockIdx.x * 16 + ct), head = blockIdx.y, key_head = head / (a.heads / a.key_heads);
  const Span sp = span_of(a, blockIdx.z);
  const T* q0 = static_cast<const T*>(a.q) + (size_t)key_head * a.dk;
  const T* k0 = static_cast<const T*>(a.k) + (size_t)key_head * a.dk;
  const T* v0 = static_cast<const T*>(a.v) + (size_t)head * a.dv;
  T* o0 = static_cast<T*>(a.out) + (size_t)head * a.dv;
  const size_t state0 = ((size_t)blockIdx.z * a.heads + head) * a.dk * a.dv + j;
  const bool on = j < a.dv;
  const int left = a.dv - j;

  f32x4_t S[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int row = rt + 16 * i;
    S[i] = f32x4_t{0, 0, 0, 0};
    if (on && a.state_in && row < a.dk) S[i] = load4<float>(a.state_in + state0 + (size_t)row * a.dv, left);
  }
  for (int t = 0; t < sp.len; ++t) {
    const size_t tok = sp.tok + t;
    float(*kq)[kDeltaMaxKey] = s_kq[t & 1];
    if ((tid & 127) < a.dk) {
      const int d = tid & 127;
      kq[tid >> 7][d] = load1<T>(tid < 128 ? k0 + tok * a.ld_k + d : q0 + tok * a.ld_q + d);
    }
    const f32x4_t v = on ? load4<T>(v0 + tok * a.ld_v + j, left) : f32x4_t{0, 0, 0, 0};
    const float decay = expf(a.log_decay[tok * a.ld_gates + head]), beta = a.beta[tok * a.ld_gates + head];
    __syncthreads();
    f32x4_t ks = {0, 0, 0, 0}, qs = {0, 0, 0, 0};
    float qk = 0.0f;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int row = rt + 16 * i;
      if (row < a.dk) {
        const float kd = kq[0][row], qd = kq[1][row];
        qk = fmaf(qd, kd, qk);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          S[i][e] = decay == 0.0f ? 0.0f : S[i][e] * decay;
          ks[e] = fmaf(kd, S[i][e], ks[e]);
          qs[e] = fmaf(qd, S[i][e], qs[e]);
        }
      }
    }
#pragma unroll
    for (int off = 16; off <= 32; off <<= 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ks[e] += __shfl_xor(ks[e], off, 64);
        qs[e] += __shfl_xor(qs[e], off, 64);
      }
      qk += __shfl_xor(qk, off, 64);
    }
    __shared__ float s_qk[2][4];
    if ((tid & 63) < 16) {
      s_part[t & 1][wave][0][ct] = ks;
      s_part[t & 1][wave][1][ct] = qs;
      s_qk[t & 1][wave] = qk;
    }
    __syncthreads();
    ks = s_part[t & 1][0][0][ct];
    qs = s_part[t & 1][0][1][ct];
    qk = s_qk[t & 1][0];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      ks += s_part[t & 1][w][0][ct];
      qs += s_part[t & 1][w][1][ct];
      qk += s_qk[t & 1][w];
    }
    f32x4_t u;
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = beta * (v[e] - ks[e]);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int row = rt + 16 * i;
      if (row < a.dk) {
        const float kd = kq[0][row];
#pragma unroll
        for (int e = 0; e < 4; ++e) S[i][e] = fmaf(kd, u[e], S[i][e]);
      }
    }
    if (rt == 0 && on) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) store1(o0 + tok * a.ld_out + j + e, fmaf(qk, u[e], qs[e]) * a.scale);
    }
  }
  if (!a.state_out || !on) return;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int row = rt + 16 * i;
    if (row >= a.dk) continue;
    float* dst = a.state_out + state0 + (size_t)row * a.dv;
    if (left >= 4) {
      *reinterpret_cast<f32x4_any_t*>(dst) = S[i];
    } else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (e < left) dst[e] = S[i][e];
    }
  }
}

// ------------------------------------------------------------------- chunks
constexpr double kLog2e = 1.4426950408889634;
constexpr float kForget = -1e4f;  // a log decay below it forgets all the same, and its sums stay finite

// A chunk's place: its sequence's and its own first token, its tokens.
struct Place {
  size_t tok;
  int n;
};
template <int C>
__device__ __forceinline__ Place place_of(const DeltaArgs& a, int chunk) {
  if (a.uniform_len >= 0) {
    const int per = (a.uniform_len + C - 1) / C, seq = chunk / per, pos = (chunk - seq * per) * C;
    return Place{(size_t)seq * a.uniform_len + pos, min(C, a.uniform_len - pos)};
  }
  int lo = 0, hi = a.n_seqs - 1;  // the last sequence whose chunks begin at or before this one
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first_chunk(a, mid) <= chunk) lo = mid; else hi = mid - 1;
  }
  const int pos = (chunk - first_chunk(a, lo)) * C;
  const uint32_t tok = first_token(a, lo);
  return Place{(size_t)tok + pos, min(C, (int)(first_token(a, lo + 1) - tok) - pos)};
}

// What is worked out ahead for a chunk and head, in units of 16 bytes: T's
// tiles of 16 x 16 where its triangle holds anything, in fp32 for both types,
// then of the tokens e^G, e^(G_n - G) and G itself (Power).  T as two bf16 parts had the products for U at half the time (a
// chunk 0.4 us of 2.6), but what they drop comes back in every chunk's state,
// and grows where keys are alike: states were off by 5e-6 of their size, and
// are by 2e-7 so.  P's fragments are 16 tokens by 32 in three parts (bf16), 16 by
// 16 (fp32).
template <bool B16>
struct Ahead {
  static constexpr int C = B16 ? 64 : 32, kTiles = C / 16, kPairs = B16 ? 6 : 3, kFrag = B16 ? 192 : 64;
  static constexpr int kTriangle = kTiles * (kTiles + 1) / 2, kGamma = kTriangle * 64, kRest = kGamma + C / 4, kSum = kRest + C / 4, kUnits = kGamma + 64;
};
// The fragment of token tile t over keys 32 h .. (bf16), 16 h .. (fp32).
template <bool B16>
__device__ __forceinline__ constexpr int pair_of(int t, int h) {
  return B16 ? (t < 2 ? t : 2 * t - 2 + h) : t + h;
}
// The tiles of a lower triangle in a row: the row of the i-th, and its column.
__device__ __forceinline__ int triangle_row(int i) { return i >= 6 ? 3 : i >= 3 ? 2 : i >= 1 ? 1 : 0; }
__device__ __forceinline__ int triangle_col(int i) { return i - triangle_row(i) * (triangle_row(i) + 1) / 2; }

// Units of a row of W elements of a type lie exchanged in LDS, so that rows
// read at one unit hit different banks.
template <bool B16, int W>
__device__ __forceinline__ int unit_in_row(int row, int u) {
  if constexpr (B16) return row_unit<W>(row, u);
  return row_unit32(row, u);
}
// Rows x .. + 15 times rows y .. + 15 of two tiles in LDS: lane l holds row
// y + l % 16 and rows x + 4 (l / 16) + e.
template <bool B16, int DKP>
__device__ __forceinline__ f32x4_t tile_product(const u32x4_t* sx, int x, const u32x4_t* sy, int y, int lane) {
  const int col = lane & 15, quad = lane >> 4;
  f32x4_t s = {0, 0, 0, 0};
#pragma unroll
  for (int b = 0; b < DKP / (B16 ? 32 : 16); ++b) {
    constexpr int ROW = DKP / (B16 ? 8 : 4);
    const u32x4_t xf = sx[(x + col) * ROW + unit_in_row<B16, DKP>(x + col, 4 * b + quad)];
    const u32x4_t yf = sy[(y + col) * ROW + unit_in_row<B16, DKP>(y + col, 4 * b + quad)];
    if constexpr (B16) {
      s = mfma(xf, yf, s);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) s = mfma32(__uint_as_float(xf[e]), __uint_as_float(yf[e]), s);
    }
  }
  return s;
}

// e^G, G summed in 64 bits, as 2^(part + whole), part in +-1/2: in one fp32
// number the whole part would leave the exponential of a difference off by up
// to 22 roundings (at e^-29), so it is by 2.
struct Power {
  float part;
  int whole;
};
__device__ __forceinline__ Power power_of(double g) {
  const double d = g * kLog2e, whole = rint(d);
  return Power{(float)(d - whole), (int)whole};
}
// From LDS as 64 bits of a type of its own: read as any other, the compiler has
// it wait for the loads into LDS that are on their way.
__device__ __forceinline__ Power power_in(double bits) {
  return Power{__int_as_float(__double2loint(bits)), __double2hiint(bits)};
}
// e^(gi - gj) where `on`, else 0: no branch, as the loads of either would wait in it.
__device__ __forceinline__ float decay_between(const Power& gi, const Power& gj, bool on) {
  const float part = gi.part - gj.part;
  return ldexpf(__builtin_amdgcn_exp2f(on ? part : -INFINITY), gi.whole - gj.whole);
}

// A chunk of one head, a wave for each 16 tokens.  A's triangle lies in LDS;
// each wave inverts one of its diagonal blocks by substitution, a column a
// lane, and follows one column of blocks down:
//   T_rc = -D_r sum_j A_rj T_jc, c <= j < r.
// Some 7 us a workgroup's way, six of them to a compute unit: 16 x 1024 tokens, 12
// heads of 64 in 23 us, waits between its steps, no unit over a third busy.
template <bool B16, int DKP>
__global__ __launch_bounds__(B16 ? 256 : 128) void delta_ahead_kernel(DeltaArgs a) {
  using Out = Ahead<B16>;
  using T = std::conditional_t<B16, Bf16, float>;
  constexpr int C = Out::C, NT = Out::kTiles, LD = C + 4, N = 16 / (int)sizeof(T), ROW = DKP / N;
  __shared__ __attribute__((aligned(256))) u32x4_t s_k[C * ROW];
  __shared__ __attribute__((aligned(16))) float s_a[C * LD];
  __shared__ Power s_g[C];
  __shared__ float s_beta[C];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, quad = lane >> 4;
  const int head = a.head0 + blockIdx.y, key_head = head / (a.heads / a.key_heads);
  const Place pl = place_of<C>(a, blockIdx.x);
  u32x4_t* out = reinterpret_cast<u32x4_t*>(a.ahead) + ((size_t)blockIdx.x * a.heads_here + blockIdx.y) * Out::kUnits;
  const T* k0 = static_cast<const T*>(a.k) + pl.tok * a.ld_k + (size_t)key_head * a.wide_k;
#pragma unroll
  for (int i = 0; i < C * ROW / (64 * NT); ++i) {
    const int at = (i * NT + wave) * 64, unit = at + lane, row = unit / ROW, c = N * unit_in_row<B16, DKP>(row, unit % ROW);
    const void* src = row < pl.n && c < a.dk ? static_cast<const void*>(k0 + row * a.ld_k + c) : g_nothing;
    __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)(s_k + at), 16, 0, 0);
  }
  if (wave == 0) {
    const bool on = lane < pl.n;
    float g = on ? a.log_decay[(pl.tok + lane) * a.ld_gates + head] : 0.0f;
    g = g < kForget ? kForget : g;
    double sum = g;
#pragma unroll
    for (int off = 1; off < C; off <<= 1) {
      const double o = __shfl_up(sum, off, 64);
      if (lane >= off) sum += o;
    }
    const double all = __shfl(sum, C - 1, 64);
    if (lane < C) {
      const Power g_i = power_of(sum);
      s_g[lane] = g_i;
      s_beta[lane] = on ? a.beta[(pl.tok + lane) * a.ld_gates + head] : 0.0f;
      float* f = reinterpret_cast<float*>(out + Out::kGamma);
      f[lane] = decay_between(g_i, Power{0.0f, 0}, true);
      f[C + lane] = decay_between(power_of(all), g_i, true);
      reinterpret_cast<Power*>(out + Out::kSum)[lane] = g_i;
    }
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
  __syncthreads();
  // A: rows 16 r + 4 quad + e, columns 16 c + col.
#pragma unroll
  for (int i = 0; i < (NT * (NT + 1) / 2 + NT - 1) / NT; ++i) {
    const int at = min(i * NT + wave, NT * (NT + 1) / 2 - 1), r = triangle_row(at), c = triangle_col(at);
    const f32x4_t s = tile_product<B16, DKP>(s_k, 16 * r, s_k, 16 * c, lane);
    const Power gk = s_g[16 * c + col];
    float w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = 16 * r + 4 * quad + e;
      w[e] = s_beta[row] * decay_between(s_g[row], gk, row > 16 * c + col);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = 16 * r + 4 * quad + e;
      s_a[row * LD + 16 * c + col] = row > 16 * c + col ? s[e] * w[e] : 0.0f;
    }
  }
  __syncthreads();
  // The inverse of the wave's diagonal block, over its block.  First of its two
  // halves of 8 x 8, a column a lane: each row as soon as it is known leaves the
  // rows below (16 x 16 at once takes three times the products, and registers
  // that let three waves share a SIMD).
  {
    float* block = s_a + 16 * wave * LD + 16 * wave;
    const float* half = block + (col >> 3) * 8 * (LD + 1);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i == (col & 7) ? 1.0f : 0.0f;
    auto leave = [&](auto first) {
      constexpr int J = decltype(first)::value;
      f32x4_t w[8 - J];
#pragma unroll
      for (int i = 1; i < 8 - J; ++i) w[i] = *reinterpret_cast<const f32x4_t*>(half + (J + i) * LD + J);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 1; i < 8 - J; ++i)
          if (i > e) x[J + i] = fmaf(-w[i][e], x[J + e], x[J + i]);
    };
    leave(std::integral_constant<int, 0>{});
    leave(std::integral_constant<int, 4>{});
    wave_sync();
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (quad == (i & 3)) block[((col & 8) + i) * LD + col] = x[i];
    wave_sync();
    // The block between them: -X2 (A21 X1), an element a lane; the block above
    // holds A21 X1 meanwhile.
    const int r = lane >> 3, c = lane & 7;
    auto times = [&](const float* left, const float* right) {
      const f32x4_t l0 = *reinterpret_cast<const f32x4_t*>(left + r * LD), l1 = *reinterpret_cast<const f32x4_t*>(left + r * LD + 4);
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) sum = fmaf(l0[e], right[e * LD + c], sum);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum = fmaf(l1[e], right[(4 + e) * LD + c], sum);
      return sum;
    };
    const float y = times(block + 8 * LD, block);
    wave_sync();
    block[r * LD + 8 + c] = y;
    wave_sync();
    const float z = times(block + 8 * LD + 8, block + 8);
    wave_sync();
    block[(8 + r) * LD + c] = -z;
    block[r * LD + 8 + c] = 0.0f;
  }
  __syncthreads();
  // The wave's column of blocks.
  f32x4_t t[NT];
#pragma unroll
  for (int e = 0; e < 4; ++e) t[0][e] = s_a[(16 * wave + 4 * quad + e) * LD + 16 * wave + col];
#pragma unroll
  for (int d = 1; d < NT; ++d) {  // the block d rows below the diagonal
    const int r = wave + d;
    t[d] = f32x4_t{0, 0, 0, 0};
    if (r >= NT) continue;  // uniform
    f32x4_t z = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < d; ++j) {
      const f32x4_t w = *reinterpret_cast<const f32x4_t*>(s_a + (16 * r + col) * LD + 16 * (wave + j) + 4 * quad);
#pragma unroll
      for (int e = 0; e < 4; ++e) z = mfma32(w[e], t[j][e], z);
    }
    const f32x4_t inv = *reinterpret_cast<const f32x4_t*>(s_a + (16 * r + col) * LD + 16 * r + 4 * quad);
#pragma unroll
    for (int e = 0; e < 4; ++e) t[d] = mfma32(-inv[e], z[e], t[d]);
  }
  __syncthreads();
  const float beta = s_beta[16 * wave + col];
#pragma unroll
  for (int d = 0; d < NT; ++d) {
    if (wave + d >= NT) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) s_a[(16 * (wave + d) + 4 * quad + e) * LD + 16 * wave + col] = t[d][e] * beta;
  }
  __syncthreads();
  // T's rows as fragments.
#pragma unroll
  for (int i = 0; i < (Out::kTriangle + NT - 1) / NT; ++i) {
    const int at = i * NT + wave, r = triangle_row(at), c = triangle_col(at);
    if (at < Out::kTriangle)
      out[64 * at + lane] = *reinterpret_cast<const u32x4_t*>(s_a + (16 * r + col) * LD + 16 * c + 4 * quad);
  }
}

// How a walk runs: the whole of an unsplit call, a segment's own state and
// transition, or a segment's outputs from its entry state.
enum { DR_WHOLE, DR_LOCAL, DR_SEGMENT };

// LDS units of a walk: two buffers of k | q | v | what was worked out ahead,
// P, and what the walking waves hand over in fp32: S, and U (bf16: its first
// half in v's place).
template <bool B16, int DKP, bool LOCAL>
struct WalkLds {
  static constexpr int C = Ahead<B16>::C, N = B16 ? 8 : 4;  // elements of a unit
  static constexpr int kK = C * DKP / N, kQ = LOCAL ? 0 : kK, kV = C * 64 / N, kBuffer = kK + kQ + kV + Ahead<B16>::kUnits;
  static constexpr int kP = 2 * kBuffer, kS = kP + (LOCAL ? 0 : Ahead<B16>::kPairs * Ahead<B16>::kFrag);
  static constexpr int kState = LOCAL ? 0 : DKP / 16 * 64;  // of a wave
  static constexpr int kU = kS + 4 * kState, kUnits = kU + (LOCAL ? 0 : 4 * 128);
  static constexpr size_t kBytes = 16 * (size_t)kUnits;
  static_assert(kBytes <= 160 * 1024, "a compute unit's LDS");
};

// The state's row of register r of tile b: as rows of k are read, 16 bytes a
// lane, so that the state's tiles are operands without a move.
template <bool B16>
__device__ __forceinline__ int state_row(int b, int quad, int r) {
  return B16 ? 32 * (b >> 1) + 8 * quad + 4 * (b & 1) + r : 16 * b + 4 * quad + r;
}
// Rows row0 + 4 quad .. + 3 and 16 more at a lane's column: 16 lanes read a 4 x
// 16 block, 4 columns each, and are handed its columns.  The lanes' columns are
// c0 + STEP (lane % 4) .. + 3.  The waves that compute bring nothing into LDS,
// so these loads wait for none.
typedef short i16x4_t __attribute__((ext_vector_type(4)));
template <int W, int STEP>
__device__ __forceinline__ u32x4_t turned(const u32x4_t* s, int row0, int c0, int lane) {
  const int row = row0 + 4 * (lane >> 4) + ((lane >> 2) & 3), c = c0 + STEP * (lane & 3);
  const u32x2_t* at = reinterpret_cast<const u32x2_t*>(s + row * (W / 8) + row_unit<W>(row, c >> 3)) + ((c >> 2) & 1);
  auto read = [](const u32x2_t* p) {
    return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                           (__attribute__((address_space(3))) i16x4_t*)(const_cast<u32x2_t*>(p))));
  };
  const u32x2_t x = read(at), y = read(at + 16 * (W / 4));
  return u32x4_t{x[0], x[1], y[0], y[1]};
}

// Two of an accumulator's tiles as an operand, in three bf16 parts.
__device__ __forceinline__ void parts_of(const f32x4_t& x, const f32x4_t& y, u32x4_t (&w)[3]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const f32x4_t& v = e < 2 ? x : y;
    uint32_t p0, p1, p2;
    split3(v[2 * (e & 1)], v[2 * (e & 1) + 1], p0, p1, p2);
    w[0][e] = p0;
    w[1][e] = p1;
    w[2][e] = p2;
  }
}

// In U's place (a NaN, which U never holds there): the walking wave runs the
// chunk token by token and stores its outputs.
constexpr uint32_t kOneByOne = ~0u;

// What a workgroup walks: a sequence's or segment's first chunk, its first
// token and its tokens.
template <int C>
struct Walk {
  int seq, chunk0;
  Span span;
};
template <int C, int MODE>
__device__ __forceinline__ Walk<C> walk_of(const DeltaArgs& a, int item) {
  Walk<C> w;
  int seg = 0;
  if (MODE == DR_WHOLE) {
    w.seq = item;
  } else if (a.uniform_len >= 0) {
    w.seq = item / a.uniform_segs;
    seg = item - w.seq * a.uniform_segs;
  } else {
    int lo = 0, hi = a.n_seqs - 1;  // the last sequence that begins at or before the item
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first_item(a, mid) <= item) lo = mid; else hi = mid - 1;
    }
    w.seq = lo;
    seg = item - first_item(a, lo);
  }
  w.span = span_of(a, w.seq);
  w.chunk0 = a.uniform_len >= 0 ? w.seq * ((a.uniform_len + C - 1) / C) : first_chunk(a, w.seq);
  if (MODE != DR_WHOLE) {
    w.chunk0 += seg * a.seg_chunks;
    w.span.tok += (size_t)seg * a.seg_chunks * C;
    w.span.len = min(w.span.len - seg * a.seg_chunks * C, a.seg_chunks * C);
  }
  return w;
}

// The walk of a sequence, a head and 64 value columns through its chunks. Four
// waves, 16 columns each, go from S to the next S; four bring the next chunk,
// four turn the S and U that they are handed into outputs, and these eight
// work out P, so that nothing but the states' own chain runs from chunk to
// chunk (where the same waves did all, issuing the loads alone took 2.3 of a
// chunk's 5.7 us, heads of 128).  A chunk takes 3.5 us at heads of 64, 5.5 at 128:
// the chain's matrix products 0.9 and 1.2 us, the rest its LDS reads, splits and
// two meetings; matrix cores and VALU are 0.3 busy each.  Of these 0.5 and 1 us
// are what outputs from S, U and P in all three parts cost (two parts, 2^-17 of
// each value off, put one bf16 output in some 900 on the wrong side of a border).
// Both outputs' helpers at once, Q S ahead of the second meeting and S handed
// over in parts came to the same times within 3%.
// A segment's own state and its transition need no outputs, and two waves bring
// their chunks, so that two workgroups fit a compute unit.  The transition is
// the state that the unit matrix becomes without values: more columns.
// (Where a segment's own bf16 walk takes over 168 registers, only one of the two fits.)
constexpr int kWalkers = 4;
template <int MODE>
constexpr int kHelpers = MODE == DR_LOCAL ? 2 : 8;
template <bool B16, int DKP, int MODE>
__global__ __launch_bounds__(64 * (kWalkers + kHelpers<MODE>), MODE != DR_LOCAL ? 1 : B16 || DKP < 128 ? 3 : 2) void delta_walk_kernel(DeltaArgs a) {
  constexpr bool LOCAL = MODE == DR_LOCAL;
  using In = Ahead<B16>;
  using Lds = WalkLds<B16, DKP, LOCAL>;
  using T = std::conditional_t<B16, Bf16, float>;
  constexpr int C = In::C, NT = In::kTiles, NB = DKP / 16, N = Lds::N;
  constexpr int BRING = LOCAL ? 2 : 4, LOADS = Lds::kBuffer / 64, PER = (LOADS + BRING - 1) / BRING;
  extern __shared__ __attribute__((aligned(256))) u32x4_t s_walk[];
  const int lane = threadIdx.x & 63, in_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = in_all % kWalkers;
  const int col = lane & 15, quad = lane >> 4;
  // The columns: of the values, or (behind them) of the transition.
  const int tiles_v = (a.dv + 63) / 64, tiles = tiles_v + (LOCAL ? (a.dk + 63) / 64 : 0);
  // Workgroups of one item that read the same keys follow one another on one
  // of the eight XCDs, so that its L2 has them once.
  const int shared = a.share * tiles, slot = blockIdx.x / 8, group = slot / shared * 8 + blockIdx.x % 8;
  const int key_groups = a.heads_here / a.share, item = group / key_groups;
  if (item >= (MODE == DR_WHOLE ? a.n_seqs : a.items)) return;
  const int tile = slot % shared % tiles, head_here = group % key_groups * a.share + slot % shared / tiles;
  const int head = a.head0 + head_here, key_head = head / (a.heads / a.key_heads);
  const Walk<C> wk = walk_of<C, MODE>(a, item);
  const Span sp = wk.span;
  const bool moves = LOCAL && tile >= tiles_v;
  const int dv0 = 64 * (tile - (moves ? tiles_v : 0));
  const size_t item_head = (size_t)item * a.heads_here + head_here;
  // The state's element at the lane's first row and its column; the others are whole rows further.
  const size_t state0 = (((size_t)wk.seq * a.heads + head) * a.dk + state_row<B16>(0, quad, 0)) * a.dv + dv0 + 16 * wave + col;
  // A segment's state lies as the waves hold it: [16 columns][tile][lane].
  f32x4_t* seg_state = reinterpret_cast<f32x4_t*>(a.seg_state) + (item_head * ((a.dv + 15) / 16) + dv0 / 16 + wave) * NB * 64 + lane;
  const int j = dv0 + 16 * wave + col;  // the lane's column

  auto issue = [&](int pos, int n, u32x4_t* buffer) {
    const size_t tok = sp.tok + pos;
    const u32x4_t* ahead = reinterpret_cast<const u32x4_t*>(a.ahead) +
                           ((size_t)(wk.chunk0 + pos / C) * a.heads_here + head_here) * In::kUnits;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int load = i * BRING + in_all - kWalkers;
      if (LOADS % BRING != 0 && load >= LOADS) continue;
      const int at = load * 64;  // first unit
      const bool is_k = at < Lds::kK, is_q = !is_k && at < Lds::kK + Lds::kQ, is_v = !is_k && !is_q && at < Lds::kK + Lds::kQ + Lds::kV;
      const void* src;
      if (is_k || is_q || is_v) {
        const int unit = at - (is_k ? 0 : is_q ? Lds::kK : Lds::kK + Lds::kQ) + lane;
        const int units = is_v ? 64 / N : DKP / N, row = unit / units, u = unit % units;
        int c;
        if constexpr (B16)
          c = N * (is_v ? row_unit<64>(row, u) : row_unit<DKP>(row, u));
        else
          c = N * row_unit32(row, u);
        const size_t ld = is_k ? a.ld_k : is_q ? a.ld_q : a.ld_v;
        const T* base = is_k   ? static_cast<const T*>(a.k) + (size_t)key_head * a.wide_k
                        : is_q ? static_cast<const T*>(a.q) + (size_t)key_head * a.wide_q
                               : static_cast<const T*>(a.v) + (size_t)head * a.wide_v + dv0;
        const int there = is_v ? (moves ? 0 : a.dv - dv0) : a.dk;
        src = row < n && c < there ? static_cast<const void*>(base + (tok + row) * ld + c) : g_nothing;
      } else {
        src = ahead + (at - Lds::kK - Lds::kQ - Lds::kV) + lane;
      }
      auto* dst = (__attribute__((address_space(3))) void*)(buffer + at);
      __builtin_amdgcn_global_load_lds(src, dst, 16, 0, 0);
    }
  };
  auto meet = [&]() {  // without __syncthreads' wait for outputs on their way
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(kLdsOnly);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  if constexpr (LOCAL) {
    if (in_all >= kWalkers) {
      u32x4_t* to = s_walk;
      if (sp.len > 0) issue(0, min(C, sp.len), to);
      for (int pos = 0; pos < sp.len; pos += C) {
        __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
        meet();  // the chunk is there, and the one before is read
        to = to == s_walk ? s_walk + Lds::kBuffer : s_walk;
        if (pos + C < sp.len) issue(pos + C, min(C, sp.len - pos - C), to);
      }
      return;
    }
  }
  u32x4_t *sP = s_walk + Lds::kP, *sS = s_walk + Lds::kS + wave * Lds::kState, *sU = s_walk + Lds::kU + wave * 128;
  // U's first half in v's place: the wave's own columns, 2 units of each row.
  auto u_place = [&](const u32x4_t* v, int h) {
    const int i = 64 * h + lane, row = i >> 1;
    return const_cast<u32x4_t*>(v) + row * 8 + row_unit<64>(row, 2 * wave + (i & 1));
  };
  if (!LOCAL && in_all >= kWalkers) {
    if constexpr (B16) {  // the halves of fragments that P does not reach
      if (wave < 2) {
#pragma unroll
        for (int part = 0; part < 3; ++part)
          reinterpret_cast<u32x2_t*>(sP + In::kFrag * pair_of<B16>(2 * wave, wave) + 64 * part + lane)[1] = u32x2_t{0, 0};
      }
    }
    const int helper = in_all - kWalkers;
    const bool brings = helper < 4;
    const u32x4_t* buffer = s_walk;
    if (brings && sp.len > 0) issue(0, min(C, sp.len), s_walk);
    for (int pos = 0; pos < sp.len; pos += C) {
      const int n = min(C, sp.len - pos);
      if (brings) __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
      meet();  // the chunk is there, and the one before is read
      const u32x4_t *sK = buffer, *sQ = sK + Lds::kK, *sV = sQ + Lds::kQ, *sT = sV + Lds::kV;
      const float* gamma = reinterpret_cast<const float*>(sT + In::kGamma);
      const double* sum = reinterpret_cast<const double*>(sT + In::kSum);
      u32x4_t* other = buffer == s_walk ? s_walk + Lds::kBuffer : s_walk;
      buffer = other;
      if (brings && pos + C < sp.len) issue(pos + C, min(C, sp.len - pos - C), other);
      // P^T: queries 16 r + col, keys 16 c + 4 quad + e.
#pragma unroll
      for (int i = 0; i < (NT * (NT + 1) / 2 + 7) / 8; ++i) {
        // The waves that bring nothing take the second round.
        const int at = i ? 8 + helper - 4 : helper, r = triangle_row(at), c = triangle_col(at);
        if (at < 8 * i || at >= NT * (NT + 1) / 2) continue;  // uniform
        f32x4_t p = tile_product<B16, DKP>(sK, 16 * c, sQ, 16 * r, lane);
        const Power gq = power_in(sum[16 * r + col]);
        float d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = 16 * c + 4 * quad + e;
          d[e] = a.scale * decay_between(gq, power_in(sum[key]), 16 * r + col >= key);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = 16 * r + col >= 16 * c + 4 * quad + e ? p[e] * d[e] : 0.0f;
        if constexpr (B16) {
          u32x2_t w[3];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t p0, p1, p2;
            split3(p[2 * e], p[2 * e + 1], p0, p1, p2);
            w[0][e] = p0;
            w[1][e] = p1;
            w[2][e] = p2;
          }
          u32x4_t* to_p = sP + In::kFrag * pair_of<B16>(r, c >> 1) + lane;
#pragma unroll
          for (int part = 0; part < 3; ++part) reinterpret_cast<u32x2_t*>(to_p + 64 * part)[c & 1] = w[part];
        } else {
          sP[In::kFrag * pair_of<B16>(r, c) + lane] = __builtin_bit_cast(u32x4_t, p);
        }
      }
      meet();  // P, S and U are there
      if (brings || (uint32_t)__builtin_amdgcn_readfirstlane(sU[0][0]) == kOneByOne) continue;
      // O^T = scale e^G (Q S)^T + (P U)^T.
      f32x4_t o[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) o[t] = f32x4_t{0, 0, 0, 0};
      if constexpr (B16) {
#pragma unroll
        for (int kp = 0; kp < DKP / 32; ++kp) {
          u32x4_t w[3];
          parts_of(__builtin_bit_cast(f32x4_t, sS[128 * kp + lane]), __builtin_bit_cast(f32x4_t, sS[128 * kp + 64 + lane]), w);
          u32x4_t qf[NT];
#pragma unroll
          for (int t = 0; t < NT; ++t) qf[t] = row_frag<DKP>(sQ, 16 * t + col, 4 * kp + quad);
#pragma unroll
          for (int p = 2; p >= 0; --p)
#pragma unroll
            for (int t = 0; t < NT; ++t) o[t] = mfma(w[p], qf[t], o[t]);
        }
      } else {
        const f32x4_t* Q32 = reinterpret_cast<const f32x4_t*>(sQ);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const f32x4_t sf = __builtin_bit_cast(f32x4_t, sS[64 * b + lane]);
          f32x4_t qf[NT];
#pragma unroll
          for (int t = 0; t < NT; ++t) qf[t] = row_frag32<DKP>(Q32, 16 * t + col, 4 * b + quad);
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int t = 0; t < NT; ++t) o[t] = mfma32(sf[r], qf[t][r], o[t]);
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) o[t] *= a.scale * gamma[16 * t + col];
      if constexpr (B16) {
        // Parts' products down to 2^-16 of the whole; the others hold some 2^-24 of it.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          u32x4_t w[3];
          if (h == 0)
            parts_of(__builtin_bit_cast(f32x4_t, *u_place(sV, 0)), __builtin_bit_cast(f32x4_t, *u_place(sV, 1)), w);
          else
            parts_of(__builtin_bit_cast(f32x4_t, sU[lane]), __builtin_bit_cast(f32x4_t, sU[64 + lane]), w);
#pragma unroll
          for (int part = 2; part >= 0; --part)
#pragma unroll
            for (int t = 2 * h; t < NT; ++t) {
              const u32x4_t pf = sP[In::kFrag * pair_of<B16>(t, h) + 64 * part + lane];
#pragma unroll
              for (int p = 2 - part; p >= 0; --p) o[t] = mfma(w[p], pf, o[t]);
            }
        }
      } else {
        f32x4_t u[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) u[t] = __builtin_bit_cast(f32x4_t, sU[64 * t + lane]);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int h = 0; h <= t; ++h) {
            const f32x4_t pf = __builtin_bit_cast(f32x4_t, sP[64 * pair_of<B16>(t, h) + lane]);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[t] = mfma32(u[h][r], pf[r], o[t]);
          }
      }
      // Tokens 16 t + col, columns 16 wave + 4 quad ..
      const int c = dv0 + 16 * wave + 4 * quad;
      T* dst = static_cast<T*>(a.out) + (sp.tok + pos) * a.ld_out + (size_t)head * a.dv + (__umul24(col, (uint32_t)a.ld_out) + c);
      auto store = [&](T* to, const f32x4_t& v) {
        if constexpr (B16)
          *reinterpret_cast<u32x2_any_t*>(to) = u32x2_t{bf16x2_bits(v[0], v[1]), bf16x2_bits(v[2], v[3])};
        else
          *reinterpret_cast<f32x4_any_t*>(to) = v;
      };
      if (n == C && dv0 + 64 <= a.dv) {
#pragma unroll
        for (int t = 0; t < NT; ++t) store(dst + (size_t)(16 * t) * a.ld_out, o[t]);
      } else {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (16 * t + col >= n || c >= a.dv) continue;
          T* to = dst + (size_t)(16 * t) * a.ld_out;
          if (c + 4 <= a.dv) {
            store(to, o[t]);
          } else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
              if (c + e < a.dv) store1(to + e, o[t][e]);
          }
        }
      }
    }
    return;
  }
  // Whether a token of the segment forgets the state before it (a NaN does not).
  float least = 0.0f;
  if (moves)
#pragma unroll 4
    for (int i = lane; i < sp.len; i += 64) least = fminf(least, a.log_decay[(sp.tok + i) * a.ld_gates + head]);
  const bool forgets = __any(expf(least) == 0.0f);
  // S: the rows of the lane's column.
  f32x4_t S[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    if constexpr (MODE == DR_SEGMENT) {
      S[b] = dv0 + 16 * wave < a.dv ? seg_state[64 * b] : f32x4_t{0, 0, 0, 0};
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = state_row<B16>(b, quad, r);
        if constexpr (LOCAL)
          S[b][r] = moves && i == j && i < a.dk ? 1.0f : 0.0f;
        else
          S[b][r] = a.state_in && i < a.dk && j < a.dv ? (a.state_in + state0)[(size_t)state_row<B16>(b, 0, r) * a.dv] : 0.0f;
      }
    }
  }
  const u32x4_t* buffer = s_walk;
  for (int pos = 0; pos < sp.len; pos += C) {
    const int n = min(C, sp.len - pos);
    meet();
    const u32x4_t *sK = buffer, *sQ = sK + Lds::kK, *sV = sQ + Lds::kQ, *sT = sV + Lds::kV;
    const float *gamma = reinterpret_cast<const float*>(sT + In::kGamma), *rest = gamma + C;
    const f32x4_t *K32 = reinterpret_cast<const f32x4_t*>(sK), *Q32 = reinterpret_cast<const f32x4_t*>(sQ),
                  *V32 = reinterpret_cast<const f32x4_t*>(sV);
    buffer = buffer == s_walk ? s_walk + Lds::kBuffer : s_walk;

    // K S (rows: tokens).
    f32x4_t x[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) x[t] = f32x4_t{0, 0, 0, 0};
    if constexpr (B16) {
#pragma unroll
      for (int kp = 0; kp < DKP / 32; ++kp) {
        u32x4_t w[3];
        parts_of(S[2 * kp], S[2 * kp + 1], w);
        if constexpr (!LOCAL) {
          sS[128 * kp + lane] = __builtin_bit_cast(u32x4_t, S[2 * kp]);
          sS[128 * kp + 64 + lane] = __builtin_bit_cast(u32x4_t, S[2 * kp + 1]);
        }
        u32x4_t kf[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) kf[t] = row_frag<DKP>(sK, 16 * t + col, 4 * kp + quad);
#pragma unroll
        for (int p = 2; p >= 0; --p)
#pragma unroll
          for (int t = 0; t < NT; ++t) x[t] = mfma(kf[t], w[p], x[t]);
      }
    } else {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        if constexpr (!LOCAL) sS[64 * b + lane] = __builtin_bit_cast(u32x4_t, S[b]);
        f32x4_t kf[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) kf[t] = row_frag32<DKP>(K32, 16 * t + col, 4 * b + quad);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int t = 0; t < NT; ++t) x[t] = mfma32(kf[t][r], S[b][r], x[t]);
      }
    }
    // X = V - e^G K S, U = T X.
    if constexpr (B16) {
      u32x4_t vf[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) vf[h] = turned<64, 4>(sV, 32 * h, 16 * wave, lane);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const f32x4_t g = *reinterpret_cast<const f32x4_t*>(gamma + 16 * t + 4 * quad);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t w = vf[t >> 1][2 * (t & 1) + (r >> 1)];
          x[t][r] = fmaf(-g[r], x[t][r], __uint_as_float(r & 1 ? w & 0xFFFF0000u : w << 16));
        }
      }
    } else {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const f32x4_t g = *reinterpret_cast<const f32x4_t*>(gamma + 16 * t + 4 * quad);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[t][r] = fmaf(-g[r], x[t][r], element32<64>(V32, 16 * t + 4 * quad + r, 16 * wave + col));
      }
    }
    f32x4_t u[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) u[t] = f32x4_t{0, 0, 0, 0};
#pragma unroll
    for (int h = 0; h < NT; ++h) {
      f32x4_t tf[NT];
#pragma unroll
      for (int t = h; t < NT; ++t) tf[t] = __builtin_bit_cast(f32x4_t, sT[64 * (t * (t + 1) / 2 + h) + lane]);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int t = h; t < NT; ++t) u[t] = mfma32(tf[t][r], x[h][r], u[t]);
    }
    float odd = 0.0f;  // NaN once a value is not finite
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) odd = fmaf(u[t][r], 0.0f, odd);
    const bool one_by_one = __any(odd != odd);
    if constexpr (!LOCAL) {
      if (lane == 0) *reinterpret_cast<uint32_t*>(sU) = 0u - (uint32_t)one_by_one;  // kOneByOne, or what U then overwrites
      if (!one_by_one) {
#pragma unroll
        for (int t = 0; t < 2; ++t) sU[64 * t + lane] = __builtin_bit_cast(u32x4_t, u[NT - 2 + t]);
        if constexpr (B16) {
#pragma unroll
          for (int t = 0; t < 2; ++t) *u_place(sV, t) = __builtin_bit_cast(u32x4_t, u[t]);
        }
      }
    }
    if constexpr (!LOCAL) meet();  // S and U are there
    if (one_by_one) {
      T* out = static_cast<T*>(a.out) + (sp.tok + pos) * a.ld_out + (size_t)head * a.dv;
      // Something is not finite; in the products 0 times it would reach
      // tokens before it.  The chunk's tokens run one by one.
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        const size_t at = (sp.tok + pos + i) * a.ld_gates + head;
        const float decay = expf(a.log_decay[at]), beta = a.beta[at];
        f32x4_t kv[NB], qv[NB];
        float v;
        if constexpr (B16) {
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const u32x2_t w = four_of<DKP>(sK, i, state_row<B16>(b, quad, 0)), y = four_of<DKP>(sQ, i, state_row<B16>(b, quad, 0));
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              kv[b][r] = __uint_as_float(r & 1 ? w[r >> 1] & 0xFFFF0000u : w[r >> 1] << 16);
              qv[b][r] = __uint_as_float(r & 1 ? y[r >> 1] & 0xFFFF0000u : y[r >> 1] << 16);
            }
          }
          const u32x2_t w = four_of<64>(sV, i, 16 * wave + (col & ~3));
          const uint32_t y = col & 2 ? w[1] : w[0];
          v = __uint_as_float(col & 1 ? y & 0xFFFF0000u : y << 16);
        } else {
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            kv[b] = row_frag32<DKP>(K32, i, 4 * b + quad);
            qv[b] = row_frag32<DKP>(Q32, i, 4 * b + quad);
          }
          v = element32<64>(V32, i, 16 * wave + col);
        }
        float ks = 0.0f, qs = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            S[b][r] = decay == 0.0f ? 0.0f : S[b][r] * decay;
            ks = fmaf(kv[b][r], S[b][r], ks);
          }
        ks += __shfl_xor(ks, 16, 64);
        ks += __shfl_xor(ks, 32, 64);
        const float w = beta * ((moves ? 0.0f : v) - ks);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            // Rows past d_key stay empty, whatever w is.
            S[b][r] = state_row<B16>(b, quad, r) < a.dk ? fmaf(kv[b][r], w, S[b][r]) : 0.0f;
            qs = fmaf(qv[b][r], S[b][r], qs);
          }
        qs += __shfl_xor(qs, 16, 64);
        qs += __shfl_xor(qs, 32, 64);
        if (!LOCAL && quad == 0 && j < a.dv) store1(out + (size_t)i * a.ld_out + j, qs * a.scale);
      }
      continue;
    }
    // S = e^(G_n) S + K^T (e^(G_n - G) U).
    const float last = gamma[C - 1];
#pragma unroll
    for (int b = 0; b < NB; ++b) S[b] *= last;
#pragma unroll
    for (int t = 0; t < NT; ++t) u[t] *= *reinterpret_cast<const f32x4_t*>(rest + 16 * t + 4 * quad);
    if constexpr (B16) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4_t w[3];
        parts_of(u[2 * h], u[2 * h + 1], w);
        constexpr int BG = NB < 4 ? NB : 4;
#pragma unroll
        for (int b0 = 0; b0 < NB; b0 += BG) {
          u32x4_t kf[BG];
#pragma unroll
          for (int b = 0; b < BG; ++b) kf[b] = turned<DKP, 8>(sK, 32 * h, state_row<B16>(b0 + b, 0, 0), lane);
#pragma unroll
          for (int p = 2; p >= 0; --p)
#pragma unroll
            for (int b = 0; b < BG; ++b) S[b0 + b] = mfma(kf[b], w[p], S[b0 + b]);
        }
      }
    } else {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int b = 0; b < NB; ++b)
            S[b] = mfma32(element32<DKP>(K32, 16 * t + 4 * quad + r, 16 * b + col), u[t][r], S[b]);
    }
  }
  if (LOCAL && moves) {  // whole rows and columns, zeros past d_key, as the scan's lanes read them: 16 bytes each
    const int k = B16 ? j / 32 * 2 + (j >> 2 & 1) : j / 16, at = B16 ? j >> 3 & 3 : j >> 2 & 3;  // j = state_row(k, at, j % 4)
    float* move = a.seg_move + item_head * DKP * DKP + (k * 64 + at * 16 + 4 * quad) * 4 + j % 4;
    // Zeros are +0 where a token forgets; where the transition has only become
    // too small for fp32, -0, and the scan multiplies by them.
    const float zero = forgets ? 0.0f : -0.0f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (j < DKP) move[(b * NB * 64 + r) * 4] = S[b][r] == 0.0f ? zero : S[b][r];
  } else if (LOCAL) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
      if (dv0 + 16 * wave < a.dv) seg_state[64 * b] = S[b];
  } else if (MODE == DR_WHOLE && a.state_out) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = state_row<B16>(b, quad, r);
        if (i < a.dk && j < a.dv) (a.state_out + state0)[(size_t)state_row<B16>(b, 0, r) * a.dv] = S[b][r];
      }
  }
}

// The scan over a sequence's segments: S goes to its transition times S plus
// its own state; every segment's own state becomes its entry state, and the
// last one's exit is the sequence's.  A workgroup takes 16 columns, a wave one
// of the state's tiles; products in fp32.  The matrices of the next segments
// are on their way meanwhile; a step of 128 x 128 still takes 1.7 us, in which
// a compute unit reads its 64 KiB (2.3 us while a load's lanes lay in 64 places).
template <int DKP>
constexpr int kScanWaves = DKP / 16;
template <bool B16, int DKP>
__global__ __launch_bounds__(64 * kScanWaves<DKP>) void delta_scan_kernel(DeltaArgs a) {
  constexpr int NB = DKP / 16, WAVES = kScanWaves<DKP>, MINE = NB / WAVES;
  __shared__ f32x4_t s_state[2][NB * 64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, quad = lane >> 4;
  const int j = blockIdx.x * 16 + col, head = a.head0 + blockIdx.y, seq = blockIdx.z;
  const int item0 = a.uniform_len >= 0 ? seq * a.uniform_segs : first_item(a, seq);
  const int item1 = a.uniform_len >= 0 ? item0 + a.uniform_segs : first_item(a, seq + 1);
  const size_t state0 = ((size_t)seq * a.heads + head) * a.dk * a.dv;
  const size_t own_step = (size_t)a.heads_here * gridDim.x * NB * 64, move_step = (size_t)a.heads_here * DKP * DKP;
  f32x4_t* own = reinterpret_cast<f32x4_t*>(a.seg_state) + ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * NB * 64 + lane;
  const float* move = a.seg_move + (size_t)blockIdx.y * DKP * DKP;
  struct Part {
    f32x4_t own[MINE], move[MINE][NB];
  };
  f32x4_t S[MINE];
#pragma unroll
  for (int m = 0; m < MINE; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = state_row<B16>(wave + WAVES * m, quad, r);
      S[m][r] = a.state_in && i < a.dk && j < a.dv ? a.state_in[state0 + (size_t)i * a.dv + j] : 0.0f;
    }
  auto load = [&](int item, Part& p) {
#pragma unroll
    for (int m = 0; m < MINE; ++m) {
      const int b = wave + WAVES * m;
      p.own[m] = own[item * own_step + 64 * b];
      // Operands: the lane's row of tile b, columns as a tile's rows lie.
      const f32x4_t* at = reinterpret_cast<const f32x4_t*>(move + item * move_step) + b * NB * 64 + lane;
#pragma unroll
      for (int k = 0; k < NB; ++k) p.move[m][k] = at[64 * k];
    }
  };
  auto step = [&](int item, const Part& p) {
    f32x4_t* s = s_state[(item - item0) & 1];
#pragma unroll
    for (int m = 0; m < MINE; ++m) s[64 * (wave + WAVES * m) + lane] = S[m];
    asm volatile("" ::: "memory");  // the next segment's loads stay in flight
    __builtin_amdgcn_s_waitcnt(kLdsOnly);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    f32x4_t next[MINE];
    uint32_t keeps = 0;  // a transition of +0 forgets whatever the state is, one of -0 passes on what is not finite
#pragma unroll
    for (int m = 0; m < MINE; ++m) {
      next[m] = f32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) keeps |= __float_as_uint(p.move[m][k][r]);
    }
    if (__any(keeps != 0)) {
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const f32x4_t w = s[64 * k + lane];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int m = 0; m < MINE; ++m) next[m] = mfma32(p.move[m][k][r], w[r], next[m]);
      }
    }
#pragma unroll
    for (int m = 0; m < MINE; ++m) {
      own[item * own_step + 64 * (wave + WAVES * m)] = S[m];
      S[m] = next[m] + p.own[m];
    }
  };
  constexpr int DEEP = DKP == 128 ? 3 : 4;
  Part p[DEEP];
#pragma unroll
  for (int d = 0; d < DEEP; ++d) load(min(item0 + d, item1 - 1), p[d]);
  int item = item0;
  for (; item + DEEP <= item1; item += DEEP) {
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      step(item + d, p[d]);
      load(min(item + d + DEEP, item1 - 1), p[d]);
    }
  }
#pragma unroll
  for (int d = 0; d < DEEP - 1; ++d)
    if (item + d < item1) step(item + d, p[d]);
  if (!a.state_out) return;
#pragma unroll
  for (int m = 0; m < MINE; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = state_row<B16>(wave + WAVES * m, quad, r);
      if (i < a.dk && j < a.dv) a.state_out[state0 + (size_t)i * a.dv + j] = S[m][r];
    }
}

// Rows at any element copied to rows of whole 16-byte units: heads of `width`
// columns to heads of `to`, zeros behind.
template <class T>
__global__ __launch_bounds__(256) void delta_rows_kernel(const T* src, size_t ld, int heads, int width, T* dst, int to, size_t tokens) {
  constexpr int N = 16 / (int)sizeof(T);
  const int units = to / N;
  const size_t at = (size_t)blockIdx.x * 256 + threadIdx.x, row = (size_t)heads * units;
  if (at >= tokens * row) return;
  const size_t tok = at / row;
  const int in = (int)(at - tok * row), head = in / units, c = in % units * N;
  T v[N];
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = c + e < width ? src[tok * ld + (size_t)head * width + c + e] : T{};
  u32x4_t w;
  __builtin_memcpy(&w, v, 16);
  *reinterpret_cast<u32x4_t*>(dst + at * N) = w;
}

template <class T>
Status launch_steps(hipStream_t stream, const DeltaArgs& a) {
  const dim3 grid((a.dv + 63) / 64, a.heads, a.n_seqs);
  if (a.dk <= 32)
    delta_steps_kernel<T, 2><<<grid, 256, 0, stream>>>(a);
  else if (a.dk <= 64)
    delta_steps_kernel<T, 4><<<grid, 256, 0, stream>>>(a);
  else
    delta_steps_kernel<T, 8><<<grid, 256, 0, stream>>>(a);
  PSSA_LAUNCH_CHECK("delta_steps_kernel");
  return Status::Ok();
}

// Calls f with the kernels for a call's type and key width.
template <bool B16, int DKP>
struct Chunked {
  static constexpr bool kBf16 = B16;
  static constexpr auto kAhead = &delta_ahead_kernel<B16, DKP>;
  static constexpr auto kScan = &delta_scan_kernel<B16, DKP>;
  static constexpr int kScanThreads = 64 * kScanWaves<DKP>;
  template <int MODE>
  static Status walk(hipStream_t stream, const DeltaArgs& a) {
    const size_t shared = (size_t)a.share * ((a.dv + 63) / 64 + (MODE == DR_LOCAL ? (a.dk + 63) / 64 : 0));
    const size_t groups = (size_t)(MODE == DR_WHOLE ? a.n_seqs : a.items) * (a.heads_here / a.share);
    const uint32_t grid = (uint32_t)((groups + 7) / 8 * 8 * shared);
    delta_walk_kernel<B16, DKP, MODE>
        <<<grid, 64 * (kWalkers + kHelpers<MODE>), WalkLds<B16, DKP, MODE == DR_LOCAL>::kBytes, stream>>>(a);
    PSSA_LAUNCH_CHECK("delta_walk_kernel");
    return Status::Ok();
  }
  template <int MODE>
  static Status attributes() {
    PSSA_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(&delta_walk_kernel<B16, DKP, MODE>),
                                     hipFuncAttributeMaxDynamicSharedMemorySize, (int)WalkLds<B16, DKP, MODE == DR_LOCAL>::kBytes));
    return Status::Ok();
  }
};
template <class F>
Status with_chunks(int dtype, int dk, F f) {
  auto wide = [&](auto b16) {
    constexpr bool B = decltype(b16)::value;
    if (dk <= 32) return f(Chunked<B, 32>{});
    if (dk <= 64) return f(Chunked<B, 64>{});
    return f(Chunked<B, 128>{});
  };
  return dtype == PSSA_HIP_BF16 ? wide(std::true_type{}) : wide(std::false_type{});
}

size_t unit_of(int dtype) { return dtype == PSSA_HIP_BF16 ? 8 : 4; }  // elements of 16 bytes
size_t whole(size_t width, size_t unit) { return (width + unit - 1) / unit * unit; }

template <class T>
Status launch_rows(hipStream_t stream, const void*& p, size_t& ld, int heads, int width, int& to, size_t tokens, char*& scratch) {
  to = (int)whole(width, 16 / sizeof(T));
  const size_t units = tokens * heads * (to * sizeof(T) / 16);
  delta_rows_kernel<T><<<(uint32_t)((units + 255) / 256), 256, 0, stream>>>(static_cast<const T*>(p), ld, heads, width,
                                                                          reinterpret_cast<T*>(scratch), to, tokens);
  PSSA_LAUNCH_CHECK("delta_rows_kernel");
  p = scratch;
  ld = (size_t)heads * to;
  scratch += delta_copy_bytes(sizeof(T) == 2 ? PSSA_HIP_BF16 : PSSA_HIP_F32, tokens, heads, width);
  return Status::Ok();
}

}  // namespace

int delta_chunk(int dtype) { return dtype == PSSA_HIP_BF16 ? Ahead<true>::C : Ahead<false>::C; }

bool delta_in_units(int dtype, const void* p, size_t ld, size_t width) {
  return (uintptr_t)p % 16 == 0 && ld % unit_of(dtype) == 0 && width % unit_of(dtype) == 0;
}
size_t delta_copy_bytes(int dtype, size_t tokens, size_t heads, size_t width) {
  const size_t unit = unit_of(dtype);
  return (tokens * heads * (whole(width, unit) / unit) * 16 + 255) & ~(size_t)255;
}

// What is worked out ahead takes 11 KiB a chunk and head (bf16; 4 KiB fp32):
// past 1 GiB of it the heads run in several launches, and where a launch would
// have 2^32 threads.
DeltaScratch delta_scratch(int dtype, size_t chunks, size_t n_seqs, size_t items, size_t heads, size_t d_key, size_t d_val) {
  DeltaScratch s;
  const size_t one = chunks * 16 * (dtype == PSSA_HIP_BF16 ? Ahead<true>::kUnits : Ahead<false>::kUnits);
  const size_t walks = std::max(n_seqs, items) * ((d_val + 63) / 64 + (items ? (d_key + 63) / 64 : 0));
  s.heads_here = (int)std::max<size_t>(1, std::min({heads, ((size_t)1 << 30) / std::max<size_t>(one, 1), 5000000 / walks}));
  s.ahead = (one * s.heads_here + 255) & ~(size_t)255;
  const size_t keys = d_key <= 32 ? 32 : d_key <= 64 ? 64 : 128;  // as the kernels hold them
  s.state = items * s.heads_here * keys * whole(d_val, 16) * 4;
  s.move = items * s.heads_here * keys * keys * 4;
  return s;
}

Status init_delta_attributes() {
  for (int dtype : {PSSA_HIP_F32, PSSA_HIP_BF16})
    for (int dk : {32, 64, 128})
      PSSA_RETURN_IF(with_chunks(dtype, dk, [&](auto c) -> Status {
        PSSA_RETURN_IF(c.template attributes<DR_WHOLE>());
        PSSA_RETURN_IF(c.template attributes<DR_LOCAL>());
        return c.template attributes<DR_SEGMENT>();
      }));
  return Status::Ok();
}

// A walk's chunk takes about 3.1 us (bf16 3.5), one of a segment's own state 2.3 us, a
// step of the scan over the segments 1.5 us, and the passes between some 12 us
// (at heads of 64 and the machine's 256 compute units, a workgroup each; wider
// heads take half as much again of all, which leaves the choice).  A call is
// split where that makes it the faster, into segments of whichever length
// costs least: nine of ten calls of 600 to 16 x 1024 tokens ran within 5% of the
// best of segments of 2, 4, 6, 8, 12, 16 and 32 chunks and of none, one within 9
// (8192 tokens, 8 heads of 128: 137 us, unsplit 569; 600 tokens, 2 heads of 64: 31
// us, unsplit 38).
constexpr size_t kComputeUnits = 256;
int delta_segment(int dtype, const uint64_t* lens, size_t n_seqs, size_t longest, size_t heads, size_t d_key, size_t d_val) {
  const size_t chunk = (size_t)delta_chunk(dtype), most = (longest + chunk - 1) / chunk;
  const size_t tiles = (d_val + 63) / 64, moves = (d_key + 63) / 64;
  auto rounds = [](size_t n) { return (double)((n + kComputeUnits - 1) / kComputeUnits); };
  auto items_of = [&](size_t seg) {
    size_t items = 0;
    for (size_t i = 0; i < (lens ? n_seqs : 1); ++i) items += std::max<size_t>(1, ((lens ? lens[i] : longest) + seg * chunk - 1) / (seg * chunk));
    return lens ? items : items * n_seqs;
  };
  double best = rounds(n_seqs * heads * tiles) * most * 3.1;
  int at = 0;
  for (size_t seg = 2; 2 * seg <= most; seg += std::max<size_t>(1, seg / 4)) {
    const size_t items = items_of(seg), steps = (most + seg - 1) / seg;
    if (items > 65535) continue;
    const double cost = rounds(items * heads * (tiles + moves)) * seg * 2.3 + steps * 1.5 + rounds(items * heads * tiles) * seg * 3.1 + 12;
    if (cost < best) {
      best = cost;
      at = (int)seg;
    }
  }
  return at;
}

Status launch_delta_rule(hipStream_t stream, int dtype, DeltaArgs a, size_t tokens, int longest, const DeltaScratch& s,
                         char* scratch) {
  if (longest <= kDeltaSteps)
    return dtype == PSSA_HIP_F32 ? launch_steps<float>(stream, a) : launch_steps<Bf16>(stream, a);
  a.ahead = scratch;
  a.seg_state = reinterpret_cast<float*>(scratch + s.ahead + s.rows);
  a.seg_move = reinterpret_cast<float*>(scratch + s.ahead + s.rows + s.state);
  char* rows = scratch + s.ahead;
  const bool b16 = dtype == PSSA_HIP_BF16;
  auto in_place = [&](const void*& p, size_t& ld, int heads, int width, int& to) -> Status {
    to = width;
    if (delta_in_units(dtype, p, ld, width)) return Status::Ok();
    return b16 ? launch_rows<Bf16>(stream, p, ld, heads, width, to, tokens, rows)
               : launch_rows<float>(stream, p, ld, heads, width, to, tokens, rows);
  };
  PSSA_RETURN_IF(in_place(a.q, a.ld_q, a.key_heads, a.dk, a.wide_q));
  PSSA_RETURN_IF(in_place(a.k, a.ld_k, a.key_heads, a.dk, a.wide_k));
  PSSA_RETURN_IF(in_place(a.v, a.ld_v, a.heads, a.dv, a.wide_v));
  return with_chunks(dtype, a.dk, [&](auto c) -> Status {
    for (a.head0 = 0; a.head0 < a.heads; a.head0 += s.heads_here) {
      a.heads_here = std::min(s.heads_here, a.heads - a.head0);
      const int rep = a.heads / a.key_heads;  // heads of the same keys
      a.share = a.head0 % rep == 0 && a.heads_here % rep == 0 ? rep : 1;
      c.kAhead<<<dim3(a.chunks, a.heads_here), c.kBf16 ? 256 : 128, 0, stream>>>(a);
      PSSA_LAUNCH_CHECK("delta_ahead_kernel");
      if (!a.seg_chunks) {
        PSSA_RETURN_IF(c.template walk<DR_WHOLE>(stream, a));
        continue;
      }
      PSSA_RETURN_IF(c.template walk<DR_LOCAL>(stream, a));
      c.kScan<<<dim3((a.dv + 15) / 16, a.heads_here, a.n_seqs), c.kScanThreads, 0, stream>>>(a);
      PSSA_LAUNCH_CHECK("delta_scan_kernel");
      PSSA_RETURN_IF(c.template walk<DR_SEGMENT>(stream, a));
    }
    return Status::Ok();
  });
}

}  // namespace pssa
