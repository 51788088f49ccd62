// Linear attention with a decay for each head: the recurrence
//   S_t = lambda_h S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t
// over packed sequences, from one token to long prompts.
//
// Prompts run in chunks of 64 tokens.  Within a chunk entered with state S
// (i, j count its tokens, n of them)
//   o_i = scale (lambda^(i+1) q_i S + sum_{j<=i} lambda^(i-j) (q_i k_j) v_j)
//   S'  = lambda^n S + sum_j k_j (lambda^(n-1-j) v_j)^T,
// four matrix products.  A workgroup of four waves walks one sequence's (or
// segment's) chunks for one head and a tile of value columns; a wave owns 16
// or 32 of the columns, its part of S stays in its accumulators, and these
// are the product q S's operand as they stand: the accumulator layout (lane l
// holds column l % 16, rows 4 (l / 16) + r) is the matrix instruction's
// operand layout once q's columns are read in the same order.
//
// Few long sequences are split into segments: the segments' own states (the
// second product alone, from zero), a scan over them that leaves every
// segment's entry state, then the chunks of all segments at once.
#include <algorithm>
#include <cstddef>
#include <type_traits>

#include "operators.h"

namespace pssa {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef f32x4_t f32x4_any_t __attribute__((aligned(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef u32x2_t u32x2_any_t __attribute__((aligned(2)));

struct Bf16 {
  uint16_t bits;
};

constexpr int LA_C = 64;  // tokens of a chunk
constexpr float kLog2e = 1.44269504088896341f;

// lambda^n from the log decay; lambda^0 is 1 for lambda = 0 too.
__device__ __forceinline__ float decay_pow(float g2, int n) { return n <= 0 ? 1.0f : __builtin_amdgcn_exp2f(g2 * (float)n); }
// The same to the last bit, for factors that a whole prompt's states pass through.
__device__ __forceinline__ float decay_pow_exact(float g, int n) { return n <= 0 ? 1.0f : (float)exp((double)g * n); }

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

// What a workgroup walks: a segment's first token and length, and where its
// state is (the sequence's, or its own one in the scratch of a split call).
struct Span {
  int seq, item;
  size_t tok;
  int len;
};
// The arguments' tables are read from the kernel's argument segment, where the
// arguments lie first: indexing the struct itself would copy it to scratch.
typedef const __attribute__((address_space(4))) char* kernarg_t;
__device__ __forceinline__ uint32_t inline_word(size_t offset, int i) {
  return reinterpret_cast<const __attribute__((address_space(4))) uint32_t*>(
      (kernarg_t)__builtin_amdgcn_kernarg_segment_ptr() + offset)[i];
}
__device__ __forceinline__ uint32_t first_token(const LinearArgs& a, int seq) {
  return a.table ? a.table[seq] : inline_word(offsetof(LinearArgs, inline_tokens), seq);
}
__device__ __forceinline__ int first_item(const LinearArgs& a, int seq) {
  return (int)(a.table ? a.table[a.n_seqs + 1 + seq] : inline_word(offsetof(LinearArgs, inline_items), seq));
}
__device__ __forceinline__ Span span_of(const LinearArgs& a, int item) {
  Span s;
  s.item = item;
  int seg, len;
  if (a.uniform_len >= 0) {
    s.seq = item / a.uniform_segs;
    seg = item - s.seq * a.uniform_segs;
    s.tok = (size_t)s.seq * a.uniform_len;
    len = a.uniform_len;
  } else {
    int lo = 0, hi = a.n_seqs - 1;  // the last sequence that begins at or before the item
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first_item(a, mid) <= item) lo = mid; else hi = mid - 1;
    }
    s.seq = lo;
    seg = item - first_item(a, lo);
    s.tok = first_token(a, lo);
    len = (int)(first_token(a, lo + 1) - s.tok);
  }
  s.tok += (size_t)seg * a.seg_len;
  s.len = min(len - seg * a.seg_len, a.seg_len);
  return s;
}

// How a chunk kernel runs: the whole of an unsplit call, a segment's own
// state, or a segment's outputs from its entry state.
enum { LA_WHOLE, LA_LOCAL, LA_SEGMENT };

// fp32 matrix products (v_mfma_f32_16x16x4_f32); bf16 inputs widened.
template <class T, int DKP, int NC, int MODE>
__global__ __launch_bounds__(256) void linear_chunks_f32_kernel(LinearArgs a) {
  constexpr int LDK = DKP + 4, LDV = 64 * NC + 4, LDP = 68, NB = DKP / 16;
  extern __shared__ float s_lin[];
  float* sQ = s_lin;
  float* sK = sQ + LA_C * LDK;
  float* sV = sK + LA_C * LDK;
  float* sP = sV + LA_C * LDV;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int dv0 = blockIdx.x * 64 * NC, head = blockIdx.y, kv_head = head / (a.heads / a.kv_heads);
  const Span sp = span_of(a, blockIdx.z);
  const float g = a.log_decay[head], g2 = g * kLog2e;
  const T* q0 = static_cast<const T*>(a.q) + (size_t)head * a.dk;
  const T* k0 = static_cast<const T*>(a.k) + (size_t)kv_head * a.dk;
  const T* v0 = static_cast<const T*>(a.v) + (size_t)kv_head * a.dv;
  T* o0 = static_cast<T*>(a.out) + (size_t)head * a.dv;
  const size_t state0 = ((size_t)(MODE == LA_WHOLE ? sp.seq : sp.item) * a.heads + head) * a.dk * a.dv;
  const float* state_in = MODE == LA_WHOLE ? a.state_in : MODE == LA_LOCAL ? nullptr : a.seg_state;
  float* state_out = MODE == LA_WHOLE ? a.state_out : MODE == LA_LOCAL ? a.seg_state : nullptr;

  // S: rows 16 b + 4 quad + r, column dv0 + 16 NC wave + 16 c + col.
  f32x4_t S[NB][NC];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * b + 4 * quad + r, j = dv0 + 16 * NC * wave + 16 * c + col;
        S[b][c][r] = state_in && i < a.dk && j < a.dv ? state_in[state0 + (size_t)i * a.dv + j] : 0.0f;
      }
  const float full = decay_pow_exact(g, LA_C);

  int singles = 0;  // tokens left of a chunk that runs one by one
  for (int pos = 0; pos < sp.len;) {
    int n = singles ? 1 : min(LA_C, sp.len - pos);
    bool odd = false;
    auto fill = [&]() {
      for (int i = tid; i < LA_C * DKP / 4; i += 256) {
        const int row = i / (DKP / 4), c = i % (DKP / 4) * 4, left = row < n ? a.dk - c : 0;
        const size_t t = sp.tok + pos + row;
        if (MODE != LA_LOCAL)
          *reinterpret_cast<f32x4_t*>(sQ + row * LDK + c) = left > 0 ? load4<T>(q0 + t * a.ld_q + c, left) : f32x4_t{0, 0, 0, 0};
        *reinterpret_cast<f32x4_t*>(sK + row * LDK + c) = left > 0 ? load4<T>(k0 + t * a.ld_k + c, left) : f32x4_t{0, 0, 0, 0};
      }
      for (int i = tid; i < LA_C * 16 * NC; i += 256) {
        const int row = i / (16 * NC), c = i % (16 * NC) * 4, left = row < n ? a.dv - dv0 - c : 0;
        const size_t t = sp.tok + pos + row;
        const f32x4_t v = left > 0 ? load4<T>(v0 + t * a.ld_v + dv0 + c, left) : f32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= !(fabsf(v[e]) < INFINITY);
        *reinterpret_cast<f32x4_t*>(sV + row * LDV + c) = v;
      }
    };
    __syncthreads();  // the chunk before is read
    fill();
    // A value that is not finite would reach the rows before it (0 times it is
    // NaN): such a chunk's tokens run one at a time.
    if (__syncthreads_or(odd) && MODE != LA_LOCAL && n > 1) {
      singles = n;
      n = 1;
      fill();
      __syncthreads();
    }

    if constexpr (MODE != LA_LOCAL) {
    // P = (q k^T) lambda^(i-j), j <= i: rows 16 wave .. of the chunk.
#pragma unroll
    for (int jt = 0; jt < 4; ++jt) {
      if (jt > wave) continue;
      f32x4_t p = {0, 0, 0, 0};
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const f32x4_t qf = *reinterpret_cast<const f32x4_t*>(sQ + (16 * wave + col) * LDK + 16 * b + 4 * quad);
        const f32x4_t kf = *reinterpret_cast<const f32x4_t*>(sK + (16 * jt + col) * LDK + 16 * b + 4 * quad);
#pragma unroll
        for (int r = 0; r < 4; ++r) p = __builtin_amdgcn_mfma_f32_16x16x4f32(qf[r], kf[r], p, 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * wave + 4 * quad + r, j = 16 * jt + col;
        sP[i * LDP + j] = j <= i ? p[r] * decay_pow(g2, i - j) : 0.0f;
      }
    }
    // q S, each row times lambda^(i+1).
    f32x4_t o[4][NC];
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) {
#pragma unroll
      for (int c = 0; c < NC; ++c) o[rt][c] = f32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const f32x4_t qf = *reinterpret_cast<const f32x4_t*>(sQ + (16 * rt + col) * LDK + 16 * b + 4 * quad);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < NC; ++c) o[rt][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(qf[r], S[b][c][r], o[rt][c], 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float f = decay_pow(g2, 16 * rt + 4 * quad + r + 1);
#pragma unroll
        for (int c = 0; c < NC; ++c) o[rt][c][r] *= f;
      }
    }
    __syncthreads();
    // + P v.
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      float vf[4][NC];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < NC; ++c) vf[r][c] = sV[(16 * kt + 4 * quad + r) * LDV + 16 * NC * wave + 16 * c + col];
#pragma unroll
      for (int rt = kt; rt < 4; ++rt) {
        const f32x4_t pf = *reinterpret_cast<const f32x4_t*>(sP + (16 * rt + col) * LDP + 16 * kt + 4 * quad);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < NC; ++c) o[rt][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(pf[r], vf[r][c], o[rt][c], 0, 0, 0);
      }
    }
#pragma unroll
    for (int rt = 0; rt < 4; ++rt)
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 16 * rt + 4 * quad + r, j = dv0 + 16 * NC * wave + 16 * c + col;
          if (i < n && j < a.dv) store1(o0 + (sp.tok + pos + i) * a.ld_out + j, o[rt][c][r] * a.scale);
        }
    }
    // S = lambda^n S + k^T (lambda^(n-1-j) v).
    const float fs = n == LA_C ? full : decay_pow_exact(g, n);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int c = 0; c < NC; ++c) S[b][c] *= fs;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 16 * kt + 4 * quad + r;
        const float w = decay_pow(g2, n - 1 - j);
        float vf[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) vf[c] = w * sV[j * LDV + 16 * NC * wave + 16 * c + col];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const float kf = sK[j * LDK + 16 * b + col];
#pragma unroll
          for (int c = 0; c < NC; ++c) S[b][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf, vf[c], S[b][c], 0, 0, 0);
        }
      }
    }
    pos += n;
    if (singles) --singles;
  }
  if (!state_out) return;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * b + 4 * quad + r, j = dv0 + 16 * NC * wave + 16 * c + col;
        if (i < a.dk && j < a.dv) state_out[state0 + (size_t)i * a.dv + j] = S[b][c][r];
      }
}

// ---------------------------------------------------------------- bf16 inputs
// The same on v_mfma_f32_16x16x32_bf16.  q k^T takes the inputs as they are;
// P and S enter as two bf16 parts (2^-17 relative, below the outputs' own
// rounding), the decayed values of the state's update as three (exact), since
// the state is an fp32 result.
//
// A 32-deep operand's lane holds eight places: 4 quad + r of one 16-row tile
// and of the next, the order in which two accumulators lie in the lane's
// registers.  Everything that meets an accumulator is kept in that order
// (columns of q and k, tokens of the transposed k and v), so S and P are
// operands without a move; P passes through LDS as ready fragments because
// one wave computes 16 rows of it and every wave needs all.
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef u32x4_t u32x4_any_t __attribute__((aligned(2)));

// 8 neighbouring elements, zeros past `left`.
__device__ __forceinline__ u32x4_t load8(const uint16_t* p, int left) {
  if (left >= 8) return *reinterpret_cast<const u32x4_any_t*>(p);
  u32x4_t v = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (i < left) v[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
  return v;
}
// Lower or upper halves of two words side by side.
__device__ __forceinline__ uint32_t lower2(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
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

// LDS in 16-byte units; a row has one more than it needs, so that 16 rows
// read at one unit lie in 16 different places.
template <int W>
__device__ __forceinline__ int row_at(int row, int u) { return row * (W / 8 + 1) + u; }
// Rows of 64 tokens.
__device__ __forceinline__ int tok_at(int row, int u) { return row * 9 + u; }
// The unit and half of columns (or tokens) c .. c + 3 in operand order.
__device__ __forceinline__ int order_unit(int c) { return (c >> 5) * 4 + ((c >> 2) & 3); }
__device__ __forceinline__ int order_half(int c) { return (c >> 4) & 1; }

// Place of query tile t's keys 32 h ..: none behind the queries.
constexpr int pair_at(int t, int h) { return t < 2 ? t : 2 * t - 2 + h; }

template <int DKP, int NC, int MODE>
__global__ __launch_bounds__(256, NC == 2 || DKP == 128 ? 1 : 2) void linear_chunks_bf16_kernel(LinearArgs a) {
  constexpr int DVT = 64 * NC, NB = DKP / 16, KP = DKP / 32;
  constexpr int QV = LA_C * DKP / 8 / 256;              // 16-byte pieces of q for a thread (DKP = 32: one)
  constexpr int TASKS = 16 * (DKP / 8 + DVT / 8);       // 4 tokens x 8 columns of k, then of v
  constexpr int TV = (TASKS + 255) / 256;
  extern __shared__ u32x4_t s_bf[];
  u32x4_t* sQ = s_bf;                       // [64][DKP], operand order
  u32x4_t* sK = sQ + (MODE == LA_LOCAL ? 0 : LA_C * (DKP / 8 + 1));
  u32x4_t* sKT = sK + (MODE == LA_LOCAL ? 0 : LA_C * (DKP / 8 + 1));  // [DKP][64 tokens]
  u32x4_t* sVT = sKT + DKP * 9;  // [DVT][64 tokens]
  u32x4_t* sP = sVT + DVT * 9;   // [6 pairs of a query tile and a key half][2 parts][64 lanes]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int dv0 = blockIdx.x * DVT, head = blockIdx.y, kv_head = head / (a.heads / a.kv_heads);
  const Span sp = span_of(a, blockIdx.z);
  const float g = a.log_decay[head], g2 = g * kLog2e;
  const uint16_t* q0 = static_cast<const uint16_t*>(a.q) + (size_t)head * a.dk;
  const uint16_t* k0 = static_cast<const uint16_t*>(a.k) + (size_t)kv_head * a.dk;
  const uint16_t* v0 = static_cast<const uint16_t*>(a.v) + (size_t)kv_head * a.dv + dv0;
  uint16_t* o0 = static_cast<uint16_t*>(a.out) + (size_t)head * a.dv;
  const size_t state0 = ((size_t)(MODE == LA_WHOLE ? sp.seq : sp.item) * a.heads + head) * a.dk * a.dv;
  const float* state_in = MODE == LA_WHOLE ? a.state_in : MODE == LA_LOCAL ? nullptr : a.seg_state;
  float* state_out = MODE == LA_WHOLE ? a.state_out : MODE == LA_LOCAL ? a.seg_state : nullptr;

  // S: rows 16 b + 4 quad + r, column dv0 + 16 NC wave + 16 c + col.
  f32x4_t S[NB][NC];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * b + 4 * quad + r, j = dv0 + 16 * NC * wave + 16 * c + col;
        S[b][c][r] = state_in && i < a.dk && j < a.dv ? state_in[state0 + (size_t)i * a.dv + j] : 0.0f;
      }
  const float full = decay_pow_exact(g, LA_C);
  float first[4];  // lambda^(i+1) of the lane's query in each tile
#pragma unroll
  for (int t = 0; t < 4; ++t) first[t] = decay_pow(g2, 16 * t + col + 1);

  u32x4_t rq[QV > 0 ? QV : 1], rt[TV][4];
  auto fetch = [&](int pos, int n) {
    if constexpr (MODE != LA_LOCAL) {
#pragma unroll
      for (int i = 0; i < QV; ++i) {
        const int at = tid + 256 * i, row = at / (DKP / 8), c = at % (DKP / 8) * 8;
        rq[i] = row < n && c < a.dk ? load8(q0 + (sp.tok + pos + row) * a.ld_q + c, a.dk - c) : u32x4_t{0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int i = 0; i < TV; ++i) {
      const int task = tid + 256 * i;
      const bool is_k = task < 16 * (DKP / 8);
      const int row = (task & 15) * 4, c = (is_k ? task >> 4 : (task >> 4) - DKP / 8) * 8;
      const int left = task < TASKS ? (is_k ? a.dk : a.dv - dv0) - c : 0;
      const uint16_t* src = is_k ? k0 : v0;
      const size_t ld = is_k ? a.ld_k : a.ld_v;
#pragma unroll
      for (int t = 0; t < 4; ++t)
        rt[i][t] = row + t < n && left > 0 ? load8(src + (sp.tok + pos + row + t) * ld + c, left) : u32x4_t{0, 0, 0, 0};
    }
  };
  // The fetched chunk into LDS; whether a value of v is not finite.
  auto place = [&]() {
    u32x2_t* q8 = reinterpret_cast<u32x2_t*>(sQ);
    u32x2_t* k8 = reinterpret_cast<u32x2_t*>(sK);
    bool odd = false;
    if constexpr (MODE != LA_LOCAL) {
#pragma unroll
      for (int i = 0; i < QV; ++i) {
        const int at = tid + 256 * i, row = at / (DKP / 8), c = at % (DKP / 8) * 8;
        q8[2 * row_at<DKP>(row, order_unit(c)) + order_half(c)] = u32x2_t{rq[i][0], rq[i][1]};
        q8[2 * row_at<DKP>(row, order_unit(c + 4)) + order_half(c)] = u32x2_t{rq[i][2], rq[i][3]};
      }
    }
#pragma unroll
    for (int i = 0; i < TV; ++i) {
      const int task = tid + 256 * i;
      if (task >= TASKS) continue;
      const bool is_k = task < 16 * (DKP / 8);
      const int row = (task & 15) * 4, c = (is_k ? task >> 4 : (task >> 4) - DKP / 8) * 8;
      if constexpr (MODE != LA_LOCAL) {
        if (is_k) {
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            k8[2 * row_at<DKP>(row + t, order_unit(c)) + order_half(c)] = u32x2_t{rt[i][t][0], rt[i][t][1]};
            k8[2 * row_at<DKP>(row + t, order_unit(c + 4)) + order_half(c)] = u32x2_t{rt[i][t][2], rt[i][t][3]};
          }
        } else {
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              odd |= (rt[i][t][e] & 0x7F80u) == 0x7F80u || (rt[i][t][e] & 0x7F800000u) == 0x7F800000u;
        }
      }
      u32x2_t* t8 = reinterpret_cast<u32x2_t*>(is_k ? sKT : sVT);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        t8[2 * tok_at(c + 2 * e, order_unit(row)) + order_half(row)] =
            u32x2_t{lower2(rt[i][0][e], rt[i][1][e]), lower2(rt[i][2][e], rt[i][3][e])};
        t8[2 * tok_at(c + 2 * e + 1, order_unit(row)) + order_half(row)] =
            u32x2_t{upper2(rt[i][0][e], rt[i][1][e]), upper2(rt[i][2][e], rt[i][3][e])};
      }
    }
    return odd;
  };

  int singles = 0;  // tokens left of a chunk that runs one by one
  if (sp.len > 0) fetch(0, min(LA_C, sp.len));
  for (int pos = 0; pos < sp.len;) {
    int n = singles ? 1 : min(LA_C, sp.len - pos);
    __syncthreads();  // the chunk before is read
    const bool odd = place();
    // A value that is not finite would reach the rows before it (0 times it is
    // NaN): such a chunk's tokens run one at a time.
    if (MODE != LA_LOCAL) {
      if (__syncthreads_or(odd) && n > 1) {
        singles = n;
        n = 1;
        fetch(pos, 1);
        place();
        __syncthreads();
      }
    } else {
      __syncthreads();
    }
    const int next = pos + n;
    if (next < sp.len) fetch(next, singles > 1 ? 1 : min(LA_C, sp.len - next));

    f32x4_t o[4][NC];
    if constexpr (MODE != LA_LOCAL) {
      // P^T = (k q^T) lambda^(i-j), j <= i, of query tile `wave`.
      f32x4_t p[4];
#pragma unroll
      for (int jt = 0; jt < 4; ++jt) {
        p[jt] = f32x4_t{0, 0, 0, 0};
        if (jt > wave) continue;  // uniform
#pragma unroll
        for (int kp = 0; kp < KP; ++kp)
          p[jt] = mfma(sK[row_at<DKP>(16 * jt + col, 4 * kp + quad)], sQ[row_at<DKP>(16 * wave + col, 4 * kp + quad)], p[jt]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 16 * wave + col, j = 16 * jt + 4 * quad + r;
          p[jt][r] = j <= i ? p[jt][r] * decay_pow(g2, i - j) : 0.0f;
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (2 * h > wave) continue;
        u32x4_t hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t x, y;
          split2(p[2 * h + (e >> 1)][2 * (e & 1)], p[2 * h + (e >> 1)][2 * (e & 1) + 1], x, y);
          hi[e] = x;
          lo[e] = y;
        }
        sP[(pair_at(wave, h) * 2 + 0) * 64 + lane] = hi;
        sP[(pair_at(wave, h) * 2 + 1) * 64 + lane] = lo;
      }
      // (q S)^T, each query's column times lambda^(i+1).
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int c = 0; c < NC; ++c) o[t][c] = f32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int kp = 0; kp < KP; ++kp) {
        u32x4_t hi[NC], lo[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t x, y;
            split2(S[2 * kp + (e >> 1)][c][2 * (e & 1)], S[2 * kp + (e >> 1)][c][2 * (e & 1) + 1], x, y);
            hi[c][e] = x;
            lo[c][e] = y;
          }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const u32x4_t qf = sQ[row_at<DKP>(16 * t + col, 4 * kp + quad)];
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            o[t][c] = mfma(lo[c], qf, o[t][c]);
            o[t][c] = mfma(hi[c], qf, o[t][c]);
          }
        }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int c = 0; c < NC; ++c) o[t][c] *= first[t];
      __syncthreads();  // P is there
    }

    // (P v)^T, and S = lambda^n S + k^T (lambda^(n-1-j) v).
    const float fs = n == LA_C ? full : decay_pow_exact(g, n);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int c = 0; c < NC; ++c) S[b][c] *= fs;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4_t w0[NC], w1[NC], w2[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const u32x4_t vf = sVT[tok_at(16 * NC * wave + 16 * c + col, 4 * h + quad)];
        if constexpr (MODE != LA_LOCAL) {
#pragma unroll
          for (int t = 2 * h; t < 4; ++t) {
            o[t][c] = mfma(vf, sP[(pair_at(t, h) * 2 + 1) * 64 + lane], o[t][c]);
            o[t][c] = mfma(vf, sP[(pair_at(t, h) * 2 + 0) * 64 + lane], o[t][c]);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = 32 * h + 16 * (e >> 1) + 4 * quad + 2 * (e & 1);  // of the word's first token
          uint32_t x, y, z;
          split3(__uint_as_float(vf[e] << 16) * decay_pow(g2, n - 1 - j),
                 __uint_as_float(vf[e] & 0xFFFF0000u) * decay_pow(g2, n - 2 - j), x, y, z);
          w0[c][e] = x;
          w1[c][e] = y;
          w2[c][e] = z;
        }
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const u32x4_t kf = sKT[tok_at(16 * b + col, 4 * h + quad)];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          S[b][c] = mfma(kf, w2[c], S[b][c]);
          S[b][c] = mfma(kf, w1[c], S[b][c]);
          S[b][c] = mfma(kf, w0[c], S[b][c]);
        }
      }
    }
    if constexpr (MODE != LA_LOCAL) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int i = 16 * t + col;
        if (i >= n) continue;
        uint16_t* dst = o0 + (sp.tok + pos + i) * a.ld_out;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int j = dv0 + 16 * NC * wave + 16 * c + 4 * quad;
          const u32x2_t v = {bf16x2_bits(o[t][c][0] * a.scale, o[t][c][1] * a.scale),
                             bf16x2_bits(o[t][c][2] * a.scale, o[t][c][3] * a.scale)};
          if (j + 4 <= a.dv) {
            *reinterpret_cast<u32x2_any_t*>(dst + j) = v;
          } else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
              if (j + e < a.dv) dst[j + e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
          }
        }
      }
    }
    pos = next;
    if (singles) --singles;
  }
  if (!state_out) return;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * b + 4 * quad + r, j = dv0 + 16 * NC * wave + 16 * c + col;
        if (i < a.dk && j < a.dv) state_out[state0 + (size_t)i * a.dv + j] = S[b][c][r];
      }
}

// The scan over the segments of a sequence: every segment's own state becomes
// its entry state, and the last one's exit is the sequence's.
__global__ __launch_bounds__(256) void linear_scan_kernel(LinearArgs a, size_t state) {
  const size_t at = (size_t)blockIdx.x * 256 + threadIdx.x;  // of one sequence's heads' states
  if (at >= state * a.heads) return;
  const int seq = blockIdx.y;
  const int item0 = a.uniform_len >= 0 ? seq * a.uniform_segs : first_item(a, seq);
  const int item1 = a.uniform_len >= 0 ? item0 + a.uniform_segs : first_item(a, seq + 1);
  const int len = a.uniform_len >= 0 ? a.uniform_len : (int)(first_token(a, seq + 1) - first_token(a, seq));
  const float g = a.log_decay[at / state], full = decay_pow_exact(g, a.seg_len);
  const size_t step = state * a.heads;
  float s = a.state_in ? a.state_in[seq * step + at] : 0.0f;
  for (int i = item0; i < item1; ++i) {
    const float own = a.seg_state[i * step + at];
    a.seg_state[i * step + at] = s;
    const int n = len - (i - item0) * a.seg_len;
    s = fmaf(n >= a.seg_len ? full : decay_pow_exact(g, n), s, own);
  }
  if (a.state_out) a.state_out[seq * step + at] = s;
}

// Sequences of few tokens: the recurrence itself, the state read and written
// once.  A workgroup's threads lie over the state's columns, four each, and
// its rows; a token's readout meets in LDS.
template <class T, int ROWS>
__global__ __launch_bounds__(256) void linear_steps_kernel(LinearArgs a, int col_threads) {
  __shared__ float s_kq[2][128];
  __shared__ f32x4_t s_o[256];
  const int tid = threadIdx.x, ct = tid % col_threads, rt = tid / col_threads, row_threads = 256 / col_threads;
  const int j = 4 * (blockIdx.x * col_threads + ct), head = blockIdx.y, kv_head = head / (a.heads / a.kv_heads);
  const Span sp = span_of(a, blockIdx.z);
  const float g = a.log_decay[head], lam = (float)exp((double)g);
  const T* q0 = static_cast<const T*>(a.q) + (size_t)head * a.dk;
  const T* k0 = static_cast<const T*>(a.k) + (size_t)kv_head * a.dk;
  const T* v0 = static_cast<const T*>(a.v) + (size_t)kv_head * a.dv;
  T* o0 = static_cast<T*>(a.out) + (size_t)head * a.dv;
  const size_t state0 = ((size_t)sp.seq * a.heads + head) * a.dk * a.dv + j;
  const bool on = rt < row_threads && j < a.dv;
  const int left = a.dv - j;

  f32x4_t S[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int row = rt + row_threads * i;
    S[i] = f32x4_t{0, 0, 0, 0};
    if (on && a.state_in && row < a.dk) S[i] = load4<float>(a.state_in + state0 + (size_t)row * a.dv, left);
  }
  for (int t = 0; t < sp.len; ++t) {
    const size_t tok = sp.tok + t;
    for (int i = tid; i < 2 * a.dk; i += 256) {
      const int d = i < a.dk ? i : i - a.dk;
      const T* src = i < a.dk ? k0 + tok * a.ld_k + d : q0 + tok * a.ld_q + d;
      s_kq[i < a.dk ? 0 : 1][d] = load4<T>(src, 1)[0];
    }
    const f32x4_t v = on ? load4<T>(v0 + tok * a.ld_v + j, left) : f32x4_t{0, 0, 0, 0};
    __syncthreads();
    f32x4_t o = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int row = rt + row_threads * i;
      if (row < a.dk) {
        const float kd = s_kq[0][row], qd = s_kq[1][row];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          S[i][e] = fmaf(lam, S[i][e], kd * v[e]);
          o[e] = fmaf(qd, S[i][e], o[e]);
        }
      }
    }
    s_o[tid] = o;
    __syncthreads();
    if (rt == 0 && on) {
      for (int p = 1; p < row_threads; ++p) o += s_o[p * col_threads + ct];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) store1(o0 + tok * a.ld_out + j + e, o[e] * a.scale);
    }
  }
  if (!a.state_out || !on) return;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int row = rt + row_threads * i;
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

template <class T>
Status launch_steps(hipStream_t stream, const LinearArgs& a) {
  // 16 column threads cover 64 columns, 16 row threads 8 rows each of up to 128.
  const int cols = (a.dv + 3) / 4, ct = cols >= 16 ? 16 : cols;
  const dim3 grid((cols + ct - 1) / ct, a.heads, a.n_seqs);
  const int rows = (a.dk + 256 / ct - 1) / (256 / ct);
  if (rows <= 2)
    linear_steps_kernel<T, 2><<<grid, 256, 0, stream>>>(a, ct);
  else if (rows <= 4)
    linear_steps_kernel<T, 4><<<grid, 256, 0, stream>>>(a, ct);
  else
    linear_steps_kernel<T, 8><<<grid, 256, 0, stream>>>(a, ct);
  PSSA_LAUNCH_CHECK("linear_steps_kernel");
  return Status::Ok();
}

template <class T, int DKP, int NC, int MODE>
struct Chunks {
  static constexpr size_t kLds = (size_t)(2 * LA_C * (DKP + 4) + LA_C * (64 * NC + 4) + LA_C * 68) * 4;
  static constexpr auto kKernel = &linear_chunks_f32_kernel<T, DKP, NC, MODE>;
};
template <int DKP, int NC, int MODE>
struct Chunks<Bf16, DKP, NC, MODE> {
  static constexpr size_t kLds = (MODE == LA_LOCAL ? 0 : 2 * LA_C * (DKP * 2 + 16) + 12288) + (DKP + 64 * NC) * 144;
  static constexpr auto kKernel = &linear_chunks_bf16_kernel<DKP, NC, MODE>;
};

// Calls f with the kernel choice for a call's head widths and type.
template <int MODE, class F>
Status with_chunks(int dtype, int dk, int dv, F f) {
  auto typed = [&](auto t) {
    using T = decltype(t);
    auto wide = [&](auto dkp) {
      constexpr int D = decltype(dkp)::value;
      return dv > 64 ? f(Chunks<T, D, 2, MODE>{}, 2) : f(Chunks<T, D, 1, MODE>{}, 1);
    };
    if (dk <= 32) return wide(std::integral_constant<int, 32>{});
    if (dk <= 64) return wide(std::integral_constant<int, 64>{});
    return wide(std::integral_constant<int, 128>{});
  };
  return dtype == PSSA_HIP_F32 ? typed(0.0f) : typed(Bf16{});
}

template <int MODE>
Status launch_chunks(hipStream_t stream, int dtype, const LinearArgs& a) {
  return with_chunks<MODE>(dtype, a.dk, a.dv, [&](auto c, int nc) -> Status {
    const dim3 grid((a.dv + 64 * nc - 1) / (64 * nc), a.heads, a.items);
    c.kKernel<<<grid, 256, c.kLds, stream>>>(a);
    PSSA_LAUNCH_CHECK("linear_chunks_kernel");
    return Status::Ok();
  });
}

template <int MODE>
Status chunks_attributes() {
  for (int dtype : {PSSA_HIP_F32, PSSA_HIP_BF16})
    for (int dk : {32, 64, 128})
      for (int dv : {64, 128})
        PSSA_RETURN_IF(with_chunks<MODE>(dtype, dk, dv, [&](auto c, int) -> Status {
          PSSA_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(c.kKernel),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, (int)c.kLds));
          return Status::Ok();
        }));
  return Status::Ok();
}

}  // namespace

Status init_linear_attributes() {
  PSSA_RETURN_IF(chunks_attributes<LA_WHOLE>());
  PSSA_RETURN_IF(chunks_attributes<LA_LOCAL>());
  return chunks_attributes<LA_SEGMENT>();
}

int linear_segment(size_t n_seqs, size_t longest, size_t tokens, size_t heads, size_t d_val) {
  if (longest <= (size_t)kLinearSteps) return 0;
  const size_t tiles = heads * ((d_val + 127) / 128);
  const size_t blocks = n_seqs * tiles;
  (void)tokens;
  if (blocks >= 256 || longest < 512) return 0;
  // Segments of whole chunks, about one workgroup for each compute unit.
  const size_t segs = (256 + blocks - 1) / blocks;
  const size_t len = std::max<size_t>(256, (longest + segs - 1) / segs);
  return (int)((len + LA_C - 1) / LA_C * LA_C);
}

Status launch_linear_attention(hipStream_t stream, int dtype, const LinearArgs& a, int longest) {
  if (longest <= kLinearSteps)
    return dtype == PSSA_HIP_F32 ? launch_steps<float>(stream, a) : launch_steps<Bf16>(stream, a);
  if (!a.seg_state) return launch_chunks<LA_WHOLE>(stream, dtype, a);
  PSSA_RETURN_IF(launch_chunks<LA_LOCAL>(stream, dtype, a));
  const size_t state = (size_t)a.dk * a.dv;
  linear_scan_kernel<<<dim3((uint32_t)((state * a.heads + 255) / 256), a.n_seqs), 256, 0, stream>>>(a, state);
  PSSA_LAUNCH_CHECK("linear_scan_kernel");
  return launch_chunks<LA_SEGMENT>(stream, dtype, a);
}

}  // namespace pssa
