// Linear attention with a decay for each head: the recurrence
//   S_t = lambda_h S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t
// over packed sequences, from one token to long prompts.
//
// Prompts run in chunks of 64 tokens (32 in fp32).  Within a chunk entered with state S
// (i, j count its tokens, n of them)
//   o_i = scale (lambda^(i+1) q_i S + sum_{j<=i} lambda^(i-j) (q_i k_j) v_j)
//   S'  = lambda^n S + sum_j k_j (lambda^(n-1-j) v_j)^T,
// four matrix products.  A workgroup walks one sequence's (or segment's)
// chunks for one head and a tile of value columns, of which a wave owns 16;
// its part of S stays in its accumulators, and these are the product q S's
// operand as they stand: the accumulator layout (lane l holds column l % 16,
// rows 4 (l / 16) + r) is the matrix instruction's operand layout once q's
// columns are read in the same order.  The next chunk's rows go straight into
// the other of two LDS buffers meanwhile.
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
// state is (the sequence's, or its own one in the scratch of a split call,
// which seg_state tells from one that is not).
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
    int lo = item, hi = item;  // not split: the tables have no items
    if (a.seg_state) lo = 0, hi = a.n_seqs - 1;  // the last sequence that begins at or before the item
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first_item(a, mid) <= item) lo = mid; else hi = mid - 1;
    }
    s.seq = lo;
    seg = a.seg_state ? item - first_item(a, lo) : 0;
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

// Any widths and alignment: bf16 inputs widened for fp32 products.
template <class T, int DKP, int NC, int MODE>
__global__ __launch_bounds__(256) void linear_chunks_any_kernel(LinearArgs a) {
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
// the state is an fp32 result.  Three parts of P and S too took 51.9 us for
// 49.3 and 44.6 for 41.1 (8192 tokens, 8 heads of 128; 16 x 1024, 12 of 64):
// then 0.03% of the outputs lie a bf16 step beside the fp32 form's instead of
// 0.24%, and the error against 64 bits is the same to three digits.
//
// A 32-deep operand's lane holds eight places: 4 quad + r of one 16-row tile
// and of the next, the order in which two accumulators lie in the lane's
// registers.  So S and P are operands without a move (P passes through LDS as
// ready fragments because one wave computes 16 rows of it and every wave
// needs all), and what meets them is read in that order: rows of q in two
// halves, columns of k and v (their tokens) by ds_read_b64_tr_b16, which gives
// a lane four rows of its column.  Rows go from memory straight into one of
// two LDS buffers while the other one's chunk is worked on.
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
// One fragment.  Written out, with their
// wait, because the compiler would let the builtin wait for the loads that
// are on their way into the other buffer.
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

// Element i of bf16 values in a register or LDS.
template <class V>
__device__ __forceinline__ float bf16_at(const V* p, int i) {
  return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << 16);
}

// Of a chunk's P the pairs of a query tile and a key half that hold anything,
// the largest first: a wave computes one or two.
constexpr int kLdsOnly = 0xF | (0x3 << 14) | (0x7 << 4);  // s_waitcnt lgkmcnt(0)
constexpr int kPairs = 6;
__device__ __forceinline__ int pair_query(int p) { return (0x201233 >> (4 * p)) & 3; }
__device__ __forceinline__ int pair_half(int p) { return (0x100010 >> (4 * p)) & 1; }
constexpr int pair_of(int t, int h) { return t == 3 ? h : t == 2 ? (h ? 5 : 2) : t == 1 ? 3 : 4; }

// What stands in for rows and columns that are not there.
__device__ uint32_t g_nothing[4];

// Groups of waves that keep the state, a part of its rows each: two where it
// is all that a workgroup computes, which otherwise would leave a SIMD one wave
// (8192 bf16 tokens, 8 heads of 128: 14.7 us against 16.5).
template <int DKP, bool LOCAL>
constexpr int kKeepers = LOCAL && DKP >= 64 ? 2 : 1;

// LDS units (16 bytes) of the kernel: two buffers of q | k | v, P, and q S.
constexpr int WAVES = 4;  // of a group: 16 value columns each
template <int DKP, bool LOCAL>
struct ChunkLds {
  static constexpr int kQ = LOCAL ? 0 : LA_C * DKP / 8, kK = LA_C * DKP / 8, kV = LA_C * 2 * WAVES;
  static constexpr int kBuffer = kQ + kK + kV;
  static constexpr size_t kBytes = 16 * (size_t)(2 * kBuffer + (LOCAL ? 0 : kPairs * 128 + WAVES * 256));
};

// A tile of 16 WAVES value columns takes two groups of as many waves: one
// computes P and P v and stores the outputs, the other keeps S, computes q S
// (handed over through LDS) and the next S.  Both halves of a chunk's work
// are about as long, and every SIMD has a wave of each (heads of 64: 5500
// cycles a chunk, against 7000 of one group that does both in turn).
// LB: bytes of one load, 16 where every row and head is so aligned, else 4.
template <int DKP, int MODE, int LB>
__global__ __launch_bounds__((64 * WAVES * (MODE == LA_LOCAL ? kKeepers<DKP, true> : 2)), (MODE == LA_LOCAL || DKP == 128 ? 2 : 4)) void linear_chunks_bf16_kernel(
    LinearArgs a) {
  constexpr bool LOCAL = MODE == LA_LOCAL;
  constexpr int KEEPERS = kKeepers<DKP, LOCAL>, ALL = (LOCAL ? 0 : WAVES) + KEEPERS * WAVES;
  using Lds = ChunkLds<DKP, LOCAL>;
  constexpr int DVT = 16 * WAVES, NB = DKP / 16 / KEEPERS, KP = DKP / 32;
  constexpr int LOADS = Lds::kBuffer / 64 * (16 / LB), PER = (LOADS + ALL - 1) / ALL;  // instructions of a chunk, of a wave
  constexpr int SLOTS = (kPairs + WAVES - 1) / WAVES;
  extern __shared__ __attribute__((aligned(256))) u32x4_t s_bf[];
  u32x4_t* sP = s_bf + 2 * Lds::kBuffer;  // [pairs][2 parts][64 lanes]
  f32x4_t* sO = reinterpret_cast<f32x4_t*>(sP + kPairs * 128);  // [column group][query tile][64 lanes]
  const int lane = threadIdx.x & 63, in_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool keeps_state = LOCAL || in_all >= WAVES;
  const int wave = in_all % WAVES;  // of its group: its 16 columns
  const int b_first = LOCAL ? NB * (in_all / WAVES) : 0;  // of the state's tiles of 16 rows
  const int dv0 = blockIdx.x * DVT, head = blockIdx.y, kv_head = head / (a.heads / a.kv_heads);
  const Span sp = span_of(a, blockIdx.z);
  const float g = a.log_decay[head], g2 = g * kLog2e;
  const size_t state0 = ((size_t)(MODE == LA_WHOLE ? sp.seq : sp.item) * a.heads + head) * a.dk * a.dv;
  const float* state_in = MODE == LA_WHOLE ? a.state_in : LOCAL ? nullptr : a.seg_state;
  float* state_out = MODE == LA_WHOLE ? a.state_out : LOCAL ? a.seg_state : nullptr;

  // The n tokens from pos on into a buffer, straight from memory.  A load's 64
  // lanes fill 64 neighbouring places, so each lane looks up what belongs in
  // its own: rows swizzled by row_unit, zeros where nothing is.
  struct Piece {
    const uint16_t* base;  // of the chunk's first row
    size_t ld;
    int row, c, width;
  };
  auto piece = [&](int i, int ln) {
    const int at = (i * ALL + in_all) * 64 / (16 / LB);  // first unit
    // Where all waves load from the same array the compiler sees which.
    constexpr int STEP = ALL * 64 / (16 / LB);
    const bool even = Lds::kQ % STEP == 0 && Lds::kK % STEP == 0;
    const int by = even ? i * STEP : at;
    const bool is_q = by < Lds::kQ, is_k = !is_q && by < Lds::kQ + Lds::kK;
    const int unit = at - (is_q ? 0 : is_k ? Lds::kQ : Lds::kQ + Lds::kK) + ln / (16 / LB);
    const int units = is_q || is_k ? DKP / 8 : DVT / 8;
    Piece p;
    p.row = unit / units;
    const int here = unit % units;
    p.c = 8 * (is_q || is_k ? row_unit<DKP>(p.row, here) : row_unit<DVT>(p.row, here)) + ln % (16 / LB) * (LB / 2);
    p.ld = is_q ? a.ld_q : is_k ? a.ld_k : a.ld_v;
    p.width = is_q || is_k ? a.dk : a.dv - dv0;
    p.base = is_q   ? static_cast<const uint16_t*>(a.q) + (size_t)head * a.dk
             : is_k ? static_cast<const uint16_t*>(a.k) + (size_t)kv_head * a.dk
                    : static_cast<const uint16_t*>(a.v) + (size_t)kv_head * a.dv + dv0;
    return p;
  };
  constexpr bool KEEP = LB == 16;  // the places of a whole chunk's pieces stay in registers
  uint32_t place[KEEP ? PER : 1];
  if constexpr (KEEP) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const Piece p = piece(i, lane);
      place[i] = __umul24(p.row, (uint32_t)p.ld) + p.c;
    }
  }
  const bool heads_fill = a.dk == DKP && a.dv - dv0 >= DVT;
  auto issue = [&](int pos, int n, u32x4_t* buffer, int ln) {
    const size_t tok = sp.tok + pos;
    const bool plain = KEEP && heads_fill && n == LA_C;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (LOADS % ALL != 0 && i * ALL + in_all >= LOADS) continue;
      auto* dst = (__attribute__((address_space(3))) void*)(reinterpret_cast<char*>(buffer) + (i * ALL + in_all) * 64 * LB);
      const Piece p = piece(i, ln);
      const uint16_t* base = p.base + tok * p.ld;
      const void* src;
      if (plain)
        src = base + place[KEEP ? i : 0];
      else
        src = p.row < n && p.c < p.width ? static_cast<const void*>(base + (__umul24(p.row, (uint32_t)p.ld) + p.c)) : g_nothing;
      if constexpr (LB == 16)
        __builtin_amdgcn_global_load_lds(src, dst, 16, 0, 0);
      else
        __builtin_amdgcn_global_load_lds(src, dst, 4, 0, 0);
    }
  };

  int n = min(LA_C, sp.len);
  if (n > 0) issue(0, n, s_bf, lane);
  // S: rows 16 (b_first + b) + 4 quad + r, column dv0 + 16 wave + col.
  f32x4_t S[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * (b_first + b) + 4 * (lane >> 4) + r, j = dv0 + 16 * wave + (lane & 15);
      S[b][r] = keeps_state && state_in && i < a.dk && j < a.dv ? state_in[state0 + (size_t)i * a.dv + j] : 0.0f;
    }
  // The state's loads end here: waited for in the loop, they would be waited
  // for together with the loads of every next chunk.
#pragma unroll
  for (int b = 0; b < NB; ++b) asm volatile("" : "+v"(S[b]));
  // Powers of the decay, as products of a lane's and a uniform one, every
  // exponent >= 0.  The first group of waves: scale lambda^(i-j) in P's
  // diagonal tiles, lambda^(i-j+15) for the others.  The second: scale
  // lambda^(i+1) for the lane's queries, lambda^(n-1-j) for its tokens of a
  // half chunk (n_left and fs = lambda^n say which).
  float pw[12], fs = 1.0f;
  int n_left = -1;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int col = lane & 15, quad = lane >> 4;
    pw[t] = LOCAL ? 0.0f : a.scale * decay_pow(g2, keeps_state ? 16 * t + col + 1 : col - 4 * quad - t);
    pw[4 + t] = LOCAL ? 0.0f : decay_pow(g2, col - 4 * quad - t + 15);
    pw[8 + t] = 0.0f;
  }
  const float tile_pow[4] = {0.0f, a.scale * decay_pow(g2, 1), a.scale * decay_pow(g2, 17), a.scale * decay_pow(g2, 33)};
  // A chunk's outputs are stored in the next one's course, before which every
  // memory operation of the chunk before has to have ended.  The waves that
  // store have no state: the outputs lie in its registers.
  auto put = [&](int pos, int n, int ln) {
    const int j = dv0 + 16 * wave + 4 * (ln >> 4);
    uint16_t* base = static_cast<uint16_t*>(a.out) + (size_t)head * a.dv + (sp.tok + pos) * a.ld_out;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int i = 16 * t + (ln & 15);
      if (i >= n || j >= a.dv) continue;
      const u32x2_t v = {__float_as_uint(S[t >> 1][2 * (t & 1)]), __float_as_uint(S[t >> 1][2 * (t & 1) + 1])};
      uint16_t* dst = base + (__umul24(i, (uint32_t)a.ld_out) + j);
      if (LB == 16 || j + 4 <= a.dv) {
        *reinterpret_cast<u32x2_any_t*>(dst) = v;
      } else {  // heads are whole in pairs
        dst[0] = (uint16_t)v[0];
        dst[1] = (uint16_t)(v[0] >> 16);
      }
    }
  };

  u32x4_t* buffer = s_bf;
  for (int pos = 0, before = 0; pos < sp.len; pos += n, before = n) {
    n = min(LA_C, sp.len - pos);
    // The lane's number, new for the compiler in each chunk: what follows from
    // it is worked out again, as kept it would take more registers than the
    // kernel's work.
    int ln = lane;
    asm volatile("" : "+v"(ln));
#pragma unroll
    for (int i = 0; i < 12; ++i) asm volatile("" : "+v"(pw[i]));
    const int col = ln & 15, quad = ln >> 4;
    __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
    __syncthreads();  // the chunk is there, and the one before is read
    u32x4_t* other = buffer == s_bf ? s_bf + Lds::kBuffer : s_bf;
    if (pos + n < sp.len) issue(pos + n, min(LA_C, sp.len - pos - n), other, ln);
    if constexpr (!LOCAL) {
      if (before && !keeps_state) put(pos - before, before, ln);
    }
    const u32x4_t *sQ = buffer, *sK = buffer + Lds::kQ, *sV = sK + Lds::kK;
    buffer = other;

    if (!LOCAL && !keeps_state) {
      // P^T = scale (k q^T) lambda^(i-j), j <= i, of the wave's pairs.
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) {
        const int p = wave + WAVES * s, qt = pair_query(p), half = pair_half(p);
        if (p >= kPairs) continue;  // uniform
        f32x4_t acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int kp = 0; kp < KP; ++kp) {
          const u32x4_t qf = row_frag<DKP>(sQ, 16 * qt + col, 4 * kp + quad);
#pragma unroll
          for (int x = 0; x < 2; ++x) acc[x] = mfma(row_frag<DKP>(sK, 32 * half + 16 * x + col, 4 * kp + quad), qf, acc[x]);
        }
        u32x4_t hi, lo;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int ahead = qt - 2 * half - x;  // tiles from the keys to the queries
          const float u = ahead == 1 ? tile_pow[1] : ahead == 2 ? tile_pow[2] : tile_pow[3];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float d = ahead == 0 ? pw[r] : pw[4 + r] * u;
            acc[x][r] = 16 * ahead + col >= 4 * quad + r ? acc[x][r] * d : 0.0f;
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t h, l;
            split2(acc[x][2 * e], acc[x][2 * e + 1], h, l);
            hi[2 * x + e] = h;
            lo[2 * x + e] = l;
          }
        }
        sP[(2 * p) * 64 + ln] = hi;
        sP[(2 * p + 1) * 64 + ln] = lo;
      }
    } else if (!LOCAL) {
      // (q S)^T, each query's column times scale lambda^(i+1).
      f32x4_t o[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) o[t] = f32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int kp = 0; kp < KP; ++kp) {
        u32x4_t hi, lo, qf[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) qf[t] = order_frag<DKP>(sQ, 16 * t + col, kp, quad);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t x, y;
          split2(S[2 * kp + (e >> 1)][2 * (e & 1)], S[2 * kp + (e >> 1)][2 * (e & 1) + 1], x, y);
          hi[e] = x;
          lo[e] = y;
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) o[t] = mfma(lo, qf[t], o[t]);
#pragma unroll
        for (int t = 0; t < 4; ++t) o[t] = mfma(hi, qf[t], o[t]);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) sO[(4 * wave + t) * 64 + ln] = o[t] * pw[t];
    }
    if constexpr (!LOCAL) {
      // P and q S are there; the next chunk's loads stay in flight (__syncthreads would wait for them).
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(kLdsOnly);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    }

    if (!LOCAL && !keeps_state) {
      // + (P v)^T, 32 tokens at a time.
      u32x4_t vf[2];
      uint32_t odd = 0;  // an exponent of ones carries into the bit above it
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        turned_frag<DVT>(turned_at<DVT>(sV, 32 * h, 16 * wave, ln), vf[h]);
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= (vf[h][e] & 0x7F807F80u) + 0x00800080u;
      }
      if (__any((odd & 0x80008000u) != 0)) {
        // Values that are not finite leave the product, where 0 times one
        // would reach the queries before it, and are added one by one.
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t carry = ((vf[h][e] & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
            vf[h][e] &= ~((carry >> 15) * 0xFFFFu);
          }
#pragma unroll 1
        for (int j = 0; j < LA_C; ++j) {
          const u32x2_t v4 = four_of<DVT>(sV, j, 16 * wave + 4 * quad);
#pragma unroll 1
          for (int t = j >> 4; t < 4; ++t) {
            const int pair = t == 3 ? j >> 5 : t == 2 ? (j >> 5 ? 5 : 2) : t == 1 ? 3 : 4;
            const float p = bf16_at(&sP[2 * pair * 64 + 16 * ((j & 15) >> 2) + col], 4 * ((j >> 4) & 1) + (j & 3));
            f32x4_t& o = sO[(4 * wave + t) * 64 + ln];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float v = __uint_as_float(r & 1 ? v4[r >> 1] & 0xFFFF0000u : v4[r >> 1] << 16);
              if (16 * t + col >= j && !(fabsf(v) < INFINITY)) o[r] += p * v;
            }
          }
        }
      }
      f32x4_t o[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) o[t] = sO[(4 * wave + t) * 64 + ln];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int part = 1; part >= 0; --part)
#pragma unroll
          for (int t = 2 * h; t < 4; ++t) o[t] = mfma(vf[h], sP[(2 * pair_of(t, h) + part) * 64 + ln], o[t]);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        S[t >> 1][2 * (t & 1)] = __uint_as_float(bf16x2_bits(o[t][0], o[t][1]));
        S[t >> 1][2 * (t & 1) + 1] = __uint_as_float(bf16x2_bits(o[t][2], o[t][3]));
      }
    } else {
      // S = lambda^n S + k^T (lambda^(n-1-j) v), 32 tokens at a time.
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int nh = min(max(n - 32 * h, 0), 32);
        if (nh != n_left) {
          n_left = nh;
          fs = decay_pow_exact(g, nh);
#pragma unroll
          for (int e = 0; e < 8; ++e) pw[4 + e] = decay_pow(g2, nh - 1 - (16 * (e >> 2) + 4 * quad + (e & 3)));
        }
        constexpr int BG = NB < 4 ? NB : 4;  // tiles whose sums run beside each other
        u32x4_t vf, kf[BG];
        turned_frags<DVT, DKP, BG>(turned_at<DVT>(sV, 32 * h, 16 * wave, ln), vf, turned_at<DKP>(sK, 32 * h, 16 * b_first, ln), kf);
        u32x4_t w[3];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t x, y, z;
          split3(__uint_as_float(vf[e] << 16) * pw[4 + 2 * e], __uint_as_float(vf[e] & 0xFFFF0000u) * pw[5 + 2 * e], x, y, z);
          w[0][e] = x;
          w[1][e] = y;
          w[2][e] = z;
        }
#pragma unroll
        for (int b0 = 0; b0 < NB; b0 += BG) {
          if constexpr (NB > 4) {
            if (b0) turned_frags<DKP>(turned_at<DKP>(sK, 32 * h, 16 * (b_first + b0), ln), kf);
          }
#pragma unroll
          for (int b = 0; b < BG; ++b) S[b0 + b] *= fs;
#pragma unroll
          for (int p = 2; p >= 0; --p)
#pragma unroll
            for (int b = 0; b < BG; ++b) S[b0 + b] = mfma(kf[b], w[p], S[b0 + b]);
        }
      }
    }
  }
  if constexpr (!LOCAL) {
    if (sp.len > 0 && !keeps_state) put(sp.len - n, n, lane);
  }
  if (!state_out || !keeps_state) return;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * (b_first + b) + 4 * (lane >> 4) + r, j = dv0 + 16 * wave + (lane & 15);
      if (i < a.dk && j < a.dv) state_out[state0 + (size_t)i * a.dv + j] = S[b][r];
    }
}

// ---------------------------------------------------------------- fp32 inputs
// The same walk on v_mfma_f32_16x16x4_f32, exact fp32 products, in chunks of
// 32 tokens: the instruction has a sixteenth of the bf16 one's rate, so a
// shorter chunk's smaller triangle of P saves more than its barriers cost.
// Its operands are single elements, four of which follow one another in an
// accumulator's rows, so rows of q and k are read 16 bytes at a time and
// columns of k and v element by element.  9 prompts of 5 to 1000 tokens, 12
// heads of 64, not split: 89 us, against 173 us of the kernel for any widths
// in chunks of 64.
constexpr int LA_C32 = 32;

template <int DKP, bool LOCAL>
struct ChunkLds32 {
  static constexpr int kQ = LOCAL ? 0 : LA_C32 * DKP / 4, kK = LA_C32 * DKP / 4, kV = LA_C32 * 16;
  static constexpr int kBuffer = kQ + kK + kV;
  static constexpr size_t kBytes = 16 * (size_t)(2 * kBuffer + (LOCAL ? 0 : 3 * 64 + 4 * 128));
};
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

template <int DKP, int MODE, int LB>
__global__ __launch_bounds__((MODE == LA_LOCAL ? 256 * kKeepers<DKP, true> : 512), (MODE == LA_LOCAL || DKP == 128 ? 2 : 4)) void linear_chunks_fp32_kernel(
    LinearArgs a) {
  constexpr bool LOCAL = MODE == LA_LOCAL;
  using Lds = ChunkLds32<DKP, LOCAL>;
  constexpr int KEEPERS = kKeepers<DKP, LOCAL>, ALL = LOCAL ? 4 * KEEPERS : 8, DVT = 64, NB = DKP / 16 / KEEPERS;
  constexpr int LOADS = Lds::kBuffer / 64 * (16 / LB), PER = (LOADS + ALL - 1) / ALL;
  extern __shared__ __attribute__((aligned(256))) f32x4_t s_f32[];
  f32x4_t* sP = s_f32 + 2 * Lds::kBuffer;  // [tiles (1, 0), (1, 1), (0, 0) of queries and keys][64 lanes]
  f32x4_t* sO = sP + 3 * 64;               // [column group][query tile][64 lanes]
  const int lane = threadIdx.x & 63, in_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool keeps_state = LOCAL || in_all >= WAVES;
  const int wave = in_all % WAVES;  // of its group: its 16 columns
  const int b_first = LOCAL ? NB * (in_all / WAVES) : 0;  // of the state's tiles of 16 rows
  const int dv0 = blockIdx.x * DVT, head = blockIdx.y, kv_head = head / (a.heads / a.kv_heads);
  const Span sp = span_of(a, blockIdx.z);
  const float g = a.log_decay[head], g2 = g * kLog2e;
  const size_t state0 = ((size_t)(MODE == LA_WHOLE ? sp.seq : sp.item) * a.heads + head) * a.dk * a.dv;
  const float* state_in = MODE == LA_WHOLE ? a.state_in : LOCAL ? nullptr : a.seg_state;
  float* state_out = MODE == LA_WHOLE ? a.state_out : LOCAL ? a.seg_state : nullptr;

  auto issue = [&](int pos, int n, f32x4_t* buffer, int ln) {
    const size_t tok = sp.tok + pos;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (LOADS % ALL != 0 && i * ALL + in_all >= LOADS) continue;
      const int at = (i * ALL + in_all) * 64 / (16 / LB);  // first unit
      constexpr int STEP = ALL * 64 / (16 / LB);
      const bool even = Lds::kQ % STEP == 0 && Lds::kK % STEP == 0;
      const int by = even ? i * STEP : at;
      const bool is_q = by < Lds::kQ, is_k = !is_q && by < Lds::kQ + Lds::kK;
      const int unit = at - (is_q ? 0 : is_k ? Lds::kQ : Lds::kQ + Lds::kK) + ln / (16 / LB);
      const int units = is_q || is_k ? DKP / 4 : DVT / 4;
      const int row = unit / units, c = 4 * row_unit32(row, unit % units) + ln % (16 / LB) * (LB / 4);
      const size_t ld = is_q ? a.ld_q : is_k ? a.ld_k : a.ld_v;
      const int width = is_q || is_k ? a.dk : a.dv - dv0;
      const float* base = (is_q   ? static_cast<const float*>(a.q) + (size_t)head * a.dk
                           : is_k ? static_cast<const float*>(a.k) + (size_t)kv_head * a.dk
                                  : static_cast<const float*>(a.v) + (size_t)kv_head * a.dv + dv0) +
                          tok * ld;
      const void* src = row < n && c < width ? static_cast<const void*>(base + (__umul24(row, (uint32_t)ld) + c)) : g_nothing;
      auto* dst = (__attribute__((address_space(3))) void*)(reinterpret_cast<char*>(buffer) + (i * ALL + in_all) * 64 * LB);
      if constexpr (LB == 16)
        __builtin_amdgcn_global_load_lds(src, dst, 16, 0, 0);
      else
        __builtin_amdgcn_global_load_lds(src, dst, 4, 0, 0);
    }
  };

  int n = min(LA_C32, sp.len);
  if (n > 0) issue(0, n, s_f32, lane);
  // S: rows 16 (b_first + b) + 4 quad + r, column dv0 + 16 wave + col.
  f32x4_t S[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * (b_first + b) + 4 * (lane >> 4) + r, j = dv0 + 16 * wave + (lane & 15);
      S[b][r] = keeps_state && state_in && i < a.dk && j < a.dv ? state_in[state0 + (size_t)i * a.dv + j] : 0.0f;
    }
#pragma unroll
  for (int b = 0; b < NB; ++b) asm volatile("" : "+v"(S[b]));  // these loads end here, see above
  // The powers as above, of 32 tokens: 4 for the diagonal tiles and 4 for the
  // other one, or 2 for the queries and, behind them, 8 for the tokens.
  float pw[12], fs = 1.0f;
  int n_left = -1;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int col = lane & 15, quad = lane >> 4;
    pw[t] = LOCAL ? 0.0f : a.scale * decay_pow(g2, keeps_state ? 16 * (t & 1) + col + 1 : col - 4 * quad - t);
    pw[4 + t] = LOCAL ? 0.0f : a.scale * decay_pow(g2, 16 + col - 4 * quad - t);
    pw[8 + t] = 0.0f;
  }
  auto put = [&](int pos, int n, int ln) {
    const int j = dv0 + 16 * wave + 4 * (ln >> 4);
    float* base = static_cast<float*>(a.out) + (size_t)head * a.dv + (sp.tok + pos) * a.ld_out;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int i = 16 * t + (ln & 15);
      if (i >= n || j >= a.dv) continue;
      float* dst = base + (__umul24(i, (uint32_t)a.ld_out) + j);
      if (j + 4 <= a.dv) {
        *reinterpret_cast<f32x4_any_t*>(dst) = S[t];
      } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (j + e < a.dv) dst[e] = S[t][e];
      }
    }
  };

  f32x4_t* buffer = s_f32;
  for (int pos = 0, before = 0; pos < sp.len; pos += n, before = n) {
    n = min(LA_C32, sp.len - pos);
    int ln = lane;  // new for the compiler, as above
    asm volatile("" : "+v"(ln));
#pragma unroll
    for (int i = 0; i < 12; ++i) asm volatile("" : "+v"(pw[i]));
    const int col = ln & 15, quad = ln >> 4;
    __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
    __syncthreads();  // the chunk is there, and the one before is read
    f32x4_t* other = buffer == s_f32 ? s_f32 + Lds::kBuffer : s_f32;
    if (pos + n < sp.len) issue(pos + n, min(LA_C32, sp.len - pos - n), other, ln);
    if constexpr (!LOCAL) {
      if (before && !keeps_state) put(pos - before, before, ln);
    }
    const f32x4_t *sQ = buffer, *sK = buffer + Lds::kQ, *sV = sK + Lds::kK;
    buffer = other;

    if (!LOCAL && !keeps_state) {
      if (wave < 3) {  // P^T = scale (k q^T) lambda^(i-j), j <= i, one tile each
        const int qt = wave < 2, kt = wave == 1;
        f32x4_t p = {0, 0, 0, 0};
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const f32x4_t kf = row_frag32<DKP>(sK, 16 * kt + col, 4 * b + quad);
          const f32x4_t qf = row_frag32<DKP>(sQ, 16 * qt + col, 4 * b + quad);
#pragma unroll
          for (int r = 0; r < 4; ++r) p = mfma32(kf[r], qf[r], p);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) p[r] = wave == 0 ? p[r] * pw[4 + r] : col >= 4 * quad + r ? p[r] * pw[r] : 0.0f;
        sP[wave * 64 + ln] = p;
      }
    } else if (!LOCAL) {
      // (q S)^T, each query's column times scale lambda^(i+1).
      f32x4_t o[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        f32x4_t qf[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) qf[t] = row_frag32<DKP>(sQ, 16 * t + col, 4 * b + quad);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int t = 0; t < 2; ++t) o[t] = mfma32(S[b][r], qf[t][r], o[t]);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) sO[(2 * wave + t) * 64 + ln] = o[t] * pw[t];
    }
    if constexpr (!LOCAL) {
      asm volatile("" ::: "memory");  // as above: no wait for the next chunk's loads
      __builtin_amdgcn_s_waitcnt(kLdsOnly);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    }

    float v[2][4];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) v[kt][r] = element32<DVT>(sV, 16 * kt + 4 * quad + r, 16 * wave + col);
    if (!LOCAL && !keeps_state) {
      // + (P v)^T; values that are not finite one by one, as above.
      bool odd = false;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) odd |= !(fabsf(v[kt][r]) < INFINITY);
      if (__any(odd)) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!(fabsf(v[kt][r]) < INFINITY)) v[kt][r] = 0.0f;
#pragma unroll 1
        for (int j = 0; j < LA_C32; ++j) {
          const f32x4_t v4 = sV[j * (DVT / 4) + row_unit32(j, 4 * wave + quad)];
#pragma unroll 1
          for (int t = j >> 4; t < 2; ++t) {
            const int tile = t == 0 ? 2 : j >> 4;
            const float p = reinterpret_cast<const float*>(&sP[tile * 64 + 16 * ((j & 15) >> 2) + col])[j & 3];
            f32x4_t& o = sO[(2 * wave + t) * 64 + ln];
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (16 * t + col >= j && !(fabsf(v4[r]) < INFINITY)) o[r] += p * v4[r];
          }
        }
      }
      f32x4_t o[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) o[t] = sO[(2 * wave + t) * 64 + ln];
      const f32x4_t p10 = sP[ln], p11 = sP[64 + ln], p00 = sP[128 + ln];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        o[0] = mfma32(v[0][r], p00[r], o[0]);
        o[1] = mfma32(v[0][r], p10[r], o[1]);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) o[1] = mfma32(v[1][r], p11[r], o[1]);
#pragma unroll
      for (int t = 0; t < 2; ++t) S[t] = o[t];
    } else {
      // S = lambda^n S + k^T (lambda^(n-1-j) v).
      if (n != n_left) {
        n_left = n;
        fs = decay_pow_exact(g, n);
#pragma unroll
        for (int e = 0; e < 8; ++e) pw[4 + e] = decay_pow(g2, n - 1 - (16 * (e >> 2) + 4 * quad + (e & 3)));
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) S[b] *= fs;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float w = v[kt][r] * pw[4 + 4 * kt + r];
#pragma unroll
          for (int b = 0; b < NB; ++b)
            S[b] = mfma32(element32<DKP>(sK, 16 * kt + 4 * quad + r, 16 * (b_first + b) + col), w, S[b]);
        }
    }
  }
  if constexpr (!LOCAL) {
    if (sp.len > 0 && !keeps_state) put(sp.len - n, n, lane);
  }
  if (!state_out || !keeps_state) return;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * (b_first + b) + 4 * (lane >> 4) + r, j = dv0 + 16 * wave + (lane & 15);
      if (i < a.dk && j < a.dv) state_out[state0 + (size_t)i * a.dv + j] = S[b][r];
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
  constexpr int AHEAD = 8;  // segments whose loads are in flight together
  for (int i0 = item0; i0 < item1; i0 += AHEAD) {
    float own[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) own[j] = a.seg_state[min(i0 + j, item1 - 1) * step + at];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (i0 + j >= item1) continue;
      a.seg_state[(i0 + j) * step + at] = s;
      const int n = len - (i0 + j - item0) * a.seg_len;
      s = fmaf(n >= a.seg_len ? full : decay_pow_exact(g, n), s, own[j]);
    }
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

// The kernel of a call and the value columns of its workgroups: loads of LB
// bytes, or (0) the one that takes any width and alignment.
template <class T, int DKP, int NC, int MODE, int LB>
struct Chunks {
  static constexpr size_t kLds = (size_t)(2 * LA_C * (DKP + 4) + LA_C * (64 * NC + 4) + LA_C * 68) * 4;
  static constexpr int kThreads = 256, kColumns = 64 * NC;
  static constexpr auto kKernel = &linear_chunks_any_kernel<T, DKP, NC, MODE>;
};
template <int DKP, int NC, int MODE, int LB>
struct ChunksBf16 {
  static constexpr size_t kLds = ChunkLds<DKP, MODE == LA_LOCAL>::kBytes;
  static constexpr int kThreads = MODE == LA_LOCAL ? 256 * kKeepers<DKP, true> : 512, kColumns = 64;
  static constexpr auto kKernel = &linear_chunks_bf16_kernel<DKP, MODE, LB>;
};
template <int DKP, int NC, int MODE>
struct Chunks<Bf16, DKP, NC, MODE, 16> : ChunksBf16<DKP, NC, MODE, 16> {};
template <int DKP, int NC, int MODE>
struct Chunks<Bf16, DKP, NC, MODE, 4> : ChunksBf16<DKP, NC, MODE, 4> {};
template <int DKP, int NC, int MODE, int LB>
struct Chunks<float, DKP, NC, MODE, LB> {
  static constexpr size_t kLds = ChunkLds32<DKP, MODE == LA_LOCAL>::kBytes;
  static constexpr int kThreads = MODE == LA_LOCAL ? 256 * kKeepers<DKP, true> : 512, kColumns = 64;
  static constexpr auto kKernel = &linear_chunks_fp32_kernel<DKP, MODE, LB>;
};

// Calls f with the kernel for a call's type, head widths and loads.
template <int MODE, class F>
Status with_chunks(int dtype, int dk, int dv, int load, F f) {
  auto typed = [&](auto t, auto lb) {
    using T = decltype(t);
    constexpr int LB = decltype(lb)::value;
    auto wide = [&](auto dkp) {
      constexpr int D = decltype(dkp)::value;
      return dv > 64 ? f(Chunks<T, D, 2, MODE, LB>{}) : f(Chunks<T, D, 1, MODE, LB>{});
    };
    if (dk <= 32) return wide(std::integral_constant<int, 32>{});
    if (dk <= 64) return wide(std::integral_constant<int, 64>{});
    return wide(std::integral_constant<int, 128>{});
  };
  const std::integral_constant<int, 16> wide_loads;
  const std::integral_constant<int, 4> short_loads;
  if (dtype == PSSA_HIP_F32) return load == 16 ? typed(0.0f, wide_loads) : typed(0.0f, short_loads);
  if (load == 16) return typed(Bf16{}, wide_loads);
  if (load == 4) return typed(Bf16{}, short_loads);
  return typed(Bf16{}, std::integral_constant<int, 0>{});
}

// The largest load that every row's and head's start is aligned to.
int load_bytes(int dtype, const LinearArgs& a) {
  const size_t all = (size_t)a.q | (size_t)a.k | (size_t)a.v |
                     (dtype == PSSA_HIP_F32 ? 4 : 2) * (a.ld_q | a.ld_k | a.ld_v | (size_t)a.dk | (size_t)a.dv);
  return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 0;
}

template <int MODE>
Status launch_chunks(hipStream_t stream, int dtype, const LinearArgs& a) {
  return with_chunks<MODE>(dtype, a.dk, a.dv, load_bytes(dtype, a), [&](auto c) -> Status {
    const dim3 grid((a.dv + c.kColumns - 1) / c.kColumns, a.heads, a.items);
    c.kKernel<<<grid, c.kThreads, c.kLds, stream>>>(a);
    PSSA_LAUNCH_CHECK("linear_chunks_kernel");
    return Status::Ok();
  });
}

template <int MODE>
Status chunks_attributes() {
  for (int dtype : {PSSA_HIP_F32, PSSA_HIP_BF16})
    for (int dk : {32, 64, 128})
      for (int dv : {64, 128})
        for (int load : {16, 4, 0})
          PSSA_RETURN_IF(with_chunks<MODE>(dtype, dk, dv, load, [&](auto c) -> Status {
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

// A walk is the way of a sequence, a head and 64 value columns through the
// tokens, in a workgroup of its own.  A call is split into the shortest
// segments that still run all at once: of one chunk if every segment then has
// a compute unit, else of two or more, two workgroups a compute unit with
// keys of up to 64 (LDS) and one with wider ones.  A split walk's chunk
// costs twice one of a whole walk, as its state is computed twice, and the
// passes between take about 12 us, 5 chunks of bf16 heads of 64 (figures that
// the rule was taken from; the first two lines' calls now take 49 and 44 us):
//                                               whole     split for 256, 512
//   8192 bf16 tokens, 8 heads of 128             366 us     54   61
//   9 fp32 prompts of 5..1000, 12 heads of 64     90        49   47
//   8 fp32 prompts of 1000, 12 heads of 64        92         -   73
//   16 bf16 prompts of 1500, 8 heads of 32        50         -   40
// (one chunk or two: a prompt of 700 fp32 tokens, 12 heads of 64 22 us and 27;
// 4 bf16 prompts of 2000, 4 heads of 64, for which 512 are needed, 27 and 22).
constexpr size_t kComputeUnits = 256;
int linear_segment(const uint64_t* lens, size_t n_seqs, size_t longest, size_t heads, size_t d_key, size_t d_val) {
  const size_t chunks = (longest + LA_C - 1) / LA_C, lanes = heads * ((d_val + 63) / 64);
  const size_t slots = (d_key <= 64 ? 2 : 1) * kComputeUnits;
  if (n_seqs * lanes > slots) return 0;
  auto fits = [&](size_t c, size_t slots) {
    size_t items = 0;
    for (size_t i = 0; i < n_seqs; ++i)
      items += lens ? std::max<size_t>(1, (lens[i] + c * LA_C - 1) / (c * LA_C)) : (longest + c * LA_C - 1) / (c * LA_C);
    return items * lanes <= slots;
  };
  size_t lo = 2, hi = std::max<size_t>(chunks, 2);  // the fewest chunks of a segment that fit; all of them do
  if (fits(1, kComputeUnits)) lo = hi = 1;
  while (lo < hi) {
    const size_t mid = (lo + hi) / 2;
    if (fits(mid, slots)) hi = mid; else lo = mid + 1;
  }
  return 2 * lo + 5 <= chunks ? (int)(lo * LA_C) : 0;
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
