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
#include <algorithm>

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

// The span of a workgroup: its sequence, first token and length.
struct Span {
  int seq;
  size_t tok;
  int len;
};
__device__ __forceinline__ Span span_of(const LinearArgs& a, int seq) {
  if (a.uniform_len >= 0) return {seq, (size_t)seq * a.uniform_len, a.uniform_len};
  const uint32_t t0 = a.table ? a.table[seq] : a.inline_table[seq];
  const uint32_t t1 = a.table ? a.table[seq + 1] : a.inline_table[seq + 1];
  return {seq, t0, (int)(t1 - t0)};
}

// fp32 matrix products (v_mfma_f32_16x16x4_f32); bf16 inputs widened.
template <class T, int DKP, int NC>
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
  const size_t state0 = ((size_t)sp.seq * a.heads + head) * a.dk * a.dv;

  // S: rows 16 b + 4 quad + r, column dv0 + 16 NC wave + 16 c + col.
  f32x4_t S[NB][NC];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * b + 4 * quad + r, j = dv0 + 16 * NC * wave + 16 * c + col;
        S[b][c][r] = a.state_in && i < a.dk && j < a.dv ? a.state_in[state0 + (size_t)i * a.dv + j] : 0.0f;
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
    if (__syncthreads_or(odd) && n > 1) {
      singles = n;
      n = 1;
      fill();
      __syncthreads();
    }

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
  if (!a.state_out) return;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * b + 4 * quad + r, j = dv0 + 16 * NC * wave + 16 * c + col;
        if (i < a.dk && j < a.dv) a.state_out[state0 + (size_t)i * a.dv + j] = S[b][c][r];
      }
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

template <class T, int DKP, int NC>
Status launch_chunks_f32(hipStream_t stream, const LinearArgs& a) {
  const size_t lds = (size_t)(2 * LA_C * (DKP + 4) + LA_C * (64 * NC + 4) + LA_C * 68) * 4;
  linear_chunks_f32_kernel<T, DKP, NC><<<dim3((a.dv + 64 * NC - 1) / (64 * NC), a.heads, a.n_seqs), 256, lds, stream>>>(a);
  PSSA_LAUNCH_CHECK("linear_chunks_f32_kernel");
  return Status::Ok();
}
template <class T>
Status launch_chunks(hipStream_t stream, const LinearArgs& a) {
  const bool wide = a.dv > 64;
  if (a.dk <= 32) return wide ? launch_chunks_f32<T, 32, 2>(stream, a) : launch_chunks_f32<T, 32, 1>(stream, a);
  if (a.dk <= 64) return wide ? launch_chunks_f32<T, 64, 2>(stream, a) : launch_chunks_f32<T, 64, 1>(stream, a);
  return wide ? launch_chunks_f32<T, 128, 2>(stream, a) : launch_chunks_f32<T, 128, 1>(stream, a);
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

template <class T, int DKP, int NC>
Status chunks_attribute() {
  PSSA_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(&linear_chunks_f32_kernel<T, DKP, NC>),
                                   hipFuncAttributeMaxDynamicSharedMemorySize,
                                   (2 * LA_C * (DKP + 4) + LA_C * (64 * NC + 4) + LA_C * 68) * 4));
  return Status::Ok();
}

}  // namespace

Status init_linear_attributes() {
  PSSA_RETURN_IF((chunks_attribute<float, 32, 2>()));
  PSSA_RETURN_IF((chunks_attribute<float, 64, 1>()));
  PSSA_RETURN_IF((chunks_attribute<float, 64, 2>()));
  PSSA_RETURN_IF((chunks_attribute<float, 128, 1>()));
  PSSA_RETURN_IF((chunks_attribute<float, 128, 2>()));
  PSSA_RETURN_IF((chunks_attribute<Bf16, 32, 2>()));
  PSSA_RETURN_IF((chunks_attribute<Bf16, 64, 1>()));
  PSSA_RETURN_IF((chunks_attribute<Bf16, 64, 2>()));
  PSSA_RETURN_IF((chunks_attribute<Bf16, 128, 1>()));
  return chunks_attribute<Bf16, 128, 2>();
}

Status launch_linear_attention(hipStream_t stream, int dtype, const LinearArgs& a, int max_len) {
  const bool f32 = dtype == PSSA_HIP_F32;
  if (max_len <= kLinearSteps) return f32 ? launch_steps<float>(stream, a) : launch_steps<Bf16>(stream, a);
  return f32 ? launch_chunks<float>(stream, a) : launch_chunks<Bf16>(stream, a);
}

}  // namespace pssa
