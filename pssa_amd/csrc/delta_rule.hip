// The gated delta rule over packed sequences, from one token to long prompts:
//   S_t = a_t (1 - beta_t k_t k_t^T) S_{t-1} + beta_t k_t v_t^T,   o_t = scale q_t S_t,
// a_t = exp(log_decay_t).  With u_t = beta_t (v_t - a_t k_t S_{t-1}) that is
//   S_t = a_t S_{t-1} + k_t u_t^T,   o_t = scale (a_t q_t S_{t-1} + (q_t k_t) u_t).
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
template <class T>
__device__ __forceinline__ float load1(const T* p);
template <>
__device__ __forceinline__ float load1<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float load1<Bf16>(const Bf16* p) { return __uint_as_float((uint32_t)p->bits << 16); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(Bf16* p, float v) { p->bits = bf16_bits_dev(v); }

// The arguments' table is read from the kernel's argument segment, where the
// arguments lie first: indexing the struct itself would copy it to scratch.
typedef const __attribute__((address_space(4))) char* kernarg_t;
__device__ __forceinline__ uint32_t first_token(const DeltaArgs& a, int seq) {
  if (a.table) return a.table[seq];
  return reinterpret_cast<const __attribute__((address_space(4))) uint32_t*>(
      (kernarg_t)__builtin_amdgcn_kernarg_segment_ptr() + offsetof(DeltaArgs, inline_tokens))[seq];
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
// apart: 16 x 16.  k S and q S of a token meet in LDS together.
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
          S[i][e] *= decay;
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

}  // namespace

Status launch_delta_rule(hipStream_t stream, int dtype, const DeltaArgs& a, int longest) {
  return dtype == PSSA_HIP_F32 ? launch_steps<float>(stream, a) : launch_steps<Bf16>(stream, a);
}

}  // namespace pssa
