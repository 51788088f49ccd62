// Beam search: the best continuations of a group's beams, and its states
// reordered by them.
//
//   value(b, v) = score[b] + logits[b][v] - log sum_u exp(logits[b][u]),
//
// the `keep` largest over a group's beams b and tokens v, equal ones by beam,
// then by token.  Within a beam the order is the logits' own, so a slice of a
// row gives its `keep` largest logits and its part of the sum, and a workgroup
// for each group joins the slices.  Values of different beams lie as near to
// each other as chance has it: the sums of exponentials, their logarithms and
// the values are in 64 bits (an fp32 logarithm would pick the wrong one of two
// candidates in some of 10^4 close calls).
#include <algorithm>

#include "operators.h"

namespace pssa {
namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef u32x4_t u32x4_any_t __attribute__((aligned(2)));

constexpr float kLog2e = 1.44269504088896341f;
constexpr uint32_t kNoToken = PSSA_HIP_NO_TOKEN;
constexpr int kThreads = 256;

struct Bf16 {
  uint16_t bits;
};
template <class T>
constexpr int vec_n() { return 16 / (int)sizeof(T); }

// Larger for larger values (-0 as 0), and never 0 for one above -inf; 0 stands for none.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) {
  return __uint_as_float(o ^ (~(uint32_t)((int32_t)o >> 31) | 0x80000000u));
}
constexpr uint32_t kOrderedLowest = 0x007FFFFFu;  // of -inf

// A logit and its token as one number: by value, then by lower id.
__device__ __forceinline__ uint64_t key_of(float v, uint32_t id) {
  const uint32_t o = ordered(v);
  return o > kOrderedLowest ? (uint64_t)o << 32 | (uint32_t)~id : 0;
}

// What a slice of a row leaves for the join.
struct SliceSum {
  double sum;    // of exp(logit - most)
  float most;
  uint32_t bad;  // a logit is NaN or +inf
};

__device__ __forceinline__ bool beam_ended(const BeamArgs& a, int row) {
  return a.last && a.eos != kNoToken && a.last[row] == a.eos;
}
__device__ __forceinline__ bool beam_runs(const BeamArgs& a, int row) {
  return !beam_ended(a, row) && fabsf(a.scores[row]) < INFINITY;
}

// A piece of a row: 16 bytes, or the `left` elements that there are, then -inf.
template <class T>
__device__ __forceinline__ u32x4_t load_piece(const T* row, int c, int left) {
  constexpr int N = vec_n<T>();
  if (left >= N) return *reinterpret_cast<const u32x4_any_t*>(row + c);
  u32x4_t u;
#pragma unroll
  for (int e = 0; e < 4; ++e) u[e] = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (j >= left) continue;
    if constexpr (sizeof(T) == 4)
      u[j] = __float_as_uint(row[c + j]);
    else
      u[j >> 1] = j & 1 ? (u[j >> 1] & 0xFFFFu) | (uint32_t)row[c + j].bits << 16 : (u[j >> 1] & 0xFFFF0000u) | row[c + j].bits;
  }
  return u;
}
template <class T>
__device__ __forceinline__ float elem(const u32x4_t& u, int j) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(u[j]);
  return __uint_as_float(j & 1 ? u[j >> 1] & 0xFFFF0000u : u[j >> 1] << 16);
}

// Of the 64 values of a wave's lanes the keep-th largest, in every lane.
__device__ __forceinline__ float keepth_largest(float v, int keep) {
  int above = 0;
#pragma unroll
  for (int i = 0; i < 64; ++i) above += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), i)) > v;
  // The least of those that fewer than keep lie above.
  float least = above < keep ? v : INFINITY;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) least = fminf(least, __shfl_xor(least, off, 64));
  return least;
}

// Places of the candidates that a workgroup puts aside; past them (rows of
// equal logits) it goes through its candidates in rounds.
constexpr int kAside = 1024;

// A slice of a row in the registers of a workgroup, NV pieces of 16 bytes a
// thread.  The largest logits of 64 groups of threads: the keep-th of these is
// a bound that keep logits reach, and few others do.  What reaches it is put
// aside and ordered (64 x 8 rows of 100003 bf16: 35 us, 3 TB/s, the VALU 0.42 busy:
// an exponential, a maximum and two widenings an element).
template <class T, int NV>
__global__ __launch_bounds__(kThreads) void beam_slice_kernel(BeamArgs a) {
  constexpr int N = vec_n<T>();
  __shared__ uint64_t s_list[kAside], s_best[4];
  __shared__ float s_group[4][64], s_bound;
  __shared__ double s_sum[4];
  __shared__ uint32_t s_count;
  const int row = blockIdx.x, slice = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (!beam_runs(a, row)) return;
  const T* logits = static_cast<const T*>(a.logits) + (size_t)row * a.ld;
  const int first = slice * kThreads * NV * N;

  u32x4_t raw[NV];
  float piece[NV], mine = -INFINITY;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = first + (tid + k * kThreads) * N;
    raw[k] = load_piece<T>(logits, c, a.vocab - c);
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    piece[k] = elem<T>(raw[k], 0);
#pragma unroll
    for (int j = 1; j < N; ++j) piece[k] = fmaxf(piece[k], elem<T>(raw[k], j));
    mine = fmaxf(mine, piece[k]);  // passes over a NaN
  }
  s_group[wave][lane] = mine;
  if (tid == 0) s_count = 0;
  __syncthreads();
  const float group = fmaxf(fmaxf(s_group[0][lane], s_group[1][lane]), fmaxf(s_group[2][lane], s_group[3][lane]));
  float most = group;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) most = fmaxf(most, __shfl_xor(most, off, 64));
  if (wave == ((row + slice) & 3)) {  // one wave, another SIMD's in neighbouring workgroups
    const float b = keepth_largest(group, a.keep);
    if (lane == 0) s_bound = b;
  }
  // A NaN makes the sum NaN; a slice of nothing else and -inf has no sum.
  const float base = most > -INFINITY ? most : 0.0f;
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    asm volatile("" : "+v"(raw[k]));  // widened again: kept, the elements would take twice the registers
    float part = 0.0f;                // few terms in fp32, these sums in 64 bits
#pragma unroll
    for (int j = 0; j < N; ++j) part += __builtin_amdgcn_exp2f((elem<T>(raw[k], j) - base) * kLog2e);
    sum += part;
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if (lane == 0) s_sum[wave] = sum;
  __syncthreads();

  // The few pieces that reach the bound are read again, so that the others
  // need no registers.
  const float bound = s_bound;
  uint32_t reach = 0;
#pragma unroll
  for (int k = 0; k < NV; ++k) reach |= (piece[k] >= bound ? 1u : 0u) << k;
  auto keys = [&](auto use) {
    for (uint32_t left = reach; left; left &= left - 1) {
      const int c = first + (tid + __builtin_ctz(left) * kThreads) * N;
      const u32x4_t u = load_piece<T>(logits, c, a.vocab - c);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float v = elem<T>(u, j);
        const uint64_t key = key_of(v, c + j);
        if (key && v >= bound) use(key);
      }
    }
  };
  keys([&](uint64_t key) {
    const uint32_t at = atomicAdd(&s_count, 1u);
    if (at < kAside) s_list[at] = key;
  });
  __syncthreads();

  const int count = (int)s_count;
  const size_t at = (size_t)row * a.slices + slice;
  uint64_t* out = a.keys + at * a.keep;
  if (count <= kAside) {
    for (int i = tid; i < count; i += kThreads) {
      const uint64_t key = s_list[i];
      int place = 0;
      for (int j = 0; j < count; ++j) place += s_list[j] > key;
      if (place < a.keep) out[place] = key;
    }
    for (int i = count + tid; i < a.keep; i += kThreads) out[i] = 0;
  } else {
    uint64_t last = ~(uint64_t)0;
    for (int i = 0; i < a.keep; ++i) {
      uint64_t best = 0;
      keys([&](uint64_t key) { best = key < last && key > best ? key : best; });
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) {
        const uint64_t o = __shfl_xor((unsigned long long)best, off, 64);
        best = o > best ? o : best;
      }
      if (lane == 0) s_best[wave] = best;
      __syncthreads();
      best = s_best[0];
#pragma unroll
      for (int w = 1; w < 4; ++w) best = s_best[w] > best ? s_best[w] : best;
      __syncthreads();
      if (tid == 0) out[i] = best;
      last = best;
    }
  }
  if (tid == 0) {
    SliceSum s;
    s.sum = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
    s.most = most;
    s.bad = !(most < INFINITY) || s.sum != s.sum;
    static_cast<SliceSum*>(a.sums)[at] = s;
  }
}

// A candidate: its value, and the beam and token that break ties.
struct Candidate {
  double value;
  uint64_t at;  // beam << 32 | token
};
__device__ __forceinline__ bool better(const Candidate& x, const Candidate& y) {
  return x.value > y.value || (x.value == y.value && x.at < y.at);
}
__device__ __forceinline__ Candidate nothing() { return Candidate{-INFINITY, ~(uint64_t)0}; }

// The join of a group's slices, with the same bound.  A slice's candidates lie
// best first.  `each` threads take every each-th one of a slice, so that the
// bound needs to look at the first `each` of a slice alone, and what does not
// reach it ends a walk.  More threads where more are kept, as one beam's few
// slices may hold all of these (a thread a slice: 64 x 8 x 100003, 8 kept, 12.8
// us, four 7.4), or where slices are few; candidates dealt out in their order met
// whole groups of threads without a slice's best (16 beams of 72320, 32 kept, the
// whole call 473 us, so 55).
__global__ __launch_bounds__(kThreads) void beam_join_kernel(BeamArgs a) {
  // The scores and which beams have ended, as the outputs may be written over them.
  __shared__ double s_lse[kMaxBeams], s_score[kMaxBeams];
  __shared__ float s_group[4][64];
  __shared__ bool s_ended[kMaxBeams];
  __shared__ Candidate s_list[kAside], s_part[4];
  __shared__ uint32_t s_count;
  const int group = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row0 = group * a.beams;
  const SliceSum* sums = static_cast<const SliceSum*>(a.sums);
  if (tid == 0) s_count = 0;
  // Each running beam's log of the sum; +inf (no candidate) where it has none.
  // A beam's slices take as many lanes as let all beams be joined at once.
  const int lanes = a.beams <= 4 ? 64 : a.beams <= 16 ? 16 : 4, b = tid / lanes;
  if (b < a.beams) {
    const SliceSum* s = sums + (size_t)(row0 + b) * a.slices;
    const int in = tid & (lanes - 1), slices = beam_runs(a, row0 + b) ? a.slices : 0;
    float most = -INFINITY;
    bool bad = false;
    for (int i = in; i < slices; i += lanes) most = fmaxf(most, s[i].most), bad |= s[i].bad != 0;
    for (int off = lanes >> 1; off >= 1; off >>= 1) {
      most = fmaxf(most, __shfl_xor(most, off, 64));
      bad |= (bool)__shfl_xor((int)bad, off, 64);
    }
    double sum = 0.0;
    for (int i = in; i < slices; i += lanes)
      if (s[i].most > -INFINITY) sum += s[i].sum * exp((double)s[i].most - (double)most);
    for (int off = lanes >> 1; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if (in == 0) {
      s_lse[b] = !bad && most > -INFINITY ? log(sum) + (double)most : INFINITY;
      s_score[b] = a.scores[row0 + b];
      s_ended[b] = beam_ended(a, row0 + b);
    }
  }
  __syncthreads();

  const int lists = a.beams * a.slices;
  int each = a.keep > 16 ? 8 : a.keep > 2 ? 4 : 1;
  while (2 * each * lists <= 64) each *= 2;
  const int sub = tid & (each - 1), list0 = tid / each, step = kThreads / each;
  auto candidate = [&](int list, int r) -> Candidate {
    const int b = list / a.slices;
    const double score = s_score[b];
    if (s_ended[b])  // it stays as it is
      return list == b * a.slices && r == 0 && fabs(score) < INFINITY ? Candidate{score, (uint64_t)b << 32 | a.eos} : nothing();
    if (!(s_lse[b] < INFINITY)) return nothing();
    const uint64_t key = a.keys[((size_t)row0 * a.slices + list) * a.keep + r];
    if (!key) return nothing();
    return Candidate{score + ((double)unordered((uint32_t)(key >> 32)) - s_lse[b]),
                     (uint64_t)b << 32 | ((uint32_t)~key + a.first_id)};
  };
  Candidate mine = nothing();
  if (sub < a.keep)
    for (int list = list0; list < lists; list += step) {
      const Candidate c = candidate(list, sub);
      if (better(c, mine)) mine = c;
    }
  s_group[wave][lane] = (float)mine.value;  // rounding keeps the order
  __syncthreads();
  const float bound = keepth_largest(fmaxf(fmaxf(s_group[0][lane], s_group[1][lane]), fmaxf(s_group[2][lane], s_group[3][lane])), a.keep);
  for (int list = list0; list < lists; list += step)
    for (int r = sub; r < a.keep; r += each) {
      const Candidate c = candidate(list, r);
      if (!(c.value > -INFINITY && (float)c.value >= bound)) break;
      const uint32_t at = atomicAdd(&s_count, 1u);
      if (at < kAside) s_list[at] = c;
    }
  __syncthreads();
  const int count = (int)s_count;
  auto put = [&](int place, const Candidate& c) {
    const size_t o = (size_t)group * a.keep + place;
    const bool some = c.value > -INFINITY;
    a.parents[o] = some ? (uint32_t)(c.at >> 32) : kNoToken;
    a.tokens[o] = some ? (uint32_t)c.at : kNoToken;
    a.out_scores[o] = some ? (float)c.value : -INFINITY;
  };
  if (count <= kAside) {
    for (int i = tid; i < count; i += kThreads) {
      const Candidate c = s_list[i];
      int place = 0;
      for (int j = 0; j < count; ++j) place += better(s_list[j], c);
      if (place < a.keep) put(place, c);
    }
    for (int i = count + tid; i < a.keep; i += kThreads) put(i, nothing());
    return;
  }
  // Rounds that each pick the best candidate left, of which only the winner's
  // thread looks for its next one: over all of its own, as values that a large
  // score has rounded to one lie in the logits' order.
  auto next = [&](auto left) {
    Candidate best = nothing();
    for (int list = list0; list < lists; list += step)
      for (int r = sub; r < a.keep; r += each) {
        const Candidate c = candidate(list, r);
        if (left(c) && better(c, best)) best = c;
      }
    return best;
  };
  mine = next([](const Candidate&) { return true; });
  for (int j = 0; j < a.keep; ++j) {
    Candidate w = mine;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
      const Candidate o{__shfl_xor(w.value, off, 64), (uint64_t)__shfl_xor((unsigned long long)w.at, off, 64)};
      if (better(o, w)) w = o;
    }
    if (lane == 0) s_part[wave] = w;
    __syncthreads();
    w = s_part[0];
#pragma unroll
    for (int i = 1; i < 4; ++i)
      if (better(s_part[i], w)) w = s_part[i];
    __syncthreads();
    if (tid == 0) put(j, w);
    if (w.value > -INFINITY && mine.at == w.at) mine = next([&](const Candidate& c) { return better(w, c); });
  }
}

// ------------------------------------------------------------------ states
// Rows of a group copied from their parents'.  A thread moves one piece of
// every row, MOST rows at a time.  Where MOST covers a group, all are loaded
// before the first is stored, and rows may be reordered where they are (64 x 8
// rows of 196 KB: 31 us, 135 MB read and written, 4.4 TB/s).
template <class V, int MOST>
__global__ __launch_bounds__(kThreads) void beam_gather_kernel(GatherArgs a) {
  typedef V any_t __attribute__((aligned(1)));
  const size_t c = ((size_t)blockIdx.x * kThreads + threadIdx.x) * sizeof(V);
  if (c >= a.row_bytes) return;
  for (int group = blockIdx.y; group < a.groups; group += gridDim.y) {
    const uint32_t* parents = a.parents + (size_t)group * a.n_out;
    const char* src = static_cast<const char*>(a.src) + (size_t)group * a.n_in * a.ld_src + c;
    char* dst = static_cast<char*>(a.dst) + (size_t)group * a.n_out * a.ld_dst + c;
    for (int j0 = 0; j0 < a.n_out; j0 += MOST) {
      V v[MOST];
#pragma unroll
      for (int j = 0; j < MOST; ++j)
        if (j0 + j < a.n_out && parents[j0 + j] < (uint32_t)a.n_in)
          v[j] = *reinterpret_cast<const any_t*>(src + parents[j0 + j] * a.ld_src);
#pragma unroll
      for (int j = 0; j < MOST; ++j)
        if (j0 + j < a.n_out && parents[j0 + j] < (uint32_t)a.n_in && !(a.src == a.dst && parents[j0 + j] == (uint32_t)(j0 + j)))
          *reinterpret_cast<any_t*>(dst + (j0 + j) * a.ld_dst) = v[j];
    }
  }
}

// The first row of every group copied to all of the group's, where the first
// rows are packed at the front: group g's rows begin behind row g, so the last
// group goes first.
__global__ __launch_bounds__(kThreads) void beam_spread_kernel(uint32_t* rows, size_t words, size_t ld, int groups, int beams) {
  const size_t c = (size_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= words) return;
  for (int g = groups - 1; g >= 0; --g) {
    const uint32_t v = rows[g * ld + c];
    for (int b = 0; b < beams; ++b) rows[((size_t)g * beams + b) * ld + c] = v;
  }
}

// The chosen tokens as the next step's inputs; where there is none, any.
__global__ __launch_bounds__(kThreads) void beam_feed_kernel(const uint32_t* tokens, uint32_t* ids, size_t n) {
  const size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x;
  if (i < n) ids[i] = tokens[i] == kNoToken ? 0 : tokens[i];
}

template <class V, int MOST>
Status launch_pieces(hipStream_t stream, const GatherArgs& a) {
  const size_t pieces = a.row_bytes / sizeof(V);
  const dim3 grid((uint32_t)((pieces + kThreads - 1) / kThreads), (uint32_t)std::min(a.groups, 65535));
  beam_gather_kernel<V, MOST><<<grid, kThreads, 0, stream>>>(a);
  PSSA_LAUNCH_CHECK("beam_gather_kernel");
  return Status::Ok();
}

template <class T>
Status launch_slices(hipStream_t stream, const BeamArgs& a, size_t rows, int pieces) {
  const dim3 grid((uint32_t)rows, a.slices);
  if (pieces == 1)
    beam_slice_kernel<T, 1><<<grid, kThreads, 0, stream>>>(a);
  else if (pieces == 2)
    beam_slice_kernel<T, 2><<<grid, kThreads, 0, stream>>>(a);
  else if (pieces == 4)
    beam_slice_kernel<T, 4><<<grid, kThreads, 0, stream>>>(a);
  else
    beam_slice_kernel<T, 8><<<grid, kThreads, 0, stream>>>(a);
  PSSA_LAUNCH_CHECK("beam_slice_kernel");
  return Status::Ok();
}

}  // namespace

BeamPlan beam_plan(int dtype, size_t rows, size_t vocab, size_t keep) {
  BeamPlan p;
  const size_t per = kThreads * (dtype == PSSA_HIP_F32 ? 4 : 8);
  for (p.pieces = 1; p.pieces < 8 && rows * ((vocab + per * p.pieces - 1) / (per * p.pieces)) > 2048; p.pieces *= 2) {}
  p.slices = (vocab + per * p.pieces - 1) / (per * p.pieces);
  p.sums_bytes = (rows * p.slices * sizeof(SliceSum) + 255) & ~(size_t)255;
  p.bytes = p.sums_bytes + rows * p.slices * keep * 8;
  return p;
}

Status launch_beam_select(hipStream_t stream, int dtype, const BeamArgs& a, size_t groups, const BeamPlan& p) {
  const size_t rows = groups * (size_t)a.beams;
  PSSA_RETURN_IF(dtype == PSSA_HIP_F32 ? launch_slices<float>(stream, a, rows, p.pieces)
                                       : launch_slices<Bf16>(stream, a, rows, p.pieces));
  beam_join_kernel<<<(uint32_t)groups, kThreads, 0, stream>>>(a);
  PSSA_LAUNCH_CHECK("beam_join_kernel");
  return Status::Ok();
}

// 16 bytes a thread and row up to 16 rows (64 registers), more rows in parts
// of 16, but for those that are reordered in place: 4 bytes of up to 64 rows.
size_t beam_gather_piece(const GatherArgs& a) {
  if (a.row_bytes % 16 == 0 && (a.n_out <= 16 || a.src != a.dst)) return 16;
  return a.row_bytes % 4 == 0 ? 4 : 1;
}
Status launch_beam_gather(hipStream_t stream, const GatherArgs& a) {
  const size_t piece = beam_gather_piece(a);
  if (piece == 16) {
    if (a.n_out <= 4) return launch_pieces<u32x4_t, 4>(stream, a);
    if (a.n_out <= 8) return launch_pieces<u32x4_t, 8>(stream, a);
    return launch_pieces<u32x4_t, 16>(stream, a);
  }
  if (piece == 4) return launch_pieces<uint32_t, kMaxBeams>(stream, a);
  return launch_pieces<uint8_t, kMaxBeams>(stream, a);
}

Status launch_beam_feed(hipStream_t stream, const uint32_t* tokens, uint32_t* ids, size_t n) {
  beam_feed_kernel<<<(uint32_t)((n + kThreads - 1) / kThreads), kThreads, 0, stream>>>(tokens, ids, n);
  PSSA_LAUNCH_CHECK("beam_feed_kernel");
  return Status::Ok();
}

Status launch_beam_spread(hipStream_t stream, void* rows, size_t words, size_t ld, size_t groups, size_t beams) {
  beam_spread_kernel<<<(uint32_t)((words + kThreads - 1) / kThreads), kThreads, 0, stream>>>(
      static_cast<uint32_t*>(rows), words, ld, (int)groups, (int)beams);
  PSSA_LAUNCH_CHECK("beam_spread_kernel");
  return Status::Ok();
}

}  // namespace pssa
