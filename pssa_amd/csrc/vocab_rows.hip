// Operators over logit rows: log probabilities of given tokens with entropy
// and top alternatives, and distillation from a teacher's top logits.
//
// Both pass a row through the registers of one workgroup, tile by tile.  Log
// probabilities take one pass: a maximum that rises rescales each thread's
// sums, and tokens that may be among the largest are put aside in LDS.
// Distillation writes its gradient from the registers that the sums were taken
// from, or reads a row past them twice.
#include <algorithm>

#include "operators.h"

namespace pssa {
namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
// 16 bytes at any element's address: rows start anywhere (gfx950 loads and
// stores them unaligned in one instruction).
typedef u32x4_t u32x4_any_t __attribute__((aligned(2)));

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLowest = -3.0e38f;  // stands for differences that overflow: exp of it is 0, products with 0 stay 0
constexpr uint32_t kNoToken = PSSA_HIP_NO_TOKEN;
constexpr size_t kComputeUnits = 256;

struct Bf16 {
  uint16_t bits;
};
template <class T>
constexpr int vec_n() { return 16 / (int)sizeof(T); }

template <class T>
__device__ __forceinline__ float elem(const u32x4_t& u, int j);
template <>
__device__ __forceinline__ float elem<float>(const u32x4_t& u, int j) { return __uint_as_float(u[j]); }
template <>
__device__ __forceinline__ float elem<Bf16>(const u32x4_t& u, int j) {
  return __uint_as_float(j & 1 ? u[j >> 1] & 0xFFFF0000u : u[j >> 1] << 16);
}
template <class T>
__device__ __forceinline__ float load1(const T* p);
template <>
__device__ __forceinline__ float load1<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float load1<Bf16>(const Bf16* p) { return __uint_as_float((uint32_t)p->bits << 16); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(Bf16* p, float v) { p->bits = bf16_bits_dev(v); }
template <class T>
__device__ __forceinline__ u32x4_t pack(const float (&v)[vec_n<T>()]);
template <>
__device__ __forceinline__ u32x4_t pack<float>(const float (&v)[4]) {
  return u32x4_t{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}
template <>
__device__ __forceinline__ u32x4_t pack<Bf16>(const float (&v)[8]) {
  return u32x4_t{bf16x2_bits(v[0], v[1]), bf16x2_bits(v[2], v[3]), bf16x2_bits(v[4], v[5]), bf16x2_bits(v[6], v[7])};
}
// -inf in one element (the other half of its word kept).
template <class T>
__device__ __forceinline__ void mask_elem(u32x4_t& u, int j);
template <>
__device__ __forceinline__ void mask_elem<float>(u32x4_t& u, int j) { u[j] = 0xFF800000u; }
template <>
__device__ __forceinline__ void mask_elem<Bf16>(u32x4_t& u, int j) {
  u[j >> 1] = j & 1 ? (u[j >> 1] & 0xFFFFu) | 0xFF800000u : (u[j >> 1] & 0xFFFF0000u) | 0xFF80u;
}

// Vector i of a row covers elements i*N .. i*N+N-1 and is loaded from
// vec_start, which moves the row's last, partial vector back to end with the
// row: every load stays inside the row, and the elements that belong to the
// vector before (all of them past the row's end) read as -inf.
template <class T>
__device__ __forceinline__ int vec_start(int V, int i) {
  constexpr int N = vec_n<T>();
  return V < N ? 0 : min(i * N, V - N);
}
template <class T>
__device__ __forceinline__ u32x4_t vec_load(const T* row, int V, int i) {
  constexpr int N = vec_n<T>();
  if (V < N) {  // uniform
    u32x4_t u = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (i == 0 && j < V) {
        if constexpr (sizeof(T) == 4)
          u[j] = reinterpret_cast<const uint32_t*>(row)[j];
        else
          u[j >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[j] << (16 * (j & 1));
      } else {
        mask_elem<T>(u, j);
      }
    }
    return u;
  }
  return *reinterpret_cast<const u32x4_any_t*>(row + vec_start<T>(V, i));
}
template <class T>
__device__ __forceinline__ void vec_mask(u32x4_t& u, int V, int i) {
  constexpr int N = vec_n<T>();
  const int lead = i * N - vec_start<T>(V, i);
  if (V >= N && lead > 0) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < lead) mask_elem<T>(u, j);
  }
}
// The tile's vectors of one thread (vector tile0 + k * 64W + tid); a k past
// the row is skipped, and one that lies inside it loaded plainly, by the
// whole workgroup.
template <class T, int W, int NV>
__device__ __forceinline__ void tile_load(u32x4_t (&u)[NV], const T* row, int V, int tile0) {
  constexpr int N = vec_n<T>();
  const uint32_t none = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;
  const T* mine = row + (size_t)(tile0 + (int)threadIdx.x) * N;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    u[k] = u32x4_t{none, none, none, none};
    if ((tile0 + (k + 1) * 64 * W) * N <= V)
      u[k] = *reinterpret_cast<const u32x4_any_t*>(mine + k * 64 * W * N);
    else if ((tile0 + k * 64 * W) * N < V)
      u[k] = vec_load<T>(row, V, tile0 + k * 64 * W + (int)threadIdx.x);
  }
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if ((tile0 + (k + 1) * 64 * W) * N > V && (tile0 + k * 64 * W) * N < V)
      vec_mask<T>(u[k], V, tile0 + k * 64 * W + (int)threadIdx.x);
}
// Between two uses of a tile: what one computed of it (bf16 values widened,
// twice the registers) is not kept for the next.
template <int NV>
__device__ __forceinline__ void tile_again(u32x4_t (&u)[NV]) {
#pragma unroll
  for (int k = 0; k < NV; ++k) asm volatile("" : "+v"(u[k]));
}
// The largest of three; a NaN is passed over.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
template <class T, int NV>
__device__ __forceinline__ float tile_max(const u32x4_t (&u)[NV]) {
  constexpr int N = vec_n<T>();
  float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      m0 = max3(m0, elem<T>(u[k], j), elem<T>(u[k], j + 1));
      m1 = max3(m1, elem<T>(u[k], j + 2), elem<T>(u[k], j + 3));
    }
  return fmaxf(m0, m1);
}

// The value of the lane whose number differs in one bit, in registers (`off`
// constant; every lane active): a step of 8 to 16 cycles, where a shuffle
// through LDS takes a hundred.
__device__ __forceinline__ uint32_t lane_xor(uint32_t v, int off) {
  switch (off) {
    case 1: return __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, true);  // quads 1 0 3 2
    case 2: return __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, true);  // quads 2 3 0 1
    case 4:  // eights mirrored, then quads
      return __builtin_amdgcn_mov_dpp(__builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, true), 0x1B, 0xF, 0xF, true);
    case 8: return __builtin_amdgcn_mov_dpp(v, 0x128, 0xF, 0xF, true);  // sixteens rotated by 8
    case 16: {
      const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
      return threadIdx.x & 16 ? r[0] : r[1];
    }
    default: {
      const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
      return threadIdx.x & 32 ? r[0] : r[1];
    }
  }
}
__device__ __forceinline__ float lane_xor(float v, int off) { return __uint_as_float(lane_xor(__float_as_uint(v), off)); }
__device__ __forceinline__ uint64_t lane_xor(uint64_t v, int off) {
  return (uint64_t)lane_xor((uint32_t)(v >> 32), off) << 32 | lane_xor((uint32_t)v, off);
}
// The value of lane 63 - lane: sixteens mirrored, then exchanged.
__device__ __forceinline__ uint64_t lane_reverse(uint64_t v) {
  const uint32_t lo = __builtin_amdgcn_mov_dpp((uint32_t)v, 0x140, 0xF, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_mov_dpp((uint32_t)(v >> 32), 0x140, 0xF, 0xF, true);
  return lane_xor(lane_xor((uint64_t)hi << 32 | lo, 16), 32);
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += lane_xor(v, o);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {  // NaN never becomes the maximum
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, lane_xor(v, o));
  return v;
}

// ------------------------------------------------------------- ordered keys
// A token's place in (logit descending, id ascending) order as one whole
// number: the logit's bits mapped to unsigned order above the complement of
// the id.  Distinct for every token; 0 is no token.
__device__ __forceinline__ uint64_t token_key(float v, int id) {
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 orders as 0
  return (uint64_t)(b ^ (b >> 31 ? 0xFFFFFFFFu : 0x80000000u)) << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __uint_as_float(b ^ (b >> 31 ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ int key_id(uint64_t k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ uint64_t key_step(uint64_t a, int off, bool keep_max) {
  const uint64_t o = lane_xor(a, off);
  return (o > a) == keep_max ? o : a;
}
__device__ __forceinline__ uint32_t value_key(float v) { return (uint32_t)(token_key(v, 0) >> 32); }
__device__ __forceinline__ uint32_t key_step(uint32_t a, int off, bool keep_max) {
  const uint32_t o = lane_xor(a, off);
  return keep_max ? max(o, a) : min(o, a);
}
// The wave's 64 keys, largest in lane 0 (bitonic, 21 exchanges).
template <class Key>
__device__ __forceinline__ Key wave_sort(Key a, int lane) {
#pragma unroll
  for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
    for (int off = size >> 1; off >= 1; off >>= 1) a = key_step(a, off, ((lane & off) == 0) == ((lane & size) == 0));
  return a;
}
// The largest 64 of two descending lists, descending; `b` is given reversed.
template <class Key>
__device__ __forceinline__ Key wave_merge(Key a, Key b_reversed, int lane) {
  a = a > b_reversed ? a : b_reversed;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) a = key_step(a, off, (lane & off) == 0);
  return a;
}

// --------------------------------------------------------- log probabilities
// With m the row's maximum and d_i = (z_i - m) / tau, the log softmax is
// d_i - log(1 + S) and the entropy log(1 + S) - T / (1 + S), where S and T sum
// exp(d_i) and exp(d_i) d_i over every token but the first maximum: kept
// apart from its 1, S carries the small probabilities that a nearly certain
// row's values consist of.
//
// Alternatives: the k-th largest of the maxima of some groups of threads (64
// groups, or every thread for itself where k is large) bounds the first
// tile's k-th largest token from below, and with it the row's.  The tokens
// that pass the bound, hardly more than k of a tile, gather in LDS until one
// wave sorts them by value and id, at the end or where they are many, which
// raises the bound.  A tile where they are too many for that (all logits
// equal, say) gives its k tokens one by one, each round the largest behind
// the one before.
//
// 8192 fp32 rows of 16384, 8 alternatives: 109 us (4.9 TB/s); 509 bf16 rows of
// 100003, 5 of them: 34 us (3.0 TB/s); one row of 16384: 7.5 us, mostly latency.
// Tiles that leave fewer tokens than are asked for, with no bound from before,
// go through LDS whole: 257 and 113 us where the first two keep 4 and 20
// tokens a row (8 alternatives).
constexpr int kCandidates = 1024;
constexpr int kSlots = 8;  // threads of a wave whose vectors are looked through at once

// MANY: the row takes several tiles, each loaded while the one before is summed.
template <class T, int W, int NV, bool MANY>
__global__ __launch_bounds__(64 * W) void token_logprobs_kernel(LogprobArgs a) {
  constexpr int N = vec_n<T>(), TILE = 64 * W * NV;
  __shared__ uint32_t s_keys[W * 64];
  __shared__ uint64_t s_round[W];
  __shared__ float s_max[2][W], s_sum[2 * W];
  __shared__ int s_owner[2], s_count;
  __shared__ u32x4_t s_hit[W][kSlots][NV];
  __shared__ int s_hit_lane[W][kSlots];
  __shared__ uint32_t s_kth;
  extern __shared__ uint64_t s_cand[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = a.vocab, top = a.top_k;
  const T* row = static_cast<const T*>(a.logits) + (size_t)blockIdx.x * a.ld;
  const float inv_tau = 1.0f / a.temperature, c2 = kLog2e * inv_tau;
  const uint32_t target = a.targets ? a.targets[blockIdx.x] : kNoToken;
  const float z_target = target < (uint32_t)V ? load1<T>(row + target) : 0.0f;
  if (tid == 0) {
    s_count = 0;
    s_owner[0] = s_owner[1] = 64 * W;
    s_kth = 0;
  }

  float m = -INFINITY, S = 0.0f, Tq = 0.0f;  // the maximum so far; this thread's sums
  uint64_t best = 0;                         // wave 0: the largest keys so far, descending
  const int vecs = (V + N - 1) / N;
  // What s_cand has gathered, n of them, into `best`; where the tile that
  // began behind the first n_before had too many, its tokens from the row.
  auto settle = [&](int n, int n_before, int tile0) {
    uint64_t list = 0;
    const bool many = n > kCandidates;
    if (many) {
      uint64_t last = ~(uint64_t)0;
      for (int i = 0; i < top; ++i) {
        uint64_t mine = 0;
        for (int e = tile0 * N + tid; e < min(V, (tile0 + TILE) * N); e += 64 * W) {  // from the cache: rare
          const float v = load1<T>(row + e);
          const uint64_t key = v > -INFINITY ? token_key(v, e) : 0;
          if (key < last && key > mine) mine = key;
        }
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) mine = key_step(mine, off, true);
        if (lane == 0) s_round[wave] = mine;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) mine = s_round[w] > mine ? s_round[w] : mine;
        __syncthreads();
        last = mine;
        if (lane == i) list = mine;
        if (!mine) break;  // uniform
      }
      n = n_before;
    }
    if (wave == 0) {
      if (many) best = wave_merge(best, lane_reverse(list), lane);
#pragma unroll 1
      for (int c = 0; c < n; c += 64) {
        const uint64_t got = wave_sort(c + lane < n ? s_cand[c + lane] : (uint64_t)0, lane);
        if (!MANY && c == 0 && !many)
          best = got;
        else
          best = wave_merge(best, lane_reverse(got), lane);
      }
      if (lane == top - 1) s_kth = (uint32_t)(best >> 32);
      if (lane == 0) s_count = 0;
    }
    __syncthreads();
  };
  int gathered = 0;  // before the tile
  u32x4_t u[NV], ahead[MANY ? NV : 1];
  tile_load<T, W, NV>(u, row, V, 0);
  for (int tile0 = 0, p = 0; tile0 < vecs; tile0 += TILE, p ^= 1) {
    tile_again(u);  // its loads end here
    if constexpr (MANY) {
      if (tile0 + TILE < vecs) tile_load<T, W, NV>(ahead, row, V, tile0 + TILE);
    }
    const float bv = tile_max<T, NV>(u);
    tile_again(u);
    float mt = wave_max(bv);
    if (lane == 0) s_max[p][wave] = mt;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) mt = fmaxf(mt, s_max[p][w]);
    if (tid == 0) s_owner[p ^ 1] = 64 * W;
    const bool rises = mt > m;
    if (rises && bv == mt) atomicMin(&s_owner[p], tid);  // this thread's first maximum is left out of the sums
    const int n = s_count;
    uint32_t kth = s_kth;
    if (top || rises) __syncthreads();  // uniform
    if (top) {
      if (MANY && n > kCandidates / 2) {
        settle(n, gathered, tile0 - TILE);
        kth = s_kth;
        gathered = 0;
        __syncthreads();
      } else {
        gathered = n;
      }
      const bool ties = kth <= value_key(-INFINITY);  // no bound yet; what equals the tile's own may be among the largest
      if (ties) {
        const bool fine = top > 24;  // every thread a group
        float gm = bv;
        if (!fine) {
#pragma unroll
          for (int off = 1; off < W; off <<= 1) gm = fmaxf(gm, lane_xor(gm, off));
        }
        uint32_t key = value_key(gm);
        if constexpr (W > 1) {
          if (fine) {
            key = wave_sort(key, lane);
            s_keys[tid] = key;
          } else if (lane % W == 0) {
            s_keys[tid / W] = key;
          }
          __syncthreads();
          if (fine) {
#pragma unroll
            for (int half = W / 2; half >= 1; half >>= 1) {
              if (wave < half) {
                key = wave_merge(key, s_keys[(wave + half) * 64 + 63 - lane], lane);
                s_keys[tid] = key;
              }
              __syncthreads();
            }
          }
        }
        if (wave == 0) {
          if (W == 1 || !fine) key = wave_sort(W == 1 ? key : s_keys[lane], lane);
          if (lane == top - 1) s_kth = key;
        }
        __syncthreads();
        kth = s_kth;
      }
      const float bound = key_value((uint64_t)kth << 32);
      // Threads with such a token hand their vectors over to their wave, a
      // token for each lane: looked for by the threads themselves, one of 32
      // here and there would keep the wave as long as the sums do.
      bool hit = ties ? bv >= bound : bv > bound;
      for (uint64_t hits = __ballot(hit); hits;) {  // uniform in the wave
        const int rank = __popcll(hits & (((uint64_t)1 << lane) - 1));
        const bool now = hit && rank < kSlots;
        if (now) {
#pragma unroll
          for (int k = 0; k < NV; ++k) s_hit[wave][rank][k] = u[k];
          s_hit_lane[wave][rank] = lane;
        }
        wave_sync();
        const uint64_t done = __ballot(now);
        const int held = __popcll(done) * NV * N;
        hits &= ~done;
        hit = hit && !now;
        for (int c = 0; c < held; c += 64) {
          const int at = min(c + lane, held - 1), slot = at / (NV * N), k = at / N % NV, j = at % N;
          const float v = load1<T>(reinterpret_cast<const T*>(&s_hit[wave][slot][k]) + j);
          const bool take = c + lane < held && (ties ? v >= bound : v > bound) && v > -INFINITY;
          const uint64_t taken = __ballot(take);
          int first = 0;
          if (lane == 0 && taken) first = atomicAdd(&s_count, __popcll(taken));
          first = __builtin_amdgcn_readfirstlane(first) + __popcll(taken & (((uint64_t)1 << lane) - 1));
          if (take && first < kCandidates)
            s_cand[first] = token_key(v, vec_start<T>(V, tile0 + (k * W + wave) * 64 + s_hit_lane[wave][slot]) + j);
        }
        wave_sync();
      }
      tile_again(u);
    }

    // The sums without the first maximum; one that was it becomes a term of the first thread's.
    if (rises) {
      const float d = fmaxf(m - mt, kLowest), f = __builtin_amdgcn_exp2f(d * c2);
      S += tid == 0 && m > -INFINITY ? 1.0f : 0.0f;
      Tq = fmaf(f, Tq, f * d * S);  // f d first: d alone may be huge where f is 0
      S *= f;
      m = mt;
    }
    const float at = m > -INFINITY ? m : 0.0f;
    bool left_out = !rises || s_owner[p] != tid;
    float st = 0.0f, tt = 0.0f;
    auto add = [&](float v) {
      const float d = v - at;
      const float e = __builtin_amdgcn_exp2f(d * c2);
      st += e;
      tt = fmaf(e, fmaxf(d, kLowest), tt);
    };
    if (__any(!left_out)) {  // one wave
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float v = elem<T>(u[k], j);
          const bool now = !left_out && v == m;
          left_out |= now;
          add(now ? -INFINITY : v);
        }
    } else {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if (MANY && (tile0 + k * 64 * W) * N >= V) continue;  // uniform: nothing is there
#pragma unroll
        for (int j = 0; j < N; ++j) add(elem<T>(u[k], j));
      }
    }
    S += st;
    Tq += tt;
    if constexpr (!MANY) break;
#pragma unroll
    for (int k = 0; k < NV; ++k) u[k] = ahead[MANY ? k : 0];
  }
  if (top) {
    __syncthreads();
    const int n = s_count;
    __syncthreads();
    settle(n, gathered, (vecs - 1) / TILE * TILE);
  }
  S = wave_sum(S);
  Tq = wave_sum(Tq);
  if constexpr (W > 1) {
    if (lane == 0) {
      s_sum[wave] = S;
      s_sum[W + wave] = Tq;
    }
    __syncthreads();
    S = s_sum[0];
    Tq = s_sum[W];
#pragma unroll
    for (int w = 1; w < W; ++w) {
      S += s_sum[w];
      Tq += s_sum[W + w];
    }
  }

  // A NaN anywhere makes S NaN, and so does a maximum of +inf (inf - inf).
  const bool bad = !(S >= 0.0f) || m == INFINITY, empty = m == -INFINITY;
  const float lse = log1pf(S);
  if (tid == 0) {
    if (a.logprobs) {
      float lp = (z_target - m) * inv_tau - lse;
      if (empty) lp = -INFINITY;
      if (bad || target >= (uint32_t)V) lp = NAN;
      a.logprobs[blockIdx.x] = target == kNoToken ? 0.0f : lp;
    }
    if (a.entropy) {
      const float h = lse - Tq * inv_tau / (1.0f + S);
      a.entropy[blockIdx.x] = bad ? NAN : empty ? 0.0f : h;
    }
  }
  if (wave == 0 && lane < top) {
    const size_t at = (size_t)blockIdx.x * top + lane;
    const bool has = best != 0 && !bad;
    a.top_ids[at] = has ? (uint32_t)key_id(best) : kNoToken;
    a.top_logprobs[at] = bad ? NAN : has ? (key_value(best) - m) * inv_tau - lse : -INFINITY;
  }
}

// -------------------------------------------------------------- distillation
// With p the softmax of the student's row and q that of the teacher's entries,
// both at temperature tau, a row's loss is w tau^2 sum_j q_j (log q_j - log p_j)
// and its gradient w tau (p - q).  The dense part p is written from the
// registers that the sums were taken from; the few teacher's tokens are then
// written again with their q.
// 8192 fp32 rows of 16384: 220 us (4.9 TB/s); 777 bf16 rows of 65537: 69 us
// (4.4 TB/s with the second read); 37 fp32 rows of 2048: 5.5 us, latency.
// MANY: the row takes several tiles, each thread with a maximum and sum of its
// own until the end, each tile loaded while the one before is summed.
template <class T, int W, int NV, bool MANY>
__global__ __launch_bounds__(64 * W) void distill_kernel(DistillArgs a) {
  constexpr int N = vec_n<T>(), TILE = 64 * W * NV;
  __shared__ float s_red[2 * W];
  __shared__ float s_teach[2];  // the teacher's maximum and log of its sum
  extern __shared__ float s_dyn[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = a.vocab, K = a.teacher_k;
  float* s_q = s_dyn;
  float* s_z = s_dyn + K;  // the student's logits at the teacher's tokens
  uint32_t* s_id = reinterpret_cast<uint32_t*>(s_dyn + 2 * K);
  const T* row = static_cast<const T*>(a.logits) + (size_t)blockIdx.x * a.ld;
  T* grad = a.grad ? static_cast<T*>(a.grad) + (size_t)blockIdx.x * a.ld_grad : nullptr;
  const float inv_tau = 1.0f / a.temperature, c2 = kLog2e * inv_tau;
  const float weight = a.row_weights ? a.row_weights[blockIdx.x] : 1.0f;
  const int vecs = (V + N - 1) / N;

  // The teacher's entries, by the first wave.
  if (wave == 0) {
    float mt = -INFINITY;
    bool bad = false;
    for (int j = lane; j < K; j += 64) {
      uint32_t id = a.teacher_ids[(size_t)blockIdx.x * K + j];
      float t = a.teacher_logits[(size_t)blockIdx.x * K + j];
      if (id != kNoToken && id >= (uint32_t)V) t = NAN;  // no such token
      if (id >= (uint32_t)V) id = kNoToken;
      bad |= id == kNoToken ? t != t && a.teacher_ids[(size_t)blockIdx.x * K + j] != kNoToken : !(t < INFINITY);
      if (id == kNoToken) t = -INFINITY;
      s_id[j] = id;
      s_q[j] = t;
      s_z[j] = id == kNoToken ? 0.0f : load1<T>(row + id);
      mt = fmaxf(mt, t);
    }
    mt = wave_max(mt);
    float z = 0.0f;
    if (mt > -INFINITY)
      for (int j = lane; j < K; j += 64) z += __builtin_amdgcn_exp2f((s_q[j] - mt) * c2);
    z = wave_sum(z);
    if (__any(bad)) mt = NAN;
    if (lane == 0) {
      s_teach[0] = mt;
      s_teach[1] = z;
    }
  }
  __syncthreads();
  const float t_max = s_teach[0], t_sum = s_teach[1];
  // A row without weight or without a teacher: zeros, whatever it holds.
  if (weight == 0.0f || t_max == -INFINITY) {
    if (tid == 0) a.losses[blockIdx.x] = 0.0f;
    if (grad) {
      for (int i = tid; i < vecs; i += 64 * W) {
        if (i * N + N <= V) {
          *reinterpret_cast<u32x4_any_t*>(grad + i * N) = u32x4_t{0, 0, 0, 0};
        } else {
          for (int e = i * N; e < V; ++e) store1(grad + e, 0.0f);
        }
      }
    }
    return;
  }

  float m = -INFINITY, S = 0.0f;
  u32x4_t u[NV], ahead[MANY ? NV : 1];
  tile_load<T, W, NV>(u, row, V, 0);
  auto sum = [&](float at, int tile0) {
    float st = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (MANY && (tile0 + k * 64 * W) * N >= V) continue;  // uniform: nothing is there
      if constexpr (NV > 8) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < N; ++j) st += __builtin_amdgcn_exp2f((elem<T>(u[k], j) - at) * c2);
    }
    tile_again(u);
    return st;
  };
  if constexpr (MANY) {
    float mine = -INFINITY;
    for (int tile0 = 0; tile0 < vecs; tile0 += TILE) {
      tile_again(u);  // its loads end here
      // Behind the last tile comes the first, for the gradient.
      tile_load<T, W, NV>(ahead, row, V, tile0 + TILE < vecs ? tile0 + TILE : 0);
      const float mn = fmaxf(mine, tile_max<T, NV>(u)), at = mn > -INFINITY ? mn : 0.0f;
      tile_again(u);
      S = (mine > -INFINITY ? S * __builtin_amdgcn_exp2f((mine - at) * c2) : S) + sum(at, tile0);
      mine = mn;
#pragma unroll
      for (int k = 0; k < NV; ++k) u[k] = ahead[k];
    }
    m = wave_max(mine);
    if (lane == 0) s_red[wave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) m = fmaxf(m, s_red[w]);
    if (mine > -INFINITY) S *= __builtin_amdgcn_exp2f((mine - m) * c2);
  } else {
    m = wave_max(tile_max<T, NV>(u));
    tile_again(u);
    if constexpr (W > 1) {
      if (lane == 0) s_red[wave] = m;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < W; ++w) m = fmaxf(m, s_red[w]);
    }
    S = sum(m > -INFINITY ? m : 0.0f, 0);
  }
  S = wave_sum(S);
  if constexpr (W > 1) {
    if (lane == 0) s_red[W + wave] = S;
    __syncthreads();
    S = s_red[W];
#pragma unroll
    for (int w = 1; w < W; ++w) S += s_red[W + w];
  }
  const bool empty = m == -INFINITY;
  const float at = empty ? 0.0f : m;

  if (wave == 0) {
    const float log_z = logf(t_sum), log_s = logf(S);
    float kl = 0.0f;
    for (int j = lane; j < K; j += 64) {
      const float t = (s_q[j] - t_max) * inv_tau, q = __builtin_amdgcn_exp2f((s_q[j] - t_max) * c2) / t_sum;
      if (!(q <= 0.0f)) kl += q * ((t - log_z) - ((s_z[j] - at) * inv_tau - log_s));
      s_q[j] = q;
    }
    kl = wave_sum(kl);
    if (empty && S == 0.0f) kl = t_max != t_max ? NAN : INFINITY;  // every token masked, yet one is taught
    if (lane == 0) a.losses[blockIdx.x] = weight * a.temperature * a.temperature * kl;
  }
  if (!grad) return;
  const float scale = weight * a.temperature * (t_max != t_max ? NAN : 1.0f);
  const float ps = S == 0.0f ? scale * 0.0f : scale / S;
  auto write = [&](int tile0) {
    T* mine = grad + (size_t)(tile0 + tid) * N;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if ((tile0 + k * 64 * W) * N >= V) continue;
      if constexpr (NV > 8) __builtin_amdgcn_sched_barrier(0);  // one vector's exponentials at a time: registers
      const int i = tile0 + k * 64 * W + tid;
      float g[N];
#pragma unroll
      for (int j = 0; j < N; ++j) g[j] = __builtin_amdgcn_exp2f((elem<T>(u[k], j) - at) * c2) * ps;
      if (i * N + N <= V) {
        *reinterpret_cast<u32x4_any_t*>(mine + k * 64 * W * N) = pack<T>(g);
      } else {
        const int s = vec_start<T>(V, i);
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (s + j >= i * N && s + j < V) store1(grad + s + j, g[j]);
      }
    }
  };
  if constexpr (!MANY) {
    write(0);
  } else {
    // In place, a partial vector's load also covers its neighbour's elements,
    // which may be written already: they are masked, as in the sums.
    for (int tile0 = 0; tile0 < vecs; tile0 += TILE) {
      tile_again(u);
      if (tile0 + TILE < vecs) tile_load<T, W, NV>(ahead, row, V, tile0 + TILE);
      write(tile0);
#pragma unroll
      for (int k = 0; k < NV; ++k) u[k] = ahead[k];
    }
  }
  // The dense stores have reached the cache before another thread's store to the same token.
  __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
  __syncthreads();
  for (int j = tid; j < K; j += 64 * W) {
    const uint32_t id = s_id[j];
    if (id == kNoToken) continue;
    float q = 0.0f;
    bool first = true;
    for (int i = 0; i < K; ++i) {
      if (s_id[i] != id) continue;
      first &= i >= j;
      q += s_q[i];
    }
    if (!first) continue;  // the token's first entry writes it
    const float p = S == 0.0f ? 0.0f : __builtin_amdgcn_exp2f((s_z[j] - at) * c2) / S;
    store1(grad + id, scale * (p - q));
  }
}

template <class T, int W, int NV, bool MANY>
Status logprobs(hipStream_t stream, const LogprobArgs& a, size_t rows) {
  const size_t lds = a.top_k ? kCandidates * 8 : 0;
  token_logprobs_kernel<T, W, NV, MANY><<<(uint32_t)rows, 64 * W, lds, stream>>>(a);
  PSSA_LAUNCH_CHECK("token_logprobs_kernel");
  return Status::Ok();
}
template <class T, int W, int NV, bool MANY>
Status distill(hipStream_t stream, const DistillArgs& a, size_t rows) {
  distill_kernel<T, W, NV, MANY><<<(uint32_t)rows, 64 * W, (size_t)a.teacher_k * 12, stream>>>(a);
  PSSA_LAUNCH_CHECK("distill_kernel");
  return Status::Ok();
}

// Waves for a row: so many that the rows fill the chip's compute units, and a
// tile that holds the row where no more than these are needed for it.
//   us, with 8 alternatives:      256 rows of          3000 rows of
//                               65537 100003 bf16    65537 100003 bf16
//     16 waves                     19     24            222    273
//     8 waves                      21     28            149    204
//     4 waves                      31     47            122    182
template <class T>
Status launch_logprobs(hipStream_t stream, const LogprobArgs& a, size_t rows) {
  const int vecs = (a.vocab + vec_n<T>() - 1) / vec_n<T>();
  if (vecs <= 64 * 1 * 4) return logprobs<T, 1, 4, false>(stream, a, rows);
  if (vecs <= 64 * 4 * 4) return logprobs<T, 4, 4, false>(stream, a, rows);
  if (vecs <= 64 * 4 * 8) return logprobs<T, 4, 8, false>(stream, a, rows);
  if (rows > 2 * kComputeUnits) return logprobs<T, 4, 4, true>(stream, a, rows);
  if (vecs <= 64 * 8 * 8) return logprobs<T, 8, 8, false>(stream, a, rows);
  if (rows > kComputeUnits) return logprobs<T, 8, 4, true>(stream, a, rows);
  if (vecs <= 64 * 16 * 8) return logprobs<T, 16, 8, false>(stream, a, rows);
  return logprobs<T, 16, 4, true>(stream, a, rows);
}

// The smallest workgroup whose registers hold the row, which the gradient is
// then written from: eight waves with 16 vectors rather than sixteen with 8
// leave room for a second one (3000 rows of 50257 bf16: 175 and 195 us).  A
// row past the registers is read again, and so is a bf16 one that would
// leave no such room, where there are rows for a second workgroup: a byte of
// bf16 costs twice the exponentials, which hide behind another's loads (us,
// tiles of 8 waves against 16 waves that hold the row: 3000 rows of 65537 242
// and 310, of 100003 380 and 395; 256 rows of 100003 33 and 31).  fp32 rows
// gain from being read once (3000 of 50257: 278 us held, 338 in tiles).
template <class T>
Status launch_distillation(hipStream_t stream, const DistillArgs& a, size_t rows) {
  const int vecs = (a.vocab + vec_n<T>() - 1) / vec_n<T>();
  if (vecs <= 64 * 1 * 4) return distill<T, 1, 4, false>(stream, a, rows);
  if (vecs <= 64 * 4 * 4) return distill<T, 4, 4, false>(stream, a, rows);
  if (vecs <= 64 * 4 * 8) return distill<T, 4, 8, false>(stream, a, rows);
  if (vecs <= 64 * 8 * 8) return distill<T, 8, 8, false>(stream, a, rows);
  if (vecs <= 64 * 8 * 16) return distill<T, 8, 16, false>(stream, a, rows);
  if (vecs > 64 * 16 * 16) return distill<T, 16, 4, true>(stream, a, rows);
  if constexpr (sizeof(T) == 2)
    if (rows > kComputeUnits) return distill<T, 8, 4, true>(stream, a, rows);
  return distill<T, 16, 16, false>(stream, a, rows);
}

}  // namespace

// A launch's threads are counted in 32 bits: more rows go in parts.
constexpr size_t kMostRows = (size_t)1 << 21;

Status launch_token_logprobs(hipStream_t stream, int dtype, const LogprobArgs& args, size_t rows) {
  LogprobArgs a = args;
  for (size_t n; rows; rows -= n) {
    n = std::min(rows, kMostRows);
    PSSA_RETURN_IF(dtype == PSSA_HIP_F32 ? launch_logprobs<float>(stream, a, n) : launch_logprobs<Bf16>(stream, a, n));
    a.logits = static_cast<const char*>(a.logits) + n * a.ld * (dtype == PSSA_HIP_F32 ? 4 : 2);
    if (a.targets) a.targets += n;
    if (a.logprobs) a.logprobs += n;
    if (a.entropy) a.entropy += n;
    if (a.top_ids) a.top_ids += n * a.top_k;
    if (a.top_logprobs) a.top_logprobs += n * a.top_k;
  }
  return Status::Ok();
}

Status launch_distill(hipStream_t stream, int dtype, const DistillArgs& args, size_t rows) {
  DistillArgs a = args;
  const size_t size = dtype == PSSA_HIP_F32 ? 4 : 2;
  for (size_t n; rows; rows -= n) {
    n = std::min(rows, kMostRows);
    PSSA_RETURN_IF(dtype == PSSA_HIP_F32 ? launch_distillation<float>(stream, a, n)
                                         : launch_distillation<Bf16>(stream, a, n));
    a.logits = static_cast<const char*>(a.logits) + n * a.ld * size;
    a.teacher_ids += n * a.teacher_k;
    a.teacher_logits += n * a.teacher_k;
    if (a.row_weights) a.row_weights += n;
    a.losses += n;
    if (a.grad) a.grad = static_cast<char*>(a.grad) + n * a.ld_grad * size;
  }
  return Status::Ok();
}

}  // namespace pssa
