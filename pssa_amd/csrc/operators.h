// Language-model operators on device-resident arrays: log probabilities and
// distillation over logit rows, linear attention with a decay for each head,
// the gated delta rule, products with 4-bit weights, norms with 8-bit rows and
// products of these, beam search.
#pragma once
#include "common.h"

namespace pssa {

// Threads of a launch along x: below 2^32, in workgroups of 256.
constexpr size_t kMostThreads = ((size_t)1 << 32) - 256;

// Dynamic LDS above the default limit, once for each device.
Status init_w4_attributes();

// ---------------------------------------------------------------- logit rows
constexpr int kMaxAlternatives = 64;  // top tokens a row can list: one wave's lanes
constexpr int kMaxTeacher = 1024;     // teacher entries of a row (held in LDS)

struct LogprobArgs {
  const void* logits = nullptr;  // row r at logits + r * ld (f32 or bf16)
  size_t ld = 0;
  int vocab = 0;
  const uint32_t* targets = nullptr;  // [rows] or null
  float temperature = 1.0f;
  int top_k = 0;
  float* logprobs = nullptr;      // [rows], with targets
  float* entropy = nullptr;       // [rows] or null
  uint32_t* top_ids = nullptr;    // [rows, top_k]
  float* top_logprobs = nullptr;  // [rows, top_k]
};
Status launch_token_logprobs(hipStream_t stream, int dtype, const LogprobArgs& a, size_t rows);

struct DistillArgs {
  const void* logits = nullptr;
  size_t ld = 0;
  int vocab = 0;
  const uint32_t* teacher_ids = nullptr;   // [rows, teacher_k]
  const float* teacher_logits = nullptr;   // [rows, teacher_k]
  int teacher_k = 0;
  float temperature = 1.0f;
  const float* row_weights = nullptr;  // [rows] or null (1)
  float* losses = nullptr;             // [rows]
  void* grad = nullptr;                // row r at grad + r * ld_grad, the logits' type, or null
  size_t ld_grad = 0;
};
Status launch_distill(hipStream_t stream, int dtype, const DistillArgs& a, size_t rows);

// -------------------------------------------------------------- 4-bit weights
struct W4View {
  const void* packed = nullptr;
  const float* scales = nullptr;   // half of each group's scale, [tile][group][16]
  const uint8_t* zeros = nullptr;  // [tile][group][16], null: 8 everywhere
  int n = 0, k = 0, group = 0;
};
size_t w4_packed_bytes(size_t n, size_t k);
size_t w4_groups_held(size_t n, size_t k, size_t group);
Status launch_w4_pack(hipStream_t stream, const uint8_t* codes, const float* scales, const uint8_t* zeros, int n, int k,
                      int group, void* packed, float* out_scales, uint8_t* out_zeros);
Status launch_matvec_w4(hipStream_t stream, int x_dtype, const void* x, size_t ld_x, int m, const W4View& w, float* y,
                        size_t ld_y);

// ------------------------------------------------------------ linear attention
constexpr int kLinearMaxKey = 128;      // d_key held in a workgroup's tiles
constexpr int kLinearSteps = 4;         // up to this length a sequence runs token by token
constexpr int kLinearInline = 256;      // sequences whose offsets travel with the kernel's arguments

struct LinearArgs {
  const void *q = nullptr, *k = nullptr, *v = nullptr;  // token t, head h at t * ld + h * width
  size_t ld_q = 0, ld_k = 0, ld_v = 0, ld_out = 0;
  const float* log_decay = nullptr;  // [heads]
  const float* state_in = nullptr;   // [n_seqs, heads, dk, dv] or null (zeros)
  float* state_out = nullptr;        // likewise, or null
  void* out = nullptr;
  float scale = 1.0f;
  int n_seqs = 0, heads = 0, kv_heads = 0, dk = 0, dv = 0;
  // The work items: whole sequences, or (split) their segments of seg_len tokens.
  int items = 0, seg_len = 0;
  float* seg_state = nullptr;       // [items, heads, dk, dv] of a split call
  int uniform_len = -1;             // every sequence's length, or -1: the tables
  int uniform_segs = 1;             // its segments
  // [n_seqs + 1] first tokens and, in a split call, as many first items: on the device, or null and here.
  const uint32_t* table = nullptr;
  uint32_t inline_tokens[kLinearInline + 1] = {};
  uint32_t inline_items[kLinearInline + 1] = {};
};
Status init_linear_attributes();
// Tokens of a segment where a call of these sizes is split, else 0.
int linear_segment(const uint64_t* lens, size_t n_seqs, size_t longest, size_t heads, size_t d_key, size_t d_val);
Status launch_linear_attention(hipStream_t stream, int dtype, const LinearArgs& a, int longest);

// ------------------------------------------------------------------- norms
constexpr size_t kRmsWidth = 65536;  // the widest row: a workgroup's registers
constexpr size_t kRmsStep = 4096;    // rows at a time, at most
constexpr size_t kRmsRows = ((size_t)1 << 31) - kRmsStep;  // a row and a step beyond it stay below 2^31

struct RmsNormArgs {
  const void *x = nullptr, *residual = nullptr;  // row r at r * ld; residual may be null
  size_t ld_x = 0, ld_residual = 0, ld_sum = 0, ld_out = 0, ld_codes = 0;
  const float* gamma = nullptr;  // [width], null: ones
  int width = 0;
  bool normed = true;  // false: codes of the rows as they are
  float eps = 0.0f;
  // Each may be null (codes and scales together); out needs gamma.
  void *sum = nullptr, *out = nullptr;
  int8_t* codes = nullptr;
  float* scales = nullptr;
};
Status launch_rms_norm(hipStream_t stream, int dtype, const RmsNormArgs& a, size_t rows);

// ---------------------------------------------------------- 8-bit products
constexpr size_t kI8Depth = 131071;  // 128 * 128 * k stays below 2^31

struct I8Args {
  const int8_t *x = nullptr, *w = nullptr;  // rows of k codes
  size_t ld_x = 0, ld_w = 0, ld_y = 0;
  const float *x_scales = nullptr, *w_scales = nullptr;  // [m], [n]
  void* y = nullptr;
  int m = 0, n = 0, k = 0;
  int splits = 1;            // parts of k
  int32_t* parts = nullptr;  // [splits, m, n] sums of each, where there are several
};
constexpr int kI8FewRows = 64;  // up to these the weights go straight to registers
// Whether rows of k codes lie in units of 16 bytes: many rows are copied where not.
bool i8_in_units(const void* p, size_t ld, size_t k);
// Parts of k of a product of these sizes, and its scratch: the parts' sums,
// and the copies of rows and weights that there are.
struct I8Plan {
  int splits = 1;
  size_t parts_bytes = 0, pack_bytes = 0;
  size_t bytes() const { return ((parts_bytes + 255) & ~(size_t)255) + pack_bytes; }
};
I8Plan i8_plan(size_t m, size_t n, size_t k, bool copy_x, bool copy_w);
Status init_i8_attributes();
Status launch_matmul_i8(hipStream_t stream, int y_dtype, I8Args a, const I8Plan& p, void* scratch);

// -------------------------------------------------------- gated delta rule
constexpr int kDeltaMaxKey = 128;   // d_key held in a workgroup's tiles
constexpr int kDeltaSteps = 4;      // up to this length a sequence runs token by token
constexpr int kDeltaInline = 256;   // sequences whose offsets travel with the kernel's arguments

struct DeltaArgs {
  const void *q = nullptr, *k = nullptr, *v = nullptr;  // token t, head h at t * ld + h * width
  size_t ld_q = 0, ld_k = 0, ld_v = 0, ld_out = 0, ld_gates = 0;
  const float *log_decay = nullptr, *beta = nullptr;  // token t, head h at t * ld_gates + h
  const float* state_in = nullptr;  // [n_seqs, heads, dk, dv] or null (zeros)
  float* state_out = nullptr;       // likewise, or null
  void* out = nullptr;
  float scale = 1.0f;
  int n_seqs = 0, heads = 0, key_heads = 0, dk = 0, dv = 0;
  int uniform_len = -1;  // every sequence's length, or -1: the tables
  // Where the call runs in chunks: what is worked out for each of them ahead,
  // [chunks, heads of one launch], and the launch's first head.
  char* ahead = nullptr;
  int head0 = 0, heads_here = 0, chunks = 0;
  int share = 1;  // neighbouring heads of the launch that read the same keys
  int wide_q = 0, wide_k = 0, wide_v = 0;  // elements from a head to the next in rows that may be copies
  // The work items: whole sequences, or (split) their segments of seg_chunks
  // chunks, whose own states and transitions are [items, heads of one launch].
  int items = 0, seg_chunks = 0, uniform_segs = 1;
  float *seg_state = nullptr, *seg_move = nullptr;
  // [n_seqs + 1] first tokens, behind them first chunks and, in a split call,
  // first items: on the device, or null and here.
  const uint32_t* table = nullptr;
  uint32_t inline_tokens[kDeltaInline + 1] = {};
  uint32_t inline_chunks[kDeltaInline + 1] = {};
  uint32_t inline_items[kDeltaInline + 1] = {};
};
// Tokens of a chunk of a type, and the scratch of a call: what is worked out
// ahead for the heads of one launch, the copies of rows that do not lie in
// units of 16 bytes, which the caller adds, and the segments' states.
int delta_chunk(int dtype);
struct DeltaScratch {
  size_t ahead = 0, rows = 0, state = 0, move = 0;  // bytes
  int heads_here = 0;                               // heads of a launch
};
// `items` segments, 0 where the call is not split.
DeltaScratch delta_scratch(int dtype, size_t chunks, size_t n_seqs, size_t items, size_t heads, size_t d_key, size_t d_val);
// Rows of heads of `width` elements that a call in chunks reads as they are,
// and the bytes of a copy of those that it does not.
bool delta_in_units(int dtype, const void* p, size_t ld, size_t width);
size_t delta_copy_bytes(int dtype, size_t tokens, size_t heads, size_t width);
// Chunks of a segment where a call of these sizes is split, else 0.
int delta_segment(int dtype, const uint64_t* lens, size_t n_seqs, size_t longest, size_t heads, size_t d_key, size_t d_val);
Status init_delta_attributes();
Status launch_delta_rule(hipStream_t stream, int dtype, DeltaArgs a, size_t tokens, int longest, const DeltaScratch& s,
                         char* scratch);

// ------------------------------------------------------------- beam search
constexpr int kMaxBeams = 64;  // of a group, before and after a step

struct BeamArgs {
  const void* logits = nullptr;  // row g * beams + b at row * ld
  size_t ld = 0;
  int vocab = 0, beams = 0, keep = 0;
  const float* scores = nullptr;   // [groups, beams]
  const uint32_t* last = nullptr;  // [groups, beams] or null
  uint32_t eos = PSSA_HIP_NO_TOKEN;
  uint32_t first_id = 0;  // the token of a row's first logit
  uint32_t *parents = nullptr, *tokens = nullptr;  // [groups, keep]
  float* out_scores = nullptr;                     // [groups, keep]
  int slices = 1;
  void* sums = nullptr;      // scratch [rows, slices]
  uint64_t* keys = nullptr;  // scratch [rows, slices, keep]
};
// How the rows of a call are cut: pieces of 16 bytes a thread, slices a row,
// and the scratch (sums, then keys).
struct BeamPlan {
  int pieces = 1;
  size_t slices = 1, sums_bytes = 0, bytes = 0;
};
BeamPlan beam_plan(int dtype, size_t rows, size_t vocab, size_t keep);
Status launch_beam_select(hipStream_t stream, int dtype, const BeamArgs& a, size_t groups, const BeamPlan& p);

struct GatherArgs {
  const void* src = nullptr;  // row i of group g at (g * n_in + i) * ld_src bytes
  void* dst = nullptr;        // may be src
  size_t ld_src = 0, ld_dst = 0, row_bytes = 0;
  int groups = 0, n_in = 0, n_out = 0;
  const uint32_t* parents = nullptr;  // [groups, n_out]; a row whose parent is not below n_in stays as it is
};
// Bytes of a row that a thread moves.
size_t beam_gather_piece(const GatherArgs& a);
Status launch_beam_gather(hipStream_t stream, const GatherArgs& a);
// Rows 0 .. groups-1 copied to rows g * beams .. + beams - 1 of the same array.
Status launch_beam_spread(hipStream_t stream, void* rows, size_t words, size_t ld, size_t groups, size_t beams);
// The chosen tokens as the next step's inputs (0 where there is none).
Status launch_beam_feed(hipStream_t stream, const uint32_t* tokens, uint32_t* ids, size_t n);

}  // namespace pssa
