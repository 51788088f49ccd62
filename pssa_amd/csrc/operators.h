// Language-model operators on device-resident arrays: log probabilities and
// distillation over logit rows, linear attention with a decay for each head,
// products with 4-bit weights.
#pragma once
#include "common.h"

namespace pssa {

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

}  // namespace pssa
