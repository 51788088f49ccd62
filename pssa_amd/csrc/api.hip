// C ABI of libpssa_hip (include/pssa_hip.h).  Validation happens before any
// allocation or launch; device failures after a launch are reported as
// PSSA_HIP_EDEVICE (fatal).
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <memory>

#include "gemm.h"
#include "memory.h"
#include "model.h"
#include "operators.h"
#include "ssm.h"

namespace pssa {
Status launch_dense_scan(hipStream_t stream, const float* A, const float* B, const float* H0, float* H,
                         int batch, int L, int s, void* scratch, size_t scratch_bytes);
// Scratch the two-level schedule needs (0: the sequential kernels run).
size_t dense_scan_scratch_bytes(int batch, int L, int s);
Status init_dense_scan_attributes();
}

using pssa::DevBuf;
using pssa::Status;

namespace {

// A temporary of one call (its block returns to the context's pool) holding
// a host array.
Status upload(pssa_hip_ctx* ctx, DevBuf& dst, const void* src, size_t bytes) {
  PSSA_RETURN_IF(dst.alloc(bytes, &ctx->pool));
  return ctx->stage.to_device(dst.p, src, bytes, ctx->stream);
}
// The same for a buffer that stays (model parameters, cached weights): moved
// by the runtime, `src` must outlive the copy.
Status upload_keep(pssa_hip_ctx* ctx, DevBuf& dst, const void* src, size_t bytes) {
  PSSA_RETURN_IF(dst.alloc(bytes));
  if (bytes) PSSA_HIP_TRY(hipMemcpyAsync(dst.p, src, bytes, hipMemcpyHostToDevice, ctx->stream));
  return Status::Ok();
}

Status download(pssa_hip_ctx* ctx, void* dst, const DevBuf& src, size_t bytes) {
  return ctx->stage.to_host(dst, src.p, bytes, ctx->stream);
}

uint16_t bf16_bits(float f) {
  uint32_t u;
  std::memcpy(&u, &f, 4);
  u += 0x7FFFu + ((u >> 16) & 1u);
  return (uint16_t)(u >> 16);
}

// Weight upload in the model's storage type.
Status upload_weight(pssa_hip_ctx* ctx, DevBuf& dst, const float* src, size_t n, int dtype) {
  if (dtype == PSSA_HIP_F32) return upload_keep(ctx, dst, src, n * 4);
  std::vector<uint16_t> tmp(n);
  for (size_t i = 0; i < n; ++i) tmp[i] = bf16_bits(src[i]);
  PSSA_RETURN_IF(upload_keep(ctx, dst, tmp.data(), n * 2));
  PSSA_HIP_TRY(hipStreamSynchronize(ctx->stream));  // tmp must outlive the copy
  return Status::Ok();
}

Status sync(pssa_hip_ctx* ctx) {
  return ctx->stage.wait(ctx->stream);
}

Status need(bool cond, const char* msg) { return cond ? Status::Ok() : Status::Invalid(msg); }

Status check_ctx(pssa_hip_ctx* ctx) { return ctx ? Status::Ok() : Status::Invalid("null context"); }

Status check_config(const pssa_hip_config& c) {
  if (c.depth < 1 || c.depth > 32) return Status::Invalid("depth must be in 1..=32");
  if (!c.d_vocab || !c.d_latent || !c.d_state || !c.d_mem_key || !c.mem_capacity || !c.adapter_rank)
    return Status::Invalid("model dimensions and memory capacity must be positive");
  if (!(std::isfinite(c.tau_mem) && c.tau_mem > 0.0f))
    return Status::Invalid("tau_mem must be finite and positive");
  if (c.d_latent > 16384 || c.d_state > 4096 || c.d_mem_key > 4096 || c.mem_capacity > 8192 ||
      c.d_vocab > (1u << 24) || c.adapter_rank > 256)
    return Status::Invalid("model dimensions exceed the supported range");
  return Status::Ok();
}

float softplus_host(float x) { return x > 20.0f ? x : log1pf(expf(x)); }

// Carries are [lanes, depth, d, s] at the ABI (h_persistent, src/pssa.rs) and
// [lanes, depth] matrices in the scan's channel-blocked layout on the device
// (pssa::carry_at).
Status carry_layout(pssa_hip_lanes* L, const float* in, float* out, bool to_device) {
  const pssa_hip_config& c = L->model->cfg;
  return pssa::launch_carry_convert(L->ctx->stream, in, out, L->lanes * c.depth * L->loops, (int)c.d_latent,
                                    (int)c.d_state, to_device);
}

// Clamps every slot of a block's bank values to `cap` (set_value_cap,
// src/memory.rs:121-134) and rebuilds the transposed readout operand.
// Every slot's value of each given block clamped to `cap` (clamp_value,
// src/memory.rs:150-170), committed only when no slot of any of them has a
// non-finite norm: such a slot fails the call, as the reference's assertion
// (src/memory.rs:151-152) does, and leaves every bank unchanged.
Status cap_bank_values(pssa_hip_model* M, const std::vector<pssa::DevBlock*>& blocks, float cap) {
  const hipStream_t st = M->ctx->stream;
  const int C = (int)M->cfg.mem_capacity, d = (int)M->cfg.d_latent;
  const size_t bytes = (size_t)C * d * 4;
  pssa::ValueCaps caps{};
  caps.c[0] = cap;
  std::vector<DevBuf> capped(blocks.size());
  DevBuf tmp, bad;
  PSSA_RETURN_IF(bad.alloc(4));
  PSSA_RETURN_IF(pssa::launch_fill_zero(st, bad.as<float>(), 1));
  for (size_t i = 0; i < blocks.size(); ++i) {
    PSSA_RETURN_IF(capped[i].alloc(bytes));
    PSSA_RETURN_IF(pssa::launch_clamp_rows(st, blocks[i]->values.as<float>(), capped[i].as<float>(), C, d,
                                           (size_t)d, caps, C, bad.as<int>()));
  }
  int flag = 0;
  PSSA_RETURN_IF(download(M->ctx, &flag, bad, 4));
  PSSA_RETURN_IF(sync(M->ctx));
  if (flag) return Status::Invalid("capped memory value must be finite");
  if (M->dtype == PSSA_HIP_BF16) PSSA_RETURN_IF(tmp.alloc(bytes));
  for (size_t i = 0; i < blocks.size(); ++i) {
    pssa::DevBlock& B = *blocks[i];
    PSSA_HIP_TRY(hipMemcpyAsync(B.values.p, capped[i].p, bytes, hipMemcpyDeviceToDevice, st));
    if (M->dtype == PSSA_HIP_F32) {
      PSSA_RETURN_IF(pssa::launch_transpose(st, B.values.as<float>(), B.values_t.as<float>(), 1, C, d, 1.0f));
    } else {
      PSSA_RETURN_IF(pssa::launch_transpose(st, B.values.as<float>(), tmp.as<float>(), 1, C, d, 1.0f));
      PSSA_RETURN_IF(pssa::launch_to_bf16(st, tmp.as<float>(), C, B.values_t.as<uint16_t>(), C, d, C));
    }
  }
  return sync(M->ctx);  // the staging buffers are freed at return
}

// Empties every lane's repetition-penalty window (a new generation,
// src/inference.rs:345-347).  Fill kernels, so the call may sit in a graph.
Status clear_history(pssa_hip_lanes* L) {
  PSSA_RETURN_IF(pssa::launch_fill_zero(L->ctx->stream, static_cast<float*>(L->hist_n.p), L->lanes));
  return pssa::launch_fill_zero(L->ctx->stream, static_cast<float*>(L->hist_pos.p), L->lanes);
}

// The device copy of a GEMM weight (CudaContext::weight_buffer,
// src/cuda.rs:198-227): reused while current, uploaded again when stale,
// uploaded and kept on first use.  Called with ctx->mu held.
Status cached_weight(pssa_hip_ctx* ctx, const void* host, size_t n, int dtype, const void** out) {
  const size_t bytes = n * (dtype == PSSA_HIP_BF16 ? 2 : 4);
  auto key = std::make_tuple((uintptr_t)host, n, dtype);
  auto it = ctx->weights.find(key);
  if (it == ctx->weights.end()) {
    pssa_hip_ctx::CachedWeight cw;
    PSSA_RETURN_IF(upload_keep(ctx, cw.buf, host, bytes));
    it = ctx->weights.emplace(key, std::move(cw)).first;
  } else if (!it->second.current) {
    PSSA_RETURN_IF(ctx->stage.to_device(it->second.buf.p, host, bytes, ctx->stream));
    it->second.current = true;
  }
  *out = it->second.buf.p;
  return Status::Ok();
}

Status stage_ids_locked(pssa_hip_lanes* L, const uint32_t* ids, size_t n_lanes, size_t T) {
  PSSA_RETURN_IF(need(ids != nullptr, "null ids"));
  PSSA_RETURN_IF(need(T > 0, "prefill requires at least one token"));
  PSSA_RETURN_IF(need(n_lanes > 0 && n_lanes <= L->lanes, "n_lanes must be in 1..=lanes"));
  PSSA_RETURN_IF(need(n_lanes * T <= L->max_tokens, "n_lanes*seq_len exceeds max_tokens"));
  const uint32_t V = (uint32_t)L->model->cfg.d_vocab;
  for (size_t i = 0; i < n_lanes * T; ++i)
    if (ids[i] >= V)
      return Status::Invalid("prompt ID " + std::to_string(ids[i]) + " outside model vocabulary");
  PSSA_RETURN_IF(L->ctx->stage.to_device(L->ids.p, ids, n_lanes * T * 4, L->ctx->stream));
  L->staged_lanes = n_lanes;
  L->staged_len = T;
  return Status::Ok();
}

}  // namespace

extern "C" {

int pssa_hip_abi_version(void) { return PSSA_HIP_ABI_VERSION; }

int pssa_hip_is_fatal(int code) { return code == PSSA_HIP_EDEVICE ? 1 : 0; }

int pssa_hip_init(int device, pssa_hip_ctx** out, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    if (!out) return Status::Invalid("null output handle");
    *out = nullptr;
    int n = 0;
    if (hipGetDeviceCount(&n) != hipSuccess || n == 0) {
      (void)hipGetLastError();
      return Status::NoDev("no HIP device visible");
    }
    if (device < 0 || device >= n) return Status::NoDev("device index out of range");
    hipDeviceProp_t prop;
    PSSA_HIP_TRY(hipGetDeviceProperties(&prop, device));
    if (std::strncmp(prop.gcnArchName, "gfx950", 6) != 0)
      return Status::NoDev(std::string("device is ") + prop.gcnArchName + ", this build targets gfx950");
    PSSA_HIP_TRY(hipSetDevice(device));
    auto ctx = std::make_unique<pssa_hip_ctx>();
    ctx->device = device;
    ctx->name = prop.name;
    ctx->cu_count = prop.multiProcessorCount;
    PSSA_HIP_TRY(hipStreamCreateWithFlags(&ctx->stream, hipStreamNonBlocking));
    PSSA_RETURN_IF(ctx->stage.init());
    PSSA_RETURN_IF(pssa::init_gemm_attributes());
    PSSA_RETURN_IF(pssa::init_retrieve_attributes());
    PSSA_RETURN_IF(pssa::init_decode_attributes());
    PSSA_RETURN_IF(pssa::init_dense_scan_attributes());
    PSSA_RETURN_IF(pssa::init_w4_attributes());
    PSSA_RETURN_IF(pssa::init_linear_attributes());
    PSSA_RETURN_IF(pssa::init_i8_attributes());
    PSSA_RETURN_IF(pssa::init_delta_attributes());
    PSSA_RETURN_IF(pssa::noalloc_scratch_address(&ctx->noalloc_scratch));
    *out = ctx.release();
    return Status::Ok();
  };
  return pssa::finish(body(), err, err_len);
}

void pssa_hip_destroy(pssa_hip_ctx* ctx) {
  if (!ctx) return;
  (void)hipSetDevice(ctx->device);
  if (ctx->stream) {
    (void)hipStreamSynchronize(ctx->stream);
    (void)hipStreamDestroy(ctx->stream);
  }
  if (ctx->scratch) (void)hipFree(ctx->scratch);
  delete ctx;
}

int pssa_hip_device_name(const pssa_hip_ctx* ctx, char* out, size_t out_len) {
  if (!ctx || !out || !out_len) return PSSA_HIP_EINVAL;
  std::snprintf(out, out_len, "hip:%s (gfx950, %d CUs)", ctx->name.c_str(), ctx->cu_count);
  return PSSA_HIP_OK;
}

int pssa_hip_device_alloc(pssa_hip_ctx* ctx, size_t bytes, void** out, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(check_ctx(ctx));
    PSSA_RETURN_IF(need(out != nullptr, "null output handle"));
    *out = nullptr;
    PSSA_RETURN_IF(need(bytes > 0 && bytes <= ((size_t)1 << 40), "allocation size must be in 1..=2^40"));
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    void* p = nullptr;
    const hipError_t e = pssa::device_malloc(&p, bytes);
    if (e != hipSuccess) return Status::NoMem(std::string("hipMalloc: ") + hipGetErrorString(e));
    *out = p;
    return Status::Ok();
  };
  return pssa::finish(body(), err, err_len);
}

void pssa_hip_device_free(pssa_hip_ctx* ctx, void* p) {
  if (!ctx || !p) return;
  std::lock_guard<std::mutex> g(ctx->mu);
  (void)hipSetDevice(ctx->device);
  (void)hipStreamSynchronize(ctx->stream);
  (void)hipFree(p);
}

int pssa_hip_memcpy(pssa_hip_ctx* ctx, void* dst, const void* src, size_t bytes, int kind, char* err,
                    size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(check_ctx(ctx));
    PSSA_RETURN_IF(need(dst && src, "memcpy: null pointer"));
    PSSA_RETURN_IF(need(kind == PSSA_HIP_H2D || kind == PSSA_HIP_D2H || kind == PSSA_HIP_D2D, "memcpy: unknown kind"));
    if (bytes == 0) return Status::Ok();
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    const hipMemcpyKind k = kind == PSSA_HIP_H2D ? hipMemcpyHostToDevice
                            : kind == PSSA_HIP_D2H ? hipMemcpyDeviceToHost
                                                   : hipMemcpyDeviceToDevice;
    if (k == hipMemcpyHostToDevice)
      PSSA_RETURN_IF(ctx->stage.to_device(dst, src, bytes, ctx->stream));
    else if (k == hipMemcpyDeviceToHost)
      PSSA_RETURN_IF(ctx->stage.to_host(dst, src, bytes, ctx->stream));
    else
      PSSA_HIP_TRY(hipMemcpyAsync(dst, src, bytes, k, ctx->stream));
    return sync(ctx);
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_synchronize(pssa_hip_ctx* ctx, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(check_ctx(ctx));
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    return sync(ctx);
  };
  return pssa::finish(body(), err, err_len);
}

// ------------------------------------------------------------------- GEMM
int pssa_hip_gemm_xwt(pssa_hip_ctx* ctx, const float* x, size_t x_len, const void* w, size_t w_len,
                      int w_dtype, size_t m, size_t n, size_t k, size_t batch, float* y,
                      size_t y_len, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(check_ctx(ctx));
    PSSA_RETURN_IF(need(x && w && y, "gemm: null buffer"));
    PSSA_RETURN_IF(need(m && n && k && batch, "GEMM dimensions must be positive"));
    PSSA_RETURN_IF(need(w_dtype == PSSA_HIP_F32 || w_dtype == PSSA_HIP_BF16, "gemm: unknown dtype"));
    size_t rows = 0, xin = 0, win = 0, yout = 0;
    PSSA_RETURN_IF(pssa::checked_count({m, batch}, &rows, "gemm rows"));
    PSSA_RETURN_IF(pssa::checked_count({rows, k}, &xin, "gemm input"));
    PSSA_RETURN_IF(pssa::checked_count({n, k}, &win, "gemm weights"));
    PSSA_RETURN_IF(pssa::checked_count({rows, n}, &yout, "gemm output"));
    if (x_len != xin || w_len != win)
      return Status::Invalid("GEMM operand lengths must be " + std::to_string(xin) + " and " +
                             std::to_string(win) + ", got " + std::to_string(x_len) + " and " +
                             std::to_string(w_len));
    if (y_len != yout) return Status::Invalid("GEMM output length mismatch");
    if (rows > INT32_MAX || n > INT32_MAX || k > INT32_MAX) return Status::Invalid("gemm: too large");
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    DevBuf dx, dxh, dy;
    PSSA_RETURN_IF(upload(ctx, dx, x, xin * 4));
    const void* dw = nullptr;
    PSSA_RETURN_IF(cached_weight(ctx, w, win, w_dtype, &dw));
    PSSA_RETURN_IF(dy.alloc(yout * 4, &ctx->pool));
    const void* a = dx.p;
    if (w_dtype == PSSA_HIP_BF16) {
      // bf16 weights multiply bf16-rounded activations (fp32 accumulation).
      PSSA_RETURN_IF(dxh.alloc(xin * 2, &ctx->pool));
      PSSA_RETURN_IF(pssa::launch_to_bf16(ctx->stream, dx.as<float>(), (int)k, dxh.as<uint16_t>(), (int)k, rows, (int)k));
      a = dxh.p;
    }
    pssa::EpiParams ep;
    ep.out32 = dy.as<float>();
    ep.ld32 = (int)n;
    PSSA_RETURN_IF(pssa::launch_gemm(ctx->stream, w_dtype, a, (int)k, dw, (int)k, (int)rows, (int)n, (int)k, ep));
    PSSA_RETURN_IF(download(ctx, y, dy, yout * 4));
    return sync(ctx);
  };
  return pssa::finish(body(), err, err_len);
}

// Shared body of gemm_nn and gemm_tn_accumulate: y = x w^T on the device
// after transposing the operands the layout asks for (`x_t`: x arrives as
// [kx, rows]; `w_t`: w arrives as [k, n]); `accumulate` adds the product to
// the caller's y.
static Status gemm_transposed(pssa_hip_ctx* ctx, const float* x, const float* w, size_t rows, size_t n, size_t k,
                              bool x_t, bool w_t, bool accumulate, float* y) {
  std::lock_guard<std::mutex> g(ctx->mu);
  PSSA_HIP_TRY(hipSetDevice(ctx->device));
  const hipStream_t st = ctx->stream;
  DevBuf dx, dw, dxt, dwt, dy, dacc;
  PSSA_RETURN_IF(upload(ctx, dx, x, rows * k * 4));
  PSSA_RETURN_IF(upload(ctx, dw, w, n * k * 4));
  const float* xa = dx.as<float>();
  const float* wa = dw.as<float>();
  if (x_t) {  // [k, rows] -> [rows, k]
    PSSA_RETURN_IF(dxt.alloc(rows * k * 4, &ctx->pool));
    PSSA_RETURN_IF(pssa::launch_transpose(st, xa, dxt.as<float>(), 1, (int)k, (int)rows, 1.0f));
    xa = dxt.as<float>();
  }
  if (w_t) {  // [k, n] -> [n, k]
    PSSA_RETURN_IF(dwt.alloc(n * k * 4, &ctx->pool));
    PSSA_RETURN_IF(pssa::launch_transpose(st, wa, dwt.as<float>(), 1, (int)k, (int)n, 1.0f));
    wa = dwt.as<float>();
  }
  PSSA_RETURN_IF(dy.alloc(rows * n * 4, &ctx->pool));
  pssa::EpiParams ep;
  ep.out32 = dy.as<float>();
  ep.ld32 = (int)n;
  if (accumulate) {
    PSSA_RETURN_IF(upload(ctx, dacc, y, rows * n * 4));
    ep.kind = pssa::EPI_ADD_AUX;
    ep.aux = dacc.as<float>();
    ep.ld_aux = (int)n;
  }
  PSSA_RETURN_IF(pssa::launch_gemm(st, PSSA_HIP_F32, xa, (int)k, wa, (int)k, (int)rows, (int)n, (int)k, ep));
  PSSA_RETURN_IF(download(ctx, y, dy, rows * n * 4));
  return sync(ctx);
}

static Status gemm_dims(size_t m, size_t k, size_t n, size_t a_len, size_t b_len, size_t out_len, size_t a_exp,
                        size_t b_exp, size_t out_exp) {
  PSSA_RETURN_IF(need(m && k && n, "GEMM dimensions must be positive"));
  if (a_exp > INT32_MAX || b_exp > INT32_MAX || out_exp > INT32_MAX) return Status::Invalid("gemm: too large");
  if (a_len != a_exp || b_len != b_exp || out_len != out_exp)
    return Status::Invalid("GEMM operand lengths must be " + std::to_string(a_exp) + ", " + std::to_string(b_exp) +
                           " and " + std::to_string(out_exp));
  return Status::Ok();
}

int pssa_hip_gemm_nn(pssa_hip_ctx* ctx, const float* a, size_t a_len, const float* b, size_t b_len, size_t m,
                     size_t k, size_t n, float* out, size_t out_len, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(check_ctx(ctx));
    PSSA_RETURN_IF(need(a && b && out, "gemm: null buffer"));
    size_t ae = 0, be = 0, oe = 0;
    PSSA_RETURN_IF(pssa::checked_count({m, k}, &ae, "gemm lhs"));
    PSSA_RETURN_IF(pssa::checked_count({k, n}, &be, "gemm rhs"));
    PSSA_RETURN_IF(pssa::checked_count({m, n}, &oe, "gemm output"));
    PSSA_RETURN_IF(gemm_dims(m, k, n, a_len, b_len, out_len, ae, be, oe));
    return gemm_transposed(ctx, a, b, m, n, k, false, true, false, out);
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_gemm_tn_accumulate(pssa_hip_ctx* ctx, const float* a, size_t a_len, const float* b, size_t b_len,
                                size_t m, size_t k, size_t n, float* out, size_t out_len, char* err,
                                size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(check_ctx(ctx));
    PSSA_RETURN_IF(need(a && b && out, "gemm: null buffer"));
    size_t ae = 0, be = 0, oe = 0;
    PSSA_RETURN_IF(pssa::checked_count({m, k}, &ae, "gemm lhs"));
    PSSA_RETURN_IF(pssa::checked_count({m, n}, &be, "gemm rhs"));
    PSSA_RETURN_IF(pssa::checked_count({k, n}, &oe, "gemm output"));
    PSSA_RETURN_IF(gemm_dims(m, k, n, a_len, b_len, out_len, ae, be, oe));
    // C(K,N) += A^T B: rows = K, reduction over M; A [M,K] and B [M,N] both
    // arrive reduction-major.
    return gemm_transposed(ctx, a, b, k, n, m, true, true, true, out);
  };
  return pssa::finish(body(), err, err_len);
}

void pssa_hip_invalidate_weights(pssa_hip_ctx* ctx) {
  if (!ctx) return;
  std::lock_guard<std::mutex> g(ctx->mu);
  for (auto& kv : ctx->weights) kv.second.current = false;
}

int pssa_hip_invalidate_weights_only(pssa_hip_ctx* ctx, const pssa_hip_weight_key* keys, size_t n_keys,
                                     char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(check_ctx(ctx));
    PSSA_RETURN_IF(need(keys || n_keys == 0, "null weight keys"));
    std::lock_guard<std::mutex> g(ctx->mu);
    for (auto& kv : ctx->weights)
      for (size_t i = 0; i < n_keys; ++i)
        if (std::get<0>(kv.first) == (uintptr_t)keys[i].ptr && std::get<1>(kv.first) == keys[i].len)
          kv.second.current = false;
    return Status::Ok();
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_weight_cache_stats(pssa_hip_ctx* ctx, size_t* entries, size_t* current, size_t* bytes) {
  if (!ctx) return PSSA_HIP_EINVAL;
  std::lock_guard<std::mutex> g(ctx->mu);
  size_t e = 0, c = 0, b = 0;
  for (const auto& kv : ctx->weights) {
    ++e;
    c += kv.second.current ? 1 : 0;
    b += kv.second.buf.bytes;
  }
  if (entries) *entries = e;
  if (current) *current = c;
  if (bytes) *bytes = b;
  return PSSA_HIP_OK;
}

int pssa_hip_softplus_in_place(pssa_hip_ctx* ctx, float* values, size_t len, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(check_ctx(ctx));
    PSSA_RETURN_IF(need(values || len == 0, "softplus: null buffer"));
    if (len == 0) return Status::Ok();
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    DevBuf dv;
    PSSA_RETURN_IF(upload(ctx, dv, values, len * 4));
    PSSA_RETURN_IF(pssa::launch_softplus(ctx->stream, dv.as<float>(), len));
    PSSA_RETURN_IF(download(ctx, values, dv, len * 4));
    return sync(ctx);
  };
  return pssa::finish(body(), err, err_len);
}

// -------------------------------------------------------------- SSM stage
// Device results of one stage-API scan (the reference's SSM tape fields,
// src/gpu_batch.rs:392-437): y [L,d], the final carry (state-major [s,d]),
// and when materialised bar_a, bar_b [L*d*s] and states [(L+1)*d*s].
struct SsmTape {
  size_t L = 0, d = 0, s = 0;
  DevBuf y, carry, carry_ds, bar_a, bar_b, states;
};

static Status check_ssm_shapes(size_t seq_len, size_t d_m, size_t d_s, size_t delta_len, size_t b_len,
                               size_t x_len, size_t rates_len, size_t c_len, size_t initial_len) {
  PSSA_RETURN_IF(need(seq_len && d_m && d_s, "ssm: dimensions must be positive"));
  size_t ld = 0, ls = 0, w = 0, lw1 = 0;
  PSSA_RETURN_IF(pssa::checked_count({seq_len, d_m}, &ld, "ssm"));
  PSSA_RETURN_IF(pssa::checked_count({seq_len, d_s}, &ls, "ssm"));
  PSSA_RETURN_IF(pssa::checked_count({d_m, d_s}, &w, "ssm"));
  PSSA_RETURN_IF(pssa::checked_count({seq_len + 1, w}, &lw1, "ssm"));
  if (delta_len != ld || x_len != ld) return Status::Invalid("ssm: delta/x_norm/y_ssm must be seq_len*d_m");
  if (b_len != ls || c_len != ls) return Status::Invalid("ssm: b_proj/c_proj must be seq_len*d_s");
  if (rates_len != w || initial_len != w) return Status::Invalid("ssm: rates/initial must be d_m*d_s");
  if (seq_len > INT32_MAX || d_m > INT32_MAX || d_s > INT32_MAX) return Status::Invalid("ssm: too large");
  return Status::Ok();
}

// Runs the scan of the stage API into `t` (called with ctx->mu held).
static Status run_stage_ssm(pssa_hip_ctx* ctx, const float* delta, const float* b_proj, const float* x_norm,
                            const float* rates, const float* c_proj, const float* initial, size_t seq_len,
                            size_t d_m, size_t d_s, bool materialize, SsmTape& t) {
  const hipStream_t st = ctx->stream;
  const size_t ld = seq_len * d_m, ls = seq_len * d_s, w = d_m * d_s;
  t.L = seq_len;
  t.d = d_m;
  t.s = d_s;
  DevBuf dd, db, dx, dr, dc, dr2;
  PSSA_RETURN_IF(upload(ctx, dd, delta, ld * 4));
  PSSA_RETURN_IF(upload(ctx, db, b_proj, ls * 4));
  PSSA_RETURN_IF(upload(ctx, dx, x_norm, ld * 4));
  PSSA_RETURN_IF(upload(ctx, dr, rates, w * 4));
  PSSA_RETURN_IF(upload(ctx, dc, c_proj, ls * 4));
  PSSA_RETURN_IF(upload(ctx, t.carry_ds, initial, w * 4));
  PSSA_RETURN_IF(t.y.alloc(ld * 4, &ctx->pool));
  // The scan keeps rates state-major ([s, d]) and states channel-blocked
  // (pssa::carry_at); the stage API speaks the reference's [d, s].
  PSSA_RETURN_IF(dr2.alloc(w * 4, &ctx->pool));
  PSSA_RETURN_IF(t.carry.alloc(w * 4, &ctx->pool));
  PSSA_RETURN_IF(pssa::launch_transpose(st, dr.as<float>(), dr2.as<float>(), 1, (int)d_m, (int)d_s,
                                        1.4426950408889634f));
  PSSA_RETURN_IF(pssa::launch_carry_convert(st, t.carry_ds.as<float>(), t.carry.as<float>(), 1, (int)d_m, (int)d_s,
                                            true));
  PSSA_RETURN_IF(pssa::launch_fill_zero(st, t.y.as<float>(), ld));
  pssa::SsmArgs a;
  a.delta = dd.as<float>();
  a.ld_delta = (int)d_m;
  a.bproj = db.as<float>();
  a.ld_b = (int)d_s;
  a.cproj = dc.as<float>();
  a.ld_c = (int)d_s;
  a.xn = dx.as<float>();
  a.ld_x = (int)d_m;
  a.rates2 = dr2.as<float>();
  a.carry = t.carry.as<float>();
  a.carry_stride = (long)w;
  a.y = t.y.as<float>();
  a.ld_y = (int)d_m;
  a.T = (int)seq_len;
  a.d = (int)d_m;
  a.s = (int)d_s;
  a.lanes = 1;
  DevBuf dpart;
  const int nz = pssa::ssm_state_blocks((int)d_s);
  if (!materialize && nz > 2) {
    PSSA_RETURN_IF(dpart.alloc((size_t)nz * ld * 4, &ctx->pool));
    a.y_part = dpart.as<float>();
  }
  if (materialize) {
    PSSA_RETURN_IF(t.bar_a.alloc(seq_len * w * 4, &ctx->pool));
    PSSA_RETURN_IF(t.bar_b.alloc(seq_len * w * 4, &ctx->pool));
    PSSA_RETURN_IF(t.states.alloc((seq_len + 1) * w * 4, &ctx->pool));
    a.bar_a = t.bar_a.as<float>();
    a.bar_b = t.bar_b.as<float>();
    a.states = t.states.as<float>();
  }
  PSSA_RETURN_IF(pssa::launch_ssm_scan(st, a));
  // Sources of the scan's inputs are freed at return: finish first.
  return sync(ctx);
}

// Copies the tape's host outputs (any may be NULL).
static Status download_ssm(pssa_hip_ctx* ctx, SsmTape& t, float* bar_a, float* bar_b, float* states, float* y_ssm,
                           float* final_state) {
  const hipStream_t st = ctx->stream;
  const size_t ld = t.L * t.d, w = t.d * t.s;
  if (y_ssm) PSSA_RETURN_IF(download(ctx, y_ssm, t.y, ld * 4));
  if (final_state) {
    PSSA_RETURN_IF(pssa::launch_carry_convert(st, t.carry.as<float>(), t.carry_ds.as<float>(), 1, (int)t.d, (int)t.s,
                                              false));
    PSSA_RETURN_IF(download(ctx, final_state, t.carry_ds, w * 4));
  }
  if (bar_a) PSSA_RETURN_IF(download(ctx, bar_a, t.bar_a, t.L * w * 4));
  if (bar_b) PSSA_RETURN_IF(download(ctx, bar_b, t.bar_b, t.L * w * 4));
  if (states) PSSA_RETURN_IF(download(ctx, states, t.states, (t.L + 1) * w * 4));
  return sync(ctx);
}

int pssa_hip_ssm_forward(pssa_hip_ctx* ctx, const float* delta, size_t delta_len,
                         const float* delta_raw, const float* b_proj, size_t b_len,
                         const float* x_norm, size_t x_len, const float* rates, size_t rates_len,
                         const float* rate_deriv, const float* c_proj, size_t c_len,
                         const float* initial, size_t initial_len, size_t seq_len, size_t d_m,
                         size_t d_s, float* bar_a, float* bar_b, float* states, float* y_ssm,
                         size_t y_len, float* final_state, char* err, size_t err_len) {
  (void)delta_raw;
  (void)rate_deriv;
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(check_ctx(ctx));
    PSSA_RETURN_IF(need(delta && b_proj && x_norm && rates && c_proj && initial && y_ssm, "ssm: null input"));
    PSSA_RETURN_IF(need((bar_a == nullptr) == (bar_b == nullptr) && (bar_a == nullptr) == (states == nullptr),
                        "ssm: bar_a, bar_b and states are materialised together"));
    PSSA_RETURN_IF(check_ssm_shapes(seq_len, d_m, d_s, delta_len, b_len, x_len, rates_len, c_len, initial_len));
    PSSA_RETURN_IF(need(y_len == seq_len * d_m, "ssm: delta/x_norm/y_ssm must be seq_len*d_m"));
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    SsmTape t;
    PSSA_RETURN_IF(run_stage_ssm(ctx, delta, b_proj, x_norm, rates, c_proj, initial, seq_len, d_m, d_s,
                                 bar_a != nullptr, t));
    return download_ssm(ctx, t, bar_a, bar_b, states, y_ssm, final_state);
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_ssm_forward_resident(pssa_hip_ctx* ctx, const float* delta, size_t delta_len, const float* delta_raw,
                                  const float* b_proj, size_t b_len, const float* x_norm, size_t x_len,
                                  const float* rates, size_t rates_len, const float* c_proj, size_t c_len,
                                  const float* initial, size_t initial_len, size_t seq_len, size_t d_m,
                                  size_t d_s, char* err, size_t err_len) {
  (void)delta_raw;
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(check_ctx(ctx));
    PSSA_RETURN_IF(need(delta && b_proj && x_norm && rates && c_proj && initial, "ssm: null input"));
    PSSA_RETURN_IF(check_ssm_shapes(seq_len, d_m, d_s, delta_len, b_len, x_len, rates_len, c_len, initial_len));
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    ctx->ssm_tape.reset();
    auto t = std::make_shared<SsmTape>();
    PSSA_RETURN_IF(run_stage_ssm(ctx, delta, b_proj, x_norm, rates, c_proj, initial, seq_len, d_m, d_s, true, *t));
    ctx->ssm_tape = t;
    return Status::Ok();
  };
  return pssa::finish(body(), err, err_len);
}

// ----------------------------------------------------------- memory stage
static Status check_memory_args(size_t seq_len, size_t d_m, size_t d_k, size_t d_val, size_t capacity,
                                size_t count, float tau, size_t top_k) {
  PSSA_RETURN_IF(need(seq_len && d_m && d_k && d_val && capacity, "memory: dimensions must be positive"));
  PSSA_RETURN_IF(need(d_val == d_m, "memory: the model path reads values of width d_latent"));
  PSSA_RETURN_IF(need(count <= capacity, "memory: count exceeds capacity"));
  PSSA_RETURN_IF(need(top_k <= (size_t)pssa::kMaxTopK, "memory: top_k must be at most 64"));
  PSSA_RETURN_IF(need(std::isfinite(tau) && tau > 0.0f, "tau must be positive and finite"));
  if (seq_len > INT32_MAX / 4 || d_m > 16384 || d_k > 4096 || capacity > 8192)
    return Status::Invalid("memory: shape exceeds the supported range");
  return Status::Ok();
}

// The memory stage of the stage API on the device copy `dy` of y_ssm
// (called with ctx->mu held).
static Status run_stage_memory(pssa_hip_ctx* ctx, const float* x_norm, const float* dy_ptr, const float* w_qx,
                               const float* w_qh, const float* w_gate, const float* w_proj, const float* keys,
                               const float* norm_sq, const float* values, size_t seq_len, size_t d_m,
                               size_t d_k, size_t capacity, size_t count, float tau, size_t top_k,
                               float* q_euc, float* q_pnc, float* q_norm, float* weights, float* m_val,
                               float* g_mem, float* m_proj, float* m_inj) {
  const hipStream_t st = ctx->stream;
  const int L = (int)seq_len, d = (int)d_m, k = (int)d_k, C = (int)capacity;
  DevBuf dx, dwqx, dwqh, dwg, dwp, dk_, dn, dv, dvt, qx, qe, qp, qn, wts, mv, gm, mp, mi;
  PSSA_RETURN_IF(upload(ctx, dx, x_norm, (size_t)L * d * 4));
  PSSA_RETURN_IF(upload(ctx, dwqx, w_qx, (size_t)k * d * 4));
  PSSA_RETURN_IF(upload(ctx, dwqh, w_qh, (size_t)k * d * 4));
  PSSA_RETURN_IF(upload(ctx, dwg, w_gate, (size_t)d * d * 4));
  PSSA_RETURN_IF(upload(ctx, dwp, w_proj, (size_t)d * d * 4));
  PSSA_RETURN_IF(upload(ctx, dk_, keys, (size_t)C * k * 4));
  PSSA_RETURN_IF(upload(ctx, dn, norm_sq, (size_t)C * 4));
  PSSA_RETURN_IF(upload(ctx, dv, values, (size_t)C * d * 4));
  std::vector<float> vt((size_t)d * C);
  for (int s2 = 0; s2 < C; ++s2)
    for (int j = 0; j < d; ++j) vt[(size_t)j * C + s2] = values[(size_t)s2 * d + j];
  PSSA_RETURN_IF(upload(ctx, dvt, vt.data(), vt.size() * 4));
  for (DevBuf* b : {&qx, &qe, &qp}) PSSA_RETURN_IF(b->alloc((size_t)L * k * 4, &ctx->pool));
  PSSA_RETURN_IF(qn.alloc((size_t)L * 4, &ctx->pool));
  PSSA_RETURN_IF(wts.alloc((size_t)L * C * 4, &ctx->pool));
  for (DevBuf* b : {&mv, &gm, &mp, &mi}) PSSA_RETURN_IF(b->alloc((size_t)L * d * 4, &ctx->pool));
  // q_euc = x W_qx^T + y W_qh^T, as dot(row_x, x) + dot(row_h, y) (src/pssa.rs:1147-1152).
  pssa::EpiParams ex;
  ex.out32 = qx.as<float>();
  ex.ld32 = k;
  PSSA_RETURN_IF(pssa::launch_gemm(st, PSSA_HIP_F32, dx.p, d, dwqx.p, d, L, k, d, ex));
  pssa::EpiParams eq;
  eq.kind = pssa::EPI_ADD_AUX;
  eq.aux = qx.as<float>();
  eq.ld_aux = k;
  eq.out32 = qe.as<float>();
  eq.ld32 = k;
  PSSA_RETURN_IF(pssa::launch_gemm(st, PSSA_HIP_F32, dy_ptr, d, dwqh.p, d, L, k, d, eq));
  pssa::RetrieveArgs ra;
  ra.q = qe.as<float>();
  ra.ld_q = k;
  ra.project = 1;
  ra.q_pnc = qp.as<float>();
  ra.q_norm = qn.as<float>();
  ra.keys = dk_.as<float>();
  ra.norm_sq = dn.as<float>();
  ra.values = dv.as<float>();
  ra.n = L;
  ra.dk = k;
  ra.dv = d;
  ra.capacity = C;
  ra.count = (int)count;
  ra.tau = tau;
  ra.top_k = (int)top_k;
  ra.weights = wts.as<float>();
  const bool sparse = top_k > 0 && top_k < count;
  if (sparse) ra.out_val = mv.as<float>();
  PSSA_RETURN_IF(pssa::launch_retrieve(st, ra));
  if (!sparse) {
    if (count > 0) {
      pssa::EpiParams em;
      em.out32 = mv.as<float>();
      em.ld32 = d;
      PSSA_RETURN_IF(pssa::launch_gemm(st, PSSA_HIP_F32, wts.p, C, dvt.p, C, L, d, (int)count, em));
    } else {
      PSSA_RETURN_IF(pssa::launch_fill_zero(st, mv.as<float>(), (size_t)L * d));
    }
  }
  pssa::EpiParams eg;
  eg.kind = pssa::EPI_SEGMENTS;
  eg.seg[0] = 0;
  eg.seg[1] = 0;
  eg.seg[2] = d;
  eg.seg[3] = d;
  eg.out32 = gm.as<float>();
  eg.ld32 = d;
  PSSA_RETURN_IF(pssa::launch_gemm(st, PSSA_HIP_F32, dx.p, d, dwg.p, d, L, d, d, eg));
  pssa::EpiParams ep2;
  ep2.out32 = mp.as<float>();
  ep2.ld32 = d;
  PSSA_RETURN_IF(pssa::launch_gemm(st, PSSA_HIP_F32, mv.p, d, dwp.p, d, L, d, d, ep2));
  PSSA_RETURN_IF(pssa::launch_mul(st, gm.as<float>(), mp.as<float>(), mi.as<float>(), (size_t)L * d));
  if (q_euc) PSSA_RETURN_IF(download(ctx, q_euc, qe, (size_t)L * k * 4));
  if (q_pnc) PSSA_RETURN_IF(download(ctx, q_pnc, qp, (size_t)L * k * 4));
  if (q_norm) PSSA_RETURN_IF(download(ctx, q_norm, qn, (size_t)L * 4));
  if (weights) PSSA_RETURN_IF(download(ctx, weights, wts, (size_t)L * C * 4));
  if (m_val) PSSA_RETURN_IF(download(ctx, m_val, mv, (size_t)L * d * 4));
  if (g_mem) PSSA_RETURN_IF(download(ctx, g_mem, gm, (size_t)L * d * 4));
  if (m_proj) PSSA_RETURN_IF(download(ctx, m_proj, mp, (size_t)L * d * 4));
  PSSA_RETURN_IF(download(ctx, m_inj, mi, (size_t)L * d * 4));
  return sync(ctx);
}

int pssa_hip_memory_forward(pssa_hip_ctx* ctx, const float* x_norm, const float* y_ssm,
                            const float* w_qx, const float* w_qh, const float* w_gate,
                            const float* w_proj, const float* keys, const float* norm_sq,
                            const float* values, size_t seq_len, size_t d_m, size_t d_k,
                            size_t d_val, size_t capacity, size_t count, float tau, size_t top_k,
                            float* q_euc, float* q_pnc, float* q_norm, float* weights,
                            float* m_val, float* g_mem, float* m_proj, float* m_inj, char* err,
                            size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(check_ctx(ctx));
    PSSA_RETURN_IF(check_memory_args(seq_len, d_m, d_k, d_val, capacity, count, tau, top_k));
    PSSA_RETURN_IF(need(x_norm && y_ssm && w_qx && w_qh && w_gate && w_proj && keys && norm_sq &&
                            values && m_inj,
                        "memory: null input"));
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    DevBuf dy;
    PSSA_RETURN_IF(upload(ctx, dy, y_ssm, seq_len * d_m * 4));
    return run_stage_memory(ctx, x_norm, dy.as<float>(), w_qx, w_qh, w_gate, w_proj, keys, norm_sq, values,
                            seq_len, d_m, d_k, capacity, count, tau, top_k, q_euc, q_pnc, q_norm, weights, m_val,
                            g_mem, m_proj, m_inj);
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_memory_forward_after_ssm(pssa_hip_ctx* ctx, const float* x_norm, const float* w_qx,
                                      const float* w_qh, const float* w_gate, const float* w_proj,
                                      const float* keys, const float* norm_sq, const float* values,
                                      size_t seq_len, size_t d_m, size_t d_k, size_t d_val, size_t capacity,
                                      size_t count, float tau, size_t top_k, float* bar_a, float* bar_b,
                                      float* states, float* y_ssm, float* q_euc, float* q_pnc, float* q_norm,
                                      float* weights, float* m_val, float* g_mem, float* m_proj, float* m_inj,
                                      char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(check_ctx(ctx));
    PSSA_RETURN_IF(check_memory_args(seq_len, d_m, d_k, d_val, capacity, count, tau, top_k));
    PSSA_RETURN_IF(need(x_norm && w_qx && w_qh && w_gate && w_proj && keys && norm_sq && values && m_inj,
                        "memory: null input"));
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_RETURN_IF(need(ctx->ssm_tape && ctx->ssm_tape->L == seq_len && ctx->ssm_tape->d == d_m,
                        "memory_forward_after_ssm: no resident SSM tape of this shape "
                        "(pssa_hip_ssm_forward_resident comes first)"));
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    std::shared_ptr<SsmTape> t = std::move(ctx->ssm_tape);  // consumed by this call
    PSSA_RETURN_IF(run_stage_memory(ctx, x_norm, t->y.as<float>(), w_qx, w_qh, w_gate, w_proj, keys, norm_sq,
                                    values, seq_len, d_m, d_k, capacity, count, tau, top_k, q_euc, q_pnc, q_norm,
                                    weights, m_val, g_mem, m_proj, m_inj));
    return download_ssm(ctx, *t, bar_a, bar_b, states, y_ssm, nullptr);
  };
  return pssa::finish(body(), err, err_len);
}

}  // extern "C"

// Grows the context's scratch to `bytes`.  Called with ctx->mu held; the
// previous buffer is released only once the stream has drained.  Where the
// caller can do without (`optional`) it stays when there is no memory.
static Status grow_scratch(pssa_hip_ctx* ctx, size_t bytes, bool optional) {
  if (ctx->scratch_bytes >= bytes) return Status::Ok();
  PSSA_HIP_TRY(hipStreamSynchronize(ctx->stream));
  void* p = nullptr;
  if (optional && pssa::device_malloc(&p, bytes) != hipSuccess) return Status::Ok();
  if (ctx->scratch) PSSA_HIP_TRY(hipFree(ctx->scratch));
  ctx->scratch = nullptr;
  ctx->scratch_bytes = 0;
  if (!p) PSSA_HIP_TRY(pssa::device_malloc(&p, bytes));
  ctx->scratch = p;
  ctx->scratch_bytes = bytes;
  return Status::Ok();
}

// Points ra.scratch at the context's scratch, grown to what the launch needs.
// Called with ctx->mu held.  A full soft read runs without where there is no
// memory.
static Status bind_retrieve_scratch(pssa_hip_ctx* ctx, pssa::RetrieveArgs& ra) {
  const size_t need_bytes = pssa::retrieve_scratch_bytes(ra);
  if (!need_bytes) return Status::Ok();
  PSSA_RETURN_IF(grow_scratch(ctx, need_bytes, !pssa::retrieve_needs_scratch(ra)));
  ra.scratch = ctx->scratch;
  ra.scratch_bytes = ctx->scratch_bytes;
  return Status::Ok();
}

// Grows the context's scratch to what the two-level dense scan needs.
// Called with ctx->mu held.
static Status bind_dense_scan_scratch(pssa_hip_ctx* ctx, int batch, int L, int s) {
  return grow_scratch(ctx, pssa::dense_scan_scratch_bytes(batch, L, s), false);
}

extern "C" {

// Host-buffer retrieval; gate/age (both or neither) select the hybrid read.
static int retrieve_host(pssa_hip_ctx* ctx, const float* q_pnc, size_t n_q, const float* keys,
                         const float* norm_sq, const float* values, size_t capacity, size_t count,
                         size_t d_key, size_t d_val, float tau, size_t top_k, const float* gate,
                         const uint64_t* age, float lam, float* out_val, float* out_min, uint32_t* out_idx,
                         float* out_weights, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(check_ctx(ctx));
    PSSA_RETURN_IF(need(n_q && d_key && d_val && capacity, "retrieve: dimensions must be positive"));
    PSSA_RETURN_IF(need(count <= capacity, "retrieve: count exceeds capacity"));
    PSSA_RETURN_IF(need(top_k <= (size_t)pssa::kMaxTopK, "retrieve: top_k must be at most 64"));
    PSSA_RETURN_IF(need(std::isfinite(tau) && tau > 0.0f, "tau must be positive and finite"));
    PSSA_RETURN_IF(need(q_pnc && keys && norm_sq && values && out_val, "retrieve: null buffer"));
    PSSA_RETURN_IF(need(!out_idx || top_k > 0, "retrieve: indices need top_k > 0"));
    const bool hybrid = gate != nullptr;
    if (hybrid) {
      PSSA_RETURN_IF(need(age != nullptr, "retrieve: the hybrid read needs gates and ages"));
      PSSA_RETURN_IF(need(std::isfinite(lam) && lam > 0.0f && lam <= 1.0f, "hybrid decay lam must be in (0.0, 1.0]"));
      for (size_t q = 0; q < count; ++q)
        PSSA_RETURN_IF(need(std::isfinite(gate[q]) && gate[q] >= 0.0f,
                            "hybrid write gate must be finite and nonnegative"));
    }
    if (n_q > INT32_MAX / 4 || d_key > 4096 || d_val > 65536 || capacity > 8192)
      return Status::Invalid("retrieve: shape exceeds the supported range");
    // The query must lie in the open ball (retrieve_soft_into's assertion).
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    const hipStream_t st = ctx->stream;
    DevBuf dq, dk_, dn, dv, dval, dmin, didx, dw, dg, da;
    PSSA_RETURN_IF(upload(ctx, dq, q_pnc, n_q * d_key * 4));
    PSSA_RETURN_IF(upload(ctx, dk_, keys, capacity * d_key * 4));
    PSSA_RETURN_IF(upload(ctx, dn, norm_sq, capacity * 4));
    PSSA_RETURN_IF(upload(ctx, dv, values, capacity * d_val * 4));
    if (hybrid && count > 0) {
      PSSA_RETURN_IF(upload(ctx, dg, gate, count * 4));
      PSSA_RETURN_IF(upload(ctx, da, age, count * 8));
    }
    PSSA_RETURN_IF(dval.alloc(n_q * d_val * 4, &ctx->pool));
    if (out_min) PSSA_RETURN_IF(dmin.alloc(n_q * 4, &ctx->pool));
    if (out_idx) PSSA_RETURN_IF(didx.alloc(n_q * top_k * 4, &ctx->pool));
    if (out_weights) PSSA_RETURN_IF(dw.alloc(n_q * capacity * 4, &ctx->pool));
    pssa::RetrieveArgs ra;
    ra.q = dq.as<float>();
    ra.ld_q = (int)d_key;
    ra.project = 0;
    ra.keys = dk_.as<float>();
    ra.norm_sq = dn.as<float>();
    ra.values = dv.as<float>();
    ra.n = (int)n_q;
    ra.dk = (int)d_key;
    ra.dv = (int)d_val;
    ra.capacity = (int)capacity;
    ra.count = (int)count;
    ra.tau = tau;
    ra.top_k = (int)top_k;
    ra.weights = out_weights ? dw.as<float>() : nullptr;
    ra.out_val = dval.as<float>();
    ra.out_min = out_min ? dmin.as<float>() : nullptr;
    ra.out_idx = out_idx ? didx.as<uint32_t>() : nullptr;
    if (hybrid && count > 0) {
      ra.hgate = dg.as<float>();
      ra.hage = da.as<unsigned long long>();
      ra.log_lam = std::log((double)lam);
    }
    PSSA_RETURN_IF(bind_retrieve_scratch(ctx, ra));
    PSSA_RETURN_IF(pssa::launch_retrieve(st, ra));
    PSSA_RETURN_IF(download(ctx, out_val, dval, n_q * d_val * 4));
    if (out_min) PSSA_RETURN_IF(download(ctx, out_min, dmin, n_q * 4));
    if (out_idx) PSSA_RETURN_IF(download(ctx, out_idx, didx, n_q * top_k * 4));
    if (out_weights) PSSA_RETURN_IF(download(ctx, out_weights, dw, n_q * capacity * 4));
    return sync(ctx);
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_retrieve(pssa_hip_ctx* ctx, const float* q_pnc, size_t n_q, const float* keys,
                      const float* norm_sq, const float* values, size_t capacity, size_t count,
                      size_t d_key, size_t d_val, float tau, size_t top_k, float* out_val,
                      float* out_min, uint32_t* out_idx, float* out_weights, char* err, size_t err_len) {
  return retrieve_host(ctx, q_pnc, n_q, keys, norm_sq, values, capacity, count, d_key, d_val, tau, top_k,
                       nullptr, nullptr, 1.0f, out_val, out_min, out_idx, out_weights, err, err_len);
}

int pssa_hip_retrieve_hybrid(pssa_hip_ctx* ctx, const float* q_pnc, size_t n_q, const float* keys,
                             const float* norm_sq, const float* values, size_t capacity, size_t count,
                             size_t d_key, size_t d_val, float tau, size_t top_k, const float* gate,
                             const uint64_t* age, float lam, float* out_val, float* out_min,
                             uint32_t* out_idx, float* out_weights, char* err, size_t err_len) {
  if (!gate || !age) {
    if (err && err_len) std::snprintf(err, err_len, "retrieve: the hybrid read needs gates and ages");
    return PSSA_HIP_EINVAL;
  }
  return retrieve_host(ctx, q_pnc, n_q, keys, norm_sq, values, capacity, count, d_key, d_val, tau, top_k, gate,
                       age, lam, out_val, out_min, out_idx, out_weights, err, err_len);
}

// Device-buffer retrieval.  no_alloc: the ranked path's scratch is the
// device's static array (kNoallocChunk queries per pass) instead of the
// context's grown buffer, so nothing is allocated.
static int retrieve_resident(pssa_hip_ctx* ctx, const float* d_q_pnc, size_t n_q, const float* d_keys,
                             const float* d_norm_sq, const float* d_values, size_t capacity, size_t count,
                             size_t d_key, size_t d_val, float tau, size_t top_k, float* d_out_val,
                             float* d_out_min, uint32_t* d_out_idx, bool no_alloc, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(check_ctx(ctx));
    PSSA_RETURN_IF(need(n_q && d_key && d_val && capacity, "retrieve: dimensions must be positive"));
    PSSA_RETURN_IF(need(count <= capacity, "retrieve: count exceeds capacity"));
    PSSA_RETURN_IF(need(top_k <= (size_t)pssa::kMaxTopK, "retrieve: top_k must be at most 64"));
    PSSA_RETURN_IF(need(std::isfinite(tau) && tau > 0.0f, "tau must be positive and finite"));
    PSSA_RETURN_IF(need(d_q_pnc && d_keys && d_norm_sq && d_values && d_out_val, "retrieve: null buffer"));
    PSSA_RETURN_IF(need(!d_out_idx || top_k > 0, "retrieve: indices need top_k > 0"));
    if (n_q > INT32_MAX / 4 || d_key > 4096 || d_val > 65536 || capacity > 8192)
      return Status::Invalid("retrieve: shape exceeds the supported range");
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    pssa::RetrieveArgs ra;
    ra.q = d_q_pnc;
    ra.ld_q = (int)d_key;
    ra.project = 0;
    ra.keys = d_keys;
    ra.norm_sq = d_norm_sq;
    ra.values = d_values;
    ra.n = (int)n_q;
    ra.dk = (int)d_key;
    ra.dv = (int)d_val;
    ra.capacity = (int)capacity;
    ra.count = (int)count;
    ra.tau = tau;
    ra.top_k = (int)top_k;
    ra.out_val = d_out_val;
    ra.out_min = d_out_min;
    ra.out_idx = d_out_idx;
    if (no_alloc) {
      ra.chunk = pssa::kNoallocChunk;
      const size_t need_bytes = pssa::retrieve_scratch_bytes(ra);
      if (need_bytes > pssa::kNoallocScratchBytes)
        return Status::Invalid("retrieve (allocation-free): needs " + std::to_string(need_bytes) +
                               " bytes of scratch, the static scratch holds " +
                               std::to_string(pssa::kNoallocScratchBytes));
      if (!ctx->noalloc_scratch) return Status::Device("retrieve (allocation-free): scratch address unresolved");
      ra.scratch = ctx->noalloc_scratch;
      ra.scratch_bytes = pssa::kNoallocScratchBytes;
    } else {
      PSSA_RETURN_IF(bind_retrieve_scratch(ctx, ra));
    }
    return pssa::launch_retrieve(ctx->stream, ra);
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_retrieve_resident(pssa_hip_ctx* ctx, const float* d_q_pnc, size_t n_q, const float* d_keys,
                               const float* d_norm_sq, const float* d_values, size_t capacity,
                               size_t count, size_t d_key, size_t d_val, float tau, size_t top_k,
                               float* d_out_val, float* d_out_min, uint32_t* d_out_idx,
                               char* err, size_t err_len) {
  return retrieve_resident(ctx, d_q_pnc, n_q, d_keys, d_norm_sq, d_values, capacity, count, d_key, d_val, tau,
                           top_k, d_out_val, d_out_min, d_out_idx, false, err, err_len);
}

int pssa_hip_retrieve_resident_noalloc(pssa_hip_ctx* ctx, const float* d_q_pnc, size_t n_q, const float* d_keys,
                                       const float* d_norm_sq, const float* d_values, size_t capacity,
                                       size_t count, size_t d_key, size_t d_val, float tau, size_t top_k,
                                       float* d_out_val, float* d_out_min, uint32_t* d_out_idx, char* err,
                                       size_t err_len) {
  return retrieve_resident(ctx, d_q_pnc, n_q, d_keys, d_norm_sq, d_values, capacity, count, d_key, d_val, tau,
                           top_k, d_out_val, d_out_min, d_out_idx, true, err, err_len);
}

// ------------------------------------------------------------------ model
int pssa_hip_model_load(pssa_hip_ctx* ctx, const pssa_hip_weights* w, int weight_dtype,
                        pssa_hip_model** out, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(check_ctx(ctx));
    PSSA_RETURN_IF(need(out != nullptr, "null output handle"));
    *out = nullptr;
    PSSA_RETURN_IF(need(w && w->embed && w->unembed && w->blocks, "weights: null pointer"));
    PSSA_RETURN_IF(need(weight_dtype == PSSA_HIP_F32 || weight_dtype == PSSA_HIP_BF16, "unknown weight dtype"));
    const pssa_hip_config& c = w->cfg;
    PSSA_RETURN_IF(check_config(c));
    const size_t V = c.d_vocab, d = c.d_latent, s = c.d_state, k = c.d_mem_key, C = c.mem_capacity,
                 r = c.adapter_rank;
    for (size_t l = 0; l < c.depth; ++l) {
      const pssa_hip_block& b = w->blocks[l];
      PSSA_RETURN_IF(need(b.norm_gamma && b.norm_beta && b.a_raw && b.w_delta && b.w_b && b.w_c &&
                              b.w_qx && b.w_qh && b.w_gate && b.w_proj && b.adapter_down &&
                              b.adapter_up && b.adapter_slow && b.mlp_w1 && b.mlp_w2 && b.mem_keys &&
                              b.mem_values && b.mem_norm_sq,
                          "weights: null block tensor"));
      PSSA_RETURN_IF(need(b.mem_count <= C, "memory count exceeds capacity"));
      PSSA_RETURN_IF(need(std::isfinite(b.mem_value_cap) && b.mem_value_cap >= 0.0f,
                          "memory value cap must be positive and finite"));
      PSSA_RETURN_IF(need(b.mem_top_k <= (uint64_t)pssa::kMaxTopK, "memory top-k above 64 is not supported"));
      if (b.mem_hybrid_enabled)
        PSSA_RETURN_IF(need(std::isfinite(b.mem_hybrid_lam) && b.mem_hybrid_lam > 0.0f && b.mem_hybrid_lam <= 1.0f,
                            "hybrid decay lam must be in (0.0, 1.0]"));
      if (b.mem_hybrid_gate)
        for (size_t q = 0; q < b.mem_count; ++q)
          PSSA_RETURN_IF(need(std::isfinite(b.mem_hybrid_gate[q]) && b.mem_hybrid_gate[q] >= 0.0f,
                              "hybrid write gate must be finite and nonnegative"));
      for (size_t q = 0; q < b.mem_count; ++q)
        PSSA_RETURN_IF(need(std::isfinite(b.mem_norm_sq[q]) && b.mem_norm_sq[q] >= 0.0f && b.mem_norm_sq[q] < 1.0f,
                            "memory key norms must lie in [0, 1)"));
    }
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    const hipStream_t st = ctx->stream;
    auto m = std::make_unique<pssa_hip_model>();
    m->ctx = ctx;
    m->cfg = c;
    m->dtype = weight_dtype;
    m->n_in = 2 * d + 2 * s + k + r;
    PSSA_RETURN_IF(upload_keep(ctx, m->embed, w->embed, V * d * 4));
    PSSA_RETURN_IF(upload_weight(ctx, m->unembed, w->unembed, V * d, weight_dtype));
    m->blocks.resize(c.depth);
    std::vector<float> tmp;
    for (size_t l = 0; l < c.depth; ++l) {
      const pssa_hip_block& b = w->blocks[l];
      pssa::DevBlock& B = m->blocks[l];
      // Fused input projection rows: W_delta | W_B | W_C | W_qx | W_gate | D.
      tmp.assign(m->n_in * d, 0.0f);
      float* p = tmp.data();
      auto put = [&](const float* src, size_t rows) {
        std::memcpy(p, src, rows * d * 4);
        p += rows * d;
      };
      put(b.w_delta, d);
      put(b.w_b, s);
      put(b.w_c, s);
      put(b.w_qx, k);
      put(b.w_gate, d);
      put(b.adapter_down, r);
      PSSA_RETURN_IF(upload_weight(ctx, B.w_in, tmp.data(), tmp.size(), weight_dtype));
      PSSA_RETURN_IF(upload_weight(ctx, B.w_qh, b.w_qh, k * d, weight_dtype));
      PSSA_RETURN_IF(upload_weight(ctx, B.w_proj, b.w_proj, d * d, weight_dtype));
      PSSA_RETURN_IF(upload_weight(ctx, B.mlp_w1, b.mlp_w1, 2 * d * d, weight_dtype));
      PSSA_RETURN_IF(upload_weight(ctx, B.mlp_w2, b.mlp_w2, d * 2 * d, weight_dtype));
      std::vector<float> ueff(d * r), rates(d * s), vt(d * C);
      for (size_t i = 0; i < d * r; ++i) ueff[i] = b.adapter_up[i] + b.adapter_slow[i];
      // State-major [s, d] for the scan.
      for (size_t i = 0; i < d; ++i)
        for (size_t j = 0; j < s; ++j) rates[j * d + i] = -softplus_host(b.a_raw[i * s + j]) * 1.4426950408889634f;
      for (size_t q = 0; q < C; ++q)
        for (size_t j = 0; j < d; ++j) vt[j * C + q] = b.mem_values[q * d + j];
      PSSA_RETURN_IF(upload_weight(ctx, B.u_eff, ueff.data(), ueff.size(), weight_dtype));
      PSSA_RETURN_IF(upload_keep(ctx, B.u_fast, b.adapter_up, d * r * 4));
      PSSA_RETURN_IF(upload_keep(ctx, B.u_slow, b.adapter_slow, d * r * 4));
      std::vector<float> conf(C, 1.0f);
      std::vector<unsigned long long> last(C, 0ull);
      if (b.mem_confidence) std::memcpy(conf.data(), b.mem_confidence, C * 4);
      if (b.mem_last_seen)
        for (size_t q = 0; q < C; ++q) last[q] = b.mem_last_seen[q];
      const int meta[2] = {(int)b.mem_count, (int)(b.mem_write_head % C)};
      std::vector<float> hg(C, 1.0f);
      std::vector<unsigned long long> ha(C, 0ull);
      if (b.mem_hybrid_gate) std::memcpy(hg.data(), b.mem_hybrid_gate, C * 4);
      if (b.mem_hybrid_age)
        for (size_t q = 0; q < C; ++q) ha[q] = b.mem_hybrid_age[q];
      B.hybrid = b.mem_hybrid_enabled != 0;
      B.lam = b.mem_hybrid_lam;
      B.top_k = (int)b.mem_top_k;
      B.value_cap = b.mem_value_cap;
      PSSA_RETURN_IF(upload_keep(ctx, B.hgate, hg.data(), C * 4));
      PSSA_RETURN_IF(upload_keep(ctx, B.hage, ha.data(), C * 8));
      PSSA_RETURN_IF(upload_keep(ctx, B.conf, conf.data(), C * 4));
      PSSA_RETURN_IF(upload_keep(ctx, B.last_seen, last.data(), C * 8));
      PSSA_RETURN_IF(upload_keep(ctx, B.meta, meta, sizeof(meta)));
      PSSA_RETURN_IF(upload_keep(ctx, B.rates2, rates.data(), rates.size() * 4));
      PSSA_RETURN_IF(upload_keep(ctx, B.gamma, b.norm_gamma, d * 4));
      PSSA_RETURN_IF(upload_keep(ctx, B.beta, b.norm_beta, d * 4));
      PSSA_RETURN_IF(upload_keep(ctx, B.keys, b.mem_keys, C * k * 4));
      PSSA_RETURN_IF(upload_keep(ctx, B.norm_sq, b.mem_norm_sq, C * 4));
      PSSA_RETURN_IF(upload_keep(ctx, B.values, b.mem_values, C * d * 4));
      PSSA_RETURN_IF(upload_weight(ctx, B.values_t, vt.data(), vt.size(), weight_dtype));
      PSSA_RETURN_IF(sync(ctx));  // host staging vectors are reused
      // Values of a capped bank are capped (a no-op for values that were).
      if (B.value_cap > 0.0f) PSSA_RETURN_IF(cap_bank_values(m.get(), {&B}, B.value_cap));
    }
    const unsigned long long step0 = 0;
    PSSA_RETURN_IF(upload_keep(ctx, m->step, &step0, 8));
    PSSA_RETURN_IF(sync(ctx));
    *out = m.release();
    return Status::Ok();
  };
  return pssa::finish(body(), err, err_len);
}

void pssa_hip_model_free(pssa_hip_model* model) {
  if (!model) return;
  (void)hipSetDevice(model->ctx->device);
  (void)hipStreamSynchronize(model->ctx->stream);
  delete model;
}

int pssa_hip_lanes_create(pssa_hip_ctx* ctx, const pssa_hip_model* model, size_t lanes,
                          size_t max_tokens, pssa_hip_lanes** out, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(check_ctx(ctx));
    PSSA_RETURN_IF(need(model && out, "null model or output handle"));
    *out = nullptr;
    PSSA_RETURN_IF(need(lanes > 0 && max_tokens >= lanes, "lanes must be positive and max_tokens >= lanes"));
    PSSA_RETURN_IF(need(max_tokens <= (1u << 24), "max_tokens exceeds 2^24"));
    const pssa_hip_config& c = model->cfg;
    const size_t d = c.d_latent, s = c.d_state, k = c.d_mem_key, C = c.mem_capacity;
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    auto L = std::make_unique<pssa_hip_lanes>();
    L->ctx = ctx;
    L->model = model;
    L->lanes = lanes;
    L->max_tokens = max_tokens;
    const size_t n = max_tokens;
    PSSA_RETURN_IF(L->carry.alloc(lanes * c.depth * d * s * 4));
    PSSA_RETURN_IF(L->ids.alloc(n * 4));
    const size_t es = model->dtype == PSSA_HIP_BF16 ? 2 : 4;  // operand element size
    PSSA_RETURN_IF(L->X.alloc(n * d * 4));
    PSSA_RETURN_IF(L->XN.alloc(n * d * 4));
    PSSA_RETURN_IF(L->P.alloc(n * model->n_in * 4));
    PSSA_RETURN_IF(L->Y.alloc(n * d * 4));
    PSSA_RETURN_IF(L->Q.alloc(n * k * 4));
    PSSA_RETURN_IF(L->Zraw.alloc(n * d * 4));
    if (es == 2) {
      PSSA_RETURN_IF(L->XNh.alloc(n * d * 2));
      PSSA_RETURN_IF(L->Yh.alloc(n * d * 2));
      PSSA_RETURN_IF(L->Zrawh.alloc(n * d * 2));
    }
    PSSA_RETURN_IF(L->Wm.alloc(n * C * es));
    PSSA_RETURN_IF(L->Mval.alloc(n * d * es));
    PSSA_RETURN_IF(L->H1.alloc(n * 2 * d * es));
    PSSA_RETURN_IF(L->logits.alloc(lanes * c.d_vocab * 4));
    const int nz = pssa::ssm_state_blocks((int)s);
    if (nz > 2) PSSA_RETURN_IF(L->Ypart.alloc((size_t)nz * n * d * 4));
    PSSA_RETURN_IF(pssa::launch_fill_zero(ctx->stream, L->carry.as<float>(), lanes * c.depth * d * s));
    PSSA_RETURN_IF(L->hist.alloc(lanes * pssa_hip_lanes::kHist * 4));
    PSSA_RETURN_IF(L->hist_n.alloc(lanes * 4));
    PSSA_RETURN_IF(L->hist_pos.alloc(lanes * 4));
    // [0] non-finite logits, [1] non-finite capped bank value, [2] invalid sampling mass
    PSSA_RETURN_IF(L->nonfinite.alloc(16));
    PSSA_RETURN_IF(clear_history(L.get()));
    PSSA_HIP_TRY(hipEventCreateWithFlags(&L->ev_fork, hipEventDisableTiming));
    PSSA_HIP_TRY(hipEventCreateWithFlags(&L->ev_tail_fork, hipEventDisableTiming));
    PSSA_HIP_TRY(hipEventCreateWithFlags(&L->ev_tail_join, hipEventDisableTiming));
    for (int g = 0; g < pssa_hip_lanes::kMaxGroups - 1; ++g) {
      PSSA_HIP_TRY(hipStreamCreateWithFlags(&L->aux_stream[g], hipStreamNonBlocking));
      PSSA_HIP_TRY(hipEventCreateWithFlags(&L->ev_first[g], hipEventDisableTiming));
      PSSA_HIP_TRY(hipEventCreateWithFlags(&L->ev_join[g], hipEventDisableTiming));
    }
    PSSA_RETURN_IF(sync(ctx));
    *out = L.release();
    return Status::Ok();
  };
  return pssa::finish(body(), err, err_len);
}

void pssa_hip_lanes_free(pssa_hip_lanes* lanes) {
  if (!lanes) return;
  (void)hipSetDevice(lanes->ctx->device);
  (void)hipStreamSynchronize(lanes->ctx->stream);
  delete lanes;
}

int pssa_hip_lanes_reset(pssa_hip_lanes* L, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(need(L != nullptr, "null lanes"));
    std::lock_guard<std::mutex> g(L->ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(L->ctx->device));
    const pssa_hip_config& c = L->model->cfg;
    PSSA_RETURN_IF(pssa::launch_fill_zero(L->ctx->stream, L->carry.as<float>(),
                                          L->lanes * c.depth * L->loops * c.d_latent * c.d_state));
    PSSA_RETURN_IF(clear_history(L));
    // No prefill logits to continue from (reset_recurrent_state is followed
    // by a fresh prefill, src/inference.rs:347-355).
    L->logit_lanes = 0;
    return sync(L->ctx);
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_lanes_get_carry(pssa_hip_lanes* L, float* out, size_t len, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(need(L && out, "null argument"));
    const pssa_hip_config& c = L->model->cfg;
    const size_t n = L->lanes * c.depth * L->loops * c.d_latent * c.d_state;
    PSSA_RETURN_IF(need(len == n, "carry length must be lanes*depth*loops*d_latent*d_state"));
    std::lock_guard<std::mutex> g(L->ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(L->ctx->device));
    DevBuf tmp;
    PSSA_RETURN_IF(tmp.alloc(n * 4, &L->ctx->pool));
    PSSA_RETURN_IF(carry_layout(L, L->carry.as<float>(), tmp.as<float>(), false));
    PSSA_RETURN_IF(download(L->ctx, out, tmp, n * 4));
    return sync(L->ctx);
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_lanes_set_carry(pssa_hip_lanes* L, const float* in, size_t len, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(need(L && in, "null argument"));
    const pssa_hip_config& c = L->model->cfg;
    const size_t n = L->lanes * c.depth * L->loops * c.d_latent * c.d_state;
    PSSA_RETURN_IF(need(len == n, "carry length must be lanes*depth*loops*d_latent*d_state"));
    std::lock_guard<std::mutex> g(L->ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(L->ctx->device));
    DevBuf tmp;
    PSSA_RETURN_IF(upload(L->ctx, tmp, in, n * 4));
    PSSA_RETURN_IF(carry_layout(L, tmp.as<float>(), L->carry.as<float>(), true));
    // The prefill logits belong to the replaced carries.
    L->logit_lanes = 0;
    return sync(L->ctx);
  };
  return pssa::finish(body(), err, err_len);
}

static Status invalid_prefix_locked(pssa_hip_lanes* L, const uint32_t* ids, size_t n_lanes, size_t T);

int pssa_hip_prefill(pssa_hip_lanes* L, const uint32_t* ids, size_t n_lanes, size_t seq_len,
                     float* logits_last, size_t logits_len, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(need(L != nullptr, "null lanes"));
    const size_t V = L->model->cfg.d_vocab;
    if (logits_last) PSSA_RETURN_IF(need(logits_len == n_lanes * V, "logits length must be n_lanes*d_vocab"));
    PSSA_RETURN_IF(need(ids != nullptr, "null ids"));
    PSSA_RETURN_IF(need(seq_len > 0, "prefill requires at least one token"));
    PSSA_RETURN_IF(need(n_lanes > 0 && n_lanes <= L->lanes, "n_lanes must be in 1..=lanes"));
    PSSA_RETURN_IF(need(n_lanes * seq_len <= L->max_tokens, "n_lanes*seq_len exceeds max_tokens"));
    std::lock_guard<std::mutex> g(L->ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(L->ctx->device));
    PSSA_RETURN_IF(invalid_prefix_locked(L, ids, n_lanes, seq_len));
    PSSA_RETURN_IF(stage_ids_locked(L, ids, n_lanes, seq_len));
    PSSA_RETURN_IF(pssa::run_prefill(L, n_lanes, seq_len));
    L->logit_lanes = n_lanes;
    if (logits_last) PSSA_RETURN_IF(download(L->ctx, logits_last, L->logits, n_lanes * V * 4));
    return sync(L->ctx);
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_forward_inference(pssa_hip_lanes* L, const uint32_t* ids, size_t n_lanes, float* logits,
                               size_t logits_len, char* err, size_t err_len) {
  return pssa_hip_prefill(L, ids, n_lanes, 1, logits, logits_len, err, err_len);
}

// Lanes of their own lengths as the device runs them: one pass over all
// rows, lane after lane, each stage once per layer (time segments of the lanes
// still running cost a pass of small launches per distinct length).  Longest
// lanes first, dealt to the concurrent lane groups of a prefill.
struct RaggedPlan {
  std::vector<size_t> order;  // launch lane -> index into the caller's lengths
  std::vector<size_t> row;    // first row of each launch lane in the packed rows
  std::vector<uint32_t> meta; // spans, last rows, positions: the upload
  pssa::RaggedRows rows;
};

// lens[i] tokens on lane lane_of[i] (0: does not run); tokens > 0.
static void plan_ragged(const pssa_hip_lanes* L, const std::vector<uint64_t>& lens, const std::vector<uint64_t>& lane_of,
                        RaggedPlan& p) {
  std::vector<size_t> sorted;
  for (size_t i = 0; i < lens.size(); ++i)
    if (lens[i] > 0) sorted.push_back(i);
  std::stable_sort(sorted.begin(), sorted.end(), [&](size_t a, size_t b) { return lens[a] > lens[b]; });
  pssa::RaggedRows& r = p.rows;
  r.max_len = lens[sorted[0]];
  r.groups = pssa::prefill_lane_groups(L, sorted.size(), r.max_len);
  for (int g = 0; g < r.groups; ++g) {
    r.lane0[g] = p.order.size();
    for (size_t i = 0; i < sorted.size(); ++i)
      if (r.groups == 1 || ((i & 3) == 0 || (i & 3) == 3) == (g == 0)) p.order.push_back(sorted[i]);
  }
  r.lane0[r.groups] = p.order.size();
  size_t row = 0;
  for (int g = 0; g < r.groups; ++g) {
    r.row0[g] = row;
    for (size_t l = r.lane0[g]; l < r.lane0[g + 1]; ++l) {
      p.row.push_back(row);
      p.meta.push_back((uint32_t)(row - r.row0[g]));
      p.meta.push_back((uint32_t)lens[p.order[l]]);
      p.meta.push_back((uint32_t)lane_of[p.order[l]]);
      row += lens[p.order[l]];
    }
  }
  r.row0[r.groups] = row;
}

// Copies the plan's metadata to the device (p.meta must stay until the
// stream is synchronised) and points the rows at it.
static Status upload_plan(pssa_hip_lanes* L, RaggedPlan& p, size_t n_last, size_t n_pos) {
  if (!L->row_meta.p) PSSA_RETURN_IF(L->row_meta.alloc((4 * L->lanes + L->max_tokens) * 4));
  const size_t n_span = 3 * p.order.size();
  PSSA_RETURN_IF(L->ctx->stage.to_device(L->row_meta.p, p.meta.data(), p.meta.size() * 4, L->ctx->stream));
  p.rows.spans = L->row_meta.as<int>();
  if (n_last) p.rows.last = L->row_meta.as<uint32_t>() + n_span;
  if (n_pos) p.rows.pos = L->row_meta.as<uint32_t>() + n_span + n_last;
  p.rows.n_lanes = n_last;
  return Status::Ok();
}

// Ragged prefill with L->ctx->mu held: lane i consumes lens[i] ids (0 leaves
// the lane untouched), packed in lane order.  Each lane's last-token logits
// end in row i of lanes->logits (lanes of length 0: undefined).
static Status ragged_locked(pssa_hip_lanes* L, const uint32_t* ids, const uint64_t* lens, size_t n_lanes) {
  size_t tokens = 0;
  std::vector<size_t> offset(n_lanes);
  std::vector<uint64_t> lens_v(lens, lens + n_lanes), lane_of(n_lanes);
  for (size_t i = 0; i < n_lanes; ++i) {
    offset[i] = tokens;
    tokens += lens[i];
    lane_of[i] = i;
  }
  if (tokens == 0) return Status::Ok();
  RaggedPlan p;
  plan_ragged(L, lens_v, lane_of, p);
  std::vector<uint32_t> ids_h(tokens);
  std::vector<uint32_t> last(n_lanes, ~0u);
  bool hybrid = false;
  for (const pssa::DevBlock& B : L->model->blocks) hybrid |= B.hybrid;
  for (size_t l = 0; l < p.order.size(); ++l) {
    const size_t i = p.order[l];
    std::memcpy(&ids_h[p.row[l]], ids + offset[i], lens[i] * 4);
    last[i] = (uint32_t)(p.row[l] + lens[i] - 1);
  }
  p.meta.insert(p.meta.end(), last.begin(), last.end());
  if (hybrid)
    for (size_t l = 0; l < p.order.size(); ++l)
      for (size_t t = 0; t < lens[p.order[l]]; ++t) p.meta.push_back((uint32_t)t);
  PSSA_RETURN_IF(L->ctx->stage.to_device(L->ids.p, ids_h.data(), tokens * 4, L->ctx->stream));
  PSSA_RETURN_IF(upload_plan(L, p, n_lanes, hybrid ? tokens : 0));
  p.rows.ids = L->ids.as<uint32_t>();
  PSSA_RETURN_IF(pssa::run_prefill_ragged(L, p.rows));
  return sync(L->ctx);  // the staging vectors are freed at return
}

// Ids [n_lanes, T] after the reference's rule for invalid ids (src/pssa.rs:
// 2411-2418: every token before the first invalid one is processed, then the
// call fails and leaves the logits alone), with L->ctx->mu held.  Returns
// Ok when every id is valid (nothing run); otherwise advances each lane
// through its valid prefix and returns the error of the first invalid id.
static Status invalid_prefix_locked(pssa_hip_lanes* L, const uint32_t* ids, size_t n_lanes, size_t T) {
  const uint32_t V = (uint32_t)L->model->cfg.d_vocab;
  std::vector<uint64_t> lens(n_lanes);
  bool all = true;
  uint32_t first_bad = 0;
  for (size_t i = 0; i < n_lanes; ++i) {
    size_t v = 0;
    while (v < T && ids[i * T + v] < V) ++v;
    lens[i] = v;
    if (v < T && all) first_bad = ids[i * T + v];
    all &= v == T;
  }
  if (all) return Status::Ok();
  std::vector<uint32_t> packed;
  for (size_t i = 0; i < n_lanes; ++i) packed.insert(packed.end(), ids + i * T, ids + i * T + lens[i]);
  PSSA_RETURN_IF(ragged_locked(L, packed.data(), lens.data(), n_lanes));
  L->staged_lanes = L->staged_len = 0;
  L->logit_lanes = 0;  // no decode continues from a failed prompt
  return Status::Invalid("prompt ID " + std::to_string(first_bad) + " outside model vocabulary");
}

int pssa_hip_prefill_ragged(pssa_hip_lanes* L, const uint32_t* ids, const uint64_t* lens, size_t n_lanes,
                            float* logits_last, size_t logits_len, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(need(L && ids && lens, "null argument"));
    PSSA_RETURN_IF(need(n_lanes > 0 && n_lanes <= L->lanes, "n_lanes must be in 1..=lanes"));
    const size_t V = L->model->cfg.d_vocab;
    size_t tokens = 0;
    for (size_t i = 0; i < n_lanes; ++i) {
      PSSA_RETURN_IF(need(lens[i] > 0, "prefill requires at least one token"));
      PSSA_RETURN_IF(need(lens[i] <= L->max_tokens, "the lanes' tokens exceed max_tokens"));
      tokens += lens[i];
    }
    PSSA_RETURN_IF(need(tokens <= L->max_tokens, "the lanes' tokens exceed max_tokens"));
    for (size_t i = 0; i < tokens; ++i)
      if (ids[i] >= V) return Status::Invalid("prompt ID " + std::to_string(ids[i]) + " outside model vocabulary");
    if (logits_last) PSSA_RETURN_IF(need(logits_len == n_lanes * V, "logits length must be n_lanes*d_vocab"));
    std::lock_guard<std::mutex> g(L->ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(L->ctx->device));
    PSSA_RETURN_IF(ragged_locked(L, ids, lens, n_lanes));
    L->staged_lanes = L->staged_len = 0;  // `ids` holds the packed prompts
    L->logit_lanes = n_lanes;             // decode may continue from these logits
    if (logits_last) PSSA_RETURN_IF(download(L->ctx, logits_last, L->logits, n_lanes * V * 4));
    return sync(L->ctx);
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_prefill_cancellable(pssa_hip_lanes* L, const uint32_t* ids, size_t n_lanes, size_t seq_len,
                                 size_t chunk, pssa_hip_cancel_fn cancelled, void* user, float* logits_last,
                                 size_t logits_len, size_t* processed, char* err, size_t err_len) {
  bool was_cancelled = false;
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(need(L != nullptr && ids != nullptr, "null argument"));
    PSSA_RETURN_IF(need(seq_len > 0, "prefill requires at least one token"));
    PSSA_RETURN_IF(need(n_lanes > 0 && n_lanes <= L->lanes, "n_lanes must be in 1..=lanes"));
    PSSA_RETURN_IF(need(chunk > 0, "chunk must be positive"));
    const size_t c = std::min(chunk, seq_len);
    PSSA_RETURN_IF(need(n_lanes * c <= L->max_tokens, "n_lanes*chunk exceeds max_tokens"));
    const size_t V = L->model->cfg.d_vocab;
    if (logits_last) PSSA_RETURN_IF(need(logits_len == n_lanes * V, "logits length must be n_lanes*d_vocab"));
    if (processed) *processed = 0;
    std::lock_guard<std::mutex> g(L->ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(L->ctx->device));
    std::vector<uint32_t> part(n_lanes * c);
    for (size_t t0 = 0; t0 < seq_len; t0 += c) {
      // The reference asks before every token (src/pssa.rs:2412-2415); here
      // before every chunk of `chunk` tokens (1: every token).
      if (cancelled && cancelled(user)) {
        was_cancelled = true;
        L->staged_lanes = L->staged_len = 0;
        L->logit_lanes = 0;
        return Status::Ok();
      }
      const size_t T = std::min(c, seq_len - t0);
      for (size_t i = 0; i < n_lanes; ++i)
        std::memcpy(&part[i * T], ids + i * seq_len + t0, T * 4);
      PSSA_RETURN_IF(invalid_prefix_locked(L, part.data(), n_lanes, T));
      PSSA_RETURN_IF(L->ctx->stage.to_device(L->ids.p, part.data(), n_lanes * T * 4, L->ctx->stream));
      PSSA_RETURN_IF(pssa::run_prefill(L, n_lanes, T));
      PSSA_RETURN_IF(sync(L->ctx));  // `part` is refilled next
      if (processed) *processed = t0 + T;
    }
    L->staged_lanes = L->staged_len = 0;  // `ids` holds the last chunk
    L->logit_lanes = n_lanes;
    if (logits_last) PSSA_RETURN_IF(download(L->ctx, logits_last, L->logits, n_lanes * V * 4));
    return sync(L->ctx);
  };
  const int rc = pssa::finish(body(), err, err_len);
  return rc == PSSA_HIP_OK && was_cancelled ? PSSA_HIP_CANCELLED : rc;
}

int pssa_hip_batch_forward(pssa_hip_lanes* L, const pssa_hip_sequence* seqs, size_t n_seqs, float* out_loss,
                           float* token_losses, size_t token_losses_len, float* logits, size_t logits_len,
                           char* err, size_t err_len) {
  auto body = [&]() -> Status {
    // Validation in SequenceBatch::forward's order (src/sequence_batch.rs:243-272),
    // all before any carry changes.
    PSSA_RETURN_IF(need(L && out_loss, "null lanes or loss output"));
    PSSA_RETURN_IF(need(n_seqs >= 1 && n_seqs <= L->lanes && seqs,
                        "sequence count must be between 1 and the configured batch size"));
    const pssa_hip_model* M = L->model;
    const pssa_hip_config& c = M->cfg;
    const size_t V = c.d_vocab;
    if (L->loops != 1)
      return Status{PSSA_HIP_EUNSUPPORTED, "the batched training forward runs one loop here (set_loops 1)"};
    std::vector<char> used(L->lanes, 0);
    size_t tokens = 0;
    for (size_t i = 0; i < n_seqs; ++i) {
      const pssa_hip_sequence& q = seqs[i];
      PSSA_RETURN_IF(need(q.lane < L->lanes && !used[q.lane],
                          "each sequence needs a distinct lane within the configured batch size"));
      used[q.lane] = 1;
      PSSA_RETURN_IF(need(q.inputs && q.targets && q.len > 0 && q.len <= L->max_tokens,
                          "each sequence needs matching nonempty input/target slices no longer than max_tokens"));
      tokens += q.len;
    }
    PSSA_RETURN_IF(need(tokens <= L->max_tokens, "the batch's tokens exceed the lanes' max_tokens"));
    for (size_t i = 0; i < n_seqs; ++i)
      for (size_t t = 0; t < seqs[i].len; ++t)
        if (seqs[i].inputs[t] >= V || seqs[i].targets[t] >= V)
          return Status::Invalid("batch token ID is outside the model vocabulary");
    for (const pssa::DevBlock& B : M->blocks)
      PSSA_RETURN_IF(need(!B.hybrid, "hybrid read currently requires the CPU backend"));
    if (token_losses)
      PSSA_RETURN_IF(need(token_losses_len == tokens, "token_losses length must equal the batch's token count"));
    if (logits) PSSA_RETURN_IF(need(logits_len == tokens * V, "logits length must be tokens*d_vocab"));

    std::lock_guard<std::mutex> g(L->ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(L->ctx->device));
    const hipStream_t st = L->ctx->stream;
    const size_t cw = c.depth * L->loops * c.d_latent * c.d_state;  // floats of one lane's carry
    if (!L->tok_logits.p) {
      PSSA_RETURN_IF(L->tok_logits.alloc(L->max_tokens * V * 4));
      PSSA_RETURN_IF(L->tok_meta.alloc(2 * L->max_tokens * 4));
      PSSA_RETURN_IF(L->tok_loss.alloc(L->max_tokens * 4));
    }
    L->logit_lanes = 0;  // lanes->logits no longer follows a prefill
    L->tok_row.clear();

    std::vector<size_t> offset(n_seqs);  // packed token offsets in the given order
    std::vector<uint64_t> lens(n_seqs), lane_of(n_seqs);
    for (size_t i = 0, o = 0; i < n_seqs; o += seqs[i].len, ++i) {
      offset[i] = o;
      lens[i] = seqs[i].len;
      lane_of[i] = seqs[i].lane;
    }
    // Carries to reset, runs of neighbouring lanes in one fill.
    float* carry = L->carry.as<float>();
    std::vector<char> reset(L->lanes, 0);
    for (size_t i = 0; i < n_seqs; ++i) reset[seqs[i].lane] = seqs[i].reset != 0;
    for (size_t a = 0; a < L->lanes; ++a) {
      if (!reset[a]) continue;
      size_t e = a + 1;
      while (e < L->lanes && reset[e]) ++e;
      PSSA_RETURN_IF(pssa::launch_fill_zero(st, carry + a * cw, (e - a) * cw));
      a = e;
    }

    RaggedPlan p;
    plan_ragged(L, lens, lane_of, p);
    std::vector<uint32_t> ids_h(tokens), meta_h(2 * tokens), row_h(tokens), target_h(tokens);
    for (size_t l = 0; l < p.order.size(); ++l) {
      const pssa_hip_sequence& q = seqs[p.order[l]];
      std::memcpy(&ids_h[p.row[l]], q.inputs, q.len * 4);
      std::memcpy(&meta_h[p.row[l]], q.targets, q.len * 4);
      for (size_t t = 0; t < q.len; ++t) {
        const size_t at = offset[p.order[l]] + t;
        meta_h[tokens + p.row[l] + t] = (uint32_t)at;
        row_h[at] = (uint32_t)(p.row[l] + t);
        target_h[at] = q.targets[t];
      }
    }
    PSSA_RETURN_IF(L->ctx->stage.to_device(L->ids.p, ids_h.data(), tokens * 4, L->ctx->stream));
    PSSA_RETURN_IF(L->ctx->stage.to_device(L->tok_meta.p, meta_h.data(), 2 * tokens * 4, L->ctx->stream));
    PSSA_RETURN_IF(upload_plan(L, p, 0, 0));
    p.rows.ids = L->ids.as<uint32_t>();
    p.rows.targets = L->tok_meta.as<uint32_t>();
    p.rows.index = L->tok_meta.as<uint32_t>() + tokens;
    p.rows.logits = L->tok_logits.as<float>();
    p.rows.loss = L->tok_loss.as<float>();
    PSSA_RETURN_IF(pssa::run_train_forward(L, p.rows));

    std::vector<float> loss_h(tokens);
    PSSA_RETURN_IF(download(L->ctx, loss_h.data(), L->tok_loss, tokens * 4));
    if (logits)
      for (size_t l = 0; l < p.order.size(); ++l)
        PSSA_RETURN_IF(L->ctx->stage.to_host(logits + offset[p.order[l]] * V,
                                             L->tok_logits.as<float>() + p.row[l] * V, lens[p.order[l]] * V * 4, st));
    PSSA_RETURN_IF(sync(L->ctx));
    L->tok_row.swap(row_h);
    L->tok_target.swap(target_h);
    // The token mean in packed order, summed left to right in f32
    // (stage_logits_loss, src/gpu_batch.rs:1246-1249).
    float total = 0.0f;
    for (size_t i = 0; i < tokens; ++i) total += loss_h[i];
    const float loss = total / (float)tokens;
    if (token_losses) std::memcpy(token_losses, loss_h.data(), tokens * 4);
    *out_loss = loss;
    if (!std::isfinite(loss)) return Status::Invalid("batch forward: non-finite training loss");
    return Status::Ok();
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_lanes_stage_ids(pssa_hip_lanes* L, const uint32_t* ids, size_t n_lanes, size_t seq_len,
                             char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(need(L != nullptr, "null lanes"));
    std::lock_guard<std::mutex> g(L->ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(L->ctx->device));
    PSSA_RETURN_IF(stage_ids_locked(L, ids, n_lanes, seq_len));
    return sync(L->ctx);
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_lanes_prefill_staged(pssa_hip_lanes* L, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(need(L != nullptr, "null lanes"));
    PSSA_RETURN_IF(need(L->staged_len > 0, "no ids staged"));
    std::lock_guard<std::mutex> g(L->ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(L->ctx->device));
    PSSA_RETURN_IF(pssa::run_prefill(L, L->staged_lanes, L->staged_len));
    L->logit_lanes = L->staged_lanes;
    return Status::Ok();
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_lanes_read_logits(pssa_hip_lanes* L, float* out, size_t len, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(need(L && out, "null argument"));
    const size_t n = L->logit_lanes * L->model->cfg.d_vocab;
    PSSA_RETURN_IF(need(n > 0, "no prefill logits to read"));
    PSSA_RETURN_IF(need(len == n, "logits length must be the last prefill's lanes*d_vocab"));
    std::lock_guard<std::mutex> g(L->ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(L->ctx->device));
    PSSA_RETURN_IF(download(L->ctx, out, L->logits, n * 4));
    return sync(L->ctx);
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_lanes_stage_times(pssa_hip_lanes* L, int enable, const char** names, float* ms, size_t cap) {
  if (!L) return PSSA_HIP_EINVAL;
  if (enable >= 0) L->timing = enable != 0;
  size_t n = 0;
  for (int s2 = 0; s2 < pssa::ST_COUNT && n < cap; ++s2) {
    if (names) names[n] = pssa::kStageNames[s2];
    if (ms) ms[n] = L->stage_ms[s2];
    ++n;
  }
  return (int)n;
}

int pssa_hip_model_get_plastic(pssa_hip_model* M, size_t layer, float* adapter_up, float* keys,
                               float* values, float* norm_sq, float* confidence, uint64_t* last_seen,
                               uint64_t* count, uint64_t* write_head, uint64_t* step, char* err,
                               size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(need(M != nullptr, "null model"));
    const pssa_hip_config& c = M->cfg;
    PSSA_RETURN_IF(need(layer < c.depth, "layer out of range"));
    std::lock_guard<std::mutex> g(M->ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(M->ctx->device));
    const hipStream_t st = M->ctx->stream;
    const pssa::DevBlock& B = M->blocks[layer];
    const size_t d = c.d_latent, k = c.d_mem_key, C = c.mem_capacity, r = c.adapter_rank;
    if (adapter_up) PSSA_RETURN_IF(download(M->ctx, adapter_up, B.u_fast, d * r * 4));
    if (keys) PSSA_RETURN_IF(download(M->ctx, keys, B.keys, C * k * 4));
    if (values) PSSA_RETURN_IF(download(M->ctx, values, B.values, C * d * 4));
    if (norm_sq) PSSA_RETURN_IF(download(M->ctx, norm_sq, B.norm_sq, C * 4));
    if (confidence) PSSA_RETURN_IF(download(M->ctx, confidence, B.conf, C * 4));
    std::vector<unsigned long long> last(C);
    if (last_seen) PSSA_RETURN_IF(download(M->ctx, last.data(), B.last_seen, C * 8));
    int meta[2] = {0, 0};
    PSSA_RETURN_IF(download(M->ctx, meta, B.meta, sizeof(meta)));
    unsigned long long stp = 0;
    PSSA_RETURN_IF(download(M->ctx, &stp, M->step, 8));
    PSSA_RETURN_IF(sync(M->ctx));
    if (last_seen)
      for (size_t q = 0; q < C; ++q) last_seen[q] = last[q];
    if (count) *count = (uint64_t)meta[0];
    if (write_head) *write_head = (uint64_t)meta[1];
    if (step) *step = stp;
    return Status::Ok();
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_model_set_hybrid_read(pssa_hip_model* M, int enabled, float lam, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(need(M != nullptr, "null model"));
    PSSA_RETURN_IF(need(std::isfinite(lam) && lam > 0.0f && lam <= 1.0f, "hybrid decay lam must be in (0.0, 1.0]"));
    std::lock_guard<std::mutex> g(M->ctx->mu);
    for (auto& B : M->blocks) {
      B.hybrid = enabled != 0;
      B.lam = lam;
    }
    ++M->hybrid_epoch;
    return Status::Ok();
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_model_set_value_cap(pssa_hip_model* M, float cap, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(need(M != nullptr, "null model"));
    PSSA_RETURN_IF(need(std::isfinite(cap) && cap >= 0.0f, "memory value cap must be positive and finite"));
    std::lock_guard<std::mutex> g(M->ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(M->ctx->device));
    std::vector<pssa::DevBlock*> all;
    for (pssa::DevBlock& B : M->blocks) all.push_back(&B);
    if (cap > 0.0f) PSSA_RETURN_IF(cap_bank_values(M, all, cap));
    for (pssa::DevBlock& B : M->blocks) B.value_cap = cap;
    ++M->hybrid_epoch;  // captured bank writes hold the old cap
    return sync(M->ctx);
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_model_set_memory_top_k(pssa_hip_model* M, size_t top_k, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(need(M != nullptr, "null model"));
    PSSA_RETURN_IF(need(top_k <= (size_t)pssa::kMaxTopK, "memory top-k above 64 is not supported"));
    std::lock_guard<std::mutex> g(M->ctx->mu);
    for (pssa::DevBlock& B : M->blocks) B.top_k = (int)top_k;
    ++M->hybrid_epoch;
    return Status::Ok();
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_model_get_hybrid(pssa_hip_model* M, size_t layer, float* gate, uint64_t* age, char* err,
                              size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(need(M != nullptr, "null model"));
    PSSA_RETURN_IF(need(layer < M->cfg.depth, "layer out of range"));
    std::lock_guard<std::mutex> g(M->ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(M->ctx->device));
    const hipStream_t st = M->ctx->stream;
    const pssa::DevBlock& B = M->blocks[layer];
    const size_t C = M->cfg.mem_capacity;
    if (gate) PSSA_RETURN_IF(download(M->ctx, gate, B.hgate, C * 4));
    std::vector<unsigned long long> a(C);
    if (age) PSSA_RETURN_IF(download(M->ctx, a.data(), B.hage, C * 8));
    PSSA_RETURN_IF(sync(M->ctx));
    if (age)
      for (size_t q = 0; q < C; ++q) age[q] = a[q];
    return Status::Ok();
  };
  return pssa::finish(body(), err, err_len);
}

}  // extern "C"

namespace {

// Recurrent depth loops and the hybrid read are not combined on the device.
Status loops_allow_hybrid(const pssa_hip_lanes* L) {
  if (L->loops > 1)
    for (const pssa::DevBlock& B : L->model->blocks)
      if (B.hybrid) return Status{PSSA_HIP_EUNSUPPORTED, "the hybrid read runs one loop here (set_loops 1)"};
  return Status::Ok();
}

Status ensure_decode_buffers(pssa_hip_lanes* L, size_t n_lanes, size_t steps) {
  const pssa_hip_config& c = L->model->cfg;
  if (L->dec_lanes < L->lanes) {
    const size_t n = L->lanes, D = c.depth;
    PSSA_RETURN_IF(L->tap_q.alloc(D * n * c.d_mem_key * 4));
    PSSA_RETURN_IF(L->tap_z.alloc(D * n * c.d_latent * 4));
    PSSA_RETURN_IF(L->tap_a.alloc(D * n * c.d_latent * 4));
    PSSA_RETURN_IF(L->tap_act.alloc(D * n * c.adapter_rank * 4));
    PSSA_RETURN_IF(L->tap_gmean.alloc(D * n * 4));
    PSSA_RETURN_IF(L->tap_zcap.alloc(D * n * c.d_latent * 4));
    PSSA_RETURN_IF(L->surprise.alloc(n * 4));
    PSSA_RETURN_IF(L->hebb_rate.alloc(D * n * 4));  // [depth, lanes]
    PSSA_RETURN_IF(L->bank_writer.alloc(D * c.mem_capacity * 4));
    PSSA_RETURN_IF(L->gen_pos.alloc(4));
    L->dec_lanes = n;
  }
  if (L->gen_cap < steps) {
    const size_t cap = std::max<size_t>(steps, 128);
    PSSA_RETURN_IF(L->gen_ids.alloc(cap * L->lanes * 4));
    L->gen_cap = cap;
    // The captured step holds the old buffer's address.
    if (L->graph_exec) (void)hipGraphExecDestroy(L->graph_exec);
    if (L->graph) (void)hipGraphDestroy(L->graph);
    L->graph_exec = nullptr;
    L->graph = nullptr;
    L->graph_lanes = 0;
  }
  (void)n_lanes;
  return Status::Ok();
}

Status capture_decode_step(pssa_hip_lanes* L, size_t n_lanes, bool plastic) {
  if (L->graph_exec && L->graph_lanes == n_lanes && L->graph_plastic == (plastic ? 1 : 0) &&
      L->graph_hybrid_epoch == L->model->hybrid_epoch && L->graph_penalty == L->rep_penalty &&
      L->graph_temperature == L->temperature && L->graph_top_p == L->top_p && L->graph_top_k == L->top_k)
    return Status::Ok();
  if (L->graph_exec) (void)hipGraphExecDestroy(L->graph_exec);
  if (L->graph) (void)hipGraphDestroy(L->graph);
  L->graph_exec = nullptr;
  L->graph = nullptr;
  const hipStream_t st = L->ctx->stream;
  const bool timing = L->timing;
  L->timing = false;  // no event records inside the graph
  PSSA_HIP_TRY(hipStreamBeginCapture(st, hipStreamCaptureModeThreadLocal));
  Status s = pssa::run_decode_step(L, n_lanes, plastic);
  hipGraph_t graph = nullptr;
  const hipError_t e = hipStreamEndCapture(st, &graph);
  L->timing = timing;
  PSSA_RETURN_IF(s);
  if (e != hipSuccess) return Status::Device(std::string("hipStreamEndCapture: ") + hipGetErrorString(e));
  L->graph = graph;
  PSSA_HIP_TRY(hipGraphInstantiate(&L->graph_exec, graph, nullptr, nullptr, 0));
  L->graph_lanes = n_lanes;
  L->graph_plastic = plastic ? 1 : 0;
  L->graph_hybrid_epoch = L->model->hybrid_epoch;
  L->graph_penalty = L->rep_penalty;
  L->graph_temperature = L->temperature;
  L->graph_top_p = L->top_p;
  L->graph_top_k = L->top_k;
  return Status::Ok();
}

}  // namespace

extern "C" {

int pssa_hip_lanes_get_taps(pssa_hip_lanes* L, size_t layer, size_t n_lanes, float* q_pnc, float* z_final,
                            float* ad_out, float* act, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(need(L != nullptr, "null lanes"));
    std::lock_guard<std::mutex> g(L->ctx->mu);
    const pssa_hip_config& c = L->model->cfg;
    PSSA_RETURN_IF(need(L->tap_lanes > 0, "no plastic decode step has recorded taps"));
    PSSA_RETURN_IF(need(n_lanes == L->tap_lanes, "n_lanes must be the last plastic step's lane count"));
    PSSA_RETURN_IF(need(layer < c.depth, "layer out of range"));
    PSSA_HIP_TRY(hipSetDevice(L->ctx->device));
    const hipStream_t st = L->ctx->stream;
    const size_t n = n_lanes, d = c.d_latent, k = c.d_mem_key, r = c.adapter_rank;
    auto part = [&](float* dst, const DevBuf& src, size_t w) -> Status {
      if (!dst) return Status::Ok();
      PSSA_RETURN_IF(L->ctx->stage.to_host(dst, src.as<float>() + layer * n * w, n * w * 4, st));
      return Status::Ok();
    };
    PSSA_RETURN_IF(part(q_pnc, L->tap_q, k));
    PSSA_RETURN_IF(part(z_final, L->tap_z, d));
    PSSA_RETURN_IF(part(ad_out, L->tap_a, d));
    PSSA_RETURN_IF(part(act, L->tap_act, r));
    return sync(L->ctx);
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_lanes_set_repetition_penalty(pssa_hip_lanes* L, float penalty, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(need(L != nullptr, "null lanes"));
    PSSA_RETURN_IF(need(std::isfinite(penalty) && penalty >= 1.0f, "repetition penalty must be finite and >= 1"));
    std::lock_guard<std::mutex> g(L->ctx->mu);
    L->rep_penalty = penalty;
    return Status::Ok();
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_lanes_set_loops(pssa_hip_lanes* L, size_t loops, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(need(L != nullptr, "null lanes"));
    PSSA_RETURN_IF(need(loops >= 1 && loops <= 32, "--loops must be between 1 and 32; use --loops 1 for the original model"));
    std::lock_guard<std::mutex> g(L->ctx->mu);
    if (loops == L->loops) return Status::Ok();
    if (loops > 1)
      for (const pssa::DevBlock& B : L->model->blocks)
        if (B.hybrid) return Status{PSSA_HIP_EUNSUPPORTED, "the hybrid read runs one loop here (set_loops 1)"};
    PSSA_HIP_TRY(hipSetDevice(L->ctx->device));
    const hipStream_t st = L->ctx->stream;
    const pssa_hip_config& c = L->model->cfg;
    const size_t hs = c.d_latent * c.d_state, per = L->lanes * c.depth;
    // Loop 0 keeps each block's persistent carry; the other loops start from
    // zero, as resize_loop_tape leaves them (src/pssa.rs:2147-2167).
    DevBuf carry;
    PSSA_RETURN_IF(carry.alloc(per * loops * hs * 4));
    PSSA_RETURN_IF(pssa::launch_fill_zero(st, carry.as<float>(), per * loops * hs));
    PSSA_HIP_TRY(hipMemcpy2DAsync(carry.p, loops * hs * 4, L->carry.p, L->loops * hs * 4, hs * 4, per,
                                  hipMemcpyDeviceToDevice, st));
    if (loops > 1 && !L->Xin.p) PSSA_RETURN_IF(L->Xin.alloc(L->max_tokens * c.d_latent * 4));
    PSSA_RETURN_IF(sync(L->ctx));
    std::swap(L->carry, carry);
    L->loops = loops;
    // The captured step and the prefill logits belong to the old carries.
    if (L->graph_exec) (void)hipGraphExecDestroy(L->graph_exec);
    if (L->graph) (void)hipGraphDestroy(L->graph);
    L->graph_exec = nullptr;
    L->graph = nullptr;
    L->graph_lanes = 0;
    L->logit_lanes = 0;
    return Status::Ok();
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_lanes_set_sampling(pssa_hip_lanes* L, float temperature, float top_p, size_t top_k, uint64_t seed,
                                char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(need(L != nullptr, "null lanes"));
    // InferenceConfig validation (src/inference.rs:87-100).
    PSSA_RETURN_IF(need(std::isfinite(temperature) && temperature >= 0.0f, "temperature must be finite and >= 0"));
    PSSA_RETURN_IF(need(std::isfinite(top_p) && top_p > 0.0f && top_p <= 1.0f, "top-p must be finite in (0, 1]"));
    PSSA_RETURN_IF(need(top_k > 0, "top-k must be positive"));
    if (temperature > 0.0f && top_k > 64)
      return Status{PSSA_HIP_EUNSUPPORTED, "sampling on the device supports top-k up to 64"};
    std::lock_guard<std::mutex> g(L->ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(L->ctx->device));
    const hipStream_t st = L->ctx->stream;
    if (temperature > 0.0f) {
      if (!L->rng.p) PSSA_RETURN_IF(L->rng.alloc(L->lanes * 8));
      if (!L->probs.p && L->model->cfg.d_vocab > (size_t)pssa::kSampleRowMaxV)
        PSSA_RETURN_IF(L->probs.alloc(L->lanes * L->model->cfg.d_vocab * 4));
      // SimpleRng::new (src/linalg.rs:7-11): every lane starts from `seed`.
      std::vector<uint64_t> st0(L->lanes, seed == 0 ? 0x853c49e6748fea9bULL : seed);
      PSSA_RETURN_IF(L->ctx->stage.to_device(L->rng.p, st0.data(), L->lanes * 8, L->ctx->stream));
      PSSA_RETURN_IF(sync(L->ctx));
    }
    L->temperature = temperature;
    L->top_p = top_p;
    L->top_k = (int)std::min<size_t>(top_k, 64);
    return Status::Ok();
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_decode(pssa_hip_lanes* L, const uint32_t* first_ids, size_t n_lanes, size_t steps,
                    int flags, uint32_t* out_ids, size_t out_len, float* logits_last,
                    size_t logits_len, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(need(L != nullptr, "null lanes"));
    PSSA_RETURN_IF(need((flags & ~(PSSA_HIP_DECODE_PLASTIC | PSSA_HIP_DECODE_GRAPH)) == 0, "unknown decode flags"));
    PSSA_RETURN_IF(need(n_lanes > 0 && n_lanes <= L->lanes, "n_lanes must be in 1..=lanes"));
    PSSA_RETURN_IF(need(steps > 0 && steps <= (1u << 20), "steps must be in 1..=2^20"));
    PSSA_RETURN_IF(need(out_ids != nullptr && out_len == steps * n_lanes, "out_ids length must be steps*n_lanes"));
    const size_t V = L->model->cfg.d_vocab;
    if (logits_last) PSSA_RETURN_IF(need(logits_len == n_lanes * V, "logits length must be n_lanes*d_vocab"));
    if (first_ids) {
      for (size_t i = 0; i < n_lanes; ++i)
        if (first_ids[i] >= V)
          return Status::Invalid("prompt ID " + std::to_string(first_ids[i]) + " outside model vocabulary");
    } else {
      PSSA_RETURN_IF(need(L->logit_lanes == n_lanes, "decode without first ids continues the last prefill of n_lanes lanes"));
    }
    const bool plastic = (flags & PSSA_HIP_DECODE_PLASTIC) != 0;
    if (plastic && L->loops != 1)
      return Status{PSSA_HIP_EUNSUPPORTED, "plastic decode runs one loop here (set_loops 1)"};
    // Refused before the choice kernel runs: it records a token and advances
    // every lane's generator.
    PSSA_RETURN_IF(loops_allow_hybrid(L));
    if (plastic) {
      PSSA_RETURN_IF(need(pssa::bank_write_lds((int)L->model->cfg.mem_capacity, (int)n_lanes) <= 160 * 1024,
                          "plastic decode: mem_capacity and n_lanes exceed the bank-write LDS budget"));
      PSSA_RETURN_IF(need(L->model->cfg.adapter_rank <= 256 &&
                              pssa::hebbian_lds((int)L->model->cfg.adapter_rank, (int)n_lanes) <= 160 * 1024,
                          "plastic decode: adapter rank and n_lanes exceed the Hebbian-update LDS budget"));
    }
    std::lock_guard<std::mutex> g(L->ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(L->ctx->device));
    const hipStream_t st = L->ctx->stream;
    PSSA_RETURN_IF(ensure_decode_buffers(L, n_lanes, steps));
    PSSA_RETURN_IF(pssa::launch_fill_zero(st, static_cast<float*>(L->nonfinite.p), 3));
    const int zero = 0;
    PSSA_RETURN_IF(L->ctx->stage.to_device(L->gen_pos.p, &zero, 4, L->ctx->stream));
    // After a prefill the first generated token is the choice from its logits
    // (src/inference.rs:367-379), and each later one costs a forward step of
    // the token before it; given first ids, every token costs a step.
    size_t fwd_steps = steps;
    if (first_ids) {
      PSSA_RETURN_IF(L->ctx->stage.to_device(L->ids.p, first_ids, n_lanes * 4, L->ctx->stream));
    } else {
      PSSA_RETURN_IF(pssa::run_greedy_from_logits(L, n_lanes, true));
      fwd_steps = steps - 1;
    }
    if (fwd_steps > 0 && (flags & PSSA_HIP_DECODE_GRAPH)) {
      PSSA_RETURN_IF(capture_decode_step(L, n_lanes, plastic));
      for (size_t t = 0; t < fwd_steps; ++t) PSSA_HIP_TRY(hipGraphLaunch(L->graph_exec, st));
    } else {
      for (size_t t = 0; t < fwd_steps; ++t) PSSA_RETURN_IF(pssa::run_decode_step(L, n_lanes, plastic));
    }
    PSSA_RETURN_IF(download(L->ctx, out_ids, L->gen_ids, steps * n_lanes * 4));
    if (logits_last) PSSA_RETURN_IF(download(L->ctx, logits_last, L->logits, n_lanes * V * 4));
    int nonfinite[3] = {0, 0, 0};
    PSSA_RETURN_IF(download(L->ctx, nonfinite, L->nonfinite, 12));
    // The last generated token has not been consumed: a continuation passes
    // it as first_ids.  `ids` now holds the step tokens.
    L->staged_lanes = L->staged_len = 0;
    L->logit_lanes = 0;
    PSSA_RETURN_IF(sync(L->ctx));
    // sample() refuses non-finite logits (src/inference.rs:110-112).
    if (nonfinite[0]) return Status::Invalid("model emitted non-finite logits");
    // clamp_value refuses a non-finite value (src/memory.rs:151-152).
    if (nonfinite[1]) return Status::Invalid("capped memory value must be finite");
    if (nonfinite[2]) return Status::Invalid("invalid sampling probability mass");
    return Status::Ok();
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_dense_scan(pssa_hip_ctx* ctx, const float* a, const float* b, const float* h0,
                        size_t batch, size_t seq_len, size_t d_state, float* h, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(check_ctx(ctx));
    PSSA_RETURN_IF(need(a && b && h, "dense scan: null buffer"));
    PSSA_RETURN_IF(need(batch && seq_len && d_state, "dense scan: dimensions must be positive"));
    PSSA_RETURN_IF(need(d_state <= 64, "dense scan: d_state above 64 is not supported"));
    size_t na = 0, nb = 0;
    PSSA_RETURN_IF(pssa::checked_count({batch, seq_len, d_state, d_state}, &na, "dense scan"));
    PSSA_RETURN_IF(pssa::checked_count({batch, seq_len, d_state}, &nb, "dense scan"));
    if (batch > INT32_MAX || seq_len > INT32_MAX) return Status::Invalid("dense scan: too large");
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    const hipStream_t st = ctx->stream;
    DevBuf da, db, dh0, dh;
    PSSA_RETURN_IF(upload(ctx, da, a, na * 4));
    PSSA_RETURN_IF(upload(ctx, db, b, nb * 4));
    if (h0) PSSA_RETURN_IF(upload(ctx, dh0, h0, batch * d_state * 4));
    PSSA_RETURN_IF(dh.alloc(nb * 4));
    PSSA_RETURN_IF(bind_dense_scan_scratch(ctx, (int)batch, (int)seq_len, (int)d_state));
    PSSA_RETURN_IF(pssa::launch_dense_scan(st, da.as<float>(), db.as<float>(), h0 ? dh0.as<float>() : nullptr,
                                           dh.as<float>(), (int)batch, (int)seq_len, (int)d_state, ctx->scratch,
                                           ctx->scratch_bytes));
    PSSA_RETURN_IF(download(ctx, h, dh, nb * 4));
    return sync(ctx);
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_dense_scan_resident(pssa_hip_ctx* ctx, const float* d_a, const float* d_b,
                                 const float* d_h0, size_t batch, size_t seq_len, size_t d_state,
                                 float* d_h, char* err, size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(check_ctx(ctx));
    PSSA_RETURN_IF(need(d_a && d_b && d_h, "dense scan: null buffer"));
    PSSA_RETURN_IF(need(batch && seq_len && d_state, "dense scan: dimensions must be positive"));
    PSSA_RETURN_IF(need(d_state <= 64, "dense scan: d_state above 64 is not supported"));
    if (batch > INT32_MAX || seq_len > INT32_MAX) return Status::Invalid("dense scan: too large");
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    PSSA_RETURN_IF(bind_dense_scan_scratch(ctx, (int)batch, (int)seq_len, (int)d_state));
    return pssa::launch_dense_scan(ctx->stream, d_a, d_b, d_h0, d_h, (int)batch, (int)seq_len, (int)d_state,
                                   ctx->scratch, ctx->scratch_bytes);
  };
  return pssa::finish(body(), err, err_len);
}

int pssa_hip_dense_scan_reserve(pssa_hip_ctx* ctx, size_t batch, size_t seq_len, size_t d_state, char* err,
                                size_t err_len) {
  auto body = [&]() -> Status {
    PSSA_RETURN_IF(check_ctx(ctx));
    PSSA_RETURN_IF(need(batch && seq_len && d_state, "dense scan: dimensions must be positive"));
    PSSA_RETURN_IF(need(d_state <= 64, "dense scan: d_state above 64 is not supported"));
    if (batch > INT32_MAX || seq_len > INT32_MAX) return Status::Invalid("dense scan: too large");
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    return bind_dense_scan_scratch(ctx, (int)batch, (int)seq_len, (int)d_state);
  };
  return pssa::finish(body(), err, err_len);
}

}  // extern "C"

// ------------------------------------------------- language-model operators

// 4-bit weights on the device.
struct pssa_hip_w4 {
  pssa_hip_ctx* ctx = nullptr;
  DevBuf data;  // codes, scales and zero points, one behind the other
  pssa::W4View view;
};

namespace {

// Runs an entry point's body; no C++ exception leaves it.
template <class Body>
int guarded(Body body, char* err, size_t err_len) {
  try {
    return pssa::finish(body(), err, err_len);
  } catch (const std::exception& e) {
    return pssa::finish(Status::NoMem(std::string("host: ") + e.what()), err, err_len);
  }
}

bool temperature_ok(float t) { return t >= 1e-6f && t <= 1e6f; }
bool dtype_ok(int dtype) { return dtype == PSSA_HIP_F32 || dtype == PSSA_HIP_BF16; }
size_t dtype_size(int dtype) { return dtype == PSSA_HIP_BF16 ? 2 : 4; }
bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// A matrix of logit rows: its type, extent and alignment.
Status check_rows(const void* p, int dtype, size_t rows, size_t vocab, size_t ld, const char* what) {
  PSSA_RETURN_IF(need(dtype_ok(dtype), "unknown dtype"));
  if (!rows || !vocab) return Status::Invalid(std::string(what) + ": dimensions must be positive");
  if (vocab > ((size_t)1 << 24) || rows > INT32_MAX) return Status::Invalid(std::string(what) + ": too large");
  if (ld < vocab) return Status::Invalid(std::string(what) + ": row stride below the vocabulary");
  size_t n = 0;
  PSSA_RETURN_IF(pssa::checked_count({rows, ld}, &n, what));
  if (!aligned_to(p, dtype_size(dtype))) return Status::Invalid(std::string(what) + ": misaligned buffer");
  return Status::Ok();
}

// Rows of `width` words between packed token order (host) and the device
// rows of the last batch forward.
template <class T>
void rows_to_device_order(const std::vector<uint32_t>& row, const T* in, size_t width, std::vector<T>& out) {
  out.resize(row.size() * width);
  for (size_t i = 0; i < row.size(); ++i) std::memcpy(&out[row[i] * width], in + i * width, width * sizeof(T));
}

// A device array in batch-row order, copied to `out` in packed token order.
template <class T>
Status rows_to_host(pssa_hip_lanes* L, T* out, const DevBuf& buf, size_t width) {
  std::vector<T> h(L->tok_row.size() * width);
  PSSA_RETURN_IF(download(L->ctx, h.data(), buf, h.size() * sizeof(T)));
  PSSA_RETURN_IF(sync(L->ctx));
  for (size_t i = 0; i < L->tok_row.size(); ++i)
    std::memcpy(out + i * width, &h[L->tok_row[i] * width], width * sizeof(T));
  return Status::Ok();
}

Status check_batch(const pssa_hip_lanes* L, size_t n_tokens) {
  PSSA_RETURN_IF(need(!L->tok_row.empty(), "no batch forward has left logits on these lanes"));
  return need(n_tokens == L->tok_row.size(), "token count must be the last batch forward's");
}

// Token ids of a host array: the model's or none.
Status check_tokens(const uint32_t* ids, size_t n, size_t V, const char* what) {
  for (size_t i = 0; i < n; ++i)
    if (ids[i] >= V && ids[i] != PSSA_HIP_NO_TOKEN)
      return Status::Invalid(std::string(what) + " token ID " + std::to_string(ids[i]) + " outside model vocabulary");
  return Status::Ok();
}

Status check_w4(size_t n, size_t k, size_t group) {
  PSSA_RETURN_IF(need(n && k, "4-bit weights: dimensions must be positive"));
  PSSA_RETURN_IF(need(group == 32 || group == 64 || group == 128, "4-bit weights: group must be 32, 64 or 128"));
  // The layout's kernel has a thread for each 16 packed bytes, counted in 32 bits.
  return need(n <= ((size_t)1 << 30) && k <= ((size_t)1 << 24) && pssa::w4_packed_bytes(n, k) <= (size_t)1 << 35,
              "4-bit weights: too large");
}

// Lays device arrays out into a new handle; the caller waits for the stream.
Status load_w4(pssa_hip_ctx* ctx, const uint8_t* codes, const float* scales, const uint8_t* zeros, size_t n, size_t k,
               size_t group, std::unique_ptr<pssa_hip_w4>& w) {
  w = std::make_unique<pssa_hip_w4>();
  w->ctx = ctx;
  const size_t held = pssa::w4_groups_held(n, k, group), packed = pssa::w4_packed_bytes(n, k);
  PSSA_RETURN_IF(w->data.alloc(packed + held * (zeros ? 5 : 4)));
  char* base = w->data.as<char>();
  float* held_scales = reinterpret_cast<float*>(base + packed);
  uint8_t* held_zeros = zeros ? reinterpret_cast<uint8_t*>(held_scales + held) : nullptr;
  PSSA_RETURN_IF(
      pssa::launch_w4_pack(ctx->stream, codes, scales, zeros, (int)n, (int)k, (int)group, base, held_scales, held_zeros));
  w->view.packed = base;
  w->view.scales = held_scales;
  w->view.zeros = held_zeros;
  w->view.n = (int)n;
  w->view.k = (int)k;
  w->view.group = (int)group;
  return Status::Ok();
}

bool disjoint(const void* a, size_t na, const void* b, size_t nb) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return x + na <= y || y + nb <= x;
}

// Token rows `w` wide at stride ld apart from rows `wo` wide at stride ldo:
// in memory, or as other columns of the same rows.
bool rows_disjoint(const void* p, size_t ld, size_t w, const void* o, size_t ldo, size_t wo, size_t rows, size_t size) {
  if (!rows || disjoint(p, ((rows - 1) * ld + w) * size, o, ((rows - 1) * ldo + wo) * size)) return true;
  const intptr_t d = (intptr_t)o - (intptr_t)p;
  if (ld != ldo || d % (intptr_t)size) return false;
  const intptr_t row = (intptr_t)ld;
  const size_t at = (size_t)((d / (intptr_t)size % row + row) % row);
  return at >= w && at + wo <= ld;
}

// The sequences of a linear attention call and their split into work items.
struct LinearPlan {
  std::vector<uint32_t> table;  // first tokens (and a split call's items), where the arguments do not hold them
  size_t tokens = 0, longest = 0;
  size_t states = 0;  // bytes of the scratch before the table: a split call's states, one for each item

  size_t scratch_bytes() const { return states + table.size() * 4; }
};
Status plan_sequences(const uint64_t* lens, size_t n_seqs, size_t seq_len, size_t heads, size_t d_key,
                      size_t d_val, pssa::LinearArgs& a, LinearPlan& p) {
  PSSA_RETURN_IF(need(n_seqs >= 1 && n_seqs <= 65535, "linear attention: sequences must be in 1..=65535"));
  a.n_seqs = (int)n_seqs;
  const size_t most = INT32_MAX;
  bool same = true;
  for (size_t i = 0; i < n_seqs; ++i) {
    const size_t len = lens ? lens[i] : seq_len;
    PSSA_RETURN_IF(need(len <= most && p.tokens + len <= most, "linear attention: too many tokens"));
    p.tokens += len;
    p.longest = std::max(p.longest, len);
    same &= !lens || lens[i] == lens[0];
  }
  const size_t seg = (size_t)pssa::linear_segment(lens, n_seqs, p.longest, heads, d_key, d_val);
  a.seg_len = (int)(seg ? seg : std::max<size_t>(p.longest, 1));
  a.uniform_len = same ? (int)p.longest : -1;
  a.uniform_segs = (int)std::max<size_t>(1, (p.longest + a.seg_len - 1) / a.seg_len);
  if (same) {
    a.items = (int)n_seqs * a.uniform_segs;
  } else {
    const bool inside = n_seqs <= (size_t)pssa::kLinearInline;
    if (!inside) p.table.resize((seg ? 2 : 1) * (n_seqs + 1));
    uint32_t* tok = inside ? a.inline_tokens : p.table.data();
    uint32_t* item = !seg ? nullptr : inside ? a.inline_items : p.table.data() + n_seqs + 1;
    uint32_t t = 0, w = 0;
    for (size_t i = 0; i < n_seqs; ++i) {
      tok[i] = t;
      if (item) item[i] = w;
      t += (uint32_t)lens[i];
      w += (uint32_t)std::max<size_t>(1, (lens[i] + a.seg_len - 1) / a.seg_len);
    }
    tok[n_seqs] = t;
    if (item) item[n_seqs] = w;
    a.items = (int)w;
  }
  if (a.items > a.n_seqs) p.states = ((size_t)a.items * heads * d_key * d_val * 4 + 255) & ~(size_t)255;
  return Status::Ok();
}

Status check_heads(size_t heads, size_t d_key, size_t d_val) {
  PSSA_RETURN_IF(need(heads && d_key && d_val, "linear attention: dimensions must be positive"));
  PSSA_RETURN_IF(need(heads <= 65535, "linear attention: at most 65535 heads"));
  PSSA_RETURN_IF(need(d_key <= (size_t)pssa::kLinearMaxKey, "linear attention: d_key above 128 is not supported"));
  return need(d_val <= 4096, "linear attention: d_val above 4096 is not supported");
}

}  // namespace

extern "C" {

int pssa_hip_token_logprobs_resident(pssa_hip_ctx* ctx, const void* d_logits, int dtype, size_t rows, size_t vocab,
                                     size_t ld, const uint32_t* d_targets, float temperature, size_t top_k,
                                     float* d_logprobs, float* d_entropy, uint32_t* d_top_ids,
                                     float* d_top_logprobs, char* err, size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(need(d_logits != nullptr, "token logprobs: null buffer"));
    PSSA_RETURN_IF(check_rows(d_logits, dtype, rows, vocab, ld, "token logprobs"));
    PSSA_RETURN_IF(need(temperature_ok(temperature), "token logprobs: temperature must be in [1e-6, 1e6]"));
    PSSA_RETURN_IF(need(top_k <= (size_t)pssa::kMaxAlternatives, "token logprobs: top_k must be at most 64"));
    PSSA_RETURN_IF(need(!top_k || (d_top_ids && d_top_logprobs), "token logprobs: top_k needs both of its outputs"));
    PSSA_RETURN_IF(need(!d_logprobs || d_targets, "token logprobs: log probabilities need targets"));
    PSSA_RETURN_IF(need(d_logprobs || d_entropy || top_k, "token logprobs: no output asked for"));
    PSSA_RETURN_IF(need(aligned_to(d_targets, 4) && aligned_to(d_logprobs, 4) && aligned_to(d_entropy, 4) &&
                            aligned_to(d_top_ids, 4) && aligned_to(d_top_logprobs, 4),
                        "token logprobs: misaligned buffer"));
    PSSA_RETURN_IF(check_ctx(ctx));
    pssa::LogprobArgs a;
    a.logits = d_logits;
    a.ld = ld;
    a.vocab = (int)vocab;
    a.targets = d_targets;
    a.temperature = temperature;
    a.top_k = (int)top_k;
    a.logprobs = d_logprobs;
    a.entropy = d_entropy;
    a.top_ids = d_top_ids;
    a.top_logprobs = d_top_logprobs;
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    return pssa::launch_token_logprobs(ctx->stream, dtype, a, rows);
  }, err, err_len);
}

int pssa_hip_distill_resident(pssa_hip_ctx* ctx, const void* d_logits, int dtype, size_t rows, size_t vocab,
                              size_t ld, const uint32_t* d_teacher_ids, const float* d_teacher_logits,
                              size_t teacher_k, float temperature, const float* d_row_weights, float* d_losses,
                              void* d_grad, size_t ld_grad, char* err, size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(need(d_logits && d_teacher_ids && d_teacher_logits && d_losses, "distill: null buffer"));
    PSSA_RETURN_IF(check_rows(d_logits, dtype, rows, vocab, ld, "distill"));
    PSSA_RETURN_IF(need(teacher_k >= 1 && teacher_k <= (size_t)pssa::kMaxTeacher,
                        "distill: teacher_k must be in 1..=1024"));
    PSSA_RETURN_IF(need(temperature_ok(temperature), "distill: temperature must be in [1e-6, 1e6]"));
    PSSA_RETURN_IF(need(aligned_to(d_teacher_ids, 4) && aligned_to(d_teacher_logits, 4) &&
                            aligned_to(d_row_weights, 4) && aligned_to(d_losses, 4),
                        "distill: misaligned buffer"));
    if (d_grad) {
      PSSA_RETURN_IF(check_rows(d_grad, dtype, rows, vocab, ld_grad, "distill gradient"));
      if (d_grad == d_logits) {
        PSSA_RETURN_IF(need(ld_grad == ld, "distill: a gradient in place needs the logits' row stride"));
      } else {
        const uintptr_t x = (uintptr_t)d_logits, y = (uintptr_t)d_grad;
        const size_t nx = ((rows - 1) * ld + vocab) * dtype_size(dtype);
        const size_t ny = ((rows - 1) * ld_grad + vocab) * dtype_size(dtype);
        PSSA_RETURN_IF(need(x + nx <= y || y + ny <= x, "distill: the gradient overlaps the logits"));
      }
    }
    PSSA_RETURN_IF(check_ctx(ctx));
    pssa::DistillArgs a;
    a.logits = d_logits;
    a.ld = ld;
    a.vocab = (int)vocab;
    a.teacher_ids = d_teacher_ids;
    a.teacher_logits = d_teacher_logits;
    a.teacher_k = (int)teacher_k;
    a.temperature = temperature;
    a.row_weights = d_row_weights;
    a.losses = d_losses;
    a.grad = d_grad;
    a.ld_grad = ld_grad;
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    return pssa::launch_distill(ctx->stream, dtype, a, rows);
  }, err, err_len);
}

int pssa_hip_batch_token_logprobs(pssa_hip_lanes* L, const uint32_t* targets, size_t n_tokens, float temperature,
                                  size_t top_k, float* logprobs, float* entropy, uint32_t* top_ids,
                                  float* top_logprobs, char* err, size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(need(L != nullptr, "null lanes"));
    PSSA_RETURN_IF(need(temperature_ok(temperature), "token logprobs: temperature must be in [1e-6, 1e6]"));
    PSSA_RETURN_IF(need(top_k <= (size_t)pssa::kMaxAlternatives, "token logprobs: top_k must be at most 64"));
    std::lock_guard<std::mutex> g(L->ctx->mu);
    PSSA_RETURN_IF(check_batch(L, n_tokens));
    pssa_hip_ctx* ctx = L->ctx;
    const size_t V = L->model->cfg.d_vocab;
    if (targets) PSSA_RETURN_IF(check_tokens(targets, n_tokens, V, "token logprobs: target"));
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    std::vector<uint32_t> target_h;
    rows_to_device_order(L->tok_row, targets ? targets : L->tok_target.data(), 1, target_h);
    DevBuf dt, lp, en, id, tl;
    PSSA_RETURN_IF(upload(ctx, dt, target_h.data(), n_tokens * 4));
    PSSA_RETURN_IF(lp.alloc(n_tokens * 4, &ctx->pool));
    PSSA_RETURN_IF(en.alloc(n_tokens * 4, &ctx->pool));
    PSSA_RETURN_IF(id.alloc(n_tokens * top_k * 4, &ctx->pool));
    PSSA_RETURN_IF(tl.alloc(n_tokens * top_k * 4, &ctx->pool));
    pssa::LogprobArgs a;
    a.logits = L->tok_logits.p;
    a.ld = V;
    a.vocab = (int)V;
    a.targets = dt.as<uint32_t>();
    a.temperature = temperature;
    a.top_k = (int)top_k;
    a.logprobs = lp.as<float>();
    a.entropy = en.as<float>();
    a.top_ids = id.as<uint32_t>();
    a.top_logprobs = tl.as<float>();
    PSSA_RETURN_IF(pssa::launch_token_logprobs(ctx->stream, PSSA_HIP_F32, a, n_tokens));
    if (logprobs) PSSA_RETURN_IF(rows_to_host(L, logprobs, lp, 1));
    if (entropy) PSSA_RETURN_IF(rows_to_host(L, entropy, en, 1));
    if (top_ids && top_k) PSSA_RETURN_IF(rows_to_host(L, top_ids, id, top_k));
    if (top_logprobs && top_k) PSSA_RETURN_IF(rows_to_host(L, top_logprobs, tl, top_k));
    return sync(ctx);
  }, err, err_len);
}

int pssa_hip_batch_distill(pssa_hip_lanes* L, const uint32_t* teacher_ids, const float* teacher_logits,
                           size_t n_tokens, size_t teacher_k, float temperature, const float* row_weights,
                           float* losses, float* grad_logits, char* err, size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(need(L && teacher_ids && teacher_logits && losses, "distill: null buffer"));
    PSSA_RETURN_IF(need(teacher_k >= 1 && teacher_k <= (size_t)pssa::kMaxTeacher,
                        "distill: teacher_k must be in 1..=1024"));
    PSSA_RETURN_IF(need(temperature_ok(temperature), "distill: temperature must be in [1e-6, 1e6]"));
    std::lock_guard<std::mutex> g(L->ctx->mu);
    PSSA_RETURN_IF(check_batch(L, n_tokens));
    pssa_hip_ctx* ctx = L->ctx;
    const size_t V = L->model->cfg.d_vocab;
    PSSA_RETURN_IF(check_tokens(teacher_ids, n_tokens * teacher_k, V, "distill: teacher"));
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    std::vector<uint32_t> ids_h;
    std::vector<float> t_h, w_h;
    rows_to_device_order(L->tok_row, teacher_ids, teacher_k, ids_h);
    rows_to_device_order(L->tok_row, teacher_logits, teacher_k, t_h);
    if (row_weights) rows_to_device_order(L->tok_row, row_weights, 1, w_h);
    DevBuf ids, t, w, loss, grad;
    PSSA_RETURN_IF(upload(ctx, ids, ids_h.data(), ids_h.size() * 4));
    PSSA_RETURN_IF(upload(ctx, t, t_h.data(), t_h.size() * 4));
    if (row_weights) PSSA_RETURN_IF(upload(ctx, w, w_h.data(), w_h.size() * 4));
    PSSA_RETURN_IF(loss.alloc(n_tokens * 4, &ctx->pool));
    if (grad_logits) PSSA_RETURN_IF(grad.alloc(n_tokens * V * 4, &ctx->pool));
    pssa::DistillArgs a;
    a.logits = L->tok_logits.p;
    a.ld = V;
    a.vocab = (int)V;
    a.teacher_ids = ids.as<uint32_t>();
    a.teacher_logits = t.as<float>();
    a.teacher_k = (int)teacher_k;
    a.temperature = temperature;
    a.row_weights = row_weights ? w.as<float>() : nullptr;
    a.losses = loss.as<float>();
    a.grad = grad_logits ? grad.p : nullptr;
    a.ld_grad = V;
    PSSA_RETURN_IF(pssa::launch_distill(ctx->stream, PSSA_HIP_F32, a, n_tokens));
    PSSA_RETURN_IF(rows_to_host(L, losses, loss, 1));
    if (grad_logits) {
      // Runs of neighbouring rows go down together, without a second host copy.
      for (size_t i = 0; i < n_tokens;) {
        size_t e = i + 1;
        while (e < n_tokens && L->tok_row[e] == L->tok_row[e - 1] + 1) ++e;
        PSSA_RETURN_IF(ctx->stage.to_host(grad_logits + i * V, grad.as<float>() + (size_t)L->tok_row[i] * V,
                                          (e - i) * V * 4, ctx->stream));
        i = e;
      }
    }
    return sync(ctx);
  }, err, err_len);
}

int pssa_hip_w4_load_resident(pssa_hip_ctx* ctx, const uint8_t* d_codes, const float* d_scales, const uint8_t* d_zeros,
                              size_t n, size_t k, size_t group, pssa_hip_w4** out, char* err, size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(need(out != nullptr, "null output handle"));
    *out = nullptr;
    PSSA_RETURN_IF(need(d_codes && d_scales, "4-bit weights: null buffer"));
    PSSA_RETURN_IF(check_w4(n, k, group));
    PSSA_RETURN_IF(need(aligned_to(d_scales, 4), "4-bit weights: misaligned buffer"));
    PSSA_RETURN_IF(check_ctx(ctx));
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    std::unique_ptr<pssa_hip_w4> w;
    PSSA_RETURN_IF(load_w4(ctx, d_codes, d_scales, d_zeros, n, k, group, w));
    PSSA_RETURN_IF(sync(ctx));
    *out = w.release();
    return Status::Ok();
  }, err, err_len);
}

int pssa_hip_w4_load(pssa_hip_ctx* ctx, const uint8_t* codes, size_t codes_len, const float* scales, size_t scales_len,
                     const uint8_t* zeros, size_t n, size_t k, size_t group, pssa_hip_w4** out, char* err,
                     size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(need(out != nullptr, "null output handle"));
    *out = nullptr;
    PSSA_RETURN_IF(need(codes && scales, "4-bit weights: null buffer"));
    PSSA_RETURN_IF(check_w4(n, k, group));
    const size_t groups = n * ((k + group - 1) / group);
    PSSA_RETURN_IF(need(codes_len == n * k && scales_len == groups,
                        "4-bit weights: codes must be [n, k] and scales [n, ceil(k / group)]"));
    PSSA_RETURN_IF(check_ctx(ctx));
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    DevBuf dc, ds, dz;
    PSSA_RETURN_IF(upload(ctx, dc, codes, codes_len));
    PSSA_RETURN_IF(upload(ctx, ds, scales, groups * 4));
    if (zeros) PSSA_RETURN_IF(upload(ctx, dz, zeros, groups));
    std::unique_ptr<pssa_hip_w4> w;
    PSSA_RETURN_IF(load_w4(ctx, dc.as<uint8_t>(), ds.as<float>(), zeros ? dz.as<uint8_t>() : nullptr, n, k, group, w));
    PSSA_RETURN_IF(sync(ctx));
    *out = w.release();
    return Status::Ok();
  }, err, err_len);
}

void pssa_hip_w4_free(pssa_hip_w4* w) {
  if (!w) return;
  {
    std::lock_guard<std::mutex> g(w->ctx->mu);
    (void)hipSetDevice(w->ctx->device);
    (void)hipStreamSynchronize(w->ctx->stream);
  }
  delete w;
}

int pssa_hip_matvec_w4_resident(pssa_hip_w4* w, const void* d_x, int x_dtype, size_t m, size_t ld_x, float* d_y,
                                size_t ld_y, char* err, size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(need(w && d_x && d_y, "4-bit product: null weights or buffer"));
    PSSA_RETURN_IF(need(dtype_ok(x_dtype), "unknown dtype"));
    PSSA_RETURN_IF(need(m >= 1, "4-bit product: dimensions must be positive"));
    PSSA_RETURN_IF(need(m <= 65535, "4-bit product: at most 65535 rows"));
    const size_t n = (size_t)w->view.n, k = (size_t)w->view.k;
    PSSA_RETURN_IF(need(ld_x >= k && ld_y >= n, "4-bit product: row stride below the row"));
    size_t nx = 0, ny = 0;
    PSSA_RETURN_IF(pssa::checked_count({m, ld_x}, &nx, "4-bit product input"));
    PSSA_RETURN_IF(pssa::checked_count({m, ld_y}, &ny, "4-bit product output"));
    PSSA_RETURN_IF(need(aligned_to(d_x, dtype_size(x_dtype)) && aligned_to(d_y, 4), "4-bit product: misaligned buffer"));
    const uintptr_t x = (uintptr_t)d_x, y = (uintptr_t)d_y;
    PSSA_RETURN_IF(need(x + ((m - 1) * ld_x + k) * dtype_size(x_dtype) <= y || y + ((m - 1) * ld_y + n) * 4 <= x,
                        "4-bit product: the output overlaps the input"));
    std::lock_guard<std::mutex> g(w->ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(w->ctx->device));
    return pssa::launch_matvec_w4(w->ctx->stream, x_dtype, d_x, ld_x, (int)m, w->view, d_y, ld_y);
  }, err, err_len);
}

int pssa_hip_matvec_w4(pssa_hip_w4* w, const float* x, size_t x_len, size_t m, float* y, size_t y_len, char* err,
                       size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(need(w && x && y, "4-bit product: null weights or buffer"));
    PSSA_RETURN_IF(need(m >= 1 && m <= 65535, "4-bit product: rows must be in 1..=65535"));
    const size_t n = (size_t)w->view.n, k = (size_t)w->view.k;
    PSSA_RETURN_IF(need(x_len == m * k && y_len == m * n, "4-bit product: x must be [m, k] and y [m, n]"));
    pssa_hip_ctx* ctx = w->ctx;
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    DevBuf dx, dy;
    PSSA_RETURN_IF(upload(ctx, dx, x, x_len * 4));
    PSSA_RETURN_IF(dy.alloc(y_len * 4, &ctx->pool));
    PSSA_RETURN_IF(pssa::launch_matvec_w4(ctx->stream, PSSA_HIP_F32, dx.p, k, (int)m, w->view, dy.as<float>(), n));
    PSSA_RETURN_IF(download(ctx, y, dy, y_len * 4));
    return sync(ctx);
  }, err, err_len);
}

int pssa_hip_linear_attention_resident(pssa_hip_ctx* ctx, int dtype, const void* d_q, size_t ld_q, const void* d_k,
                                       size_t ld_k, const void* d_v, size_t ld_v, const float* d_log_decay,
                                       const float* d_state_in, const uint64_t* lens, size_t n_seqs, size_t seq_len,
                                       size_t heads, size_t kv_heads, size_t d_key, size_t d_val, float scale,
                                       void* d_out, size_t ld_out, float* d_state_out, char* err, size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(need(d_q && d_k && d_v && d_log_decay && d_out, "linear attention: null buffer"));
    PSSA_RETURN_IF(need(dtype_ok(dtype), "unknown dtype"));
    PSSA_RETURN_IF(check_heads(heads, d_key, d_val));
    PSSA_RETURN_IF(need(kv_heads && heads % kv_heads == 0, "linear attention: kv_heads must divide heads"));
    PSSA_RETURN_IF(need(std::isfinite(scale), "linear attention: scale must be finite"));
    const size_t size = dtype_size(dtype), wq = heads * d_key, wk = kv_heads * d_key, wv = kv_heads * d_val,
                 wo = heads * d_val;
    PSSA_RETURN_IF(need(ld_q >= wq && ld_k >= wk && ld_v >= wv && ld_out >= wo,
                        "linear attention: row stride below the heads' width"));
    PSSA_RETURN_IF(need(std::max(std::max(ld_q, ld_k), std::max(ld_v, ld_out)) < ((size_t)1 << 24),
                        "linear attention: row strides must be below 2^24"));
    PSSA_RETURN_IF(need(aligned_to(d_q, size) && aligned_to(d_k, size) && aligned_to(d_v, size) &&
                            aligned_to(d_out, size) && aligned_to(d_log_decay, 4) && aligned_to(d_state_in, 4) &&
                            aligned_to(d_state_out, 4),
                        "linear attention: misaligned buffer"));
    pssa::LinearArgs a;
    LinearPlan plan;
    PSSA_RETURN_IF(plan_sequences(lens, n_seqs, seq_len, heads, d_key, d_val, a, plan));
    const size_t tokens = plan.tokens;
    size_t n = 0;
    for (size_t ld : {ld_q, ld_k, ld_v, ld_out}) PSSA_RETURN_IF(pssa::checked_count({tokens, ld}, &n, "linear attention"));
    PSSA_RETURN_IF(pssa::checked_count({n_seqs, heads, d_key, d_val}, &n, "linear attention states"));
    PSSA_RETURN_IF(need(rows_disjoint(d_q, ld_q, wq, d_out, ld_out, wo, tokens, size) &&
                            rows_disjoint(d_k, ld_k, wk, d_out, ld_out, wo, tokens, size) &&
                            rows_disjoint(d_v, ld_v, wv, d_out, ld_out, wo, tokens, size),
                        "linear attention: the output overlaps its inputs"));
    if (tokens) {
      const size_t out_bytes = ((tokens - 1) * ld_out + wo) * size;
      PSSA_RETURN_IF(need(disjoint(d_log_decay, heads * 4, d_out, out_bytes), "linear attention: the output overlaps its inputs"));
      PSSA_RETURN_IF(need(!d_state_in || disjoint(d_state_in, n * 4, d_out, out_bytes),
                          "linear attention: the output overlaps the states"));
    }
    if (d_state_out) {
      PSSA_RETURN_IF(need(disjoint(d_log_decay, heads * 4, d_state_out, n * 4), "linear attention: the states overlap"));
      PSSA_RETURN_IF(need(!d_state_in || d_state_in == d_state_out || disjoint(d_state_in, n * 4, d_state_out, n * 4),
                          "linear attention: the states overlap"));
      if (tokens)
        for (auto [p, ld, w] : {std::tuple{d_q, ld_q, wq}, {d_k, ld_k, wk}, {d_v, ld_v, wv}, {(const void*)d_out, ld_out, wo}})
          PSSA_RETURN_IF(need(disjoint(p, ((tokens - 1) * ld + w) * size, d_state_out, n * 4),
                              "linear attention: the states overlap"));
    }
    PSSA_RETURN_IF(check_ctx(ctx));
    a.q = d_q;
    a.k = d_k;
    a.v = d_v;
    a.ld_q = ld_q;
    a.ld_k = ld_k;
    a.ld_v = ld_v;
    a.ld_out = ld_out;
    a.log_decay = d_log_decay;
    a.state_in = d_state_in;
    a.state_out = d_state_out;
    a.out = d_out;
    a.scale = scale;
    a.heads = (int)heads;
    a.kv_heads = (int)kv_heads;
    a.dk = (int)d_key;
    a.dv = (int)d_val;
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    PSSA_RETURN_IF(grow_scratch(ctx, plan.scratch_bytes(), false));
    if (plan.states) a.seg_state = static_cast<float*>(ctx->scratch);
    if (!plan.table.empty()) {
      uint32_t* table = reinterpret_cast<uint32_t*>(static_cast<char*>(ctx->scratch) + plan.states);
      PSSA_RETURN_IF(ctx->stage.to_device(table, plan.table.data(), plan.table.size() * 4, ctx->stream));
      a.table = table;
    }
    return pssa::launch_linear_attention(ctx->stream, dtype, a, (int)plan.longest);
  }, err, err_len);
}

int pssa_hip_linear_attention_reserve(pssa_hip_ctx* ctx, int dtype, const uint64_t* lens, size_t n_seqs, size_t seq_len,
                                      size_t heads, size_t d_key, size_t d_val, char* err, size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(need(dtype_ok(dtype), "unknown dtype"));
    PSSA_RETURN_IF(check_heads(heads, d_key, d_val));
    pssa::LinearArgs a;
    LinearPlan plan;
    PSSA_RETURN_IF(plan_sequences(lens, n_seqs, seq_len, heads, d_key, d_val, a, plan));
    PSSA_RETURN_IF(check_ctx(ctx));
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    return grow_scratch(ctx, plan.scratch_bytes(), false);
  }, err, err_len);
}

}  // extern "C"

namespace {

// The sequences of a delta rule call and the scratch that it takes.
struct DeltaPlan {
  std::vector<uint32_t> table;  // first tokens and chunks, where the arguments do not hold them
  size_t tokens = 0, longest = 0;
  bool chunked = false;
  pssa::DeltaScratch scratch;

  // What is worked out ahead, row copies, the segments' states and transitions, then the table.
  size_t table_at() const { return scratch.ahead + scratch.rows + scratch.state + scratch.move; }
  size_t scratch_bytes() const { return table_at() + table.size() * 4; }
};
Status plan_delta(int dtype, const uint64_t* lens, size_t n_seqs, size_t seq_len, size_t heads, size_t d_key, size_t d_val,
                  pssa::DeltaArgs& a, DeltaPlan& p) {
  PSSA_RETURN_IF(need(n_seqs >= 1 && n_seqs <= 65535, "delta rule: sequences must be in 1..=65535"));
  a.n_seqs = (int)n_seqs;
  const size_t chunk = (size_t)pssa::delta_chunk(dtype);
  bool same = true;
  for (size_t i = 0; i < n_seqs; ++i) {
    const size_t len = lens ? lens[i] : seq_len;
    PSSA_RETURN_IF(need(len <= INT32_MAX && p.tokens + len <= INT32_MAX, "delta rule: too many tokens"));
    p.tokens += len;
    p.longest = std::max(p.longest, len);
    same &= !lens || lens[i] == lens[0];
  }
  a.uniform_len = same ? (int)p.longest : -1;
  p.chunked = p.longest > (size_t)pssa::kDeltaSteps;
  a.seg_chunks = p.chunked ? pssa::delta_segment(dtype, lens, n_seqs, p.longest, heads, d_key, d_val) : 0;
  const size_t seg = (size_t)a.seg_chunks * chunk;
  auto segments = [&](size_t len) { return seg ? std::max<size_t>(1, (len + seg - 1) / seg) : 1; };
  size_t chunks = 0, items = 0;
  const bool inside = n_seqs <= (size_t)pssa::kDeltaInline;
  if (!same && !inside) p.table.resize((seg ? 3 : 2) * (n_seqs + 1));
  uint32_t* tok = inside ? a.inline_tokens : p.table.data();
  uint32_t* first = inside ? a.inline_chunks : p.table.data() + n_seqs + 1;
  uint32_t* item = inside ? a.inline_items : p.table.data() + 2 * (n_seqs + 1);
  uint32_t t = 0;
  for (size_t i = 0; i <= n_seqs; ++i) {
    if (!same) {
      tok[i] = t;
      first[i] = (uint32_t)chunks;
      if (seg) item[i] = (uint32_t)items;
    }
    if (i == n_seqs) break;
    const size_t len = lens ? lens[i] : seq_len;
    t += (uint32_t)len;
    chunks += (len + chunk - 1) / chunk;
    items += segments(len);
  }
  PSSA_RETURN_IF(need(chunks < ((size_t)1 << 24), "delta rule: too many tokens"));
  a.chunks = (int)chunks;
  a.items = (int)items;
  a.uniform_segs = (int)segments(p.longest);
  if (p.chunked) p.scratch = pssa::delta_scratch(dtype, chunks, n_seqs, seg ? items : 0, heads, d_key, d_val);
  return Status::Ok();
}
Status check_delta_heads(size_t heads, size_t d_key, size_t d_val) {
  PSSA_RETURN_IF(need(heads && d_key && d_val, "delta rule: dimensions must be positive"));
  PSSA_RETURN_IF(need(heads <= 65535, "delta rule: at most 65535 heads"));
  PSSA_RETURN_IF(need(d_key <= (size_t)pssa::kDeltaMaxKey, "delta rule: d_key above 128 is not supported"));
  return need(d_val <= 4096, "delta rule: d_val above 4096 is not supported");
}

// Rows `w` bytes wide at stride ld bytes: an array of a call that its outputs must not touch.
struct Rows {
  const void* p;
  size_t rows, ld, w;
};
// Apart in memory, or other columns of the same rows.
bool apart(const Rows& a, const Rows& b) {
  if (!a.p || !b.p) return true;
  if (a.rows == b.rows && a.ld && b.ld) return rows_disjoint(a.p, a.ld, a.w, b.p, b.ld, b.w, a.rows, 1);
  return !a.rows || !b.rows || disjoint(a.p, (a.rows - 1) * a.ld + a.w, b.p, (b.rows - 1) * b.ld + b.w);
}
// A matrix of rows: its extent.
Status check_matrix(size_t rows, size_t width, size_t ld, const char* what) {
  if (!rows || !width) return Status::Invalid(std::string(what) + ": dimensions must be positive");
  if (ld < width) return Status::Invalid(std::string(what) + ": row stride below the row");
  if (rows > INT32_MAX || ld > INT32_MAX) return Status::Invalid(std::string(what) + ": too large");
  size_t n = 0;
  return pssa::checked_count({rows, ld}, &n, what);
}
Status check_i8(size_t m, size_t n, size_t k) {
  PSSA_RETURN_IF(need(m && n && k, "8-bit product: dimensions must be positive"));
  PSSA_RETURN_IF(need(k <= pssa::kI8Depth, "8-bit product: k above 131071 is not supported"));
  return need(m <= ((size_t)1 << 20) && n <= ((size_t)1 << 24), "8-bit product: too large");
}
Status check_beams(size_t groups, size_t beams, size_t vocab, size_t keep) {
  PSSA_RETURN_IF(need(groups && vocab, "beam selection: dimensions must be positive"));
  PSSA_RETURN_IF(need(beams >= 1 && beams <= (size_t)pssa::kMaxBeams && keep >= 1 && keep <= (size_t)pssa::kMaxBeams,
                      "beam selection: beams and keep must be in 1..=64"));
  return need(vocab <= ((size_t)1 << 24) && groups <= (((size_t)1 << 24) - 1) / beams, "beam selection: too large");
}

// The selection of one step on the context's stream, its scratch grown to what it needs.
Status select_beams(pssa_hip_ctx* ctx, int dtype, pssa::BeamArgs& a, size_t groups) {
  const pssa::BeamPlan p = pssa::beam_plan(dtype, groups * (size_t)a.beams, (size_t)a.vocab, (size_t)a.keep);
  PSSA_RETURN_IF(grow_scratch(ctx, p.bytes, false));
  a.slices = (int)p.slices;
  a.sums = ctx->scratch;
  a.keys = reinterpret_cast<uint64_t*>(static_cast<char*>(ctx->scratch) + p.sums_bytes);
  return pssa::launch_beam_select(ctx->stream, dtype, a, groups, p);
}

Status reorder_rows(pssa_hip_ctx* ctx, const DevBuf& rows, size_t row_bytes, size_t groups, size_t beams,
                    const uint32_t* parents) {
  pssa::GatherArgs a;
  a.src = a.dst = rows.p;
  a.ld_src = a.ld_dst = a.row_bytes = row_bytes;
  a.groups = (int)groups;
  a.n_in = a.n_out = (int)beams;
  a.parents = parents;
  return pssa::launch_beam_gather(ctx->stream, a);
}

}  // namespace

extern "C" {

int pssa_hip_delta_rule_resident(pssa_hip_ctx* ctx, int dtype, const void* d_q, size_t ld_q, const void* d_k,
                                 size_t ld_k, const void* d_v, size_t ld_v, const float* d_log_decay,
                                 const float* d_beta, size_t ld_gates, const float* d_state_in, const uint64_t* lens,
                                 size_t n_seqs, size_t seq_len, size_t heads, size_t key_heads, size_t d_key,
                                 size_t d_val, float scale, void* d_out, size_t ld_out, float* d_state_out, char* err,
                                 size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(need(d_q && d_k && d_v && d_log_decay && d_beta && d_out, "delta rule: null buffer"));
    PSSA_RETURN_IF(need(dtype_ok(dtype), "unknown dtype"));
    PSSA_RETURN_IF(check_delta_heads(heads, d_key, d_val));
    PSSA_RETURN_IF(need(key_heads && heads % key_heads == 0, "delta rule: key_heads must divide heads"));
    PSSA_RETURN_IF(need(std::isfinite(scale), "delta rule: scale must be finite"));
    const size_t size = dtype_size(dtype), wk = key_heads * d_key, wv = heads * d_val;
    PSSA_RETURN_IF(need(ld_q >= wk && ld_k >= wk && ld_v >= wv && ld_out >= wv && ld_gates >= heads,
                        "delta rule: row stride below the heads' width"));
    PSSA_RETURN_IF(need(std::max({ld_q, ld_k, ld_v, ld_out, ld_gates}) < ((size_t)1 << 24),
                        "delta rule: row strides must be below 2^24"));
    PSSA_RETURN_IF(need(aligned_to(d_q, size) && aligned_to(d_k, size) && aligned_to(d_v, size) &&
                            aligned_to(d_out, size) && aligned_to(d_log_decay, 4) && aligned_to(d_beta, 4) &&
                            aligned_to(d_state_in, 4) && aligned_to(d_state_out, 4),
                        "delta rule: misaligned buffer"));
    pssa::DeltaArgs a;
    DeltaPlan plan;
    PSSA_RETURN_IF(plan_delta(dtype, lens, n_seqs, seq_len, heads, d_key, d_val, a, plan));
    const size_t tokens = plan.tokens;
    if (plan.chunked) {
      auto copied = [&](const void* p, size_t ld, size_t n, size_t width) {
        return pssa::delta_in_units(dtype, p, ld, width) ? 0 : pssa::delta_copy_bytes(dtype, tokens, n, width);
      };
      const size_t q = copied(d_q, ld_q, key_heads, d_key), k = copied(d_k, ld_k, key_heads, d_key), v = copied(d_v, ld_v, heads, d_val);
      PSSA_RETURN_IF(need(std::max({q, k, v}) / 16 <= pssa::kMostThreads, "delta rule: too large for rows not in units of 16 bytes"));
      plan.scratch.rows = q + k + v;
    }
    size_t n = 0;
    for (size_t ld : {ld_q, ld_k, ld_v, ld_out, ld_gates})
      PSSA_RETURN_IF(pssa::checked_count({tokens, ld}, &n, "delta rule"));
    PSSA_RETURN_IF(pssa::checked_count({n_seqs, heads, d_key, d_val}, &n, "delta rule states"));
    const Rows out{d_out, tokens, ld_out * size, wv * size}, in{d_state_in, 1, 0, n * 4}, kept{d_state_out, 1, 0, n * 4};
    for (const Rows& r : {Rows{d_q, tokens, ld_q * size, wk * size}, Rows{d_k, tokens, ld_k * size, wk * size},
                          Rows{d_v, tokens, ld_v * size, wv * size}, Rows{d_log_decay, tokens, ld_gates * 4, heads * 4},
                          Rows{d_beta, tokens, ld_gates * 4, heads * 4}}) {
      PSSA_RETURN_IF(need(apart(r, out), "delta rule: the output overlaps its inputs"));
      PSSA_RETURN_IF(need(apart(r, kept), "delta rule: the states overlap"));
    }
    PSSA_RETURN_IF(need(apart(in, out) && apart(kept, out), "delta rule: the output overlaps the states"));
    PSSA_RETURN_IF(need(d_state_in == d_state_out || apart(in, kept), "delta rule: the states overlap"));
    PSSA_RETURN_IF(check_ctx(ctx));
    a.q = d_q;
    a.k = d_k;
    a.v = d_v;
    a.ld_q = ld_q;
    a.ld_k = ld_k;
    a.ld_v = ld_v;
    a.ld_out = ld_out;
    a.ld_gates = ld_gates;
    a.log_decay = d_log_decay;
    a.beta = d_beta;
    a.state_in = d_state_in;
    a.state_out = d_state_out;
    a.out = d_out;
    a.scale = scale;
    a.heads = (int)heads;
    a.key_heads = (int)key_heads;
    a.dk = (int)d_key;
    a.dv = (int)d_val;
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    PSSA_RETURN_IF(grow_scratch(ctx, plan.scratch_bytes(), false));
    char* scratch = static_cast<char*>(ctx->scratch);
    if (!plan.table.empty()) {
      uint32_t* table = reinterpret_cast<uint32_t*>(scratch + plan.table_at());
      PSSA_RETURN_IF(ctx->stage.to_device(table, plan.table.data(), plan.table.size() * 4, ctx->stream));
      a.table = table;
    }
    return pssa::launch_delta_rule(ctx->stream, dtype, a, tokens, (int)plan.longest, plan.scratch, scratch);
  }, err, err_len);
}

int pssa_hip_delta_rule_reserve(pssa_hip_ctx* ctx, int dtype, const uint64_t* lens, size_t n_seqs, size_t seq_len,
                                size_t heads, size_t d_key, size_t d_val, char* err, size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(need(dtype_ok(dtype), "unknown dtype"));
    PSSA_RETURN_IF(check_delta_heads(heads, d_key, d_val));
    pssa::DeltaArgs a;
    DeltaPlan plan;
    PSSA_RETURN_IF(plan_delta(dtype, lens, n_seqs, seq_len, heads, d_key, d_val, a, plan));
    if (plan.chunked)
      plan.scratch.rows = 2 * pssa::delta_copy_bytes(dtype, plan.tokens, heads, d_key) + pssa::delta_copy_bytes(dtype, plan.tokens, heads, d_val);
    PSSA_RETURN_IF(check_ctx(ctx));
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    return grow_scratch(ctx, plan.scratch_bytes(), false);
  }, err, err_len);
}

int pssa_hip_rms_norm_resident(pssa_hip_ctx* ctx, int dtype, const void* d_x, size_t ld_x, const void* d_residual,
                               size_t ld_residual, const float* d_gamma, float eps, size_t rows, size_t width,
                               void* d_sum, size_t ld_sum, void* d_out, size_t ld_out, int8_t* d_codes,
                               size_t ld_codes, float* d_scales, char* err, size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(need(d_x && d_gamma, "rms norm: null buffer"));
    PSSA_RETURN_IF(need(dtype_ok(dtype), "unknown dtype"));
    PSSA_RETURN_IF(need(eps >= 1e-12f && eps <= 1.0f, "rms norm: eps must be in [1e-12, 1]"));
    PSSA_RETURN_IF(need(width <= pssa::kRmsWidth, "rms norm: rows above 65536 elements are not supported"));
    PSSA_RETURN_IF(need(rows <= pssa::kRmsRows, "rms norm: too large"));
    PSSA_RETURN_IF(need(!d_codes == !d_scales, "rms norm: codes and scales belong together"));
    PSSA_RETURN_IF(need(d_sum || d_out || d_codes, "rms norm: no output asked for"));
    PSSA_RETURN_IF(check_matrix(rows, width, ld_x, "rms norm"));
    if (d_residual) PSSA_RETURN_IF(check_matrix(rows, width, ld_residual, "rms norm residual"));
    if (d_sum) PSSA_RETURN_IF(check_matrix(rows, width, ld_sum, "rms norm sum"));
    if (d_out) PSSA_RETURN_IF(check_matrix(rows, width, ld_out, "rms norm output"));
    if (d_codes) PSSA_RETURN_IF(check_matrix(rows, width, ld_codes, "rms norm codes"));
    const size_t size = dtype_size(dtype);
    PSSA_RETURN_IF(need(aligned_to(d_x, size) && aligned_to(d_residual, size) && aligned_to(d_sum, size) &&
                            aligned_to(d_out, size) && aligned_to(d_gamma, 4) && aligned_to(d_scales, 4),
                        "rms norm: misaligned buffer"));
    const Rows ins[3] = {{d_x, rows, ld_x * size, width * size}, {d_residual, rows, ld_residual * size, width * size},
                         {d_gamma, 1, 0, width * 4}};
    const Rows outs[4] = {{d_sum, rows, ld_sum * size, width * size}, {d_out, rows, ld_out * size, width * size},
                          {d_codes, rows, ld_codes, width}, {d_scales, 1, 0, rows * 4}};
    for (int o = 0; o < 4; ++o) {
      for (int i = 0; i < 3; ++i) {
        const bool in_place = o < 2 && i < 2 && outs[o].p == ins[i].p && outs[o].ld == ins[i].ld;
        PSSA_RETURN_IF(need(in_place || apart(outs[o], ins[i]), "rms norm: an output overlaps an input"));
      }
      for (int i = 0; i < o; ++i) PSSA_RETURN_IF(need(apart(outs[o], outs[i]), "rms norm: the outputs overlap"));
    }
    PSSA_RETURN_IF(check_ctx(ctx));
    pssa::RmsNormArgs a;
    a.x = d_x;
    a.residual = d_residual;
    a.ld_x = ld_x;
    a.ld_residual = ld_residual;
    a.ld_sum = ld_sum;
    a.ld_out = ld_out;
    a.ld_codes = ld_codes;
    a.gamma = d_gamma;
    a.width = (int)width;
    a.eps = eps;
    a.sum = d_sum;
    a.out = d_out;
    a.codes = d_codes;
    a.scales = d_scales;
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    return pssa::launch_rms_norm(ctx->stream, dtype, a, rows);
  }, err, err_len);
}

int pssa_hip_quantize_i8_resident(pssa_hip_ctx* ctx, int dtype, const void* d_x, size_t ld_x, size_t rows, size_t width,
                                  int8_t* d_codes, size_t ld_codes, float* d_scales, char* err, size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(need(d_x && d_codes && d_scales, "8-bit rows: null buffer"));
    PSSA_RETURN_IF(need(dtype_ok(dtype), "unknown dtype"));
    PSSA_RETURN_IF(need(width <= pssa::kRmsWidth, "8-bit rows: above 65536 elements are not supported"));
    PSSA_RETURN_IF(need(rows <= pssa::kRmsRows, "8-bit rows: too large"));
    PSSA_RETURN_IF(check_matrix(rows, width, ld_x, "8-bit rows"));
    PSSA_RETURN_IF(check_matrix(rows, width, ld_codes, "8-bit rows' codes"));
    const size_t size = dtype_size(dtype);
    PSSA_RETURN_IF(need(aligned_to(d_x, size) && aligned_to(d_scales, 4), "8-bit rows: misaligned buffer"));
    const Rows x{d_x, rows, ld_x * size, width * size}, codes{d_codes, rows, ld_codes, width}, scales{d_scales, 1, 0, rows * 4};
    PSSA_RETURN_IF(need(apart(x, codes) && apart(x, scales) && apart(codes, scales), "8-bit rows: the arrays overlap"));
    PSSA_RETURN_IF(check_ctx(ctx));
    pssa::RmsNormArgs a;
    a.x = d_x;
    a.ld_x = ld_x;
    a.ld_codes = ld_codes;
    a.width = (int)width;
    a.normed = false;
    a.codes = d_codes;
    a.scales = d_scales;
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    return pssa::launch_rms_norm(ctx->stream, dtype, a, rows);
  }, err, err_len);
}

int pssa_hip_matmul_i8_resident(pssa_hip_ctx* ctx, const int8_t* d_x, size_t ld_x, const float* d_x_scales,
                                const int8_t* d_w, size_t ld_w, const float* d_w_scales, size_t m, size_t n, size_t k,
                                void* d_y, int y_dtype, size_t ld_y, char* err, size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(need(d_x && d_x_scales && d_w && d_w_scales && d_y, "8-bit product: null buffer"));
    PSSA_RETURN_IF(need(dtype_ok(y_dtype), "unknown dtype"));
    PSSA_RETURN_IF(check_i8(m, n, k));
    PSSA_RETURN_IF(check_matrix(m, k, ld_x, "8-bit product rows"));
    PSSA_RETURN_IF(check_matrix(n, k, ld_w, "8-bit product weights"));
    PSSA_RETURN_IF(check_matrix(m, n, ld_y, "8-bit product output"));
    const size_t size = dtype_size(y_dtype);
    PSSA_RETURN_IF(need(aligned_to(d_x_scales, 4) && aligned_to(d_w_scales, 4) && aligned_to(d_y, size),
                        "8-bit product: misaligned buffer"));
    const Rows y{d_y, m, ld_y * size, n * size};
    for (const Rows& r : {Rows{d_x, m, ld_x, k}, Rows{d_w, n, ld_w, k}, Rows{d_x_scales, 1, 0, m * 4},
                          Rows{d_w_scales, 1, 0, n * 4}})
      PSSA_RETURN_IF(need(apart(r, y), "8-bit product: the output overlaps its inputs"));
    const bool copy_x = !pssa::i8_in_units(d_x, ld_x, k), copy_w = !pssa::i8_in_units(d_w, ld_w, k);
    const pssa::I8Plan plan = pssa::i8_plan(m, n, k, copy_x, copy_w);
    PSSA_RETURN_IF(need(m <= pssa::kI8FewRows || ((copy_x ? m : 0) + (copy_w ? n : 0)) * ((k + 15) / 16) <= pssa::kMostThreads,
                        "8-bit product: too large for rows not in units of 16 bytes"));
    PSSA_RETURN_IF(check_ctx(ctx));
    pssa::I8Args a;
    a.x = d_x;
    a.w = d_w;
    a.ld_x = ld_x;
    a.ld_w = ld_w;
    a.ld_y = ld_y;
    a.x_scales = d_x_scales;
    a.w_scales = d_w_scales;
    a.y = d_y;
    a.m = (int)m;
    a.n = (int)n;
    a.k = (int)k;
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    PSSA_RETURN_IF(grow_scratch(ctx, plan.bytes(), false));
    return pssa::launch_matmul_i8(ctx->stream, y_dtype, a, plan, ctx->scratch);
  }, err, err_len);
}

int pssa_hip_matmul_i8_reserve(pssa_hip_ctx* ctx, size_t m, size_t n, size_t k, char* err, size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(check_i8(m, n, k));
    PSSA_RETURN_IF(check_ctx(ctx));
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    return grow_scratch(ctx, pssa::i8_plan(m, n, k, true, true).bytes(), false);
  }, err, err_len);
}

int pssa_hip_beam_select_resident(pssa_hip_ctx* ctx, const void* d_logits, int dtype, size_t groups, size_t beams,
                                  size_t vocab, size_t ld, const float* d_scores, const uint32_t* d_last, uint32_t eos,
                                  size_t keep, uint32_t* d_parents, uint32_t* d_tokens, float* d_out_scores, char* err,
                                  size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(need(d_logits && d_scores && d_parents && d_tokens && d_out_scores, "beam selection: null buffer"));
    PSSA_RETURN_IF(check_beams(groups, beams, vocab, keep));
    const size_t rows = groups * beams;
    PSSA_RETURN_IF(check_rows(d_logits, dtype, rows, vocab, ld, "beam selection"));
    PSSA_RETURN_IF(need(aligned_to(d_scores, 4) && aligned_to(d_last, 4) && aligned_to(d_parents, 4) &&
                            aligned_to(d_tokens, 4) && aligned_to(d_out_scores, 4),
                        "beam selection: misaligned buffer"));
    const size_t size = dtype_size(dtype), kept = groups * keep * 4;
    const Rows ins[3] = {{d_logits, rows, ld * size, vocab * size}, {d_scores, 1, 0, rows * 4}, {d_last, 1, 0, rows * 4}};
    const Rows outs[3] = {{d_parents, 1, 0, kept}, {d_out_scores, 1, 0, kept}, {d_tokens, 1, 0, kept}};
    for (int o = 0; o < 3; ++o) {
      for (int i = 0; i < 3; ++i) {
        const bool in_place = o && o == i && keep == beams && outs[o].p == ins[i].p;
        PSSA_RETURN_IF(need(in_place || apart(outs[o], ins[i]), "beam selection: an output overlaps an input"));
      }
      for (int i = 0; i < o; ++i) PSSA_RETURN_IF(need(apart(outs[o], outs[i]), "beam selection: the outputs overlap"));
    }
    PSSA_RETURN_IF(check_ctx(ctx));
    pssa::BeamArgs a;
    a.logits = d_logits;
    a.ld = ld;
    a.vocab = (int)vocab;
    a.beams = (int)beams;
    a.keep = (int)keep;
    a.scores = d_scores;
    a.last = d_last;
    a.eos = eos;
    a.parents = d_parents;
    a.tokens = d_tokens;
    a.out_scores = d_out_scores;
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    return select_beams(ctx, dtype, a, groups);
  }, err, err_len);
}

int pssa_hip_beam_select_reserve(pssa_hip_ctx* ctx, size_t groups, size_t beams, size_t vocab, size_t keep, char* err,
                                 size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(check_beams(groups, beams, vocab, keep));
    PSSA_RETURN_IF(check_ctx(ctx));
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    const size_t rows = groups * beams;
    return grow_scratch(ctx, std::max(pssa::beam_plan(PSSA_HIP_F32, rows, vocab, keep).bytes,
                                      pssa::beam_plan(PSSA_HIP_BF16, rows, vocab, keep).bytes), false);
  }, err, err_len);
}

int pssa_hip_beam_gather_resident(pssa_hip_ctx* ctx, const void* d_src, size_t ld_src, void* d_dst, size_t ld_dst,
                                  size_t row_bytes, size_t groups, size_t n_in, const uint32_t* d_parents,
                                  size_t n_out, char* err, size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(need(d_src && d_dst && d_parents, "beam states: null buffer"));
    PSSA_RETURN_IF(need(row_bytes && groups, "beam states: dimensions must be positive"));
    PSSA_RETURN_IF(need(n_in >= 1 && n_in <= (size_t)pssa::kMaxBeams && n_out >= 1 && n_out <= (size_t)pssa::kMaxBeams,
                        "beam states: rows of a group must be in 1..=64"));
    PSSA_RETURN_IF(need(ld_src >= row_bytes && ld_dst >= row_bytes, "beam states: row stride below the row"));
    PSSA_RETURN_IF(need(row_bytes <= ((size_t)1 << 38) && groups <= INT32_MAX / pssa::kMaxBeams, "beam states: too large"));
    size_t n = 0;
    PSSA_RETURN_IF(pssa::checked_count({groups, n_in, ld_src}, &n, "beam states"));
    PSSA_RETURN_IF(pssa::checked_count({groups, n_out, ld_dst}, &n, "beam states"));
    PSSA_RETURN_IF(need(aligned_to(d_parents, 4), "beam states: misaligned buffer"));
    const Rows src{d_src, groups * n_in, ld_src, row_bytes}, dst{d_dst, groups * n_out, ld_dst, row_bytes};
    const bool in_place = d_src == d_dst && n_in == n_out && ld_src == ld_dst;
    PSSA_RETURN_IF(need(in_place || apart(src, dst), "beam states: the rows overlap"));
    PSSA_RETURN_IF(need(apart(dst, Rows{d_parents, 1, 0, groups * n_out * 4}), "beam states: the rows overlap the parents"));
    pssa::GatherArgs a;
    a.src = d_src;
    a.dst = d_dst;
    a.ld_src = ld_src;
    a.ld_dst = ld_dst;
    a.row_bytes = row_bytes;
    a.groups = (int)groups;
    a.n_in = (int)n_in;
    a.n_out = (int)n_out;
    a.parents = d_parents;
    PSSA_RETURN_IF(need(row_bytes / pssa::beam_gather_piece(a) <= pssa::kMostThreads, "beam states: too large"));
    PSSA_RETURN_IF(check_ctx(ctx));
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    return pssa::launch_beam_gather(ctx->stream, a);
  }, err, err_len);
}

int pssa_hip_beam_search(pssa_hip_lanes* L, size_t n_groups, size_t beams, size_t steps, uint32_t eos,
                         uint32_t* out_ids, size_t out_len, float* out_scores, size_t scores_len, char* err,
                         size_t err_len) {
  return guarded([&]() -> Status {
    PSSA_RETURN_IF(need(L && out_ids && out_scores, "beam search: null argument"));
    PSSA_RETURN_IF(need(beams >= 1 && beams <= (size_t)pssa::kMaxBeams, "beam search: beams must be in 1..=64"));
    PSSA_RETURN_IF(need(steps >= 1 && steps <= (1u << 20), "beam search: steps must be in 1..=2^20"));
    PSSA_RETURN_IF(need(n_groups >= 1 && n_groups <= L->lanes && n_groups * beams <= L->lanes,
                        "beam search: n_groups*beams must be in 1..=lanes"));
    const size_t n = n_groups * beams, V = L->model->cfg.d_vocab;
    PSSA_RETURN_IF(need(out_len == n * steps && scores_len == n,
                        "beam search: out_ids must be [n_groups, beams, steps] and out_scores [n_groups, beams]"));
    PSSA_RETURN_IF(need(V >= 2, "beam search: the vocabulary has no token but 0"));
    pssa_hip_ctx* ctx = L->ctx;
    std::lock_guard<std::mutex> g(ctx->mu);
    PSSA_RETURN_IF(need(L->logit_lanes == n_groups, "beam search continues the last prefill of n_groups lanes"));
    if (L->rep_penalty != 1.0f || L->temperature > 0.0f)
      return Status{PSSA_HIP_EUNSUPPORTED, "beam search runs without a repetition penalty or a sampling temperature"};
    PSSA_RETURN_IF(loops_allow_hybrid(L));
    PSSA_HIP_TRY(hipSetDevice(ctx->device));
    const hipStream_t st = ctx->stream;
    const pssa_hip_config& c = L->model->cfg;
    const size_t carry = c.depth * L->loops * c.d_latent * c.d_state;
    DevBuf parents, tokens, scores, start;
    PSSA_RETURN_IF(parents.alloc(steps * n * 4, &ctx->pool));
    PSSA_RETURN_IF(tokens.alloc(steps * n * 4, &ctx->pool));
    PSSA_RETURN_IF(scores.alloc(n * 4, &ctx->pool));
    PSSA_RETURN_IF(start.alloc(n_groups * 4, &ctx->pool));
    PSSA_RETURN_IF(pssa::launch_fill_zero(st, start.as<float>(), n_groups));
    // From here on the lanes are no longer the prefill's.
    L->staged_lanes = L->staged_len = 0;
    L->logit_lanes = 0;
    PSSA_RETURN_IF(pssa::launch_beam_spread(st, L->carry.p, carry, carry, n_groups, beams));
    PSSA_RETURN_IF(pssa::launch_beam_spread(st, L->hist.p, pssa_hip_lanes::kHist, pssa_hip_lanes::kHist, n_groups, beams));
    PSSA_RETURN_IF(pssa::launch_beam_spread(st, L->hist_n.p, 1, 1, n_groups, beams));
    PSSA_RETURN_IF(pssa::launch_beam_spread(st, L->hist_pos.p, 1, 1, n_groups, beams));
    pssa::BeamArgs a;
    a.logits = L->logits.as<float>() + 1;
    a.ld = V;
    a.vocab = (int)(V - 1);
    a.first_id = 1;
    a.eos = eos;
    a.keep = (int)beams;
    a.out_scores = scores.as<float>();
    for (size_t t = 0; t < steps; ++t) {
      a.parents = parents.as<uint32_t>() + t * n;
      a.tokens = tokens.as<uint32_t>() + t * n;
      if (t) {
        PSSA_RETURN_IF(pssa::launch_beam_feed(st, tokens.as<uint32_t>() + (t - 1) * n, L->ids.as<uint32_t>(), n));
        PSSA_RETURN_IF(pssa::run_prefill(L, n, 1));
        a.last = tokens.as<uint32_t>() + (t - 1) * n;
      }
      a.beams = (int)(t ? beams : 1);
      a.scores = t ? scores.as<float>() : start.as<float>();
      PSSA_RETURN_IF(select_beams(ctx, PSSA_HIP_F32, a, n_groups));
      if (!t) continue;  // every beam of a group has the same state so far
      PSSA_RETURN_IF(reorder_rows(ctx, L->carry, carry * 4, n_groups, beams, a.parents));
      PSSA_RETURN_IF(reorder_rows(ctx, L->hist, pssa_hip_lanes::kHist * 4, n_groups, beams, a.parents));
      PSSA_RETURN_IF(reorder_rows(ctx, L->hist_n, 4, n_groups, beams, a.parents));
      PSSA_RETURN_IF(reorder_rows(ctx, L->hist_pos, 4, n_groups, beams, a.parents));
    }
    std::vector<uint32_t> from(steps * n), id(steps * n);
    PSSA_RETURN_IF(download(ctx, from.data(), parents, steps * n * 4));
    PSSA_RETURN_IF(download(ctx, id.data(), tokens, steps * n * 4));
    PSSA_RETURN_IF(download(ctx, out_scores, scores, n * 4));
    PSSA_RETURN_IF(sync(ctx));
    // Each beam's tokens from its last one back through its parents.
    for (size_t i = 0; i < n; ++i) {
      size_t beam = i % beams;
      const size_t first = i - beam;
      for (size_t t = steps; t-- > 0;) {
        out_ids[i * steps + t] = id[t * n + first + beam];
        const uint32_t p = from[t * n + first + beam];
        if (t && p < beams) beam = p;
      }
    }
    return Status::Ok();
  }, err, err_len);
}

}  // extern "C"
