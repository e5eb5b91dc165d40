// Bindings of the operators around a paged cache that many sequences share: head norms
// with rotation and append (head_norm_store.hip), decode attention over shared prefixes
// (shared_prefix.hip).
//
// Every argument is looked at before the device is, so that a call is refused the same
// way wherever its tensors lie.

#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <torch/extension.h>

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <initializer_list>
#include <optional>
#include <utility>

#include "cache_ops.h"

extern "C" {
void launch_head_norm_store(const HeadNormStore*, bool, bool, hipStream_t);
void shared_prefix_plan(int, int, int, int, int, int*, int*);
void launch_shared_prefix(const SharedPrefix*, bool, hipStream_t);
}

namespace {

using torch::Tensor;

void check_type(const Tensor& t, at::ScalarType type, const char* name) {
  TORCH_CHECK(t.scalar_type() == type, name, " must be ", type, ", not ",
              t.scalar_type());
}

void check_list(const Tensor& t, at::ScalarType type, int64_t n, const char* name) {
  check_type(t, type, name);
  TORCH_CHECK(t.dim() == 1 && t.size(0) == n && t.is_contiguous(), name,
              " must have one value for each of ", n, ", contiguous");
}

// rows of heads, each of neighbouring values
void check_heads(const Tensor& t, const char* name) {
  check_type(t, at::kBFloat16, name);
  TORCH_CHECK(t.dim() == 3 && (t.stride(2) == 1 || t.size(2) == 1), name,
              " must be [rows, heads, values] with neighbouring values");
}

// K by rows [NB, Hk, BS, D], V transposed [NB, Hk, D, BS]
void check_cache(const Tensor& k, const Tensor& v, int64_t Hk, int64_t D) {
  TORCH_CHECK(k.scalar_type() == at::kBFloat16 ||
                  k.scalar_type() == at::kFloat8_e4m3fn,
              "k_cache must be bf16 or fp8_e4m3fn");
  check_type(v, k.scalar_type(), "v_cache");
  TORCH_CHECK(k.dim() == 4 && k.size(1) == Hk && k.size(3) == D,
              "k_cache must be [blocks, ", Hk, ", tokens, ", D, "]");
  TORCH_CHECK(v.dim() == 4 && v.size(0) == k.size(0) && v.size(1) == Hk &&
                  v.size(2) == D && v.size(3) == k.size(2),
              "v_cache must be k_cache's [blocks, heads, ", D, ", tokens]");
  TORCH_CHECK(k.is_contiguous() && v.is_contiguous(), "caches must be contiguous");
  TORCH_CHECK(k.size(0) <= INT_MAX && k.size(2) >= 1, "cache sizes");
}

void check_device(const Tensor& like, std::initializer_list<const Tensor*> others) {
  TORCH_CHECK(like.is_cuda(), "q must be on GPU");
  for (const Tensor* t : others)
    TORCH_CHECK(t->device() == like.device(), "all tensors must be on ",
                like.device(), ", not ", t->device());
}

void check_no_grad(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : tensors)
    TORCH_CHECK(!t->requires_grad(), "there is no gradient: call it under no_grad");
}

// of 32 bits, as the kernels take it and its inverse
void check_scale(double s, const char* name) {
  TORCH_CHECK(s > 0 && std::isfinite((float)s) && std::isfinite((float)(1.0 / s)), name,
              " must be above 0, itself and its inverse within 32 bits");
}

Tensor from16(const Tensor& t) { return (uintptr_t)t.data_ptr() % 16 ? t.clone() : t; }

hipStream_t stream() { return at::hip::getCurrentHIPStream().stream(); }

}  // namespace

Tensor qk_norm_rope_and_cache(Tensor q, Tensor k, Tensor v, Tensor q_weight,
                              Tensor k_weight, double eps, Tensor k_cache,
                              Tensor v_cache, Tensor positions, Tensor cos_sin,
                              Tensor slot_mapping, bool neox, double k_scale,
                              double v_scale) {
  check_heads(q, "q");
  check_heads(k, "k");
  check_heads(v, "v");
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2), Hk = k.size(1);
  TORCH_CHECK(k.size(0) == T && k.size(2) == D, "k must have q's rows and width");
  TORCH_CHECK(v.sizes() == k.sizes(), "v must have k's sizes");
  TORCH_CHECK(Hq >= 1 && Hk >= 1 && D >= 1 && D <= 1024,
              "heads of 1 to 1024 values, one at least");
  TORCH_CHECK(Hq + 2 * Hk <= 1 << 20, "at most 2^20 heads");
  check_list(q_weight, at::kBFloat16, D, "q_weight");
  check_list(k_weight, at::kBFloat16, D, "k_weight");
  check_cache(k_cache, v_cache, Hk, D);
  check_list(positions, at::kInt, T, "positions");
  check_list(slot_mapping, at::kLong, T, "slot_mapping");
  check_type(cos_sin, at::kFloat, "cos_sin");
  TORCH_CHECK(cos_sin.dim() == 2 && cos_sin.is_contiguous(),
              "cos_sin must be a contiguous table");
  const int64_t rot = cos_sin.size(1), P = cos_sin.size(0);
  TORCH_CHECK(rot % 2 == 0 && rot <= D && P <= INT_MAX && (P >= 1 || T == 0),
              "cos_sin must have a row a position, of an even width up to ", D);
  TORCH_CHECK(eps >= 0 && std::isfinite((float)eps),
              "eps must not be negative, and within 32 bits");
  TORCH_CHECK(T * (Hq + 2 * Hk) <= INT_MAX && k_cache.size(2) <= INT_MAX, "too many rows");
  check_scale(k_scale, "k_scale");
  check_scale(v_scale, "v_scale");
  check_no_grad({&q, &k, &v, &q_weight, &k_weight, &k_cache, &v_cache, &cos_sin});
  check_device(q, {&k, &v, &q_weight, &k_weight, &k_cache, &v_cache, &positions,
                   &cos_sin, &slot_mapping});
  const c10::DeviceGuard guard(q.device());
  auto out = torch::empty({T, Hq, D}, q.options());
  if (T == 0) return out;
  HeadNormStore a = {};
  a.out = (uint16_t*)out.data_ptr();
  a.q = (const uint16_t*)q.data_ptr();
  a.k = (const uint16_t*)k.data_ptr();
  a.v = (const uint16_t*)v.data_ptr();
  a.q_w = (const uint16_t*)q_weight.data_ptr();
  a.k_w = (const uint16_t*)k_weight.data_ptr();
  a.k_cache = k_cache.data_ptr();
  a.v_cache = v_cache.data_ptr();
  a.positions = positions.data_ptr<int>();
  a.cos_sin = cos_sin.data_ptr<float>();
  a.slots = slot_mapping.data_ptr<int64_t>();
  a.T = T, a.Hq = Hq, a.Hk = Hk, a.D = D, a.rot = rot, a.BS = k_cache.size(2), a.P = P;
  a.num_slots = k_cache.size(0) * k_cache.size(2);
  a.q_row = q.stride(0), a.q_head = q.stride(1);
  a.k_row = k.stride(0), a.k_head = k.stride(1);
  a.v_row = v.stride(0), a.v_head = v.stride(1);
  a.eps = (float)eps;
  a.inv_k = (float)(1.0 / k_scale), a.inv_v = (float)(1.0 / v_scale);
  launch_head_norm_store(&a, neox, k_cache.scalar_type() == at::kFloat8_e4m3fn,
                         stream());
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return out;
}

Tensor shared_prefix_attention_decode(Tensor q, Tensor k_cache, Tensor v_cache,
                                      Tensor block_tables, Tensor seq_lens,
                                      Tensor prefix_group, Tensor prefix_lens,
                                      double scale, int64_t sliding_window,
                                      double softcap, std::optional<Tensor> sinks,
                                      double k_scale, double v_scale) {
  check_heads(q, "q");
  const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2);
  TORCH_CHECK(k_cache.dim() == 4, "k_cache must be [blocks, heads, tokens, values]");
  const int64_t Hk = k_cache.size(1), BS = k_cache.size(2);
  check_cache(k_cache, v_cache, Hk, D);
  TORCH_CHECK(Hk >= 1 && Hq >= 1 && Hq % Hk == 0 && Hq / Hk <= 16,
              "query heads must be 1 to 16 times the cache's heads");
  TORCH_CHECK(D == 64 || D == 128, "head_dim must be 64 or 128");
  TORCH_CHECK(BS == 16 || BS == 32 || BS == 64, "block size must be 16/32/64");
  TORCH_CHECK(q.stride(1) == D || Hq == 1, "q's heads must be neighbours");
  check_type(block_tables, at::kInt, "block_tables");
  TORCH_CHECK(block_tables.dim() == 2 && block_tables.size(0) == B &&
                  block_tables.is_contiguous(),
              "block_tables must be [", B, ", blocks], contiguous");
  check_list(seq_lens, at::kInt, B, "seq_lens");
  check_list(prefix_group, at::kInt, B, "prefix_group");
  TORCH_CHECK(prefix_lens.dim() == 1, "prefix_lens must be a list");
  const int64_t N = prefix_lens.size(0);
  check_list(prefix_lens, at::kInt, N, "prefix_lens");
  TORCH_CHECK(B <= 4096 && N <= 256, "at most 4096 rows and 256 groups");
  const int64_t max_blocks = block_tables.size(1);
  // key tiles of all item tiles, and suffix tiles of all rows, are counted in 32 bits
  TORCH_CHECK(max_blocks * BS < INT_MAX / 4 &&
                  (B * Hq / Hk / 128 + N) * (max_blocks * BS / 64 + 1) < INT_MAX / 2 &&
                  B * (max_blocks * BS / 32 + 1) < INT_MAX / 2 &&
                  Hk * BS * D <= INT_MAX && Hq <= 65535,
              "too many tokens or heads");
  TORCH_CHECK(std::isfinite((float)scale) && std::isfinite(softcap) && softcap >= 0,
              "scale and softcap must be finite, softcap not negative, scale within 32 bits");
  if (sinks) check_list(*sinks, at::kFloat, Hq, "sinks");
  check_scale(k_scale, "k_scale");
  check_scale(v_scale, "v_scale");
  const bool fp8 = k_cache.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(!fp8 || std::isfinite((float)(scale * k_scale)),
              "scale times k_scale must be within 32 bits");
  check_no_grad({&q, &k_cache, &v_cache});
  if (sinks) check_no_grad({&*sinks});
  check_device(q, {&k_cache, &v_cache, &block_tables, &seq_lens, &prefix_group,
                   &prefix_lens});
  if (sinks) check_device(q, {&*sinks});
  const c10::DeviceGuard guard(q.device());
  auto out = torch::empty({B, Hq, D}, q.options());
  if (B == 0) return out;
  // copied to LDS and read by 16 bytes at once
  k_cache = from16(k_cache);
  v_cache = from16(v_cache);
  if ((uintptr_t)q.data_ptr() % 16 || q.stride(0) % 8) q = q.clone(at::MemoryFormat::Contiguous);
  if (max_blocks == 0 || k_cache.size(0) == 0) return out.zero_();
  SharedPrefix a = {};
  a.out = (uint16_t*)out.data_ptr();
  a.q = (const uint16_t*)q.data_ptr();
  a.k = (const uint8_t*)k_cache.data_ptr();
  a.v = (const uint8_t*)v_cache.data_ptr();
  a.tables = block_tables.data_ptr<int>();
  a.lens = seq_lens.data_ptr<int>();
  a.group = prefix_group.data_ptr<int>();
  a.prefix = prefix_lens.data_ptr<int>();
  a.sinks = sinks ? sinks->data_ptr<float>() : nullptr;
  a.B = B, a.N = N, a.Hq = Hq, a.Hk = Hk, a.D = D;
  a.shift = BS == 16 ? 4 : BS == 32 ? 5 : 6;
  a.max_blocks = max_blocks, a.num_pages = k_cache.size(0);
  a.q_stride = q.stride(0);
  a.scale = (float)(fp8 ? scale * k_scale : scale);
  a.v_scale = fp8 ? (float)v_scale : 1.f;
  // within fp32: below, nothing is left of a score; above, all of it
  a.softcap = softcap > 0 ? (float)std::clamp(softcap, 1e-30, (double)FLT_MAX) : 0.f;
  a.window = sliding_window > 0 ? (int)std::min<int64_t>(sliding_window, INT_MAX) : 0;
  int tiles;
  shared_prefix_plan(a.B, a.N, a.Hq, a.Hk, a.D, &a.runs, &tiles);
  // fp32 words: of a part its sums, then maxima and sums of weights; then where a row's
  // parts lie
  const int64_t p_items = N > 0 ? (int64_t)(a.runs + tiles) * Hk * 128 : 0;
  const int64_t s_items = (4 * a.runs + B) * Hq;
  const int64_t words = (p_items + s_items) * (D + 2) + B * Hq * 4 + B * 3;
  auto work = torch::empty({words}, q.options().dtype(at::kFloat));
  float* at = work.data_ptr<float>();
  auto take = [&](int64_t n) { return std::exchange(at, at + n); };
  a.p_acc = take(p_items * D);
  a.s_acc = take(s_items * D);
  a.p_info = (int4*)take(B * Hq * 4);
  a.p_ml = take(p_items * 2);
  a.s_ml = take(s_items * 2);
  a.s_info = (int2*)take(B * 2);
  a.has = (int*)take(B);
  launch_shared_prefix(&a, fp8, stream());
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return out;
}
