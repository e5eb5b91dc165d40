// Head norms, rotation and append in one pass for gfx950.
//
// Of every token t and query or key head x of D values, at position p and slot s:
//   y = x w / sqrt(mean(x^2) + eps)
//   z1 = y1 cos - y2 sin,  z2 = y2 cos + y1 sin   over the rot leading values, whose
//        pairs lie half of rot apart (NEOX) or next to each other; cos and sin are row
//        p of the table
// Queries go to rows of their own, keys to k_cache[s / BS, h, s % BS], values, as they
// are, to the transposed v_cache[s / BS, h, :, s % BS]; an fp8 cache holds them over
// its scale, clamped to +-448. All in fp32, rounded once where it is stored.
//
// A position outside the table makes NaN and a slot outside the cache stores nothing:
// both are the caller's fault, and neither may read or write past a buffer.

#include "cache_ops.h"
#include "common.h"

namespace {

DEVINL uint16_t to_bf16(float x) {
  return __builtin_bit_cast(uint16_t, (__bf16)x);
}

// to e4m3, clamped; NaN stays NaN
DEVINL uint8_t to_e4m3(float x) {
  const float c = x != x ? x : fminf(fmaxf(x, -448.f), 448.f);
  return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, c, 0, false);
}

}  // namespace

// Any sizes: a wave a head, whose normed values lie in LDS for the pairs.
template <bool NEOX, bool FP8>
__global__ __launch_bounds__(256) void head_norm_store_kernel(const HeadNormStore a) {
  __shared__ float rows[4][1024];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int heads = a.Hq + 2 * a.Hk;
  const int64_t item = (int64_t)blockIdx.x * 4 + wid;
  const bool on = item < (int64_t)a.T * heads;
  const int t = on ? (int)(item / heads) : 0;
  const int n = on ? (int)(item % heads) : 0;
  const int kind = n < a.Hq ? 0 : n < a.Hq + a.Hk ? 1 : 2;  // q, k, v
  const int h = kind == 0 ? n : kind == 1 ? n - a.Hq : n - a.Hq - a.Hk;
  const uint16_t* x = kind == 0   ? a.q + t * a.q_row + h * a.q_head
                      : kind == 1 ? a.k + t * a.k_row + h * a.k_head
                                  : a.v + t * a.v_row + h * a.v_head;
  float* y = rows[wid];
  float ss = 0.f;
  if (on)
    for (int d = lane; d < a.D; d += 64) {
      const float f = bf16_bits_to_f32(x[d]);
      ss = fmaf(f, f, ss);
      y[d] = f;
    }
  const float r = 1.f / sqrtf(wave_reduce_sum(ss) / a.D + a.eps);
  if (on && kind < 2)
    for (int d = lane; d < a.D; d += 64)
      y[d] *= r * bf16_bits_to_f32((kind == 0 ? a.q_w : a.k_w)[d]);
  __syncthreads();
  if (!on) return;
  const int64_t slot = kind == 0 ? 0 : a.slots[t];
  if (slot < 0 || slot >= a.num_slots) return;
  const int64_t row = (slot / a.BS) * a.Hk + h;
  const int in = (int)(slot % a.BS);
  const int p = a.positions[t], half = a.rot / 2;
  const bool known = p >= 0 && p < a.P;
  const float* cs = a.cos_sin + (int64_t)(known ? p : 0) * a.rot;
  for (int d = lane; d < a.D; d += 64) {
    float z = y[d];
    if (kind < 2 && d < a.rot) {
      const int j = NEOX ? d % half : d / 2;
      const bool second = NEOX ? d >= half : d % 2;
      const int other = NEOX ? (second ? d - half : d + half) : d ^ 1;
      const float c = known ? cs[j] : __builtin_nanf("");
      const float s = known ? cs[half + j] : __builtin_nanf("");
      z = fmaf(z, c, second ? y[other] * s : -y[other] * s);
    }
    if (kind == 0) {
      a.out[((int64_t)t * a.Hq + h) * a.D + d] = to_bf16(z);
    } else {
      const int64_t at =
          kind == 1 ? (row * a.BS + in) * a.D + d : (row * a.D + d) * a.BS + in;
      void* cache = kind == 1 ? a.k_cache : a.v_cache;
      if constexpr (FP8)
        ((uint8_t*)cache)[at] = to_e4m3(z * (kind == 1 ? a.inv_k : a.inv_v));
      else
        ((uint16_t*)cache)[at] = kind == 1 ? to_bf16(z) : x[d];
    }
  }
}

extern "C" void launch_head_norm_store(const HeadNormStore* a, bool neox, bool fp8,
                                       hipStream_t stream) {
  const int64_t items = (int64_t)a->T * (a->Hq + 2 * a->Hk);
  const dim3 grid((unsigned)((items + 3) / 4));
  auto run = [&](auto kernel) { kernel<<<grid, 256, 0, stream>>>(*a); };
  if (neox) fp8 ? run(head_norm_store_kernel<true, true>)
                : run(head_norm_store_kernel<true, false>);
  else fp8 ? run(head_norm_store_kernel<false, true>)
           : run(head_norm_store_kernel<false, false>);
}
