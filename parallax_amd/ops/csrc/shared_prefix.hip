// Decode attention of a batch whose sequences share prefixes, for gfx950.
//
//   s_i = cap(scale q . k_i),  o = sum_i exp(s_i - m) v_i / sum_i exp(s_i - m)
// over the tokens i < L of a row that its window leaves, a sink in the denominator.
// Row b belongs to group g = prefix_group[b] if 0 <= g < N and its length is at least
// prefix_lens[g] > 0; its tokens before prefix_lens[g] are then those of the pages of
// the group's first row, the others those of its own. All other rows have no group.

#include "common.h"
#include "decode_common.h"

struct SharedPrefix {
  uint16_t* out;           // [B, Hq, D]
  const uint16_t* q;       // [B, Hq, D] rows at q_stride
  const uint8_t *k, *v;    // [NB, Hk, BS, D], [NB, Hk, D, BS], bf16 | fp8
  const int *tables, *lens, *group, *prefix;  // [B, max_blocks], [B], [B], [N]
  const float* sinks;      // [Hq] or null
  int B, N, Hq, Hk, D, shift, max_blocks, num_pages;
  int64_t q_stride;
  float scale, v_scale, softcap;  // scale: with that of an fp8 cache's keys
  int window;
};

namespace {

constexpr float kLog2e = 1.4426950408889634f;

DEVINL int prefix_of(const SharedPrefix& a, int b) {
  const int g = a.group[b];
  const int p = g >= 0 && g < a.N ? a.prefix[g] : 0;
  return p > 0 && a.lens[b] >= p ? p : 0;
}

}  // namespace

template <bool FP8>
__global__ __launch_bounds__(64) void shared_prefix_kernel(const SharedPrefix a) {
  __shared__ float qs[128];
  const int lane = threadIdx.x, h = blockIdx.x, b = blockIdx.y;
  const int hk = h / (a.Hq / a.Hk), BS = 1 << a.shift, D = a.D;
  const int L = a.lens[b], P = prefix_of(a, b);
  const int lo = a.window > 0 ? max(0, L - a.window) : 0;
  int first = b;
  if (P > 0)
    for (int i = b - 1; i >= 0; --i)
      if (a.group[i] == a.group[b] && prefix_of(a, i) > 0) first = i;
  for (int d = lane; d < D; d += 64)
    qs[d] = bf16_bits_to_f32(a.q[b * a.q_stride + h * D + d]);
  __syncthreads();
  float m = -1e30f, l = 0.f, o[2] = {};
  for (int t0 = lo; t0 < L; t0 += 64) {
    const int tok = t0 + lane;
    const bool on = tok < L;
    const int at = min(tok, L - 1);
    const int* table = a.tables + (int64_t)(at < P ? first : b) * a.max_blocks;
    const int page = min(max(table[at >> a.shift], 0), a.num_pages - 1);
    const int64_t row = (int64_t)page * a.Hk + hk;
    const int64_t k0 = (row * BS + (at & (BS - 1))) * D;
    float s = 0.f;
    for (int d = 0; d < D; ++d)
      s = fmaf(FP8 ? fp8_e4m3_to_f32(a.k[k0 + d])
                   : bf16_bits_to_f32(((const uint16_t*)a.k)[k0 + d]), qs[d], s);
    s *= a.scale;
    if (a.softcap > 0.f) s = a.softcap * tanhf(s / a.softcap);
    s = on ? s * kLog2e : -__builtin_inff();
    const float m2 = fmaxf(m, wave_reduce_max(s));
    const float f = exp2f(m - m2), p = exp2f(s - m2);
    m = m2;
    l = l * f + p;
    o[0] *= f;
    o[1] *= f;
    for (int j = 0; j < 64 && t0 + j < L; ++j) {
      const float w = __shfl(p, j, WAVE_SIZE);
      const int64_t r = (int64_t)__shfl(page, j, WAVE_SIZE) * a.Hk + hk;
      for (int i = 0; i < D / 64; ++i) {
        const int64_t v0 = (r * D + i * 64 + lane) * BS + ((t0 + j) & (BS - 1));
        o[i] = fmaf(w, FP8 ? fp8_e4m3_to_f32(a.v[v0])
                           : bf16_bits_to_f32(((const uint16_t*)a.v)[v0]), o[i]);
      }
    }
  }
  l = wave_reduce_sum(l);
  if (a.sinks != nullptr) l += exp2f(a.sinks[h] * kLog2e - m);
  const float inv = L > 0 ? a.v_scale / l : 0.f;
  for (int i = 0; i < D / 64; ++i)
    a.out[((int64_t)b * a.Hq + h) * D + i * 64 + lane] =
        (uint16_t)pack_bf16(o[i] * inv, 0.f);
}

extern "C" void launch_shared_prefix(const SharedPrefix* a, bool fp8, hipStream_t stream) {
  const dim3 grid(a->Hq, a->B);
  auto run = [&](auto kernel) { kernel<<<grid, 64, 0, stream>>>(*a); };
  fp8 ? run(shared_prefix_kernel<true>) : run(shared_prefix_kernel<false>);
}
