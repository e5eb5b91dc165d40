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
//
// What bounds it: prompts memory, 8,192 tokens of 32 and 8 heads of 128 in bf16 (206 MB)
// 38.5 us or 5.3 TB/s in a row of calls, 43 among calls on other tensors; into an fp8
// cache 36. Decode latency: one token 2.7 us, 96 4.1, 200 rows of 64 and 8 heads
// into an fp8 cache 6.1. Copies, norms and rope_and_cache() apart: one token 6.6, 8,192
// 173, those 200 rows 24.7.

#include <type_traits>

#include "cache_ops.h"
#include "common.h"
#include "decode_common.h"

namespace {

DEVINL uint16_t to_bf16(float x) {
  return __builtin_bit_cast(uint16_t, (__bf16)x);
}

// clamped to what e4m3 holds; NaN stays NaN
DEVINL float in_range(float x) {
  return x != x ? x : __builtin_amdgcn_fmed3f(x, -448.f, 448.f);
}
DEVINL uint8_t to_e4m3(float x) {
  const float c = in_range(x);
  return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, c, 0, false);
}
DEVINL uint32_t pack_e4m3(const float* x) {  // four, in range
  return __builtin_amdgcn_cvt_pk_fp8_f32(
      x[2], x[3], __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false), true);
}

// eight neighbouring values
DEVINL void store8(uint16_t* dst, const float* x) {
  *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]),
                                              pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}
DEVINL void store8(uint8_t* dst, const float* x) {
  float f[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) f[r] = in_range(x[r]);
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack_e4m3(f), pack_e4m3(f + 4));
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
  if (kind > 0 && (slot < 0 || slot >= a.num_slots)) return;
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

// Vectors of 16 bytes. The first v_blocks workgroups transpose v, the others take 16
// values of a query or key head a lane: LPH lanes a head (a power of two, of which D / 16
// have values), U heads one after the other a group of lanes, for which the token's angles
// are read once.
template <int LPH, int U, bool NEOX, bool FP8, bool RUNS>
__global__ __launch_bounds__(256) void head_norm_store16_kernel(const HeadNormStore a,
                                                               const int v_blocks) {
  using C = std::conditional_t<FP8, uint8_t, uint16_t>;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  if ((int)blockIdx.x >= v_blocks) {
    // ---- queries and keys --------------------------------------------------------------
    constexpr int HPW = 64 / LPH;  // heads a wave at once
    const int heads = a.Hq + a.Hk;
    const int per_token = (heads + HPW * U - 1) / (HPW * U);
    const int64_t item = (int64_t)(blockIdx.x - v_blocks) * 4 + wid;
    const int t = (int)(item / per_token);
    if (t >= a.T) return;
    const int h0 = (int)(item % per_token) * (HPW * U) + lane / LPH;
    const int piece = lane % LPH, half = a.rot / 2;
    const bool on = piece * 16 < a.D, turned = piece * 16 < a.rot;
    // the lane's two runs of eight values
    const int i1 = !on ? 0 : NEOX && turned ? piece * 8 : piece * 16;
    const int i2 = !on ? 0 : NEOX && turned ? piece * 8 + half : piece * 16 + 8;
    const int p = a.positions[t];
    const int64_t slot = a.slots[t];
    const bool stored = slot >= 0 && slot < a.num_slots;
    bf16x8 x[U][2], w[2][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int n = min(h0 + u * HPW, heads - 1);
      const uint16_t* src = n < a.Hq ? a.q + t * a.q_row + n * a.q_head
                                     : a.k + t * a.k_row + (n - a.Hq) * a.k_head;
      x[u][0] = load_bf16x8(src + i1);
      x[u][1] = load_bf16x8(src + i2);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[i][0] = load_bf16x8((i ? a.k_w : a.q_w) + i1);
      w[i][1] = load_bf16x8((i ? a.k_w : a.q_w) + i2);
    }
    const bool known = p >= 0 && p < a.P;
    float c[8], s[8];
    if (turned) {
      const float* cs = a.cos_sin + (int64_t)(known ? p : 0) * a.rot + piece * 8;
#pragma unroll
      for (int r = 0; r < 8; r += 4) {
        *reinterpret_cast<f32x4v*>(c + r) = *reinterpret_cast<const f32x4v*>(cs + r);
        *reinterpret_cast<f32x4v*>(s + r) = *reinterpret_cast<const f32x4v*>(cs + half + r);
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        c[r] = known ? c[r] : __builtin_nanf("");
        s[r] = known ? s[r] : __builtin_nanf("");
      }
    } else {
#pragma unroll
      for (int r = 0; r < 8; ++r) c[r] = 1.f, s[r] = 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int n = h0 + u * HPW;
      const bool is_k = n >= a.Hq;
      float y[16];
      float ss = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        y[r] = bf16x8_get(x[u][r >> 3], r & 7);
        ss = fmaf(y[r], y[r], ss);
      }
      ss = on ? ss : 0.f;
#pragma unroll
      for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor(ss, o, WAVE_SIZE);
      const float rs = 1.f / sqrtf(ss / a.D + a.eps);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        y[r] *= rs * bf16x8_get(is_k ? w[1][r >> 3] : w[0][r >> 3], r & 7);
      float z[16];
      if (turned) {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int n1 = NEOX ? r : 2 * r, n2 = NEOX ? 8 + r : 2 * r + 1;
          z[n1] = fmaf(y[n1], c[r], -y[n2] * s[r]);
          z[n2] = fmaf(y[n2], c[r], y[n1] * s[r]);
        }
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) z[r] = y[r];
      }
      if (!on || n >= heads) continue;
      if (!is_k) {
        uint16_t* dst = a.out + ((int64_t)t * a.Hq + n) * a.D;
        store8(dst + i1, z);
        store8(dst + i2, z + 8);
      } else if (stored) {
        C* dst = (C*)a.k_cache +
                 (((slot / a.BS) * a.Hk + n - a.Hq) * a.BS + slot % a.BS) * a.D;
        if constexpr (FP8) {
#pragma unroll
          for (int r = 0; r < 16; ++r) z[r] *= a.inv_k;
        }
        store8(dst + i1, z);
        store8(dst + i2, z + 8);
      }
    }
    return;
  }
  // ---- values ----------------------------------------------------------------------------
  const int per_token = a.Hk * (a.D / 8);  // eights of values
  auto place = [&](int64_t slot, int h, int d) {
    return (C*)a.v_cache + (((slot / a.BS) * a.Hk + h) * a.D + d) * a.BS + slot % a.BS;
  };
  auto put = [&](int t, int64_t slot, int h, int d) {  // eight values of one token
    const bf16x8 x = load_bf16x8(a.v + t * a.v_row + h * a.v_head + d);
    C* dst = place(slot, h, d);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const float f = bf16x8_get(x, r);
      if constexpr (FP8) dst[r * a.BS] = to_e4m3(f * a.inv_v);
      else dst[r * a.BS] = to_bf16(f);
    }
  };
  if constexpr (!RUNS) {
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int t = (int)(e / per_token), i = (int)(e % per_token) * 8;
    if (t >= a.T) return;
    const int64_t slot = a.slots[t];
    if (slot >= 0 && slot < a.num_slots) put(t, slot, i / a.D, i % a.D);
  } else {
    // A wave has 32 tokens, four groups of lanes eight each, and 16 eights of values.
    // Eight neighbouring slots from a multiple of 8 on are stored at once by the group in
    // whose tokens they begin; what lies in no such run goes by itself.
    const int chunks = (per_token + 15) / 16;
    const int64_t wave = (int64_t)blockIdx.x * 4 + wid;
    // the waves of a workgroup: two chunks of two neighbouring runs of 32 tokens, whose
    // halves of a line of a page of 64 meet in one L2
    const int pairs = (chunks + 1) / 2;
    const int64_t quad = wave >> 2;
    const int t0 = (int)(quad / pairs) * 64 + (int)(wave & 1) * 32;
    const int part = (int)(quad % pairs) * 2 + (int)((wave >> 1) & 1);
    if (t0 >= a.T) return;
    const int near = t0 - 8 + lane;  // lanes 8 .. 39: this wave's tokens
    int64_t slot = lane < 48 && near >= 0 && near < a.T ? a.slots[near] : -1;
    if (slot >= a.num_slots) slot = -1;
    const bool next = slot >= 0 && __shfl_down(slot, 1, WAVE_SIZE) == slot + 1;
    const unsigned long long follows = __ballot(next);
    const unsigned long long begins = __ballot(
        slot >= 0 && slot % 8 == 0 && a.BS % 8 == 0 && ((follows >> lane) & 0x7f) == 0x7f);
    const int group = lane >> 4;
    const int earlier = (int)(begins >> (8 * group)) & 0xff;
    const int mine = (int)(begins >> (8 * group + 8)) & 0xff;
    const int before = earlier ? __ffs(earlier) - 1 : 0;  // tokens of a run from there
    const int here = mine ? __ffs(mine) - 1 : 8;
    const int i = part * 16 + (lane & 15);
    const bool on = i < per_token;
    const int h = on ? i * 8 / a.D : 0, d = on ? i * 8 % a.D : 0;
    const int tg = t0 + group * 8;
    const bool run = on && here < 8;
    bf16x8 x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (run) x[j] = load_bf16x8(a.v + (tg + here + j) * a.v_row + h * a.v_head + d);
    const int64_t s0 = __shfl(slot, 8 + 8 * group + (here & 7), WAVE_SIZE);
#pragma unroll 1
    for (int j = 0; j < 8; ++j) {
      const int64_t s1 = __shfl(slot, 8 + 8 * group + j, WAVE_SIZE);
      if (on && j >= before && j < here && s1 >= 0) put(tg + j, s1, h, d);
    }
    if (!run) return;
    C* dst = place(s0, h, d);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if constexpr (FP8) {
        uint32_t o[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float f[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            f[k] = in_range(bf16x8_get(x[4 * j + k], r) * a.inv_v);
          o[j] = pack_e4m3(f);
        }
        *reinterpret_cast<uint2*>(dst + r * a.BS) = make_uint2(o[0], o[1]);
      } else {
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t lo = reinterpret_cast<const uint32_t*>(&x[2 * j].raw)[r >> 1];
          const uint32_t hi = reinterpret_cast<const uint32_t*>(&x[2 * j + 1].raw)[r >> 1];
          o[j] = __builtin_amdgcn_perm(hi, lo, r & 1 ? 0x07060302 : 0x05040100);
        }
        *reinterpret_cast<uint4*>(dst + r * a.BS) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
  }
}

// many: as prompts are; vectors: everything lies as vectors need it
static void launch_portion(const HeadNormStore* a, bool neox, bool fp8, bool many,
                           bool vectors, hipStream_t stream) {
  if (!vectors) {
    const int64_t items = (int64_t)a->T * (a->Hq + 2 * a->Hk);
    const dim3 grid((unsigned)((items + 3) / 4));
    auto run = [&](auto kernel) { kernel<<<grid, 256, 0, stream>>>(*a); };
    if (neox) fp8 ? run(head_norm_store_kernel<true, true>)
                  : run(head_norm_store_kernel<true, false>);
    else fp8 ? run(head_norm_store_kernel<false, true>)
             : run(head_norm_store_kernel<false, false>);
    return;
  }
  const int64_t eights = (int64_t)a->Hk * (a->D / 8);
  const int64_t v_blocks =
      many ? (int64_t)ceil_div(a->T, 64) * (((eights + 15) / 16 + 1) / 2)
           : ((int64_t)a->T * eights + 255) / 256;
  auto run = [&](auto lph, auto u, auto n, auto f, auto runs) {
    constexpr int L = decltype(lph)::value, U = decltype(u)::value;
    const int64_t per_token = ceil_div(a->Hq + a->Hk, 64 / L * U);
    const unsigned blocks = (unsigned)(v_blocks + (a->T * per_token + 3) / 4);
    auto kernel = head_norm_store16_kernel<L, U, decltype(n)::value, decltype(f)::value,
                                           decltype(runs)::value>;
    kernel<<<blocks, 256, 0, stream>>>(*a, (int)v_blocks);
  };
  auto flags = [&](auto lph, auto u, auto runs) {
    const std::true_type yes;
    const std::false_type no;
    if (neox) fp8 ? run(lph, u, yes, yes, runs) : run(lph, u, yes, no, runs);
    else fp8 ? run(lph, u, no, yes, runs) : run(lph, u, no, no, runs);
  };
  auto width = [&](auto lph) {
    if (many) flags(lph, std::integral_constant<int, 2>{}, std::true_type{});
    else flags(lph, std::integral_constant<int, 1>{}, std::false_type{});
  };
  if (a->D <= 64) width(std::integral_constant<int, 4>{});
  else if (a->D <= 128) width(std::integral_constant<int, 8>{});
  else if (a->D <= 256) width(std::integral_constant<int, 16>{});
  else width(std::integral_constant<int, 32>{});
}

extern "C" void launch_head_norm_store(const HeadNormStore* a, bool neox, bool fp8,
                                       hipStream_t stream) {
  const uintptr_t at = (uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v |
                       (uintptr_t)a->q_w | (uintptr_t)a->k_w | (uintptr_t)a->out |
                       (uintptr_t)a->k_cache | (uintptr_t)a->v_cache |
                       (uintptr_t)a->cos_sin;
  const int64_t strides =
      a->q_row | a->q_head | a->k_row | a->k_head | a->v_row | a->v_head;
  const bool vectors = !(at % 16 || strides % 8 || a->D % 16 || a->rot % 16 || a->D > 512);
  // Runs of slots and two heads a lane for prompts, a token's eight values a thread for
  // decode. us without / with, 32 and 8 heads of 128 in bf16, two prompts: 256 tokens 5.6
  // / 5.5, 512 8.4 / 5.6, 2,048 21 / 11.2, 8,192 84 / 38.5 (one head a lane 40.4, four
  // 39.8); 96 and 256 requests of a slot each 4.1 / 12.3 and 6.9 / 14.8. Requests of a slot
  // each pay for the rule from 512 on, as it knows rows alone: 511 10.1, 512 17.1, 1,024
  // 30.6, where the launches apart take 31.6, 31.3 and 53.4.
  const bool many = a->T >= 512;
  // A launch has less than 2^32 threads, 2^24 workgroups: of n tokens' heads either form
  // has half of that at most, for up to 2^20 heads.
  const int n = (1 << 25) / (a->Hq + 2 * a->Hk);
  for (int64_t t0 = 0; t0 < a->T; t0 += n) {
    HeadNormStore b = *a;
    b.T = (int)(a->T - t0 < n ? a->T - t0 : n);
    b.out += t0 * a->Hq * a->D;
    b.q += t0 * a->q_row, b.k += t0 * a->k_row, b.v += t0 * a->v_row;
    b.positions += t0, b.slots += t0;
    launch_portion(&b, neox, fp8, many, vectors, stream);
  }
}
