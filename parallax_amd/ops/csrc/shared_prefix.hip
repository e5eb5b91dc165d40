// Decode attention of a batch whose sequences share prefixes, for gfx950.
//
//   s_i = cap(scale q . k_i),  o = sum_i exp(s_i - m) v_i / sum_i exp(s_i - m)
// over the tokens i < L of a row that its window leaves, a sink in the denominator.
// Row b belongs to group g = prefix_group[b] if 0 <= g < N and its length is at least
// prefix_lens[g] > 0; its tokens before prefix_lens[g] are then those of the pages of
// the group's first row, the others those of its own. All other rows have no group.
//
// One launch has two kinds of workgroups, whose parts (a maximum, a sum of weights and
// a sum of weighted values, in fp32) a second launch joins:
//
// Prefixes. The (row, query head) items of a group and key/value head are columns, 128
// a tile, 32 a wave; keys go by in tiles of 64 that all of them read:
//   S^T[64 x 32] = K . Q^T    O^T[D x 32] += V^T . P     mfma_f32_32x32x16_bf16
// K rows are taken with bits 2 and 3 of their number swapped, so that an accumulator
// half of S^T is eight neighbouring tokens, the operand of the second product: P stays
// in registers. The key tiles of all item tiles of all groups form one list, of which
// every workgroup takes an equal run.
//
// Suffixes. The tokens behind the prefix (of a row without a group: all) are decode
// attention as in paged_decode.hip: a wave copies tiles of 32 tokens into LDS of its
// own, a key/value head's query heads are 16 columns. The tiles of all rows form one
// list, dealt in equal runs to the waves, which never wait for each other.
//
// Lengths, groups and prefixes are read on the device, by every workgroup itself; the
// grid depends on sizes alone.
//
// What bounds it, replayed in graphs on several cards, 32 query heads over 8 of 128 in bf16
// unless said:
// Long prefixes by the products with the softmax's instructions beside them, and by the
// card's power: 64 rows, 64 heads over 8, 60,000 shared tokens 152 to 160 us, of which this
// launch has 143 to 151, 830 to 880 TFLOP/s, where a product of 8192^3 reaches 1,213; at
// 1.9 GHz matrix and vector units are busy 42% and 44% of the time, and neither the order of
// a turn nor how far ahead operands are read moves it. Of an fp8 cache 149 to 155, 182 to
// 189 with up to 4,000 more tokens a row. Under a softcap, whose turns are all of the kind
// for any, 203 to 210 in bf16. Suffixes by the stream of their keys and values: 8 rows over
// 100,000, where the prefix is little more than a stream too, 92 us, 4.5 TB/s. Both
// together: 256 rows over 8,000, up to 600 of their own, 98, of which the prefix alone is 58
// and the rest alone 91. Small batches by waits in a row, of lengths, lists, page numbers, a
// tile, and by the second launch: 4 rows over 700 tokens, 14 heads over 2 of 64, 11.0; 16
// rows over 500, up to 300 of their own, 15, where paged_decode.hip starts with 6. The
// second launch is 4 to 10 of each, 10 where it reads the 34 MB that 512 workgroups leave.
//
// Keys and values of 16-bit caches go to LDS by buffer instructions: behind global ones
// the compiler waits for all reads of LDS at once, 164 us where these took 151.

#include <algorithm>
#include <cfloat>
#include <climits>
#include <type_traits>

#include "cache_ops.h"
#include "common.h"
#include "decode_common.h"
#include "decode_tiles.h"

#define SP_KT 64       // keys of a prefix tile
#define SP_ITEMS 128   // items of one: 4 waves x 32
#define SP_THREADS 256
#define SP_UNIT 32     // tokens of a suffix tile
#define SP_GROUPS 256  // at most
#define SP_ROWS 4096   // at most
#define SP_SPANS 512

typedef float f32x16v __attribute__((ext_vector_type(16)));

namespace {

// tokens of a row, of those that its table has pages for
DEVINL int length(const SharedPrefix& a, int b) {
  return min(a.lens[b], a.max_blocks << a.shift);
}

DEVINL int window_start(const SharedPrefix& a, int L) {
  return a.window > 0 ? max(0, L - a.window) : 0;
}

// suffix tiles of a row's tokens [lo, L)
DEVINL int suffix_units(int lo, int L) {
  return L > lo ? (L + SP_UNIT - 1) / SP_UNIT - lo / SP_UNIT : 0;
}

DEVINL int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
DEVINL int of_lane(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }

// inclusive sum over the lanes of a wave, without LDS
DEVINL int sum_to_lane(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // of the row: 1 before
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // of the row before
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // of both before
  return v;
}

DEVINL int page_at(const SharedPrefix& a, int entry) {
  return min(max(entry, 0), a.num_pages - 1);
}

// log2(e) cap tanh(y / cap) of a product s, whose score is y, by the exponential of
// 2 y / cap: off by some 2^-22 of the cap, 2^-15 of a weight at a cap of 64, which is less
// than products in fp32 are off by. HIGH: of caps above that, below a quarter of them, by
// tanh's series, the next term of which is 2^-26 of the result: what it multiplies is y
// itself, so that caps far above the scores leave them as they are.
template <bool HIGH>
struct Cap {
  float flat, twice, cap;  // log2(e) |scale|, 2 log2(e) |scale| / cap, log2(e) cap
  DEVINL explicit Cap(const SharedPrefix& a)
      : flat(kLog2e * fabsf(a.scale)),
        twice(fminf(2.f * kLog2e * fabsf(a.scale) / fmaxf(a.softcap, 1e-30f), FLT_MAX)),
        cap(kLog2e * a.softcap) {}
  DEVINL float operator()(float s) const {
    const float y2 = s * twice;
    const float e = __builtin_amdgcn_exp2f(y2);
    float bent = cap * (1.f - 2.f * __builtin_amdgcn_rcpf(1.f + e));
    if constexpr (!HIGH) return bent;
    const float x2 = y2 * y2 * (0.25f / (kLog2e * kLog2e));  // (y / cap)^2
    const float p = fmaf(fmaf(fmaf(fmaf(62.f / 2835, x2, -17.f / 315), x2, 2.f / 15), x2,
                              -1.f / 3), x2, 1.f);
    asm volatile("" : "+v"(bent));  // both and a choice: a branch a score takes registers
    return x2 < 0.0625f ? s * flat * p : bent;
  }
};

// A sum of weights at maximum m with that of a sink, whichever is larger at 1. The weights
// go by the square of what is returned, which may lie below what an exponential gives.
DEVINL float beside_sink(float sink, float m, float& l) {
  const float g = __builtin_amdgcn_exp2f(0.5f * fminf(m - sink, 0.f));
  l = l * g * g + (sink > m ? 1.f : __builtin_amdgcn_exp2f(sink - m));  // NaN stays
  return g;
}

// n / g of n below 2^20, exactly: n + 1/2 is 1/32 at least from where a quotient changes
DEVINL int over(int n, int g) {
  return (int)(((float)n + 0.5f) * __builtin_amdgcn_rcpf((float)g));
}

template <class F>
DEVINL float over_halves(float v, F f) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v),
                                                  __float_as_uint(v), false, false);
  return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

constexpr int tiles_bytes(int D) { return 4 * SP_KT * D * 2; }
constexpr int lds_bytes(int D) {
  return tiles_bytes(D) + (3 * SP_GROUPS + SP_ITEMS + 4) * 4 + SP_SPANS * 8 + SP_ROWS * 2;
}

// What a workgroup finds of the batch, in LDS behind its tiles.
struct Lists {
  int* prefix;      // the groups' lengths
  int* count;       // rows of a group
  int* low;         // where the first window of a group's rows begins
  int* rows;        // of an item tile; [SP_ITEMS]: its group's first row, then a flag
  int2* span;       // of the first SP_SPANS rows: where a row's own tokens begin and end
  int16_t* member;  // a row's group, -1: none
  int* units;       // a row's suffix tiles; here the tiles come to lie

  // item tiles of a group, and its key tiles [*begin, result), one at least
  DEVINL int tiles(int g, int G) const { return (count[g] * G + SP_ITEMS - 1) / SP_ITEMS; }
  DEVINL int keys(int g, int* begin) const {
    const int end = (prefix[g] + SP_KT - 1) / SP_KT;
    *begin = min(low[g] / SP_KT, end - 1);
    return end;
  }
  DEVINL int key_tiles(int g) const {
    int begin;
    const int end = keys(g, &begin);
    return end - begin;
  }
  template <class F>
  DEVINL int sum_over(int groups, F f) const {  // of f(group), for groups with rows
    const int lane = threadIdx.x & 63;
    int all = 0;
    for (int g0 = 0; g0 < groups; g0 += 64) {
      const int g = g0 + lane;
      all += of_lane(sum_to_lane(g < groups && count[g] > 0 ? f(g) : 0), 63);
    }
    return all;
  }
};

// ---- prefixes ----------------------------------------------------------------------

template <int D, bool FP8, bool HIGH>
DEVINL void prefix_role(const SharedPrefix& a, const Lists& w, uint8_t* S, const int hk,
                        const int run, const int total, int per, const bool apart) {
  constexpr int KCH = D / 8;            // 16-byte chunks of a K row
  constexpr int KPER = SP_KT * KCH / SP_THREADS;  // chunks that a thread copies
  constexpr int VPER = D * 8 / SP_THREADS;
  constexpr int KSTEPS = D / 16;
  constexpr int DT = D / 32;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wid = uniform(tid >> 6);
  const int half = lane >> 5;
  const int l31 = lane & 31;
  const int G = a.Hq / a.Hk, BS = 1 << a.shift;

  constexpr int TILE = SP_KT * D;
  uint16_t* const K0 = (uint16_t*)S;  // K and V of two tiles
  uint16_t* const V0 = K0 + TILE;
  uint16_t* const K1 = V0 + TILE;
  uint16_t* const V1 = K1 + TILE;

  // ---- this workgroup's run of key tiles ------------------------------------------
  // the group that has this run: its place in the list of what is dealt
  const int begin = apart ? run : run * per;
  int g = 0, at = -1, tile0 = 0, before = 0;
  for (int g0 = 0; g0 < a.N; g0 += 64) {
    const int x = g0 + lane;
    int n = 0, t = 0;
    if (x < a.N && w.count[x] > 0) {
      t = w.tiles(x, G);
      n = t * (apart ? (w.key_tiles(x) + per - 1) / per : w.key_tiles(x));
    }
    const int ns = sum_to_lane(n), ts = sum_to_lane(t);
    const unsigned long long hit = __ballot(before + ns > begin);
    if (hit) {
      const int src = __ffsll(hit) - 1;
      g = g0 + src;
      at = begin - before - of_lane(ns, src) + of_lane(n, src);
      tile0 += of_lane(ts, src) - of_lane(t, src);
      break;
    }
    before += of_lane(ns, 63);
    tile0 += of_lane(ts, 63);
  }
  if (at < 0) return;  // nothing is left for it
  int todo = uniform(min(per, total - begin));
  if (apart) {
    const int keys = uniform(w.key_tiles(g)), n = uniform((keys + per - 1) / per);
    const int tile = uniform(at / n), i = at - tile * n;
    per = uniform((keys + n - 1) / n);  // even
    at = tile * keys + i * per;
    todo = min(per, keys - i * per);
    if (todo <= 0) return;
  }

  // ---- what a lane copies and reads -------------------------------------------------
  // A wave copies 16 tokens, which lie in one page: of K two steps of 16 values at once,
  // of V 32 rows. LDS holds both as operands are read, K as [16 tokens][step][token][16
  // values], V as [16 tokens][row][16 tokens], the two chunks of 32 bytes exchanged
  // every 8 rows: the lanes that read together then meet in no bank.
  constexpr int ES = FP8 ? 1 : 2;
  constexpr int GROUP = 16 * D;  // values of 16 tokens
  const int line = (lane >> 1) & 15, chunk = (lane & 1) ^ ((lane >> 4) & 1);
  const uint32_t page_bytes = (uint32_t)a.Hk * BS * D * ES;
  const uint32_t in_page = (wid * 16) & (BS - 1);
  const uint32_t koff =
      ((hk * BS + in_page + line) * D + (lane >> 5) * 16 + chunk * 8) * ES;
  const uint32_t voff = ((hk * D + (lane >> 1)) * BS + in_page + chunk * 8) * ES;
  // K rows in the order that swaps bits 2 and 3
  const int krow = (l31 & 0x13) | ((l31 & 4) << 1) | ((l31 & 8) >> 1);
  const int k_at = (krow >> 4) * GROUP + (krow & 15) * 16 + (half ^ ((krow >> 3) & 1)) * 8;
  const int v_at = l31 * 16 + (half ^ ((l31 >> 3) & 1)) * 8;
  auto k_frag = [&](const uint16_t* Kl, int ks, int t) INL {
    return *reinterpret_cast<const bf16x8v*>(Kl + k_at + t * 2 * GROUP + ks * 256);
  };
  auto v_frag = [&](const uint16_t* Vl, int ks, int t) INL {
    return *reinterpret_cast<const bf16x8v*>(Vl + v_at + ks * GROUP + t * 512);
  };
  // above 0 also for a scale of 0: hidden scores are multiplied by it too
  const float c = a.softcap > 0.f ? 1.f : fmaxf(fabsf(a.scale) * kLog2e, 1e-20f);
  const Cap<HIGH> capped(a);

  int done = 0;
  bool careful = false;  // a segment's second time, see part_numbers()
  while (todo > 0) {
    const int n_items = uniform(w.count[g]) * G;
    const int P = uniform(w.prefix[g]);
    int kb;
    const int kend = uniform(w.keys(g, &kb));
    kb = uniform(kb);
    const int keys = kend - kb;
    const int tile = at < keys ? 0 : uniform(at / keys);
    const int k0 = kb + at - tile * keys, k1 = min(kend, k0 + todo);

    // ---- the tile's items ---------------------------------------------------------
    const int r0 = uniform(over(tile * SP_ITEMS, G));
    const int r1 = uniform(over(min((tile + 1) * SP_ITEMS, n_items) - 1, G));
    __syncthreads();  // the buffers and the list are free
    if (wid == 0) {
      if (lane == 0) w.rows[SP_ITEMS + 1] = 0;
      int rank = 0;
      for (int b0 = 0; b0 < a.B && rank <= r1; b0 += 64) {
        const bool is = b0 + lane < a.B && w.member[b0 + lane] == g;
        const unsigned long long all = __ballot(is);
        const int mine = rank + __popcll(all & ((1ull << lane) - 1));
        if (is && mine >= r0 && mine <= r1) w.rows[mine - r0] = b0 + lane;
        if (is && mine == 0) w.rows[SP_ITEMS] = b0 + lane;
        rank += __popcll(all);
      }
    }
    __syncthreads();
    const int item = tile * SP_ITEMS + wid * 32 + l31;
    const bool on = item < n_items;
    const int r = over(min(item, n_items - 1), G);
    const int row = w.rows[r - r0];
    const int h = hk * G + min(item, n_items - 1) - r * G;
    const int lo = a.window > 0 ? window_start(a, length(a, row)) : 0;
    // constant memory: read by the scalar unit
    const auto* table = (const __attribute__((address_space(4))) int*)(
        a.tables + (size_t)uniform(w.rows[SP_ITEMS]) * a.max_blocks);
    const bool wave_on = tile * SP_ITEMS + wid * 32 < n_items;
    int lo_most = lo;
    if (a.window > 0) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1)
        lo_most = max(lo_most, __shfl_xor(lo_most, o, WAVE_SIZE));
    }
    lo_most = uniform(lo_most);
    const int lo_least = uniform(w.low[g]);
    int lo_last = 0;  // of the tile's rows, if careful
    if (careful) {
      for (int i = lane; i <= r1 - r0; i += 64)
        lo_last = max(lo_last, window_start(a, length(a, w.rows[i])));
#pragma unroll
      for (int i = 1; i < 64; i <<= 1)
        lo_last = max(lo_last, __shfl_xor(lo_last, i, WAVE_SIZE));
      lo_last = uniform(lo_last);
    }
    const int part0 = apart ? run : run + tile0 + tile;

    if (k0 == kb && half == 0 && on)
      a.p_info[(int64_t)row * a.Hq + h] =
          make_int4(part0, apart ? (keys + per - 1) / per
                                 : (begin + done + keys - 1) / per - run + 1,
                    item - tile * SP_ITEMS, 0);

    bf16x8v qf[KSTEPS];
    {
      const uint16_t* src = a.q + row * a.q_stride + h * D + half * 8;
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s) {
        qf[s] = *reinterpret_cast<const bf16x8v*>(src + s * 16);
      }
    }

    // Pages of the 16 tokens that this wave copies next, of K and of V, by the scalar
    // unit a turn before. Tokens past the end are hidden later; their place is in the
    // last page.
    int kpage, vpage;
    auto look = [&](int kt) INL {
      return page_at(a, table[min(min(kt, k1 - 1) * SP_KT + wid * 16, P - 1) >> a.shift]);
    };
    auto k_src = [&](int i) INL {
      return a.k + (uint64_t)(uint32_t)kpage * page_bytes + i * 32 * ES + koff;
    };
    auto v_src = [&](int i) INL {
      return a.v + ((uint64_t)(uint32_t)vpage * page_bytes + (uint32_t)(i * 32 * BS * ES)) +
             voff;
    };
    // where a lane's chunk i goes: a copy writes 1 KB, 16 bytes a lane
    auto to = [&](uint16_t* l, int i) INL { return l + wid * GROUP + i * 512; };
    auto copy = [&](const uint8_t* page, uint32_t off, uint32_t more, uint16_t* l) INL {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          __builtin_amdgcn_make_buffer_rsrc((void*)page, 0, (int)page_bytes, 0x00027000),
          (__attribute__((address_space(3))) void*)l, 16, off, more, 0, 0);
    };
    auto copy_k = [&](uint16_t* l, int i) INL {
      copy(a.k + (uint64_t)(uint32_t)kpage * page_bytes, koff, i * 32 * ES, to(l, i));
    };
    auto copy_v = [&](uint16_t* l, int i) INL {
      copy(a.v + (uint64_t)(uint32_t)vpage * page_bytes, voff, i * 32 * BS * ES, to(l, i));
    };
    uint64_t kraw[FP8 ? KPER : 1], vraw[FP8 ? VPER : 1];  // fp8 passes registers
    auto fetch_k = [&]() INL {
#pragma unroll
      for (int i = 0; i < KPER; ++i)
        kraw[i] = *reinterpret_cast<const uint64_t*>(k_src(i));
    };
    auto fetch_v = [&]() INL {
#pragma unroll
      for (int i = 0; i < VPER; ++i)
        vraw[i] = *reinterpret_cast<const uint64_t*>(v_src(i));
    };
    auto settle_k = [&](uint16_t* l) INL {
#pragma unroll
      for (int i = 0; i < KPER; ++i)
        *reinterpret_cast<bf16x8v*>(to(l, i) + lane * 8) =
            widen((uint32_t)kraw[i], (uint32_t)(kraw[i] >> 32));
    };
    auto settle_v = [&](uint16_t* l) INL {
#pragma unroll
      for (int i = 0; i < VPER; ++i)
        *reinterpret_cast<bf16x8v*>(to(l, i) + lane * 8) =
            widen((uint32_t)vraw[i], (uint32_t)(vraw[i] >> 32));
    };

    f32x16v o[DT] = {}, s0[2] = {}, s1[2];
    float m = kLowest, l = 0.f, lsum = 0.f;
    float mx = kLowest;  // of the scores whose weights come next
    // weights of two tokens, part j of a B operand of 16
    auto weigh = [&](const f32x16v(&s)[2], int ks, int j) INL {
      const int e = (ks & 1) * 8 + 2 * j;
      const float x = __builtin_amdgcn_exp2f(fmaf(s[ks >> 1][e], c, -m));
      const float y = __builtin_amdgcn_exp2f(fmaf(s[ks >> 1][e + 1], c, -m));
      lsum += x;
      lsum += y;
      return pack_bf16(x, y);
    };
    auto larger = [](float x, const f32x16v& s) INL {
#pragma unroll
      for (int e = 0; e < 16; ++e) x = fmaxf(x, s[e]);
      return x;
    };
    auto top_of = [&](float x) INL {
      return over_halves(x, [](float p, float q) { return fmaxf(p, q); }) * c;
    };
    // Rescaled whenever a maximum moved, which 32 items have in three turns of four: the
    // largest weight is then 1, without error. Only at moves by more than 2^8, 64 rows
    // over 60,000 tokens took 149 us for 157 on one card, but the error against 64 bits
    // goes from 1.8e-3 of the result, of which its own rounding has 1.6e-3, to 2.3e-3.
    auto raise = [&]() INL {
      if (__any(mx > m)) {
        const float m2 = fmaxf(m, mx);
        const float f = __builtin_amdgcn_exp2f(m - m2);
        m = m2;
        l *= f;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[t][e] *= f;
      }
    };
    // All copies and stores to LDS, of all waves; but those of this thread that may be
    // under way.
    auto meet = [&](auto left) INL {
      constexpr int n = decltype(left)::value;
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0x0070 | n);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    using none = std::integral_constant<int, 0>;

    // What no item sees of a tile's V may be anything, also no number, and its weight 0
    // times it: zeros in its place. Only where a mask cuts the tile for all.
    auto clean = [&](int base, uint16_t* Vl) INL {
      const int end = P - base - wid * 16, first = lo_least - base - wid * 16;
      u32x4v keep[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int tok = 8 * (i ^ ((lane >> 3) & 1)) + 2 * j;
          keep[i][j] = (tok >= first && tok < end ? 0xffffu : 0u) |
                       (tok + 1 >= first && tok + 1 < end ? 0xffff0000u : 0u);
        }
#pragma unroll 1
      for (int d = lane; d < D; d += 64) {  // rows that leave the lane's bit 3 as it is
        u32x4v* row = reinterpret_cast<u32x4v*>(Vl + wid * GROUP + d * 16);
        row[0] &= keep[0];
        row[1] &= keep[1];
      }
    };

    // What one item sees and another's window hides stays in the product, and the other's
    // weight 0 times NaN or infinity is NaN. Where that shows in a segment's sums it is gone
    // through again, carefully: a tile that has such values loses them here, and the items
    // that see them get them as they are, behind their rescaling.
    auto part_numbers = [&](int base, uint16_t* Vl) INL {
      raise();
#pragma unroll 1
      for (int tok = 0; tok < SP_KT; ++tok) {
        const bool seen = base + tok >= lo && base + tok < P;
        // value d = 32 t + 8 i + 4 half + e of the token, its chunks exchanged for odd i
        const uint16_t* at = Vl + (tok >> 4) * GROUP + half * 64 + (tok & 7);
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int i = e >> 2;
            const uint16_t x =
                at[(32 * t + 8 * i + (e & 3)) * 16 + ((tok & 8) ^ (i & 1) * 8)];
            if (seen && (x & 0x7f80) == 0x7f80) o[t][e] += bf16_bits_to_f32(x);
            if ((e & 3) == 3) __builtin_amdgcn_sched_barrier(0);
          }
      }
      __syncthreads();
      u32x4v* const mine = reinterpret_cast<u32x4v*>(Vl + wid * GROUP);
#pragma unroll 1
      for (int i = lane; i < GROUP / 8; i += 64) {
        u32x4v f = mine[i];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          f[j] &= ((f[j] & 0x7f80u) == 0x7f80u ? 0u : 0xffffu) |
                  ((f[j] & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u);
        mine[i] = f;
      }
      __syncthreads();
    };

    // A turn takes the scores of tile kt and the weights and values of the tile before,
    // which depend on nothing of this turn. It copies K of the next tile and V of its
    // own. Any turn: also the first and the last, a softcap, a mask. `odd` (0 or 1): of
    // a segment's turns, which begin with K0 and V0.
    auto cut_turn = [&](int kt, int odd) INL {
      const uint16_t* Kl = K0 + odd * (2 * TILE);
      uint16_t* Kn = K1 - odd * (2 * TILE);
      uint16_t* Vl = V1 - odd * (2 * TILE);
      uint16_t* Vn = V0 + odd * (2 * TILE);
      const bool more = kt < k1, first = kt == k0;
      if (first) meet(std::integral_constant<int, FP8 ? 0 : KPER + VPER>{});
      else meet(none{});
      if (more && !first) {  // past the last tile K's copy is the last again
        if constexpr (FP8) {
          fetch_k();
          fetch_v();
        } else {
#pragma unroll
          for (int i = 0; i < KPER; ++i) copy_k(Kn, i);
#pragma unroll
          for (int i = 0; i < VPER; ++i) copy_v(Vn, i);
        }
        vpage = kpage;
        kpage = look(kt + 2);
      }
      if (!first && (kt * SP_KT > P || (kt - 1) * SP_KT < lo_least)) {
        clean((kt - 1) * SP_KT, Vl);
        __syncthreads();
      }
      if (!first && (kt - 1) * SP_KT < lo_last && kt * SP_KT > lo_least)
        part_numbers((kt - 1) * SP_KT, Vl);
      // operands are read AHEAD products early here too
      constexpr int AHEAD = 4;
      bf16x8v fr[AHEAD];
      if (wave_on && !first) {
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) fr[n] = v_frag(Vl, n / DT, n % DT);
        raise();
        u32x4v w;
#pragma unroll
        for (int n = 0; n < 4 * DT; ++n) {
          const int ks = n / DT, t = n % DT;
          if (t == 0)
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = weigh(s0, ks, j);
          __builtin_amdgcn_sched_barrier(0);
          o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              fr[n % AHEAD], __builtin_bit_cast(bf16x8v, w), o[t], 0, 0, 0);
          if (n + AHEAD < 4 * DT)
            fr[n % AHEAD] = v_frag(Vl, (n + AHEAD) / DT, (n + AHEAD) % DT);
        }
        l += lsum;
        lsum = 0.f;
      }
      if (wave_on && more) {
        const int base = kt * SP_KT;
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) fr[n] = k_frag(Kl, n / 2, n % 2);
        s0[0] = s0[1] = f32x16v{};
#pragma unroll
        for (int n = 0; n < 2 * KSTEPS; ++n) {
          __builtin_amdgcn_sched_barrier(0);
          s0[n % 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr[n % AHEAD], qf[n / 2],
                                                              s0[n % 2], 0, 0, 0);
          if (n + AHEAD < 2 * KSTEPS)
            fr[n % AHEAD] = k_frag(Kl, (n + AHEAD) / 2, (n + AHEAD) % 2);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (a.softcap > 0.f) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              s0[t][e] = capped(s0[t][e]);
        }
        if (base + SP_KT > P || base < lo_most) {
          int begin = lo - base - 8 * half;  // tokens [begin, begin + count) are seen
          uint32_t count = max(P - lo, 0);
          asm volatile("" : "+v"(begin));  // not computed where no mask is applied
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int tok = 32 * t + 16 * (e >> 3) + (e & 7);
              s0[t][e] = (uint32_t)(tok - begin) < count ? s0[t][e] : kHidden;
            }
        }
        mx = top_of(larger(larger(s0[0][0], s0[0]), s0[1]));
      }
      if constexpr (FP8)
        if (more) {
          settle_k(Kn);
          if (!first) settle_v(Vn);
        }
    };

    // A tile seen whole behind another. The order is the one that is written here, a
    // matrix instruction and what fits beside it at a time, operands read AHEAD
    // instructions early; the compiler's own puts every read right before its use.
    auto whole_turn = [&](int kt, const uint16_t* Kl, uint16_t* Kn, const uint16_t* Vl,
                          uint16_t* Vn, f32x16v(&sn)[2], const f32x16v(&sp)[2]) INL {
      meet(none{});
      raise();
      constexpr int NS = 2 * KSTEPS, NM = NS + 4 * DT, AHEAD = 4;
      bf16x8v fr[AHEAD];
      u32x4v w[4];
      auto load = [&](int n) INL {
        fr[n % AHEAD] = n < NS ? k_frag(Kl, n % KSTEPS, n / KSTEPS)
                               : v_frag(Vl, (n - NS) / DT, (n - NS) % DT);
      };
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) load(n);
      if constexpr (FP8) {
        fetch_k();
        fetch_v();
      }
#pragma unroll
      for (int n = 0; n < NM; ++n) {
        __builtin_amdgcn_sched_barrier(0);
        if (n < NS) {
          const int t = n / KSTEPS, ks = n % KSTEPS;
          sn[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              fr[n % AHEAD], qf[ks], ks ? sn[t] : f32x16v{}, 0, 0, 0);
        } else {
          const int t = (n - NS) % DT, ks = (n - NS) / DT;
          o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              fr[n % AHEAD], __builtin_bit_cast(bf16x8v, w[ks]), o[t], 0, 0, 0);
        }
        if (n + AHEAD < NM) load(n + AHEAD);
        // 16 pairs of weights; each slice of four comes before its first product
#pragma unroll
        for (int u = 0; u < 16; ++u)
          if (u * (NM - 4) / 16 == n) w[u / 4][u % 4] = weigh(sp, u / 4, u % 4);
        if constexpr (!FP8) {
          if (n < KPER) copy_k(Kn, n);
          else if (n - KPER < VPER) copy_v(Vn, n - KPER);
        }
        if (n == KPER + VPER) {
          vpage = kpage;
          kpage = look(kt + 2);
        }
        if (n == NS) mx = larger(sn[0][0], sn[0]);
      }
      __builtin_amdgcn_sched_barrier(0);
      mx = top_of(larger(mx, sn[1]));
      l += lsum;
      lsum = 0.f;
      if constexpr (FP8) {
        settle_k(Kn);
        settle_v(Vn);
      }
    };

    // careful: the same turns for all waves, which have more barriers than one
    const int whole = careful ? max(k0 + 1, (lo_last + SP_KT - 1) / SP_KT + 1)
                              : max(max(k0 + 1, (lo_least + SP_KT - 1) / SP_KT + 1),
                                    (lo_most + SP_KT - 1) / SP_KT);
    const int cut = wave_on && a.softcap <= 0.f ? min(k1, P / SP_KT) : 0;

    // The first turn's K, and behind it what that turn would ask for: the buffers are
    // free, and short prefixes are rows of such waits.
    {
      kpage = vpage = look(k0);
      const int second = look(k0 + 1), third = look(k0 + 2);
      if constexpr (FP8) {
        fetch_k();
        fetch_v();
        settle_k(K0);
        kpage = second;
        fetch_k();
        settle_v(V0);
      } else {
#pragma unroll
        for (int i = 0; i < KPER; ++i) copy_k(K0, i);
        asm volatile("" ::: "memory");
        kpage = second;
#pragma unroll
        for (int i = 0; i < KPER; ++i) copy_k(K1, i);
#pragma unroll
        for (int i = 0; i < VPER; ++i) copy_v(V0, i);
      }
      vpage = second;
      kpage = third;
    }
    if (a.scale < 0.f)  // the sign goes with q; here, as it waits for q
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s)
        qf[s] = __builtin_bit_cast(
            bf16x8v, __builtin_bit_cast(u32x4v, qf[s]) ^ 0x80008000u);
    // Whole turns apart only of 128: with heads of 64 the compiler runs out of the 168
    // registers of three workgroups a CU. 64 heads over 8, without / with, us: 100 rows in
    // five groups over 5,000 tokens 37.7 / 39.1; of an fp8 cache 16 rows over 500 14.4 /
    // 15.1, 64 over 2,000 22.1 / 23.1, 256 over 8,000 70.7 / 67.3.
    for (int kt = k0, odd = 0; kt <= k1; ++kt, odd ^= 1) {
      if (D == 128 && odd == 0)
        for (; kt >= whole && kt + 1 < cut; kt += 2) {
          whole_turn(kt, K0, K1, V1, V0, s1, s0);
          whole_turn(kt + 1, K1, K0, V0, V1, s0, s1);
        }
      cut_turn(kt, odd);
    }
    if (a.window > 0 && !careful) {
      uint32_t any = 0;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          any |= (__float_as_uint(o[t][e]) & 0x7f800000u) + 0x00800000u;
      if (any >> 31) w.rows[SP_ITEMS + 1] = 1;
      __syncthreads();
      careful = uniform(w.rows[SP_ITEMS + 1]);
      if (careful) continue;
    }
    careful = false;

    l = over_halves(l, [](float x, float y) { return x + y; });
    if (on) {
      const int64_t part = ((int64_t)part0 * a.Hk + hk) * SP_ITEMS +
                           item - tile * SP_ITEMS;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f32x4v x;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = o[t][4 * i + e];
          *reinterpret_cast<f32x4v*>(a.p_acc + part * D + t * 32 + 8 * i + 4 * half) = x;
        }
      if (half == 0) *reinterpret_cast<f32x2v*>(a.p_ml + part * 2) = f32x2v{m, l};
    }

    todo -= k1 - k0;
    done += k1 - k0;
    at += k1 - k0;
    if (apart) break;
    const int tiles = uniform(w.tiles(g, G));
    if (at == tiles * keys) {
      at = 0;
      tile0 += tiles;
      do ++g;
      while (g < a.N && w.count[g] == 0);
      g = uniform(g);
    }
  }
}

// ---- suffixes ----------------------------------------------------------------------

template <int D, bool FP8, bool HIGH>
DEVINL void suffix_role(const SharedPrefix& a, const Lists& w, uint8_t* S, const int hk,
                        const int run, const int total, const int runs) {
  constexpr int KT = SP_UNIT;
  constexpr int ES = FP8 ? 1 : 2;
  constexpr int RB = D * ES;             // bytes a K row
  constexpr int CPR = RB / 16;
  constexpr int VB = KT * ES;            // bytes of a V row in a tile
  constexpr int TILE = KT * RB;          // bytes of K, and of V, in a tile
  constexpr int NC = TILE / 1024;        // copies of K, and of V
  constexpr int KC = D / 32;
  constexpr int MT = D / 16;
  constexpr int W = SP_THREADS / 64;
  static_assert(W * 2 * TILE <= tiles_bytes(D) && SP_ROWS * 4 <= tiles_bytes(D), "");
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wid = uniform(tid >> 6);
  const int l15 = lane & 15;
  const int l4 = lane >> 4;
  const int G = a.Hq / a.Hk, BS = 1 << a.shift;

  // ---- this wave's run of tiles --------------------------------------------------------
  const int wave = run * W + wid;
  const int per = max((total + 4 * runs - 1) / (4 * runs), 1);
  const int begin = wave * per;
  const int todo = uniform(max(0, min(per, total - begin)));
  int seq = 0, at = 0, before = 0;
  for (int b0 = 0; b0 < a.B && todo > 0; b0 += 64) {
    const int n = b0 + lane < a.B ? w.units[b0 + lane] : 0;
    const int s = sum_to_lane(n);
    const unsigned long long hit = __ballot(before + s > begin);
    if (hit) {
      const int src = __ffsll(hit) - 1;
      seq = b0 + src;
      at = begin - before - of_lane(s, src) + of_lane(n, src);
      break;
    }
    before += of_lane(s, 63);
  }
  __syncthreads();  // the list is read
  if (todo == 0) return;

  uint8_t* Kt = S + wid * (2 * TILE);
  uint8_t* Vt = Kt + TILE;
  // ---- what a lane copies: byte offsets within a page ------------------------------
  const uint32_t k_row = lane / CPR;
  const uint32_t k_ch = (lane % CPR) ^ swz_k<CPR>(k_row);
  const uint32_t v_row = lane / (VB / 16);
  const uint32_t v_tok = ((lane % (VB / 16)) ^ swz_v<FP8>(v_row)) * (16 / ES);
  const bool v_second = v_tok >= (uint32_t)BS;  // of two pages of 16
  const uint32_t v_off = (v_row * BS + (v_tok & (BS - 1))) * ES;
  const int64_t page_bytes = (int64_t)a.Hk * BS * RB;
  const int64_t head_off = (int64_t)hk * BS * RB;
  // ---- what a lane reads ------------------------------------------------------------
  const int rr = 8 * (l15 >> 2) + (l15 & 3);
  const uint32_t k_at = lds_at(Kt) + rr * RB + (l4 ^ swz_k<CPR>(rr)) * 16;
  const uint32_t v_at =
      FP8 ? lds_at(Vt) + l15 * VB + ((l4 >> 1) ^ swz_v<FP8>(l15)) * 16 + (l4 & 1) * 8
          : lds_at(Vt) + l15 * VB + (l4 ^ swz_v<FP8>(l15)) * 16;
  const float c = a.softcap > 0.f ? 1.f : fmaxf(fabsf(a.scale) * kLog2e, 1e-20f);
  const Cap<HIGH> capped(a);

  // Rows 64 at a time, one a lane: where its own tokens begin and end.
  int rows0 = -64, row_lo = 0, row_end = 0;
  unsigned long long filled = 0, grouped = 0;
  auto look = [&](int b0) INL {
    rows0 = b0;
    const int b = min(b0 + lane, a.B - 1), g = w.member[b];
    if (b0 < SP_SPANS) {
      const int2 x = w.span[min(b, SP_SPANS - 1)];
      row_lo = x.x;
      row_end = x.y;
    } else {
      row_end = length(a, b);
      row_lo = max(g >= 0 ? w.prefix[g] : 0, window_start(a, row_end));
    }
    grouped = __ballot(g >= 0);
    filled = __ballot(b0 + lane < a.B && row_lo < row_end);
  };
  // One tile after the other, across rows: while one is computed, the next is copied
  // and the pages of the one behind that are looked up.
  struct Tile {
    int row, tok, lo, end;  // a row, the tile's first token, the row's own tokens
    int p0, p1;             // pages of the tile's two halves
    int grouped;
  };
  auto row_of = [&](Tile& t, int row) INL {
    t.row = row;
    t.lo = __builtin_amdgcn_readlane(row_lo, row - rows0);
    t.end = __builtin_amdgcn_readlane(row_end, row - rows0);
    t.grouped = (int)(grouped >> (row - rows0)) & 1;
  };
  auto pages = [&](Tile& t) INL {
    // constant memory: read by the scalar unit, no vector load among the copies
    const auto* table = (const __attribute__((address_space(4))) int*)(
        a.tables + (size_t)t.row * a.max_blocks);
    t.p0 = page_at(a, table[t.tok >> a.shift]);
    t.p1 = page_at(a, table[min(a.shift == 4 ? t.tok + 16 : t.tok, t.end - 1) >> a.shift]);
  };
  auto next = [&](const Tile& t) INL {  // the same where no row has one
    Tile n = t;
    n.tok += KT;
    if (n.tok >= t.end) {
      unsigned long long rest =
          t.row >= rows0 + 63 ? 0 : filled & (~0ull << (t.row + 1 - rows0));
      while (rest == 0 && rows0 + 64 < a.B) {
        look(rows0 + 64);
        rest = filled;
      }
      if (rest == 0) return t;
      row_of(n, rows0 + __ffsll(rest) - 1);
      n.tok = n.lo & ~(KT - 1);
    }
    pages(n);
    return n;
  };
  auto issue_k = [&](const Tile& t) INL {
    const int64_t in = head_off + (int64_t)(t.tok & (BS - 1)) * RB;
    const uint8_t* b0 = a.k + t.p0 * page_bytes + in;
    const uint8_t* b1 = a.k + t.p1 * page_bytes + in;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      constexpr int RC = 64 / CPR;  // rows a copy
      const uint32_t off = k_row * RB + (k_ch ^ swz_k<CPR>(i * RC)) * 16;
      // the second 16 rows: of the second page, if pages have 16
      const uint8_t* b = i < NC / 2 ? b0 + i * 1024
                         : a.shift == 4 ? b1 + (i - NC / 2) * 1024
                                        : b0 + i * 1024;
      copy16_to_lds(b + off, Kt + i * 1024);
    }
  };
  auto issue_v = [&](const Tile& t) INL {
    const int64_t in = head_off + (int64_t)(t.tok & (BS - 1)) * ES;
    const int64_t page = v_second ? t.p1 : t.p0;
    const uint8_t* b = a.v + in + page * page_bytes + v_off;
#pragma unroll
    for (int i = 0; i < NC; ++i)
      copy16_to_lds(b + i * (1024 / VB) * BS * ES, Vt + i * 1024);
  };
  bf16x8v qf[KC];
  auto load_q = [&](int row) INL {
    const uint16_t* src = a.q + row * a.q_stride + (hk * G + min(l15, G - 1)) * D;
#pragma unroll
    for (int s = 0; s < KC; ++s)
      qf[s] = *(const bf16x8v*)(src + (FP8 ? ((s >> 1) * 4 + l4) * 16 + (s & 1) * 8
                                           : s * 32 + l4 * 8));
  };

  const float sink = a.sinks != nullptr ? a.sinks[hk * G + min(l15, G - 1)] * kLog2e
                                        : kHidden;
  look(seq & ~63);
  Tile t0 = {};
  row_of(t0, seq);
  t0.tok = (t0.lo & ~(KT - 1)) + at * KT;
  pages(t0);
  load_q(t0.row);
  issue_k(t0);
  issue_v(t0);
  // past the run the copies are of its last tile again: the count of copies in flight
  // stays the same
  Tile t1 = todo > 1 ? next(t0) : t0;
  int from = t0.tok;  // this wave's first token of the row
  f32x4v o[MT] = {};
  float m = kLowest, l = 0.f;

  for (int i = 0; i < todo; ++i) {
    const int tok = t0.tok, lo = t0.lo, L = t0.end;
    if (tok <= lo && hk == 0 && lane == 0)  // a row's first tile
      a.s_info[t0.row] =
          make_int2(wave, wave + (i + suffix_units(lo, L) - 1) / per);
    wait_copies<NC>();
    u32x4v kr[KC * ES];  // [chunk group][t]
    if constexpr (CPR == 16)
      read8<4 * RB>(kr, k_at, k_at ^ 64, k_at ^ 128, k_at ^ 192);
    else if constexpr (CPR == 8)
      read4<4 * RB>(kr, k_at, k_at ^ 64);
    else
      read2<4 * RB>(kr, k_at);
    issue_k(t1);

    // token of s[t][r]: tok + 8 l4 + 4 t + r
    f32x4v s[2] = {};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int k = 0; k < KC; ++k) {
        bf16x8v x;
        if constexpr (FP8) {
          const u32x4v r = kr[(k >> 1) * 2 + t];
          x = k & 1 ? widen(r[2], r[3]) : widen(r[0], r[1]);
        } else {
          x = __builtin_bit_cast(bf16x8v, kr[k * 2 + t]);
        }
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, qf[k], s[t], 0, 0, 0);
      }
    if (a.scale < 0.f) {  // maxima are taken of the scores of -q
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e >> 2][e & 3] = -s[e >> 2][e & 3];
    }
    if (a.softcap > 0.f) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        s[e >> 2][e & 3] = capped(s[e >> 2][e & 3]);
    }
    const bool cut = tok + KT > L || tok < lo;
    if (cut) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int k = tok + 8 * l4 + e;
        s[e >> 2][e & 3] = k >= lo && k < L ? s[e >> 2][e & 3] : kHidden;
      }
    }
    float mx = s[0][0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[e >> 2][e & 3]);
    mx = over_head(mx, [](float x, float y) { return fmaxf(x, y); }) * c;
    if (__any(mx > m)) {
      const float m2 = fmaxf(m, mx);
      const float f = __builtin_amdgcn_exp2f(m - m2);
      m = m2;
      l *= f;
#pragma unroll
      for (int t = 0; t < MT; ++t) o[t] *= f;
    }
    u32x4v pk;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float p0 = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][e & 3], c, -m));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][(e & 3) + 1], c, -m));
      l += p0 + p1;
      pk[e >> 1] = pack_bf16(p0, p1);
    }
    // Not right behind the products: where paths meet there, one of them without
    // instructions, the compiler leaves out the wait for their results (seen in what it
    // wrote, and in the last score of four).
    if (t1.row != t0.row) load_q(t1.row);

    wait_copies<NC>();
    using VR = std::conditional_t<FP8, u32x2v, u32x4v>;
    VR vr[MT];
    read_rows(vr, v_at);
    issue_v(t1);
    const Tile t2 = i + 2 < todo ? next(t1) : t1;
    bf16x8v vb[MT];
#pragma unroll
    for (int d = 0; d < MT; ++d) {
      if constexpr (FP8)
        vb[d] = widen(vr[d][0], vr[d][1]);
      else
        vb[d] = __builtin_bit_cast(bf16x8v, vr[d]);
    }
    // slots past the end, and before the row's own tokens, may hold anything:
    // weight 0 times it
    if (cut) {
      const int first = lo - tok - 8 * l4, end = L - tok - 8 * l4;
      u32x4v keep;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        keep[j] = (2 * j >= first && 2 * j < end ? 0xffffu : 0u) |
                  (2 * j + 1 >= first && 2 * j + 1 < end ? 0xffff0000u : 0u);
      asm volatile("" : "+v"(keep));  // a branch, not 32 instructions for every tile
#pragma unroll
      for (int d = 0; d < MT; ++d)
        vb[d] = __builtin_bit_cast(bf16x8v, __builtin_bit_cast(u32x4v, vb[d]) & keep);
    }
    const bf16x8v pb = __builtin_bit_cast(bf16x8v, pk);
#pragma unroll
    for (int d = 0; d < MT; ++d)
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb[d], pb, o[d], 0, 0, 0);

    // ---- out: column l15 = head, rows of O^T = d -----------------------------------------
    if (t1.row != t0.row || i + 1 == todo) {
      l = over_head(l, [](float x, float y) { return x + y; });
      if (l15 < G) {
        const int h = hk * G + l15;
        if (!t0.grouped && from <= lo && tok + KT >= L) {  // all that it sees
          const float g = beside_sink(sink, m, l);
          const float f = a.v_scale * g / l;
          uint16_t* dst = a.out + ((int64_t)t0.row * a.Hq + h) * D + l4 * 4;
#pragma unroll
          for (int t = 0; t < MT; ++t)
            *reinterpret_cast<uint2*>(dst + t * 16) =
                make_uint2(pack_bf16(o[t][0] * f * g, o[t][1] * f * g),
                           pack_bf16(o[t][2] * f * g, o[t][3] * f * g));
        } else {
          const int64_t part = (int64_t)(wave + t0.row) * a.Hq + h;
#pragma unroll
          for (int t = 0; t < MT; ++t)
            *reinterpret_cast<f32x4v*>(a.s_acc + part * D + t * 16 + l4 * 4) = o[t];
          if (l4 == 0) *reinterpret_cast<f32x2v*>(a.s_ml + part * 2) = f32x2v{m, l};
        }
      }
#pragma unroll
      for (int t = 0; t < MT; ++t) o[t] = f32x4v{};
      m = kLowest;
      l = 0.f;
      from = t1.tok;
    }
    t0 = t1;
    t1 = t2;
  }
  wait_copies<0>();
}

}  // namespace

template <int D, bool FP8, bool HIGH>
__global__ __launch_bounds__(SP_THREADS, D == 64 ? 3 : 2) void shared_prefix_kernel(
    const SharedPrefix a) {
  __shared__ __attribute__((aligned(1024))) uint8_t S[lds_bytes(D)];
  const int hk = blockIdx.x % a.Hk, run = blockIdx.x / a.Hk;
  const int tid = threadIdx.x, lane = tid & 63;
  Lists w;
  w.units = (int*)S;
  w.prefix = (int*)(S + tiles_bytes(D));
  w.count = w.prefix + SP_GROUPS;
  w.low = w.count + SP_GROUPS;
  w.rows = w.low + SP_GROUPS;
  w.span = (int2*)(w.rows + SP_ITEMS + 4);
  w.member = (int16_t*)(w.span + SP_SPANS);
  int* const sum = w.rows;  // of all units
  int L = 0, group = -1;  // of this thread's first row, asked for with the prefixes
  if (tid < a.B) {
    L = length(a, tid);
    group = a.group[tid];
  }
  for (int g = tid; g < a.N; g += SP_THREADS) {
    w.prefix[g] = a.prefix[g];
    w.count[g] = 0;
    w.low[g] = INT_MAX;
  }
  if (tid == 0) *sum = 0;
  __syncthreads();
  int mine = 0;
  for (int b = tid; b < a.B; b += SP_THREADS) {
    if (b >= SP_THREADS) {
      L = length(a, b);
      group = a.group[b];
    }
    const int g = group;
    int P = g >= 0 && g < a.N ? w.prefix[g] : 0;
    if (P <= 0 || L < P) P = 0;
    const int lo = window_start(a, L);
    w.member[b] = (int16_t)(P > 0 ? g : -1);
    if (P > 0) {
      atomicAdd(w.count + g, 1);
      atomicMin(w.low + g, lo);
    }
    const int n = suffix_units(max(P, lo), L);
    if (b < SP_SPANS) w.span[b] = make_int2(max(P, lo), L);
    w.units[b] = n;
    mine += n;
    if (blockIdx.x == 0) a.has[b] = (P > 0) + 2 * (n > 0);
  }
  mine = sum_to_lane(mine);
  if (lane == 63) atomicAdd(sum, mine);
  __syncthreads();
  const int s_total = uniform(*sum);
  const int G = a.Hq / a.Hk;
  const int tiles = w.sum_over(a.N, [&](int g) { return w.tiles(g, G); });
  const int p_total =
      w.sum_over(a.N, [&](int g) { return w.tiles(g, G) * w.key_tiles(g); });
  __syncthreads();  // the sum is read

  // Workgroups for prefixes, by what the key tiles and the suffix tiles cost.
  int p_runs = 0, per = 1;
  bool apart = false;
  if (p_total > 0) {
    p_runs = a.runs;
    if (s_total > 0) {
      // By measurement; us with 0.15 / 0.25 / 0.4 of fp8: 64 rows, 64 heads over 8, 4,000
      // shared, up to 3,000 more 54.8 / 52.2 / 61.5; of 60,000 and 4,000 180 / 181 / 194.
      // bf16, 0.18 / 0.3 / 0.5: 64 rows, 2,048 and 2,000 64.1 / 62.5 / 71.4; 256 rows,
      // 8,000 and 600 97.0 / 97.9 / 102.8; 512 rows, 500 and 500 142.7 / 141.7 / 168.4.
      const float p_cost = p_total, s_cost = s_total * (FP8 ? 0.25f : 0.3f);
      p_runs = uniform((int)(a.runs * (p_cost / (p_cost + s_cost)) + 0.5f));
      p_runs = min(max(p_runs, 1), a.runs - 1);
    }
    // Where there are no more item tiles than workgroups, each has a run of one item
    // tile's key tiles, the shortest length that this gives for all; otherwise equal runs
    // of the list of all of them. A run's begin and end cost as much as four key tiles.
    per = uniform((p_total + p_runs - 1) / p_runs);
    apart = tiles <= p_runs;
    int used = (p_total + per - 1) / per;
    while (apart) {  // ends where per is the longest group's at the latest
      used = w.sum_over(a.N, [&](int g) {
        return w.tiles(g, G) * ((w.key_tiles(g) + per - 1) / per);
      });
      if (used <= p_runs) break;
      per = uniform(max(per + 1, (int)((float)per * used / p_runs)));
    }
    p_runs = uniform(used);  // the others are for suffixes
  }
  if (run < p_runs)
    prefix_role<D, FP8, HIGH>(a, w, S, hk, run, p_total, per, apart);
  else
    suffix_role<D, FP8, HIGH>(a, w, S, hk, run - p_runs, s_total, a.runs - p_runs);
}

// Joins the parts of every row and query head, W waves each. A lane takes a part for
// the weights; groups of D / 4 lanes take the parts in turn, in a fixed order.
template <int D, int W>
__global__ __launch_bounds__(256) void shared_prefix_join_kernel(const SharedPrefix a) {
  constexpr int Q = D / 4, GROUPS = 64 / Q, AHEAD = W > 1 ? 4 : 2;
  __shared__ f32x4v sums[W > 1 ? W : 1][Q];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int h = W > 1 ? blockIdx.x : blockIdx.x * 4 + wid, b = blockIdx.y;
  if (h >= a.Hq) return;
  const int wv = W > 1 ? wid : 0;
  const int hk = h / (a.Hq / a.Hk);
  const int d = lane % Q * 4, grp = lane / Q;
  // asked for together: what is not there is not looked at
  const int has = a.has[b];
  int4 pi = a.p_info[(int64_t)b * a.Hq + h];
  int2 sr = a.s_info[b];
  uint16_t* out = a.out + ((int64_t)b * a.Hq + h) * D + d;
  if (has == 0) {  // no tokens: zeros
    if (wv == 0 && grp == 0) *reinterpret_cast<uint2*>(out) = make_uint2(0, 0);
    return;
  }
  if (!(has & 1)) pi = make_int4(0, 0, 0, 0);
  if (!(has & 2)) sr = make_int2(0, -1);
  if (has == 2 && sr.x == sr.y) return;  // finished by its wave
  const int np = pi.y, parts = np + sr.y - sr.x + 1;
  // the place of part i
  auto at = [&](int i) INL {
    return i < np ? ((int64_t)(pi.x + i) * a.Hk + hk) * SP_ITEMS + pi.z
                  : (int64_t)(sr.x + i - np + b) * a.Hq + h;
  };
  auto load = [&](int i) INL {
    return *reinterpret_cast<const f32x4v*>((i < np ? a.p_acc : a.s_acc) + at(i) * D + d);
  };
  const int first = wv * GROUPS + grp;
  float M = kLowest, l = 0.f;
  f32x4v s = {};
  for (int i0 = 0; i0 < parts; i0 += 64) {
    const int n = min(64, parts - i0);
    f32x4v x[AHEAD];  // on their way while the weights are found
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) x[j] = load(i0 + min(first + j * W * GROUPS, n - 1));
    f32x2v v = {kLowest, 0.f};
    if (lane < n)
      v = *reinterpret_cast<const f32x2v*>((i0 + lane < np ? a.p_ml : a.s_ml) +
                                           at(i0 + lane) * 2);
    const float M2 = fmaxf(M, wave_reduce_max(v[0]));
    const float f = __builtin_amdgcn_exp2f(M - M2);
    const float w = __builtin_amdgcn_exp2f(v[0] - M2);
    M = M2;
    l = l * f + wave_reduce_sum(v[1] * w);
    s *= f;
    for (int j0 = 0; j0 < n; j0 += AHEAD * W * GROUPS) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int i = j0 + first + j * W * GROUPS;
        const float y = __shfl(w, min(i, n - 1), WAVE_SIZE);
        const f32x4v z = x[j] * y;  // past the end a part again, of infinities perhaps
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += i < n ? z[e] : 0.f;
      }
      if (j0 + AHEAD * W * GROUPS < n)
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
          x[j] = load(i0 + min(j0 + first + (AHEAD + j) * W * GROUPS, n - 1));
    }
  }
#pragma unroll
  for (int o = Q; o < 64; o <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += __shfl_xor(s[e], o, WAVE_SIZE);
  if constexpr (W > 1) {
    if (grp == 0) sums[wv][lane] = s;
    __syncthreads();
    if (wv > 0) return;
#pragma unroll
    for (int k = 1; k < W; ++k) s += sums[k][lane % Q];
  }
  float g = 1.f;
  if (a.sinks != nullptr) g = beside_sink(a.sinks[h] * kLog2e, M, l);
  s *= a.v_scale * g / l;
  s *= g;
  if (grp == 0)
    *reinterpret_cast<uint2*>(out) =
        make_uint2(pack_bf16(s[0], s[1]), pack_bf16(s[2], s[3]));
}

// Workgroups of a key/value head, as many as the chip holds at once, and the item tiles
// that B rows of N groups make at most.
extern "C" void shared_prefix_plan(int B, int N, int Hq, int Hk, int D, int* runs,
                                   int* tiles) {
  *runs = std::max(2, (D == 128 ? 512 : 768) / Hk);
  *tiles = N > 0 ? (int)((int64_t)B * (Hq / Hk) / SP_ITEMS) + std::min(N, B) : 0;
}

extern "C" void launch_shared_prefix(const SharedPrefix* a, bool fp8, hipStream_t stream) {
  const dim3 grid(a->runs * a->Hk);
  auto run = [&](auto kernel) { kernel<<<grid, SP_THREADS, 0, stream>>>(*a); };
  auto pick = [&](auto high) {
    constexpr bool H = decltype(high)::value;
    if (a->D == 128) fp8 ? run(shared_prefix_kernel<128, true, H>)
                         : run(shared_prefix_kernel<128, false, H>);
    else fp8 ? run(shared_prefix_kernel<64, true, H>)
             : run(shared_prefix_kernel<64, false, H>);
  };
  // us by the exponential / the series: 256 rows over 8,000 103 / 117, 100 rows in five
  // groups over 5,000 of 64 42 / 51, 64 over 60,000 of an fp8 cache 250 / 316.
  if (a->softcap > 64.f) pick(std::true_type{});
  else pick(std::false_type{});
  // Few rows: four waves each, which share its parts. One / four, us of the call: 8
  // rows of 32 heads over 100,000 tokens 96.6 / 91.2, 256 over 8,000 98.6 / 108.6, 128 rows
  // of 64 heads over 256 tokens 26.0 / 34.6.
  const bool wide = a->B * a->Hq <= 1024;
  const dim3 heads(wide ? a->Hq : (a->Hq + 3) / 4, a->B);
  auto join = [&](auto kernel) { kernel<<<heads, 256, 0, stream>>>(*a); };
  if (a->D == 128) wide ? join(shared_prefix_join_kernel<128, 4>)
                        : join(shared_prefix_join_kernel<128, 1>);
  else wide ? join(shared_prefix_join_kernel<64, 4>)
            : join(shared_prefix_join_kernel<64, 1>);
}
