// Tiles of 32 tokens of a paged cache, as a wave of decode attention copies them to LDS
// and reads them back as operands.
#pragma once

#include "common.h"

#define INL __attribute__((always_inline))

typedef unsigned int u32x2v __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4v __attribute__((ext_vector_type(4)));

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHidden = -__builtin_inff();  // score of a key that is not seen
constexpr float kLowest = -1e30f;              // where a maximum starts

DEVINL void copy16_to_lds(const void* src, void* dst) {
  __builtin_amdgcn_global_load_lds(
      (const __attribute__((address_space(1))) void*)src,
      (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}

template <int N>
DEVINL void wait_copies() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | ((N & 48) << 10));
  asm volatile("" ::: "memory");
}

DEVINL uint32_t lds_at(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// Operands out of LDS, each block with its own wait: before plain loads the
// compiler waits for every copy in flight.
#define RD "ds_read_b128 "
template <int OFF>
DEVINL void read2(u32x4v (&v)[2], uint32_t a) {
  asm volatile(RD "%0, %2\n\t" RD "%1, %2 offset:%3\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(v[0]), "=&v"(v[1]) : "v"(a), "n"(OFF) : "memory");
}
template <int OFF>
DEVINL void read4(u32x4v (&v)[4], uint32_t a, uint32_t b) {
  asm volatile(RD "%0, %4\n\t" RD "%1, %4 offset:%6\n\t" RD "%2, %5\n\t"
               RD "%3, %5 offset:%6\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
               : "v"(a), "v"(b), "n"(OFF) : "memory");
}
template <int OFF>
DEVINL void read8(u32x4v (&v)[8], uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile(RD "%0, %8\n\t" RD "%1, %8 offset:%12\n\t" RD "%2, %9\n\t"
               RD "%3, %9 offset:%12\n\t" RD "%4, %10\n\t"
               RD "%5, %10 offset:%12\n\t" RD "%6, %11\n\t"
               RD "%7, %11 offset:%12\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]),
                 "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
               : "v"(a), "v"(b), "v"(c), "v"(d), "n"(OFF) : "memory");
}
DEVINL void read_rows(u32x4v (&v)[4], uint32_t a) {
  asm volatile(RD "%0, %4\n\t" RD "%1, %4 offset:1*1024\n\t"
               RD "%2, %4 offset:2*1024\n\t" RD "%3, %4 offset:3*1024\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
               : "v"(a) : "memory");
}
DEVINL void read_rows(u32x4v (&v)[8], uint32_t a) {
  asm volatile(RD "%0, %8\n\t" RD "%1, %8 offset:1*1024\n\t"
               RD "%2, %8 offset:2*1024\n\t" RD "%3, %8 offset:3*1024\n\t"
               RD "%4, %8 offset:4*1024\n\t" RD "%5, %8 offset:5*1024\n\t"
               RD "%6, %8 offset:6*1024\n\t" RD "%7, %8 offset:7*1024\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]),
                 "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
               : "v"(a) : "memory");
}
#undef RD
#define RD "ds_read_b64 "
DEVINL void read_rows(u32x2v (&v)[4], uint32_t a) {
  asm volatile(RD "%0, %4\n\t" RD "%1, %4 offset:1*512\n\t"
               RD "%2, %4 offset:2*512\n\t" RD "%3, %4 offset:3*512\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
               : "v"(a) : "memory");
}
DEVINL void read_rows(u32x2v (&v)[8], uint32_t a) {
  asm volatile(RD "%0, %8\n\t" RD "%1, %8 offset:1*512\n\t"
               RD "%2, %8 offset:2*512\n\t" RD "%3, %8 offset:3*512\n\t"
               RD "%4, %8 offset:4*512\n\t" RD "%5, %8 offset:5*512\n\t"
               RD "%6, %8 offset:6*512\n\t" RD "%7, %8 offset:7*512\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]),
                 "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
               : "v"(a) : "memory");
}
#undef RD

// 8 e4m3 values to bf16, exact
DEVINL bf16x8v widen(uint32_t lo, uint32_t hi) {
  u32x4v r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true));
  return __builtin_bit_cast(bf16x8v, r);
}

// Where chunk c of a row lies: at c ^ swz(row), linear over xor in the row's bits.
// 16 lanes read at a time (0-3, 12-15 and 20-23, 24-27, ..): rows of two lane
// groups, which differ in bit 0 of the chunk. four(): 0, 2, 3, 1.
DEVINL constexpr int four(int a) { return ((a & 1) << 1) ^ ((a >> 1) & 1) * 3; }
template <int CPR>  // chunks a K row; its rows go 8 (l15 / 4) + (l15 & 3)
DEVINL constexpr int swz_k(int r) {
  return CPR == 16 ? ((r >> 3) & 3) * 4 + (r & 3)
         : CPR == 8 ? ((r >> 3) & 3) * 2 + ((r >> 1) & 1)
                    : four((r >> 3) & 3);
}
template <bool FP8>  // V rows: 4 chunks (bf16), 2 (fp8)
DEVINL constexpr int swz_v(int d) {
  return FP8 ? (d >> 3) & 1 : four((d >> 2) & 3);
}

// inclusive sum over the lanes of a wave
DEVINL int scan64(int v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int t = __shfl_up(v, o, WAVE_SIZE);
    if (lane >= o) v += t;
  }
  return v;
}

}  // namespace
