// The 8-bit key/value cache: layout, number formats and the checks that every kernel on it makes.
//
// k, v [num_blocks, n_kv_heads, block_size, head_dim], one byte per element; k_scale, v_scale [num_blocks, n_kv_heads]
// float: value = stored * scale.  A block of one head is one contiguous piece.  A sequence's tokens lie in the blocks
// that its row of the block table names, in order: slot t in block t / block_size of the row.
//
// Scales that this library writes are powers of two, the least one that keeps the block's values in range.  A scale
// amax / top would use the int8 range better (up to one bit, half a bit on average; for e4m3, whose step follows the
// value, nothing), but every change of a block's scale or move to another block would round every value again: a token
// would lose up to half a step at each eviction.  With powers of two a move rounds only what a larger scale cannot
// hold, and a value read back to 16 bits is exact.
#pragma once
#include <cuda_fp16.h>
#include <cuda_bf16.h>

#include "rswa_common.cuh"
#include "tc05.cuh"

namespace rswa {

// device-side error codes of these kernels (the host's text goes by them)
enum : int {
  kErrBlockTable = 110,  // an entry of the block table that a sequence's length reaches is no block of the cache
  kErrSeqLen = 111,      // a length or an offset that is negative, or beyond what the table, the tokens given or the weights hold
};

struct CacheView {
  uint8_t* data[2];   // k, v
  float* scale[2];
  int num_blocks, hkv, bs, head_dim, kind;
};

// (These kernels may be brought up before the one in front of them has ended, and read after griddep_wait() what that
// one wrote: with ordinary loads, not through the read-only path.)

// the block that holds block index j of sequence b, or -1 (reported)
__device__ __forceinline__ int table_entry(const int* table, long long stride, int b, int j, int num_blocks, int* status,
                                           int* mirror) {
  const int page = table[b * stride + j];
  if (page >= 0 && page < num_blocks) return page;
  raise_status(status, mirror, kErrBlockTable);
  return -1;
}

// Least power of two 2^e with amax <= top * 2^e, e >= -100 (a block of zeros keeps a finite reciprocal).  An infinity or
// a NaN in the block makes the scale, and with it every value of the block, NaN; zeros are stored under it, so that the
// NaN reaches those who see the block's tokens and nobody who has a weight of 0 for them.
template <bool kInt8>
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  if (bits >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
  // amax = m * 2^E with m in [1, 2): 127 = 1.984375 * 2^6, 448 = 1.75 * 2^8
  const int e = static_cast<int>(bits >> 23) - (kInt8 ? 6 : 8) + ((bits & 0x7fffffu) > (kInt8 ? 0x7e0000u : 0x600000u) ? 1 : 0);
  return __uint_as_float(static_cast<uint32_t>(max(e, 127 - 100)) << 23);
}

// four floats, already divided by the scale, to four stored bytes (round to nearest even)
template <bool kInt8>
__device__ __forceinline__ uint32_t to_bytes(float a, float b, float c, float d) {
  if constexpr (kInt8) {
    // 1.5 * 2^23 + x: the low byte of the sum is round(x) in two's complement (|x| <= 127)
    const float m = 12582912.f;
    const uint32_t ab = __byte_perm(__float_as_uint(a + m), __float_as_uint(b + m), 0x0040);
    const uint32_t cd = __byte_perm(__float_as_uint(c + m), __float_as_uint(d + m), 0x0040);
    return __byte_perm(ab, cd, 0x5410);
  } else {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
  }
}

// The four bytes of a word as two registers of two fp16 numbers (every stored value is one exactly).
// kPairs: bytes 0, 1 and 2, 3; else bytes 0, 2 and 1, 3.
// int8: as 1024 + 128 + q, minus 1152.  e4m3: two converting instructions (with shifts and masks, exponents moved to where
// fp16 has them, it takes seven: 161 MB of attention tiles in 42 instead of 34 us).
template <bool kInt8, bool kPairs>
__device__ __forceinline__ void to_half2(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (kInt8) {
    const uint32_t x = w ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    uint32_t a = __byte_perm(x, 0x64646464u, kPairs ? 0x4140 : 0x4240), b = __byte_perm(x, 0x64646464u, kPairs ? 0x4342 : 0x4341);
    const __half2 l = __hsub2(*reinterpret_cast<__half2*>(&a), off), h = __hsub2(*reinterpret_cast<__half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&l);
    hi = *reinterpret_cast<const uint32_t*>(&h);
  } else {
    if (!kPairs) w = __byte_perm(w, 0, 0x3120);
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}\n" : "=r"(lo), "=r"(hi) : "r"(w));
  }
}

// the four values of a word as floats, byte 0 first
template <bool kInt8>
__device__ __forceinline__ float4 to_float4(uint32_t w) {
  uint32_t lo, hi;
  to_half2<kInt8, true>(w, lo, hi);
  const float2 l = __half22float2(*reinterpret_cast<__half2*>(&lo)), h = __half22float2(*reinterpret_cast<__half2*>(&hi));
  return make_float4(l.x, l.y, h.x, h.y);
}

// largest magnitude of a word's four values
template <bool kInt8>
__device__ __forceinline__ uint32_t abs_bytes(uint32_t w) { return kInt8 ? __vabs4(w) : (w & 0x7f7f7f7fu); }  // |-128| = 128
template <bool kInt8>
__device__ __forceinline__ float byte_to_float(uint32_t b) {  // of a magnitude
  if constexpr (kInt8) return static_cast<float>(b);
  return __half2float(__ushort_as_half(static_cast<unsigned short>(b << 7))) * 256.f;
}

// host side
int check_cache(const rswa_cache_t& c, const char* what);
CacheView cache_view(const rswa_cache_t& c);

}  // namespace rswa
