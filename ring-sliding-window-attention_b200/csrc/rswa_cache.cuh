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

constexpr float kLeastScale = 7.888609052210118e-31f;  // 2^-100, of those that are written here

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

// Stored values to another scale, four at a time: round(value * ratio), ratio = old scale / new scale.
// Ratios that are powers of two (all that scales written here give) keep to packed fp16, where everything up to the one
// rounding is exact: e4m3 numbers times a power of two, then the converting instruction; int8 as 1152 + q, which an FMA
// turns into 1536 + q * ratio, whose low byte is the result.  12 instructions an element through 32-bit floats made
// the packing of an eviction wait for its arithmetic: 134 MB 69 us.
template <bool kInt8>
struct Rescale {
  float ratio;
  uint32_t mul, add;
  int how;  // 0: as they are, 1: packed, 2: through floats, 3: all zero
  __device__ __forceinline__ explicit Rescale(float r) : ratio(r), mul(0), add(0) {
    const bool pow2 = (__float_as_uint(r) & 0x807fffffu) == 0;
    how = r == 1.f ? 0 : 2;
    if (pow2 && r != 1.f) {
      if (kInt8) {
        if (r < 0.0078125f) how = 3;  // (at most 128 * 2^-8, which is rounded to 0)
        else if (r <= 32.f) how = 1;
      } else if (r >= 6.103515625e-5f && r <= 32768.f) {
        how = 1;
      }
      if (how == 1) {
        const __half2 m = __float2half2_rn(r), a = __float2half2_rn(1536.f - 1152.f * r);  // (both exact)
        mul = *reinterpret_cast<const uint32_t*>(&m);
        add = *reinterpret_cast<const uint32_t*>(&a);
      }
    }
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t w) const {
    if (how == 0) return w;
    if (how == 3) return 0;
    if (how == 2) {
      const float4 f = to_float4<kInt8>(w);
      return to_bytes<kInt8>(f.x * ratio, f.y * ratio, f.z * ratio, f.w * ratio);
    }
    uint32_t lo, hi, r;
    if (kInt8) {
      const uint32_t x = w ^ 0x80808080u;
      lo = __byte_perm(x, 0x64646464u, 0x4240), hi = __byte_perm(x, 0x64646464u, 0x4341);
      asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(lo) : "r"(mul), "r"(add));
      asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(hi) : "r"(mul), "r"(add));
      r = __byte_perm(lo, hi, 0x6240);
    } else {
      to_half2<false, true>(w, lo, hi);
      asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(lo) : "r"(mul));
      asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(hi) : "r"(mul));
      asm("{\n\t.reg .b16 a, b;\n\tcvt.rn.satfinite.e4m3x2.f16x2 a, %1;\n\tcvt.rn.satfinite.e4m3x2.f16x2 b, %2;\n\tmov.b32 %0, {a, b};\n\t}\n" : "=r"(r) : "r"(lo), "r"(hi));
    }
    return r;
  }
};

// Largest magnitude of many words' stored values: two 16-bit lanes each, since there is no packed maximum of bytes.
template <bool kInt8>
struct Largest {
  uint32_t a, b;  // e4m3: largest magnitude bits (a); int8: largest and smallest 128 + q
  __device__ __forceinline__ Largest() : a(kInt8 ? 0x00800080u : 0u), b(0x00800080u) {}
  __device__ __forceinline__ void add(uint32_t w) {
    if (kInt8) {
      const uint32_t x = w ^ 0x80808080u, e = x & 0x00ff00ffu, o = (x >> 8) & 0x00ff00ffu;
      a = __vmaxu2(a, __vmaxu2(e, o));
      b = __vminu2(b, __vminu2(e, o));
    } else {
      a = __vmaxu2(a, __vmaxu2(w & 0x007f007fu, (w >> 8) & 0x007f007fu));
    }
  }
  __device__ __forceinline__ float value() const {
    const uint32_t m = max(a & 0xffffu, a >> 16);
    if (kInt8) return static_cast<float>(max(static_cast<int>(m) - 128, 128 - static_cast<int>(min(b & 0xffffu, b >> 16))));
    return __half2float(__ushort_as_half(static_cast<unsigned short>(m << 7))) * 256.f;
  }
};

// host side
int check_cache(const rswa_cache_t& c, const char* what);
CacheView cache_view(const rswa_cache_t& c);

}  // namespace rswa
