// The 8-bit key/value cache: new tokens into it (append) and a prefix back to 16 bits (read).
// Layout and number formats: rswa_cache.cuh.
#include <type_traits>

#include "rswa_cache.cuh"

namespace rswa {

namespace {

constexpr int kThreads = 128;

struct AppendKernelParams {
  CacheView c;
  const uint16_t* src[2];
  long long s_b[2], s_t[2], s_h[2];
  const int* cu;
  long long tokens;
  int per_seq;  // new tokens of every sequence (without cu)
  const int* table;
  long long table_stride;
  int batch, max_blocks;
  const int* lens;
  int* status;
  int* mirror;
};

// New tokens of sequence b: first row in src, their number, and the slots before them.  0 tokens if something is wrong.
__device__ __forceinline__ int new_tokens(const AppendKernelParams& p, int b, long long& row0, int& len) {
  len = p.lens[b];
  int n = p.per_seq;
  row0 = 0;
  bool ok = len >= 0;
  if (p.cu != nullptr) {
    const int lo = p.cu[b], hi = p.cu[b + 1];
    ok = ok && lo >= 0 && hi >= lo && hi <= p.tokens;
    row0 = lo, n = hi - lo;
  }
  if (ok && len + static_cast<long long>(n) > static_cast<long long>(p.max_blocks) * p.c.bs) ok = false;
  if (!ok) {
    raise_status(p.status, p.mirror, kErrSeqLen);
    return 0;
  }
  return n;
}
__device__ __forceinline__ int blocks_touched(int len, int n, int bs) { return n == 0 ? 0 : (len % bs + n + bs - 1) / bs; }

// One CTA per touched block, head and K or V: the block's new values stay in registers between the search for the
// largest magnitude and the rounding, so that they are read once.  The older tokens of a block are only read when the
// block's scale grows.  kPasses: 16-byte pieces of a block per thread.
// Bound by HBM (2 bytes in, 1 out per element) for prompts; for a decoding step by the latency of
// lens -> block table -> scale -> store.
template <int kD, int kPasses, bool kInt8>
__global__ void __launch_bounds__(kThreads) cache_append_kernel(const __grid_constant__ AppendKernelParams p, bool bf16) {
  constexpr int kCols = kD / 8;  // 16-byte pieces of a row
  __shared__ uint32_t s_max[kThreads / 32];
  const int lane = threadIdx.x & 31;
  const int bs = p.c.bs;
  griddep_launch();
  griddep_wait();
  // which block of which sequence: every warp counts the touched blocks of 32 sequences at a time (or divides)
  int b = 0, unit = blockIdx.x, n = 0, len = 0;
  long long row0 = 0;
  if (p.cu == nullptr) {
    const int most = (p.per_seq + 2 * bs - 2) / bs;
    b = unit / most;
    unit -= b * most;
    n = new_tokens(p, b, row0, len);
    if (unit >= blocks_touched(len, n, bs)) return;
  } else {
    bool found = false;
    for (int base = 0; base < p.batch && !found; base += 32) {
      int l = 0, m = 0;
      long long r = 0;
      if (base + lane < p.batch) m = new_tokens(p, base + lane, r, l);
      const int mine = blocks_touched(l, m, bs);
      int sum = mine;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int o = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += o;
      }
      const int total = __shfl_sync(0xffffffffu, sum, 31);
      if (unit < total) {
        const uint32_t behind = __ballot_sync(0xffffffffu, unit < sum);
        const int who = __ffs(behind) - 1;
        unit -= __shfl_sync(0xffffffffu, sum - mine, who);
        b = base + who;
        n = __shfl_sync(0xffffffffu, m, who);
        len = __shfl_sync(0xffffffffu, l, who);
        row0 = __shfl_sync(0xffffffffu, r, who);
        found = true;
      } else {
        unit -= total;
      }
    }
    if (!found) return;
  }
  const int j = len / bs + unit;  // block of the sequence
  const int page = p.table[b * p.table_stride + j];  // (looked at below: the values do not wait for it)
  const int which = blockIdx.y & 1, h = blockIdx.y >> 1;
  const int first = max(len - j * bs, 0);                                   // slots before it hold older tokens
  const int end = static_cast<int>(min(static_cast<long long>(bs), static_cast<long long>(len) + n - static_cast<long long>(j) * bs));
  const uint16_t* src = p.src[which] + (p.cu == nullptr ? b * p.s_b[which] : 0) + h * p.s_h[which] +
                        (row0 + static_cast<long long>(j) * bs - len) * p.s_t[which];  // row of the block's slot 0

  uint4 x[kPasses];
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int at = i * kThreads + threadIdx.x, row = at / kCols, col = at % kCols;
    x[i] = make_uint4(0, 0, 0, 0);
    if (row >= first && row < end) x[i] = *reinterpret_cast<const uint4*>(src + row * p.s_t[which] + col * 8);
  }
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    // magnitudes of 16-bit floats compare like their bits, NaN above infinity above the rest
    most = __vmaxu2(most, __vmaxu2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu));
    most = __vmaxu2(most, __vmaxu2(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu));
  }
  most = __reduce_max_sync(0xffffffffu, max(most & 0xffffu, most >> 16));
  if (page < 0 || page >= p.c.num_blocks) {
    raise_status(p.status, p.mirror, kErrBlockTable);
    return;
  }
  float* const scale_at = p.c.scale[which] + static_cast<long long>(page) * p.c.hkv + h;
  const float before = first > 0 ? *scale_at : 0.f;
  if (lane == 0) s_max[threadIdx.x >> 5] = most;
  __syncthreads();
  most = max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3]));
  const float amax = bf16 ? __uint_as_float(most << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(most)));
  const float need = scale_for<kInt8>(amax);
  // (a scale from elsewhere need not be a power of two: what counts is whether the values fit, at a scale with a finite reciprocal)
  const bool grows = first == 0 || amax > (kInt8 ? 127.f : 448.f) * before || before < kLeastScale || need != need;
  const float after = grows ? need : before;
  const bool poisoned = after != after;
  const float inv = 1.f / after;
  uint8_t* const dst = p.c.data[which] + (static_cast<long long>(page) * p.c.hkv + h) * bs * kD;
  if (threadIdx.x == 0 && grows) *scale_at = after;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int at = i * kThreads + threadIdx.x, row = at / kCols;
    uint2* const to = reinterpret_cast<uint2*>(dst) + at;
    if (poisoned) {
      if (row < end) *to = make_uint2(0, 0);
    } else if (row >= first && row < end) {
      const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
      float2 f[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        f[k] = bf16 ? make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u))
                    : __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
      *to = make_uint2(to_bytes<kInt8>(f[0].x * inv, f[0].y * inv, f[1].x * inv, f[1].y * inv),
                       to_bytes<kInt8>(f[2].x * inv, f[2].y * inv, f[3].x * inv, f[3].y * inv));
    } else if (row < first && grows) {
      const uint2 old = *to;
      const Rescale<kInt8> to_new(before * inv);
      *to = make_uint2(to_new(old.x), to_new(old.y));
    }
  }
}

struct ReadKernelParams {
  CacheView c;
  uint16_t* dst[2];
  const int* table;
  long long table_stride;
  int batch, max_blocks, rows;
  const int* lens;
  int* status;
  int* mirror;
};

// One CTA per block of the result, head and K or V.  HBM-bound: 1 byte in, 2 out per element.
template <int kD, int kPasses, bool kInt8>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const __grid_constant__ ReadKernelParams p, bool bf16) {
  constexpr int kCols = kD / 16;  // 16-byte pieces of a stored row
  const int bs = p.c.bs;
  const int blocks = (p.rows + bs - 1) / bs;
  const int b = blockIdx.x / blocks, j = blockIdx.x - b * blocks;
  const int which = blockIdx.y & 1, h = blockIdx.y >> 1;
  griddep_launch();
  griddep_wait();
  const int len_b = p.lens[b];
  const int entry = j < p.max_blocks ? p.table[b * p.table_stride + j] : -1;  // (of no meaning behind the sequence's end)
  int len = min(len_b, p.rows);
  if (len_b < 0 || len_b > static_cast<long long>(p.max_blocks) * bs) {
    raise_status(p.status, p.mirror, kErrSeqLen);
    len = 0;
  }
  int held = min(max(len - j * bs, 0), bs);           // slots of this block that hold tokens
  const int wanted = min(p.rows - j * bs, bs);        // rows of the result in it
  float scale = 0.f;
  const uint8_t* src = nullptr;
  if (held > 0) {
    if (entry >= 0 && entry < p.c.num_blocks) {
      const long long at = static_cast<long long>(entry) * p.c.hkv + h;
      scale = p.c.scale[which][at];
      src = p.c.data[which] + at * bs * kD;
    } else {
      raise_status(p.status, p.mirror, kErrBlockTable);
      held = 0;
    }
  }
  uint16_t* const dst = p.dst[which] + ((static_cast<long long>(b) * p.rows + static_cast<long long>(j) * bs) * p.c.hkv + h) * kD;
  uint4 x[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int at = i * kThreads + threadIdx.x, row = at / kCols;
    x[i] = make_uint4(0, 0, 0, 0);
    if (row < held) x[i] = reinterpret_cast<const uint4*>(src)[at];
  }
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int at = i * kThreads + threadIdx.x, row = at / kCols, col = at % kCols;
    if (row >= wanted) continue;
    uint32_t out[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (row < held) {
      const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float4 f = to_float4<kInt8>(w[k]);
        out[2 * k] = bf16 ? tc05::pack2<true>(f.x * scale, f.y * scale) : tc05::pack2<false>(f.x * scale, f.y * scale);
        out[2 * k + 1] = bf16 ? tc05::pack2<true>(f.z * scale, f.w * scale) : tc05::pack2<false>(f.z * scale, f.w * scale);
      }
    }
    tc05::st_global_v8(dst + static_cast<long long>(row) * p.c.hkv * kD + col * 16, out);
  }
}

template <typename Launch>
int by_block(int head_dim, int bs, Launch launch) {
  // (head_dim * bs of 1024 to 16384 bytes a block)
  if (head_dim == 64) {
    switch (bs) {
      case 16: return launch(std::integral_constant<int, 64>(), std::integral_constant<int, 16>());
      case 32: return launch(std::integral_constant<int, 64>(), std::integral_constant<int, 32>());
      case 64: return launch(std::integral_constant<int, 64>(), std::integral_constant<int, 64>());
      default: return launch(std::integral_constant<int, 64>(), std::integral_constant<int, 128>());
    }
  }
  switch (bs) {
    case 16: return launch(std::integral_constant<int, 128>(), std::integral_constant<int, 16>());
    case 32: return launch(std::integral_constant<int, 128>(), std::integral_constant<int, 32>());
    case 64: return launch(std::integral_constant<int, 128>(), std::integral_constant<int, 64>());
    default: return launch(std::integral_constant<int, 128>(), std::integral_constant<int, 128>());
  }
}

int launched(cudaError_t e, const char* what) {
  if (e != cudaSuccess) {
    set_error("%s: launch failed: %s", what, cudaGetErrorString(e));
    return RSWA_E_CUDA;
  }
  count_launches(1);
  return RSWA_OK;
}

bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace

int check_cache(const rswa_cache_t& c, const char* what) {
  if (c.kind != RSWA_CACHE_INT8 && c.kind != RSWA_CACHE_E4M3) {
    set_error("%s: unknown cache kind %d", what, c.kind);
    return RSWA_E_UNSUPPORTED;
  }
  if (c.head_dim != 64 && c.head_dim != 128) {
    set_error("%s: head_dim must be 64 or 128, got %d", what, c.head_dim);
    return RSWA_E_UNSUPPORTED;
  }
  if (c.block_size != 16 && c.block_size != 32 && c.block_size != 64 && c.block_size != 128) {
    set_error("%s: block_size must be 16, 32, 64 or 128, got %d", what, c.block_size);
    return RSWA_E_UNSUPPORTED;
  }
  if (c.n_kv_heads <= 0 || c.num_blocks <= 0 || c.num_blocks > 0x7fffffffLL) {
    set_error("%s: a cache needs at least one block and one head", what);
    return RSWA_E_ARG;
  }
  if (c.n_kv_heads > 32767) {
    set_error("%s: at most 32767 key/value heads", what);
    return RSWA_E_UNSUPPORTED;
  }
  if (c.k == nullptr || c.v == nullptr || c.k_scale == nullptr || c.v_scale == nullptr || off16(c.k) || off16(c.v) ||
      ((reinterpret_cast<uintptr_t>(c.k_scale) | reinterpret_cast<uintptr_t>(c.v_scale)) & 3) != 0) {
    set_error("%s: the cache's tensors must be there, keys and values 16-byte aligned", what);
    return RSWA_E_ARG;
  }
  return RSWA_OK;
}

CacheView cache_view(const rswa_cache_t& c) {
  CacheView v;
  v.data[0] = static_cast<uint8_t*>(c.k), v.data[1] = static_cast<uint8_t*>(c.v);
  v.scale[0] = c.k_scale, v.scale[1] = c.v_scale;
  v.num_blocks = static_cast<int>(c.num_blocks);
  v.hkv = c.n_kv_heads, v.bs = c.block_size, v.head_dim = c.head_dim, v.kind = c.kind;
  return v;
}

int check_table(const rswa_block_table_t& t, bool written, const int32_t* lens, const int32_t* status, int block_size, const char* what) {
  if (t.batch < 0 || t.max_blocks < 0 || (t.batch > 0 && ((t.entries == nullptr && t.max_blocks > 0) || lens == nullptr)) || status == nullptr) {
    set_error("%s: block table, lens and status are required", what);
    return RSWA_E_ARG;
  }
  if (written ? t.stride < t.max_blocks && t.batch > 1 : t.stride < 0) {
    set_error("%s: rows of a block table of blocks to write to overlap", what);
    return RSWA_E_ARG;
  }
  // (the kernels may step up to 2^14 slots beyond a sequence's end before they compare)
  if (static_cast<long long>(t.max_blocks) * block_size > 0x7ff00000LL) {
    set_error("%s: positions overflow int32", what);
    return RSWA_E_UNSUPPORTED;
  }
  return RSWA_OK;
}

}  // namespace rswa

using namespace rswa;

extern "C" int rswa_cache_append(const rswa_cache_append_params_t* p, void* stream) {
  const char* what = "rswa_cache_append";
  if (p == nullptr) {
    set_error("%s: null params", what);
    return RSWA_E_ARG;
  }
  int rc = check_cache(p->cache, what);
  if (rc == RSWA_OK) rc = check_table(p->table, true, p->lens, p->status, p->cache.block_size, what);
  if (rc != RSWA_OK) return rc;
  if (p->dtype != RSWA_DTYPE_BF16 && p->dtype != RSWA_DTYPE_FP16) {
    set_error("%s: dtype must be bf16 (0) or fp16 (1), got %d", what, p->dtype);
    return RSWA_E_UNSUPPORTED;
  }
  const int64_t batch = p->table.batch;
  if (p->tokens < 0 || p->tokens > 0x7fffffffLL || (p->cu_seqlens == nullptr && batch > 0 && p->tokens % batch != 0)) {
    set_error("%s: %lld new tokens for %lld sequences", what, static_cast<long long>(p->tokens), static_cast<long long>(batch));
    return RSWA_E_ARG;
  }
  if (p->tokens == 0 || batch == 0) return RSWA_OK;
  if (p->k == nullptr || p->v == nullptr || off16(p->k) || off16(p->v) || p->k_stride_b % 8 || p->k_stride_t % 8 || p->k_stride_h % 8 ||
      p->v_stride_b % 8 || p->v_stride_t % 8 || p->v_stride_h % 8) {
    set_error("%s: k and v must be 16-byte aligned with strides that are multiples of 8 elements", what);
    return RSWA_E_ARG;
  }
  AppendKernelParams kp;
  kp.c = cache_view(p->cache);
  kp.src[0] = static_cast<const uint16_t*>(p->k), kp.src[1] = static_cast<const uint16_t*>(p->v);
  kp.s_b[0] = p->k_stride_b, kp.s_t[0] = p->k_stride_t, kp.s_h[0] = p->k_stride_h;
  kp.s_b[1] = p->v_stride_b, kp.s_t[1] = p->v_stride_t, kp.s_h[1] = p->v_stride_h;
  kp.cu = p->cu_seqlens;
  kp.tokens = p->tokens;
  kp.per_seq = p->cu_seqlens == nullptr ? static_cast<int>(p->tokens / batch) : 0;
  kp.table = p->table.entries;
  kp.table_stride = p->table.stride;
  kp.batch = p->table.batch, kp.max_blocks = p->table.max_blocks;
  kp.lens = p->lens;
  kp.status = p->status;
  kp.mirror = status_mirror(p->status);
  // Blocks that can be touched: a sequence with n > 0 new tokens touches at most n / bs + 2, and never more than n.
  const int64_t bs = p->cache.block_size;
  const int64_t units = p->cu_seqlens == nullptr ? batch * ((kp.per_seq + 2 * bs - 2) / bs)
                                                 : (p->tokens < p->tokens / bs + 2 * batch ? p->tokens : p->tokens / bs + 2 * batch);
  if (units > 0x7fffffffLL) {
    set_error("%s: too many blocks in one call", what);
    return RSWA_E_UNSUPPORTED;
  }
  const dim3 grid(static_cast<unsigned>(units), static_cast<unsigned>(2 * p->cache.n_kv_heads));
  const bool bf16 = p->dtype == RSWA_DTYPE_BF16;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_block(p->cache.head_dim, p->cache.block_size, [&](auto d, auto n) {
    constexpr int kD = decltype(d)::value, kPasses = kD * decltype(n)::value / 8 / kThreads;
    return launched(p->cache.kind == RSWA_CACHE_INT8 ? launch_kernel(cache_append_kernel<kD, kPasses, true>, grid, kThreads, 0, s, true, kp, bf16)
                                                     : launch_kernel(cache_append_kernel<kD, kPasses, false>, grid, kThreads, 0, s, true, kp, bf16),
                    what);
  });
}

extern "C" int rswa_cache_read(const rswa_cache_read_params_t* p, void* stream) {
  const char* what = "rswa_cache_read";
  if (p == nullptr) {
    set_error("%s: null params", what);
    return RSWA_E_ARG;
  }
  int rc = check_cache(p->cache, what);
  if (rc == RSWA_OK) rc = check_table(p->table, false, p->lens, p->status, p->cache.block_size, what);
  if (rc != RSWA_OK) return rc;
  if (p->dtype != RSWA_DTYPE_BF16 && p->dtype != RSWA_DTYPE_FP16) {
    set_error("%s: dtype must be bf16 (0) or fp16 (1), got %d", what, p->dtype);
    return RSWA_E_UNSUPPORTED;
  }
  if (p->rows < 0) {
    set_error("%s: rows must be non-negative", what);
    return RSWA_E_ARG;
  }
  if (p->rows == 0 || p->table.batch == 0) return RSWA_OK;
  if (p->k == nullptr || p->v == nullptr || (reinterpret_cast<uintptr_t>(p->k) & 31) != 0 || (reinterpret_cast<uintptr_t>(p->v) & 31) != 0) {
    set_error("%s: k and v must be there and 32-byte aligned", what);
    return RSWA_E_ARG;
  }
  ReadKernelParams kp;
  kp.c = cache_view(p->cache);
  kp.dst[0] = static_cast<uint16_t*>(p->k), kp.dst[1] = static_cast<uint16_t*>(p->v);
  kp.table = p->table.entries;
  kp.table_stride = p->table.stride;
  kp.batch = p->table.batch, kp.max_blocks = p->table.max_blocks, kp.rows = p->rows;
  kp.lens = p->lens;
  kp.status = p->status;
  kp.mirror = status_mirror(p->status);
  const int64_t bs = p->cache.block_size;
  const int64_t units = p->table.batch * ((p->rows + bs - 1) / bs);
  if (units > 0x7fffffffLL) {
    set_error("%s: too many blocks in one call", what);
    return RSWA_E_UNSUPPORTED;
  }
  const dim3 grid(static_cast<unsigned>(units), static_cast<unsigned>(2 * p->cache.n_kv_heads));
  const bool bf16 = p->dtype == RSWA_DTYPE_BF16;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_block(p->cache.head_dim, p->cache.block_size, [&](auto d, auto n) {
    constexpr int kD = decltype(d)::value, kPasses = (kD * decltype(n)::value / 16 + kThreads - 1) / kThreads;
    return launched(p->cache.kind == RSWA_CACHE_INT8 ? launch_kernel(cache_read_kernel<kD, kPasses, true>, grid, kThreads, 0, s, true, kp, bf16)
                                                     : launch_kernel(cache_read_kernel<kD, kPasses, false>, grid, kThreads, 0, s, true, kp, bf16),
                    what);
  });
}
