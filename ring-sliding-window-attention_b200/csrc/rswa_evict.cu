// Thinning out cached sequences by accumulated attention weight (see rswa_cache_evict in rswa.h), in two kernels:
// one chooses the slots that stay, per sequence and key/value head, the other packs their keys and values into new blocks.
#include <type_traits>

#include "rswa_cache.cuh"

namespace rswa {

int check_table(const rswa_block_table_t& t, const int32_t* lens, const int32_t* status, int block_size, const char* what);

namespace {

constexpr int kSelect = 1024;     // threads of a choosing CTA
constexpr int kBins = 2048;       // of a radix pass: 11, 11 and 10 bits
constexpr int kPack = 128;        // threads of a packing CTA

struct EvictKernelParams {
  CacheView c;
  const int* table;
  long long table_stride;
  int batch, max_blocks;
  const int* lens;
  const float* weights;
  long long w_sb, w_sh;
  int budget, n_sink, n_recent, new_w_len;
  const int* new_table;
  long long new_table_stride;
  int new_max_blocks;
  int* new_lens;
  float* new_weights;
  int* kept;
  int* status;
  int* mirror;
};

// a sequence's length, 0 (reported) if it cannot be
__device__ __forceinline__ int checked_len(const EvictKernelParams& p, int b) {
  const int len = p.lens[b];
  if (len >= 0 && len <= static_cast<long long>(p.max_blocks) * p.c.bs) return len;
  raise_status(p.status, p.mirror, kErrSeqLen);
  return 0;
}

// Bits that order like the weights, larger ones first in the order of unsigned numbers: NaN above +inf, -0 equal to 0.
__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One CTA per (sequence, head).  The k-th largest key between the sinks and the newest tokens is found digit by digit
// (11, 11, 10 bits; a histogram of the candidates' digits each time), then two ordered sweeps write what is above it and
// the first ones of those equal to it.  The weights come from L2 after the first of the five sweeps.
__global__ void __launch_bounds__(kSelect) evict_select_kernel(const __grid_constant__ EvictKernelParams p) {
  __shared__ int s_hist[kBins];
  __shared__ int s_warp[kSelect / 32], s_warp_eq[kSelect / 32];
  __shared__ int s_digit, s_left;
  griddep_wait();
  const int b = blockIdx.x / p.c.hkv, h = blockIdx.x - b * p.c.hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = checked_len(p, b);
  const int keep = min(len, p.budget);
  const float* const w = p.weights + b * p.w_sb + h * p.w_sh;
  int* const kept = p.kept + static_cast<long long>(blockIdx.x) * p.budget;
  float* const new_w = p.new_weights + static_cast<long long>(blockIdx.x) * p.new_w_len;
  if (h == 0 && threadIdx.x == 0) p.new_lens[b] = keep;
  // candidates: slots [lo, hi), of which `left` stay
  int lo = 0, hi = len, left = len;
  uint32_t bound = 0;  // keys above it stay, and `left` of those equal to it
  if (len > p.budget) {
    lo = p.n_sink, hi = len - p.n_recent;  // (n_sink + n_recent <= budget < len)
    left = p.budget - p.n_sink - p.n_recent;
    uint32_t mask = 0;
    if (left > 0) {
#pragma unroll
      for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass < 2 ? 2048 : 1024;
        for (int i = threadIdx.x; i < bins; i += kSelect) s_hist[i] = 0;
        __syncthreads();
        for (int i = lo + threadIdx.x; i < hi; i += kSelect) {
          const uint32_t key = order_key(w[i]);
          if ((key & mask) == bound) atomicAdd(&s_hist[(key >> shift) & (bins - 1)], 1);
        }
        __syncthreads();
        // the digit with which the count from above reaches `left`: every thread two bins, largest first
        const int at = bins - 1 - 2 * threadIdx.x;
        const int c0 = at >= 1 ? s_hist[at] : 0, c1 = at >= 1 ? s_hist[at - 1] : 0;
        int sum = c0 + c1;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
          const int o = __shfl_up_sync(0xffffffffu, sum, d);
          if (lane >= d) sum += o;
        }
        if (lane == 31) s_warp[warp] = sum;
        __syncthreads();
        int before = 0;
        for (int i = 0; i < warp; ++i) before += s_warp[i];
        const int above = before + sum - c0 - c1;  // keys of larger digits
        if (at >= 1 && above < left && above + c0 + c1 >= left) {
          const bool first = above + c0 >= left;
          s_digit = first ? at : at - 1;
          s_left = left - above - (first ? 0 : c0);
        }
        __syncthreads();
        left = s_left;
        bound |= static_cast<uint32_t>(s_digit) << shift;
        mask |= static_cast<uint32_t>(bins - 1) << shift;
        __syncthreads();
      }
    } else {
      bound = 0xffffffffu;  // nothing in between (a NaN would be equal to it: left is 0)
    }
  }
  // Every warp takes a contiguous piece of all slots: how many of its tokens stay, then where they go.
  const bool all = len <= p.budget;
  const int piece = (len + kSelect / 32 * 32 - 1) / (kSelect / 32 * 32) * 32;
  const int begin = min(len, warp * piece), end = min(len, begin + piece);
  int n_above = 0, n_equal = 0;
  for (int i = begin; i < end; i += 32) {
    const int slot = i + lane;
    bool above = false, equal = false;
    if (slot < end) {
      const bool must = all || slot < lo || slot >= hi;
      const uint32_t key = must ? 0 : order_key(w[slot]);
      above = must || key > bound;
      equal = !must && key == bound;
    }
    n_above += __popc(__ballot_sync(0xffffffffu, above));
    n_equal += __popc(__ballot_sync(0xffffffffu, equal));
  }
  if (lane == 0) s_warp[warp] = n_above, s_warp_eq[warp] = n_equal;
  __syncthreads();
  int at = 0, equal_before = 0;
  for (int i = 0; i < warp; ++i) {
    // (of the equal ones, those in front take the room first)
    at += s_warp[i] + max(0, min(s_warp_eq[i], left - equal_before));
    equal_before += s_warp_eq[i];
  }
  for (int i = begin; i < end; i += 32) {
    const int slot = i + lane;
    bool stays = false, equal = false;
    float x = 0.f;
    if (slot < end) {
      x = w[slot];
      const bool must = all || slot < lo || slot >= hi;
      const uint32_t key = order_key(x);
      stays = must || key > bound;
      equal = !must && key == bound;
    }
    const uint32_t before = (1u << lane) - 1;
    const uint32_t equals = __ballot_sync(0xffffffffu, equal);
    stays = stays || (equal && equal_before + __popc(equals & before) < left);
    const uint32_t stay = __ballot_sync(0xffffffffu, stays);
    if (stays) {
      const int to = at + __popc(stay & before);
      kept[to] = slot;
      if (to < p.new_w_len) new_w[to] = x;
    }
    at += __popc(stay);
    equal_before += __popc(equals);
  }
  for (int i = keep + threadIdx.x; i < p.budget; i += kSelect) kept[i] = -1;
  for (int i = keep + threadIdx.x; i < p.new_w_len; i += kSelect) new_w[i] = 0.f;
}

// One CTA per new block, head and K or V: the kept rows (scattered, head_dim bytes each) are read once, stay in
// registers while their largest magnitude is found, and are written at the new block's scale.
// Bound by HBM: one byte in, one out per element.
template <int kD, int kBs, bool kInt8>
__global__ void __launch_bounds__(kPack) evict_pack_kernel(const __grid_constant__ EvictKernelParams p) {
  constexpr int kCols = kD / 16;  // 16-byte pieces of a row
  constexpr int kPasses = (kBs * kCols + kPack - 1) / kPack;
  __shared__ long long s_row[kBs];  // offset of the row, -1: none
  __shared__ float s_scale[kBs];
  __shared__ float s_max[kPack / 32];
  __shared__ int s_nan;
  const int j = blockIdx.x % p.new_max_blocks, b = blockIdx.x / p.new_max_blocks;
  const int which = blockIdx.y & 1, h = blockIdx.y >> 1;
  griddep_wait();
  const int keep = min(checked_len(p, b), p.budget);
  const int rows = min(keep - j * kBs, kBs);
  if (rows <= 0) return;
  const int to = table_entry(p.new_table, p.new_table_stride, b, j, p.c.num_blocks, p.status, p.mirror);
  if (to < 0) return;
  const int* kept = p.kept + (static_cast<long long>(b) * p.c.hkv + h) * p.budget + static_cast<long long>(j) * kBs;
  for (int r = threadIdx.x; r < kBs; r += kPack) {
    long long at = -1;
    float scale = 0.f;
    if (r < rows) {
      const int slot = kept[r];
      const int page = table_entry(p.table, p.table_stride, b, slot / kBs, p.c.num_blocks, p.status, p.mirror);
      if (page >= 0) {
        at = static_cast<long long>(page) * p.c.hkv + h;
        scale = p.c.scale[which][at];
        at = at * kBs + slot % kBs;
      }
    }
    s_row[r] = at;
    s_scale[r] = scale;
  }
  if (threadIdx.x == 0) s_nan = 0;
  __syncthreads();
  uint4 x[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int at = i * kPack + threadIdx.x, row = at / kCols;
    x[i] = make_uint4(0, 0, 0, 0);
    if (row < rows && s_row[row] >= 0) x[i] = *reinterpret_cast<const uint4*>(p.c.data[which] + s_row[row] * kD + at % kCols * 16);
  }
  float most = 0.f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int row = (i * kPack + threadIdx.x) / kCols;
    if (row >= rows) continue;
    uint32_t m = __vmaxu4(__vmaxu4(abs_bytes<kInt8>(x[i].x), abs_bytes<kInt8>(x[i].y)), __vmaxu4(abs_bytes<kInt8>(x[i].z), abs_bytes<kInt8>(x[i].w)));
    m = __vmaxu4(m, m >> 16);
    m = max(m & 0xffu, (m >> 8) & 0xffu);
    const float scale = s_scale[row];
    most = fmaxf(most, byte_to_float<kInt8>(m) * scale);
    bad = bad || !(scale <= 3.4028235e38f);
  }
  if (bad) s_nan = 1;
#pragma unroll
  for (int d = 16; d > 0; d /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = most;
  __syncthreads();
  most = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
  const float after = s_nan != 0 ? __uint_as_float(0x7fffffffu) : scale_for<kInt8>(most);
  const float inv = 1.f / after;
  const long long block = static_cast<long long>(to) * p.c.hkv + h;
  if (threadIdx.x == 0) p.c.scale[which][block] = after;
  uint4* const dst = reinterpret_cast<uint4*>(p.c.data[which] + block * kBs * kD);
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int at = i * kPack + threadIdx.x, row = at / kCols;
    if (row >= rows) continue;
    const float scale = s_scale[row];
    if (after != after) x[i] = make_uint4(0, 0, 0, 0);
    uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float4 f = to_float4<kInt8>(w[k]);
      if (after == after) w[k] = to_bytes<kInt8>(f.x * scale * inv, f.y * scale * inv, f.z * scale * inv, f.w * scale * inv);
    }
    dst[at] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int kD, int kBs>
cudaError_t launch_pack(const EvictKernelParams& kp, dim3 grid, cudaStream_t s) {
  return kp.c.kind == RSWA_CACHE_INT8 ? launch_kernel(evict_pack_kernel<kD, kBs, true>, grid, kPack, 0, s, true, kp)
                                      : launch_kernel(evict_pack_kernel<kD, kBs, false>, grid, kPack, 0, s, true, kp);
}

}  // namespace

}  // namespace rswa

using namespace rswa;

extern "C" int rswa_cache_evict(const rswa_cache_evict_params_t* p, void* stream) {
  const char* what = "rswa_cache_evict";
  if (p == nullptr) {
    set_error("%s: null params", what);
    return RSWA_E_ARG;
  }
  int rc = check_cache(p->cache, what);
  if (rc == RSWA_OK) rc = check_table(p->table, p->lens, p->status, p->cache.block_size, what);
  if (rc == RSWA_OK) rc = check_table(p->new_table, p->lens, p->status, p->cache.block_size, what);
  if (rc != RSWA_OK) return rc;
  if (p->budget <= 0 || p->n_sink < 0 || p->n_recent < 0 || static_cast<int64_t>(p->n_sink) + p->n_recent > p->budget) {
    set_error("%s: budget must be positive and hold the sink tokens and the newest ones (budget %d, %d and %d)", what, p->budget, p->n_sink, p->n_recent);
    return RSWA_E_ARG;
  }
  const int64_t bs = p->cache.block_size, cap = p->table.max_blocks * bs, new_cap = p->new_table.max_blocks * bs;
  if (p->new_table.batch != p->table.batch || new_cap < (p->budget < cap ? p->budget : cap) || p->new_w_len < new_cap) {
    set_error("%s: new_table must have a row for each sequence and hold min(budget, tokens of the table); new_weights its tokens", what);
    return RSWA_E_ARG;
  }
  if (p->table.batch == 0) return RSWA_OK;
  if (p->weights == nullptr || p->new_lens == nullptr || p->new_weights == nullptr || p->kept == nullptr) {
    set_error("%s: weights, new_lens, new_weights and kept are required", what);
    return RSWA_E_ARG;
  }
  const int64_t items = static_cast<int64_t>(p->table.batch) * p->cache.n_kv_heads;
  const int64_t units = static_cast<int64_t>(p->table.batch) * p->new_table.max_blocks;
  if (items > 0x7fffffffLL || units > 0x7fffffffLL) {
    set_error("%s: too many sequences in one call", what);
    return RSWA_E_UNSUPPORTED;
  }
  EvictKernelParams kp;
  kp.c = cache_view(p->cache);
  kp.table = p->table.entries, kp.table_stride = p->table.stride;
  kp.batch = p->table.batch, kp.max_blocks = p->table.max_blocks;
  kp.lens = p->lens;
  kp.weights = p->weights;
  kp.w_sb = p->w_stride_b, kp.w_sh = p->w_stride_h;
  kp.budget = p->budget, kp.n_sink = p->n_sink, kp.n_recent = p->n_recent, kp.new_w_len = p->new_w_len;
  kp.new_table = p->new_table.entries, kp.new_table_stride = p->new_table.stride, kp.new_max_blocks = p->new_table.max_blocks;
  kp.new_lens = p->new_lens;
  kp.new_weights = p->new_weights;
  kp.kept = p->kept;
  kp.status = p->status;
  kp.mirror = status_mirror(p->status);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = launch_kernel(evict_select_kernel, dim3(static_cast<unsigned>(items)), kSelect, 0, s, true, kp);
  if (e == cudaSuccess) count_launches(1);
  if (e == cudaSuccess && units > 0) {
    const dim3 grid(static_cast<unsigned>(units), static_cast<unsigned>(2 * p->cache.n_kv_heads));
    const int key = p->cache.head_dim * 1000 + p->cache.block_size;
    switch (key) {
      case 64016: e = launch_pack<64, 16>(kp, grid, s); break;
      case 64032: e = launch_pack<64, 32>(kp, grid, s); break;
      case 64064: e = launch_pack<64, 64>(kp, grid, s); break;
      case 64128: e = launch_pack<64, 128>(kp, grid, s); break;
      case 128016: e = launch_pack<128, 16>(kp, grid, s); break;
      case 128032: e = launch_pack<128, 32>(kp, grid, s); break;
      case 128064: e = launch_pack<128, 64>(kp, grid, s); break;
      default: e = launch_pack<128, 128>(kp, grid, s); break;
    }
    if (e == cudaSuccess) count_launches(1);
  }
  if (e != cudaSuccess) {
    set_error("%s: launch failed: %s", what, cudaGetErrorString(e));
    return RSWA_E_CUDA;
  }
  return RSWA_OK;
}
