// Thinning out cached sequences by accumulated attention weight (see rswa_cache_evict in rswa.h), in two kernels:
// one chooses the slots that stay, per sequence and key/value head, the other packs their keys and values into new blocks.
#include <atomic>

#include "rswa_cache.cuh"

namespace rswa {

int check_table(const rswa_block_table_t& t, bool written, const int32_t* lens, const int32_t* status, int block_size, const char* what);

namespace {

constexpr int kSelect = 1024;     // threads of a choosing CTA
constexpr int kDigits = 3;        // of a key: 11, 11 and 10 bits
constexpr int kPack = 128;        // threads of a packing CTA
constexpr int kCacheKeys = 47104; // keys that a choosing CTA keeps in shared memory
constexpr int kMostRanks = 8;     // choosing CTAs of a head at most
constexpr int kRankKeys = 6144;   // slots that are worth a CTA of their own

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

// the weight a key was made of (a NaN of any kind as the canonical one, -0 as 0)
__device__ __forceinline__ float key_weight(uint32_t key) {
  if (key == 0xffffffffu) return __uint_as_float(0x7fffffffu);
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// s[0] + ... + s[warp - 1], for all lanes of a warp (at most 32 values)
__device__ __forceinline__ int sum_below(const int* s, int warp) {
  const int lane = threadIdx.x & 31;
  return __reduce_add_sync(0xffffffffu, lane < warp ? s[lane] : 0);
}

// All threads of a cluster, with what they wrote to shared memory.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// the same place in another CTA's shared memory
__device__ __forceinline__ uint32_t cluster_addr(const void* at, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(tc05::smem_u32(at)), "r"(rank));
  return a;
}
__device__ __forceinline__ int ld_cluster(const int* at, int rank) {
  int x;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(x) : "r"(cluster_addr(at, rank)) : "memory");
  return x;
}
__device__ __forceinline__ int2 ld_cluster(const int2* at, int rank) {
  int2 x;
  asm volatile("ld.shared::cluster.v2.s32 {%0, %1}, [%2];" : "=r"(x.x), "=r"(x.y) : "r"(cluster_addr(at, rank)) : "memory");
  return x;
}
__device__ __forceinline__ int2 operator+(int2 a, int2 b) { return make_int2(a.x + b.x, a.y + b.y); }
// *at, or the sum of it over a cluster's CTAs
template <bool kMany, typename T>
__device__ __forceinline__ T sum_ranks(const T* at, int ranks) {
  if (!kMany) return *at;
  T x = {};
#pragma unroll
  for (int r = 0; r < kMostRanks; ++r)
    if (r < ranks) x = x + ld_cluster(at, r);
  return x;
}

// One CTA per (sequence, head), or a cluster of `ranks` (kMany), each with a contiguous piece of the slots.  The k-th
// largest key between the sinks and the newest tokens is found digit by digit (11, 11, 10 bits; a histogram of the
// candidates' digits each time, added up over the cluster), then two ordered sweeps write what is above it and the first
// ones of those equal to it.  The weights are read once, into shared memory, unless there are more than fit (then the
// later sweeps read them from L2).  The number of cluster barriers depends on nothing that is read.
// Bound by the SM's issue rate, 0.6 us for 1000 slots of a CTA, and 8 us of latencies (13 in a cluster: four exchanges).
// Whole evictions, by single CTAs and by the clusters chosen below: 8 heads of 131072 slots (8192 stay) 143 and 32 us,
// of 40000 38 and 24, of 8192 16.5 (two CTAs: 18); 64 heads of 16384 (half stay) 87 and 82.
template <bool kMany>
__global__ void __launch_bounds__(kSelect) evict_select_kernel(const __grid_constant__ EvictKernelParams p, int n_cached, int ranks_) {
  extern __shared__ __align__(16) uint32_t s_keys[];  // [n_cached]
  // Histograms, two of each digit: neighbouring lanes count apart where the weights are much alike.  Their sums over 64 bins
  // each, a warp's, largest digits first.
  __shared__ __align__(16) int s_hist[2 * (2048 + 2048 + 1024)];
  __shared__ int s_part[kDigits][kSelect / 32];
  __shared__ int2 s_found[kDigits];
  __shared__ int s_warp[kSelect / 32], s_warp_eq[kSelect / 32];
  __shared__ int2 s_stay;
  griddep_launch();
  for (int i = threadIdx.x; i < 2 * (2048 + 2048 + 1024) / 4; i += kSelect) reinterpret_cast<uint4*>(s_hist)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  griddep_wait();
  const int ranks = kMany ? ranks_ : 1;
  const int item = blockIdx.x / ranks, rank = blockIdx.x - item * ranks;
  const int b = item / p.c.hkv, h = item - b * p.c.hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = checked_len(p, b);
  const int keep = min(len, p.budget);
  const float* const w = p.weights + b * p.w_sb + h * p.w_sh;
  int* const kept = p.kept + static_cast<long long>(item) * p.budget;
  float* const new_w = p.new_weights + static_cast<long long>(item) * p.new_w_len;
  if (h == 0 && rank == 0 && threadIdx.x == 0) p.new_lens[b] = keep;
  // this CTA's slots: [from, to)
  constexpr int kStep = 128;  // slots of a warp at a time, four a lane
  const int per = ((len + ranks - 1) / ranks + kStep - 1) / kStep * kStep;
  const int from = min(static_cast<long long>(len), static_cast<long long>(rank) * per), to = min(static_cast<long long>(len), static_cast<long long>(from) + per);
  const bool cached = per <= n_cached;
  // candidates: slots [lo, hi), of which `left` stay
  const bool all = len <= p.budget;
  const int lo = all ? 0 : p.n_sink, hi = all ? len : len - p.n_recent;  // (n_sink + n_recent <= budget < len)
  int left = all ? len : p.budget - p.n_sink - p.n_recent;
  const bool choose = !all && left > 0;
  // keys above it stay, and `left` of those equal to it (nothing in between: a NaN would be equal to it, left is 0)
  uint32_t bound = choose || all ? 0 : 0xffffffffu;
  if (!all) {
    constexpr int kAhead = 8;
    for (int i0 = from + threadIdx.x; i0 < to; i0 += kAhead * kSelect) {
      float x[kAhead];
#pragma unroll
      for (int e = 0; e < kAhead; ++e) x[e] = i0 + e * kSelect < to ? w[i0 + e * kSelect] : 0.f;
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        const int i = i0 + e * kSelect;
        const uint32_t key = order_key(x[e]);
        if (cached && i < to) s_keys[i - from] = key;
        if (choose && i >= lo && i < min(hi, to)) atomicAdd(&s_hist[(lane & 1) * 2048 + (key >> 21)], 1);
      }
    }
  }
  __syncthreads();
  // the keys of four slots, from a multiple of four behind the first on (behind the last one: anything)
  const auto keys4 = [&](int i) {
    if (cached) return *reinterpret_cast<const uint4*>(s_keys + (i - from));
    return make_uint4(order_key(w[i]), i + 1 < len ? order_key(w[i + 1]) : 0, i + 2 < len ? order_key(w[i + 2]) : 0, i + 3 < len ? order_key(w[i + 3]) : 0);
  };
  uint32_t mask = 0;
#pragma unroll
  for (int pass = 0; pass < kDigits; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass < 2 ? 2048 : 1024;
    int* const hist = s_hist + pass * 2 * 2048;
    if (choose) {
      if (pass > 0) {
#pragma unroll 2
        for (int i = from + 4 * threadIdx.x; i < min(hi, to); i += 4 * kSelect) {
          const uint4 k4 = keys4(i);
          const uint32_t keys[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (i + e >= lo && i + e < min(hi, to) && (keys[e] & mask) == bound) atomicAdd(hist + (lane & 1) * bins + ((keys[e] >> shift) & (bins - 1)), 1);
        }
        __syncthreads();
      }
      const int at = bins - 2 - 2 * threadIdx.x;
      int2 c = make_int2(0, 0);
      if (at >= 0) {
        int2* const h2 = reinterpret_cast<int2*>(hist + at);
        c = *h2 + h2[bins / 2];
        *h2 = c;
      }
      const int sum = __reduce_add_sync(0xffffffffu, c.x + c.y);
      if (lane == 0) s_part[pass][warp] = sum;
      if (!kMany) __syncthreads();
    }
    if (kMany) cluster_sync();
    if (choose) {
      // the digit with which the count from above reaches `left`: which 64 bins, then which of them
      if (warp == 0) {
        const auto scan = [&](int x) {
#pragma unroll
          for (int d = 1; d < 32; d *= 2) {
            const int o = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += o;
          }
          return x;
        };
        const int part = sum_ranks<kMany>(&s_part[pass][lane], ranks);
        int above = scan(part) - part;
        int src = __ffs(__ballot_sync(0xffffffffu, above < left && above + part >= left)) - 1;
        above = __shfl_sync(0xffffffffu, above, src);
        const int at = max(0, bins - 2 - 2 * (32 * src + lane));
        const int2 c = sum_ranks<kMany>(reinterpret_cast<const int2*>(hist + at), ranks);
        above += scan(c.x + c.y) - c.x - c.y;
        src = __ffs(__ballot_sync(0xffffffffu, above < left && above + c.x + c.y >= left)) - 1;
        const bool first = above + c.y >= left;
        const int digit = __shfl_sync(0xffffffffu, first ? at + 1 : at, src);
        above = __shfl_sync(0xffffffffu, above + (first ? 0 : c.y), src);
        if (lane == 0) s_found[pass] = make_int2(digit, left - above);
      }
      __syncthreads();
      bound |= static_cast<uint32_t>(s_found[pass].x) << shift;
      left = s_found[pass].y;
      mask |= static_cast<uint32_t>(bins - 1) << shift;
    }
  }
  // Every warp takes a contiguous piece of the CTA's slots: how many of its tokens stay, then where they go.
  const int piece = (to - from + kSelect / 32 * kStep - 1) / (kSelect / 32 * kStep) * kStep;
  const int begin = min(to, from + warp * piece), end = min(to, begin + piece);
  // whether the slots i .. i + 3 stay for certain (bits 0 to 3), or if there is room for them (bits 8 to 11)
  const auto stand = [&](int i, uint32_t (&keys)[4]) {
    uint32_t r = 0;
    if (i < end) {
      if (!all) {
        const uint4 k4 = keys4(i);
        keys[0] = k4.x, keys[1] = k4.y, keys[2] = k4.z, keys[3] = k4.w;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int slot = i + e;
        if (slot >= end) continue;
        if (all || slot < lo || slot >= hi || keys[e] > bound) r |= 1u << e;
        else if (keys[e] == bound) r |= 256u << e;
      }
    }
    return r;
  };
  int n_above = 0, n_equal = 0;
  for (int i = begin + 4 * lane; i - 4 * lane < end; i += kStep) {
    uint32_t keys[4] = {0, 0, 0, 0};
    const uint32_t r = stand(i, keys);
    n_above += __popc(r & 15u);
    n_equal += __popc(r >> 8);
  }
  n_above = __reduce_add_sync(0xffffffffu, n_above);
  n_equal = __reduce_add_sync(0xffffffffu, n_equal);
  if (lane == 0) s_warp[warp] = n_above, s_warp_eq[warp] = n_equal;
  __syncthreads();
  // (of the equal ones, those in front take the room first)
  int equal_before = sum_below(s_warp_eq, warp), above_before = sum_below(s_warp, warp);
  if (kMany) {
    if (threadIdx.x == kSelect - 1) s_stay = make_int2(above_before + n_above, equal_before + n_equal);
    cluster_sync();
    const int2 o = lane < rank ? ld_cluster(&s_stay, lane) : make_int2(0, 0);
    above_before += __reduce_add_sync(0xffffffffu, o.x);
    equal_before += __reduce_add_sync(0xffffffffu, o.y);
  }
  int at = above_before + min(equal_before, left);
  const uint32_t before = (1u << lane) - 1;
  for (int i = begin + 4 * lane; i - 4 * lane < end; i += kStep) {
    uint32_t keys[4] = {0, 0, 0, 0};
    uint32_t r = stand(i, keys);
    // how many of the lanes in front of this one: four votes each, since a lane has four slots
    int equal_here = 0, equal_all = 0;
    if (__any_sync(0xffffffffu, r >> 8)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t v = __ballot_sync(0xffffffffu, r >> (8 + e) & 1u);
        equal_here += __popc(v & before);
        equal_all += __popc(v);
      }
      int n = equal_before + equal_here;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (r >> (8 + e) & 1u) r |= (n++ < left ? 1u : 0u) << e;
    }
    int n = at;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t v = __ballot_sync(0xffffffffu, r >> e & 1u);
      n += __popc(v & before);
      at += __popc(v);
    }
    equal_before += equal_all;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (r >> e & 1u) {
        if (n < p.budget) kept[n] = i + e;  // (always, unless somebody changes the weights meanwhile)
        if (n < p.new_w_len) new_w[n] = cached && !all ? key_weight(keys[e]) : w[i + e];
        ++n;
      }
  }
  for (long long i = keep + rank * kSelect + threadIdx.x; i < p.budget; i += ranks * kSelect) kept[i] = -1;
  for (long long i = keep + rank * kSelect + threadIdx.x; i < p.new_w_len; i += ranks * kSelect) new_w[i] = 0.f;
  if (kMany) cluster_sync();  // (nobody's shared memory goes while somebody may read it)
}

// A CTA packs `run` new blocks of a head, K and V (or one block, K or V, where there are too few for that): it looks all
// their rows up first, then reads the rows of one block while it finds the largest magnitude of the one before and writes
// it at its new scale.  A row is read once (head_dim bytes, scattered) and stays in registers.
// Bound by HBM, one byte in and one out per element; what a CTA waits for before its first byte (length, kept slots,
// block table, scales: four loads in a row) is paid once a run.  134 MB in and 134 MB out in blocks of 64 take 51 us with
// runs of two, 57 with four (too few CTAs for even waves), 41 at a copy's rate; in blocks of 16 four are 5 % faster.
template <int kBs>
constexpr int kRunOf = kBs >= 64 ? 2 : 4;
template <int kD, int kBs, bool kInt8>
__global__ void __launch_bounds__(kPack) evict_pack_kernel(const __grid_constant__ EvictKernelParams p, int run) {
  constexpr int kCols = kD / 16;  // 16-byte pieces of a row
  constexpr int kPasses = (kBs * kCols + kPack - 1) / kPack;
  constexpr int kRun = kRunOf<kBs>;
  __shared__ int s_page[kRun * kBs], s_slot[kRun * kBs];  // block and head of a row (-1: none), token in the block
  __shared__ float s_scale[2][kRun * kBs];
  __shared__ float s_max[2][kPack / 32];
  const int groups = (p.new_max_blocks + run - 1) / run;
  const int b = blockIdx.x / groups, j0 = (blockIdx.x - b * groups) * run;
  // which of K and V
  const int h = run > 1 ? blockIdx.y : blockIdx.y >> 1, first = run > 1 ? 0 : blockIdx.y & 1, kinds = run > 1 ? 2 : 1;
  griddep_launch();
  griddep_wait();
  const int keep = min(checked_len(p, b), p.budget);
  const int rows = min(keep - j0 * kBs, run * kBs);
  if (rows <= 0) return;
  const int* kept = p.kept + (static_cast<long long>(b) * p.c.hkv + h) * p.budget + static_cast<long long>(j0) * kBs;
  for (int r = threadIdx.x; r < rows; r += kPack) {
    const int slot = kept[r];
    const int page = table_entry(p.table, p.table_stride, b, slot / kBs, p.c.num_blocks, p.status, p.mirror);
    const int at = page < 0 ? -1 : page * p.c.hkv + h;
    s_page[r] = at;
    s_slot[r] = slot % kBs;
    for (int k = 0; k < 2; ++k) s_scale[k][r] = at < 0 ? 0.f : p.c.scale[k][at];
  }
  __syncthreads();
  const int units = (rows + kBs - 1) / kBs * kinds;  // (block, K or V)
  const auto load = [&](int u, uint4 (&x)[kPasses]) {
    const int base = u / kinds * kBs;
    const uint8_t* const data = p.c.data[first + u % kinds];
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int at = i * kPack + threadIdx.x, row = base + at / kCols;
      x[i] = make_uint4(0, 0, 0, 0);
      if (at < kBs * kCols && row < rows && s_page[row] >= 0)
        x[i] = *reinterpret_cast<const uint4*>(data + (static_cast<long long>(s_page[row]) * kBs + s_slot[row]) * kD + at % kCols * 16);
    }
  };
  const auto store = [&](int u, uint4 (&x)[kPasses]) {
    const int j = u / kinds, base = j * kBs, which = first + u % kinds;
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int at = i * kPack + threadIdx.x, row = base + at / kCols;
      if (at >= kBs * kCols || row >= rows) continue;
      Largest<kInt8> m;
      m.add(x[i].x), m.add(x[i].y), m.add(x[i].z), m.add(x[i].w);
      // (a scale that is not finite makes the new block's NaN: infinity stands for that here)
      const float scale = s_scale[which][row];
      most = fmaxf(most, scale <= 3.4028235e38f ? m.value() * scale : INFINITY);
    }
#pragma unroll
    for (int d = 16; d > 0; d /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
    float* const all = s_max[u & 1];
    if ((threadIdx.x & 31) == 0) all[threadIdx.x >> 5] = most;
    __syncthreads();
    most = fmaxf(fmaxf(all[0], all[1]), fmaxf(all[2], all[3]));
    const float after = scale_for<kInt8>(most);
    const float inv = 1.f / after;
    const int to = table_entry(p.new_table, p.new_table_stride, b, j0 + j, p.c.num_blocks, p.status, p.mirror);
    if (to < 0) return;
    const long long block = static_cast<long long>(to) * p.c.hkv + h;
    if (threadIdx.x == 0) p.c.scale[which][block] = after;
    uint4* const dst = reinterpret_cast<uint4*>(p.c.data[which] + block * kBs * kD);
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int at = i * kPack + threadIdx.x, row = base + at / kCols;
      if (at >= kBs * kCols || row >= rows) continue;
      if (after != after) {
        dst[at] = make_uint4(0, 0, 0, 0);
        continue;
      }
      const Rescale<kInt8> to_new(s_scale[which][row] * inv);
      dst[at] = make_uint4(to_new(x[i].x), to_new(x[i].y), to_new(x[i].z), to_new(x[i].w));
    }
  };
  uint4 x[2][kPasses];
  load(0, x[0]);
  for (int u = 0; u < units; u += 2) {
    if (u + 1 < units) load(u + 1, x[1]);
    store(u, x[0]);
    if (u + 1 >= units) break;
    if (u + 2 < units) load(u + 2, x[0]);
    store(u + 1, x[1]);
  }
}

// The choosing kernel may use as much shared memory as it needs at most: set once per device.
cudaError_t allow_shared(int bytes) {
  if (bytes <= 6 * 1024) return cudaSuccess;  // (48 KB with what it has of fixed size need no permission)
  static std::atomic<uint64_t> set{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && (set.load(std::memory_order_relaxed) >> dev & 1))) return e;
  e = cudaFuncSetAttribute(evict_select_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kCacheKeys * 4);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(evict_select_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kCacheKeys * 4);
  if (e == cudaSuccess && dev < 64) set.fetch_or(1ull << dev, std::memory_order_relaxed);
  return e;
}

template <int kD, int kBs>
cudaError_t launch_pack(const EvictKernelParams& kp, dim3 grid, int run, cudaStream_t s) {
  return kp.c.kind == RSWA_CACHE_INT8 ? launch_kernel(evict_pack_kernel<kD, kBs, true>, grid, kPack, 0, s, true, kp, run)
                                      : launch_kernel(evict_pack_kernel<kD, kBs, false>, grid, kPack, 0, s, true, kp, run);
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
  if (rc == RSWA_OK) rc = check_table(p->table, false, p->lens, p->status, p->cache.block_size, what);
  if (rc == RSWA_OK) rc = check_table(p->new_table, true, p->lens, p->status, p->cache.block_size, what);
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
  if (items * kMostRanks > 0x7fffffffLL || units > 0x7fffffffLL) {
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
  // (several CTAs a head where there are SMs for them and enough slots, or where the keys do not fit one's shared memory)
  int ranks = 1;
  while (ranks < kMostRanks && ((items * 2 * ranks <= sm_count() && cap >= 2LL * ranks * kRankKeys) || cap > static_cast<int64_t>(ranks) * kCacheKeys)) ranks *= 2;
  const int64_t per = ((cap + ranks - 1) / ranks + 127) / 128 * 128, keys = per < kCacheKeys ? per : kCacheKeys;
  const int smem = static_cast<int>(keys) * 4;
  cudaError_t e = allow_shared(smem);
  if (e == cudaSuccess) e = launch_clusters(ranks > 1 ? evict_select_kernel<true> : evict_select_kernel<false>, dim3(static_cast<unsigned>(items * ranks)), ranks, kSelect, smem, s, true, kp, static_cast<int>(keys), ranks);
  if (e == cudaSuccess) count_launches(1);
  if (e == cudaSuccess && units > 0) {
    // (several blocks, K and V, a CTA where that still gives every SM four CTAs)
    const int most = bs >= 64 ? kRunOf<64> : kRunOf<16>;
    const int run = units * p->cache.n_kv_heads >= 4LL * most * sm_count() ? most : 1;
    const dim3 grid(static_cast<unsigned>(p->table.batch * ((p->new_table.max_blocks + run - 1LL) / run)), static_cast<unsigned>((run > 1 ? 1 : 2) * p->cache.n_kv_heads));
    const int key = p->cache.head_dim * 1000 + p->cache.block_size;
    switch (key) {
      case 64016: e = launch_pack<64, 16>(kp, grid, run, s); break;
      case 64032: e = launch_pack<64, 32>(kp, grid, run, s); break;
      case 64064: e = launch_pack<64, 64>(kp, grid, run, s); break;
      case 64128: e = launch_pack<64, 128>(kp, grid, run, s); break;
      case 128016: e = launch_pack<128, 16>(kp, grid, run, s); break;
      case 128032: e = launch_pack<128, 32>(kp, grid, run, s); break;
      case 128064: e = launch_pack<128, 64>(kp, grid, run, s); break;
      default: e = launch_pack<128, 128>(kp, grid, run, s); break;
    }
    if (e == cudaSuccess) count_launches(1);
  }
  if (e != cudaSuccess) {
    set_error("%s: launch failed: %s", what, cudaGetErrorString(e));
    return RSWA_E_CUDA;
  }
  return RSWA_OK;
}
