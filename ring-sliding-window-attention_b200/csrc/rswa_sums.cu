// How much softmax weight the queries of a prompt gave to each of its keys, per key/value head:
//
//   w[t] = sum over the group's query heads and the queries i that see t of exp(scale * q_i.k_t - lse_i)
//
// what an eviction from a cache by accumulated weight starts with (the decoding steps add theirs, rswa_cache_attn.cu).
//
// S^T = K Q^T on the tensor cores with the keys as rows: a thread then owns a key, and the sum over queries is a sum
// over the columns it reads from tensor memory, with no exchange between threads.  A step of the pipeline is 256 keys
// (two tiles) by 128 queries of one head: each Q tile that comes out of L2 feeds two products.  Eight warps work on a tile, 64
// query columns each: four a scheduler, so that one's loads from tensor memory hide behind the others' arithmetic (with 128
// columns and half the warps a step took 3270 cycles).
// 2 * head_dim FLOPs and one exponential per (query head, pair): at 128 elements the exponentials (16 per clock and SM,
// 2048 cycles a step) outweigh the products (1024).  One pair in eight is computed on the FMA pipe (fma_exp2): none
// 624 us, 1/8 621, 1/4 631 (16384 tokens, 32/8 heads, window 4096): the card is at its power cap there when call follows
// call (548 us on a cool one), and an exponential on the FMA pipe costs more than it saves beyond that.  Besides, 6 us go for the
// look at each step's sum: a NaN may come from a query that has to be left out, and is added up again pair by pair (with the
// queries left out in the ordinary code 15 us).
//
// Work: the steps of all (batch row, key/value head, 256 keys) in one order, cut into equal shares, one per CTA and round,
// whatever the mask makes of an item's length (a sink token is seen by its whole sequence): nothing is longer than the rest.
// Rounds, because a query tile is read by as many CTAs as the window has key tiles: with 134 MB of queries in one round
// they do not meet in L2 (1.3 GB from HBM, whose power the card lacks elsewhere: 680 us; two rounds 621, five 623, ten 641).
// An item that is cut leaves partial sums in the workspace, added up in order by a second kernel: deterministic.
// A thread's running sum is compensated: a key may be seen by 10^5 queries and more.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "rswa_common.cuh"
#include "tc05.cuh"

namespace rswa {
using namespace tc05;

namespace {

constexpr int kKeys = 2 * kTile;   // keys of an item
constexpr int kSumWarps = 16;
constexpr int kThreads = 128 + kSumWarps * 32;  // warp 0 TMA, warp 1 MMA, warp 2 log-sum-exps, warp 3 idle, warps 4-19 sums
constexpr int kScan = 256;         // threads of the prefix sums
constexpr int kQStages = 3;
constexpr int kTmemCols = 512;
constexpr long long kRoundBytes = 68ll << 20;  // of queries at most
constexpr int kMinShare = 2;       // steps of a CTA at least
constexpr int kMaxRounds = 8, kRoundSteps = 32;  // shares of a CTA at most, and steps of each at least

struct SumsKernelParams {
  CUtensorMap q_map, k_map;
  const float* lse;
  long long l_sb, l_sh;
  int batch, len, hq, hkv, group;
  int window, n_sink;
  float scale_log2;
  const int* cu;
  int n_seqs;
  float* out;    // [batch, hkv, len]
  float* part;   // [shares][2][kKeys]
  int n_items;   // per batch row and head
  int ctas, rounds;
  int* status;
  int* mirror;
};

// query tiles that see a key of item kt: the first is the one the keys begin in
__device__ __forceinline__ int item_q_tiles(const SumsKernelParams& p, int kt) {
  const int t0 = kt * kKeys, t_last = min(t0 + kKeys, p.len) - 1;
  int s, e;
  seq_of(p.cu, p.n_seqs, t_last, s, e);
  e = min(e, p.len);
  // (a tile that holds a sink token of the sequence that goes on behind it: all of that sequence)
  const bool sink = p.n_sink > 0 && t0 - s < p.n_sink;
  const int last = sink || e - 1 - t_last <= p.window ? e - 1 : t_last + p.window;
  // (at least one: boundaries that are not in order must not send the walk over the items astray)
  return max(1, last / kTile - t0 / kTile + 1);
}

// prefix sums of the items' query tiles, by the first kScan threads; s_prefix[kScan] is the sum
__device__ __forceinline__ void item_prefix(const SumsKernelParams& p, long long* s_prefix, long long* s_warp) {
  const int per = (p.n_items + kScan - 1) / kScan;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long mine = 0, sum = 0;
  if (threadIdx.x < kScan) {
    for (int i = 0; i < per; ++i) {
      const int kt = threadIdx.x * per + i;
      if (kt < p.n_items) mine += item_q_tiles(p, kt);
    }
    sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const long long o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    if (lane == 31) s_warp[warp] = sum;
  }
  __syncthreads();
  if (threadIdx.x < kScan) {
    long long before = 0;
    for (int w = 0; w < warp; ++w) before += s_warp[w];
    s_prefix[threadIdx.x] = before + sum - mine;
    if (threadIdx.x == kScan - 1) s_prefix[kScan] = before + sum;
  }
  __syncthreads();
}

// Shares of the work: `rounds` for each CTA, the ones of a round side by side, unless there is too little.
__device__ __forceinline__ long long n_shares(long long total, const SumsKernelParams& p) {
  const long long rounds = p.rounds == 1 ? 1 : max(1LL, min(static_cast<long long>(p.rounds), total / (static_cast<long long>(p.ctas) * kRoundSteps)));
  return min(rounds * p.ctas, max(1LL, total / kMinShare));
}
__device__ __forceinline__ long long share_begin(long long total, long long shares, long long c) { return total * c / shares; }

// An item, and how far into it a place is: steps are query heads of the group, then query tiles.
struct Item {
  int bh, kt, n_qt, n;  // n = n_qt * group
  long long first;      // index of its first step
  __device__ __forceinline__ void next(const SumsKernelParams& p) {
    first += n;
    if (++kt == p.n_items) kt = 0, ++bh;
    n_qt = item_q_tiles(p, kt);
    n = n_qt * p.group;
  }
};
__device__ __forceinline__ Item item_at(const SumsKernelParams& p, const long long* s_prefix, long long step) {
  const long long row = s_prefix[kScan] * p.group;  // steps of a batch row and head
  Item it;
  it.bh = static_cast<int>(step / row);
  const long long rest = step - it.bh * row;
  int lo = 0, hi = kScan - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s_prefix[mid] * p.group <= rest) lo = mid; else hi = mid - 1;
  }
  // (threads behind the last item hold none and have the whole sum in front of them: never chosen)
  it.kt = lo * ((p.n_items + kScan - 1) / kScan);
  it.first = it.bh * row + s_prefix[lo] * p.group;
  it.n_qt = item_q_tiles(p, it.kt);
  it.n = it.n_qt * p.group;
  while (step >= it.first + it.n) it.next(p);
  return it;
}

// A share: where it begins (`start` steps into an item), and its steps.
struct Share {
  int n, bh, kt, n_qt, start;
};
// The same, walked item by item by every role: steps [start, stop) of the item are this share's.
struct Walk {
  int left, bh, kt, n_qt, start, stop;
  __device__ __forceinline__ Walk(const SumsKernelParams& p, const Share& s) : left(s.n), bh(s.bh), kt(s.kt), n_qt(s.n_qt), start(s.start) { cut(p); }
  __device__ __forceinline__ int n(const SumsKernelParams& p) const { return n_qt * p.group; }
  __device__ __forceinline__ void cut(const SumsKernelParams& p) { stop = start + min(left, n(p) - start); }
  __device__ __forceinline__ void next(const SumsKernelParams& p) {
    left -= stop - start;
    start = 0;
    if (left == 0) return;
    if (++kt == p.n_items) kt = 0, ++bh;
    n_qt = item_q_tiles(p, kt);
    cut(p);
  }
};

// 2^x for two values on the FMA pipe: x = n + f with n = round(x) and f in [-0.5, 0.5]; 2^f by the polynomial of degree 5 with
// the least relative error there (7.5e-8, found by exchange of its extrema; 2.1e-7 in 32 bits), times 2^n from n's bits.  From
// -126.5 down (hidden pairs are -inf) exactly 0, since n = -127 gives an exponent field of 0; NaN stays NaN.
__device__ __forceinline__ float2 fma_exp2(float2 x) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.x) : "f"(-127.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.y) : "f"(-127.f));
  const float2 t = __fadd2_rn(x, make_float2(12582912.f, 12582912.f));  // 1.5 * 2^23: n lands in the low mantissa bits
  const float2 n = __fadd2_rn(t, make_float2(-12582912.f, -12582912.f));
  const float2 f = __ffma2_rn(n, make_float2(-1.f, -1.f), x);
  float2 q = __ffma2_rn(make_float2(0.0013276472454890609f, 0.0013276472454890609f), f, make_float2(0.009675540961325169f, 0.009675540961325169f));
  q = __ffma2_rn(q, f, make_float2(0.05550713092088699f, 0.05550713092088699f));
  q = __ffma2_rn(q, f, make_float2(0.24022120237350464f, 0.24022120237350464f));
  q = __ffma2_rn(q, f, make_float2(0.6931469440460205f, 0.6931469440460205f));
  q = __ffma2_rn(q, f, make_float2(1.0000001192092896f, 1.0000001192092896f));
  const float2 p = make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u), __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u));
  return __fmul2_rn(q, p);
}

// barrier of the summing warps; whether all of them are well
__device__ __forceinline__ bool all_sum_warps(bool ok) {
  int all;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, 1, %2, p;\n\tselp.s32 %0, 1, 0, q;\n\t}\n"
               : "=r"(all)
               : "r"(static_cast<int>(ok)), "n"(kSumWarps * 32)
               : "memory");
  return all != 0;
}

struct Ctl {
  uint64_t k_full[2], k_free[2], q_full[kQStages], q_free[kQStages], s_ready[2][2], s_free[2][2], drained;  // (of the steps' parity, and of the two tiles)
  uint32_t tmem_base;
  int err;
  Share share[kMaxRounds];  // of the CTA
};

constexpr int kSmemK = 0, kSmemQ = 4 * kTileBytes, kSmemLse = kSmemQ + kQStages * kTileBytes;
constexpr int kSmemHalf = kSmemLse + 2 * kTile * 4, kSmemCtl = kSmemHalf + kKeys * 4;
constexpr int kSmemBytes = kSmemCtl + 512;
static_assert(sizeof(Ctl) <= 512 && kSmemBytes <= 232448, "shared memory budget");

template <int kD, bool kBf16>
__global__ void __launch_bounds__(kThreads, 1) weight_sums_kernel(const __grid_constant__ SumsKernelParams p) {
  constexpr uint32_t kLoadBytes = kD / 64 * kBoxBytes;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* const sK = smem + kSmemK;  // [2 items][2 tiles]
  uint8_t* const sQ = smem + kSmemQ;
  float* const sLse = reinterpret_cast<float*>(smem + kSmemLse);  // [2][128]: -lse * log2(e)
  Ctl* const ctl = reinterpret_cast<Ctl*>(smem + kSmemCtl);
  long long* const s_prefix = reinterpret_cast<long long*>(sQ);  // (until the loads begin)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl->k_full[i], 1);
      mbar_init(&ctl->k_free[i], 1);
      for (int t = 0; t < 2; ++t) {
        mbar_init(&ctl->s_ready[i][t], 2);  // the products, and their row of log-sum-exps
        mbar_init(&ctl->s_free[i][t], kSumWarps / 2);
      }
    }
    for (int i = 0; i < kQStages; ++i) {
      mbar_init(&ctl->q_full[i], 1);
      mbar_init(&ctl->q_free[i], 1);
    }
    mbar_init(&ctl->drained, 1);
    mbar_fence_init();
    prefetch_tmap(&p.q_map);
    prefetch_tmap(&p.k_map);
  }
  if (warp == 1) {
    tmem_alloc(&ctl->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  griddep_wait();
  if (threadIdx.x == 0) ctl->err = (smem_u32(smem) & 1023u) ? 199 : status_code(p.status, p.mirror);
  item_prefix(p, s_prefix, s_prefix + kScan + 1);
  const long long total = s_prefix[kScan] * p.group * p.hkv * p.batch;
  const long long shares = n_shares(total, p);
  const int rounds = ctl->err != 0 || blockIdx.x >= shares ? 0 : (static_cast<int>(shares) - 1 - static_cast<int>(blockIdx.x)) / p.ctas + 1;
  if (threadIdx.x < rounds) {
    const long long share = blockIdx.x + static_cast<long long>(threadIdx.x) * p.ctas, begin = share_begin(total, shares, share);
    const Item it = item_at(p, s_prefix, begin);
    ctl->share[threadIdx.x] = {static_cast<int>(share_begin(total, shares, share + 1) - begin), it.bh, it.kt, it.n_qt, static_cast<int>(begin - it.first)};
  }
  tc_fence_before();
  fence_proxy_async_smem();  // (the prefix sums have been read: loads may land there)
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem_base;
  volatile int* err = &ctl->err;
  constexpr uint32_t kTile16 = kTileBytes >> 4;

  if (warp < 4) {
    setmaxnreg_dec<64>();
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------------- loads
      bool ok = true;
      int g = 0, ni = 0;  // steps and items so far
      for (int r = 0; r < rounds && ok; ++r)
      for (Walk it(p, ctl->share[r]); it.left > 0 && ok; it.next(p), ++ni) {
        const int b = it.bh / p.hkv, h = it.bh - b * p.hkv, kb = ni & 1;
        if (ni >= 2) ok = mbar_wait<200>(&ctl->k_free[kb], ((ni >> 1) - 1) & 1, err, kErrWaitProducer);
        if (!ok) break;
        const int t0 = it.kt * kKeys;
        const int tiles = t0 + kTile < p.len ? 2 : 1;  // (a tile wholly behind the end: its rows are not looked at)
        mbar_expect_tx(&ctl->k_full[kb], tiles * kLoadBytes);
        for (int t = 0; t < tiles; ++t) {
          uint8_t* const dst = sK + (kb * 2 + t) * kTileBytes;
          tma_load_4d(dst, &p.k_map, &ctl->k_full[kb], 0, h, t0 + t * kTile, b);
          if (kD > 64) tma_load_4d(dst + kBoxBytes, &p.k_map, &ctl->k_full[kb], 64, h, t0 + t * kTile, b);
        }
        for (int i = it.start; i < it.stop; ++i, ++g) {
          const int st = g % kQStages, hd = h * p.group + i / it.n_qt, q0 = t0 + i % it.n_qt * kTile;
          if (g >= kQStages) ok = mbar_wait<200>(&ctl->q_free[st], (g / kQStages - 1) & 1, err, kErrWaitProducer);
          if (!ok) break;
          uint8_t* const dst = sQ + st * kTileBytes;
          mbar_expect_tx(&ctl->q_full[st], kLoadBytes);
          tma_load_4d(dst, &p.q_map, &ctl->q_full[st], 0, hd, q0, b);
          if (kD > 64) tma_load_4d(dst + kBoxBytes, &p.q_map, &ctl->q_full[st], 64, hd, q0, b);
        }
      }
      if (!ok) {
        // loads still on their way must not outlive the CTA's shared memory (each wait is limited)
        int own = 0;
        for (int i = max(0, g - kQStages); i < g; ++i) mbar_wait(&ctl->q_full[i % kQStages], (i / kQStages) & 1, &own, kErrWaitProducer);
        for (int i = max(0, ni - 1); i <= ni; ++i)
          if (i < ni || g > 0) mbar_wait(&ctl->k_full[i & 1], (i >> 1) & 1, &own, kErrWaitProducer);
      }
    } else if (warp == 1 && elect_one()) {
      // ---------------------------------------------------------------- products
      constexpr uint32_t id = idesc_f16(128, 128, kBf16 ? 1 : 0, 0, 0);
      const uint64_t dK = smem_desc_sw128(smem_u32(sK), 16, 1024), dQ = smem_desc_sw128(smem_u32(sQ), 16, 1024);
      bool ok = true;
      int g = 0, ni = 0;
      for (int r = 0; r < rounds && ok; ++r)
      for (Walk it(p, ctl->share[r]); it.left > 0 && ok; it.next(p), ++ni) {
        const int kb = ni & 1;
        ok = mbar_wait(&ctl->k_full[kb], (ni >> 1) & 1, err, kErrWaitMma);
        for (int i = it.start; i < it.stop && ok; ++i, ++g) {
          const int st = g % kQStages, sb = g & 1;
          ok = mbar_wait(&ctl->q_full[st], (g / kQStages) & 1, err, kErrWaitMma);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (ok && g >= 2) ok = mbar_wait(&ctl->s_free[sb][t], ((g >> 1) - 1) & 1, err, kErrWaitMma);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < kD / 16; ++k) {
              const uint32_t off = ((k >> 2) * kBoxBytes + (k & 3) * 32) >> 4;
              mma_ss(tmem + sb * 256 + t * 128, dK + (kb * 2 + t) * kTile16 + off, dQ + st * kTile16 + off, id, k > 0 ? 1u : 0u);
            }
            mma_commit(&ctl->s_ready[sb][t]);
          }
          if (!ok) break;
          mma_commit(&ctl->q_free[st]);
        }
        mma_commit(&ctl->k_free[kb]);
      }
      if (!ok) {
        // products under way must not outlive the CTA's tensor memory (a limited wait)
        int own = 0;
        mma_commit(&ctl->drained);
        mbar_wait(&ctl->drained, 0, &own, kErrWaitMma);
      }
    } else if (warp == 2) {
      // ---------------------------------------------------------------- rows of -lse * log2(e)
      bool ok = true;
      int g = 0;
      for (int r = 0; r < rounds && ok; ++r)
      for (Walk it(p, ctl->share[r]); it.left > 0 && ok; it.next(p)) {
        const int b = it.bh / p.hkv, h = it.bh - b * p.hkv;
        for (int i = it.start; i < it.stop; ++i, ++g) {
          const int sb = g & 1, hd = h * p.group + i / it.n_qt, q0 = it.kt * kKeys + i % it.n_qt * kTile;
          const float* src = p.lse + b * p.l_sb + hd * p.l_sh + q0;
          float x[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int r = k * 32 + lane;
            x[k] = q0 + r < p.len ? src[r] * -1.4426950408889634f : -INFINITY;
            if (x[k] == INFINITY) x[k] = -INFINITY;  // a query that saw nothing
          }
          for (int t = 0; t < 2 && ok && g >= 2; ++t) ok = mbar_wait_w<100>(&ctl->s_free[sb][t], ((g >> 1) - 1) & 1, err, kErrWaitProducer);
          if (!ok) break;
#pragma unroll
          for (int k = 0; k < 4; ++k) sLse[sb * kTile + k * 32 + lane] = x[k];
          __syncwarp();
          if (lane < 2) mbar_arrive(&ctl->s_ready[sb][lane]);
        }
      }
    }
  } else {
    setmaxnreg_inc<104>();  // 128 x 64 + 512 x 104 <= 640 x 96 (the launch allocation)
    // ---------------------------------------------------------------- sums
    const int tile = (warp - 4) >> 3, half = (warp - 4) >> 2 & 1, key = tile * kTile + (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    float* const s_half = reinterpret_cast<float*>(smem + kSmemHalf);  // [kKeys]: the sums of the upper 64 columns
    const float2 sl = make_float2(p.scale_log2, p.scale_log2);
    bool ok = true;
    int g = 0;
    for (int r = 0; r < rounds && ok; ++r)
    for (Walk it(p, ctl->share[r]); it.left > 0 && ok; it.next(p)) {
      const int t0 = it.kt * kKeys, t = t0 + key;
      // the queries that see this key
      int lo = 0x7fffffff, hi = -1;
      if (t < p.len) {
        int s, e;
        seq_of(p.cu, p.n_seqs, t, s, e);
        e = min(e, p.len);
        lo = t;
        hi = t - s < p.n_sink || e - 1 - t <= p.window ? e - 1 : t + p.window;
      }
      const uint32_t seen = static_cast<uint32_t>(max(hi - lo + 1, 0));
      float sum = 0.f, lost = 0.f;
      int qt = it.start % it.n_qt - 1;
      for (int i = it.start; i < it.stop; ++i, ++g) {
        if (++qt == it.n_qt) qt = 0;
        const int sb = g & 1, q0 = t0 + qt * kTile + half * 64;
        ok = mbar_wait_w(&ctl->s_ready[sb][tile], (g >> 1) & 1, err, kErrWaitSoftmax);
        if (!ok) break;
        tc_fence_after();
        const bool none = q0 + 63 < lo || q0 > hi, full = q0 >= lo && q0 + 63 <= hi;
        if (!__all_sync(0xffffffffu, none)) {
          const bool masked = !__all_sync(0xffffffffu, full);
          const float* lse = sLse + sb * kTile + half * 64;
          const uint32_t from = tmem + sb * 256 + tile * 128 + half * 64 + lane_off;
          float2 acc[4] = {};
          uint32_t x[2][32];
          tmem_ld32(from, x[0]);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            tmem_ld_wait();
            if (c == 0) tmem_ld32(from + 32, x[1]);
            // (hidden pairs are taken out of the exponents, behind the log-sum-exps: one that is NaN is not theirs)
            const uint32_t at0 = static_cast<uint32_t>(q0 + c * 32 - lo);
            const auto add = [&](auto some_hidden) {
#pragma unroll
              for (int k = 0; k < 32; k += 4) {
                const float4 l = *reinterpret_cast<const float4*>(lse + c * 32 + k);
                float2 a = __ffma2_rn(make_float2(__uint_as_float(x[c][k]), __uint_as_float(x[c][k + 1])), sl, make_float2(l.x, l.y));
                float2 b = __ffma2_rn(make_float2(__uint_as_float(x[c][k + 2]), __uint_as_float(x[c][k + 3])), sl, make_float2(l.z, l.w));
                if (decltype(some_hidden)::value) {
                  a.x = at0 + k < seen ? a.x : -INFINITY, a.y = at0 + k + 1 < seen ? a.y : -INFINITY;
                  b.x = at0 + k + 2 < seen ? b.x : -INFINITY, b.y = at0 + k + 3 < seen ? b.y : -INFINITY;
                }
                const float2 ea = make_float2(ex2f(a.x), ex2f(a.y));
                const float2 eb = k % 16 == 0 ? fma_exp2(b) : make_float2(ex2f(b.x), ex2f(b.y));
                acc[k / 4 % 2 * 2] = __fadd2_rn(acc[k / 4 % 2 * 2], ea);
                acc[k / 4 % 2 * 2 + 1] = __fadd2_rn(acc[k / 4 % 2 * 2 + 1], eb);
              }
            };
            if (masked) add(std::true_type()); else add(std::false_type());
          }
          const float2 s2 = __fadd2_rn(__fadd2_rn(acc[0], acc[1]), __fadd2_rn(acc[2], acc[3]));
          float s1 = s2.x + s2.y;
          if (__any_sync(0xffffffffu, s1 != s1)) {
            // once more, pair by pair: a query that saw nothing adds nothing, even where its scores are not finite
            s1 = 0.f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              tmem_ld32(from + c * 32, x[0]);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 32; ++k) {
                const float l = lse[c * 32 + k];
                if (static_cast<uint32_t>(q0 + c * 32 + k - lo) < seen && l != -INFINITY) s1 += ex2f(__fmaf_rn(__uint_as_float(x[0][k]), p.scale_log2, l));
              }
            }
          }
          // (compensated: `lost` is what the last addition rounded away)
          const float y = s1 - lost, z = sum + y;
          lost = (z - sum) - y;
          sum = z;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->s_free[sb][tile]);
      }
      // the two halves of the columns.  (All of these warps come here, whatever happened, and go on or leave together.)
      if (half == 1) s_half[key] = sum;
      ok = all_sum_warps(ok);
      if (half == 0) sum += s_half[key];
      ok = all_sum_warps(ok);
      if (ok && half == 0) {
        const bool whole = it.start == 0 && it.stop == it.n(p);
        if (whole) {
          if (t < p.len) p.out[static_cast<long long>(it.bh) * p.len + t] = sum;
        } else {
          p.part[((blockIdx.x + static_cast<long long>(r) * p.ctas) * 2 + (it.start == 0 ? 1 : 0)) * kKeys + key] = sum;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
  if (threadIdx.x == 0 && ctl->err != 0) raise_status(p.status, p.mirror, ctl->err);
}

// Adds the pieces of an item that more than one CTA worked on, in order.  CTA c looks at the boundary between the shares c
// and c + 1; of the boundaries inside an item, the first one's CTA does the work.
__global__ void __launch_bounds__(kKeys) weight_sums_join_kernel(const __grid_constant__ SumsKernelParams p) {
  __shared__ long long s_prefix[kScan + 1 + kScan / 32];
  griddep_wait();
  item_prefix(p, s_prefix, s_prefix + kScan + 1);
  const long long total = s_prefix[kScan] * p.group * p.hkv * p.batch;
  const long long shares = n_shares(total, p);
  if (blockIdx.x + 1 >= shares) return;
  const long long at = share_begin(total, shares, blockIdx.x + 1);
  const Item it = item_at(p, s_prefix, at);
  if (it.first == at || it.first < share_begin(total, shares, blockIdx.x)) return;
  float sum = 0.f;
  for (long long c = blockIdx.x; c < shares && share_begin(total, shares, c) < it.first + it.n; ++c)
    sum += p.part[(c * 2 + (c == blockIdx.x ? 1 : 0)) * kKeys + threadIdx.x];
  const int t = it.kt * kKeys + threadIdx.x;
  if (t < p.len) p.out[static_cast<long long>(it.bh) * p.len + t] = sum;
}

int64_t part_bytes(int shares) { return static_cast<int64_t>(shares) * 2 * kKeys * 4; }

template <int kD, bool kBf16>
cudaError_t launch_sums(const SumsKernelParams& kp, cudaStream_t s) {
  const auto kern = weight_sums_kernel<kD, kBf16>;
  static std::atomic<uint64_t> set{0};  // devices on which the kernel's shared memory has been allowed
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !(set.load(std::memory_order_relaxed) >> dev & 1)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (e != cudaSuccess) return e;
    if (dev < 64) set.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  e = launch_kernel(kern, dim3(kp.ctas), kThreads, kSmemBytes, s, true, kp);
  if (e != cudaSuccess) return e;
  count_launches(1);
  if (kp.ctas * kp.rounds > 1) {
    e = launch_kernel(weight_sums_join_kernel, dim3(kp.ctas * kp.rounds - 1), kKeys, 0, s, true, kp);
    if (e != cudaSuccess) return e;
    count_launches(1);
  }
  return cudaSuccess;
}

// CTAs of a call: one per SM, fewer where the keys' own tiles alone are fewer steps
int sums_ctas(const rswa_weight_sums_params_t& p) {
  const long long steps = static_cast<long long>(p.batch) * p.n_q_heads * ((p.len + kTile - 1) / kTile) * 8;
  const int sms = sm_count();
  return static_cast<int>(steps < sms ? steps : sms);
}

// Rounds: the queries of one fit into L2, with room for what else passes through
int sums_rounds(const rswa_weight_sums_params_t& p) {
  const long long bytes = static_cast<long long>(p.batch) * p.len * p.n_q_heads * p.head_dim * 2;
  return static_cast<int>(std::min<long long>(kMaxRounds, (bytes + kRoundBytes - 1) / kRoundBytes));
}

int check_sums(const rswa_weight_sums_params_t* p) {
  const char* what = "rswa_weight_sums";
  if (p == nullptr) {
    set_error("%s: null params", what);
    return RSWA_E_ARG;
  }
  if (p->dtype != RSWA_DTYPE_BF16 && p->dtype != RSWA_DTYPE_FP16) {
    set_error("%s: dtype must be bf16 (0) or fp16 (1), got %d", what, p->dtype);
    return RSWA_E_UNSUPPORTED;
  }
  if (p->head_dim != 64 && p->head_dim != 128) {
    set_error("%s: head_dim must be 64 or 128, got %d", what, p->head_dim);
    return RSWA_E_UNSUPPORTED;
  }
  if (p->batch <= 0 || p->len <= 0 || p->n_q_heads <= 0 || p->n_kv_heads <= 0 || p->window < 0 || p->n_sink < 0) {
    set_error("%s: batch, len and head counts must be positive, window and n_sink not negative", what);
    return RSWA_E_ARG;
  }
  if (p->n_q_heads % p->n_kv_heads != 0) {
    set_error("%s: Number of query heads must be divisible by number of key/value heads", what);
    return RSWA_E_ARG;
  }
  if (p->len > 0x7fffffff - 4 * kTile || p->batch > 0x7fffffff / p->n_kv_heads) {
    set_error("%s: positions overflow int32", what);
    return RSWA_E_UNSUPPORTED;
  }
  // (a CTA counts its steps in 32 bits: 40 minutes of work.  At most: what the window spans for every item, and all query
  // tiles for those with a sink token)
  const double tiles = p->len / kTile + 1.0, items = p->len / kKeys + 1.0;
  const double steps = items * std::min(tiles, p->window / static_cast<double>(kTile) + 4.0) + tiles * (p->n_sink / static_cast<double>(kKeys) + 2.0);
  if (steps * p->n_q_heads * p->batch > 100.0 * 0x7fffffff) {
    set_error("%s: too many tiles in one call", what);
    return RSWA_E_UNSUPPORTED;
  }
  if (p->cu_seqlens != nullptr && (p->batch != 1 || p->n_seqs <= 0)) {
    set_error("%s: packed (cu_seqlens) input needs batch == 1 and n_seqs > 0", what);
    return RSWA_E_ARG;
  }
  if (!(p->softmax_scale > 0.f)) {
    set_error("%s: softmax_scale must be positive", what);
    return RSWA_E_ARG;
  }
  return RSWA_OK;
}

}  // namespace

}  // namespace rswa

using namespace rswa;

extern "C" int64_t rswa_weight_sums_workspace_bytes(const rswa_weight_sums_params_t* p) {
  const int rc = check_sums(p);
  return rc != RSWA_OK ? rc : part_bytes(sums_ctas(*p) * sums_rounds(*p));
}

extern "C" int rswa_weight_sums(const rswa_weight_sums_params_t* p, void* stream) {
  const char* what = "rswa_weight_sums";
  int rc = check_sums(p);
  if (rc != RSWA_OK) return rc;
  if (p->lse == nullptr || p->out == nullptr || p->status == nullptr) {
    set_error("%s: lse, out and status are required", what);
    return RSWA_E_ARG;
  }
  SumsKernelParams kp;
  kp.ctas = sums_ctas(*p);
  kp.rounds = sums_rounds(*p);
  const int shares = kp.ctas * kp.rounds;
  if (p->workspace == nullptr || p->workspace_bytes < part_bytes(shares)) {
    set_error("%s: the workspace must hold %lld bytes", what, static_cast<long long>(part_bytes(shares)));
    return RSWA_E_ARG;
  }
  rc = make_tile_map(&kp.q_map, p->q, p->dtype, p->batch, p->len, p->n_q_heads, p->head_dim, p->q_stride_b, p->q_stride_t, p->q_stride_h);
  if (rc == RSWA_OK) rc = make_tile_map(&kp.k_map, p->k, p->dtype, p->batch, p->len, p->n_kv_heads, p->head_dim, p->k_stride_b, p->k_stride_t, p->k_stride_h);
  if (rc != RSWA_OK) return rc;
  kp.lse = p->lse;
  kp.l_sb = p->lse_stride_b, kp.l_sh = p->lse_stride_h;
  kp.batch = p->batch, kp.len = p->len, kp.hq = p->n_q_heads, kp.hkv = p->n_kv_heads, kp.group = p->n_q_heads / p->n_kv_heads;
  // (beyond the prompt's length nothing changes)
  kp.window = p->window < p->len ? p->window : p->len;
  kp.n_sink = p->n_sink < p->len ? p->n_sink : p->len;
  kp.scale_log2 = p->softmax_scale * 1.4426950408889634f;
  kp.cu = p->cu_seqlens;
  kp.n_seqs = p->n_seqs;
  kp.out = p->out;
  kp.part = static_cast<float*>(p->workspace);
  kp.n_items = (p->len + kKeys - 1) / kKeys;
  kp.status = p->status;
  kp.mirror = status_mirror(p->status);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf16 = p->dtype == RSWA_DTYPE_BF16;
  const cudaError_t e = p->head_dim == 64 ? (bf16 ? launch_sums<64, true>(kp, s) : launch_sums<64, false>(kp, s))
                                          : (bf16 ? launch_sums<128, true>(kp, s) : launch_sums<128, false>(kp, s));
  if (e != cudaSuccess) {
    set_error("%s: launch failed: %s", what, cudaGetErrorString(e));
    return RSWA_E_CUDA;
  }
  return RSWA_OK;
}
