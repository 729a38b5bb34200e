// Attention of the newest token(s) of every sequence over its cached tokens (see rswa_cache_attn in rswa.h).
//
//   out = sum_t p_t v_t,  p_t = exp(scale * q.k_t - lse)  over the visible slots t
//
// in one pass over K and V: running maximum and sum per row, K and V brought in by TMA and never in any form but the
// stored bytes until they are operands.  What has to be moved is 2 * head_dim bytes per visible token and key/value
// head; the products are 4 * head_dim FLOPs on them per query head, 16 a byte with 8 of them: 105 TFLOP/s at the rate of
// HBM, which is more than the FMA pipe gives and a fifth of what mma.m16n8k16 does (8 cycles each, measured).
// Streaming runs at 5 to 6 TB/s; what is left is the way in (lengths, block table, first tiles: 5 us), the end of the
// pieces and their joining (4 us), and that SMs get unequal shares of the bandwidth (the last group ends 8 us behind
// the median one of 40).  161 MB (32 requests of 300 to 8192 tokens, 32/8 heads, e4m3) 40.1 us: 4.0 TB/s.
//
// Products: mma.m16n8k16 with the KEYS (the V columns) as the 16 rows and the query rows as the 8 columns, so that a
// group of up to 8 rows wastes nothing on the operand that costs: the one converted from bytes.  (tcgen05 wants 128
// rows of A, both operands in the same 8-bit or 16-bit type in shared memory: the bytes would have to be converted and
// written back there, or the queries and weights rounded to 8 bits.)  A word of four stored bytes becomes two operand
// registers in place.  For K the order of the head dimension inside a product is free (the queries are laid out the
// same way); for V the two registers are two columns of the head, whose weights are the same.
//   S^T[token][row] = K q^T        ldmatrix: lane (g, c) of a quad layout holds d = 16 s + 4c .. 4c + 3 of token g
//   O^T[d][row]    += V^T P^T      ldmatrix.trans: lane holds d = 16 m + 2g, 2g + 1 of tokens 2c, 2c + 1
// P^T comes out of S^T's accumulators by two 8x8 transposes (movmatrix) per 16 tokens.
//
// Queries and weights are fp16 operands: a bf16 query is scaled by a power of two to the top of the fp16 range (exact
// but for elements 2^-28 smaller than the row's largest), the weights are at most 2^14 with 11 bits each.  The scale of
// a V block goes into its tokens' exponents (s + log2 of the scale), so that the running reference covers both;
// the sum of the weights takes it back out.  Scores, sums and the output are 32-bit.  (The sum of the weights is kept in units
// of 2^8 of the reference, and takes exponentials of its own from blocks of V with scales below 2^-20, such as blocks of zeros: with
// the scale in it a weight falls out of the range of 32 bits where another block's V is 2^100 times larger.  That, and V's
// scales that are not finite, are a copy of the code that forms the weights, taken for tiles that have them: in one with the usual
// code the exponentials of a tile no longer overlap, 28.6 us become 29.3 for the four windows of 8192 below.)
//
// Work: the 32-token tiles of all (sequence, key/value head, 8 or 16 query rows) in one order, cut evenly whatever the
// lengths over groups of warps.  The warps of a group take its tiles in turn and add up at the end of each piece; each item
// counts one tile per warp more than it has, for that and for its queries (32 requests of 300 to 8192 tokens: 43.6 us
// without, 40 with it).  Where there are more (sequence, head, row tile)s than SMs a group is four warps, because the end of a piece and the next one's queries
// cost every warp that takes part as much as several tiles (the same requests: 48 us, and 69 with
// all 16 warps of an SM in one group); else it is all warps of the SM, which leaves fewer pieces to join.
// Every warp loads for itself: K of its next tile as soon as the scores are formed, V as soon as the output is, on over
// sequence boundaries; its lanes look 32 tiles up in the block table at a time, so that the table's latency is paid once for
// all of them.  The pieces of an item that is cut go to the workspace, and the group that delivers the last one joins them,
// in order: results do not depend on timing.
#include <atomic>
#include <type_traits>

#include "rswa_cache.cuh"

namespace rswa {

int make_rows_map(CUtensorMap* map, const void* base, long long rows, int row_bytes, int box_rows);
int check_table(const rswa_block_table_t& t, bool written, const int32_t* lens, const int32_t* status, int block_size, const char* what);

using namespace tc05;

namespace {

constexpr int kTok = 32;     // tokens of a tile
constexpr int kScan = 256;   // threads of the prefix sums over sequences
constexpr int kAdd = 256;    // threads of a CTA that adds weights up
constexpr float kRoom = 14.f;  // a weight may grow to 2^14 before the reference is raised (fp16 ends at 2^16)
constexpr float kLow = 4.f;    // and is raised to the maximum minus 4, so that not every new maximum raises it
constexpr float kSumUnit = 8.f;    // sums of weights are in units of 2^8: 2^21 tokens of weight 2^14 under V's least scale, 2^-100, stay finite
constexpr float kSumScale = 1.f / 256;
constexpr float kTinyV = -20.f;    // log2 of V's scale, below which the sum has exponentials of its own

constexpr int kNoTile = -1, kBlank = -1024;  // rows of the cache: of a tile that is not there, and in front of the first one (loads give zeros)

struct AttnKernelParams {
  CUtensorMap map[2];
  CacheView c;
  const int* table;
  long long table_stride;
  int batch, max_blocks;
  const int* lens;
  const uint16_t* q;
  long long q_sb, q_st, q_sh;
  int q_len, hq, group, rows, row_tiles;  // rows = q_len * group, in tiles of 8 * kNT
  int window, n_sink;                     // window < 0: all
  float scale_log2;
  int bf16;
  uint16_t* out;
  float* lse;        // or null
  float* part_o;     // [groups][2][8 * kNT][head_dim]
  float* part_ml;    // [groups][2][8 * kNT][2]
  int* arrived;      // [groups], 0 between calls: pieces of the item that a group begins and does not finish
  float* scores;     // [tiles][kTok][8 * kNT], or null: what the weights need
  int* first;        // [batch]: index of a sequence's first tile, with scores
  float* weights;
  long long w_sb, w_sh;
  int groups;
  int* status;
  int* mirror;
};

// The tiles of one sequence: the ones its sink tokens lie in, then the ones from its oldest visible token on.
// An item of n tiles counts as n + kOver (kOver ones that are not there, then its tiles), one without any as none.
struct SeqTiles {
  int len, n_sink_tiles, n;
  int oldest;  // the first slot in the window of any query
};
template <int kOver>
__device__ __forceinline__ SeqTiles seq_tiles(const AttnKernelParams& p, int b) {
  SeqTiles s;
  int len = p.lens[b];
  const int cap = p.max_blocks * p.c.bs;
  if (len < 0 || len > cap) {
    raise_status(p.status, p.mirror, kErrSeqLen);
    len = 0;
  }
  s.oldest = p.window < 0 ? 0 : max(0, max(0, len - p.q_len) - p.window);
  s.len = len;
  s.n_sink_tiles = min((min(p.n_sink, len) + kTok - 1) / kTok, s.oldest / kTok);
  const int n = s.n_sink_tiles + (len + kTok - 1) / kTok - s.oldest / kTok;
  s.n = n > 0 ? n + kOver : 0;
  return s;
}
__device__ __forceinline__ int tile_slot(const SeqTiles& s, int i) { return (i < s.n_sink_tiles ? i : s.oldest / kTok + i - s.n_sink_tiles) * kTok; }

// Where the work of a group begins and ends: equal shares of all tiles.  Not more of them than there is a tile per warp for,
// but one for each item at least: a group that takes short items one after the other pays for each of them.
struct Shares {
  int n, each, more;  // `more` shares have each + 1 tiles, the others each
  __device__ __forceinline__ Shares(int total, int groups, int items, int over, int warps) {
    n = max(1, min(min(groups, total), max(items, (total - items * over) / warps)));
    each = total / n;
    more = total - each * n;
  }
  __device__ __forceinline__ int begin(int c) const { return c * each + min(c, more); }
  __device__ __forceinline__ int of(int tile) const {
    const int large = more * (each + 1);
    return tile < large ? tile / (each + 1) : more + (tile - large) / each;
  }
};

// (counted with the kOver from here on)
// Prefix sums of the sequences' tiles (per key/value head and row tile): thread i of the first kScan holds `per`
// sequences.  s_prefix[i]: tiles in front of thread i's sequences; s_prefix[kScan]: all.
template <int kOver>
__device__ __forceinline__ void tile_prefix(const AttnKernelParams& p, int* s_prefix, int* s_warp) {
  const int per = (p.batch + kScan - 1) / kScan;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int mine = 0, sum = 0;
  if (threadIdx.x < kScan) {
    for (int i = 0; i < per; ++i) {
      const int b = threadIdx.x * per + i;
      if (b < p.batch) mine += seq_tiles<kOver>(p, b).n;
    }
    sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    if (lane == 31) s_warp[warp] = sum;
  }
  __syncthreads();
  if (threadIdx.x < kScan) {
    int before = 0;
    for (int w = 0; w < warp; ++w) before += s_warp[w];
    before += sum - mine;
    s_prefix[threadIdx.x] = before;
    if (threadIdx.x == kScan - 1) s_prefix[kScan] = before + mine;
    if (p.first != nullptr && blockIdx.x == 0) {
      const int items = p.c.hkv * p.row_tiles;
      for (int i = 0; i < per; ++i) {
        const int b = threadIdx.x * per + i;
        if (b >= p.batch) break;
        p.first[b] = before * items;
        before += seq_tiles<kOver>(p, b).n;
      }
    }
  }
  __syncthreads();
}

// A place in the order of all tiles: sequence, then head, then row tile, then tile.
template <int kOver>
struct Cursor {
  int b, item, i;       // item = head * row_tiles + row tile
  SeqTiles s;
  int at;         // index among all tiles
  // moves forward by n tiles; false: behind the last
  __device__ __forceinline__ void skip(const AttnKernelParams& p, int n, int end) {
    at += n;
    if (at >= end) return;
    int k = i + n;
    const int items = p.c.hkv * p.row_tiles;
    while (k >= s.n) {
      k -= s.n;
      if (++item == items) {
        item = 0;
        do s = seq_tiles<kOver>(p, ++b); while (s.n == 0);
      }
    }
    i = k;
  }
};
template <int kOver>
__device__ __forceinline__ Cursor<kOver> cursor_at(const AttnKernelParams& p, const int* s_prefix, int tile) {
  const int items = p.c.hkv * p.row_tiles;
  const int per = (p.batch + kScan - 1) / kScan;
  int lo = 0, hi = kScan - 1;  // the last thread whose prefix is not behind the tile
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s_prefix[mid] * items <= tile) lo = mid; else hi = mid - 1;
  }
  // (threads of no tiles share a prefix: the last of them holds the tile, or has no sequences and the walk starts
  // at a sequence of its own)
  Cursor<kOver> c;
  c.at = tile;
  c.b = lo * per;
  int rest = tile - s_prefix[lo] * items;
  c.s = seq_tiles<kOver>(p, c.b);
  while (rest >= c.s.n * items) {
    rest -= c.s.n * items;
    c.s = seq_tiles<kOver>(p, ++c.b);
  }
  c.item = rest / c.s.n;
  c.i = rest - c.item * c.s.n;
  return c;
}

template <int kD>
struct Ring {
  static constexpr int kTileBytes = kTok * kD;      // of K, and of V
  static constexpr int kStageBytes = 2 * kTileBytes;
};

// 16 warps of 128 registers a thread, or for 16 query rows 8 of 255 (12 of 168 spill: 4 x 128k tokens with sinks, 4 queries:
// 32 us, and 28.6 so; a second tile in flight per warp then gives nothing).  A tile in flight per warp is 128 KB or 64 an SM,
// where the latency of a load asks for about 50.
// kAll: all warps are one group.
template <int kD, int kNT, bool kAll>
struct Layout {
  static constexpr int kWarps = kNT == 1 ? 16 : 8;
  static constexpr int kThreads = kWarps * 32, kGroup = kAll ? kWarps : 4, kGroups = kWarps / kGroup;
  struct Ctl {
    uint64_t full[kWarps][2];           // K, V
    float4 scale[kWarps][32][2];        // the looked-up tiles: of the first 16 tokens and the last 16 K's scale, log2 of V's, 2^-kSumUnit / V's (negative: see put_scales)
    int2 row[kWarps][32];               // and where their K and V lie
    float ml[kWarps][8 * kNT][2];       // reference and sum of every warp's piece
    int prefix[kScan + 1 + kScan / 32];
    int last[kGroups];                  // whether the group's piece was the last one to arrive
    int err;
  };
  static constexpr int kRings = kWarps * Ring<kD>::kStageBytes;
  static constexpr int kMerge = kWarps * 8 * kD * 4;
  // [tiles][sums of the warps' pieces][control]
  static constexpr int kBytes = kRings + kMerge + static_cast<int>(sizeof(Ctl));
  static_assert(kBytes <= 232448, "shared memory budget");
};

__device__ __forceinline__ void tma_load_rows(void* dst, const CUtensorMap* m, uint64_t* bar, int row) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(0), "r"(row)
      : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16-byte piece `chunk` of row `row` of a tile, as TMA's swizzle left it
template <int kD>
__device__ __forceinline__ uint32_t piece(uint32_t base, int row, int chunk) {
  return base + row * kD + ((kD == 128 ? chunk ^ (row & 7) : chunk ^ ((row >> 1) & 3)) << 4);
}

template <int kThreads>
__device__ __forceinline__ void sync_group(int group) {
  asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(kThreads) : "memory");
}
// four elements of a finished row, and its log-sum-exp
template <int kD>
__device__ __forceinline__ void store_row(const AttnKernelParams& p, int b, int h, int row, int d4, float4 x, float top, float sum) {
  const int i = row / p.group, hd = h * p.group + row - i * p.group;
  const float inv = sum == 0.f ? 0.f : 1.f / sum * kSumScale;
  uint16_t* const to = p.out + ((static_cast<long long>(b) * p.q_len + i) * p.hq + hd) * kD + d4 * 4;
  *reinterpret_cast<uint2*>(to) = p.bf16 ? make_uint2(pack2<true>(x.x * inv, x.y * inv), pack2<true>(x.z * inv, x.w * inv))
                                         : make_uint2(pack2<false>(x.x * inv, x.y * inv), pack2<false>(x.z * inv, x.w * inv));
  if (p.lse != nullptr && d4 == 0)
    p.lse[(static_cast<long long>(b) * p.hq + hd) * p.q_len + i] = sum == 0.f ? -INFINITY : (top + kSumUnit + __log2f(sum)) * 0.6931471805599453f;
}

// The rows of the sequences that have nothing to attend to, by the first kPeers threads of every CTA.
template <int kD, int kPeers>
__device__ __forceinline__ void empty_rows(const AttnKernelParams& p) {
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
    if (seq_tiles<0>(p, b).n > 0) continue;
    for (int row = threadIdx.x / (kD / 4); row < p.rows * p.c.hkv; row += kPeers / (kD / 4))
      store_row<kD>(p, b, row / p.rows, row % p.rows, threadIdx.x % (kD / 4), make_float4(0.f, 0.f, 0.f, 0.f), 0.f, 0.f);
  }
}

// Joins the pieces of an item in the order of the groups `lo` to lo + pieces - 1 that worked on it; by the kPeers threads
// of one group.  With more threads than a row tile has 16-byte parts the pieces are dealt out to several of them, whose sums
// are added in order.  (The other groups' pieces are read past L1, which does not see what other SMs write.)
template <int kD, int kNT, int kPeers>
__device__ __forceinline__ void join_pieces(const AttnKernelParams& p, float* merge, int group, int b, int h, int row0, int lo, int pieces) {
  constexpr int kRows = 8 * kNT, kUnits = kRows * kD / 4, kParts = kPeers >= 2 * kUnits ? kPeers / kUnits : 1;
  const int t = threadIdx.x - group * kPeers;
  const int part = kParts > 1 ? t / kUnits : 0;
  float4* const s_x = reinterpret_cast<float4*>(merge);                              // [kParts][kUnits]
  float2* const s_ml = reinterpret_cast<float2*>(merge + kParts * kUnits * 4);       // [kParts][kRows]
  for (int u = kParts > 1 ? t % kUnits : t; u < kUnits; u += kParts > 1 ? kUnits : kPeers) {
    const int r = u / (kD / 4), d4 = u % (kD / 4), row = row0 + r;
    const auto place = [&](int k) { return (static_cast<long long>(lo + k) * 2 + (k == 0 ? 1 : 0)) * kRows + r; };
    float top = -INFINITY, sum = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    const auto add = [&](float m, float l, float4 y) {  // a later piece
      const float next = fmaxf(top, m);
      // (references may lie so far apart, by V's scales, that the factor is 0 where a sum times the factor is not)
      const float fh = sum == 0.f ? 0.f : ex2f(0.5f * (top - next)), wh = l == 0.f ? 0.f : ex2f(0.5f * (m - next));
      const float f = fh * fh, w = wh * wh;
      top = next;
      sum = sum * fh * fh + l * wh * wh;
      x.x = x.x * f + y.x * w, x.y = x.y * f + y.y * w, x.z = x.z * f + y.z * w, x.w = x.w * f + y.w * w;
    };
    if (row < p.rows && part < kParts) {
#pragma unroll 4
      for (int k = part; k < pieces; k += kParts) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml + place(k) * 2));
        add(ml.x, ml.y, __ldcg(reinterpret_cast<const float4*>(p.part_o + place(k) * kD + d4 * 4)));
      }
      if (kParts == 1) store_row<kD>(p, b, h, row, d4, x, top, sum);
    }
    if (kParts > 1) {
      s_x[part * kUnits + u] = x;
      if (d4 == 0) s_ml[part * kRows + r] = make_float2(top, sum);
      sync_group<kPeers>(group);
      if (part == 0 && row < p.rows) {
#pragma unroll
        for (int k = 1; k < kParts; ++k) {
          const float2 ml = s_ml[k * kRows + r];
          add(ml.x, ml.y, s_x[k * kUnits + u]);
        }
        store_row<kD>(p, b, h, row, d4, x, top, sum);
      }
      sync_group<kPeers>(group);  // (before the next piece's sums)
    }
  }
}

// kNT: query rows in columns of 8.
template <int kD, int kNT, bool kInt8, bool kAll>
__global__ void __launch_bounds__((Layout<kD, kNT, kAll>::kThreads), 1) cache_attn_kernel(const __grid_constant__ AttnKernelParams p) {
  using L = Layout<kD, kNT, kAll>;
  using R = Ring<kD>;
  constexpr int kKS = kD / 16, kGroup = L::kGroup, kPeers = kGroup * 32, kOver = kGroup;
  constexpr int kRows = 8 * kNT;
  extern __shared__ __align__(1024) uint8_t smem[];
  auto& ctl = *reinterpret_cast<typename L::Ctl*>(smem + L::kRings + L::kMerge);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int group = warp / kGroup, wg = warp % kGroup;
  // (the first groups of all CTAs come first: a call too small for all of them spreads over the SMs)
  const int me = group * gridDim.x + blockIdx.x;
  float* const merge = reinterpret_cast<float*>(smem + L::kRings) + group * kGroup * 8 * kD;
  auto& ml = *reinterpret_cast<float(*)[kGroup][kRows][2]>(ctl.ml[group * kGroup]);
  uint8_t* const own = smem + warp * R::kStageBytes;  // this warp's tile: K, then V
  uint64_t* const full = ctl.full[warp];

  griddep_launch();
  if (threadIdx.x == 0) {
    ctl.err = 0;
    prefetch_tmap(&p.map[0]);
    prefetch_tmap(&p.map[1]);
  }
  if (lane < 2) mbar_init(full + lane, 1);
  mbar_fence_init();
  griddep_wait();
  tile_prefix<kOver>(p, ctl.prefix, ctl.prefix + kScan + 1);
  const int total = ctl.prefix[kScan] * p.c.hkv * p.row_tiles;
  const Shares shares(total, p.groups, p.batch * p.c.hkv * p.row_tiles, kOver, kGroup);
  if (me >= shares.n || total == 0) {
    if (group == 0) empty_rows<kD, kPeers>(p);
    return;
  }
  const int begin = shares.begin(me), end = shares.begin(me + 1);
  const int box = min(p.c.bs, kTok);

  // The tiles of this warp, counted: tile i is the share's tile wg + i * kGroup.  Looks 32 of them up, one a lane.
  // (The warp is told of a tile that is not there by a row of kNoTile.)
  const int n_own = (end - begin - wg + kGroup - 1) / kGroup;
  int page[2], tokens;  // of this lane's tile
  auto look_up = [&](int i) {
    const int at = begin + wg + (i + lane) * kGroup;
    page[0] = page[1] = -1, tokens = 0;
    __syncwarp();
    if (at < end) {
      const auto lc = cursor_at<kOver>(p, ctl.prefix, at);
      int2 row = make_int2(kNoTile, kNoTile);
      if (lc.i >= kOver) {
        const int bs = p.c.bs, slot = tile_slot(lc.s, lc.i - kOver), h = lc.item / p.row_tiles, j = slot / bs;
        // a tile is part of one block, or two blocks of 16, of which one may have no slot that anybody sees (behind the sinks, in
        // front of the window, behind the end): that one is not looked at, and loads zeros
        // (an entry that is no block has been reported; any block will do then)
        const int* const entry = p.table + lc.b * p.table_stride + j;
        const int e0 = entry[0], e1 = entry[bs < kTok && slot + bs < lc.s.len];  // (one latency; what is not looked at may be anything)
        const auto block = [&](int e) {
          if (e >= 0 && e < p.c.num_blocks) return e * p.c.hkv + h;
          raise_status(p.status, p.mirror, kErrBlockTable);
          return h;
        };
        const auto seen = [&](int from) { return from < lc.s.len && (from < p.n_sink || from + 16 > lc.s.oldest); };
        if (bs >= kTok || seen(slot)) page[0] = block(e0);
        if (bs >= kTok) page[1] = page[0];
        else if (seen(slot + 16)) page[1] = block(e1);
        tokens = lc.s.len - slot;
        row = make_int2(page[0] < 0 ? kBlank : page[0] * bs + slot % bs, page[1] < 0 ? kBlank : page[1] * bs + slot % bs);
      }
      ctl.row[warp][lane] = row;
    }
    __syncwarp();
  };
  float scale[2][2];  // K's and V's, of the first 16 tokens and the last 16
  auto fetch_scales = [&]() {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const bool some = 16 * t < tokens && page[t] >= 0;  // (tokens behind the end: their block may not even have a scale)
      scale[0][t] = some ? p.c.scale[0][page[t]] : 1.f;
      scale[1][t] = some ? p.c.scale[1][page[t]] : 1.f;
    }
  };
  auto put_scales = [&]() {  // (V's counts as kLeastScale at least)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      // (V's scale is not finite: 1 for the sum of the weights, which depends on K alone.  Such scales and tiny ones have a
      // negative reciprocal, with a logarithm of 0 or a negative one)
      const bool spoiled = !(fabsf(scale[1][t]) <= 3.4028235e38f);
      const float sv = spoiled ? 1.f : fmaxf(scale[1][t], kLeastScale), lg = __log2f(sv), inv = 1.f / sv * kSumScale;
      ctl.scale[warp][lane][t] = make_float4(scale[0][t], lg, spoiled || lg < kTinyV ? -inv : inv, 0.f);
    }
    __syncwarp();
  };
  int loaded[2] = {0, 0};  // loads so far
  auto load = [&](int i, int kv) {
    ++loaded[kv];
    if (lane == 0) {
      const int2 row = ctl.row[warp][i & 31];
      mbar_expect_tx(full + kv, R::kTileBytes);
      tma_load_rows(own + kv * R::kTileBytes, &p.map[kv], full + kv, row.x);
      if (box < kTok) tma_load_rows(own + kv * R::kTileBytes + box * kD, &p.map[kv], full + kv, row.y);
    }
  };
  int own_i = 0, done = 0;  // this warp's next tile, and how many it has been through
  auto advance = [&](int i) {  // the next tile from i on that is there
    while (i < n_own) {
      if ((i & 31) == 0 && i > 0) {
        look_up(i);
        fetch_scales();
        put_scales();
      }
      if (ctl.row[warp][i & 31].x != kNoTile) break;
      ++i;
    }
    return i;
  };
  // The piece this group works on, and its end: a piece has at least one tile that is there.  Its queries (row g of each
  // column block, elements 16 s + 4c .. 4c + 3) are fetched while the one before it is added up; 16 rows of them do not
  // fit the registers then and are fetched behind that.
  auto cc = cursor_at<kOver>(p, ctl.prefix, begin);
  int piece_end = begin;
  uint2 raw[kNT][kKS];
  auto next_piece = [&](int from) {
    cc.skip(p, from - cc.at, end);
    while (cc.at < end) {
      piece_end = min(end, cc.at + cc.s.n - cc.i);
      if (cc.i + piece_end - cc.at > kOver) break;
      cc.skip(p, piece_end - cc.at, end);
    }
  };
  auto fetch_queries = [&]() {
    if (cc.at >= end) return;
    const int h = cc.item / p.row_tiles, row0 = (cc.item - h * p.row_tiles) * kRows;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      const int row = row0 + nt * 8 + g, i = row / p.group, hd = h * p.group + row - i * p.group;
      const uint16_t* src = p.q + cc.b * p.q_sb + i * p.q_st + hd * p.q_sh + c * 4;
#pragma unroll
      for (int s = 0; s < kKS; ++s) raw[nt][s] = row < p.rows ? *reinterpret_cast<const uint2*>(src + s * 16) : make_uint2(0, 0);
    }
  };
  // (Queries and scales are asked for in front of the first tiles: behind them they would wait until 20 MB have
  // arrived, 2 to 3 us.)
  next_piece(begin);
  fetch_queries();
  if (n_own > 0) {
    look_up(0);
    fetch_scales();
    while (own_i < min(n_own, 32) && ctl.row[warp][own_i].x == kNoTile) ++own_i;
    if (own_i < min(n_own, 32)) {
      load(own_i, 0);
      load(own_i, 1);
    }
    put_scales();
    if (own_i == 32) {  // (none of them is there: sequences of hardly any tokens)
      own_i = advance(own_i);
      if (own_i < n_own) {
        load(own_i, 0);
        load(own_i, 1);
      }
    }
  }
  bool dead = false;
  while (cc.at < end) {
    const int h = cc.item / p.row_tiles, row0 = (cc.item - h * p.row_tiles) * kRows;
    uint32_t qf[kNT][kKS][2];
    float rs[kNT][2];  // factor of the scores of rows 2c, 2c + 1, log2(e) in it
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
      for (int s = 0; s < kKS; ++s) qf[nt][s][0] = raw[nt][s].x, qf[nt][s][1] = raw[nt][s].y;
      float factor = row0 + nt * 8 + g < p.rows ? 1.f : 0.f;
      if (p.bf16) {
        uint32_t most = 0;
#pragma unroll
        for (int s = 0; s < kKS; ++s) most = __vmaxu2(most, __vmaxu2(qf[nt][s][0] & 0x7fff7fffu, qf[nt][s][1] & 0x7fff7fffu));
        most = max(most & 0xffffu, most >> 16);
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // largest element to [2^14, 2^15); exponents below 2^-100 are taken for it.  Not finite: the whole row NaN
        const int e = max(static_cast<int>(most >> 7), 27);
        const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 + 127 - e) << 23);
        const float mul = most >= 0x7f80u ? __uint_as_float(0x7fffffffu) : up;
#pragma unroll
        for (int s = 0; s < kKS; ++s)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t w = qf[nt][s][k];
            qf[nt][s][k] = pack2<false>(__uint_as_float(w << 16) * mul, __uint_as_float(w & 0xffff0000u) * mul);
          }
        factor *= __uint_as_float(static_cast<uint32_t>(e - 14) << 23);
      }
      factor *= p.scale_log2;
      rs[nt][0] = __shfl_sync(0xffffffffu, factor, c * 8);
      rs[nt][1] = __shfl_sync(0xffffffffu, factor, c * 8 + 4);
    }
    // what the rows of this lane's accumulators (2c, 2c + 1 of each column block) see: slots up to last, from first on
    int last[kNT][2], first[kNT][2];
    int last_min = 0x7fffffff, first_max = 0;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int row = row0 + nt * 8 + 2 * c + k;
        const int pos = cc.s.len - p.q_len + min(row, p.rows - 1) / p.group;  // (rows behind the last one are not stored)
        last[nt][k] = pos;
        first[nt][k] = p.window < 0 ? 0 : max(0, pos - p.window);
        last_min = min(last_min, pos);
        first_max = max(first_max, first[nt][k]);
      }
    last_min = __reduce_min_sync(0xffffffffu, last_min);
    first_max = __reduce_max_sync(0xffffffffu, first_max);

    float o[kNT][kKS][4], m[kNT][2], l[kNT][2];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
      for (int s = 0; s < kKS; ++s) o[nt][s][0] = o[nt][s][1] = o[nt][s][2] = o[nt][s][3] = 0.f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }
    // this warp's tiles of the piece: those whose index from `begin` is `wg` modulo kGroup
    for (int at; (at = begin + wg + own_i * kGroup) < piece_end && own_i < n_own;) {
      const float4 sc0 = ctl.scale[warp][own_i & 31][0], sc1 = ctl.scale[warp][own_i & 31][1];
      if (!dead) dead = !mbar_wait_w(full, done & 1, &ctl.err, kErrWaitProducer);
      const int slot = tile_slot(cc.s, cc.i + at - cc.at - kOver);
      const uint32_t k_base = smem_u32(own), v_base = k_base + R::kTileBytes;
      const float sk[2] = {sc0.x, sc1.x}, lv[2] = {sc0.y, sc1.y}, iv[2] = {sc0.z, sc1.z};
      // ---- scores
      float acc[2][kNT][4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) acc[t][nt][0] = acc[t][nt][1] = acc[t][nt][2] = acc[t][nt][3] = 0.f;
#pragma unroll
      for (int s = 0; s < kKS; ++s) {
        uint32_t w[4], lo[4], hi[4];
        ldsm4(w, piece<kD>(k_base, lane, s));
#pragma unroll
        for (int k = 0; k < 4; ++k) to_half2<kInt8, true>(w[k], lo[k], hi[k]);
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          mma16816(acc[0][nt], lo[0], lo[1], hi[0], hi[1], qf[nt][s][0], qf[nt][s][1]);
          mma16816(acc[1][nt], lo[2], lo[3], hi[2], hi[3], qf[nt][s][0], qf[nt][s][1]);
        }
      }
      // every lane has read K: the next tile's
      const int next_i = advance(own_i + 1);
      __syncwarp();
      if (next_i < n_own && !dead) load(next_i, 0);
      // ---- to base 2, hidden ones to -inf
      const bool plain = slot + kTok - 1 <= last_min && (slot >= first_max || slot + kTok <= p.n_sink);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[t][nt][k] *= rs[nt][k & 1] * sk[t];
      if (!plain) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int tok = slot + 16 * t + g + 8 * (k >> 1);
              if (!(tok <= last[nt][k & 1] && (tok >= first[nt][k & 1] || tok < p.n_sink))) acc[t][nt][k] = -INFINITY;
            }
      }
      if (p.scores != nullptr) {
        float* const to = p.scores + static_cast<long long>(at) * (kTok * kRows);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt) {
            *reinterpret_cast<float2*>(to + (16 * t + g) * kRows + nt * 8 + 2 * c) = make_float2(acc[t][nt][0], acc[t][nt][1]);
            *reinterpret_cast<float2*>(to + (16 * t + g + 8) * kRows + nt * 8 + 2 * c) = make_float2(acc[t][nt][2], acc[t][nt][3]);
          }
      }
      // ---- running reference
      float top[kNT][2];
      bool raise = false;
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = k; e < 4; e += 2)  // (a hidden token stays hidden whatever its block's scale is)
              acc[t][nt][e] = !plain && acc[t][nt][e] == -INFINITY ? -INFINITY : acc[t][nt][e] + lv[t];
          top[nt][k] = fmaxf(fmaxf(acc[0][nt][k], acc[0][nt][k + 2]), fmaxf(acc[1][nt][k], acc[1][nt][k + 2]));
          raise = raise || top[nt][k] > m[nt][k] + kRoom;
        }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float x = top[nt][k];
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            const float old = m[nt][k];
            const float next = x - kLow > old ? x - kLow : old;
            const float h = next > old ? ex2f(0.5f * (old - next)) : 1.f, f = h * h;
            m[nt][k] = next;
            l[nt][k] = l[nt][k] * h * h;  // (not times h * h, see join_pieces)
#pragma unroll
            for (int s = 0; s < kKS; ++s) o[nt][s][k] *= f, o[nt][s][k + 2] *= f;
          }
      }
      // ---- weights, as the right operand of V^T P^T
      uint32_t pf[2][kNT][2];
      const auto weigh = [&](auto usual) {
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          const float m0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], m1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const float(&x)[4] = acc[t][nt];
            float a = ex2f(x[0] - m0), b = ex2f(x[1] - m1), d = ex2f(x[2] - m0), e = ex2f(x[3] - m1);
            if (decltype(usual)::value || iv[t] > 0.f || lv[t] == 0.f) {
              l[nt][0] += (a + d) * fabsf(iv[t]);
              l[nt][1] += (b + e) * fabsf(iv[t]);
            } else {
              const float u = lv[t] + kSumUnit;
              l[nt][0] += ex2f(x[0] - m0 - u) + ex2f(x[2] - m0 - u);
              l[nt][1] += ex2f(x[1] - m1 - u) + ex2f(x[3] - m1 - u);
            }
            if (!decltype(usual)::value && iv[t] < 0.f && lv[t] == 0.f) {  // NaN for the rows that see it, whatever the weight
              const float nan = __uint_as_float(0x7fffffffu);
              a = x[0] == -INFINITY ? 0.f : nan, b = x[1] == -INFINITY ? 0.f : nan;
              d = x[2] == -INFINITY ? 0.f : nan, e = x[3] == -INFINITY ? 0.f : nan;
            }
            pf[t][nt][0] = transpose8(pack2<false>(a, b));
            pf[t][nt][1] = transpose8(pack2<false>(d, e));
          }
        }
      };
      if (fminf(iv[0], iv[1]) > 0.f) weigh(std::true_type()); else weigh(std::false_type());
      // ---- output
      if (!dead) dead = !mbar_wait_w(full + 1, done & 1, &ctl.err, kErrWaitProducer);
      if (!kInt8 && slot + kTok > cc.s.len) {
        // the slots behind the last token hold anything: a weight of 0 does not take a NaN away
        if (slot + lane >= cc.s.len)
          for (int k = 0; k < kD / 16; ++k) *reinterpret_cast<uint4*>(own + R::kTileBytes + lane * kD + k * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();  // (the next load of V comes behind these stores)
        __syncwarp();
      }
#pragma unroll
      for (int s = 0; s < kKS; ++s) {
        uint32_t w[4], lo[4], hi[4];
        ldsm4_t(w, piece<kD>(v_base, lane, s));
#pragma unroll
        for (int k = 0; k < 4; ++k) to_half2<kInt8, false>(w[k], lo[k], hi[k]);
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          mma16816(o[nt][s], lo[0], hi[0], lo[1], hi[1], pf[0][nt][0], pf[0][nt][1]);
          mma16816(o[nt][s], lo[2], hi[2], lo[3], hi[3], pf[1][nt][0], pf[1][nt][1]);
        }
      }
      __syncwarp();  // every lane has read V
      if (next_i < n_own && !dead) load(next_i, 1);
      own_i = next_i;
      ++done;
    }

    // ---- the warps' sums of this piece
    // (the first piece is the one with the item's first tile)
    const int item0 = cc.at - cc.i, lo = shares.of(item0 + kOver), pieces = shares.of(item0 + cc.s.n - 1) - lo + 1;
    const bool whole = pieces == 1;
    const int b = cc.b;
    next_piece(piece_end);
    if (kNT == 1) fetch_queries();
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float x = l[nt][k];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (g == 0) {
          ml[wg][nt * 8 + 2 * c + k][0] = m[nt][k];
          ml[wg][nt * 8 + 2 * c + k][1] = x;
        }
      }
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      // (float d of row r lies at d ^ 8 * (r / 2): no bank twice in a half-warp's stores)
      float* const mine = merge + wg * 8 * kD;
#pragma unroll
      for (int s = 0; s < kKS; ++s) {
        *reinterpret_cast<float2*>(mine + (2 * c) * kD + ((s * 16 + 2 * g) ^ (8 * c))) = make_float2(o[nt][s][0], o[nt][s][2]);
        *reinterpret_cast<float2*>(mine + (2 * c + 1) * kD + ((s * 16 + 2 * g) ^ (8 * c))) = make_float2(o[nt][s][1], o[nt][s][3]);
      }
      sync_group<kPeers>(group);
      const int t = threadIdx.x - group * kPeers, d4 = t % (kD / 4);
#pragma unroll
      for (int r = t / (kD / 4); r < 8; r += kPeers / (kD / 4)) {
        const int row = row0 + nt * 8 + r;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kGroup; ++w) top = fmaxf(top, ml[w][nt * 8 + r][0]);
        float sum = 0.f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kGroup; ++w) {
          const float lw = ml[w][nt * 8 + r][1];
          const float fh = lw == 0.f ? 0.f : ex2f(0.5f * (ml[w][nt * 8 + r][0] - top)), f = fh * fh;  // (0: no visible token)
          const float4 y = *reinterpret_cast<const float4*>(merge + (w * 8 + r) * kD + ((d4 * 4) ^ (r / 2 * 8)));
          sum += lw * fh * fh;
          x.x += y.x * f, x.y += y.y * f, x.z += y.z * f, x.w += y.w * f;
        }
        if (row < p.rows) {
          if (whole) {
            store_row<kD>(p, b, h, row, d4, x, top, sum);
          } else {
            const long long to = (static_cast<long long>(me) * 2 + (me == lo ? 1 : 0)) * kRows + nt * 8 + r;
            *reinterpret_cast<float4*>(p.part_o + to * kD + d4 * 4) = x;
            if (d4 == 0) *reinterpret_cast<float2*>(p.part_ml + to * 2) = make_float2(top, sum);
          }
        }
      }
      sync_group<kPeers>(group);
    }
    if (!whole) {
      // the group that delivers an item's last piece joins them all
      if (threadIdx.x == group * kPeers) {
        __threadfence();
        const int last = atomicAdd(p.arrived + lo, 1) == pieces - 1;
        if (last) {
          p.arrived[lo] = 0;
          __threadfence();
        }
        ctl.last[group] = last;
      }
      sync_group<kPeers>(group);
      if (ctl.last[group] != 0) join_pieces<kD, kNT, kPeers>(p, merge, group, b, h, row0, lo, pieces);
    }
    if (kNT > 1) fetch_queries();
  }
  if (dead) {
    // copies still on their way must not outlive the CTA's shared memory (each wait is limited)
    int own_err = 0;
    for (int kv = 0; kv < 2; ++kv)
      if (loaded[kv] > 0) mbar_wait(full + kv, (loaded[kv] - 1) & 1, &own_err, kErrWaitProducer);
    if (lane == 0) raise_status(p.status, p.mirror, kErrWaitProducer);
  }
  if (group == 0) empty_rows<kD, kPeers>(p);
}

// Adds every visible slot's softmax weights up, from the scores that the first kernel kept and the final log-sum-exp.
// One CTA per (sequence, head) and kWeightTiles tiles.
constexpr int kWeightTiles = 16;
template <int kNT, int kOver>
__global__ void __launch_bounds__(kAdd) cache_weights_kernel(const __grid_constant__ AttnKernelParams p, int chunks) {
  constexpr int kRows = 8 * kNT;
  extern __shared__ float s_lse[];  // [row_tiles * kRows], base 2; +inf for rows that see nothing and rows behind the last
  griddep_wait();
  const int bh = blockIdx.x / chunks, b = bh / p.c.hkv, h = bh - b * p.c.hkv;
  const SeqTiles s = seq_tiles<kOver>(p, b);
  const int t0 = (blockIdx.x - bh * chunks) * kWeightTiles;
  const int n = s.n - kOver;  // tiles
  if (t0 >= n) return;
  // (what the loads below depend on is one step behind them: lengths and the sequence's first tile, then everything else)
  const int first = p.first[b] + h * p.row_tiles * s.n;
  const int t1 = min(t0 + kWeightTiles, n);
  constexpr int kEach = kWeightTiles * kTok / kAdd;
  float4 x[kEach][kRows / 4];
  float old[kEach];
  float* to[kEach];
  const auto load = [&](int rt) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int k = t0 * kTok + e * kAdd + threadIdx.x, tile = k / kTok;
      const float4* from = reinterpret_cast<const float4*>(p.scores + (static_cast<long long>(first + rt * s.n + kOver + tile) * kTok + k % kTok) * kRows);
#pragma unroll
      for (int v = 0; v < kRows / 4; ++v) x[e][v] = to[e] != nullptr ? from[v] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    }
  };
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int k = t0 * kTok + e * kAdd + threadIdx.x, tile = k / kTok, tok = tile_slot(s, tile) + k % kTok;
    to[e] = tile < t1 && tok < s.len ? p.weights + b * p.w_sb + h * p.w_sh + tok : nullptr;
    old[e] = to[e] != nullptr ? *to[e] : 0.f;
  }
  load(0);
  for (int r = threadIdx.x; r < p.row_tiles * kRows; r += kAdd) {
    float l = INFINITY;
    if (r < p.rows) {
      const int i = r / p.group;
      l = p.lse[(static_cast<long long>(b) * p.hq + h * p.group + r - i * p.group) * p.q_len + i] * 1.4426950408889634f;
      if (l == -INFINITY) l = INFINITY;
    }
    s_lse[r] = l;
  }
  __syncthreads();
  float sum[kEach] = {};
  for (int rt = 0; rt < p.row_tiles; ++rt) {
    if (rt > 0) load(rt);
#pragma unroll
    for (int e = 0; e < kEach; ++e)
#pragma unroll
      for (int v = 0; v < kRows / 4; ++v) {
        const float* lse = s_lse + rt * kRows + v * 4;
        // (a hidden slot's score is -inf: nothing from that row, not even where the row's log-sum-exp is NaN)
        const auto part = [](float s, float l) { return s == -INFINITY ? 0.f : ex2f(s - l); };
        sum[e] += part(x[e][v].x, lse[0]) + part(x[e][v].y, lse[1]) + part(x[e][v].z, lse[2]) + part(x[e][v].w, lse[3]);
      }
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e)
    if (to[e] != nullptr) *to[e] = old[e] + sum[e];
}

struct Plan {
  int nt, row_tiles, groups, ctas;
  bool all;  // all warps of a CTA are one group
  long long most_tiles;  // of a sequence, per head and row tile, and as they are counted
  int over;
  int64_t o_bytes, ml_bytes, first_bytes, score_bytes;
  int64_t total() const { return o_bytes + ml_bytes + first_bytes + score_bytes; }
};

// kNT = 1 up to 8 query rows per key/value head, else row tiles of 16.
int make_plan(const rswa_cache_attn_params_t& a, Plan& plan) {
  const long long rows = static_cast<long long>(a.q_len) * (a.n_q_heads / a.cache.n_kv_heads);
  plan.nt = rows <= 8 ? 1 : 2;
  const long long per_tile = 8 * plan.nt;
  const long long row_tiles = (rows + per_tile - 1) / per_tile;
  const long long cap = static_cast<long long>(a.table.max_blocks) * a.cache.block_size;
  long long most = (cap + kTok - 1) / kTok;
  if (a.window >= 0) {
    const long long seen = (static_cast<long long>(a.window) + a.q_len + kTok - 1) / kTok + 1 + (static_cast<long long>(a.n_sink) + kTok - 1) / kTok;
    most = most < seen ? most : seen;
  }
  plan.most_tiles = most;
  const long long items = static_cast<long long>(a.table.batch) * a.cache.n_kv_heads * row_tiles;
  // (a row tile's log-sum-exps lie in shared memory while the weights are added up)
  if (row_tiles > 512 || items > 0x7fffffffLL) {
    set_error("rswa_cache_attn: too many queries in one call");
    return RSWA_E_UNSUPPORTED;
  }
  plan.row_tiles = static_cast<int>(row_tiles);
  const int sms = sm_count(), warps = plan.nt == 1 ? Layout<128, 1, true>::kWarps : Layout<128, 2, true>::kWarps;
  plan.all = items <= sms;
  plan.over = plan.all ? warps : 4;
  most += plan.over;
  if (items * most > 0x7fffffffLL) {
    set_error("rswa_cache_attn: too many tokens in one call");
    return RSWA_E_UNSUPPORTED;
  }
  const long long by_tiles = items * plan.most_tiles / plan.over, shares = by_tiles > items ? by_tiles : items, most_groups = plan.all ? sms : static_cast<long long>(sms) * warps / 4;
  plan.groups = static_cast<int>(shares < 1 ? 1 : shares < most_groups ? shares : most_groups);
  if (plan.groups > RSWA_CACHE_ATTN_COUNTERS) plan.groups = RSWA_CACHE_ATTN_COUNTERS;
  plan.ctas = plan.groups < sms ? plan.groups : sms;
  plan.o_bytes = 2LL * plan.groups * per_tile * a.cache.head_dim * 4;
  plan.ml_bytes = (2LL * plan.groups * per_tile * 2 * 4 + 255) / 256 * 256;
  plan.first_bytes = a.weights != nullptr ? (a.table.batch * 4LL + 255) / 256 * 256 : 0;
  plan.score_bytes = a.weights != nullptr ? items * most * kTok * per_tile * 4 : 0;
  return RSWA_OK;
}

int check_attn(const rswa_cache_attn_params_t* p) {
  const char* what = "rswa_cache_attn";
  if (p == nullptr) {
    set_error("%s: null params", what);
    return RSWA_E_ARG;
  }
  const rswa_cache_t& c = p->cache;
  if ((c.head_dim != 64 && c.head_dim != 128) || (c.block_size != 16 && c.block_size != 32 && c.block_size != 64 && c.block_size != 128)) {
    set_error("%s: head_dim must be 64 or 128 (got %d), block_size 16, 32, 64 or 128 (got %d)", what, c.head_dim, c.block_size);
    return RSWA_E_UNSUPPORTED;
  }
  if (c.n_kv_heads <= 0 || c.n_kv_heads > 32767 || p->n_q_heads <= 0 || p->q_len < 0 || p->n_sink < 0 || p->table.batch < 0 || p->table.max_blocks < 0) {
    set_error("%s: batch, lengths, sink tokens and head counts must not be negative", what);
    return RSWA_E_ARG;
  }
  if (p->n_q_heads % c.n_kv_heads != 0) {
    set_error("%s: Number of query heads must be divisible by number of key/value heads", what);
    return RSWA_E_ARG;
  }
  return RSWA_OK;
}

template <int kD, int kNT, bool kInt8, bool kAll>
cudaError_t launch_tiles(const AttnKernelParams& kp, const Plan& plan, cudaStream_t s) {
  using L = Layout<kD, kNT, kAll>;
  const auto kern = cache_attn_kernel<kD, kNT, kInt8, kAll>;
  static std::atomic<uint64_t> set{0};  // devices on which the kernel's shared memory has been allowed
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !(set.load(std::memory_order_relaxed) >> dev & 1)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
    if (e != cudaSuccess) return e;
    if (dev < 64) set.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  return launch_kernel(kern, dim3(plan.ctas), L::kThreads, L::kBytes, s, true, kp);
}

template <int kD, int kNT, bool kInt8>
cudaError_t launch_attn(const AttnKernelParams& kp, const Plan& plan, cudaStream_t s) {
  cudaError_t e = plan.all ? launch_tiles<kD, kNT, kInt8, true>(kp, plan, s) : launch_tiles<kD, kNT, kInt8, false>(kp, plan, s);
  if (e != cudaSuccess) return e;
  count_launches(1);
  if (kp.weights != nullptr && plan.most_tiles > 0) {
    const long long chunks = (plan.most_tiles + kWeightTiles - 1) / kWeightTiles;
    const dim3 grid(static_cast<unsigned>(static_cast<long long>(kp.batch) * kp.c.hkv * chunks));
    e = launch_kernel(plan.all ? cache_weights_kernel<kNT, Layout<kD, kNT, true>::kGroup> : cache_weights_kernel<kNT, Layout<kD, kNT, false>::kGroup>, grid, kAdd,
                      plan.row_tiles * 8 * kNT * 4, s, true, kp, static_cast<int>(chunks));
    if (e != cudaSuccess) return e;
    count_launches(1);
  }
  return cudaSuccess;
}

}  // namespace

}  // namespace rswa

using namespace rswa;

extern "C" int64_t rswa_cache_attn_workspace_bytes(const rswa_cache_attn_params_t* p) {
  int rc = check_attn(p);
  if (rc != RSWA_OK) return rc;
  Plan plan;
  rc = make_plan(*p, plan);
  return rc != RSWA_OK ? rc : plan.total();
}

extern "C" int rswa_cache_attn(const rswa_cache_attn_params_t* p, void* stream) {
  const char* what = "rswa_cache_attn";
  int rc = check_attn(p);
  if (rc == RSWA_OK) rc = check_cache(p->cache, what);
  if (rc == RSWA_OK) rc = check_table(p->table, false, p->lens, p->status, p->cache.block_size, what);
  if (rc != RSWA_OK) return rc;
  if (p->dtype != RSWA_DTYPE_BF16 && p->dtype != RSWA_DTYPE_FP16) {
    set_error("%s: dtype must be bf16 (0) or fp16 (1), got %d", what, p->dtype);
    return RSWA_E_UNSUPPORTED;
  }
  if (!(p->softmax_scale > 0.f)) {
    set_error("%s: softmax_scale must be positive", what);
    return RSWA_E_ARG;
  }
  if (p->table.batch == 0 || p->q_len == 0) return RSWA_OK;
  const auto off = [](const void* x, uintptr_t n) { return x == nullptr || reinterpret_cast<uintptr_t>(x) % n != 0; };
  if (off(p->q, 16) || off(p->out, 16) || p->q_stride_b % 8 || p->q_stride_t % 8 || p->q_stride_h % 8) {
    set_error("%s: q and out must be 16-byte aligned, q with strides that are multiples of 8 elements", what);
    return RSWA_E_ARG;
  }
  if (p->arrived == nullptr) {
    set_error("%s: arrived is required", what);
    return RSWA_E_ARG;
  }
  if (p->weights != nullptr && p->lse == nullptr) {
    set_error("%s: weights need lse", what);
    return RSWA_E_ARG;
  }
  Plan plan;
  rc = make_plan(*p, plan);
  if (rc != RSWA_OK) return rc;
  if (p->workspace_bytes < plan.total() || off(p->workspace, 256)) {
    set_error("%s: the workspace must be 256-byte aligned and hold %lld bytes", what, static_cast<long long>(plan.total()));
    return RSWA_E_ARG;
  }
  const rswa_cache_t& c = p->cache;
  if (c.num_blocks * c.n_kv_heads * c.block_size > 0x7fffffffLL) {
    set_error("%s: a cache of more than 2^31 rows (blocks x heads x tokens)", what);
    return RSWA_E_UNSUPPORTED;
  }
  AttnKernelParams kp;
  const long long rows = c.num_blocks * c.n_kv_heads * c.block_size;
  const int box = c.block_size < kTok ? c.block_size : kTok;
  rc = make_rows_map(&kp.map[0], c.k, rows, c.head_dim, box);
  if (rc == RSWA_OK) rc = make_rows_map(&kp.map[1], c.v, rows, c.head_dim, box);
  if (rc != RSWA_OK) return rc;
  kp.c = cache_view(c);
  kp.table = p->table.entries, kp.table_stride = p->table.stride;
  kp.batch = p->table.batch, kp.max_blocks = p->table.max_blocks;
  kp.lens = p->lens;
  kp.q = static_cast<const uint16_t*>(p->q);
  kp.q_sb = p->q_stride_b, kp.q_st = p->q_stride_t, kp.q_sh = p->q_stride_h;
  kp.q_len = p->q_len, kp.hq = p->n_q_heads, kp.group = p->n_q_heads / c.n_kv_heads;
  kp.rows = kp.q_len * kp.group, kp.row_tiles = plan.row_tiles;
  kp.window = p->window < 0 ? -1 : p->window, kp.n_sink = p->n_sink;
  kp.scale_log2 = p->softmax_scale * 1.4426950408889634f;
  kp.bf16 = p->dtype == RSWA_DTYPE_BF16;
  kp.out = static_cast<uint16_t*>(p->out);
  kp.lse = p->lse;
  uint8_t* ws = static_cast<uint8_t*>(p->workspace);
  kp.part_o = reinterpret_cast<float*>(ws);
  kp.part_ml = reinterpret_cast<float*>(ws += plan.o_bytes);
  ws += plan.ml_bytes;
  kp.first = p->weights != nullptr ? reinterpret_cast<int*>(ws) : nullptr;
  kp.scores = p->weights != nullptr ? reinterpret_cast<float*>(ws + plan.first_bytes) : nullptr;
  kp.weights = p->weights;
  kp.w_sb = p->w_stride_b, kp.w_sh = p->w_stride_h;
  kp.groups = plan.groups;
  kp.arrived = p->arrived;
  kp.status = p->status;
  kp.mirror = status_mirror(p->status);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool int8 = c.kind == RSWA_CACHE_INT8;
  cudaError_t e;
  if (c.head_dim == 64)
    e = plan.nt == 1 ? (int8 ? launch_attn<64, 1, true>(kp, plan, s) : launch_attn<64, 1, false>(kp, plan, s))
                     : (int8 ? launch_attn<64, 2, true>(kp, plan, s) : launch_attn<64, 2, false>(kp, plan, s));
  else
    e = plan.nt == 1 ? (int8 ? launch_attn<128, 1, true>(kp, plan, s) : launch_attn<128, 1, false>(kp, plan, s))
                     : (int8 ? launch_attn<128, 2, true>(kp, plan, s) : launch_attn<128, 2, false>(kp, plan, s));
  if (e != cudaSuccess) {
    set_error("%s: launch failed: %s", what, cudaGetErrorString(e));
    return RSWA_E_CUDA;
  }
  return RSWA_OK;
}
