// Choice of the key blocks that each query block attends to (the lists of
// sparse_attn.cu), from INT8 Q/K and their scales.
//
//   qm_i = sum over the 128 queries of block i of q_scale * Q8     (fp64)
//   S_j  = sum over the n_j visible keys of block j (64 keys) of K8 (exact)
//   score(i, j) = (qm_i . S_j) * k_scale_j / n_j
// which ranks as the mean score of the pair's query-key grid does (sm_scale and
// the query count change no rank), and the `keep` blocks of the highest score
// in ascending order, ties to the lowest block.  block_policy takes a block out
// (-1) or ranks it above every score (1); a NaN score ranks lowest.
//
// Which of two near blocks is kept is decided by the last digits, so the dot
// product is integer: qm_i is rounded to 40 bits below the power of two above
// its largest channel and written as six digits of base 128 in [-64, 63], S_j
// (14 bits) as two, and the tensor core multiplies the digit planes exactly
// (kind::i8, INT32 sums below 2^20).  The planes join in 64-bit integers, and
// the product with k_scale_j / n_j is the first fp64 rounding.  The sum order
// never matters, equal blocks score equal.
//
//   1. block_sums_kernel: 16-byte loads, channel sums as packed 16-bit lanes of
//      the biased bytes; a warp per key block, a CTA per query block (a warp
//      per 16-token scale tile).  HBM-bound: the only pass over Q and K.
//   2. block_select_kernel: a CTA takes up to 8 query blocks of one key head
//      (its query heads' blocks in a row) and all key blocks, 128 at a time:
//      M = 128 key blocks, N = 8 query blocks x 6 digits, K = channels, twice
//      for the two digits of S.  Warp 8 loads digit planes by TMA into a
//      4-stage ring, warp 9 issues the MMAs into two TMEM buffers, warps 0-3
//      and 4-7 take the tiles in turn and leave the top word of each score's
//      sortable bits in shared memory.  Then one warp per query block finds the
//      keep-th word by bracketing it, and, where that word is shared by more blocks
//      than fit, again with their low words from the digits.  Two CTAs per SM
//      (up to 1300 key blocks): one's search runs under the other's products.
#include <algorithm>

#define TB_TRY_WAIT_NO_HINT 1
#include "attn_common.cuh"
#include "tb_capi_internal.h"
#include "tb_tu.cuh"

namespace tb {
namespace {

constexpr int kQueryBlock = 128;
constexpr int kKeyBlock = 64;
constexpr int kTileRows = 16;            // tokens of one q_scale
constexpr int kSumThreads = 256;
constexpr int kSumWarps = kSumThreads / 32;
static_assert(kSumWarps * kTileRows == kQueryBlock, "one warp per scale tile");
constexpr int kChannels = 128;           // of a digit plane's row (64-channel heads: half zero)
constexpr int kQDigits = 6;
constexpr int kKDigits = 2;
constexpr int kFixBits = 40;

constexpr int kMaxRows = 8;              // query blocks per CTA
constexpr int kTileKeys = 128;           // key blocks per MMA
constexpr int kMmaN = kMaxRows * kQDigits;
constexpr int kStages = 4;
constexpr int kStageBytes = kTileKeys * kChannels;   // one digit plane of a tile
constexpr int kQTileBytes = kMmaN * kChannels;
constexpr int kEpilogueWarps = 8;
constexpr int kLoadWarp = 8;
constexpr int kMmaWarp = 9;
constexpr int kSelectThreads = 320;
constexpr uint32_t kBufCols = kKDigits * kMmaN;      // TMEM columns of one buffer
constexpr uint32_t kTmemCols = 256;
static_assert(2 * kBufCols <= kTmemCols, "two TMEM buffers");
constexpr int kMaxKeyBlocks = 24576;

struct SelectParams {
  const int8_t* q;
  const int8_t* k;
  const float* q_scale;
  const float* k_scale;
  const int32_t* key_lengths;  // [B] or null
  const int8_t* policy;        // [policy_rows, key_blocks] or null
  int64_t q_s[3], k_s[3];      // batch, head, token strides
  int B, Hq, Hk, Lq, Lk;
  int query_blocks, key_blocks, keep, policy_rows;
  int q_tiles_scale;
  int rows_cta;                // query blocks per CTA, <= kMaxRows
  int groups;                  // CTAs per key head
  int8_t* q_digits;            // [B * Hq * query_blocks, kQDigits, kChannels]
  int8_t* k_digits;            // [kKDigits, B * Hk, key_blocks, kChannels]
  int32_t* out;                // [B * Hq * query_blocks, keep]
};

struct __align__(8) SelectBarriers {
  uint64_t q_full;
  uint64_t full[kStages];
  uint64_t empty[kStages];
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort_flag;
};
constexpr int kFixedSmem = kQTileBytes + kStages * kStageBytes + sizeof(SelectBarriers);
static_assert(kFixedSmem % 8 == 0 && kQTileBytes % 1024 == 0, "tile alignment");

__device__ __forceinline__ int visible_keys(const SelectParams& p, int b) {
  return p.key_lengths != nullptr ? max(0, min(__ldg(p.key_lengths + b), p.Lk)) : p.Lk;
}

// Sums of the channels of 16 bytes, kept as biased (byte + 128) 16-bit lanes:
// word w holds channels 4w and 4w + 2 in `even`, 4w + 1 and 4w + 3 in `odd`.
struct ByteSums {
  uint32_t even[4] = {0u, 0u, 0u, 0u}, odd[4] = {0u, 0u, 0u, 0u};
  __device__ __forceinline__ void add(const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = w[i] ^ 0x80808080u;
      even[i] += u & 0x00ff00ffu;
      odd[i] += (u >> 8) & 0x00ff00ffu;
    }
  }
  // Over the lanes that hold the same channels of other rows.
  template <int LANES_PER_ROW>
  __device__ __forceinline__ void reduce() {
#pragma unroll
    for (int m = LANES_PER_ROW; m < 32; m <<= 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        even[i] += __shfl_xor_sync(0xffffffffu, even[i], m);
        odd[i] += __shfl_xor_sync(0xffffffffu, odd[i], m);
      }
    }
  }
  // Channel c (0..15) without the bias of n rows.
  __device__ __forceinline__ int channel(int c, int n) const {
    const uint32_t pair = c & 1 ? odd[c >> 2] : even[c >> 2];
    return static_cast<int>(c & 2 ? pair >> 16 : pair & 0xffffu) - 128 * n;
  }
};

// Adds rows [0, n) of a ROWS-row tile, all of its loads in flight.
template <int D, int ROWS>
__device__ __forceinline__ void sum_rows(ByteSums& sums, const int8_t* src, int64_t stride, int sub,
                                         int n) {
  constexpr int kStep = 32 / (D / 16);
  src += sub * stride;
  uint4 v[ROWS / kStep];
#pragma unroll
  for (int i = 0; i < ROWS / kStep; ++i) {
    // Bytes 0x80 are -128, a biased zero: rows past the end add nothing.
    v[i] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
    if (i * kStep + sub < n) v[i] = *reinterpret_cast<const uint4*>(src + i * kStep * stride);
  }
#pragma unroll
  for (int i = 0; i < ROWS / kStep; ++i) sums.add(v[i]);
  sums.reduce<D / 16>();
}

// Block and (batch, head) of a task, in the order that memory is laid out:
// where a token's heads lie side by side, the heads of a block come one after
// another.
__device__ __forceinline__ void block_of(int64_t task, int B, int H, int blocks,
                                         const int64_t (&stride)[3], int& block, int& bh) {
  if (stride[1] < stride[2]) {
    const int64_t rest = task / H;
    block = static_cast<int>(rest % blocks);
    bh = static_cast<int>(rest / blocks) * H + static_cast<int>(task % H);
  } else {
    block = static_cast<int>(task % blocks);
    bh = static_cast<int>(task / blocks);
  }
}

__device__ __forceinline__ int low_digit(int64_t v) {
  return static_cast<int>((v + 64) & 127) - 64;
}

template <int D>
__global__ void __launch_bounds__(kSumThreads, 3) block_sums_kernel(const SelectParams p) {
  constexpr int kLanesPerRow = D / 16;
  __shared__ double part[kSumWarps][kChannels];
  __shared__ int top;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = (lane % kLanesPerRow) * 16;
  const int sub = lane / kLanesPerRow;
  const int64_t key_tasks = static_cast<int64_t>(p.B) * p.Hk * p.key_blocks;
  const int64_t key_ctas = (key_tasks + kSumWarps - 1) / kSumWarps;
  ByteSums sums;
  if (blockIdx.x < key_ctas) {
    const int64_t task = static_cast<int64_t>(blockIdx.x) * kSumWarps + warp;
    if (task >= key_tasks) return;
    int j, bh;
    block_of(task, p.B, p.Hk, p.key_blocks, p.k_s, j, bh);
    const int b = bh / p.Hk;
    const int n = min(kKeyBlock, visible_keys(p, b) - j * kKeyBlock);
    if (n <= 0) return;  // never scored
    sum_rows<D, kKeyBlock>(sums, p.k + b * p.k_s[0] + (bh % p.Hk) * p.k_s[1] +
                                     static_cast<int64_t>(j) * kKeyBlock * p.k_s[2] + col,
                           p.k_s[2], sub, n);
    if (sub < kKDigits) {  // lane group d writes digit plane d
      uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const int s = sums.channel(c, n);
        const int lo = low_digit(s);
        const int digit = sub == 0 ? lo : (s - lo) >> 7;
        w[c >> 2] |= static_cast<uint32_t>(digit & 255) << (8 * (c & 3));
      }
      const int64_t at = static_cast<int64_t>(bh) * p.key_blocks + j;
      int8_t* dst = p.k_digits + (sub * key_tasks + at) * kChannels + col;
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
      if (D < kChannels) *reinterpret_cast<uint4*>(dst + D) = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  int i, bh;
  block_of(blockIdx.x - key_ctas, p.B, p.Hq, p.query_blocks, p.q_s, i, bh);
  const int64_t at = static_cast<int64_t>(bh) * p.query_blocks + i;
  const int row0 = i * kQueryBlock + warp * kTileRows;
  const int n = max(0, min(kTileRows, p.Lq - row0));
  if (threadIdx.x == 0) top = 0;
  sum_rows<D, kTileRows>(sums, p.q + (bh / p.Hq) * p.q_s[0] + (bh % p.Hq) * p.q_s[1] +
                                   row0 * p.q_s[2] + col,
                         p.q_s[2], sub, n);
  const double scale =
      n > 0 ? static_cast<double>(__ldg(p.q_scale + static_cast<int64_t>(bh) * p.q_tiles_scale +
                                        row0 / kTileRows))
            : 0.0;
  if (sub < 4) {  // lane group s keeps the four channels of word s
    uint32_t e = sums.even[0], o = sums.odd[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      e = sub == w ? sums.even[w] : e;
      o = sub == w ? sums.odd[w] : o;
    }
    // Exact: a 16-bit sum in the low mantissa bits of 2^52.
    const double bias = 4503599627370496.0 + 128.0 * n;
    auto scaled = [&](uint32_t v) {
      return scale * (__hiloint2double(0x43300000, static_cast<int>(v)) - bias);
    };
    double2* dst = reinterpret_cast<double2*>(&part[warp][col + sub * 4]);
    dst[0] = make_double2(scaled(e & 0xffffu), scaled(o & 0xffffu));
    dst[1] = make_double2(scaled(e >> 16), scaled(o >> 16));
  }
  __syncthreads();
  const int c = threadIdx.x;
  double m = 0.0;
  if (c < kChannels) {
    if (c < D) {
#pragma unroll
      for (int w = 0; w < kSumWarps; ++w) m += part[w][c];
    }
    // Exponent field of the largest channel (NaN and infinity: 0x7ff).
    const int e = (__double2hiint(m) >> 20) & 0x7ff;
    const int we = __reduce_max_sync(0xffffffffu, static_cast<unsigned>(e));
    if (lane == 0) atomicMax(&top, we);
  }
  __syncthreads();
  if (c < kChannels) {
    // |m| < 2^(top - 1022).  A block whose mean is not finite scores 0 everywhere.
    int64_t v = top == 0x7ff ? 0 : llrint(ldexp(m, kFixBits - (top - 1022)));
    int8_t* dst = p.q_digits + at * (kQDigits * kChannels) + c;
#pragma unroll
    for (int d = 0; d < kQDigits; ++d) {
      const int digit = low_digit(v);
      dst[d * kChannels] = static_cast<int8_t>(digit);
      v = (v - digit) >> 7;
    }
  }
}

// Orders fp64 scores as unsigned integers, -0 as 0 and NaN as -infinity; below
// every score lies 0 (a block that cannot be chosen), above it ~0.
__device__ __forceinline__ uint64_t sort_key(double score) {
  if (isnan(score)) score = -INFINITY;
  const int64_t bits = __double_as_longlong(score + 0.0);
  return bits < 0 ? ~static_cast<uint64_t>(bits)
                  : static_cast<uint64_t>(bits) | 0x8000000000000000ull;
}

__device__ __forceinline__ double block_factor(const SelectParams& p, int64_t kv, int j, int n) {
  return static_cast<double>(__ldg(p.k_scale + kv * p.key_blocks + j)) / n;
}

struct Edge {
  uint32_t word;  // the keep-th highest key
  int left;       // keys equal to it that are kept, lowest first
  bool shared;    // more keys equal it than are kept
};

// Score whose sort key starts with `word`.
__device__ __forceinline__ double key_score(uint32_t word) {
  return __hiloint2double(
      static_cast<int>(word & 0x80000000u ? word ^ 0x80000000u : ~word), 0);
}

// The keep-th highest of n keys, the warp together; with no more than `keep`
// keys above 0 all of those are kept.  Brackets the edge between two keys whose
// counts enclose `keep` and shrinks the bracket: by interpolating the counts
// over the scores, by the middle score, and by the middle key, which alone
// would end after 32 steps (scores of one row: 8 steps instead of 22).  The
// first PER_LANE * 32 keys stay in registers; longer rows read shared memory.
template <int PER_LANE>
__device__ __forceinline__ Edge find_edge(const uint32_t* row, int n, int keep) {
  const int lane = static_cast<int>(lane_id());
  uint32_t own[PER_LANE];
  const int rest = PER_LANE * 32 + lane;
  uint32_t low = ~0u, top = 0u;  // of the keys that scores gave
  int total = 0, ranked = 0;     // keys above 0; keys above every score
  auto see = [&](uint32_t key) {
    total += key != 0u;
    ranked += key == ~0u;
    if (key != 0u) low = min(low, key);
    if (key != ~0u) top = max(top, key);
  };
#pragma unroll
  for (int i = 0; i < PER_LANE; ++i) {
    own[i] = i * 32 + lane < n ? row[i * 32 + lane] : 0u;
    see(own[i]);
  }
#pragma unroll 4
  for (int j = rest; j < n; j += 32) see(row[j]);
  auto sum = [](int v) {
    return static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(v)));
  };
  total = sum(total);
  ranked = sum(ranked);
  if (total <= keep) return {1u, keep, false};
  if (ranked >= keep) return {~0u, keep, ranked > keep};
  uint32_t lo = __reduce_min_sync(0xffffffffu, low);
  uint32_t hi = __reduce_max_sync(0xffffffffu, top) + 1u;  // top < ~0
  int above_lo = total, above_hi = ranked;  // keys >= lo (> keep), >= hi (< keep)
  for (int step = 0; hi - lo > 1u; ++step) {
    uint32_t t = lo + (hi - lo) / 2;
    if ((step & 3) != 3) {
      const double a = key_score(lo), b = key_score(hi);
      const double part = step & 1 ? 0.5
                                   : static_cast<double>(above_lo - keep) /
                                         static_cast<double>(above_lo - above_hi);
      const uint32_t guess = static_cast<uint32_t>(sort_key(a + (b - a) * part) >> 32);
      if (guess > lo && guess < hi) t = guess;
    }
    int count = 0;
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) count += own[i] >= t;
#pragma unroll 4
    for (int j = rest; j < n; j += 32) count += row[j] >= t;
    count = sum(count);
    if (count == keep) return {t, keep, false};
    if (count > keep) {
      lo = t;
      above_lo = count;
    } else {
      hi = t;
      above_hi = count;
    }
  }
  return {lo, keep - above_hi, true};
}

constexpr int kRegisterKeys = 40;  // per lane: rows up to 1280 key blocks

__global__ void __launch_bounds__(kSelectThreads, 2)
    block_select_kernel(const __grid_constant__ CUtensorMap tm_q,
                        const __grid_constant__ CUtensorMap tm_k, const SelectParams p) {
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* ring = smem + kQTileBytes;
  SelectBarriers* bar = reinterpret_cast<SelectBarriers*>(ring + kStages * kStageBytes);
  uint32_t* keys = reinterpret_cast<uint32_t*>(bar + 1);  // [rows][visible blocks]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t kv = blockIdx.x / p.groups;               // (batch, key head)
  const int b = static_cast<int>(kv / p.Hk);
  const int head_rows = p.Hq / p.Hk * p.query_blocks;     // query blocks of the key head
  const int row_in_head = (blockIdx.x % p.groups) * p.rows_cta;
  const int rows = min(p.rows_cta, head_rows - row_in_head);
  const int64_t row0 = kv * head_rows + row_in_head;
  const int key_len = visible_keys(p, b);
  const int blocks = (key_len + kKeyBlock - 1) / kKeyBlock;
  int tiles = (blocks + kTileKeys - 1) / kTileKeys;

  if (threadIdx.x == 0) {
    mbar_init(&bar->q_full, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bar->full[s], 1);
      mbar_init(&bar->empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->tmem_full[i], 1);
      mbar_init(&bar->tmem_empty[i], kEpilogueWarps / 2);
    }
    mbar_init(&bar->drain, 1);
    bar->abort_flag = 0;
    fence_barrier_init();
    if ((smem_u32(smem) & 1023u) != 0) {  // the swizzle atoms' alignment
      record_device_error(kDevBadLaunch);
      bar->abort_flag = 1;
    }
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&bar->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar->tmem_base;
  volatile int* abort_flag = &bar->abort_flag;
  if (*abort_flag) tiles = 0;

  if (warp == kLoadWarp) {
    if (lane == 0 && tiles > 0) {
      mbar_arrive_expect_tx(&bar->q_full, kQTileBytes);
      for (int d = 0; d < kQDigits; ++d)
        tma_load_3d(smem + d * (kMaxRows * kChannels), &tm_q, &bar->q_full, 0, d,
                    static_cast<int>(row0));
      int issued = 0;
      for (; issued < kKDigits * tiles; ++issued) {
        const int s = issued % kStages;
        if (!mbar_wait(&bar->empty[s], (static_cast<uint32_t>(issued / kStages) & 1u) ^ 1u,
                       abort_flag, kDevWaitTimeoutProducer))
          break;
        mbar_arrive_expect_tx(&bar->full[s], kStageBytes);
        tma_load_4d(ring + s * kStageBytes, &tm_k, &bar->full[s], 0, issued / kKDigits * kTileKeys,
                    static_cast<int>(kv), issued % kKDigits);
      }
      // Every copy lands before the CTA exits.
      drain_wait(&bar->q_full, 0);
      for (int i = max(0, issued - kStages); i < issued; ++i)
        drain_wait(&bar->full[i % kStages], static_cast<uint32_t>(i / kStages) & 1u);
    }
  } else if (warp == kMmaWarp) {
    if (lane == 0 && tiles > 0) {
      constexpr uint32_t idesc = idesc_i8(kTileKeys, kMmaN);
      const uint64_t q_desc = umma_desc_sw128(smem_u32(smem));
      bool ok = mbar_wait(&bar->q_full, 0, abort_flag, kDevWaitTimeoutMma);
      for (int t = 0; t < tiles && ok; ++t) {
        ok = mbar_wait(&bar->tmem_empty[t & 1], (static_cast<uint32_t>(t >> 1) & 1u) ^ 1u,
                       abort_flag, kDevWaitTimeoutMma);
        for (int d = 0; d < kKDigits && ok; ++d) {
          const int i = t * kKDigits + d, s = i % kStages;
          ok = mbar_wait(&bar->full[s], static_cast<uint32_t>(i / kStages) & 1u, abort_flag,
                         kDevWaitTimeoutMma);
          if (!ok) break;
          tc_fence_after();
          const uint64_t k_desc = umma_desc_sw128(smem_u32(ring) + s * kStageBytes);
          const uint32_t d_tmem = tmem + static_cast<uint32_t>(t & 1) * kBufCols +
                                  static_cast<uint32_t>(d * kMmaN);
#pragma unroll
          for (int kk = 0; kk < kChannels / 32; ++kk)
            mma_i8_ss(d_tmem, k_desc + 2u * kk, q_desc + 2u * kk, idesc, kk > 0 ? 1u : 0u);
          mma_commit(&bar->empty[s]);
        }
        if (ok) mma_commit(&bar->tmem_full[t & 1]);
      }
      mma_commit(&bar->drain);
      drain_wait(&bar->drain, 0);
    }
  } else {
    // Warps 0-3 take the even tiles, 4-7 the odd ones: one key block per thread.
    const int buf = warp >> 2, quad = warp & 3;
    for (int t = buf; t < tiles; t += 2) {
      const int j = t * kTileKeys + quad * 32 + lane;
      const int n = min(kKeyBlock, key_len - j * kKeyBlock);
      const double factor = n > 0 ? block_factor(p, kv, j, n) : 0.0;
      if (!__all_sync(0xffffffffu,
                      mbar_wait(&bar->tmem_full[buf], static_cast<uint32_t>(t >> 1) & 1u,
                                abort_flag, kDevWaitTimeoutEpilogue)))
        break;
      tc_fence_after();
      const uint32_t src = tmem + (static_cast<uint32_t>(quad * 32) << 16) +
                           static_cast<uint32_t>(buf) * kBufCols;
#pragma unroll 1
      for (int r0 = 0; r0 < rows; r0 += 4) {
        uint32_t lo[kQDigits][4], hi[kQDigits][4];
#pragma unroll
        for (int d = 0; d < kQDigits; ++d) {
          tmem_ld4(src + d * kMaxRows + r0, lo[d]);
          tmem_ld4(src + kMmaN + d * kMaxRows + r0, hi[d]);
        }
#pragma unroll
        for (int d = 0; d < kQDigits; ++d) {
          tmem_wait_ld_regs4(lo[d]);
          tmem_wait_ld_regs4(hi[d]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // Digit sums of weight 128^w, two to a 32-bit integer, in int64.
          int w[kQDigits + 1];
          w[0] = static_cast<int>(lo[0][i]);
#pragma unroll
          for (int d = 1; d < kQDigits; ++d)
            w[d] = static_cast<int>(lo[d][i]) + static_cast<int>(hi[d - 1][i]);
          w[kQDigits] = static_cast<int>(hi[kQDigits - 1][i]);
          const int64_t v = static_cast<int64_t>(w[1] * 128 + w[0]) +
                            static_cast<int64_t>(w[3] * 128 + w[2]) * (1ll << 14) +
                            static_cast<int64_t>(w[5] * 128 + w[4]) * (1ll << 28) +
                            static_cast<int64_t>(w[6]) * (1ll << 42);
          const int r = r0 + i;
          if (n > 0 && r < rows) {
            uint32_t key = static_cast<uint32_t>(sort_key(static_cast<double>(v) * factor) >> 32);
            if (p.policy != nullptr) {
              const int prow = p.policy_rows == 1 ? 0 : (row_in_head + r) % p.query_blocks;
              const int pol = p.policy[static_cast<int64_t>(prow) * p.key_blocks + j];
              key = pol < 0 ? 0u : (pol > 0 ? ~0u : key);
            }
            keys[static_cast<int64_t>(r) * blocks + j] = key;
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->tmem_empty[buf]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
  if (warp >= rows || *abort_flag) return;

  uint32_t* row = keys + static_cast<int64_t>(warp) * blocks;
  const int64_t grow = row0 + warp;
  Edge edge = find_edge<kRegisterKeys>(row, blocks, p.keep);
  if (edge.shared && edge.word != ~0u) {
    // Blocks share the edge's top word: their low words decide.  The digits give
    // the same integer, so the same fp64 score, as the tensor core did.
    const int8_t* qd = p.q_digits + grow * (kQDigits * kChannels) + lane * 4;
    int64_t q[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      q[c] = 0;
#pragma unroll
      for (int d = kQDigits - 1; d >= 0; --d) q[c] = q[c] * 128 + qd[d * kChannels + c];
    }
    const int64_t plane = static_cast<int64_t>(p.B) * p.Hk * p.key_blocks * kChannels;
    for (int j = 0; j < blocks; ++j) {
      const uint32_t word = row[j];
      uint32_t next = word > edge.word ? ~0u : 0u;
      if (word == edge.word) {
        const int8_t* kd = p.k_digits + (kv * p.key_blocks + j) * kChannels + lane * 4;
        int64_t v = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) v += q[c] * (kd[plane + c] * 128 + kd[c]);
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
        const int n = min(kKeyBlock, key_len - j * kKeyBlock);
        const uint64_t full = sort_key(static_cast<double>(v) * block_factor(p, kv, j, n));
        next = 1u + (static_cast<uint32_t>(full) >> 1);
      }
      __syncwarp();
      if (lane == 0) row[j] = next;
    }
    __syncwarp();
    edge = find_edge<kRegisterKeys>(row, blocks, p.keep);
  }
  int32_t* out = p.out + grow * p.keep;
  const uint32_t before = (1u << lane) - 1u;
  int count = 0, left = edge.left;
  for (int j0 = 0; j0 < blocks; j0 += 32) {
    const int j = j0 + lane;
    const uint32_t key = j < blocks ? row[j] : 0u;
    const bool equal = key == edge.word;
    const uint32_t equals = __ballot_sync(0xffffffffu, equal);
    const bool take = key > edge.word || (equal && __popc(equals & before) < left);
    const uint32_t taken = __ballot_sync(0xffffffffu, take);
    if (take) out[count + __popc(taken & before)] = j;
    count += __popc(taken);
    left -= min(left, __popc(equals));
  }
  for (int j = count + lane; j < p.keep; j += 32) out[j] = -1;
}

struct SelectWorkspace {
  int64_t q_bytes, k_bytes;
};
SelectWorkspace select_workspace(int64_t B, int64_t Hq, int64_t Hk, int64_t Lq, int64_t Lk) {
  const int64_t qb = (Lq + kQueryBlock - 1) / kQueryBlock;
  const int64_t kb = (Lk + kKeyBlock - 1) / kKeyBlock;
  return {B * Hq * qb * kQDigits * kChannels, B * Hk * kb * kKDigits * kChannels};
}

void check_select(int64_t B, int64_t Hq, int64_t Hk, int64_t Lq, int64_t Lk, int64_t D) {
  TB_REQUIRE(D == 64 || D == 128, "the block choice takes head_dim 64 or 128");
  TB_REQUIRE(B > 0 && Hq > 0 && Hk > 0 && Lq > 0 && Lk > 0,
             "empty Q/K sequences are not supported");
  TB_REQUIRE(Hq % Hk == 0, "num_qo_heads must be divisible by num_kv_heads");
  TB_REQUIRE(Lq <= INT32_MAX - 256 && Lk <= static_cast<int64_t>(kMaxKeyBlocks) * kKeyBlock,
             "the block choice takes at most 1572864 keys");
  TB_REQUIRE(B <= INT32_MAX / Hq &&
                 B * Hq <= INT32_MAX / std::max((Lq + kQueryBlock - 1) / kQueryBlock,
                                                (Lk + kKeyBlock - 1) / kKeyBlock) / 2,
             "batch, heads and blocks exceed the grid range");
}

void select_launch(SelectParams& p, cudaStream_t stream) {
  // Query blocks per CTA: fewer where their keys outgrow shared memory or where
  // the CTAs would not fill the SMs (the search is a warp per query block, the
  // products of idle rows cost nothing that matters).
  const int64_t head_rows = static_cast<int64_t>(p.Hq) / p.Hk * p.query_blocks;
  const int64_t heads = static_cast<int64_t>(p.B) * p.Hk;
  auto smem_of = [&](int rows) {
    return static_cast<size_t>(kFixedSmem) + static_cast<size_t>(rows) * p.key_blocks * 4;
  };
  p.rows_cta = kMaxRows;
  while (p.rows_cta > 1 &&
         (smem_of(p.rows_cta) > device_smem_optin() ||
          heads * ((head_rows + p.rows_cta - 1) / p.rows_cta) < device_sm_count()))
    p.rows_cta /= 2;
  p.groups = static_cast<int>((head_rows + p.rows_cta - 1) / p.rows_cta);
  CUtensorMap tq, tk;
  {
    const uint64_t dims[3] = {kChannels, kQDigits, static_cast<uint64_t>(heads * head_rows)};
    const uint64_t strides[2] = {kChannels, kQDigits * kChannels};
    const uint32_t box[3] = {kChannels, 1, kMaxRows};
    encode_tensor_map(&tq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, p.q_digits, dims, strides, box,
                      CU_TENSOR_MAP_SWIZZLE_128B);
  }
  {
    const uint64_t nk = static_cast<uint64_t>(p.key_blocks), nh = static_cast<uint64_t>(heads);
    const uint64_t dims[4] = {kChannels, nk, nh, kKDigits};
    const uint64_t strides[3] = {kChannels, nk * kChannels, nh * nk * kChannels};
    const uint32_t box[4] = {kChannels, kTileKeys, 1, 1};
    encode_tensor_map(&tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, p.k_digits, dims, strides, box,
                      CU_TENSOR_MAP_SWIZZLE_128B);
  }
  const size_t smem = smem_of(p.rows_cta);
  TB_CUDA_CHECK(cudaFuncSetAttribute(block_select_kernel,
                                     cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(smem)));
  block_select_kernel<<<static_cast<unsigned>(heads * p.groups), kSelectThreads, smem, stream>>>(
      tq, tk, p);
  TB_CUDA_CHECK(cudaGetLastError());
}

}  // namespace
}  // namespace tb

using tb::guarded;

extern "C" int tb_select_key_blocks_workspace(int64_t B, int64_t Hq, int64_t Hk, int64_t Lq,
                                              int64_t Lk, int64_t D, int64_t* bytes) {
  return guarded([&] {
    TB_REQUIRE(bytes != nullptr, "the workspace size needs a place");
    tb::check_select(B, Hq, Hk, Lq, Lk, D);
    const tb::SelectWorkspace w = tb::select_workspace(B, Hq, Hk, Lq, Lk);
    *bytes = w.q_bytes + w.k_bytes;
  });
}

extern "C" int tb_select_key_blocks(const int8_t* q, const int8_t* k, const float* q_scale,
                                    const float* k_scale, const int32_t* key_lengths,
                                    const int8_t* block_policy, int64_t policy_rows,
                                    int32_t* block_index, void* workspace,
                                    int64_t workspace_bytes, int64_t B, int64_t Hq, int64_t Hk,
                                    int64_t Lq, int64_t Lk, int64_t D, int64_t keep,
                                    const int64_t* strides, tb_stream_t stream) {
  return guarded([&] {
    using namespace tb;
    TB_REQUIRE(q && k && q_scale && k_scale && block_index && workspace && strides,
               "query, key, scales and block_index must be CUDA tensors");
    check_select(B, Hq, Hk, Lq, Lk, D);
    const int64_t query_blocks = (Lq + kQueryBlock - 1) / kQueryBlock;
    const int64_t key_blocks = (Lk + kKeyBlock - 1) / kKeyBlock;
    TB_REQUIRE(keep > 0 && keep <= key_blocks, "keep must be between 1 and the key blocks");
    TB_REQUIRE(block_policy == nullptr || policy_rows == 1 || policy_rows == query_blocks,
               "block_policy must have one row or one row per query block");
    const SelectWorkspace w = select_workspace(B, Hq, Hk, Lq, Lk);
    TB_REQUIRE(workspace_bytes >= w.q_bytes + w.k_bytes,
               "the block choice needs the workspace tb_select_key_blocks_workspace names");
    auto aligned = [](const void* ptr, uintptr_t a) {
      return (reinterpret_cast<uintptr_t>(ptr) & (a - 1)) == 0;
    };
    TB_REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(workspace, 16),
               "Q/K and the workspace must be 16-byte aligned");
    TB_REQUIRE(aligned(q_scale, 4) && aligned(k_scale, 4) && aligned(key_lengths, 4) &&
                   aligned(block_index, 4),
               "scales, key_lengths and block_index must be 4-byte aligned");
    for (int i = 0; i < 6; ++i)
      TB_REQUIRE(strides[i] % 16 == 0, "Q/K strides must be multiples of 16 bytes");
    require_sm100();
    SelectParams p{};
    p.q = q;
    p.k = k;
    p.q_scale = q_scale;
    p.k_scale = k_scale;
    p.key_lengths = key_lengths;
    p.policy = block_policy;
    for (int i = 0; i < 3; ++i) {
      p.q_s[i] = strides[i];
      p.k_s[i] = strides[3 + i];
    }
    p.B = static_cast<int>(B);
    p.Hq = static_cast<int>(Hq);
    p.Hk = static_cast<int>(Hk);
    p.Lq = static_cast<int>(Lq);
    p.Lk = static_cast<int>(Lk);
    p.query_blocks = static_cast<int>(query_blocks);
    p.key_blocks = static_cast<int>(key_blocks);
    p.keep = static_cast<int>(keep);
    p.policy_rows = static_cast<int>(policy_rows);
    p.q_tiles_scale = static_cast<int>((Lq + 63) / 64 * 4);
    p.q_digits = static_cast<int8_t*>(workspace);
    p.k_digits = p.q_digits + w.q_bytes;
    p.out = block_index;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int64_t key_ctas = (B * Hk * key_blocks + kSumWarps - 1) / kSumWarps;
    const unsigned grid = static_cast<unsigned>(key_ctas + B * Hq * query_blocks);
    if (D == 128) block_sums_kernel<128><<<grid, kSumThreads, 0, s>>>(p);
    else block_sums_kernel<64><<<grid, kSumThreads, 0, s>>>(p);
    TB_CUDA_CHECK(cudaGetLastError());
    select_launch(p, s);
  });
}
