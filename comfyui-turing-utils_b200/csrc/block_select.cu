// Choice of the key blocks that each query block attends to (the lists of
// sparse_attn.cu), from INT8 Q/K and their scales.
//
//   qm_i = sum over the 128 queries of block i of q_scale * Q8     (fp64)
//   S_j  = sum over the n_j visible keys of block j (64 keys) of K8 (exact)
//   score(i, j) = (qm_i . S_j) * k_scale_j / n_j
// which ranks as the mean score of the pair's query-key grid does (sm_scale and
// the query count change no rank), and the `keep` blocks of the highest score
// in ascending order, ties to the lowest block.  block_policy takes a block out
// (-1) or ranks it above every score (1); a NaN score, as under a k_scale that is
// not finite, ranks lowest.
//
// Which of two near blocks is kept is decided by the last digits, so the dot
// product is integer: qm_i is rounded to 40 bits below the power of two above
// its largest channel and written as six digits of base 128 in [-64, 63], S_j
// (14 bits) as two, and the tensor core multiplies the digit planes exactly
// (kind::i8, INT32 sums below 2^20).  The planes join in 64-bit integers.  fp64
// rounds the sum (past 2^53), k_scale_j / n_j and their product.  The sum order
// never matters, equal blocks score equal.
//
//   1. block_sums_kernel: 16-byte loads, channel sums by dp4a of transposed
//      words; a warp per key block, a CTA per query block (a warp per 16-token
//      scale tile).  HBM-bound: the only pass over Q and K.
//   2. block_select_kernel: a CTA takes up to 8 query blocks of one key head
//      (its query heads' blocks in a row) and all key blocks, 128 at a time:
//      M = 128 key blocks, N = 8 query blocks x 6 digits, K = channels, twice
//      for the two digits of S.  Warp 8 loads digit planes by TMA into a
//      4-stage ring, warp 9 issues the MMAs into two TMEM buffers, warps 0-3
//      and 4-7 take the tiles in turn and leave the top word of each score's
//      sortable bits in shared memory.  Then one warp per query block finds the
//      keep-th word (choose_row), and, where that word is shared by more blocks
//      than fit, again with their low words from the digits, one block after the
//      other: rare, but a query block of zeros (padding) ties all blocks (one such
//      among 1182 key blocks: 1.0 ms in all; 30 of 591 in each of 40 heads 1.4 ms,
//      0.38 without; 24576 key blocks 19 ms).  Two CTAs per SM
//      (up to 1300 key blocks): one's search runs under the other's products.
//      Bound by the latency of the scores' read-back and of the search, not by the
//      tensor core: 75600 tokens x 40 heads, 1182 key blocks: 174 us, after 136 us
//      (5.7 TB/s) of sums.
#include <algorithm>
#include <cmath>

#include "attn_common.cuh"
#include "tb_capi_internal.h"
#include "tb_tu.cuh"

namespace tb {
namespace {

constexpr int kQueryBlock = 128;
constexpr int kKeyBlock = 64;
constexpr int kTileRows = 16;            // tokens of one q_scale
constexpr int kSumThreads = 128;
constexpr int kSumWarps = kSumThreads / 32;
constexpr int kTiles = kQueryBlock / kTileRows;
static_assert(kTiles == 2 * kSumWarps && kSumThreads == 128, "two scale tiles per warp, a thread per channel");
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
  int groups;                  // row groups per key head
  int cluster;                 // CTAs that share a row group's key blocks
  float z, slope;              // normal quantile that `keep` of the key blocks exceed; deviations
                               // that one block more or less moves it there
  int8_t* q_digits;            // [B * Hq * query_blocks, kQDigits, kChannels]
  int8_t* k_digits;            // [kKDigits, B * Hk, key_blocks, kChannels]
  double* k_factor;            // [B * Hk, key_blocks]: k_scale / visible keys
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

// Channel sums of INT8 rows: a lane owns 16 channels of every kStep-th row.
// Four rows' words are transposed (8 byte permutes) so that one dp4a adds four
// rows of a channel: 12 instructions per 16 bytes, a third of widening them.
struct ChannelSums {
  int acc[16];
  __device__ __forceinline__ ChannelSums() {
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0;
  }
  __device__ __forceinline__ void add4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, int word) {
    const uint32_t ab = __byte_perm(a, b, 0x5140), cd = __byte_perm(c, d, 0x5140);
    const uint32_t ef = __byte_perm(a, b, 0x7362), gh = __byte_perm(c, d, 0x7362);
    constexpr int kOnes = 0x01010101;
    int* s = acc + 4 * word;
    s[0] = __dp4a(static_cast<int>(__byte_perm(ab, cd, 0x5410)), kOnes, s[0]);
    s[1] = __dp4a(static_cast<int>(__byte_perm(ab, cd, 0x7632)), kOnes, s[1]);
    s[2] = __dp4a(static_cast<int>(__byte_perm(ef, gh, 0x5410)), kOnes, s[2]);
    s[3] = __dp4a(static_cast<int>(__byte_perm(ef, gh, 0x7632)), kOnes, s[3]);
  }
  // Rows [0, n) of ROWS, all of the loads in flight; src is the lane's first row.
  template <int ROWS, int STEP>
  __device__ __forceinline__ void add_rows(const int8_t* src, int64_t stride, int sub, int n) {
    constexpr int kLoads = ROWS / STEP;
    uint4 v[(kLoads + 3) / 4 * 4];
#pragma unroll
    for (int i = 0; i < (kLoads + 3) / 4 * 4; ++i) {
      v[i] = make_uint4(0u, 0u, 0u, 0u);
      if (i < kLoads && i * STEP + sub < n)
        v[i] = *reinterpret_cast<const uint4*>(src + i * STEP * stride);
    }
#pragma unroll
    for (int i = 0; i < kLoads; i += 4) {
      add4(v[i].x, v[i + 1].x, v[i + 2].x, v[i + 3].x, 0);
      add4(v[i].y, v[i + 1].y, v[i + 2].y, v[i + 3].y, 1);
      add4(v[i].z, v[i + 1].z, v[i + 2].z, v[i + 3].z, 2);
      add4(v[i].w, v[i + 1].w, v[i + 2].w, v[i + 3].w, 3);
    }
  }
  // Over the lanes that own the same channels: pair i holds channels 2i and
  // 2i + 1 as S1 * 2^16 + S0 (exact: both fit 16 bits signed, and sums of such
  // pairs are pairs of sums).
  template <int LANES_PER_ROW>
  __device__ __forceinline__ void reduce(int (&pair)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) pair[i] = acc[2 * i + 1] * 65536 + acc[2 * i];
#pragma unroll
    for (int m = LANES_PER_ROW; m < 32; m <<= 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) pair[i] += __shfl_xor_sync(0xffffffffu, pair[i], m);
    }
  }
};

// Block and (batch, head) of a task, in the order that memory is laid out:
// where a token's heads lie side by side, the heads of a block come one after
// another (75600 tokens x 40 heads: 136 us, 146 by heads first).
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

template <int D>
__global__ void __launch_bounds__(kSumThreads, 8) block_sums_kernel(const SelectParams p) {
  constexpr int kLanesPerRow = D / 16;
  __shared__ double part[kTiles][kChannels];
  __shared__ int top;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = (lane % kLanesPerRow) * 16;
  const int sub = lane / kLanesPerRow;
  const int64_t key_tasks = static_cast<int64_t>(p.B) * p.Hk * p.key_blocks;
  const int64_t key_ctas = (key_tasks + kSumWarps - 1) / kSumWarps;
  constexpr int kStep = 32 / kLanesPerRow;
  ChannelSums sums;
  int pair[8];
  if (blockIdx.x < key_ctas) {
    const int64_t task = static_cast<int64_t>(blockIdx.x) * kSumWarps + warp;
    if (task >= key_tasks) return;
    int j, bh;
    block_of(task, p.B, p.Hk, p.key_blocks, p.k_s, j, bh);
    const int b = bh / p.Hk;
    const int n = min(kKeyBlock, visible_keys(p, b) - j * kKeyBlock);
    if (n <= 0) return;  // never scored
    const int8_t* src = p.k + b * p.k_s[0] + (bh % p.Hk) * p.k_s[1] +
                        static_cast<int64_t>(j) * kKeyBlock * p.k_s[2] + col;
    const int64_t at = static_cast<int64_t>(bh) * p.key_blocks + j;
    const float scale = __ldg(p.k_scale + at);
    // Eight loads in flight per lane: twice as many cost occupancy.
    constexpr int kPart = 8 * kStep;
    static_assert(kKeyBlock % kPart == 0, "whole parts");
    src += sub * p.k_s[2];
#pragma unroll 1
    for (int r = 0; r < n; r += kPart)
      sums.add_rows<kPart, kStep>(src + r * p.k_s[2], p.k_s[2], sub, n - r);
    sums.reduce<kLanesPerRow>(pair);
    if (sub < kKDigits) {  // lane group d writes digit plane d
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // S + 64 * 129 in [0, 2^14], in two 16-bit lanes each: the two digits,
        // each plus 64.
        const uint32_t x = static_cast<uint32_t>(pair[2 * i]) + 64u * 129u * 0x00010001u;
        const uint32_t y = static_cast<uint32_t>(pair[2 * i + 1]) + 64u * 129u * 0x00010001u;
        const uint32_t xd = (sub == 0 ? x & 0x007f007fu : (x >> 7) & 0x01ff01ffu) + 0x00c000c0u;
        const uint32_t yd = (sub == 0 ? y & 0x007f007fu : (y >> 7) & 0x01ff01ffu) + 0x00c000c0u;
        w[i] = __byte_perm(xd, yd, 0x6420);  // the low byte of every lane: minus 64 mod 256
      }
      int8_t* dst = p.k_digits + (sub * key_tasks + at) * kChannels + col;
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
      if (D < kChannels) *reinterpret_cast<uint4*>(dst + D) = make_uint4(0, 0, 0, 0);
    }
    // Under an infinite scale the dequantized keys are infinities of both signs and
    // 0 * inf: the block's mean is no number, as under a NaN.
    if (lane == 0)
      p.k_factor[at] = isfinite(scale) ? static_cast<double>(scale) / n : static_cast<double>(NAN);
    return;
  }
  int i, bh;
  block_of(blockIdx.x - key_ctas, p.B, p.Hq, p.query_blocks, p.q_s, i, bh);
  const int64_t at = static_cast<int64_t>(bh) * p.query_blocks + i;
  if (threadIdx.x == 0) top = 0;
  const int8_t* src = p.q + (bh / p.Hq) * p.q_s[0] + (bh % p.Hq) * p.q_s[1] + col;
  const float* scales = p.q_scale + static_cast<int64_t>(bh) * p.q_tiles_scale + i * kTiles;
  ChannelSums other;
  float scale[2];
  // Both tiles' loads are in flight before either is added up.
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int row0 = i * kQueryBlock + (2 * warp + t) * kTileRows;
    const int n = min(kTileRows, p.Lq - row0);
    scale[t] = n > 0 ? __ldg(scales + 2 * warp + t) : 0.0f;
    (t == 0 ? sums : other)
        .add_rows<kTileRows, kStep>(src + (row0 + sub) * p.q_s[2], p.q_s[2], sub, n);
  }
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    (t == 0 ? sums : other).reduce<kLanesPerRow>(pair);
    if (sub < 4) {  // lane group s keeps channels 4s .. 4s + 3
      int a = pair[0], b = pair[1];
#pragma unroll
      for (int w = 1; w < 4; ++w) {
        a = sub == w ? pair[2 * w] : a;
        b = sub == w ? pair[2 * w + 1] : b;
      }
      auto scaled = [&](int v) {  // v in the low mantissa bits of 2^52 + 2^31: exact
        return static_cast<double>(scale[t]) *
               (__hiloint2double(0x43300000, v ^ static_cast<int>(0x80000000u)) -
                4503601774854144.0);
      };
      const int a0 = static_cast<int16_t>(a), b0 = static_cast<int16_t>(b);
      // Stored by lane, 32 bytes apart: no bank conflicts.
      double2* dst = reinterpret_cast<double2*>(
          &part[2 * warp + t][(sub * kLanesPerRow + col / 16) * 4]);
      dst[0] = make_double2(scaled(a0), scaled((a - a0) >> 16));
      dst[1] = make_double2(scaled(b0), scaled((b - b0) >> 16));
    }
  }
  __syncthreads();
  const int x = threadIdx.x;  // place in `part`
  double m = 0.0;
  if (x < kChannels) {
    if (x < D) {
#pragma unroll
      for (int w = 0; w < kTiles; ++w) m += part[w][x];
    }
    // Exponent field of the largest channel (NaN and infinity: 0x7ff).
    const unsigned e = (__double2hiint(m) >> 20) & 0x7ff;
    const unsigned we = __reduce_max_sync(0xffffffffu, e);
    if (lane == 0) atomicMax(&top, static_cast<int>(we));
  }
  __syncthreads();
  if (x < kChannels) {
    // |m| < 2^(top - 1022); v = m * 2^(kFixBits + 1022 - top) to the nearest
    // integer, by the rounding of an addition to 1.5 * 2^52.  (fp32 scales keep
    // top above 800.)  A block whose mean is not finite scores 0 everywhere.
    int64_t v = 0;
    if (top > 64 && top < 0x7ff) {
      const double unit = __hiloint2double((1023 + kFixBits + 1022 - top) << 20, 0);
      const double magic = 6755399441055744.0;
      v = __double_as_longlong(fma(m, unit, magic)) - __double_as_longlong(magic);
    }
    // Digits plus 64 of v + 64 (128^6 - 1) / 127.
    const uint64_t u = static_cast<uint64_t>(v + 64 * ((1ll << (7 * kQDigits)) - 1) / 127);
    const int c = x < D ? (x / 4 % kLanesPerRow) * 16 + x / (4 * kLanesPerRow) * 4 + x % 4 : x;
    int8_t* dst = p.q_digits + at * (kQDigits * kChannels) + c;
#pragma unroll
    for (int d = 0; d < kQDigits; ++d)
      dst[d * kChannels] = static_cast<int8_t>(static_cast<int>((u >> (7 * d)) & 127) - 64);
  }
}

// score = v * factor as a sortable 64-bit integer: -0 as 0, NaN as -infinity;
// below every score lies 0 (a block that cannot be chosen), above it ~0.  v is
// converted by two exact pieces and one rounding (the conversion unit would
// bound the kernel).
__device__ __forceinline__ double exact_score(int64_t v, double factor) {
  const double hi = __hiloint2double(0x45300000, static_cast<int>(v >> 32) ^ 0x80000000);
  const double lo = __hiloint2double(0x43300000, static_cast<int>(v));
  const double x = (hi - 19342822341709703277445120.0) + lo;  // 2^84 + 2^63 + 2^52
  return fma(x, factor, 0.0);
}
__device__ __forceinline__ uint32_t top_word(double score) {
  uint32_t hi = static_cast<uint32_t>(__double2hiint(score));
  if ((hi & 0x7fffffffu) > 0x7ff00000u) hi = 0xfff00000u;  // NaN
  return hi ^ (static_cast<uint32_t>(static_cast<int>(hi) >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint32_t low_word(double score) {
  const uint32_t lo = static_cast<uint32_t>(__double2loint(score));
  return isnan(score) ? 0xffffffffu : (__double2hiint(score) < 0 ? ~lo : lo);
}

// The score that a key starts, to fp32's range and precision, and back.  Only
// used to guess.
__device__ __forceinline__ float key_value(uint32_t key) {
  const uint32_t hi = key & 0x80000000u ? key ^ 0x80000000u : ~key;
  const int mag = static_cast<int>(hi & 0x7fffffffu) - (896 << 20);
  const int fit = max(0, min(mag, 0x0fdfffff));
  return __uint_as_float((hi & 0x80000000u) | (static_cast<uint32_t>(fit) << 3));
}
__device__ __forceinline__ uint32_t value_key(float x) {
  const uint32_t bits = __float_as_uint(x);
  const uint32_t hi = (bits & 0x80000000u) | (((bits & 0x7fffffffu) >> 3) + (896u << 20));
  return hi ^ (static_cast<uint32_t>(static_cast<int>(hi) >> 31) | 0x80000000u);
}

// Keys of a row that each lane of its search owns: an odd number, so that the
// lanes' first keys lie in different banks.
__host__ __device__ constexpr int keys_per_lane(int n) { return ((n + 31) / 32) | 1; }

// The `keep` highest of a row's n keys: their places into out, ascending, equals
// lowest first, -1 where fewer keys are above 0; the warp together.  Returns
// false, with the edge, where more keys equal the edge than fit and `settle` is
// not set (the caller then refines the keys).  Lane l owns keys l per .. (l + 1)
// per - 1 (zeros past n), the first PER_LANE of them in registers.
//
// The edge: thresholds are counted (four counters hide the compare-and-add
// latency) until one counts exactly `keep` or the bracket holds one key.  The
// first guess is the normal quantile (`z`) of the scores' mean and deviation;
// until both ends of the bracket are scores it moves by the count's error over
// the normal density (`slope`), then interpolates the counts (an end that stays
// twice counts half); after 12 steps the middle key, which needs at most 32
// more.  About 6 thresholds a row; halving the key range took 22.
template <int PER_LANE>
__device__ __forceinline__ bool choose_row(uint32_t* row, int n, int keep, float z,
                                           float slope, bool settle, int32_t* out,
                                           uint32_t& edge) {
  const int lane = static_cast<int>(lane_id());
  const int per = keys_per_lane(n);
  const int first = lane * per;
  uint32_t own[PER_LANE];
#pragma unroll
  for (int i = 0; i < PER_LANE; ++i) own[i] = i < per ? row[first + i] : 0u;
  auto sum = [](int v) {
    return static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(v)));
  };
  int mine = 0;  // of the keys that `reach` counted last, this lane's
  auto reach = [&](uint32_t t) {
    int c[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) c[i & 3] += own[i] >= t ? 1 : 0;
    for (int i = PER_LANE; i < per; ++i) c[0] += row[first + i] >= t ? 1 : 0;
    mine = (c[0] + c[1]) + (c[2] + c[3]);
    return sum(mine);
  };
  int left = keep;  // equals of the edge that are kept
  bool exact = false;
  if (n > keep) {
    // A few keys of every lane are sample enough.
    float sx = 0.0f, sxx = 0.0f, used = 0.0f;
#pragma unroll
    for (int i = 0; i < PER_LANE; i += (PER_LANE + 7) / 8) {
      const bool in = own[i] + 1u > 1u;  // a score: neither 0 nor ~0
      const float x = in ? key_value(own[i]) : 0.0f;
      used += in ? 1.0f : 0.0f;
      sx += x;
      sxx = fmaf(x, x, sxx);
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) {
      sx += __shfl_xor_sync(0xffffffffu, sx, m);
      sxx += __shfl_xor_sync(0xffffffffu, sxx, m);
      used += __shfl_xor_sync(0xffffffffu, used, m);
    }
    const float part = __fdividef(1.0f, used);
    const float mean = sx * part;
    const float dev = sqrtf(fmaxf(0.0f, sxx * part - mean * mean));
    float guess = mean + z * dev;
    uint32_t lo = 0u, hi = ~0u;            // counts > keep at lo, <= at hi ...
    int above_lo = n, above_hi = 0;
    bool seen_lo = false, seen_hi = false;  // ... each once it was counted
    float half_lo = 1.0f, half_hi = 1.0f;
    int last = 0;
    for (int step = 0; hi - lo > 1u; ++step) {
      uint32_t t = lo + (hi - lo) / 2;
      if (step < 12) {
        const uint32_t g = value_key(guess);
        if (g > lo && g < hi) t = g;
      }
      const int c = reach(t);
      if (c == keep) {
        lo = t;
        exact = true;
        break;
      }
      if (c > keep) {
        lo = t;
        above_lo = c;
        seen_lo = true;
        half_lo = 1.0f;
        if (last == 1) half_hi *= 0.5f;
        last = 1;
      } else {
        hi = t;
        above_hi = c;
        seen_hi = true;
        half_hi = 1.0f;
        if (last == -1) half_lo *= 0.5f;
        last = -1;
      }
      if (seen_lo && seen_hi) {
        const float a = key_value(lo), b = key_value(hi);
        const float fa = static_cast<float>(above_lo - keep) * half_lo;
        const float fb = static_cast<float>(keep - above_hi) * half_hi;
        guess = a + (b - a) * __fdividef(fa, fa + fb);
      } else {
        guess += static_cast<float>(c - keep + last) * slope * dev;
      }
    }
    edge = lo;
    if (!exact) {
      // One key is left: `lo`, or ~0 (blocks before any score) where hi stayed
      // there uncounted.
      if (!seen_hi) {
        above_hi = reach(~0u);
        if (above_hi >= keep) {
          edge = ~0u;
          above_hi = 0;
        }
      }
      if (edge != 0u) {
        if (edge != ~0u && !settle) return false;
        left = keep - above_hi;
      }
    }
  } else {
    edge = 0u;
  }
  if (edge == 0u) {  // no more than `keep` keys are above 0: all of those
    edge = 1u;
    exact = true;
    reach(edge);
  }
  // Places of this lane's kept keys: after those of the lanes before it.
  int equal = 0;
  if (!exact) {
    int c = 0, e = 0;
    for (int i = 0; i < per; ++i) {
      const uint32_t key = row[first + i];
      c += key > edge ? 1 : 0;
      e += key == edge ? 1 : 0;
    }
    int before = e;  // equals of this lane and the lanes before it
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, before, m);
      if (lane >= m) before += v;
    }
    equal = max(0, min(e, left - (before - e)));
    mine = c + equal;
  }
  int at = mine;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, at, m);
    if (lane >= m) at += v;
  }
  const int total = __shfl_sync(0xffffffffu, at, 31);
  at -= mine;
  if (exact && per <= PER_LANE) {
    // The keys are in registers: their places gather in the row's memory and
    // leave it side by side.
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {
      const bool take = own[i] >= edge;
      if (take) row[at] = static_cast<uint32_t>(first + i);
      at += take ? 1 : 0;
    }
    __syncwarp();
    for (int j = lane; j < total; j += 32) out[j] = static_cast<int32_t>(row[j]);
  } else if (exact) {
    for (int i = 0; i < per; ++i)
      if (row[first + i] >= edge) out[at++] = first + i;
  } else {
    for (int i = 0; i < per; ++i) {
      const uint32_t key = row[first + i];
      if (key > edge || (key == edge && equal > 0)) {
        equal -= key == edge ? 1 : 0;
        out[at++] = first + i;
      }
    }
  }
  for (int j = total + lane; j < keep; j += 32) out[j] = -1;
  return true;
}

__device__ __forceinline__ void store_cluster(uint32_t cluster_addr, uint32_t value) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(value) : "memory");
}
__device__ __forceinline__ int64_t mad_wide(int a, int b, int c) {
  int64_t d;
  asm("mad.wide.s32 %0, %1, %2, %3;" : "=l"(d) : "r"(a), "r"(b), "l"(static_cast<int64_t>(c)));
  return d;
}
// Keeps uses of a tmem_ld4's registers behind the tmem_wait_ld before it.
__device__ __forceinline__ void after_wait(uint32_t (&r)[4]) {
  asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]));
}

// PER_LANE: keys of a row that a lane of the search keeps in registers.
template <int PER_LANE>
__global__ void __launch_bounds__(kSelectThreads, 2)
    block_select_kernel(const __grid_constant__ CUtensorMap tm_q,
                        const __grid_constant__ CUtensorMap tm_k, const SelectParams p) {
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* ring = smem + kQTileBytes;
  SelectBarriers* bar = reinterpret_cast<SelectBarriers*>(ring + kStages * kStageBytes);
  uint32_t* keys = reinterpret_cast<uint32_t*>(bar + 1);  // [rows][row_keys], zeros past `blocks`

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % p.cluster;
  const int group = static_cast<int>(blockIdx.x) / p.cluster;
  const int64_t kv = group / p.groups;                    // (batch, key head)
  const int b = static_cast<int>(kv / p.Hk);
  const int head_rows = p.Hq / p.Hk * p.query_blocks;     // query blocks of the key head
  const int row_in_head = (group % p.groups) * p.rows_cta;
  const int rows = min(p.rows_cta, head_rows - row_in_head);
  const int64_t row0 = kv * head_rows + row_in_head;
  const int key_len = visible_keys(p, b);
  const int blocks = (key_len + kKeyBlock - 1) / kKeyBlock;
  // This CTA takes every cluster-th tile from its rank on.
  const int all_tiles = (blocks + kTileKeys - 1) / kTileKeys;
  int tiles = (all_tiles - rank + p.cluster - 1) / p.cluster;
  const int row_keys = 32 * keys_per_lane(blocks);

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
  } else if (warp < rows) {
    for (int j = blocks + lane; j < row_keys; j += 32) keys[warp * row_keys + j] = 0u;
  }
  tc_fence_before();
  __syncthreads();
  if (p.cluster > 1) cluster_sync_all();  // rank 0 has started: its keys can be written
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
        tma_load_4d(ring + s * kStageBytes, &tm_k, &bar->full[s], 0,
                    (issued / kKDigits * p.cluster + rank) * kTileKeys,
                    static_cast<int>(kv), issued % kKDigits);
      }
      // Every copy lands before the CTA exits.
      drain_wait(&bar->q_full, 0);
      for (int i = max(0, issued - kStages); i < issued; ++i)
        drain_wait(&bar->full[i % kStages], static_cast<uint32_t>(i / kStages) & 1u);
    }
  } else if (warp == kMmaWarp) {
    if (tiles > 0) {
      constexpr uint32_t idesc = idesc_i8(kTileKeys, kMmaN);
      const uint32_t elected = elect_one();
      const uint64_t q_desc = umma_desc_sw128(smem_u32(smem));
      auto warp_wait = [&](uint64_t* bar_, int phase) {
        return __all_sync(0xffffffffu, mbar_wait(bar_, static_cast<uint32_t>(phase) & 1u,
                                                 abort_flag, kDevWaitTimeoutMma)) != 0;
      };
      bool ok = warp_wait(&bar->q_full, 0);
      for (int t = 0; t < tiles && ok; ++t) {
        ok = warp_wait(&bar->tmem_empty[t & 1], (t >> 1) + 1);
        for (int d = 0; d < kKDigits && ok; ++d) {
          const int i = t * kKDigits + d, s = i % kStages;
          ok = warp_wait(&bar->full[s], i / kStages);
          if (!ok) break;
          tc_fence_after();
          const uint64_t k_desc = umma_desc_sw128(smem_u32(ring) + s * kStageBytes);
          const uint32_t d_tmem = tmem + static_cast<uint32_t>(t & 1) * kBufCols +
                                  static_cast<uint32_t>(d * kMmaN);
#pragma unroll
          for (int kk = 0; kk < kChannels / 32; ++kk)
            mma_i8_ss_warp(d_tmem, k_desc + 2u * kk, q_desc + 2u * kk, idesc, kk > 0 ? 1u : 0u,
                           elected);
          mma_commit_warp(&bar->empty[s], elected);
        }
        if (ok) mma_commit_warp(&bar->tmem_full[t & 1], elected);
      }
      mma_commit_warp(&bar->drain, elected);
      if (lane == 0) drain_wait(&bar->drain, 0);
      __syncwarp();
    }
  } else {
    // Warps 0-3 take the even tiles, 4-7 the odd ones: one key block per thread.
    const int buf = warp >> 2, quad = warp & 3;
    const double* factors = p.k_factor + kv * p.key_blocks;
    const int stride = 2 * p.cluster * kTileKeys;  // to this warp's next tile
    int j = (buf * p.cluster + rank) * kTileKeys + quad * 32 + lane;
    double next_factor = j < blocks ? factors[j] : 0.0;
    // Rank 0 keeps the keys.
    const uint32_t keys_at = p.cluster > 1 ? mapa_shared(smem_u32(keys), 0u) : 0u;
    for (int t = buf; t < tiles; t += 2, j += stride) {
      const double factor = next_factor;
      if (j + stride < blocks) next_factor = factors[j + stride];
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
        tmem_wait_ld();
#pragma unroll
        for (int d = 0; d < kQDigits; ++d) {
          after_wait(lo[d]);
          after_wait(hi[d]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // Digit sums of weight 128^w, two to a 32-bit integer, four to an int64.
          const int w0 = lo[0][i], w1 = lo[1][i] + hi[0][i], w2 = lo[2][i] + hi[1][i],
                    w3 = lo[3][i] + hi[2][i], w4 = lo[4][i] + hi[3][i], w5 = lo[5][i] + hi[4][i],
                    w6 = hi[5][i];
          const int64_t low = mad_wide(w3 * 128 + w2, 1 << 14, w1 * 128 + w0);
          const int64_t high = mad_wide(w6, 1 << 14, w5 * 128 + w4);
          const uint32_t key =
              top_word(exact_score(low + static_cast<int64_t>(static_cast<uint64_t>(high) << 28),
                                   factor));
          if (j < blocks && r0 + i < rows) {
            const int at = (r0 + i) * row_keys + j;
            if (p.cluster > 1) store_cluster(keys_at + 4u * static_cast<uint32_t>(at), key);
            else keys[at] = key;
          }
        }
      }
      if (p.policy != nullptr && j < blocks) {
        for (int r = 0; r < rows; ++r) {
          const int prow = p.policy_rows == 1 ? 0 : (row_in_head + r) % p.query_blocks;
          const int pol = p.policy[static_cast<int64_t>(prow) * p.key_blocks + j];
          if (pol != 0) {
            const int at = r * row_keys + j;
            const uint32_t key = pol < 0 ? 0u : ~0u;
            if (p.cluster > 1) store_cluster(keys_at + 4u * static_cast<uint32_t>(at), key);
            else keys[at] = key;
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
  if (p.cluster > 1) cluster_sync_all();  // every tile's keys are in rank 0's memory
  if (rank != 0 || warp >= rows || *abort_flag) return;

  uint32_t* row = keys + warp * row_keys;
  const int64_t grow = row0 + warp;
  int32_t* out = p.out + grow * p.keep;
  uint32_t edge = 0u;
  if (choose_row<PER_LANE>(row, blocks, p.keep, p.z, p.slope, false, out, edge)) return;
  // Blocks share the edge's top word: their low words decide, without the last bit
  // (0 and ~0 are taken) and then by it.  The digits give the same integer, so the
  // same fp64 score, as the tensor core did.
  const int8_t* qd = p.q_digits + grow * (kQDigits * kChannels) + lane * 4;
  int64_t q[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    q[c] = 0;
#pragma unroll
    for (int d = kQDigits - 1; d >= 0; --d) q[c] = q[c] * 128 + qd[d * kChannels + c];
  }
  const int64_t plane = static_cast<int64_t>(p.B) * p.Hk * p.key_blocks * kChannels;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    for (int j = 0; j < blocks; ++j) {
      const uint32_t word = row[j];
      uint32_t next = word > edge ? ~0u : 0u;
      if (word == edge) {
        const int8_t* kd = p.k_digits + (kv * p.key_blocks + j) * kChannels + lane * 4;
        int64_t v = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) v += q[c] * (kd[plane + c] * 128 + kd[c]);
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
        const uint32_t low = low_word(exact_score(v, p.k_factor[kv * p.key_blocks + j]));
        next = 1u + (pass == 0 ? low >> 1 : low & 1u);
      }
      __syncwarp();
      if (lane == 0) row[j] = next;
    }
    __syncwarp();
    if (choose_row<PER_LANE>(row, blocks, p.keep, p.z, p.slope, pass == 1, out, edge)) return;
  }
}

// Quantile of the standard normal distribution by bisection of erfc: a guess's
// precision is enough.
double normal_quantile(double q) {
  double lo = -6.0, hi = 6.0;
  for (int i = 0; i < 24; ++i) {
    const double x = 0.5 * (lo + hi);
    (0.5 * std::erfc(-x * 0.70710678118654752) < q ? lo : hi) = x;
  }
  return lo;
}

struct SelectWorkspace {
  int64_t q_bytes, k_bytes, factor_bytes;
  int64_t total() const { return q_bytes + k_bytes + factor_bytes; }
};
SelectWorkspace select_workspace(int64_t B, int64_t Hq, int64_t Hk, int64_t Lq, int64_t Lk) {
  const int64_t qb = (Lq + kQueryBlock - 1) / kQueryBlock;
  const int64_t kb = (Lk + kKeyBlock - 1) / kKeyBlock;
  return {B * Hq * qb * kQDigits * kChannels, B * Hk * kb * kKDigits * kChannels, B * Hk * kb * 8};
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
  // products of idle rows cost nothing that matters).  Where the SMs would not fill,
  // sums included, by the rule and with full CTAs (heads x query blocks, key blocks):
  // 1 x 591, 1182: 18.8 and 22.2 us; 8 x 8, 313: 13.2 and 14.0; 1 x 8, 313: 10.0 and
  // 10.9; 5 x 118, 236: 12.6 and 12.9; 12 x 33, 73: the same; the other way 40 x 2, 128:
  // 14.5 and 14.4; 2 x 256, 512: 15.2 and 14.2.
  const int64_t head_rows = static_cast<int64_t>(p.Hq) / p.Hk * p.query_blocks;
  const int64_t heads = static_cast<int64_t>(p.B) * p.Hk;
  auto smem_of = [&](int rows) {
    return static_cast<size_t>(kFixedSmem) + static_cast<size_t>(rows) * 32 * keys_per_lane(p.key_blocks) * 4;
  };
  p.rows_cta = kMaxRows;
  while (p.rows_cta > 1 &&
         (smem_of(p.rows_cta) > device_smem_optin() ||
          heads * ((head_rows + p.rows_cta - 1) / p.rows_cta) < device_sm_count()))
    p.rows_cta /= 2;
  p.groups = static_cast<int>((head_rows + p.rows_cta - 1) / p.rows_cta);
  // Few row groups (single tokens): a cluster shares each one's key blocks, as
  // many CTAs as fill two per SM with at least two tiles each (one token, 32 heads,
  // 2048 key blocks: 30 us alone, 18 with clusters of 8).
  const int64_t tiles = (p.key_blocks + kTileKeys - 1) / kTileKeys;
  p.cluster = 1;
  while (p.cluster < 8 && 2 * p.cluster * heads * p.groups <= 2 * device_sm_count() &&
         4 * p.cluster <= tiles)
    p.cluster *= 2;
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
  auto launch = [&](auto kern) {
    // The limit is the kernel's, shared by all host threads: always the same value, or
    // one thread's shorter row would refuse another's launch.
    TB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(device_smem_optin())));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(heads * p.groups * p.cluster));
    cfg.blockDim = dim3(kSelectThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(p.cluster);
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    TB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, tq, tk, p));
  };
  // As many register keys as a row needs; past 41 a lane (1312 key blocks) the
  // rest of a row is read from shared memory: 81 in registers cost the second CTA
  // of an SM (one token, 2048 key blocks: 22 against 18 us).
  const int per_lane = keys_per_lane(p.key_blocks);
  if (per_lane <= 9) launch(block_select_kernel<9>);
  else if (per_lane <= 17) launch(block_select_kernel<17>);
  else launch(block_select_kernel<41>);
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
    *bytes = w.total();
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
    TB_REQUIRE(workspace_bytes >= w.total(),
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
    p.k_factor = reinterpret_cast<double*>(p.k_digits + w.k_bytes);
    const double z = normal_quantile(1.0 - (keep - 0.5) / static_cast<double>(key_blocks));
    p.z = static_cast<float>(z);
    p.slope = static_cast<float>(2.5066282746310002 * std::exp(0.5 * z * z) / key_blocks);
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
