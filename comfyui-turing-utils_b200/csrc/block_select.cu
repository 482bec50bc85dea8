// Choice of the key blocks that each query block attends to (the lists of
// sparse_attn.cu), from INT8 Q/K and their scales.
//
//   qm_i = mean over the 128 queries of block i of q_scale * Q8
//   km_j = mean over the visible keys of block j (64 keys) of k_scale * K8
//   score(i, j) = qm_i . km_j  =  the mean score of the pair's query-key grid
//                                 (up to sm_scale, which changes no rank)
// and the `keep` blocks of the highest score in ascending order, ties to the
// lowest block.  block_policy takes a block out (-1) or ranks it above every
// score (1); a NaN score ranks lowest.
//
// Which of two near blocks is kept is decided by the last digits, so scores are
// exact integers as far as they go and fp64 after that: the sums of codes are
// exact (64 * 127 fits 16 bits), a query block's scaled sum takes 8 fp64
// products of 38 bits, and one score rounds 128 fp64 FMAs.
//
//   1. block_sums_kernel: one warp per key block or query block, 16-byte loads,
//      channel sums as packed 16-bit lanes of the biased bytes (HBM-bound: the
//      only pass over Q and K).
//   2. block_select_kernel: a CTA scores R query blocks against all key blocks
//      (keys sorted as 64-bit integers stay in shared memory), then one warp
//      per query block finds the keep-th key bit by bit and writes the list.
#include <algorithm>

#include "tb_capi_internal.h"
#include "tb_tu.cuh"

namespace tb {
namespace {

constexpr int kQueryBlock = 128;
constexpr int kKeyBlock = 64;
constexpr int kTileRows = 16;            // tokens of one q_scale
constexpr int kSumThreads = 256;
constexpr int kSelectThreads = 256;
constexpr int kMaxKeyBlocks = 24576;     // one query block's keys fill 192 KB

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
  double* q_sums;              // [B * Hq, query_blocks, D]
  int16_t* k_sums;             // [B * Hk, key_blocks, D]
  int32_t* out;                // [B * Hq, query_blocks, keep]
};

__device__ __forceinline__ int visible_keys(const SelectParams& p, int b) {
  return p.key_lengths != nullptr ? max(0, min(__ldg(p.key_lengths + b), p.Lk)) : p.Lk;
}

// Sums of the channels of 16 bytes, kept as biased (byte + 128) 16-bit lanes:
// word w holds channels 4w and 4w + 2 in `even`, 4w + 1 and 4w + 3 in `odd`.
struct ByteSums {
  uint32_t even[4], odd[4];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 4; ++i) even[i] = odd[i] = 0u;
  }
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
};

template <int D>
__global__ void __launch_bounds__(kSumThreads) block_sums_kernel(const SelectParams p) {
  constexpr int kLanesPerRow = D / 16;
  constexpr int kRowsPerStep = 32 / kLanesPerRow;
  const int lane = threadIdx.x & 31;
  const int col = (lane % kLanesPerRow) * 16;
  const int sub = lane / kLanesPerRow;
  const int64_t task = static_cast<int64_t>(blockIdx.x) * (kSumThreads / 32) + (threadIdx.x >> 5);
  const int64_t key_tasks = static_cast<int64_t>(p.B) * p.Hk * p.key_blocks;
  ByteSums sums;
  if (task < key_tasks) {
    const int j = static_cast<int>(task % p.key_blocks);
    const int bh = static_cast<int>(task / p.key_blocks);
    const int b = bh / p.Hk;
    const int n = min(kKeyBlock, visible_keys(p, b) - j * kKeyBlock);
    if (n <= 0) return;  // never scored
    const int8_t* src = p.k + b * p.k_s[0] + (bh % p.Hk) * p.k_s[1] +
                        static_cast<int64_t>(j) * kKeyBlock * p.k_s[2] + col;
    sums.clear();
#pragma unroll
    for (int r = 0; r < kKeyBlock; r += kRowsPerStep)
      if (r + sub < n) sums.add(*reinterpret_cast<const uint4*>(src + (r + sub) * p.k_s[2]));
    sums.reduce<kLanesPerRow>();
    if (sub == 0) {
      const uint32_t bias = static_cast<uint32_t>(n) * 128u;
      uint32_t o[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t c0 = (sums.even[i] & 0xffffu) - bias, c2 = (sums.even[i] >> 16) - bias;
        const uint32_t c1 = (sums.odd[i] & 0xffffu) - bias, c3 = (sums.odd[i] >> 16) - bias;
        o[2 * i] = (c0 & 0xffffu) | (c1 << 16);
        o[2 * i + 1] = (c2 & 0xffffu) | (c3 << 16);
      }
      uint4* dst = reinterpret_cast<uint4*>(p.k_sums + task * D + col);
      dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
      dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
    return;
  }
  const int64_t at = task - key_tasks;
  if (at >= static_cast<int64_t>(p.B) * p.Hq * p.query_blocks) return;
  const int i = static_cast<int>(at % p.query_blocks);
  const int bh = static_cast<int>(at / p.query_blocks);
  const int row0 = i * kQueryBlock;
  const int n = min(kQueryBlock, p.Lq - row0);
  const int8_t* src = p.q + (bh / p.Hq) * p.q_s[0] + (bh % p.Hq) * p.q_s[1] + row0 * p.q_s[2] + col;
  const float* scale = p.q_scale + static_cast<int64_t>(bh) * p.q_tiles_scale + row0 / kTileRows;
  // Lane group `sub` keeps the four channels of word sub % 4.
  const int word = sub & 3;
  double acc[4] = {0.0, 0.0, 0.0, 0.0};
  for (int t = 0; t * kTileRows < n; ++t) {
    const int rows = min(kTileRows, n - t * kTileRows);
    sums.clear();
#pragma unroll
    for (int r = 0; r < kTileRows; r += kRowsPerStep)
      if (r + sub < rows)
        sums.add(*reinterpret_cast<const uint4*>(src + (t * kTileRows + r + sub) * p.q_s[2]));
    sums.reduce<kLanesPerRow>();
    uint32_t e = sums.even[0], o = sums.odd[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      e = word == w ? sums.even[w] : e;
      o = word == w ? sums.odd[w] : o;
    }
    const int bias = rows * 128;
    const double s = static_cast<double>(__ldg(scale + t));
    acc[0] = fma(s, static_cast<double>(static_cast<int>(e & 0xffffu) - bias), acc[0]);
    acc[1] = fma(s, static_cast<double>(static_cast<int>(o & 0xffffu) - bias), acc[1]);
    acc[2] = fma(s, static_cast<double>(static_cast<int>(e >> 16) - bias), acc[2]);
    acc[3] = fma(s, static_cast<double>(static_cast<int>(o >> 16) - bias), acc[3]);
  }
  if (sub < 4) {
    double* dst = p.q_sums + at * D + col + word * 4;
#pragma unroll
    for (int c = 0; c < 4; ++c) dst[c] = acc[c];
  }
}

// Orders fp64 scores as unsigned integers; 0 is left for blocks that cannot be
// chosen.  -0 counts as 0.
__device__ __forceinline__ uint64_t sort_key(double score) {
  if (isnan(score)) score = -INFINITY;
  const int64_t bits = __double_as_longlong(score + 0.0);
  return bits < 0 ? ~static_cast<uint64_t>(bits)
                  : static_cast<uint64_t>(bits) | 0x8000000000000000ull;
}

template <int D, int R>
__global__ void __launch_bounds__(kSelectThreads) block_select_kernel(const SelectParams p) {
  extern __shared__ __align__(16) unsigned char select_smem[];
  double* qs = reinterpret_cast<double*>(select_smem);                     // [D][R]
  uint64_t* keys = reinterpret_cast<uint64_t*>(select_smem) + D * R;       // [R][key_blocks]
  const int groups = (p.query_blocks + R - 1) / R;
  const int bh = blockIdx.x / groups;
  const int i0 = (blockIdx.x % groups) * R;
  const int b = bh / p.Hq;
  const int hk = (bh % p.Hq) / (p.Hq / p.Hk);
  const int rows = min(R, p.query_blocks - i0);
  for (int x = threadIdx.x; x < D * R; x += kSelectThreads) {
    const int r = x / D, d = x % D;
    qs[d * R + r] =
        r < rows ? p.q_sums[(static_cast<int64_t>(bh) * p.query_blocks + i0 + r) * D + d] : 0.0;
  }
  __syncthreads();
  const int key_len = visible_keys(p, b);
  const int64_t kv = static_cast<int64_t>(b) * p.Hk + hk;
  for (int j = threadIdx.x; j < p.key_blocks; j += kSelectThreads) {
    const int n = min(kKeyBlock, key_len - j * kKeyBlock);
    double acc[R];
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r] = 0.0;
    double factor = 0.0;
    if (n > 0) {
      const uint4* ks = reinterpret_cast<const uint4*>(p.k_sums + (kv * p.key_blocks + j) * D);
#pragma unroll 2
      for (int d = 0; d < D; d += 8) {
        const uint4 v = ks[d / 8];
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const int s = static_cast<int16_t>(c & 1 ? w[c / 2] >> 16 : w[c / 2] & 0xffffu);
          const double kd = static_cast<double>(s);
#pragma unroll
          for (int r = 0; r < R; ++r) acc[r] = fma(qs[(d + c) * R + r], kd, acc[r]);
        }
      }
      factor = static_cast<double>(__ldg(p.k_scale + kv * p.key_blocks + j)) / n;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      uint64_t key = 0;
      if (n > 0 && r < rows) {
        const int pol = p.policy == nullptr
            ? 0
            : p.policy[static_cast<int64_t>(p.policy_rows == 1 ? 0 : i0 + r) * p.key_blocks + j];
        key = pol < 0 ? 0ull : (pol > 0 ? ~0ull : sort_key(acc[r] * factor));
      }
      keys[static_cast<int64_t>(r) * p.key_blocks + j] = key;
    }
  }
  __syncthreads();
  const int r = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (r >= rows) return;
  const uint64_t* row = keys + static_cast<int64_t>(r) * p.key_blocks;
  // The largest threshold that at least `keep` keys reach, from the top bit.
  uint64_t edge = 0;
  bool exact = false;  // exactly `keep` keys reach it
  for (int bit = 63; bit >= 0 && !exact; --bit) {
    const uint64_t cand = edge | (1ull << bit);
    int n = 0;
    for (int j = lane; j < p.key_blocks; j += 32) n += row[j] >= cand ? 1 : 0;
    n = __reduce_add_sync(0xffffffffu, n);
    if (n >= p.keep) edge = cand;
    exact = n == p.keep;
  }
  int left = p.keep;  // equals of the edge that fit
  if (edge == 0) {    // fewer than `keep` blocks can be chosen: all of them
    edge = 1;
  } else if (!exact) {
    int above = 0;
    for (int j = lane; j < p.key_blocks; j += 32) above += row[j] > edge ? 1 : 0;
    left = p.keep - __reduce_add_sync(0xffffffffu, above);
  }
  int32_t* out = p.out + (static_cast<int64_t>(bh) * p.query_blocks + i0 + r) * p.keep;
  const uint32_t before = (1u << lane) - 1u;
  int count = 0;
  for (int j0 = 0; j0 < p.key_blocks; j0 += 32) {
    const int j = j0 + lane;
    const uint64_t key = j < p.key_blocks ? row[j] : 0ull;
    const bool equal = key == edge;
    const uint32_t equals = __ballot_sync(0xffffffffu, equal);
    const bool take = key > edge || (equal && __popc(equals & before) < left);
    const uint32_t taken = __ballot_sync(0xffffffffu, take);
    if (take) out[count + __popc(taken & before)] = j;
    count += __popc(taken);
    left -= min(left, __popc(equals));
  }
  for (int j = count + lane; j < p.keep; j += 32) out[j] = -1;
}

size_t select_smem_bytes(int rows, int64_t D, int64_t key_blocks) {
  return static_cast<size_t>(rows) * (D + key_blocks) * 8;
}

struct SelectWorkspace {
  int64_t q_bytes, k_bytes;
};
SelectWorkspace select_workspace(int64_t B, int64_t Hq, int64_t Hk, int64_t Lq, int64_t Lk,
                                 int64_t D) {
  const int64_t qb = (Lq + kQueryBlock - 1) / kQueryBlock;
  const int64_t kb = (Lk + kKeyBlock - 1) / kKeyBlock;
  return {B * Hq * qb * D * 8, B * Hk * kb * D * 2};
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

template <int D, int R>
void select_launch(const SelectParams& p, cudaStream_t stream) {
  const size_t smem = select_smem_bytes(R, D, p.key_blocks);
  auto kern = block_select_kernel<D, R>;
  TB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(smem)));
  const unsigned grid =
      static_cast<unsigned>(p.B) * p.Hq * ((p.query_blocks + R - 1) / R);
  kern<<<grid, kSelectThreads, smem, stream>>>(p);
  TB_CUDA_CHECK(cudaGetLastError());
}

template <int D>
void run_select(const SelectParams& p, cudaStream_t stream) {
  const int64_t tasks = static_cast<int64_t>(p.B) * p.Hk * p.key_blocks +
                        static_cast<int64_t>(p.B) * p.Hq * p.query_blocks;
  constexpr int kPerCta = kSumThreads / 32;
  block_sums_kernel<D><<<static_cast<unsigned>((tasks + kPerCta - 1) / kPerCta), kSumThreads, 0,
                         stream>>>(p);
  TB_CUDA_CHECK(cudaGetLastError());
  // As many query blocks per CTA as two CTAs per SM leave room for.
  const size_t room = 100 * 1024;
  if (select_smem_bytes(8, D, p.key_blocks) <= room) select_launch<D, 8>(p, stream);
  else if (select_smem_bytes(4, D, p.key_blocks) <= room) select_launch<D, 4>(p, stream);
  else select_launch<D, 1>(p, stream);
}

}  // namespace
}  // namespace tb

using tb::guarded;

extern "C" int tb_select_key_blocks_workspace(int64_t B, int64_t Hq, int64_t Hk, int64_t Lq,
                                              int64_t Lk, int64_t D, int64_t* bytes) {
  return guarded([&] {
    TB_REQUIRE(bytes != nullptr, "the workspace size needs a place");
    tb::check_select(B, Hq, Hk, Lq, Lk, D);
    const tb::SelectWorkspace w = tb::select_workspace(B, Hq, Hk, Lq, Lk, D);
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
    const SelectWorkspace w = select_workspace(B, Hq, Hk, Lq, Lk, D);
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
    p.q_sums = static_cast<double*>(workspace);
    p.k_sums = reinterpret_cast<int16_t*>(static_cast<unsigned char*>(workspace) + w.q_bytes);
    p.out = block_index;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (D == 128) run_select<128>(p, s);
    else run_select<64>(p, s);
  });
}
