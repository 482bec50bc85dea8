// Block-sparse Sage INT8 attention for sm_100a (tcgen05 + TMA + TMEM).
//
// Each block of 128 query rows attends to the key blocks (64 keys, one k_scale
// block) that its list names; with L the listed keys below key_lengths[b],
//   S_int = Q8 . K8^T                      (exact INT32, tensor core kind::i8)
//   s     = S_int * (sm_scale * log2 e * q_scale[row / 16] * k_scale[key / 64])
//   p = 2^(s - m), d = sum_L p, O = sum_L p V, out = O / d, lse = ln sum_L e^..
// with the running reference m of one pass over the list (moved, and O and d
// rescaled, only when a row's max grows far beyond it).  A row that
// sees no key gives 0 and lse = -inf.  S, m, d and O are INT32 / fp32; p is
// rounded to V's 16-bit type for the second contraction, the operand type that the
// tensor core takes (up to half a step, 2^-8 bf16 and 2^-11 fp16 relative, in fp16
// at least 2^-25), while d sums the unrounded p.  The errors of a row's keys average,
// to about the size of the output's own rounding: in all 0.0023 relative in bf16 and
// 0.00029 in fp16, 0.0017 and 0.00021 with p in fp32.  s - m is one FMA of the exact
// integer score with a factor of three fp32 roundings: off by |s| times some 2^-24.
//
// Lists of neighbouring query blocks differ, so nothing is shared between query
// tiles: a CTA takes one query block (128 rows x one head) and two CTAs share
// an SM (113 KB of shared memory, 256 TMEM columns, 192 threads each), one's
// barrier waits and tile ends filled by the other:
//   warps 0-3  softmax, one query row per thread (TMEM lane quadrant = warp);
//   warp 4     TMA producer: Q once, then K (8 KB) and V (16 KB) of the listed
//              blocks into two 4-stage rings (128B swizzle): K is read two
//              blocks before V, so one ring for both would hold a slot for
//              three blocks and leave one to hide the loads' latency;
//   warp 5     MMA issuer: S = Q K_j^T into one of two S buffers, O += P V_j.
// TMEM columns: O [0, 128), S(b) at 128 + 64 b; P(j) overwrites the first 32
// columns of its S buffer.  While the softmax turns S(j) into P, the tensor
// core computes S(j + 1).
//
// The softmax is bound by the latency of its own steps: of 1440 clocks a block
// and warp (one CTA per SM) the exponentials took 770 (their unit needs 512); with
// two CTAs an SM finishes a block every 868 clocks (75600 tokens x 40 heads, 128
// blocks a list: 10.6 ms, 1.2 PFLOP/s).
// So what can overlap them does: the second half of S loads under the first
// half's exponentials and the first half of the next block's S while P is stored,
// the producer follows the list and fetches the K scales, the issuer has looked
// at the rings before P comes, and everything rare is out of the way.  Taking an
// eighth or a quarter of the exponentials off their unit by a polynomial costs more
// issue slots than it frees (32760 tokens x 40 heads, 64 blocks a list: 2.17 ms,
// 2.25 and 2.35 with it; medians of three).
//
// Few query blocks (single tokens): the list is split over CTAs, which write
// unnormalized O, m and d; sparse_combine_kernel joins them.
//
// List entries that name no block with visible keys (negative, or at or past
// the end) are skipped: the producer walks the list 32 entries at a time with a
// warp vote and leaves each block's K scale and visible keys in a ring of notes
// for the softmax; the count the prologue takes bounds all loops.  A block named
// twice counts twice.
#define TB_TRY_WAIT_NO_HINT 1
#include <algorithm>
#include <cmath>

#include "attn_common.cuh"
#include "tb_capi_internal.h"
#include "tb_tu.cuh"

namespace tb {
namespace {

constexpr int kRows = 128;   // query block
constexpr int kKeys = 64;    // key block
constexpr int kDim = 128;
constexpr int kStages = 4;
// Slot j % kNotes is written with K(j), which waits for S(j - 4), so for P(j - 6):
// the softmax has read the slot's last note, j - 8.
constexpr int kNotes = 8;
constexpr int kSoftmaxWarps = 4;
constexpr int kProducerWarp = 4;
constexpr int kMmaWarp = 5;
constexpr int kThreads = 192;
constexpr int kQuarter = kKeys / 4;
constexpr int kQBytes = kRows * kDim;
constexpr int kKBytes = kKeys * kDim;
constexpr int kVBytes = kKeys * kDim * 2;
constexpr int kDataBytes = kQBytes + kStages * (kKBytes + kVBytes);
constexpr uint32_t kTmemCols = 256;
constexpr uint32_t kSBase = 128;
constexpr int kCombineWarps = 4;

struct SparseParams {
  int Hq, Hk, Lq, Lk, groups;   // groups = Hq / Hk
  int query_blocks, keep, splits, chunk;
  int q_tiles_scale, k_tiles_scale;
  const float* q_scale;
  const float* k_scale;
  const int32_t* lists;         // [B, Hq, query_blocks, keep]
  const int32_t* key_lengths;   // [B] or null
  void* out;
  int64_t o_sb, o_sh, o_sl;
  float* lse;                   // [B, Hq, Lq] natural logarithm, or null
  float sm_scale_log2;
  float* part_o;                // [B * Hq * Lq, splits, kDim] when splits > 1
  float2* part_md;              // [B * Hq * Lq, splits] (m, d)
};

struct BlockNote {  // what the softmax has to know of a listed block
  float k_scale;
  int valid;        // visible keys, 1 .. 64
};

struct __align__(8) SparseBarriers {
  uint64_t q_full;
  uint64_t k_full[kStages], k_empty[kStages];
  uint64_t v_full[kStages], v_empty[kStages];
  uint64_t s_full[2];   // S buffer b computed
  uint64_t p_full[2];   // the 4 softmax warps stored P in buffer b
  uint64_t o_done;      // after each of the last two PVs
  uint64_t o_final;     // after the last PV
  uint64_t drain;
  BlockNote note[kNotes];
  uint32_t tmem_base;
  int abort_flag;
};
constexpr int kSmemBytes = kDataBytes + static_cast<int>(sizeof(SparseBarriers));
static_assert(2 * (kSmemBytes + 1024) <= 228 * 1024, "two CTAs must fit one SM");

// Walks the visible entries of a list slice, the warp together.
struct ListCursor {
  const int32_t* list;
  int n, visible, base, value;
  uint32_t mask;
  __device__ __forceinline__ ListCursor(const int32_t* l, int count, int visible_blocks)
      : list(l), n(count), visible(visible_blocks), base(-32), value(0), mask(0) {}
  __device__ __forceinline__ int next() {
    while (mask == 0 && base + 32 < n) {
      base += 32;
      const int i = base + static_cast<int>(lane_id());
      value = i < n ? __ldg(list + i) : -1;
      mask = __ballot_sync(0xffffffffu, static_cast<uint32_t>(value) <
                                            static_cast<uint32_t>(visible));
    }
    const int at = mask != 0 ? __ffs(static_cast<int>(mask)) - 1 : 0;
    mask &= mask - 1;
    const int v = __shfl_sync(0xffffffffu, value, at);
    // Always a block of the tensor, whatever the list holds by now.
    return static_cast<uint32_t>(v) < static_cast<uint32_t>(visible) ? v : 0;
  }
};

// How far (log2) a row's max may grow over the reference point before O and d
// are rescaled: p stays within V's 16-bit type and the sums within fp32.
template <typename TV>
__device__ constexpr float kGrowth = std::is_same<TV, __nv_bfloat16>::value ? 32.0f : 12.0f;

// p = 2^(s c - m) of the 16 scores in x; the packed pairs of V's type go to
// out[AT .. AT + 7] (which may be x's own first half).  `sum2` gathers the
// unrounded p.  MASKED zeroes keys >= valid.
template <typename TV, int AT, bool MASKED>
__device__ __forceinline__ void exp_scores(uint32_t (&x)[kQuarter], uint32_t (&out)[kQuarter],
                                           uint64_t c2, uint64_t nm2, int valid,
                                           uint64_t (&sum2)[2]) {
#pragma unroll
  for (int i = 0; i < kQuarter / 2; ++i) {
    uint64_t p2 = ex2_pair(f2_fma(score_pair_f32(x[2 * i], x[2 * i + 1]), c2, nm2));
    if (MASKED)
      p2 = f2_pack(2 * i < valid ? f2_lo(p2) : 0.0f, 2 * i + 1 < valid ? f2_hi(p2) : 0.0f);
    sum2[i & 1] = f2_add(sum2[i & 1], p2);
    out[AT + i] = pack_pair<TV>(p2);
  }
}

__device__ __forceinline__ int max_score(const uint32_t (&x)[kQuarter], int m) {
  int m2 = INT32_MIN;
#pragma unroll
  for (int i = 0; i < kQuarter; i += 4) {
    m = __vimax3_s32(m, static_cast<int>(x[i]), static_cast<int>(x[i + 1]));
    m2 = __vimax3_s32(m2, static_cast<int>(x[i + 2]), static_cast<int>(x[i + 3]));
  }
  return max(m, m2);
}

// Keeps uses of loaded registers behind the tmem_wait_ld before it.
__device__ __forceinline__ void after_wait(uint32_t (&r)[kQuarter]) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}

template <typename TV>
__global__ void __launch_bounds__(kThreads, 2)
    sparse_attn_kernel(const __grid_constant__ CUtensorMap tm_q,
                       const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const SparseParams p) {
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* k_smem = smem + kQBytes;
  unsigned char* v_smem = k_smem + kStages * kKBytes;
  SparseBarriers* bar = reinterpret_cast<SparseBarriers*>(smem + kDataBytes);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  const int split = blockIdx.x % p.splits;
  const int tile = blockIdx.x / p.splits;
  const int qb = tile % p.query_blocks;
  const int bh = tile / p.query_blocks;
  const int b = bh / p.Hq;
  const int h = bh % p.Hq;
  const int hk = h / p.groups;
  const int q0 = qb * kRows;
  const int key_len = p.key_lengths != nullptr ? max(0, min(__ldg(p.key_lengths + b), p.Lk)) : p.Lk;
  const int visible = (key_len + kKeys - 1) / kKeys;
  const int32_t* list = p.lists + (static_cast<int64_t>(bh) * p.query_blocks + qb) * p.keep +
                        static_cast<int64_t>(split) * p.chunk;
  const int n_list = min(p.chunk, p.keep - split * p.chunk);

  if (threadIdx.x == 0) {
    mbar_init(&bar->q_full, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bar->k_full[s], 1);
      mbar_init(&bar->k_empty[s], 1);
      mbar_init(&bar->v_full[s], 1);
      mbar_init(&bar->v_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->s_full[i], 1);
      mbar_init(&bar->p_full[i], kSoftmaxWarps);
    }
    mbar_init(&bar->o_done, 1);
    mbar_init(&bar->o_final, 1);
    mbar_init(&bar->drain, 1);
    bar->abort_flag = 0;
    fence_barrier_init();
    // The swizzle atoms need 1024-byte aligned tiles (the array asks for it).
    if ((smem_u32(smem) & 1023u) != 0) {
      record_device_error(kDevBadLaunch);
      bar->abort_flag = 1;
    }
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&bar->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  int n_kv = 0;
  for (int i = 0; i < n_list; i += kThreads) {
    const int at = i + static_cast<int>(threadIdx.x);
    n_kv += __syncthreads_count(at < n_list && static_cast<uint32_t>(__ldg(list + at)) <
                                                   static_cast<uint32_t>(visible));
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar->tmem_base;
  volatile int* abort_flag = &bar->abort_flag;
  if (*abort_flag) n_kv = 0;

  if (warp == kProducerWarp) {
    // ------------------------------------------------------------ producer
    if (n_kv > 0) {
      if (lane == 0) {
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
        mbar_arrive_expect_tx(&bar->q_full, kQBytes);
        tma_load_4d(smem, &tm_q, &bar->q_full, 0, q0, h, b);
      }
      ListCursor cur(list, n_list, visible);
      const float* ks_row = p.k_scale + static_cast<int64_t>(b * p.Hk + hk) * p.k_tiles_scale;
      auto load_k = [&](int j, int blk) {
        const int s = j % kStages;
        if (!mbar_wait(&bar->k_empty[s], (static_cast<uint32_t>(j / kStages) & 1u) ^ 1u,
                       abort_flag, kDevWaitTimeoutProducer))
          return false;
        bar->note[j % kNotes] = {__ldg(ks_row + blk), min(kKeys, key_len - blk * kKeys)};
        mbar_arrive_expect_tx(&bar->k_full[s], kKBytes);  // releases the note
        tma_load_4d(k_smem + s * kKBytes, &tm_k, &bar->k_full[s], 0, blk * kKeys, hk, b);
        return true;
      };
      auto load_v = [&](int j, int blk) {
        const int s = j % kStages;
        if (!mbar_wait(&bar->v_empty[s], (static_cast<uint32_t>(j / kStages) & 1u) ^ 1u,
                       abort_flag, kDevWaitTimeoutProducer))
          return false;
        mbar_arrive_expect_tx(&bar->v_full[s], kVBytes);
#pragma unroll
        for (int dh = 0; dh < kDim / 64; ++dh)
          tma_load_4d(v_smem + s * kVBytes + dh * (kKeys * 128), &tm_v, &bar->v_full[s], dh * 64,
                      blk * kKeys, hk, b);
        return true;
      };
      // K runs two blocks ahead of V, as S does of PV.
      int blk0 = 0, blk1 = 0, blk2 = 0, k_issued = 0, v_issued = 0;
      for (int j = -2; j < n_kv; ++j) {
        blk0 = blk1;
        blk1 = blk2;
        bool ok = true;
        if (j + 2 < n_kv) {
          blk2 = cur.next();
          if (lane == 0) ok = load_k(j + 2, blk2);
          k_issued += ok;
        }
        if (j >= 0 && lane == 0 && ok) {
          ok = load_v(j, blk0);
          v_issued += ok;
        }
        if (!__shfl_sync(0xffffffffu, static_cast<int>(ok), 0)) break;
      }
      if (lane == 0) {
        // Every copy issued by this CTA lands before it exits.
        drain_wait(&bar->q_full, 0);
        for (int i = max(0, k_issued - kStages); i < k_issued; ++i)
          drain_wait(&bar->k_full[i % kStages], static_cast<uint32_t>(i / kStages) & 1u);
        for (int i = max(0, v_issued - kStages); i < v_issued; ++i)
          drain_wait(&bar->v_full[i % kStages], static_cast<uint32_t>(i / kStages) & 1u);
      }
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------ MMA issuer
    if (n_kv > 0) {
      const uint32_t elected = elect_one();
      constexpr uint32_t idesc_qk = idesc_i8(kRows, kKeys);
      constexpr uint32_t idesc_pv = idesc_f16(
          kRows, kDim, std::is_same<TV, __nv_bfloat16>::value, /*b_mn_major=*/true);
      const uint32_t k_addr = smem_u32(k_smem), v_addr = smem_u32(v_smem);
      const uint64_t q_desc = umma_desc_sw128(smem_u32(smem));
      auto issue_s = [&](int j) {
        const uint32_t d_tmem = tmem + kSBase + static_cast<uint32_t>(j & 1) * kKeys;
        const uint64_t bk = umma_desc_sw128(k_addr + (j % kStages) * kKBytes);
#pragma unroll
        for (int kk = 0; kk < kDim / 32; ++kk)
          mma_i8_ss_warp(d_tmem, q_desc + 2u * kk, bk + 2u * kk, idesc_qk, kk > 0 ? 1u : 0u,
                         elected);
      };
      auto warp_wait = [&](uint64_t* b, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(b, parity, abort_flag, kDevWaitTimeoutMma)) != 0;
      };
      auto wait_ring = [&](uint64_t* full, int j) {
        return warp_wait(&full[j % kStages], static_cast<uint32_t>(j / kStages) & 1u);
      };
      bool ok = warp_wait(&bar->q_full, 0);
      for (int j = 0; j < 2 && j < n_kv && ok; ++j) {
        ok = wait_ring(bar->k_full, j);
        if (ok) {
          tc_fence_after();
          issue_s(j);
          mma_commit_warp(&bar->s_full[j & 1], elected);
          mma_commit_warp(&bar->k_empty[j % kStages], elected);
        }
      }
      // All waits of a block first, then PV(j) and S(j + 2) back to back, then
      // the commits.  The s_full commit of S(j + 2) also says that PV(j) is
      // done; o_done marks the last two PVs, which no S commit follows.
      for (int j = 0; j < n_kv && ok; ++j) {
        const bool next_s = j + 2 < n_kv;
        ok = wait_ring(bar->v_full, j) && (!next_s || wait_ring(bar->k_full, j + 2)) &&
             warp_wait(&bar->p_full[j & 1], static_cast<uint32_t>(j >> 1) & 1u);
        if (!ok) break;
        tc_fence_after();
        const uint32_t v_tile = v_addr + (j % kStages) * kVBytes;
        const uint32_t p_tmem = tmem + kSBase + static_cast<uint32_t>(j & 1) * kKeys;
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk) {
          const uint64_t bv = umma_desc_sw128_mn(v_tile + kk * 2048, kKeys * 128, 1024);
          mma_f16_ts_warp(tmem, p_tmem + static_cast<uint32_t>(kk * 8), bv, idesc_pv,
                          (j > 0 || kk > 0) ? 1u : 0u, elected);
        }
        if (next_s) {
          issue_s(j + 2);
          mma_commit_warp(&bar->s_full[j & 1], elected);
          mma_commit_warp(&bar->k_empty[(j + 2) % kStages], elected);
        } else {
          mma_commit_warp(&bar->o_done, elected);
        }
        mma_commit_warp(&bar->v_empty[j % kStages], elected);
        if (j + 1 == n_kv) mma_commit_warp(&bar->o_final, elected);
      }
      mma_commit_warp(&bar->drain, elected);
      if (lane == 0) drain_wait(&bar->drain, 0);
      __syncwarp();
    }
  } else if (warp < kSoftmaxWarps) {
    // ------------------------------------------------------------ softmax
    const int row = q0 + warp * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t s_tmem0 = tmem + lane_off + kSBase;
    const uint32_t o_tmem = tmem + lane_off;
    const float cq = row < p.Lq ? p.sm_scale_log2 * __ldg(p.q_scale + static_cast<int64_t>(bh) *
                                                              p.q_tiles_scale + row / 16)
                                : 0.0f;
    float m_ref = -INFINITY;  // exponent reference point
    float dsum = 0.0f;
    bool ok = n_kv > 0;
    // The usual path takes the largest integer for the largest score: not so where a
    // factor is negative.
    const bool rising = !__any_sync(0xffffffffu, cq < 0.0f);
    bool primed = false;  // every row of the warp has a reference point
    bool loaded = false;  // keys 0-31 of this block's S and its note were fetched by the last one
    BlockNote note{0.0f, kKeys};
    // One block: keys 0-31 in (l1, l2), 32-63 in (h1, h2), 16 each.  Their packed
    // P stays in l1 and h1, so h2 and l2 are free for keys 0-31 of the next block,
    // whose call therefore gets (h2, l2, h1, l1).  The usual path has no branch
    // but the loop's and the one of the vote; the rest is kept out of its way.
    auto block = [&](int j, uint32_t(&l1)[kQuarter], uint32_t(&l2)[kQuarter],
                     uint32_t(&h1)[kQuarter], uint32_t(&h2)[kQuarter]) {
      const uint32_t s_tmem = s_tmem0 + static_cast<uint32_t>(j & 1) * kKeys;
      if (__builtin_expect(!loaded, 0)) {
        ok = __all_sync(0xffffffffu,
                        mbar_wait(&bar->s_full[j & 1], static_cast<uint32_t>(j >> 1) & 1u,
                                  abort_flag, kDevWaitTimeoutSoftmax));
        if (!ok) return;
        tc_fence_after();
        tmem_ld16(s_tmem, l1);
        tmem_ld16(s_tmem + 16, l2);
        note = bar->note[j % kNotes];
      }
      tmem_wait_ld();
      after_wait(l1);
      after_wait(l2);
      tmem_ld16(s_tmem + 32, h1);
      tmem_ld16(s_tmem + 48, h2);
      const int valid = note.valid;
      const float c = cq * note.k_scale;
      const uint64_t c2 = f2_pack(c, c);
      const bool more = j + 1 < n_kv;
      uint64_t sum2[2] = {0ull, 0ull};
      bool done = false;
      loaded = false;
      if (__builtin_expect(primed && valid == kKeys && note.k_scale >= 0.0f, 1)) {
        // The reference stands, so the exponentials need not wait for the row
        // max; if it moved past, the block is read again below.
        const uint64_t nm2 = f2_pack(-m_ref, -m_ref);
        const int mx_low = max_score(l2, max_score(l1, INT32_MIN));
        exp_scores<TV, 0, false>(l1, l1, c2, nm2, kKeys, sum2);
        exp_scores<TV, 8, false>(l2, l1, c2, nm2, kKeys, sum2);
        tmem_wait_ld();
        after_wait(h1);
        after_wait(h2);
        // Both votes are taken under exponentials that do not wait for them.
        const int mx = max_score(h2, max_score(h1, mx_low));
        const bool past = __any_sync(0xffffffffu, i2f_exact(mx) * c > m_ref + kGrowth<TV>);
        exp_scores<TV, 0, false>(h1, h1, c2, nm2, kKeys, sum2);
        // S(j + 1) was issued when P(j - 1) came: not sooner than here is it there.
        asm volatile("" : "+l"(sum2[0]));
        const uint32_t next_s = static_cast<uint32_t>(j + 1) & 1u;
        const bool ready = mbar_try_wait(smem_u32(&bar->s_full[next_s]),
                                         static_cast<uint32_t>((j + 1) >> 1) & 1u);
        exp_scores<TV, 8, false>(h2, h1, c2, nm2, kKeys, sum2);
        done = !past;
        loaded = done && more && __all_sync(0xffffffffu, ready);
        if (__builtin_expect(loaded, 1)) {
          tc_fence_after();
          tmem_ld16(s_tmem0 + next_s * kKeys, h2);
          tmem_ld16(s_tmem0 + next_s * kKeys + 16, l2);
          note = bar->note[(j + 1) % kNotes];
        }
      }
      if (__builtin_expect(!done, 0)) {
        // The first block, a partly visible one, one that moves the reference
        // point of some row, or one under a negative scale: the row max first.
        tmem_wait_ld();
        after_wait(h1);
        after_wait(h2);
        tmem_ld16(s_tmem, l1);
        tmem_ld16(s_tmem + 16, l2);
        tmem_ld16(s_tmem + 32, h1);
        tmem_ld16(s_tmem + 48, h2);
        tmem_wait_ld();
        after_wait(l1);
        after_wait(l2);
        after_wait(h1);
        after_wait(h2);
        // Under a negative factor the smallest integer is the largest score (both ends
        // taken here: 131 us as before for 3 x 4111 queries, 20 heads, 19 blocks; a
        // branch for negative factors 137).
        const int some = static_cast<int>(l1[0]);  // a visible key's
        int mx = some, mn = some;
#pragma unroll
        for (int i = 0; i < kQuarter; ++i) {
          const int a = i < valid ? static_cast<int>(l1[i]) : some;
          const int b = i + 16 < valid ? static_cast<int>(l2[i]) : some;
          const int d = i + 32 < valid ? static_cast<int>(h1[i]) : some;
          const int e = i + 48 < valid ? static_cast<int>(h2[i]) : some;
          mx = __vimax3_s32(__vimax3_s32(mx, a, b), d, e);
          mn = __vimin3_s32(__vimin3_s32(mn, a, b), d, e);
        }
        const float m_blk = fmaxf(i2f_exact(mx) * c, i2f_exact(mn) * c);
        const bool move = m_blk > m_ref + kGrowth<TV>;
        const bool rescale = move && m_ref != -INFINITY;
        const float f = rescale ? ex2(m_ref - m_blk) : 1.0f;
        dsum *= f;
        if (move) m_ref = m_blk;
        primed = rising && __all_sync(0xffffffffu, m_ref != -INFINITY);
        const float nm = m_ref == -INFINITY ? 0.0f : -m_ref;
        sum2[0] = sum2[1] = 0ull;
        exp_scores<TV, 0, true>(l1, l1, c2, f2_pack(nm, nm), valid, sum2);
        exp_scores<TV, 8, true>(l2, l1, c2, f2_pack(nm, nm), valid - 16, sum2);
        exp_scores<TV, 0, true>(h1, h1, c2, f2_pack(nm, nm), valid - 32, sum2);
        exp_scores<TV, 8, true>(h2, h1, c2, f2_pack(nm, nm), valid - 48, sum2);
        if (valid < kKeys && key_len < p.Lk) {
          // V rows past key_lengths hold whatever the padding holds; a NaN there
          // times p = 0 would still be NaN, so the rows are cleared.
          ok = __all_sync(0xffffffffu,
                          mbar_wait(&bar->v_full[j % kStages],
                                    static_cast<uint32_t>(j / kStages) & 1u, abort_flag,
                                    kDevWaitTimeoutSoftmax));
          if (!ok) return;
          unsigned char* vt = v_smem + (j % kStages) * kVBytes;
          for (int i = threadIdx.x; i < (kKeys - valid) * 16; i += kSoftmaxWarps * 32)
            *reinterpret_cast<uint4*>(vt + (i & 8 ? kKeys * 128 : 0) + (valid + (i >> 4)) * 128 +
                                      (i & 7) * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
        }
        if (__any_sync(0xffffffffu, rescale)) {
          // O holds PV(0 .. j-1) once the commit after PV(j - 1) arrived; PV(j)
          // waits for this warp's p_full arrival below.
          const bool waited =
              more
                  ? mbar_wait(&bar->s_full[(j + 1) & 1], static_cast<uint32_t>((j + 1) >> 1) & 1u,
                              abort_flag, kDevWaitTimeoutSoftmax)
                  : mbar_wait(&bar->o_done, 0u, abort_flag, kDevWaitTimeoutSoftmax);
          ok = __all_sync(0xffffffffu, waited);
          if (!ok) return;
          tc_fence_after();
#pragma unroll 1
          for (int cc = 0; cc < kDim / 16; ++cc) {
            uint32_t o[16];
            tmem_ld16(o_tmem + cc * 16, o);
            tmem_wait_ld();
            after_wait(o);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st16(o_tmem + cc * 16, o);
          }
        }
      }
      tmem_st16(s_tmem, l1);
      tmem_st16(s_tmem + 16, h1);
      const uint64_t s01 = f2_add(sum2[0], sum2[1]);
      dsum += f2_lo(s01) + f2_hi(s01);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->p_full[j & 1]);
    };
    uint32_t r0[kQuarter], r1[kQuarter], r2[kQuarter], r3[kQuarter];
    for (int j = 0; j < n_kv && ok; j += 2) {
      block(j, r0, r1, r2, r3);
      if (ok && j + 1 < n_kv) block(j + 1, r3, r1, r2, r0);
    }
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&bar->o_final, 0u, abort_flag,
                                                   kDevWaitTimeoutSoftmax));
    if (ok || n_kv == 0) {
      tc_fence_after();
      const float inv = dsum > 0.0f ? 1.0f / dsum : (dsum == 0.0f ? 0.0f : dsum);
      const int64_t flat = static_cast<int64_t>(bh) * p.Lq + row;
      TV* orow = static_cast<TV*>(p.out) + b * p.o_sb + h * p.o_sh +
                 static_cast<int64_t>(row) * p.o_sl;
      float* prow = p.splits > 1 ? p.part_o + (flat * p.splits + split) * kDim : nullptr;
#pragma unroll 1
      for (int cc = 0; cc < kDim / 16; ++cc) {
        uint32_t o[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = 0u;
        if (n_kv > 0) {
          tmem_ld16(o_tmem + cc * 16, o);
          tmem_wait_ld();
        }
        if (row < p.Lq) {
          if (prow != nullptr) {
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              *reinterpret_cast<uint4*>(prow + cc * 16 + i) =
                  make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          } else {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
              w[i] =
                  pack2<TV>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
            *reinterpret_cast<uint4*>(orow + cc * 16) = make_uint4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<uint4*>(orow + cc * 16 + 8) = make_uint4(w[4], w[5], w[6], w[7]);
          }
        }
        __syncwarp();
      }
      if (row < p.Lq) {
        if (p.splits > 1) p.part_md[flat * p.splits + split] = make_float2(m_ref, dsum);
        else if (p.lse != nullptr)
          p.lse[flat] = dsum == 0.0f ? -INFINITY : (m_ref + log2f(dsum)) * 0.6931471805599453f;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the partial results of a split list: one warp per row, four channels
// per lane; O = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) d_s.  Lane s holds the
// m and d of part s (32 at a time), so the loads of one row do not wait for one
// another.
template <typename TV>
__global__ void __launch_bounds__(kCombineWarps * 32) sparse_combine_kernel(const SparseParams p,
                                                                            int64_t rows) {
  const int64_t flat = static_cast<int64_t>(blockIdx.x) * kCombineWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (flat >= rows) return;
  const float2* md = p.part_md + flat * p.splits;
  const float* part = p.part_o + flat * p.splits * kDim + lane * 4;
  float M = -INFINITY;
  for (int s = lane; s < p.splits; s += 32) {
    const float2 t = md[s];
    if (t.y != 0.0f) M = fmaxf(M, t.x);
  }
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, m));
  float d = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int s0 = 0; s0 < p.splits; s0 += 32) {
    const int n = min(32, p.splits - s0);
    const float2 mine = lane < n ? md[s0 + lane] : make_float2(0.0f, 0.0f);
    // d = 0: saw no key.  m = -inf with d != 0: every score of the part was NaN.
    const float w = mine.y == 0.0f ? 0.0f : (mine.x == -INFINITY ? 1.0f : ex2(mine.x - M));
#pragma unroll 8
    for (int s = 0; s < n; ++s) {
      const float ws = __shfl_sync(0xffffffffu, w, s);
      const float ds = __shfl_sync(0xffffffffu, mine.y, s);
      const float4 q = *reinterpret_cast<const float4*>(part + (s0 + s) * kDim);
      if (ds != 0.0f) {
        d = fmaf(ws, ds, d);
        o.x = fmaf(ws, q.x, o.x);
        o.y = fmaf(ws, q.y, o.y);
        o.z = fmaf(ws, q.z, o.z);
        o.w = fmaf(ws, q.w, o.w);
      }
    }
  }
  const float inv = d > 0.0f ? 1.0f / d : (d == 0.0f ? 0.0f : d);
  const int bh = static_cast<int>(flat / p.Lq);
  const int64_t row = flat - static_cast<int64_t>(bh) * p.Lq;
  TV* out = static_cast<TV*>(p.out) + (bh / p.Hq) * p.o_sb + (bh % p.Hq) * p.o_sh + row * p.o_sl +
            lane * 4;
  *reinterpret_cast<uint2*>(out) =
      make_uint2(pack2<TV>(o.x * inv, o.y * inv), pack2<TV>(o.z * inv, o.w * inv));
  if (p.lse != nullptr && lane == 0)
    p.lse[flat] = d == 0.0f ? -INFINITY : (M + log2f(d)) * 0.6931471805599453f;
}

// lse += sm_scale * q_scale * (Q8 . mean) of each row: the part of every score that
// K smoothing took off (the scores of the codes are those against K - mean).  Eight
// lanes a row, 16 channels each, whose means stay in registers over 16 rows; the
// products are exact in fp32.  Bound by the latency of its loads and shuffles:
// 75600 queries x 40 heads 137 us (3.0 TB/s; four rows in flight, for which fewer
// warps fit, 148).
constexpr int kShiftThreads = 256;
constexpr int kShiftLanes = kDim / 16;
constexpr int kShiftStep = kShiftThreads / kShiftLanes;  // rows of a CTA at a time
constexpr int kShiftRows = 16 * kShiftStep;

// Byte i of x plus 128, minus 128, as a float: exact, and off the conversion unit.
// x: the four codes with their sign bits turned.
__device__ __forceinline__ float code_f32(uint32_t x, int i) {
  return __uint_as_float(__byte_perm(x, 0x4b000000u, 0x7440 + i)) - 8388736.0f;
}

template <typename TM>
__global__ void __launch_bounds__(kShiftThreads, 5)
    smoothed_lse_kernel(const int8_t* q, int64_t q_sb, int64_t q_sh, int64_t q_sl,
                        const float* q_scale, const TM* mean, float* lse, int chunks, int Hq,
                        int Lq, int groups, int q_tiles_scale, float sm_scale) {
  const int bh = static_cast<int>(blockIdx.x) / chunks;
  // Unsigned: rows past the last one are counted past 2^31 in the longest sequences.
  const uint32_t row0 =
      blockIdx.x % static_cast<uint32_t>(chunks) * kShiftRows + threadIdx.x / kShiftLanes;
  const int part = threadIdx.x % kShiftLanes;
  const int b = bh / Hq, h = bh % Hq;
  const uint4* m = reinterpret_cast<const uint4*>(
      mean + static_cast<int64_t>(b * (Hq / groups) + h / groups) * kDim + part * 16);
  const uint4 m0 = __ldg(m), m1 = __ldg(m + 1);
  const uint32_t mw[8] = {m0.x, m0.y, m0.z, m0.w, m1.x, m1.y, m1.z, m1.w};
  float mv[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (std::is_same<TM, __nv_bfloat16>::value) {
      mv[2 * i] = __uint_as_float(mw[i] << 16);
      mv[2 * i + 1] = __uint_as_float(mw[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&mw[i]));
      mv[2 * i] = f.x;
      mv[2 * i + 1] = f.y;
    }
  }
  const int8_t* src = q + b * q_sb + h * q_sh + part * 16;
  const float* scales = q_scale + static_cast<int64_t>(bh) * q_tiles_scale;
  float* out = lse + static_cast<int64_t>(bh) * Lq;
  constexpr int kFly = 2;  // rows in flight
#pragma unroll 1
  for (uint32_t r0 = row0; r0 < row0 + kShiftRows; r0 += kFly * kShiftStep) {
    uint4 x[kFly];
    float scale[kFly], old[kFly];
#pragma unroll
    for (int u = 0; u < kFly; ++u) {
      const uint32_t r = r0 + u * kShiftStep;
      x[u] = make_uint4(0u, 0u, 0u, 0u);
      scale[u] = old[u] = 0.0f;
      if (r < static_cast<uint32_t>(Lq)) {
        x[u] = *reinterpret_cast<const uint4*>(src + r * q_sl);
        scale[u] = __ldg(scales + r / 16);
        old[u] = out[r];
      }
    }
#pragma unroll
    for (int u = 0; u < kFly; ++u) {
      const uint32_t w[4] = {x[u].x ^ 0x80808080u, x[u].y ^ 0x80808080u, x[u].z ^ 0x80808080u,
                             x[u].w ^ 0x80808080u};
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) sum = fmaf(code_f32(w[i / 4], i & 3), mv[i], sum);
#pragma unroll
      for (int i = kShiftLanes / 2; i > 0; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
      const uint32_t r = r0 + u * kShiftStep;
      // A row that saw no key stays -inf.
      if (part == 0 && r < static_cast<uint32_t>(Lq) && old[u] != -INFINITY)
        out[r] = fmaf(sm_scale * scale[u], sum, old[u]);
    }
  }
}

// CTAs that share one list: as many as fill two per SM, each with at least
// four blocks (one full ring).  With the join, one token of 32 heads, 64 blocks:
// 22.5 us, whole 52.4; 300 tokens of 8 heads, 16 blocks: 18.0 us, whole 19.7, at
// least two 21.8, at least eight 19.6.  Lists of up to eight stay whole: 14.0 us,
// in two 14.6.
int split_count(int64_t tiles, int64_t keep) {
  const int64_t slots = 2LL * device_sm_count();
  if (tiles >= slots || keep <= 8) return 1;
  const int64_t s = std::max<int64_t>(1, std::min(slots / tiles, (keep + 3) / 4));
  const int64_t chunk = (keep + s - 1) / s;
  return static_cast<int>((keep + chunk - 1) / chunk);
}

void check_geometry(int64_t B, int64_t Hq, int64_t Lq, int64_t keep) {
  TB_REQUIRE(B > 0 && Hq > 0 && Lq > 0, "empty Q/K sequences are not supported");
  TB_REQUIRE(keep > 0 && keep <= (1 << 24), "block_index must name 1 to 2^24 blocks a list");
  TB_REQUIRE(Lq <= INT32_MAX - 256, "sequence length exceeds the kernel range");
  TB_REQUIRE(B <= INT32_MAX / Hq && B * Hq <= INT32_MAX / ((Lq + kRows - 1) / kRows),
             "batch, heads and query blocks exceed the grid range");
}

}  // namespace
}  // namespace tb

using tb::guarded;

extern "C" int tb_sparse_attn_workspace(int64_t B, int64_t Hq, int64_t Lq, int64_t keep,
                                        int64_t* bytes) {
  return guarded([&] {
    TB_REQUIRE(bytes != nullptr, "the workspace size needs a place");
    tb::check_geometry(B, Hq, Lq, keep);
    tb::require_sm100();
    const int splits = tb::split_count(B * Hq * ((Lq + tb::kRows - 1) / tb::kRows), keep);
    *bytes = splits > 1 ? B * Hq * Lq * splits * (tb::kDim + 2) * 4 : 0;
  });
}

extern "C" int tb_sparse_attn(const int8_t* q, const int8_t* k, const void* v, int v_dtype,
                              void* out, const float* q_scale, const float* k_scale,
                              const int32_t* block_index, const int32_t* key_lengths, float* lse,
                              void* workspace, int64_t workspace_bytes, int64_t B, int64_t Hq,
                              int64_t Hk, int64_t Lq, int64_t Lk, int64_t D, int64_t keep,
                              const int64_t* strides, float sm_scale, tb_stream_t stream) {
  return guarded([&] {
    using namespace tb;
    TB_REQUIRE(q && k && v && out && q_scale && k_scale && block_index && strides,
               "query, key, value, output, scales and block_index must be CUDA tensors");
    TB_REQUIRE(D == kDim, "the sparse attention kernel takes head_dim 128 (pad smaller heads)");
    TB_REQUIRE(v_dtype == TB_DTYPE_BF16 || v_dtype == TB_DTYPE_F16,
               "value must be float16 or bfloat16");
    check_geometry(B, Hq, Lq, keep);
    TB_REQUIRE(Hk > 0 && Lk > 0, "empty Q/K sequences are not supported");
    TB_REQUIRE(Hq % Hk == 0, "num_qo_heads must be divisible by num_kv_heads");
    TB_REQUIRE(Lk <= INT32_MAX - 256, "sequence length exceeds the kernel range");
    TB_REQUIRE(std::isfinite(sm_scale), "sm_scale must be finite");
    for (int i = 0; i < 6; ++i)
      TB_REQUIRE(strides[i] % 16 == 0, "Q/K strides must be multiples of 16 bytes");
    for (int i = 6; i < 12; ++i)
      TB_REQUIRE(strides[i] % 8 == 0, "V/O strides must be multiples of 16 bytes");
    auto aligned = [](const void* ptr, uintptr_t a) {
      return (reinterpret_cast<uintptr_t>(ptr) & (a - 1)) == 0;
    };
    TB_REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 16),
               "Q/K/V/O must be 16-byte aligned");
    TB_REQUIRE(aligned(q_scale, 4) && aligned(k_scale, 4) && aligned(block_index, 4) &&
                   aligned(key_lengths, 4) && aligned(lse, 4),
               "scales, block_index, key_lengths and lse must be 4-byte aligned");
    require_sm100();
    const int64_t query_blocks = (Lq + kRows - 1) / kRows;
    const int64_t tiles = B * Hq * query_blocks;
    SparseParams p{};
    p.splits = split_count(tiles, keep);
    p.chunk = static_cast<int>((keep + p.splits - 1) / p.splits);
    if (p.splits > 1) {
      TB_REQUIRE(workspace != nullptr && aligned(workspace, 16) &&
                     workspace_bytes >= B * Hq * Lq * p.splits * (kDim + 2) * 4,
                 "the split sparse attention needs the workspace tb_sparse_attn_workspace names");
      TB_REQUIRE(tiles * p.splits <= INT32_MAX,
                 "batch, heads and query blocks exceed the grid range");
      p.part_o = static_cast<float*>(workspace);
      p.part_md = reinterpret_cast<float2*>(p.part_o + B * Hq * Lq * p.splits * kDim);
    }
    p.Hq = static_cast<int>(Hq);
    p.Hk = static_cast<int>(Hk);
    p.Lq = static_cast<int>(Lq);
    p.Lk = static_cast<int>(Lk);
    p.groups = static_cast<int>(Hq / Hk);
    p.query_blocks = static_cast<int>(query_blocks);
    p.keep = static_cast<int>(keep);
    p.q_tiles_scale = static_cast<int>((Lq + 63) / 64 * 4);
    p.k_tiles_scale = static_cast<int>((Lk + 63) / 64);
    p.q_scale = q_scale;
    p.k_scale = k_scale;
    p.lists = block_index;
    p.key_lengths = key_lengths;
    p.out = out;
    p.o_sb = strides[9];
    p.o_sh = strides[10];
    p.o_sl = strides[11];
    p.lse = lse;
    p.sm_scale_log2 = sm_scale * 1.4426950408889634f;
    CUtensorMap tq, tk, tv;
    make_map_4d(&tq, CU_TENSOR_MAP_DATA_TYPE_UINT8, q, D, Lq, Hq, B, strides[2], strides[1],
                strides[0], 1, kDim, kRows);
    make_map_4d(&tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, k, D, Lk, Hk, B, strides[5], strides[4],
                strides[3], 1, kDim, kKeys);
    make_map_4d(&tv,
                v_dtype == TB_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                         : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                v, D, Lk, Hk, B, strides[8], strides[7], strides[6], 2, 64, kKeys);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int64_t rows = B * Hq * Lq;
    auto launch = [&](auto kern, auto combine) {
      TB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         kSmemBytes));
      kern<<<static_cast<unsigned>(tiles * p.splits), kThreads, kSmemBytes, s>>>(tq, tk, tv, p);
      TB_CUDA_CHECK(cudaGetLastError());
      if (p.splits > 1) {
        combine<<<static_cast<unsigned>((rows + kCombineWarps - 1) / kCombineWarps),
                  kCombineWarps * 32, 0, s>>>(p, rows);
        TB_CUDA_CHECK(cudaGetLastError());
      }
    };
    if (v_dtype == TB_DTYPE_BF16)
      launch(sparse_attn_kernel<__nv_bfloat16>, sparse_combine_kernel<__nv_bfloat16>);
    else
      launch(sparse_attn_kernel<__half>, sparse_combine_kernel<__half>);
  });
}

extern "C" int tb_smoothed_lse(const int8_t* q, const float* q_scale, const void* key_mean,
                               int mean_dtype, float* lse, int64_t B, int64_t Hq, int64_t Hk,
                               int64_t Lq, int64_t D, const int64_t* strides, float sm_scale,
                               tb_stream_t stream) {
  return guarded([&] {
    using namespace tb;
    TB_REQUIRE(q && q_scale && key_mean && lse && strides,
               "query, its scales, key_mean and lse must be CUDA tensors");
    TB_REQUIRE(D == kDim, "the smoothed log-sum-exp takes head_dim 128 (pad smaller heads)");
    TB_REQUIRE(mean_dtype == TB_DTYPE_BF16 || mean_dtype == TB_DTYPE_F16,
               "key_mean must be float16 or bfloat16");
    check_geometry(B, Hq, Lq, 1);
    TB_REQUIRE(Hk > 0 && Hq % Hk == 0, "num_qo_heads must be divisible by num_kv_heads");
    TB_REQUIRE(std::isfinite(sm_scale), "sm_scale must be finite");
    auto aligned = [](const void* ptr, uintptr_t a) {
      return (reinterpret_cast<uintptr_t>(ptr) & (a - 1)) == 0;
    };
    TB_REQUIRE(aligned(q, 16) && aligned(key_mean, 16), "Q and key_mean must be 16-byte aligned");
    TB_REQUIRE(aligned(q_scale, 4) && aligned(lse, 4), "scales and lse must be 4-byte aligned");
    for (int i = 0; i < 3; ++i)
      TB_REQUIRE(strides[i] % 16 == 0, "Q strides must be multiples of 16 bytes");
    require_sm100();
    const int64_t chunks = (Lq + kShiftRows - 1) / kShiftRows;
    TB_REQUIRE(B * Hq * chunks <= INT32_MAX, "batch, heads and queries exceed the grid range");
    auto launch = [&](auto kern, auto* mean) {
      kern<<<static_cast<unsigned>(B * Hq * chunks), kShiftThreads, 0,
             static_cast<cudaStream_t>(stream)>>>(
          q, strides[0], strides[1], strides[2], q_scale, mean, lse, static_cast<int>(chunks),
          static_cast<int>(Hq), static_cast<int>(Lq), static_cast<int>(Hq / Hk),
          static_cast<int>((Lq + 63) / 64 * 4), sm_scale);
      TB_CUDA_CHECK(cudaGetLastError());
    };
    if (mean_dtype == TB_DTYPE_BF16)
      launch(smoothed_lse_kernel<__nv_bfloat16>, static_cast<const __nv_bfloat16*>(key_mean));
    else launch(smoothed_lse_kernel<__half>, static_cast<const __half*>(key_mean));
  });
}
