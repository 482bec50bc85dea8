// Rotary positions: applied to Q and K, or written as the 2x2 rotation matrices
// that the fused Q/K prologue reads.
//
//   angle(t, p) = position[t, axis(p)] * inv_freq[p]       for each channel pair p
//   y[c0] = scale * (x[c0] cos - x[c1] sin)
//   y[c1] = scale * (x[c1] cos + x[c0] sin)
// (c0, c1) = (2p, 2p + 1) interleaved or (p, p + rot_dim / 2) split-half;
// channels from rot_dim on pass through.  The gradient with respect to x is the
// same rotation by the negative angle (`inverse`).
//
// The angle is taken in fp64 and reduced to a fraction of a turn there: a
// position of 10^6 at frequency 1 loses 0.06 rad in fp32.  The reduced turn,
// its sine and cosine and the rotation are fp32 (fp32 matrices are off by 3.6e-8,
// 2.9e-8 where the angle stays fp64), rounded once to the tensor's type.
//
// HBM-bound (each value is read once and written once; 3 flops per value), so
// the layout follows the bytes: one 16-byte pack (split-half: the two packs
// that hold a pair's members) per step and thread, four steps of loads in
// flight.  A thread keeps one token and one pack of channels and walks over the
// heads of Q and then K, so its sines and cosines are computed once in
// registers and reused by every head, with no table in memory and no barrier.
// 32760 tokens x 40 heads, interleaved: bf16 118 us (5.7 TB/s), fp32 211 us (6.4
// TB/s).  Tensors that do not allow 16-byte packs (strides, alignment, a head or
// rotated part that is no whole number of packs) go by single pairs: 307 and 321 us.
#include <algorithm>
#include <cmath>

#include "tb_capi_internal.h"
#include "tb_tu.cuh"

namespace tb {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeInFlight = 4;
constexpr int kMaxAxes = 4;
constexpr double kTwoOverPi = 0.6366197723675814;

struct RopePositions {
  const void* ptr;
  const double* inv_freq;
  int type;                 // TB_POS_*
  int axes;
  int64_t batch_stride;     // elements; 0 when all batch rows share the positions
  int axis_end[kMaxAxes];   // pairs [axis_end[a - 1], axis_end[a]) turn with axis a
  float scale, scale_lo;    // the fp64 scale as the sum of two floats
  float sign;               // -1: inverse rotation
};

struct RopeParams {
  const void* in[2];        // Q, K
  void* out[2];
  int64_t in_s[2][3];       // element strides (batch, head, token)
  int64_t out_s[2][3];
  RopePositions pos;
  int length, q_heads, heads, head_dim, rot_dim;
  int items;                // packs of channels per token and head
  int items_cta;            // of them per CTA
  int tok_lanes, head_lanes, token_blocks;
};

__device__ __forceinline__ double load_position(const RopePositions& p, int64_t i) {
  switch (p.type) {
    case TB_POS_I32: return static_cast<double>(static_cast<const int32_t*>(p.ptr)[i]);
    case TB_POS_I64: {
      // Exact up to 2^51 by the mantissa of 1.5 * 2^52 (64-bit conversions are slow;
      // larger positions have no phase left in fp64).
      const int64_t v = static_cast<const int64_t*>(p.ptr)[i];
      return __longlong_as_double(v + 0x4338000000000000ll) - 6755399441055744.0;
    }
    case TB_POS_F32: return static_cast<double>(static_cast<const float*>(p.ptr)[i]);
    default: return static_cast<const double*>(p.ptr)[i];
  }
}

__device__ __forceinline__ int axis_of(const RopePositions& p, int pair) {
  int a = 0;
#pragma unroll
  for (int i = 0; i < kMaxAxes - 1; ++i) a += (i + 1 < p.axes && pair >= p.axis_end[i]) ? 1 : 0;
  return a;
}

// scale * cos and scale * sin of position * inv_freq.  In fp64 the angle is
// counted in quarter turns and split into the nearest whole number (the low bits
// of its sum with 1.5 * 2^52) and a rest r in [-1/2, 1/2]; sin and cos of r
// quarter turns are polynomials in r^2 (interpolated at the Chebyshev nodes of
// [0, 1/4]; off by at most 1 ulp with fp32 arithmetic), turned by the quadrant.
__device__ __forceinline__ void turn(const RopePositions& p, double position, double inv_freq,
                                     float& c, float& s) {
  const double quarters = position * inv_freq * kTwoOverPi;
  const double shifted = quarters + 6755399441055744.0;
  const int q = __double2loint(shifted);
  const float r = static_cast<float>(quarters - (shifted - 6755399441055744.0));
  const float z = r * r;
  float a = fmaf(z, -0.004602149128913879f, 0.07968021929264069f);
  a = fmaf(z, a, -0.6459634900093079f);
  a = fmaf(z, a, -4.371138828673793e-08f);  // pi / 2 in two words
  a = fmaf(r, 1.5707963705062866f, r * a);
  float b = fmaf(z, 0.0009067399078048766f, -0.02086152881383896f);
  b = fmaf(z, b, 0.253669410943985f);
  b = fmaf(z, b, -1.2337005138397217f);
  b = fmaf(z, b, 1.0f);
  const float sn = q & 1 ? b : a, cs = q & 1 ? a : b;
  s = __uint_as_float(__float_as_uint(sn) ^ (static_cast<uint32_t>(q & 2) << 30));
  c = __uint_as_float(__float_as_uint(cs) ^ (static_cast<uint32_t>((q + 1) & 2) << 30));
  c = fmaf(c, p.scale, c * p.scale_lo);
  s = fmaf(s, p.scale, s * p.scale_lo);
}

template <typename T>
struct Pack {  // 16 bytes
  static constexpr int kN = 16 / static_cast<int>(sizeof(T));
};

__device__ __forceinline__ void unpack(const uint4& v, float (&f)[4], const float*) {
  f[0] = __uint_as_float(v.x);
  f[1] = __uint_as_float(v.y);
  f[2] = __uint_as_float(v.z);
  f[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ uint4 repack(const float (&f)[4], const float*) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                    __float_as_uint(f[3]));
}
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[8], const __nv_bfloat16*) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 repack(const float (&f)[8], const __nv_bfloat16*) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                    pack_bf16x2(f[6], f[7]));
}
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[8], const __half*) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
__device__ __forceinline__ uint4 repack(const float (&f)[8], const __half*) {
  return make_uint4(pack_f16x2(f[0], f[1]), pack_f16x2(f[2], f[3]), pack_f16x2(f[4], f[5]),
                    pack_f16x2(f[6], f[7]));
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float v, float* p) { *p = v; }
__device__ __forceinline__ void from_f32(float v, __half* p) { *p = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16* p) { *p = __float2bfloat16_rn(v); }

// VEC: 16-byte packs; otherwise one pair (or one passed-through channel) per
// item, for widths, strides or addresses that no pack fits.
template <typename T, bool SPLIT, bool VEC>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeParams p) {
  constexpr int E = VEC ? Pack<T>::kN : 1;
  constexpr int NP = VEC ? (SPLIT ? E : E / 2) : 1;  // pairs per item
  const int item = blockIdx.y * p.items_cta + threadIdx.x % p.items_cta;
  const int lane = threadIdx.x / p.items_cta;
  const int b = blockIdx.x / p.token_blocks;
  const int token = (blockIdx.x % p.token_blocks) * p.tok_lanes + lane % p.tok_lanes;
  const int head_lane = lane / p.tok_lanes;
  if (item >= p.items || head_lane >= p.head_lanes || token >= p.length) return;

  const int half = p.rot_dim / 2;
  const int pair0 = item * NP;
  const bool rotated = pair0 < half;
  int c0, c1;  // first channels of the item's one or two packs
  if (rotated) {
    c0 = (VEC && !SPLIT) ? 2 * pair0 : (SPLIT ? pair0 : 2 * pair0);
    c1 = SPLIT ? pair0 + half : 2 * pair0 + 1;
  } else if (VEC && !SPLIT) {
    c0 = c1 = item * E;
  } else {
    c0 = c1 = p.rot_dim + (item - half / NP) * E;
  }
  float cs[NP], sn[NP];
  if (rotated) {
    const int64_t at = b * p.pos.batch_stride + static_cast<int64_t>(token) * p.pos.axes;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      turn(p.pos, load_position(p.pos, at + axis_of(p.pos, pair0 + i)),
           p.pos.inv_freq[pair0 + i], cs[i], sn[i]);
      sn[i] *= p.pos.sign;
    }
  }
  const int step = p.head_lanes * gridDim.z;
  const int h0 = head_lane + p.head_lanes * blockIdx.z;
  auto src = [&](int h) {
    const int w = h >= p.q_heads;
    return static_cast<const T*>(p.in[w]) + b * p.in_s[w][0] +
           (h - (w ? p.q_heads : 0)) * p.in_s[w][1] + token * p.in_s[w][2];
  };
  auto dst = [&](int h) {
    const int w = h >= p.q_heads;
    return static_cast<T*>(p.out[w]) + b * p.out_s[w][0] +
           (h - (w ? p.q_heads : 0)) * p.out_s[w][1] + token * p.out_s[w][2];
  };
  if constexpr (VEC) {
    const T* const tag = nullptr;
    for (int hb = h0; hb < p.heads; hb += kRopeInFlight * step) {
      uint4 va[kRopeInFlight], vb[SPLIT ? kRopeInFlight : 1];
#pragma unroll
      for (int u = 0; u < kRopeInFlight; ++u) {
        const int h = hb + u * step;
        if (h < p.heads) {
          const T* s = src(h);
          va[u] = *reinterpret_cast<const uint4*>(s + c0);
          if (SPLIT && rotated) vb[SPLIT ? u : 0] = *reinterpret_cast<const uint4*>(s + c1);
        }
      }
#pragma unroll
      for (int u = 0; u < kRopeInFlight; ++u) {
        const int h = hb + u * step;
        if (h >= p.heads) break;
        T* d = dst(h);
        if (!rotated) {
          *reinterpret_cast<uint4*>(d + c0) = va[u];
          continue;
        }
        float x[E], y[E];
        unpack(va[u], x, tag);
        if constexpr (SPLIT) {
          float z[E], w[E];
          unpack(vb[u], z, tag);
#pragma unroll
          for (int i = 0; i < E; ++i) {
            y[i] = fmaf(x[i], cs[i], -(z[i] * sn[i]));
            w[i] = fmaf(z[i], cs[i], x[i] * sn[i]);
          }
          *reinterpret_cast<uint4*>(d + c0) = repack(y, tag);
          *reinterpret_cast<uint4*>(d + c1) = repack(w, tag);
        } else {
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            y[2 * i] = fmaf(x[2 * i], cs[i], -(x[2 * i + 1] * sn[i]));
            y[2 * i + 1] = fmaf(x[2 * i + 1], cs[i], x[2 * i] * sn[i]);
          }
          *reinterpret_cast<uint4*>(d + c0) = repack(y, tag);
        }
      }
    }
  } else {
    for (int h = h0; h < p.heads; h += step) {
      const T* s = src(h);
      T* d = dst(h);
      if (!rotated) {
        d[c0] = s[c0];
        continue;
      }
      const float x = to_f32(s[c0]), z = to_f32(s[c1]);
      from_f32(fmaf(x, cs[0], -(z * sn[0])), d + c0);
      from_f32(fmaf(z, cs[0], x * sn[0]), d + c1);
    }
  }
}

// out [batch, length, pairs, 2, 2] = scale * [[cos, -sin], [sin, cos]]: the
// thread of G pairs writes 4 G values at once (16-bit types: 16 bytes; 75600 tokens x
// 64 pairs 14.6 us, 15.6 with G = 1).
template <typename T, int G>
__global__ void __launch_bounds__(kRopeThreads)
    rope_freqs_kernel(const RopePositions pos, T* __restrict__ out, int length, int pairs,
                      int groups_cta, int tok_lanes) {
  const int g = blockIdx.y * groups_cta + threadIdx.x % groups_cta;
  const int lane = threadIdx.x / groups_cta;
  if (g * G >= pairs || lane >= tok_lanes) return;
  double f[G];
  int axis[G];
#pragma unroll
  for (int i = 0; i < G; ++i) {
    f[i] = pos.inv_freq[g * G + i];
    axis[i] = axis_of(pos, g * G + i);
  }
  const int64_t b = blockIdx.z;
  const int step = static_cast<int>(gridDim.x) * tok_lanes;
#pragma unroll 2
  for (int t = static_cast<int>(blockIdx.x) * tok_lanes + lane; t < length; t += step) {
    const int64_t at = b * pos.batch_stride + static_cast<int64_t>(t) * pos.axes;
    float v[4 * G];
    double position = load_position(pos, at + axis[0]);
#pragma unroll
    for (int i = 0; i < G; ++i) {
      float c, s;
      if (i > 0 && axis[i] != axis[i - 1]) position = load_position(pos, at + axis[i]);
      turn(pos, position, f[i], c, s);
      v[4 * i] = c;
      v[4 * i + 1] = -s;
      v[4 * i + 2] = s;
      v[4 * i + 3] = c;
    }
    T* o = out + ((b * length + t) * pairs + g * G) * 4;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      uint32_t w[2 * G];
#pragma unroll
      for (int i = 0; i < 2 * G; ++i) {
        if constexpr (std::is_same<T, __half>::value) w[i] = pack_f16x2(v[2 * i], v[2 * i + 1]);
        else w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
      }
      if constexpr (G == 2) *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
      else *reinterpret_cast<uint2*>(o) = make_uint2(w[0], w[1]);
    }
  }
}

RopePositions make_positions(const void* positions, int position_type, int64_t position_batches,
                             const double* inv_freq, const int32_t* axis_pairs, int axes,
                             int64_t pairs, int64_t batch, int64_t length, double scale,
                             int inverse) {
  TB_REQUIRE(position_type >= TB_POS_I32 && position_type <= TB_POS_F64,
             "positions must be int32, int64, float32, or float64");
  TB_REQUIRE(position_batches == 1 || position_batches == batch,
             "positions must have one row or one row per batch entry");
  TB_REQUIRE(axes >= 1 && axes <= kMaxAxes, "positions must have 1 to 4 axes");
  TB_REQUIRE(std::isfinite(scale), "scale must be finite");
  RopePositions p{};
  p.ptr = positions;
  p.inv_freq = inv_freq;
  p.type = position_type;
  p.axes = axes;
  p.batch_stride = position_batches == 1 ? 0 : length * axes;
  int64_t end = 0;
  for (int a = 0; a < axes; ++a) {
    const int64_t n = axis_pairs != nullptr ? axis_pairs[a] : pairs;
    TB_REQUIRE(n >= 0, "axis_pairs must not be negative");
    end += n;
    TB_REQUIRE(end <= pairs, "axis_pairs must add up to the number of channel pairs");
    p.axis_end[a] = static_cast<int>(end);
  }
  TB_REQUIRE(end == pairs, "axis_pairs must add up to the number of channel pairs");
  p.scale = static_cast<float>(scale);
  p.scale_lo = static_cast<float>(scale - static_cast<double>(p.scale));
  p.sign = inverse ? -1.0f : 1.0f;
  return p;
}

bool fits16(const void* ptr, const int64_t* strides, int elem_bytes) {
  bool ok = (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0;
  for (int i = 0; i < 3; ++i) ok = ok && (strides[i] * elem_bytes) % 16 == 0;
  return ok;
}

template <typename T>
void rope_launch(RopeParams& p, int64_t batch, int split_half, cudaStream_t stream) {
  constexpr int E = Pack<T>::kN;
  bool vec = p.head_dim % E == 0 && p.rot_dim % (split_half ? 2 * E : E) == 0;
  for (int w = 0; w < 2; ++w) {
    if (p.in[w] == nullptr) continue;
    vec = vec && fits16(p.in[w], p.in_s[w], sizeof(T)) && fits16(p.out[w], p.out_s[w], sizeof(T));
  }
  const int half = p.rot_dim / 2;
  if (vec) p.items = split_half ? half / E + (p.head_dim - p.rot_dim) / E : p.head_dim / E;
  else p.items = half + p.head_dim - p.rot_dim;
  // Threads of a CTA: items x tokens x heads.  Tokens come first (a thread's
  // sines serve all heads); heads share the CTA and then the grid where there
  // are too few tokens to fill the SMs (4 CTAs each; 40 heads: 64 tokens 2.9 us, 13.4
  // unsplit, 512 tokens 5.0 us, 7.3 with 16 CTAs each).
  p.items_cta = std::min(p.items, kRopeThreads);
  const int lanes = kRopeThreads / p.items_cta;
  p.tok_lanes = static_cast<int>(std::min<int64_t>(lanes, p.length));
  p.head_lanes = std::min(lanes / p.tok_lanes, p.heads);
  p.token_blocks = (p.length + p.tok_lanes - 1) / p.tok_lanes;
  const int64_t ctas_x = batch * p.token_blocks;
  const int chunks = (p.items + p.items_cta - 1) / p.items_cta;
  TB_REQUIRE(ctas_x <= INT32_MAX, "rotary dimensions exceed the CUDA kernel range");
  const int64_t want = 4LL * device_sm_count();
  const int64_t per_thread = (p.heads + p.head_lanes - 1) / p.head_lanes;
  const int64_t split =
      std::max<int64_t>(1, std::min(per_thread, want / std::max<int64_t>(1, ctas_x * chunks)));
  const dim3 grid(static_cast<unsigned>(ctas_x), static_cast<unsigned>(chunks),
                  static_cast<unsigned>(split));
  if (vec) {
    if (split_half) rope_kernel<T, true, true><<<grid, kRopeThreads, 0, stream>>>(p);
    else rope_kernel<T, false, true><<<grid, kRopeThreads, 0, stream>>>(p);
  } else {
    if (split_half) rope_kernel<T, true, false><<<grid, kRopeThreads, 0, stream>>>(p);
    else rope_kernel<T, false, false><<<grid, kRopeThreads, 0, stream>>>(p);
  }
  TB_CUDA_CHECK(cudaGetLastError());
}

template <typename T>
void freqs_launch(const RopePositions& pos, void* out, int64_t batch, int64_t length, int pairs,
                  cudaStream_t stream) {
  const bool two = sizeof(T) == 2 && pairs % 2 == 0;
  const int groups = two ? pairs / 2 : pairs;
  const int groups_cta = std::min(groups, kRopeThreads);
  const int tok_lanes = kRopeThreads / groups_cta;
  // Eight CTAs fit an SM; two rounds of them, whose tokens share a thread's
  // frequencies (75600 tokens x 64 pairs in bf16, a call on memory not in L2: 16.5 us,
  // 18.2 with one round, 18.4 with four; in a loop over memory in L2 one token a
  // thread takes 44 % longer than two rounds).
  const int64_t blocks = (length + tok_lanes - 1) / tok_lanes;
  const int64_t want = std::max<int64_t>(1, 16LL * device_sm_count() / batch);
  TB_REQUIRE(batch <= 65535, "batch exceeds the grid range");
  const dim3 grid(static_cast<unsigned>(std::min(blocks, want)),
                  static_cast<unsigned>((groups + groups_cta - 1) / groups_cta),
                  static_cast<unsigned>(batch));
  T* o = static_cast<T*>(out);
  const int L = static_cast<int>(length);
  if constexpr (sizeof(T) == 2) {
    if (two) {
      rope_freqs_kernel<T, 2><<<grid, kRopeThreads, 0, stream>>>(pos, o, L, pairs, groups_cta,
                                                                  tok_lanes);
      TB_CUDA_CHECK(cudaGetLastError());
      return;
    }
  }
  rope_freqs_kernel<T, 1><<<grid, kRopeThreads, 0, stream>>>(pos, o, L, pairs, groups_cta,
                                                             tok_lanes);
  TB_CUDA_CHECK(cudaGetLastError());
}

}  // namespace
}  // namespace tb

using tb::guarded;

extern "C" int tb_rope(const void* query, const void* key, void* query_out, void* key_out,
                       const void* positions, int position_type, int64_t position_batches,
                       const double* inv_freq, const int32_t* axis_pairs, int axes, int64_t batch,
                       int64_t query_heads, int64_t key_heads, int64_t length, int64_t head_dim,
                       int64_t rot_dim, const int64_t* strides, int split_half, int inverse,
                       int dtype, double scale, tb_stream_t stream) {
  return guarded([&] {
    TB_REQUIRE(query && query_out && positions && inv_freq && strides,
               "rotary tensors must be CUDA tensors");
    TB_REQUIRE((key != nullptr) == (key_out != nullptr) && (key != nullptr) == (key_heads > 0),
               "key, its output and its heads must be given together");
    TB_REQUIRE(dtype == TB_DTYPE_BF16 || dtype == TB_DTYPE_F16 || dtype == TB_DTYPE_F32,
               "rotary input must be float16, bfloat16, or float32");
    TB_REQUIRE(batch > 0 && query_heads > 0 && length > 0 && head_dim > 0 && key_heads >= 0,
               "rotary input dimensions must be positive");
    TB_REQUIRE(rot_dim > 0 && rot_dim % 2 == 0 && rot_dim <= head_dim,
               "rot_dim must be even and within the head dimension");
    TB_REQUIRE(head_dim <= 65536 && query_heads + key_heads <= INT32_MAX / 8 &&
                   length <= INT32_MAX / 2 && batch <= INT32_MAX,
               "rotary dimensions exceed the CUDA kernel range");
    tb::RopeParams p{};
    p.pos = tb::make_positions(positions, position_type, position_batches, inv_freq, axis_pairs,
                               axes, rot_dim / 2, batch, length, scale, inverse);
    tb::require_sm100();
    p.in[0] = query;
    p.in[1] = key;
    p.out[0] = query_out;
    p.out[1] = key_out;
    for (int i = 0; i < 3; ++i) {
      p.in_s[0][i] = strides[i];
      p.in_s[1][i] = strides[3 + i];
      p.out_s[0][i] = strides[6 + i];
      p.out_s[1][i] = strides[9 + i];
    }
    p.length = static_cast<int>(length);
    p.q_heads = static_cast<int>(query_heads);
    p.heads = static_cast<int>(query_heads + key_heads);
    p.head_dim = static_cast<int>(head_dim);
    p.rot_dim = static_cast<int>(rot_dim);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == TB_DTYPE_BF16) tb::rope_launch<__nv_bfloat16>(p, batch, split_half, s);
    else if (dtype == TB_DTYPE_F16) tb::rope_launch<__half>(p, batch, split_half, s);
    else tb::rope_launch<float>(p, batch, split_half, s);
  });
}

extern "C" int tb_rope_freqs(const void* positions, int position_type, int64_t position_batches,
                             const double* inv_freq, const int32_t* axis_pairs, int axes,
                             void* output, int64_t batch, int64_t length, int64_t pairs,
                             int dtype, double scale, tb_stream_t stream) {
  return guarded([&] {
    TB_REQUIRE(positions && inv_freq && output, "rotary tensors must be CUDA tensors");
    TB_REQUIRE(dtype == TB_DTYPE_BF16 || dtype == TB_DTYPE_F16 || dtype == TB_DTYPE_F32,
               "rotary matrices must be float16, bfloat16, or float32");
    TB_REQUIRE(batch > 0 && length > 0 && pairs > 0, "rotary input dimensions must be positive");
    TB_REQUIRE(pairs <= 32768 && length <= INT32_MAX / 2 && batch <= INT32_MAX,
               "rotary dimensions exceed the CUDA kernel range");
    TB_REQUIRE((reinterpret_cast<uintptr_t>(output) & 15u) == 0,
               "rotary matrices must be 16-byte aligned");
    const tb::RopePositions p =
        tb::make_positions(positions, position_type, position_batches, inv_freq, axis_pairs, axes,
                           pairs, batch, length, scale, 0);
    tb::require_sm100();
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int n = static_cast<int>(pairs);
    if (dtype == TB_DTYPE_BF16) tb::freqs_launch<__nv_bfloat16>(p, output, batch, length, n, s);
    else if (dtype == TB_DTYPE_F16) tb::freqs_launch<__half>(p, output, batch, length, n, s);
    else tb::freqs_launch<float>(p, output, batch, length, n, s);
  });
}
