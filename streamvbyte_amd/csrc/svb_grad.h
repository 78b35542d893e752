// Gradient operators: the global norm of many tensors, clipping by it, and the quantising encoder that carries its
// error over to the next step.
#pragma once
#include "svb_device.h"
#include "svb_encode.h"
#include "svb_lookback.h"

namespace svb {

constexpr int kF32 = 0, kF16 = 1, kBF16 = 2;                 // SVBGPU_F32, _F16, _BF16
constexpr int kNormMax = 0, kNormSum = 1, kNormEuclid = 2;  // SVBGPU_NORM_MAX, _L1, _L2
constexpr double kNormEps = 1e-6;                            // added to the norm before it divides

// ---- element types ------------------------------------------------------------------------------------
// The empty asm in the conversions of float16 keep them, and the float32 arithmetic between them, out of
// mixed-precision multiply-adds, which round differently and turn -0 into 0.
__device__ __forceinline__ float f16_to_f32(u32 h) {
  float x = (float)__builtin_bit_cast(_Float16, (unsigned short)h);
  asm("" : "+v"(x));
  return x;
}
__device__ __forceinline__ float bf16_to_f32(u32 h) { return __uint_as_float(h << 16); }
// The one rounding of a result to 16 bits: to nearest, ties to even.
__device__ __forceinline__ u32 f32_to_f16(float x) {
  asm("" : "+v"(x));
  return __builtin_bit_cast(unsigned short, (_Float16)x);
}
__device__ __forceinline__ u32 f32_to_bf16(float x) { return __builtin_bit_cast(unsigned short, (__bf16)x); }

template <int T>
constexpr u32 kElemBytes = T == kF32 ? 4u : 2u;
template <int T>
constexpr u32 kVecElems = 16u / kElemBytes<T>;  // elements of a 16-byte vector

// Tensors are aligned to their element and to nothing more; gfx950 executes wide accesses at any address.
typedef u32x4_t u32x4_a2 __attribute__((aligned(2)));
typedef u32 u32x2_t __attribute__((ext_vector_type(2)));
typedef u32x2_t u32x2_a2 __attribute__((aligned(2)));

template <int T>
__device__ __forceinline__ float load_elem(const u8* p, u64 i) {
  if (T == kF32) return reinterpret_cast<const float*>(p)[i];
  const u32 h = reinterpret_cast<const unsigned short*>(p)[i];
  return T == kF16 ? f16_to_f32(h) : bf16_to_f32(h);
}
template <int T>
__device__ __forceinline__ void store_elem(u8* p, u64 i, float x) {
  if (T == kF32) reinterpret_cast<float*>(p)[i] = x;
  else reinterpret_cast<unsigned short*>(p)[i] = (unsigned short)(T == kF16 ? f32_to_f16(x) : f32_to_bf16(x));
}
// Element k of a 16-byte vector.
template <int T>
__device__ __forceinline__ float vec_elem(const u32x4_t& v, u32 k) {
  if (T == kF32) return __uint_as_float(v[k]);
  const u32 h = (k & 1u) ? v[k >> 1] >> 16 : v[k >> 1] & 0xFFFFu;
  return T == kF16 ? f16_to_f32(h) : bf16_to_f32(h);
}
template <int T>
__device__ __forceinline__ u32x4_t scale_vec(const u32x4_t& v, float c) {
  u32x4_t r;
#pragma unroll
  for (u32 d = 0; d < 4; ++d) {
    if (T == kF32) r[d] = __float_as_uint(__fmul_rn(__uint_as_float(v[d]), c));
    else if (T == kF16) r[d] = f32_to_f16(__fmul_rn(vec_elem<T>(v, 2 * d), c)) | (f32_to_f16(__fmul_rn(vec_elem<T>(v, 2 * d + 1), c)) << 16);
    else r[d] = f32_to_bf16(__fmul_rn(vec_elem<T>(v, 2 * d), c)) | (f32_to_bf16(__fmul_rn(vec_elem<T>(v, 2 * d + 1), c)) << 16);
  }
  return r;
}

// ---- tables of tensors ----------------------------------------------------------------------------------
// A launch carries its tensors in its arguments (4 KiB at most), so nothing is copied to the device, nothing is kept
// there, and a captured launch holds all it needs.  Every tensor is cut into chunks of `chunk_bytes`; a workgroup
// takes one, and finds the tensor it belongs to by a binary search on the first chunks.
struct GradSpan {
  u64 addr;   // bits 57..56 the type, below them the address
  u64 where;  // bits 63..40 the launch's index of the tensor's first chunk, below them its elements
};
constexpr u32 kMaxSpans = 240;       // spans of a launch without outputs
constexpr u32 kMaxSpansOut = 160;    // ... and with an output address each
constexpr int kAddrBits = 56, kCountBits = 40;
template <u32 N>
struct GradTable {
  GradSpan span[N];
  u32 n;
  u32 chunk_bytes;  // a multiple of kGradStep vectors
};
template <u32 N>
struct GradOuts {
  u64 addr[N];
};
constexpr u32 kGradThreads = 256;
constexpr u32 kGradUnroll = 8;                              // 16-byte loads a lane has in flight
constexpr u32 kGradStep = kGradThreads * kGradUnroll;       // vectors of one round of a workgroup
constexpr u32 kGradMinChunk = 2 * 16 * kGradStep;           // 64 KiB

struct GradChunk {
  u32 span;
  int type;
  u64 first;  // first element in the tensor
  u32 count;  // elements
};
template <u32 N>
__device__ __forceinline__ GradChunk find_chunk(const GradTable<N>& t, u32 chunk) {
  u32 lo = 0, hi = t.n;  // span[lo] starts at or before the chunk, span[hi] after it
  while (hi - lo > 1) {
    const u32 mid = (lo + hi) >> 1;
    if ((u32)(t.span[mid].where >> kCountBits) <= chunk) lo = mid;
    else hi = mid;
  }
  const u64 where = t.span[lo].where;
  GradChunk c;
  c.span = lo;
  c.type = (int)(t.span[lo].addr >> kAddrBits);
  const u32 elems = c.type == kF32 ? t.chunk_bytes >> 2 : t.chunk_bytes >> 1;
  c.first = (u64)(chunk - (u32)(where >> kCountBits)) * elems;
  c.count = (u32)min((u64)elems, (where & ((1ull << kCountBits) - 1)) - c.first);
  return c;
}

// ---- norm -------------------------------------------------------------------------------------------------
// N = (sum |x|^p)^(1/p) over every element of every tensor.  Squares and sums are in 64 bits: the square of a float32
// is exact there and neither overflows nor vanishes, and the order of the sums cannot be seen after the one rounding
// at the end.  The maximum is taken on the bits of |x|, where NaN stands above everything.
template <int KIND>
struct NormSum {
  double s0 = 0.0, s1 = 0.0;
  u32 m = 0;
  __device__ __forceinline__ void add(float x, bool odd) {
    if (KIND == kNormMax) m = max(m, __float_as_uint(x) & 0x7FFFFFFFu);
    else {
      const double d = (double)x, v = KIND == kNormEuclid ? d : fabs(d);
      double& s = odd ? s1 : s0;
      s = KIND == kNormEuclid ? fma(v, v, s) : s + v;
    }
  }
};
// Combination over the workgroup, the same in every run; result in thread 0.
template <int KIND>
__device__ __forceinline__ u64 norm_block(double s, u32 m, u64* s_tmp, u32 waves) {
  if (KIND == kNormMax) {
#pragma unroll
    for (int d = 32; d; d >>= 1) m = max(m, (u32)__shfl_xor((int)m, d));
  } else {
#pragma unroll
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
  }
  if (lane_id() == 0) s_tmp[wave_id()] = KIND == kNormMax ? (u64)m : (u64)__double_as_longlong(s);
  __syncthreads();
  u64 r = s_tmp[0];
  for (u32 w = 1; w < waves; ++w)
    r = KIND == kNormMax ? max(r, s_tmp[w])
                         : (u64)__double_as_longlong(__longlong_as_double((long long)r) + __longlong_as_double((long long)s_tmp[w]));
  return r;
}
template <int KIND, int T>
__device__ __forceinline__ void norm_chunk(const u8* p, u32 count, NormSum<KIND>& acc) {
  const u32 nv = count / kVecElems<T>;
  const u32x4_a2* v = reinterpret_cast<const u32x4_a2*>(p);
  for (u32 base = threadIdx.x; base < nv; base += kGradStep) {
    u32x4_t x[kGradUnroll];
#pragma unroll
    for (u32 i = 0; i < kGradUnroll; ++i) {
      x[i] = u32x4_t{0, 0, 0, 0};
      if (base + i * kGradThreads < nv) x[i] = v[base + i * kGradThreads];
    }
#pragma unroll
    for (u32 i = 0; i < kGradUnroll; ++i)
#pragma unroll
      for (u32 k = 0; k < kVecElems<T>; ++k) acc.add(vec_elem<T>(x[i], k), k & 1u);
  }
  const u32 rest = nv * kVecElems<T> + threadIdx.x;
  if (rest < count) acc.add(load_elem<T>(p, rest), false);
}
template <int KIND>
__global__ __launch_bounds__(kGradThreads) void k_grad_norm(GradTable<kMaxSpans> t, u64* __restrict__ partial) {
  __shared__ u64 s_tmp[kGradThreads / 64];
  const GradChunk c = find_chunk(t, blockIdx.x);
  const u8* p = reinterpret_cast<const u8*>(t.span[c.span].addr & ((1ull << kAddrBits) - 1)) + c.first * (c.type == kF32 ? 4u : 2u);
  NormSum<KIND> acc;
  if (c.type == kF32) norm_chunk<KIND, kF32>(p, c.count, acc);
  else if (c.type == kF16) norm_chunk<KIND, kF16>(p, c.count, acc);
  else norm_chunk<KIND, kBF16>(p, c.count, acc);
  const u64 r = norm_block<KIND>(acc.s0 + acc.s1, acc.m, s_tmp, kGradThreads / 64);
  if (threadIdx.x == 0) partial[blockIdx.x] = r;
}
// The chunks' sums to the norm: one workgroup.
template <int KIND>
__global__ __launch_bounds__(1024) void k_grad_finish(const u64* __restrict__ partial, u32 n, float* __restrict__ norm) {
  __shared__ u64 s_tmp[16];
  double s = 0.0;
  u32 m = 0;
  for (u32 i = threadIdx.x; i < n; i += 1024) {
    if (KIND == kNormMax) m = max(m, (u32)partial[i]);
    else s += __longlong_as_double((long long)partial[i]);
  }
  const u64 r = norm_block<KIND>(s, m, s_tmp, 16);
  if (threadIdx.x == 0) {
    const double total = __longlong_as_double((long long)r);
    *norm = KIND == kNormMax ? __uint_as_float((u32)r) : (float)(KIND == kNormEuclid ? sqrt(total) : total);
  }
}

// ---- clipping ----------------------------------------------------------------------------------------------
// The factor min(1, limit / (N + 1e-6)), worked out in 64 bits from the float32 norm and rounded once, so that it is
// the same whoever worked out the norm.  NaN stays NaN.
__device__ __forceinline__ float clip_factor(float norm, double limit) {
  const double n = (double)norm + kNormEps;
  return n <= limit ? 1.0f : (float)(limit / n);
}
template <int T>
__device__ __forceinline__ void scale_chunk(const u8* p, u8* q, u32 count, float c) {
  const u32 nv = count / kVecElems<T>;
  const u32x4_a2* v = reinterpret_cast<const u32x4_a2*>(p);
  u32x4_a2* w = reinterpret_cast<u32x4_a2*>(q);
  for (u32 base = threadIdx.x; base < nv; base += kGradStep) {
    u32x4_t x[kGradUnroll];
#pragma unroll
    for (u32 i = 0; i < kGradUnroll; ++i)
      if (base + i * kGradThreads < nv) x[i] = v[base + i * kGradThreads];
#pragma unroll
    for (u32 i = 0; i < kGradUnroll; ++i)
      if (base + i * kGradThreads < nv) w[base + i * kGradThreads] = scale_vec<T>(x[i], c);
  }
  const u32 rest = nv * kVecElems<T> + threadIdx.x;
  if (rest < count) store_elem<T>(q, rest, __fmul_rn(load_elem<T>(p, rest), c));
}
// y = x * factor, rounded to the tensor's type; in place unless `outs` says otherwise, and then a factor of 1 leaves
// nothing to do.
template <bool OUT>
__global__ __launch_bounds__(kGradThreads) void k_grad_scale(GradTable<kMaxSpansOut> t, GradOuts<kMaxSpansOut> outs,
                                                             const float* __restrict__ norm, double limit) {
  const float f = clip_factor(*norm, limit);
  if (!OUT && f == 1.0f) return;
  const GradChunk c = find_chunk(t, blockIdx.x);
  const u64 skip = c.first * (c.type == kF32 ? 4u : 2u);
  const u64 from = t.span[c.span].addr & ((1ull << kAddrBits) - 1);
  const u8* p = reinterpret_cast<const u8*>(from) + skip;
  u8* q = reinterpret_cast<u8*>(OUT ? outs.addr[c.span] : from) + skip;
  if (c.type == kF32) scale_chunk<kF32>(p, q, c.count, f);
  else if (c.type == kF16) scale_chunk<kF16>(p, q, c.count, f);
  else scale_chunk<kBF16>(p, q, c.count, f);
}

// ---- quantise with feedback, then encode -----------------------------------------------------------------
// What an encoder of quantised gradients throws away -- everything below half a step, which for most gradients is all
// of it -- is added to the same gradient of the next step instead:
//     e = g * factor + r      q = int32(nearest-even(e * scale))      r' = e - q * step,   step = 1 / scale
// every operation rounded to float32 by itself, so the integers do not depend on who computes them.  q saturates; an
// element whose e is not finite sends 0 and keeps its r.
struct FeedArgs {
  const float* norm;  // nullptr: factor 1
  double limit;
  float scale, step;
  const float* r_in;
  float* r_out;  // r_in itself or apart from it
};
__device__ __forceinline__ u32 feed_one(float g, float& r, float c, float scale, float step) {
#pragma clang fp contract(off)
  const float e = g * c + r;
  const bool finite = (__float_as_uint(e) & 0x7F800000u) != 0x7F800000u;
  const float f = rintf(e * scale);
  const int big = f >= 2147483648.0f ? 2147483647 : (int)fmaxf(f, -2147483648.0f);
  const int q = finite ? big : 0;
  const float left = e - (float)q * step;
  r = finite ? left : r;
  return (u32)q;
}
// Four gradients of a group, as they lie in memory.
template <int T>
struct Grad4 {
  u32x4_t w;  // float32: four dwords; 16 bits: two
  __device__ __forceinline__ void load(const u8* g, u64 first) {
    if (T == kF32) w = *reinterpret_cast<const u32x4_a4*>(g + 4 * first);
    else {
      const u32x2_t h = *reinterpret_cast<const u32x2_a2*>(g + 2 * first);
      w = u32x4_t{h.x, h.y, 0, 0};
    }
  }
  __device__ __forceinline__ float get(u32 k) const { return vec_elem<T>(w, k); }
};

// One pass, tile by tile like k_encode: a workgroup of NW waves draws a tile of NW * QW wave tiles, loads gradients and
// residuals, quantises, stores the new residuals, finds the tile's place by look-back and assembles its bytes.
// A wave that runs past the end of the stream takes its groups one element at a time.
template <int V, int T, int NW, int QW>
__global__ __launch_bounds__(NW * 64, 4) void k_feedback_encode(const u8* __restrict__ grad, u32 count, u32 n_tiles,
                                                                u8* __restrict__ out, FeedArgs fa, WsHeader* __restrict__ hdr,
                                                                LbWords lb, u64* __restrict__ written) {
  __shared__ EncWaveLds s_lds[NW];
  __shared__ u32 s_wave_tot[NW];
  __shared__ u64 s_prefix;
  __shared__ u32 s_tile;
  const int lane = lane_id(), wave = wave_id();
  if (threadIdx.x == 0) s_tile = atomicAdd(&hdr->ticket, 1u);
  __syncthreads();
  const u32 tile = __builtin_amdgcn_readfirstlane(s_tile);
  const u64 keylen = ((u64)count + 3) >> 2;
  constexpr u64 kTileInts = (u64)NW * QW * kWtInts;
  const u64 wave_first = (u64)tile * kTileInts + (u64)wave * QW * kWtInts;
  const float c = fa.norm ? clip_factor(*fa.norm, fa.limit) : 1.0f;

  uint4 x[QW][4];  // the zigzagged integers
  u32 lane_tot = 0;
  const bool full = wave_first + QW * kWtInts <= count;  // wave-uniform
  if (full) {
#pragma unroll
    for (int q = 0; q < QW; ++q) {
      Grad4<T> g[4];
      u32x4_t r[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u64 first = wave_first + (u32)(q * kWtInts + 4 * (j * 64 + lane));
        g[j].load(grad, first);
        r[j] = *reinterpret_cast<const u32x4_a4*>(fa.r_in + first);
      }
      u32 k4 = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u64 first = wave_first + (u32)(q * kWtInts + 4 * (j * 64 + lane));
        u32 z[4];
#pragma unroll
        for (u32 k = 0; k < 4; ++k) {
          float left = __uint_as_float(r[j][k]);
          z[k] = zz_enc(feed_one(g[j].get(k), left, c, fa.scale, fa.step));
          r[j][k] = __float_as_uint(left);
        }
        *reinterpret_cast<u32x4_a4*>(fa.r_out + first) = r[j];
        x[q][j] = make_uint4(z[0], z[1], z[2], z[3]);
        k4 |= classify_key<V>(x[q][j]) << (8 * j);
      }
      lane_tot += word_len<V>(k4, 16u);
    }
  } else {
#pragma unroll
    for (int q = 0; q < QW; ++q)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u64 first = wave_first + (u32)(q * kWtInts + 4 * (j * 64 + lane));
        u32 z[4] = {0, 0, 0, 0};
#pragma unroll
        for (u32 k = 0; k < 4; ++k)
          if (first + k < count) {
            float left = fa.r_in[first + k];
            z[k] = zz_enc(feed_one(load_elem<T>(grad, first + k), left, c, fa.scale, fa.step));
            fa.r_out[first + k] = left;
          }
        x[q][j] = make_uint4(z[0], z[1], z[2], z[3]);
        const u32 nv = first < count ? (u32)min((u64)4, (u64)count - first) : 0u;
        lane_tot += gi_total(classify_group<V, false>(x[q][j], nv));
      }
  }
  const u32 wave_tot = wave_sum(lane_tot);
  if (lane == 0) s_wave_tot[wave] = wave_tot;
  __syncthreads();
  if (wave == 0) {
    u32 tile_tot = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) tile_tot += s_wave_tot[w];
    const u64 excl = lb2_exclusive_prefix<2>(lb, tile, tile_tot, lane, &hdr->error);
    if (lane == 0) {
      s_prefix = excl;
      if (tile == n_tiles - 1 && written) *written = keylen + excl + tile_tot;
      if (tile == 0u) reset_other_ticket(hdr);
    }
  }
  __syncthreads();
  u64 doff = s_prefix;
  for (int w = 0; w < wave; ++w) doff += s_wave_tot[w];
  EncWaveLds& S = s_lds[wave];
  u8* data_out = out + keylen;
#pragma unroll 1
  for (int q = 0; q < QW; ++q) {
    const u64 wt_first = wave_first + (u64)q * kWtInts;
    u32 g[4];
    if (full) {
#pragma unroll
      for (int j = 0; j < 4; ++j) g[j] = classify_group<V, true>(x[0][j], 4u);
      doff += encode_wavetile<V, true>(x[0], g, kWtInts, lane, S, data_out + doff, out + (wt_first >> 2));
    } else if (wt_first < count) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u64 first = wt_first + 4u * (j * 64 + lane);
        g[j] = classify_group<V, false>(x[0][j], first < count ? (u32)min((u64)4, (u64)count - first) : 0u);
      }
      const u32 nints = (u32)min((u64)kWtInts, (u64)count - wt_first);
      doff += encode_wavetile<V, false>(x[0], g, nints, lane, S, data_out + doff, out + (wt_first >> 2));
    }
#pragma unroll
    for (int r = 0; r + 1 < QW; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[r][j] = x[r + 1][j];
  }
}

}  // namespace svb
