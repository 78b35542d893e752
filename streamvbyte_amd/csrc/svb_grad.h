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
// there, and a captured launch holds all it needs.  Every tensor is cut into chunks of `chunk_bytes`; a workgroup (or,
// for small sets, a wave) takes one at a time.
struct GradSpan {
  u64 addr;   // bits 57..56 the type, below them the address
  u64 where;  // bits 63..40 the launch's index of the tensor's first chunk, below them its elements
};
constexpr int kAddrBits = 56, kCountBits = 40;
constexpr u32 kMaxSpans = 240;     // spans of a launch without outputs
constexpr u32 kMaxSpansOut = 160;  // ... with an output address each
constexpr u32 kMaxSpansSmall = 64; // ... of the one-workgroup kernel
template <u32 N>
struct GradTable {
  GradSpan span[N];
  u32 n;
  u32 chunk_bytes;  // a multiple of 16
  u32 chunks;
};
template <u32 N>
struct GradOuts {
  u64 addr[N];
};
struct GradChunk {
  u64 addr;   // of its first element
  u64 skip;   // bytes of the tensor before it
  u32 span;
  int type;
  u32 count;  // elements
};
// The chunk's tensor is the last span that starts at or before it.  Every lane looks at a few spans and the ballots are
// counted: one trip to the arguments, where a binary search takes eight that wait for each other.
template <u32 N>
__device__ __forceinline__ GradChunk find_chunk(const GradTable<N>& t, u32 chunk) {
  const u32 lane = lane_id();
  u32 before = 0;
#pragma unroll
  for (u32 i = 0; i < (N + 63) / 64; ++i) {
    const u32 k = i * 64 + lane;
    const bool starts = k < t.n && (u32)(t.span[min(k, N - 1)].where >> kCountBits) <= chunk;
    before += (u32)__popcll(__ballot(starts));
  }
  GradChunk c;
  c.span = __builtin_amdgcn_readfirstlane(before) - 1;  // span 0 starts at chunk 0
  const GradSpan s = t.span[c.span];
  c.type = (int)(s.addr >> kAddrBits);
  const u32 shift = c.type == kF32 ? 2u : 1u, elems = t.chunk_bytes >> shift;
  const u64 first = (u64)(chunk - (u32)(s.where >> kCountBits)) * elems;
  c.count = (u32)min((u64)elems, (s.where & ((1ull << kCountBits) - 1)) - first);
  c.skip = first << shift;
  c.addr = (s.addr & ((1ull << kAddrBits) - 1)) + c.skip;
  return c;
}

// ---- norm -------------------------------------------------------------------------------------------------
// N = (sum |x|^p)^(1/p) over every element of every tensor.  Squares and sums are in 64 bits: the square of a float32
// is exact there and neither overflows nor vanishes.  The order of the sums is that of the chunks, lanes and waves, the
// same in every run; another order of the tensors may change the last bits of 64, and so, seldom, the last of 32.  The maximum is taken on the bits of |x|, where NaN stands above everything.
template <int KIND>
struct NormSum {
  double s0 = 0.0, s1 = 0.0;  // two chains of additions
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
// What a chunk, a workgroup or the whole set comes to: the bits of a double, or those of a float32 maximum.
template <int KIND>
__device__ __forceinline__ u64 norm_join(u64 a, u64 b) {
  if (KIND == kNormMax) return max(a, b);
  return (u64)__double_as_longlong(__longlong_as_double((long long)a) + __longlong_as_double((long long)b));
}
// Combination over the workgroup, the same in every run; result in every thread.
template <int KIND, u32 WAVES>
__device__ __forceinline__ u64 norm_block(double s, u32 m, u64* s_tmp) {
  if (KIND == kNormMax) {
#pragma unroll
    for (int d = 32; d; d >>= 1) m = max(m, (u32)__shfl_xor((int)m, d));
  } else {
#pragma unroll
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
  }
  if (lane_id() == 0) s_tmp[wave_id()] = KIND == kNormMax ? (u64)m : (u64)__double_as_longlong(s);
  __syncthreads();
  u64 r[WAVES];
#pragma unroll
  for (u32 w = 0; w < WAVES; ++w) r[w] = s_tmp[w];
#pragma unroll
  for (u32 w = 1; w < WAVES; w <<= 1)
#pragma unroll
    for (u32 i = 0; i + w < WAVES; i += 2 * w) r[i] = norm_join<KIND>(r[i], r[i + w]);
  return r[0];
}
template <int KIND>
__device__ __forceinline__ float norm_value(u64 r) {
  if (KIND == kNormMax) return __uint_as_float((u32)r);
  const double total = __longlong_as_double((long long)r);
  return (float)(KIND == kNormEuclid ? sqrt(total) : total);
}
// A chunk by THREADS threads, of which this is number `id`, with UNROLL 16-byte loads in flight each.
template <int KIND, int T, bool NTL, u32 THREADS, u32 UNROLL>
__device__ __forceinline__ void norm_chunk(u64 addr, u32 count, u32 id, NormSum<KIND>& acc) {
  const u32 nv = count / kVecElems<T>;
  const u32x4_a2* v = reinterpret_cast<const u32x4_a2*>(addr);
  for (u32 base = id; base < nv; base += THREADS * UNROLL) {
    u32x4_t x[UNROLL];
#pragma unroll
    for (u32 i = 0; i < UNROLL; ++i) {
      x[i] = u32x4_t{0, 0, 0, 0};
      if (base + i * THREADS < nv) x[i] = NTL ? __builtin_nontemporal_load(v + base + i * THREADS) : v[base + i * THREADS];
    }
#pragma unroll
    for (u32 i = 0; i < UNROLL; ++i)
#pragma unroll
      for (u32 k = 0; k < kVecElems<T>; ++k) acc.add(vec_elem<T>(x[i], k), k & 1u);
  }
  const u32 rest = nv * kVecElems<T> + id;
  if (rest < count) acc.add(load_elem<T>(reinterpret_cast<const u8*>(addr), rest), false);
}
template <int KIND, bool NTL, u32 THREADS, u32 UNROLL>
__device__ __forceinline__ void norm_any(const GradChunk& c, u32 id, NormSum<KIND>& acc) {
  if (c.type == kF32) norm_chunk<KIND, kF32, NTL, THREADS, UNROLL>(c.addr, c.count, id, acc);
  else if (c.type == kF16) norm_chunk<KIND, kF16, NTL, THREADS, UNROLL>(c.addr, c.count, id, acc);
  else norm_chunk<KIND, kBF16, NTL, THREADS, UNROLL>(c.addr, c.count, id, acc);
}
// The chunks' sums.  Bound by memory: 2^28 float32 in 155 us = 6.9 TB/s, with k_grad_finish 160.  The loads are
// non-temporal (181 us without): what is read once and is larger than the caches only turns them over.  The last chunks
// of a clip's norm, from `nt_chunks` on, are read to stay, for k_grad_scale begins with them.
constexpr u32 kNormThreads = 256, kNormUnroll = 8;
template <int KIND>
__global__ __launch_bounds__(kNormThreads) void k_grad_norm(GradTable<kMaxSpans> t, u64* __restrict__ partial, u32 nt_chunks) {
  __shared__ u64 s_tmp[kNormThreads / 64];
  const GradChunk c = find_chunk(t, blockIdx.x);
  NormSum<KIND> acc;
  if (blockIdx.x < nt_chunks) norm_any<KIND, true, kNormThreads, kNormUnroll>(c, threadIdx.x, acc);
  else norm_any<KIND, false, kNormThreads, kNormUnroll>(c, threadIdx.x, acc);
  const u64 r = norm_block<KIND, kNormThreads / 64>(acc.s0 + acc.s1, acc.m, s_tmp);
  if (threadIdx.x == 0) partial[blockIdx.x] = r;
}
// The chunks' sums to the norm: one workgroup, four loads of a thread in flight.
template <int KIND>
__global__ __launch_bounds__(1024) void k_grad_finish(const u64* __restrict__ partial, u32 n, float* __restrict__ norm) {
  __shared__ u64 s_tmp[16];
  u64 s = 0;  // the bits of 0.0 as well
  for (u32 i = threadIdx.x; i < n; i += 4 * 1024) {
    u64 p[4];
#pragma unroll
    for (u32 k = 0; k < 4; ++k) p[k] = i + 1024 * k < n ? partial[i + 1024 * k] : 0;
    s = norm_join<KIND>(s, norm_join<KIND>(norm_join<KIND>(p[0], p[1]), norm_join<KIND>(p[2], p[3])));
  }
  const u64 r = norm_block<KIND, 16>(__longlong_as_double((long long)s), (u32)s, s_tmp);
  if (threadIdx.x == 0) *norm = norm_value<KIND>(r);
}

// ---- clipping ----------------------------------------------------------------------------------------------
// The factor min(1, limit / (N + 1e-6)), worked out in 64 bits from the float32 norm and rounded once, so that it is
// the same whoever worked out the norm.  NaN stays NaN.
__device__ __forceinline__ float clip_factor(float norm, double limit) {
  const double n = (double)norm + kNormEps;
  return n <= limit ? 1.0f : (float)(limit / n);
}
template <int T, bool NT, u32 THREADS, u32 UNROLL>
__device__ __forceinline__ void scale_chunk(u64 from, u64 to, u32 count, u32 id, float c) {
  const u32 nv = count / kVecElems<T>;
  const u32x4_a2* v = reinterpret_cast<const u32x4_a2*>(from);
  u32x4_a2* w = reinterpret_cast<u32x4_a2*>(to);
  for (u32 base = id; base < nv; base += THREADS * UNROLL) {
    u32x4_t x[UNROLL];
#pragma unroll
    for (u32 i = 0; i < UNROLL; ++i)
      if (base + i * THREADS < nv) x[i] = NT ? __builtin_nontemporal_load(v + base + i * THREADS) : v[base + i * THREADS];
#pragma unroll
    for (u32 i = 0; i < UNROLL; ++i)
      if (base + i * THREADS < nv) {
        const u32x4_t y = scale_vec<T>(x[i], c);
        if (NT) __builtin_nontemporal_store(y, w + base + i * THREADS);
        else w[base + i * THREADS] = y;
      }
  }
  const u32 rest = nv * kVecElems<T> + id;
  if (rest < count)
    store_elem<T>(reinterpret_cast<u8*>(to), rest, __fmul_rn(load_elem<T>(reinterpret_cast<const u8*>(from), rest), c));
}
template <bool NT, u32 THREADS, u32 UNROLL>
__device__ __forceinline__ void scale_any(const GradChunk& c, u64 to, u32 id, float f) {
  if (c.type == kF32) scale_chunk<kF32, NT, THREADS, UNROLL>(c.addr, to, c.count, id, f);
  else if (c.type == kF16) scale_chunk<kF16, NT, THREADS, UNROLL>(c.addr, to, c.count, id, f);
  else scale_chunk<kBF16, NT, THREADS, UNROLL>(c.addr, to, c.count, id, f);
}
// y = x * factor, rounded to the tensor's type; in place unless OUT, and then a factor of 1 leaves nothing to do.  The
// chunks are taken last first: the end of what the norm has just read is still in the Infinity Cache.  Bound by memory,
// read and write: 2^28 float32 in 340 us = 6.3 TB/s.  Small chunks and non-temporal accesses, so that the workgroups in
// flight cover one compact stretch and what is written does not turn the cache over (385 us with chunks of 128 KiB, in
// order and with plain accesses).
constexpr u32 kScaleThreads = 256, kScaleUnroll = 4, kScaleChunk = 16 * kScaleThreads * kScaleUnroll;
template <bool OUT, bool NT>
__global__ __launch_bounds__(kScaleThreads) void k_grad_scale(GradTable<kMaxSpansOut> t, GradOuts<kMaxSpansOut> outs,
                                                              const float* __restrict__ norm, double limit) {
  const float f = clip_factor(*norm, limit);
  if (!OUT && f == 1.0f) return;
  const GradChunk c = find_chunk(t, gridDim.x - 1 - blockIdx.x);
  scale_any<NT, kScaleThreads, kScaleUnroll>(c, OUT ? outs.addr[c.span] + c.skip : c.addr, threadIdx.x, f);
}

// A small set in one launch of one workgroup: chunk by chunk to the waves, the norm, and for a clip the chunks again.
// A launch and its place in the queue cost more than the bytes: a handful of small tensors takes 3 us this way, 6 by
// k_grad_norm and k_grad_finish.
constexpr u32 kSmallChunk = 4096, kSmallChunks = 64;  // bytes; chunks at most
template <int KIND, bool CLIP, bool OUT>
__global__ __launch_bounds__(1024) void k_grad_small(GradTable<kMaxSpansSmall> t, GradOuts<kMaxSpansSmall> outs,
                                                     float* __restrict__ norm, double limit) {
  __shared__ u64 s_tmp[16];
  NormSum<KIND> acc;
  for (u32 i = wave_id(); i < t.chunks; i += 16) norm_any<KIND, false, 64, 4>(find_chunk(t, i), lane_id(), acc);
  const float n = norm_value<KIND>(norm_block<KIND, 16>(acc.s0 + acc.s1, acc.m, s_tmp));  // its barrier: all is read
  if (threadIdx.x == 0) *norm = n;
  if (!CLIP) return;
  const float f = clip_factor(n, limit);
  if (!OUT && f == 1.0f) return;
  for (u32 i = wave_id(); i < t.chunks; i += 16) {
    const GradChunk c = find_chunk(t, i);
    scale_any<false, 64, 4>(c, OUT ? outs.addr[c.span] + c.skip : c.addr, lane_id(), f);
  }
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
// A group's four values in the common case, every |q| below 2^22: with w = 2 f + 1/2 (exact), the zigzagged integer is the
// whole part of |w|, and its width follows from w's exponent: |w| in [1/2, 1) is the integer 0, then every eight
// exponents are a byte more.  Shifted up by four the exponent's low five bits are at the top; with kWidthBias added the
// topmost two of them are the code (0124; for 1234 everything below 256 counts as 1 first).  A group is half as many
// instructions this way as by integers, and the encoder of gradients is short of issue slots, not of bytes.
template <int V>
constexpr u32 kWidthBias = V == V0124 ? 9u << 27 : 1u << 27;
constexpr float kFeedSmall = 4194304.0f;  // 2^22
template <int V>
__device__ __forceinline__ u32 feed_group(const float (&g)[4], float (&r)[4], uint4& x, float c, float scale, float step) {
#pragma clang fp contract(off)
  float f[4], left[4], w[4];
  float size = 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float e = g[k] * c + r[k];
    f[k] = rintf(e * scale);
    left[k] = e - __builtin_fmaf(f[k], step, 0.0f);  // the product; + 0 makes 0 of -0, as the integer would
    size += fabsf(f[k]);
    w[k] = __builtin_fmaf(f[k], 2.0f, 0.5f);
  }
  if (__ballot(!(size < kFeedSmall)) == 0ull) {  // also false for infinities and NaN
    u32 key = 0;
#pragma unroll
    for (int k = 3; k >= 0; --k) {
      const float m = V == V1234 ? fmaxf(fabsf(w[k]), 1.0f) : w[k];
      key = __builtin_amdgcn_alignbit(key, (__float_as_uint(m) << 4) + kWidthBias<V>, 30u);
      r[k] = left[k];
    }
    x = make_uint4((u32)fabsf(w[0]), (u32)fabsf(w[1]), (u32)fabsf(w[2]), (u32)fabsf(w[3]));
    return key;
  }
  u32 z[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) z[k] = zz_enc(feed_one(g[k], r[k], c, scale, step));
  x = make_uint4(z[0], z[1], z[2], z[3]);
  return classify_key<V>(x);
}
// Four gradients of a group, as they lie in memory.
template <int T>
struct Grad4 {
  u32x4_t w;  // float32: four dwords; 16 bits: two
  template <bool NTL>
  __device__ __forceinline__ void load(const u8* g, u64 first) {
    if (T == kF32) {
      const uint4 t = ld_stream16<NTL>(g + 4 * first);
      w = u32x4_t{t.x, t.y, t.z, t.w};
    } else {
      const u32x2_a2* p = reinterpret_cast<const u32x2_a2*>(g + 2 * first);
      const u32x2_t h = NTL ? __builtin_nontemporal_load(p) : *p;
      w = u32x4_t{h.x, h.y, 0, 0};
    }
  }
  // ... those of them that exist, 0 for the rest
  __device__ __forceinline__ void load_some(const u8* g, u64 first, u32 count) {
    w = u32x4_t{0, 0, 0, 0};
#pragma unroll
    for (u32 k = 0; k < 4; ++k)
      if (first + k < count) {
        if (T == kF32) w[k] = reinterpret_cast<const u32*>(g)[first + k];
        else w[k >> 1] |= (u32)reinterpret_cast<const unsigned short*>(g)[first + k] << (16 * (k & 1u));
      }
  }
  __device__ __forceinline__ float get(u32 k) const { return vec_elem<T>(w, k); }
};

// Byte counts of a wave tile's groups, scanned: off[j] = bytes before group j*64+lane, total = all of them.
struct WavePlaces {
  u32 off[4], total;
};
__device__ __forceinline__ WavePlaces wave_places(const u32 (&g)[4], int lane) {
  // four 16-bit counts in two dwords; a count sums to at most 64 * 16, so none carries into its neighbour
  const u32 lo = gi_total(g[0]) | (gi_total(g[1]) << 16), hi = gi_total(g[2]) | (gi_total(g[3]) << 16);
  const u32 inc_lo = wave_scan_incl(lo, lane), inc_hi = wave_scan_incl(hi, lane);
  const u32 tot_lo = wave_last(inc_lo), tot_hi = wave_last(inc_hi);
  const u32 ex_lo = inc_lo - lo, ex_hi = inc_hi - hi;
  const u32 t0 = tot_lo & 0xFFFFu, t1 = tot_lo >> 16, t2 = tot_hi & 0xFFFFu, t3 = tot_hi >> 16;
  WavePlaces p;
  p.off[0] = ex_lo & 0xFFFFu;
  p.off[1] = t0 + (ex_lo >> 16);
  p.off[2] = t0 + t1 + (ex_hi & 0xFFFFu);
  p.off[3] = t0 + t1 + t2 + (ex_hi >> 16);
  p.total = t0 + t1 + t2 + t3;
  return p;
}
// ORs the bytes of a group of at most four bytes into the zeroed image.
__device__ __forceinline__ void or_small(u8* image, u32 p, u32 L, u32 d) {
  const u32 sel = shift_selector(p);
  u32* q = reinterpret_cast<u32*>(image + (p & ~3u));
  if (L) atomicOr(q, __builtin_amdgcn_perm(d, 0u, sel));
  if (L + (p & 3u) > 4u) atomicOr(q + 1, __builtin_amdgcn_perm(0u, d, sel));
}
// A wave tile's data bytes and keys into the wave's LDS image, from byte 0 of it: where the image goes is not known yet.
// A quarter in which every value fits a byte -- most quarters of quantised gradients -- needs neither the 64-bit shifts
// of the general packing nor its five dwords a group.
template <int V, bool FULL>
__device__ __forceinline__ void assemble(const uint4 (&x)[4], const u32 (&g)[4], const WavePlaces& p, int lane, EncWaveLds& S) {
#pragma unroll
  for (int j = 0; j < 4; ++j) S.keys[j * 64 + lane] = (u8)gi_key(g[j]);
  if (V == V1234) {
    // plain dword stores, later groups first; see encode_wavetile
    u32 head[4];
#pragma unroll
    for (int j = 3; j >= 0; --j) {
      const GroupSlot s = group_slot<FULL>(S.data, p.off[j], g[j]);
      if (FULL && __ballot(gi_key(g[j]) != 0u) == 0ull) {
        const uint4 d = make_uint4(x[j].x | (x[j].y << 8) | (x[j].z << 16) | (x[j].w << 24), 0, 0, 0);
        store_dword<0, FULL>(s, d);
        store_dword<1, FULL>(s, d);
        head[j] = d.x;
      } else {
        const uint4 d = pack_group<V>(x[j], g[j]);
        store_dword<0, FULL>(s, d);
        store_dword<1, FULL>(s, d);
        store_dword<2, FULL>(s, d);
        store_dword<3, FULL>(s, d);
        store_dword<4, FULL>(s, d);
        head[j] = d.x;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) store_head<FULL>(S.data, head[j], p.off[j], g[j]);
  } else {
    const u32 nz = (p.total + 15u) >> 4;
    uint4* l16 = reinterpret_cast<uint4*>(S.data);
    for (u32 c = lane; c < nz; c += 64) l16[c] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const u32 k = gi_key(g[j]);
      if (__ballot((k & 0xAAu) != 0u) == 0ull) {  // codes 0 and 1 only
        u32 d = x[j].w;
        d = (d << ((k >> 1) & 8u)) | x[j].z;
        d = (d << ((k << 1) & 8u)) | x[j].y;
        d = (d << ((k << 3) & 8u)) | x[j].x;
        or_small(S.data, p.off[j], gi_total(g[j]), d);
      } else {
        or_into_image(S.data, p.off[j], gi_total(g[j]), pack_group<V>(x[j], g[j]));
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
typedef u32x4_t u32x4_a1 __attribute__((aligned(1)));
// The image to its place.  The stream starts anywhere, so the 16-byte stores do too.
template <bool NTS>
__device__ __forceinline__ void copy_out(const EncWaveLds& S, u32 total, u32 nkeys, int lane, u8* dst, u8* kdst) {
  const u32x4_t* l16 = reinterpret_cast<const u32x4_t*>(S.data);
  u32x4_a1* g16 = reinterpret_cast<u32x4_a1*>(dst);
  const u32 whole = total >> 4;
  for (u32 c = lane; c < whole; c += 64) {
    if (NTS) __builtin_nontemporal_store(l16[c], g16 + c);
    else g16[c] = l16[c];
  }
  const u32 rest = 16u * whole + lane;
  if (rest < total) dst[rest] = S.data[rest];
  if (4u * lane + 4u <= nkeys) st_u32(kdst + 4 * lane, reinterpret_cast<const u32*>(S.keys)[lane]);
  else
    for (u32 b = 4u * lane; b < nkeys; ++b) kdst[b] = S.keys[b];
}

// Values of the group from `first` on that exist, and of a lane's four groups of a wave tile.
__device__ __forceinline__ u32 present(u64 first, u32 count) { return first < count ? (u32)min((u64)4, (u64)count - first) : 0u; }
__device__ __forceinline__ u32 present_lane(u64 wt_first, int lane, u32 count) {
  u32 n = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) n += present(wt_first + (u32)(4 * (j * 64 + lane)), count);
  return n;
}
constexpr u32 kFeedMaxWaves = 15;  // data waves of a workgroup, at most
// One pass.  A workgroup takes tiles off a ticket, QW wave tiles (of 1024 values) for each of its first nw waves; its
// last wave, the scan wave, draws the tickets and finds the tiles' places by look-back.  A data wave's round k:
//     quantise (values and residuals have arrived), send the new residuals off, count the bytes   | barrier A |
//     assemble the bytes in LDS, request the next tile's values and residuals
//     DEFER: copy out the tile of round k - 1, whose bytes have waited in the other image;  else: | barrier B | copy out
// and the scan wave's:
//     draw the next ticket (DEFER: after the publication) | A | publish the tile's bytes, look back until the place is known | B
// (without B in all but the last round of DEFER),
// so a tile's look-back runs beside its assembly and the next tile's loads (DEFER: beside a whole round), and the polls
// never stand in a queue with a data wave's loads and stores.  The loads go out only when the bytes are assembled: sent
// at the start of the round they are ahead of the polls in the CU's memory queue, which lengthens every look-back by
// more than they gain (2^25 values 107 us instead of 87).  The barriers order LDS only: __syncthreads would wait for the
// stores as well.  What the scan wave hands over has two places, the byte counts three: nobody who still reads round k
// is passed by a writer of the round that takes the same place.  Between a tile's ticket and its publication a workgroup
// waits only for tiles with smaller tickets: the chain ends.
//
// Bound by memory, 12.8 B a value for float32 (0124): 2^26 values in 140 us = 6.2 TB/s.  What it took to get there from 187 us, the tile-at-a-time form of k_encode: assembling before the place is
// known (165), half the instructions a value (feed_group, the one-byte quarters of assemble), one workgroup of 15 data
// waves per CU instead of two (158; a look-back takes the longer the more tiles are in flight, about 20 ns each), the
// deferred copy (144; 30 wave tiles a tile without it 151), 256 tile words a look-back instead of 128 (140: all that are
// in flight, so none waits for a group's leader).  The ticket drawn after the look-back instead of before it costs 10 us.
template <int V, int T, int QW, bool DEFER, int NT>
__global__ __launch_bounds__(kFeedMaxWaves * 64 + 64, 4) void k_feedback_encode(const u8* __restrict__ grad, u32 count, u32 n_tiles,
                                                                                u32 nw, u8* __restrict__ out, FeedArgs fa,
                                                                                WsHeader* __restrict__ hdr, LbWords lb,
                                                                                u64* __restrict__ written) {
  __shared__ EncWaveLds s_lds[DEFER ? 2 : 1][kFeedMaxWaves * QW];
  __shared__ u32 s_wave_tot[3][kFeedMaxWaves];
  __shared__ u64 s_prefix[2];
  __shared__ u32 s_first, s_next[2];
  const int lane = lane_id(), wave = wave_id();
  const u64 keylen = ((u64)count + 3) >> 2;
  if (wave == (int)nw) {  // the scan wave
    auto draw = [&]() -> u32 {
      u32 t = 0;
      if (lane == 0) t = atomicAdd(&hdr->ticket, 1u);
      return __builtin_amdgcn_readfirstlane(t);
    };
    const bool once = gridDim.x >= n_tiles;  // a workgroup per tile: nobody takes a second one
    u32 tile = n_tiles > 1 ? draw() : 0u;
    if (lane == 0) s_first = tile;
    lds_barrier();
    if (tile >= n_tiles) return;
    u32 next = n_tiles;
    for (u32 k = 0;; ++k) {
      if (!DEFER || k == 0) {
        next = once ? n_tiles : draw();
        if (lane == 0) s_next[k & 1] = next;
      }
      lds_barrier();  // A
      const u32 tile_tot = wave_sum(lane < (int)nw ? s_wave_tot[k % 3][lane] : 0u);
      lb2_publish(lb, tile, tile_tot, lane, &hdr->error);
      u32 after = n_tiles;
      if (DEFER && next < n_tiles) after = draw();
      const u64 excl = lb2_resolve<4>(lb, tile, tile_tot, lane, &hdr->error);
      if (lane == 0) {
        s_prefix[k & 1] = excl;
        if (DEFER) s_next[(k + 1) & 1] = after;
        if (tile == n_tiles - 1 && written) *written = keylen + excl + tile_tot;
        if (tile == 0u) reset_other_ticket(hdr);
      }
      if (!DEFER || next >= n_tiles) lds_barrier();  // B
      if (next >= n_tiles) return;
      tile = next;
      next = after;
    }
  }
  const float c = fa.norm ? clip_factor(*fa.norm, fa.limit) : 1.0f;
  Grad4<T> gr[QW][4];
  uint4 r[QW][4];
  auto first_of = [&](u32 tile, int q) -> u64 { return (((u64)tile * nw + wave) * QW + q) * kWtInts; };
  auto request = [&](u32 tile, int q) {
    const u64 wt_first = tile < n_tiles ? first_of(tile, q) : count;
    if (wt_first + kWtInts <= count) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u64 first = wt_first + (u32)(4 * (j * 64 + lane));
        gr[q][j].template load<(NT & kNtLoads) != 0>(grad, first);
        r[q][j] = ld_stream16<(NT & kNtLoads) != 0>(fa.r_in + first);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u64 first = wt_first + (u32)(4 * (j * 64 + lane));
        gr[q][j].load_some(grad, first, count);
        r[q][j] = load_group(reinterpret_cast<const u32*>(fa.r_in), first, count);
      }
    }
  };
  u32 done = 0;          // the tile of round `k` that `totals` is about
  u32 totals[QW] = {};   // bytes of its wave tiles
  auto finish = [&](u32 k) {
    u64 doff = keylen + s_prefix[k & 1];
    for (int w = 0; w < wave; ++w) doff += s_wave_tot[k % 3][w];
#pragma unroll
    for (int q = 0; q < QW; ++q) {
      const u64 wt_first = first_of(done, q);
      if (wt_first < count)
        copy_out<(NT & kNtStores) != 0>(s_lds[DEFER ? k & 1 : 0][wave * QW + q], totals[q],
                                        (u32)((min((u64)kWtInts, (u64)count - wt_first) + 3) >> 2), lane, out + doff, out + (wt_first >> 2));
      doff += totals[q];
    }
  };
  lds_barrier();
  u32 tile = __builtin_amdgcn_readfirstlane(s_first);
  if (tile >= n_tiles) return;
#pragma unroll
  for (int q = 0; q < QW; ++q) request(tile, q);
  for (u32 k = 0;; ++k) {
    uint4 x[QW][4];  // the zigzagged integers
    u32 k4[QW];      // their groups' keys
    u32 lane_tot = 0;
#pragma unroll
    for (int q = 0; q < QW; ++q) {
      const u64 wt_first = first_of(tile, q);
      const bool full = wt_first + kWtInts <= count;  // wave-uniform
      u32 keys = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float gv[4] = {gr[q][j].get(0), gr[q][j].get(1), gr[q][j].get(2), gr[q][j].get(3)};
        float rv[4] = {__uint_as_float(r[q][j].x), __uint_as_float(r[q][j].y), __uint_as_float(r[q][j].z), __uint_as_float(r[q][j].w)};
        u32 key = feed_group<V>(gv, rv, x[q][j], c, fa.scale, fa.step);
        const u64 first = wt_first + (u32)(4 * (j * 64 + lane));
        if (full) {
          st_stream16<(NT & kNtStores) != 0>(fa.r_out + first, make_uint4(__float_as_uint(rv[0]), __float_as_uint(rv[1]),
                                                                          __float_as_uint(rv[2]), __float_as_uint(rv[3])));
        } else {
          const u32 nv = present(first, count);
#pragma unroll
          for (u32 i = 0; i < 4; ++i)
            if (i < nv) fa.r_out[first + i] = rv[i];
          zero_absent(x[q][j], first, count);
          key &= (1u << (2u * nv)) - 1u;
        }
        keys |= key << (8 * j);
      }
      asm volatile("" : "+v"(keys));  // the four keys stay in one register
      k4[q] = keys;
      lane_tot += full || V == V0124 ? word_len<V>(keys, 16u) : word_len<V>(keys, present_lane(wt_first, lane, count));
    }
    const u32 wave_tot = wave_sum(lane_tot);
    if (lane == 0) s_wave_tot[k % 3][wave] = wave_tot;
    lds_barrier();  // A
    const u32 next = __builtin_amdgcn_readfirstlane(s_next[k & 1]);
    u32 mine[QW];
#pragma unroll
    for (int q = 0; q < QW; ++q) {
      const u64 wt_first = first_of(tile, q);
      const bool full = wt_first + kWtInts <= count;
      u32 lens4 = key_lens4<V>(k4[q], 16u);
      if (!full && V == V1234) {
        lens4 = code_sums4(k4[q]);
#pragma unroll
        for (int j = 0; j < 4; ++j) lens4 += present(wt_first + (u32)(4 * (j * 64 + lane)), count) << (8 * j);
      }
      u32 g[4];  // the groups' descriptors
#pragma unroll
      for (int j = 0; j < 4; ++j) g[j] = ((k4[q] >> (8 * j)) & 0xFFu) | (((lens4 >> (8 * j)) & 0xFFu) << 24);
      const WavePlaces places = wave_places(g, lane);
      mine[q] = places.total;
      EncWaveLds& S = s_lds[DEFER ? k & 1 : 0][wave * QW + q];
      if (full) assemble<V, true>(x[q], g, places, lane, S);
      else assemble<V, false>(x[q], g, places, lane, S);
      __builtin_amdgcn_sched_barrier(0);
      request(next, q);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (DEFER && k) finish(k - 1);
    done = tile;
#pragma unroll
    for (int q = 0; q < QW; ++q) totals[q] = mine[q];
    if (!DEFER || next >= n_tiles) {
      lds_barrier();  // B
      finish(k);
    }
    if (next >= n_tiles) return;
    tile = next;
  }
}

}  // namespace svb
