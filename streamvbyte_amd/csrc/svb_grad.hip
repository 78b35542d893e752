// C ABI of the gradient operators (include/streamvbyte_gpu.h): svbgpu_grad_norm, svbgpu_grad_clip,
// svbgpu_quantize_feedback_encode.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>

#include "../../include/streamvbyte.h"
#include "../../include/streamvbyte_gpu.h"
#include "svb_grad.h"
#include "svb_host.h"

using namespace svb;

namespace {

#define GRAD_HIP(expr)                                 \
  do {                                                 \
    const hipError_t e_ = (expr);                      \
    if (e_ != hipSuccess) return host::fail_hip(e_);   \
  } while (0)

inline hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }

constexpr u64 kCacheBytes = 256ull << 20;  // Infinity Cache
constexpr u32 kNormMinChunk = 64 << 10;   // bytes of a norm's chunk ...
constexpr u32 kNormChunks = 4096;         // ... which grows so that there are no more than this many, and one a tensor
constexpr u64 kMaxSetBytes = (u64)kNormChunks << 31;  // a chunk's bytes fit 32 bits: what a workspace has words for
constexpr u32 kMaxTensors = 1u << 31;     // with it the chunks of all launches fit 32 bits

bool bad_type(int t) { return t != SVBGPU_F32 && t != SVBGPU_F16 && t != SVBGPU_BF16; }
bool bad_norm(int n) { return n != SVBGPU_NORM_MAX && n != SVBGPU_NORM_L1 && n != SVBGPU_NORM_L2; }
u32 elem_bytes(int type) { return type == SVBGPU_F32 ? 4u : 2u; }
bool overlap(const void* a, u64 an, const void* b, u64 bn) {
  const u64 x = (u64)(uintptr_t)a, y = (u64)(uintptr_t)b;
  return an && bn && x < y + bn && y < x + an;
}

// Arguments of the tensors themselves; total = bytes of all of them.
int check_tensors(const svbgpu_tensor* t, uint32_t n, u64* total) {
  *total = 0;
  if (n && !t) return SVBGPU_EINVAL;
  if (n > kMaxTensors) return SVBGPU_EINVAL;
  for (uint32_t i = 0; i < n; ++i) {
    if (bad_type(t[i].type)) return SVBGPU_EINVAL;
    if (!t[i].count) continue;
    const u32 b = elem_bytes(t[i].type);
    const u64 a = (u64)(uintptr_t)t[i].data;
    if (!a || (a & (b - 1)) || a >> kAddrBits || t[i].count >> (kCountBits - 3)) return SVBGPU_EINVAL;
    *total += t[i].count * b;
    if (*total > kMaxSetBytes) return SVBGPU_EINVAL;
  }
  return SVBGPU_OK;
}

struct Range {
  u64 begin, end;
};
bool by_begin(const Range& a, const Range& b) { return a.begin < b.begin; }
// No memory that a clip writes may be written twice, or read for another tensor than its own.
int check_written(const svbgpu_tensor* t, uint32_t n, void* const* outs) {
  Range on_stack[256];
  Range* r = n <= 256 ? on_stack : new (std::nothrow) Range[n];
  if (!r) return SVBGPU_ENOMEM;
  uint32_t m = 0;
  bool sorted = true, fine = true;
  for (uint32_t i = 0; i < n; ++i) {
    if (!t[i].count) continue;
    const u64 begin = (u64)(uintptr_t)(outs ? outs[i] : t[i].data), bytes = t[i].count * elem_bytes(t[i].type);
    if (!begin || (begin & (elem_bytes(t[i].type) - 1)) || begin >> kAddrBits) { fine = false; break; }
    if (m && begin < r[m - 1].begin) sorted = false;
    r[m++] = Range{begin, begin + bytes};
  }
  if (fine && !sorted) std::sort(r, r + m, by_begin);
  for (uint32_t i = 1; fine && i < m; ++i) fine = r[i - 1].end <= r[i].begin;
  if (fine && outs) {  // neighbours in memory are one range from here on: the views of a bucket come down to the bucket
    uint32_t k = 0;
    for (uint32_t i = 1; i < m; ++i) {
      if (r[i].begin == r[k].end) r[k].end = r[i].end;
      else r[++k] = r[i];
    }
    m = m ? k + 1 : 0;
    for (uint32_t i = 0; fine && i < n; ++i) {  // an input may meet its own output, exactly, and no other
      if (!t[i].count || outs[i] == t[i].data) continue;
      const u64 begin = (u64)(uintptr_t)t[i].data, end = begin + t[i].count * elem_bytes(t[i].type);
      const Range* after = std::lower_bound(r, r + m, Range{end, 0}, by_begin);  // the first that starts at or after the end
      fine = after == r || after[-1].end <= begin;
    }
  }
  if (r != on_stack) delete[] r;
  return fine ? SVBGPU_OK : SVBGPU_EINVAL;
}

u32 chunks_of(const svbgpu_tensor& t, u32 chunk_bytes) {
  const u64 elems = chunk_bytes / elem_bytes(t.type);
  return (u32)((t.count + elems - 1) / elems);
}
// Appends a tensor to a launch's table.
template <u32 N>
void append(GradTable<N>& table, const svbgpu_tensor& t) {
  table.span[table.n++] = GradSpan{(u64)(uintptr_t)t.data | ((u64)t.type << kAddrBits), ((u64)table.chunks << kCountBits) | t.count};
  table.chunks += chunks_of(t, table.chunk_bytes);
}
// Chunks small enough for a wave and few enough for one workgroup?
bool is_small(const svbgpu_tensor* t, uint32_t n, u64 total) {
  if (total > (u64)kSmallChunk * kSmallChunks) return false;
  u32 chunks = 0, spans = 0;
  for (uint32_t i = 0; i < n; ++i)
    if (t[i].count) {
      chunks += chunks_of(t[i], kSmallChunk);
      if (++spans > kMaxSpansSmall || chunks > kSmallChunks) return false;
    }
  return true;
}

template <int KIND>
int launch_small(const svbgpu_tensor* t, uint32_t n, void* const* outs, bool clip, float* d_norm, double limit, hipStream_t st) {
  GradTable<kMaxSpansSmall> table;
  GradOuts<kMaxSpansSmall> o;
  table.n = table.chunks = 0;
  table.chunk_bytes = kSmallChunk;
  for (uint32_t i = 0; i < n; ++i)
    if (t[i].count) {
      o.addr[table.n] = outs ? (u64)(uintptr_t)outs[i] : 0;
      append(table, t[i]);
    }
  if (!clip) hipLaunchKernelGGL((k_grad_small<KIND, false, false>), dim3(1), dim3(1024), 0, st, table, o, d_norm, limit);
  else if (outs) hipLaunchKernelGGL((k_grad_small<KIND, true, true>), dim3(1), dim3(1024), 0, st, table, o, d_norm, limit);
  else hipLaunchKernelGGL((k_grad_small<KIND, true, false>), dim3(1), dim3(1024), 0, st, table, o, d_norm, limit);
  GRAD_HIP(hipGetLastError());
  return SVBGPU_OK;
}
// keep: bytes at the end of the set that are read to stay in the cache.
template <int KIND>
int launch_norm(const svbgpu_tensor* t, uint32_t n, u64 total, u64 keep, float* d_norm, u64* partial, hipStream_t st) {
  u64 chunk = kNormMinChunk;
  while (chunk * kNormChunks < total) chunk <<= 1;  // 2^31 at most: check_tensors
  GradTable<kMaxSpans> table;
  table.chunk_bytes = (u32)chunk;
  const u64 passing = total > keep ? total - keep : 0;  // bytes read to pass
  u64 bytes = 0;                                        // ... of the set that earlier launches read
  u32 before = 0;                                       // chunks of earlier launches
  for (uint32_t i = 0; i < n;) {
    u64 mine = 0;
    table.n = table.chunks = 0;
    for (; i < n && table.n < kMaxSpans; ++i)
      if (t[i].count) {
        append(table, t[i]);
        mine += t[i].count * elem_bytes(t[i].type);
      }
    if (!table.n) break;
    const u32 nt = passing <= bytes ? 0 : passing >= bytes + mine ? table.chunks : (u32)((double)(passing - bytes) / (double)mine * table.chunks);
    hipLaunchKernelGGL(k_grad_norm<KIND>, dim3(table.chunks), dim3(kNormThreads), 0, st, table, partial + before, nt);
    GRAD_HIP(hipGetLastError());
    before += table.chunks;
    bytes += mine;
  }
  hipLaunchKernelGGL(k_grad_finish<KIND>, dim3(1), dim3(1024), 0, st, partial, before, d_norm);
  GRAD_HIP(hipGetLastError());
  return SVBGPU_OK;
}
// y = x * factor, the last tensors first.
int launch_scale(const svbgpu_tensor* t, uint32_t n, u64 total, void* const* outs, const float* d_norm, double limit, hipStream_t st) {
  const bool nt = (host::nt_policy(total, total) & kNtStores) != 0;
  GradTable<kMaxSpansOut> table;
  GradOuts<kMaxSpansOut> o;
  uint32_t of_span[kMaxSpansOut];
  table.chunk_bytes = kScaleChunk;
  while ((u64)table.chunk_bytes << 23 < total) table.chunk_bytes <<= 1;  // the chunks' index has 24 bits
  for (uint32_t i = n; i;) {
    u32 k = 0;
    for (; i && k < kMaxSpansOut; --i)
      if (t[i - 1].count) of_span[k++] = i - 1;
    if (!k) break;
    table.n = table.chunks = 0;
    while (k--) {  // in the set's order, which the kernel takes from the end
      o.addr[table.n] = outs ? (u64)(uintptr_t)outs[of_span[k]] : 0;
      append(table, t[of_span[k]]);
    }
    const dim3 grid(table.chunks), block(kScaleThreads);
    if (outs && nt) hipLaunchKernelGGL((k_grad_scale<true, true>), grid, block, 0, st, table, o, d_norm, limit);
    else if (outs) hipLaunchKernelGGL((k_grad_scale<true, false>), grid, block, 0, st, table, o, d_norm, limit);
    else if (nt) hipLaunchKernelGGL((k_grad_scale<false, true>), grid, block, 0, st, table, o, d_norm, limit);
    else hipLaunchKernelGGL((k_grad_scale<false, false>), grid, block, 0, st, table, o, d_norm, limit);
    GRAD_HIP(hipGetLastError());
  }
  return SVBGPU_OK;
}
template <int KIND>
int run_kind(const svbgpu_tensor* t, uint32_t n, u64 total, void* const* outs, bool clip, double limit, float* d_norm, void* ws,
             hipStream_t st) {
  if (is_small(t, n, total)) return launch_small<KIND>(t, n, outs, clip, d_norm, limit, st);
  const u64 keep = clip ? kCacheBytes : (host::nt_policy(total, 0) & kNtLoads) ? 0 : total;
  const int rc = launch_norm<KIND>(t, n, total, keep, d_norm, static_cast<u64*>(ws), st);
  return rc || !clip ? rc : launch_scale(t, n, total, outs, d_norm, limit, st);
}
int run(int kind, const svbgpu_tensor* t, uint32_t n, u64 total, void* const* outs, bool clip, double limit, float* d_norm, void* ws,
        hipStream_t st) {
  if (kind == SVBGPU_NORM_MAX) return run_kind<kNormMax>(t, n, total, outs, clip, limit, d_norm, ws, st);
  if (kind == SVBGPU_NORM_L1) return run_kind<kNormSum>(t, n, total, outs, clip, limit, d_norm, ws, st);
  return run_kind<kNormEuclid>(t, n, total, outs, clip, limit, d_norm, ws, st);
}

template <int V, int T, int QW, bool DEFER, int NT, u32 NW>
void launch_feedback(const void* grad, uint32_t count, uint8_t* d_out, const FeedArgs& fa, void* ws, unsigned tag2,
                     uint64_t* d_written, hipStream_t st) {
  static_assert(NW * QW >= kWaves, "the workspace has a look-back word per kWaves wave tiles");
  static_assert(NW <= kFeedMaxWaves, "the kernel's LDS holds that many waves' images");
  const WsLayout L = ws_layout(count);
  const u32 tile = NW * QW * kWtInts, tiles = (u32)(((u64)count + tile - 1) / tile);
  const u32 grid = std::min<u32>(tiles, (u32)std::max(host::device_cus(), 1));
  WsHeader* h = reinterpret_cast<WsHeader*>(static_cast<char*>(ws) + ((tag2 >> 3) & 1u) * 8);
  const LbWords lb{reinterpret_cast<u64*>(static_cast<char*>(ws) + L.off_status), (u32)((L.off_lb_group - L.off_status) / 8), tag2};
  hipLaunchKernelGGL((k_feedback_encode<V, T, QW, DEFER, NT>), dim3(grid), dim3((NW + 1) * 64), 0, st, static_cast<const u8*>(grad), count,
                     tiles, NW, d_out, fa, h, lb, d_written);
}
// The tile by size.  A large tile means few look-backs, a small one that a short stream reaches more of the device; the
// deferred copy hides the look-backs where a workgroup takes several tiles.  Measured with float32, 0124, us for QW x nw
// wave tiles a tile:
//     2^18 values: 1x4 6.3, 1x8 6.7, 1x15 7.9                2^20: 1x4 10.4, 1x8 8.6, 1x15 8.9
//     2^21: 1x8 12.4, 1x15 11.3, 2x12 12.2                   3 * 2^20: 1x15 13.2, 2x12 13.8, deferred 13.6
//     2^22: 1x15 17.4, 2x12 15.6, deferred 17.1              6 * 2^20: 1x15 22.3, 2x12 20.0, deferred 20.6
//     7 * 2^20: 2x12 26.4, 2x15 22.1, deferred 23.6          2^23: 1x15 27.0, 2x12 27.2, deferred 25.3
//     12 * 2^20: 1x15 40.6, 2x12 37.3, deferred 35.6         2^24: 1x15 51.2, 2x12 48.7, deferred 45.0
//     2^26: 1x15 163, 2x15 152, deferred 140
// Two wave tiles a wave are for streams that are one round of the device's 256 CUs that way and more with one.
// Non-temporal stores from 7 * 2^19 values (47 MB read and written, 40 MB with 16-bit gradients), non-temporal loads from
// 2^24 (215 and 180 MB): deferred, 2^23 27.9 us, with such stores 25.3, with the loads too 27.4; 2^24 47.5, 45.0, 44.2.
// What reads the stream or the residual next has not been timed with either.  16-bit gradients and 1234 go by the same
// counts, which were not measured for them.
template <int V, int T>
void launch_feedback(const void* grad, uint32_t count, uint8_t* d_out, const FeedArgs& fa, void* ws, unsigned tag2, uint64_t* d_written,
                     hipStream_t st) {
  const u32 m = count >> 19;  // in half millions
  const auto go = [&](auto launch) { launch(grad, count, d_out, fa, ws, tag2, d_written, st); };
  if (m < 1) go(launch_feedback<V, T, 1, false, 0, 4>);
  else if (m < 3) go(launch_feedback<V, T, 1, false, 0, 8>);
  else if (m < 7) go(launch_feedback<V, T, 1, false, 0, 15>);
  else if (m < 12) go(launch_feedback<V, T, 2, false, kNtStores, 12>);
  else if (m < 15) go(launch_feedback<V, T, 2, false, kNtStores, 15>);
  else if (m < 32) go(launch_feedback<V, T, 1, true, kNtStores, 15>);
  else go(launch_feedback<V, T, 1, true, kNtLoads | kNtStores, 15>);
}

}  // namespace

extern "C" {

size_t svbgpu_grad_workspace_bytes(uint32_t ntensors) { return align256(8 * ((size_t)kNormChunks + ntensors)); }

int svbgpu_grad_norm(int norm, const svbgpu_tensor* tensors, uint32_t ntensors, float* d_norm, void* ws, size_t ws_bytes, void* stream) {
  u64 total;
  if (bad_norm(norm) || !d_norm || ((uintptr_t)d_norm & 3u)) return SVBGPU_EINVAL;
  const int rc = check_tensors(tensors, ntensors, &total);
  if (rc) return rc;
  if (!ws || ((uintptr_t)ws & 255u) || ws_bytes < svbgpu_grad_workspace_bytes(ntensors)) return SVBGPU_EWORKSPACE;
  if (!host::device_ok()) return SVBGPU_ENODEVICE;
  return run(norm, tensors, ntensors, total, nullptr, false, 0.0, d_norm, ws, S(stream));
}

int svbgpu_grad_clip(int norm, const svbgpu_tensor* tensors, uint32_t ntensors, void* const* outs, double max_norm, int norm_given,
                     float* d_norm, void* ws, size_t ws_bytes, void* stream) {
  u64 total;
  if ((!norm_given && bad_norm(norm)) || !d_norm || ((uintptr_t)d_norm & 3u) || !(max_norm >= 0.0)) return SVBGPU_EINVAL;
  int rc = check_tensors(tensors, ntensors, &total);
  if (!rc) rc = check_written(tensors, ntensors, outs);
  if (rc) return rc;
  for (uint32_t i = 0; i < ntensors; ++i) {  // the norm is read while tensors are written
    const u64 bytes = tensors[i].count * elem_bytes(tensors[i].type);
    if (overlap(d_norm, 4, tensors[i].data, bytes) || (outs && overlap(d_norm, 4, outs[i], bytes))) return SVBGPU_EINVAL;
  }
  if (!norm_given && (!ws || ((uintptr_t)ws & 255u) || ws_bytes < svbgpu_grad_workspace_bytes(ntensors))) return SVBGPU_EWORKSPACE;
  if (!host::device_ok()) return SVBGPU_ENODEVICE;
  if (norm_given) return launch_scale(tensors, ntensors, total, outs, d_norm, max_norm, S(stream));
  return run(norm, tensors, ntensors, total, outs, true, max_norm, d_norm, ws, S(stream));
}

int svbgpu_quantize_feedback_encode(int variant, int type, const void* d_grad, uint32_t count, const float* d_norm, double max_norm,
                                    float scale, const float* d_residual, float* d_residual_out, uint8_t* d_out, void* ws,
                                    size_t ws_bytes, uint64_t* d_written, void* stream) {
  if ((variant != SVBGPU_1234 && variant != SVBGPU_0124) || bad_type(type)) return SVBGPU_EINVAL;
  const float step = 1.0f / scale;
  if (!std::isnormal(scale) || !(scale > 0.0f) || !std::isnormal(step)) return SVBGPU_EINVAL;
  if (d_norm && (!(max_norm >= 0.0) || ((uintptr_t)d_norm & 3u))) return SVBGPU_EINVAL;
  if (count == 0) return d_written ? host::fill_u32(d_written, 0u, 8, S(stream)) : SVBGPU_OK;
  const u64 grad_bytes = (u64)count * elem_bytes(type), res_bytes = 4ull * count, out_bytes = streamvbyte_max_compressedbytes(count);
  if (!d_grad || !d_residual || !d_residual_out || !d_out) return SVBGPU_EINVAL;
  if (((uintptr_t)d_grad & (elem_bytes(type) - 1)) || ((uintptr_t)d_residual & 3u) || ((uintptr_t)d_residual_out & 3u)) return SVBGPU_EINVAL;
  if (d_residual != d_residual_out && overlap(d_residual, res_bytes, d_residual_out, res_bytes)) return SVBGPU_EINVAL;
  if (overlap(d_grad, grad_bytes, d_residual_out, res_bytes) || overlap(d_out, out_bytes, d_grad, grad_bytes) ||
      overlap(d_out, out_bytes, d_residual, res_bytes) || overlap(d_out, out_bytes, d_residual_out, res_bytes))
    return SVBGPU_EINVAL;
  if (d_norm && (overlap(d_norm, 4, d_residual_out, res_bytes) || overlap(d_norm, 4, d_out, out_bytes))) return SVBGPU_EINVAL;
  if (!host::device_ok()) return SVBGPU_ENODEVICE;
  hipStream_t st = S(stream);
  unsigned tag2 = 0;
  const int rc = host::begin_lookback(count, ws, ws_bytes, st, &tag2);
  if (rc) return rc;
  const FeedArgs fa{d_norm, max_norm, scale, step, d_residual, d_residual_out};
  const bool v0 = variant == SVBGPU_1234;
  if (type == SVBGPU_F32) {
    if (v0) launch_feedback<V1234, kF32>(d_grad, count, d_out, fa, ws, tag2, d_written, st);
    else launch_feedback<V0124, kF32>(d_grad, count, d_out, fa, ws, tag2, d_written, st);
  } else if (type == SVBGPU_F16) {
    if (v0) launch_feedback<V1234, kF16>(d_grad, count, d_out, fa, ws, tag2, d_written, st);
    else launch_feedback<V0124, kF16>(d_grad, count, d_out, fa, ws, tag2, d_written, st);
  } else {
    if (v0) launch_feedback<V1234, kBF16>(d_grad, count, d_out, fa, ws, tag2, d_written, st);
    else launch_feedback<V0124, kBF16>(d_grad, count, d_out, fa, ws, tag2, d_written, st);
  }
  GRAD_HIP(hipGetLastError());
  return host::end_lookback(ws, st, tag2);
}

}  // extern "C"
