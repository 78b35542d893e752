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

constexpr u32 kGradChunks = 8192;      // chunks of one call, apart from one a tensor
constexpr u32 kMaxTensors = 1u << 22;  // so that a chunk's index fits 24 bits

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
  }
  return SVBGPU_OK;
}

struct Range {
  u64 begin, end;
  uint32_t index;
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
    r[m++] = Range{begin, begin + bytes, i};
  }
  if (fine && !sorted) std::sort(r, r + m, by_begin);
  for (uint32_t i = 1; fine && i < m; ++i) fine = r[i - 1].end <= r[i].begin;
  for (uint32_t i = 0; fine && outs && i < n; ++i) {  // an input may meet its own output, exactly, and no other
    if (!t[i].count || outs[i] == t[i].data) continue;
    const u64 begin = (u64)(uintptr_t)t[i].data, end = begin + t[i].count * elem_bytes(t[i].type);
    const Range* after = std::lower_bound(r, r + m, Range{end, 0, 0}, by_begin);  // the first that starts at or after the end
    fine = after == r || after[-1].end <= begin;
  }
  if (r != on_stack) delete[] r;
  return fine ? SVBGPU_OK : SVBGPU_EINVAL;
}

u32 chunk_bytes_of(u64 total) {
  u64 c = kGradMinChunk;
  while (c * kGradChunks < total) c <<= 1;
  return (u32)std::min<u64>(c, 1u << 31);
}

// Cuts the tensors into launches of at most N spans; launch(table, first tensor of span 0.., chunks, chunks before).
template <u32 N, class F>
int for_launches(const svbgpu_tensor* t, uint32_t n, u32 chunk_bytes, F launch) {
  GradTable<N> table;
  uint32_t of_span[N];
  u32 before = 0, chunks = 0;
  table.n = 0;
  table.chunk_bytes = chunk_bytes;
  for (uint32_t i = 0; i <= n; ++i) {
    if (table.n == N || (i == n && table.n)) {
      const int rc = launch(table, of_span, chunks, before);
      if (rc) return rc;
      before += chunks;
      chunks = 0;
      table.n = 0;
    }
    if (i == n || !t[i].count) continue;
    table.span[table.n] = GradSpan{(u64)(uintptr_t)t[i].data | ((u64)t[i].type << kAddrBits), ((u64)chunks << kCountBits) | t[i].count};
    of_span[table.n++] = i;
    const u64 elems = chunk_bytes / elem_bytes(t[i].type);
    chunks += (u32)((t[i].count + elems - 1) / elems);
  }
  return SVBGPU_OK;
}

template <int KIND>
int run_norm(const svbgpu_tensor* t, uint32_t n, u64 total, float* d_norm, u64* partial, hipStream_t st) {
  u32 chunks_all = 0;
  const int rc = for_launches<kMaxSpans>(t, n, chunk_bytes_of(total), [&](const GradTable<kMaxSpans>& table, const uint32_t*, u32 chunks, u32 before) {
    hipLaunchKernelGGL(k_grad_norm<KIND>, dim3(chunks), dim3(kGradThreads), 0, st, table, partial + before);
    GRAD_HIP(hipGetLastError());
    chunks_all = before + chunks;
    return SVBGPU_OK;
  });
  if (rc) return rc;
  hipLaunchKernelGGL(k_grad_finish<KIND>, dim3(1), dim3(1024), 0, st, partial, chunks_all, d_norm);
  GRAD_HIP(hipGetLastError());
  return SVBGPU_OK;
}
int norm_of(int kind, const svbgpu_tensor* t, uint32_t n, u64 total, float* d_norm, void* ws, hipStream_t st) {
  u64* partial = static_cast<u64*>(ws);
  if (kind == SVBGPU_NORM_MAX) return run_norm<kNormMax>(t, n, total, d_norm, partial, st);
  if (kind == SVBGPU_NORM_L1) return run_norm<kNormSum>(t, n, total, d_norm, partial, st);
  return run_norm<kNormEuclid>(t, n, total, d_norm, partial, st);
}

template <int V, int T, int QW, int NT>
void launch_feedback(u32 nw, const void* grad, uint32_t count, uint8_t* d_out, const FeedArgs& fa, void* ws, unsigned tag2,
                     uint64_t* d_written, hipStream_t st) {
  const WsLayout L = ws_layout(count);  // has a look-back word per kWaves wave tiles: nw * QW >= kWaves
  const u32 tile = nw * QW * kWtInts, tiles = (u32)(((u64)count + tile - 1) / tile);
  const u32 grid = std::min<u32>(tiles, (u32)std::max(host::device_cus(), 1));
  WsHeader* h = reinterpret_cast<WsHeader*>(static_cast<char*>(ws) + ((tag2 >> 3) & 1u) * 8);
  const LbWords lb{reinterpret_cast<u64*>(static_cast<char*>(ws) + L.off_status), (u32)((L.off_lb_group - L.off_status) / 8), tag2};
  hipLaunchKernelGGL((k_feedback_encode<V, T, QW, NT>), dim3(grid), dim3((nw + 1) * 64), 0, st, static_cast<const u8*>(grad), count,
                     tiles, nw, d_out, fa, h, lb, d_written);
}
// The tile by size.  A large tile means few look-backs, a small one that a short stream reaches more of the device and
// that the last round of workgroups is fuller.  Measured with float32, 0124, us for QW x nw wave tiles a tile:
//     2^18 values: 1x4 6.3, 1x8 6.7, 1x15 7.9                2^20: 1x4 10.4, 1x8 8.6, 1x15 9.0, 2x15 12.7
//     3 * 2^20: 1x8 17.5, 1x15 13.4, 2x15 14.9               2^22: 1x15 17.4, 2x15 16.5
//     6 * 2^20: 1x15 23.6, 2x15 19.8                         2^24: 1x15 49.3, 2x11 48.0, 2x15 50.9
//     2^25: 1x15 86.7, 2x11 82.7, 2x15 83.9
// Non-temporal stores from 2^23 values up and loads from 2^24, where what a call touches no longer stays in the Infinity
// Cache (2^23: 30 us, with such stores 26, with the loads too 30; 2^26: 161, 156, 151).
template <int V, int T>
void launch_feedback(const void* grad, uint32_t count, uint8_t* d_out, const FeedArgs& fa, void* ws, unsigned tag2, uint64_t* d_written,
                     hipStream_t st) {
  const u32 m = count >> 19;  // in half millions
  if (m < 4) launch_feedback<V, T, 1, 0>(m < 1 ? 4 : 8, grad, count, d_out, fa, ws, tag2, d_written, st);
  else if (m < 7) launch_feedback<V, T, 1, 0>(15, grad, count, d_out, fa, ws, tag2, d_written, st);
  else if (m < 16) launch_feedback<V, T, 2, 0>(15, grad, count, d_out, fa, ws, tag2, d_written, st);
  else if (m < 32) launch_feedback<V, T, 1, kNtStores>(15, grad, count, d_out, fa, ws, tag2, d_written, st);
  else launch_feedback<V, T, 2, kNtLoads | kNtStores>(11, grad, count, d_out, fa, ws, tag2, d_written, st);
}

}  // namespace

extern "C" {

size_t svbgpu_grad_workspace_bytes(uint32_t ntensors) { return align256(8 * ((size_t)kGradChunks + ntensors)); }

int svbgpu_grad_norm(int norm, const svbgpu_tensor* tensors, uint32_t ntensors, float* d_norm, void* ws, size_t ws_bytes, void* stream) {
  u64 total;
  if (bad_norm(norm) || !d_norm || ((uintptr_t)d_norm & 3u)) return SVBGPU_EINVAL;
  const int rc = check_tensors(tensors, ntensors, &total);
  if (rc) return rc;
  if (!ws || ((uintptr_t)ws & 255u) || ws_bytes < svbgpu_grad_workspace_bytes(ntensors)) return SVBGPU_EWORKSPACE;
  if (!host::device_ok()) return SVBGPU_ENODEVICE;
  return norm_of(norm, tensors, ntensors, total, d_norm, ws, S(stream));
}

int svbgpu_grad_clip(int norm, const svbgpu_tensor* tensors, uint32_t ntensors, void* const* outs, double max_norm, int norm_given,
                     float* d_norm, void* ws, size_t ws_bytes, void* stream) {
  u64 total;
  if (bad_norm(norm) || !d_norm || ((uintptr_t)d_norm & 3u) || !(max_norm >= 0.0)) return SVBGPU_EINVAL;
  int rc = check_tensors(tensors, ntensors, &total);
  if (!rc) rc = check_written(tensors, ntensors, outs);
  if (rc) return rc;
  if (!norm_given && (!ws || ((uintptr_t)ws & 255u) || ws_bytes < svbgpu_grad_workspace_bytes(ntensors))) return SVBGPU_EWORKSPACE;
  if (!host::device_ok()) return SVBGPU_ENODEVICE;
  hipStream_t st = S(stream);
  if (!norm_given) {
    rc = norm_of(norm, tensors, ntensors, total, d_norm, ws, st);
    if (rc) return rc;
  }
  return for_launches<kMaxSpansOut>(tensors, ntensors, chunk_bytes_of(total),
                                    [&](const GradTable<kMaxSpansOut>& table, const uint32_t* of_span, u32 chunks, u32) {
    GradOuts<kMaxSpansOut> o;
    for (u32 i = 0; i < table.n; ++i) o.addr[i] = outs ? (u64)(uintptr_t)outs[of_span[i]] : 0;
    if (outs) hipLaunchKernelGGL(k_grad_scale<true>, dim3(chunks), dim3(kGradThreads), 0, st, table, o, d_norm, max_norm);
    else hipLaunchKernelGGL(k_grad_scale<false>, dim3(chunks), dim3(kGradThreads), 0, st, table, o, d_norm, max_norm);
    GRAD_HIP(hipGetLastError());
    return SVBGPU_OK;
  });
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
