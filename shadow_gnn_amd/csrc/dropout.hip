// dropout.hip -- dropout of rows in fp32 / bf16 / fp16 from the counter hash of the fused epilogues (actnorm_common.h), with the
// residual it is added to:
//     y[r, c] = res[r, c] + (keep(r, c; seed) ? x[r, c] / (1 - p) : 0)
// The mask is a function of (seed, r, c) and never in memory: the backward pass is the same call on dy without a residual.
// Bound by HBM (x and res read once, y written once); the hash -- one murmur finaliser per two columns, two quarter-rate multiplies
// each -- stays below that.
// One thread takes one 16-byte word per trip.  Rows that are whole words ("words") take the row hash once; contiguous rows of any other
// width are walked as one flat array of words, the row and column of a word's first element from one 64-bit division per workgroup and a
// 32-bit one per thread, and counted on from there; what is neither (a pitched view with odd rows) goes element by element.
// 289127 x 256 bf16: with residual 92 us (4.8 TB/s), backward 51 us (5.8 TB/s); 50021 x 602 fp32 (flat words) 40 us (6.0 TB/s).
#include "elem.h"

using namespace shadow;

namespace {

struct DropArgs {
  const void *x, *res;
  void *y;
  int64_t ldx, ldr, ldy;
  uint64_t n;
  uint32_t F;
  uint64_t seed;
  const int64_t *d_seed;
  uint32_t thr;                             // 0: keep everything
  float scale;
};

__device__ __forceinline__ uint64_t seed_of(const DropArgs &a) { return a.d_seed ? (uint64_t)*a.d_seed : a.seed; }

__device__ __forceinline__ bool keep1(uint32_t rowh, uint32_t thr, uint32_t c) {
  const uint32_t h = mix32(rowh + (c >> 1) * 0x9E3779B1u);
  return ((c & 1) ? h >> 16 : h & 0xFFFFu) >= thr;
}

// rows of whole words: L lanes (a power of two covering the words of a row, at most the workgroup) walk a row
template <typename T, bool RES>
__global__ void __launch_bounds__(256) drop_words_kernel(DropArgs a, uint32_t lanes) {
  constexpr int V = kVec<T>;
  const uint64_t seed = seed_of(a);
  const uint32_t lo = (uint32_t)seed, hi = (uint32_t)(seed >> 32), nch = a.F / V;
  const uint32_t sub = threadIdx.x & (lanes - 1), G = 256 / lanes;
  for (uint64_t row = (uint64_t)blockIdx.x * G + threadIdx.x / lanes; row < a.n; row += (uint64_t)gridDim.x * G) {
    const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.ldx;
    const T *rs = RES ? static_cast<const T *>(a.res) + (int64_t)row * a.ldr : nullptr;
    T *y = static_cast<T *>(a.y) + (int64_t)row * a.ldy;
    const uint32_t rowh = drop_row_hash(lo, hi, row);
    for (uint32_t c = sub; c < nch; c += lanes) {
      float v[V], q[V];
      ldv<T, V>(x + c * V, v);
      if (RES) ldv<T, V>(rs + c * V, q);
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        const uint32_t k = drop_keep4_h(rowh, a.thr, c * V + j);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          v[j + i] = (k >> i) & 1u ? v[j + i] * a.scale : 0.f;
          if (RES) v[j + i] += q[j + i];
        }
      }
      stv<T, V>(y + c * V, v);
    }
  }
}

// contiguous rows of any width: flat words.  PAIRS: F is even, so a pair of columns is
// a pair of neighbouring elements and one hash serves both.
template <typename T, bool RES, bool PAIRS>
__global__ void __launch_bounds__(256) drop_flat_kernel(DropArgs a, uint64_t total) {
  constexpr int V = kVec<T>;
  const uint64_t seed = seed_of(a);
  const uint32_t lo = (uint32_t)seed, hi = (uint32_t)(seed >> 32);
  const T *x = static_cast<const T *>(a.x), *rs = static_cast<const T *>(a.res);
  T *y = static_cast<T *>(a.y);
  const uint64_t words = total / V;
  // the row and column of the workgroup's first element by one 64-bit division per trip (uniform), the thread's by a 32-bit one
  for (uint64_t w0 = (uint64_t)blockIdx.x * 256; w0 < words; w0 += (uint64_t)gridDim.x * 256) {
    const uint64_t r0 = w0 * V / a.F;
    const uint32_t c0 = (uint32_t)(w0 * V - r0 * a.F);
    const uint64_t w = w0 + threadIdx.x;
    if (w >= words) break;
    const uint64_t off = (uint64_t)c0 + threadIdx.x * V;             // < F + 2048
    uint32_t dr, c;
    if (off >> 32) { dr = (uint32_t)(off / a.F); c = (uint32_t)(off % a.F); }
    else { dr = (uint32_t)off / a.F; c = (uint32_t)off - dr * a.F; }
    uint64_t r = r0 + dr;
    float v[V], q[V];
    ldv<T, V>(x + w * V, v);
    if (RES) ldv<T, V>(rs + w * V, q);
    uint32_t rowh = drop_row_hash(lo, hi, r);
#pragma unroll
    for (int j = 0; j < V; j += PAIRS ? 2 : 1) {
      if (PAIRS) {
        const uint32_t h = mix32(rowh + (c >> 1) * 0x9E3779B1u);
        v[j] = (h & 0xFFFFu) >= a.thr ? v[j] * a.scale : 0.f;
        v[j + 1] = (h >> 16) >= a.thr ? v[j + 1] * a.scale : 0.f;
        if (RES) { v[j] += q[j]; v[j + 1] += q[j + 1]; }
        c += 2;
      } else {
        v[j] = keep1(rowh, a.thr, c) ? v[j] * a.scale : 0.f;
        if (RES) v[j] += q[j];
        c++;
      }
      if (c >= a.F) { c = 0; r++; rowh = drop_row_hash(lo, hi, r); }
    }
    stv<T, V>(y + w * V, v);
  }
  if (blockIdx.x == 0 && threadIdx.x < total % V) {
    const uint64_t e = words * V + threadIdx.x, r = e / a.F;
    float t = keep1(drop_row_hash(lo, hi, r), a.thr, (uint32_t)(e - r * a.F)) ? (float)x[e] * a.scale : 0.f;
    if (RES) t += (float)rs[e];
    y[e] = (T)t;
  }
}

// any pitch, any alignment: one element per thread and trip
template <typename T, bool RES>
__global__ void __launch_bounds__(256) drop_elem_kernel(DropArgs a, uint32_t lanes) {
  const uint64_t seed = seed_of(a);
  const uint32_t lo = (uint32_t)seed, hi = (uint32_t)(seed >> 32);
  const uint32_t sub = threadIdx.x & (lanes - 1), G = 256 / lanes;
  for (uint64_t row = (uint64_t)blockIdx.x * G + threadIdx.x / lanes; row < a.n; row += (uint64_t)gridDim.x * G) {
    const uint32_t rowh = drop_row_hash(lo, hi, row);
    for (uint32_t c = sub; c < a.F; c += lanes) {
      float t = keep1(rowh, a.thr, c) ? (float)static_cast<const T *>(a.x)[(int64_t)row * a.ldx + c] * a.scale : 0.f;
      if (RES) t += (float)static_cast<const T *>(a.res)[(int64_t)row * a.ldr + c];
      static_cast<T *>(a.y)[(int64_t)row * a.ldy + c] = (T)t;
    }
  }
}

template <typename T>
void launch(const DropArgs &a, bool words, bool flat, hipStream_t st) {
  constexpr int V = kVec<T>;
  constexpr uint64_t kMost = 4096;          // workgroups: each walks several rows of a tall operand
  if (words || !flat) {
    const uint32_t units = words ? a.F / V : a.F;
    uint32_t lanes = 1;
    while (lanes < units && lanes < 256) lanes <<= 1;
    const uint64_t need = (a.n + 256 / lanes - 1) / (256 / lanes);
    const dim3 g((uint32_t)(need < kMost ? need : kMost)), b(256);
    if (words) {
      if (a.res) hipLaunchKernelGGL((drop_words_kernel<T, true>), g, b, 0, st, a, lanes);
      else hipLaunchKernelGGL((drop_words_kernel<T, false>), g, b, 0, st, a, lanes);
    } else {
      if (a.res) hipLaunchKernelGGL((drop_elem_kernel<T, true>), g, b, 0, st, a, lanes);
      else hipLaunchKernelGGL((drop_elem_kernel<T, false>), g, b, 0, st, a, lanes);
    }
    return;
  }
  const uint64_t total = a.n * a.F, need = (total / V + 255) / 256;
  const dim3 g((uint32_t)(need < 1 ? 1 : need < kMost ? need : kMost)), b(256);
  if (a.F % 2 == 0) {
    if (a.res) hipLaunchKernelGGL((drop_flat_kernel<T, true, true>), g, b, 0, st, a, total);
    else hipLaunchKernelGGL((drop_flat_kernel<T, false, true>), g, b, 0, st, a, total);
  } else {
    if (a.res) hipLaunchKernelGGL((drop_flat_kernel<T, true, false>), g, b, 0, st, a, total);
    else hipLaunchKernelGGL((drop_flat_kernel<T, false, false>), g, b, 0, st, a, total);
  }
}

}  // namespace

extern "C" int sl_dropout(int dtype, const void *d_x, int64_t ldx, const void *d_res, int64_t ldr, uint64_t n, uint32_t F, float p,
                          uint64_t seed, const int64_t *d_seed, void *d_y, int64_t ldy, void *stream) {
  if (!elem_dtype_ok(dtype)) return set_error(SG_ERR_INVALID, "sl_dropout: type %d", dtype);
  if (!(p >= 0.f && p < 1.f)) return set_error(SG_ERR_INVALID, "sl_dropout: probability %g (0 <= p < 1)", (double)p);
  if (F > 0x7FFFFFFFu) return set_error(SG_ERR_INVALID, "sl_dropout: rows of %u elements", F);
  if (n == 0 || F == 0) return SG_OK;
  if (!d_x || !d_y || ldx < (int64_t)F || ldy < (int64_t)F || (d_res && ldr < (int64_t)F)) return set_error(SG_ERR_INVALID, "sl_dropout: operands");
  hipStream_t st = (hipStream_t)stream;
  DropArgs a = {};
  a.x = d_x; a.res = d_res; a.y = d_y; a.ldx = ldx; a.ldr = ldr; a.ldy = ldy; a.n = n; a.F = F; a.seed = seed; a.d_seed = d_seed;
  a.thr = p > 0.f ? drop_threshold16(p) : 0u;
  a.scale = 1.0f / (1.0f - p);
  SHD_PROF_FMT((double)(d_res ? 3 : 2) * n * F * elem_bytes(dtype), 0, st, "dropout_F%u", F);
  const bool words = rows_of_words(d_x, ldx, F, dtype) && rows_of_words(d_y, ldy, F, dtype) && rows_of_words(d_res, ldr, F, dtype);
  const bool flat = ldx == (int64_t)F && ldy == (int64_t)F && (!d_res || ldr == (int64_t)F) &&
                    !((reinterpret_cast<uintptr_t>(d_x) | reinterpret_cast<uintptr_t>(d_y) | reinterpret_cast<uintptr_t>(d_res)) & 15);
  SHD_DISPATCH_ELEM(dtype, launch<T>(a, words, flat, st));
  SHD_HIP(hipGetLastError());
  return SG_OK;
}
