// layer_norm.hip -- layer normalisation of rows in fp32 / bf16 / fp16, forward and backward.
//
//     d = x - mean(x),  r = (mean(d^2) + eps)^-1/2,  n = d r,  y = n s + o
//     g = dy s,  dx = r (g - mean(g) - n mean(g n)),  ds = sum_rows dy n,  do = sum_rows dy
//
// Bound by HBM: forward reads x and writes y, backward reads x and dy and writes dx.  A row stays in the registers of L lanes (16
// elements each), so the variance is the two-pass one (sum of squared differences from the mean) without a second read; the row sums
// run on the DPP network inside a wavefront, through LDS where a row takes a whole workgroup.  Statistics and sums are fp32.
// The weight gradient: every lane keeps its columns' running sums over the rows its workgroup walks (registers, no atomics), a
// workgroup leaves one row of partial sums, and a second kernel adds those in a fixed order -- the same bits every time.
// 289127 x 256 bf16: forward 61 us (4.8 TB/s), backward 87 us (5.1 TB/s) + 4.8 for the weight gradient, where a large copy runs at 5.2;
// 16385 x 800 fp16 12.5 and 18 + 4; 1024 x 256 fp32 forward 2.9; 289127 x 256 fp32 105 and 178 + 5.  Rows that are not whole 16-byte words
// go one element per load: 50021 x 602 fp32 48 and 71 + 5 (5.0 TB/s: a wavefront still reads whole lines), 20011 x 500 bf16 21 and 24 + 4
// (1.9 and 2.5 TB/s: half lines).
#include "elem.h"

using namespace shadow;

namespace {

constexpr int kElems = 16;                 // elements per lane

struct LnArgs {
  const void *x, *scale, *offset;
  void *y;
  int64_t ldx, ldy;
  float *stats;                            // [n, 2]: mean, r
  uint32_t n, F;
  float eps;
  int w_f32;
  // backward
  const void *dy;
  int64_t lddy;
  float *partial;                          // [gridDim.x, 2, F]; null with one workgroup, which writes dscale / doffset
  void *dscale, *doffset;
};

template <typename T, int V>
__device__ __forceinline__ void ld_weight(const void *w, int w_f32, uint32_t f, float (&out)[V]) {
  if (w_f32) {
#pragma unroll
    for (int j = 0; j < V; j++) out[j] = static_cast<const float *>(w)[f + j];
  } else {
#pragma unroll
    for (int j = 0; j < V; j++) out[j] = (float)static_cast<const T *>(w)[f + j];
  }
}

// sum over the L lanes of a row: DPP for L <= 64, LDS over the wavefronts of the workgroup above (the row is the workgroup's)
template <int L, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float *lds) {
  constexpr int kIn = L < 64 ? L : 64;
#pragma unroll
  for (int k = 0; k < K; k++) v[k] = group_sum<kIn>(v[k]);
  if (L > 64) {
    constexpr int W = L / 64;
    __syncthreads();                       // (the previous use of lds has been read)
    if (lane_id() == 0) {
#pragma unroll
      for (int k = 0; k < K; k++) lds[k * W + wave_id()] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; k++) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < W; w++) s += lds[k * W + w];
      v[k] = s;
    }
  }
}

template <typename T, int V, int L>
__global__ void __launch_bounds__(L < 256 ? 256 : L) ln_fwd_kernel(LnArgs a) {
  constexpr int NC = kElems / V, T_ = L < 256 ? 256 : L, G = T_ / L;
  __shared__ float lds[L > 64 ? L / 64 : 1];
  const uint32_t sub = threadIdx.x % L, nch = a.F / V;
  const float inv = 1.0f / (float)a.F;
  float s[NC][V], o[NC][V];
#pragma unroll
  for (int i = 0; i < NC; i++) {
    const uint32_t c = sub + i * L;
#pragma unroll
    for (int j = 0; j < V; j++) { s[i][j] = 1.f; o[i][j] = 0.f; }
    if (c < nch) {
      if (a.scale) ld_weight<T, V>(a.scale, a.w_f32, c * V, s[i]);
      if (a.offset) ld_weight<T, V>(a.offset, a.w_f32, c * V, o[i]);
    }
  }
  for (uint64_t row = (uint64_t)blockIdx.x * G + threadIdx.x / L; row < a.n; row += (uint64_t)gridDim.x * G) {
    const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.ldx;
    float v[NC][V], sum[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NC; i++) {
      const uint32_t c = sub + i * L;
#pragma unroll
      for (int j = 0; j < V; j++) v[i][j] = 0.f;
      if (c < nch) ldv<T, V>(x + c * V, v[i]);
#pragma unroll
      for (int j = 0; j < V; j++) sum[0] += v[i][j];
    }
    row_sum<L>(sum, lds);
    const float mean = sum[0] * inv;
    float sq[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NC; i++) {
      const bool in = sub + i * L < nch;
#pragma unroll
      for (int j = 0; j < V; j++) {
        v[i][j] -= mean;
        sq[0] += in ? v[i][j] * v[i][j] : 0.f;
      }
    }
    row_sum<L>(sq, lds);
    const float r = rsqrtf(sq[0] * inv + a.eps);
    if (a.stats && sub == 0) { a.stats[2 * row] = mean; a.stats[2 * row + 1] = r; }
    T *y = static_cast<T *>(a.y) + (int64_t)row * a.ldy;
#pragma unroll
    for (int i = 0; i < NC; i++) {
      const uint32_t c = sub + i * L;
#pragma unroll
      for (int j = 0; j < V; j++) v[i][j] = v[i][j] * r * s[i][j] + o[i][j];
      if (c < nch) stv<T, V>(y + c * V, v[i]);
    }
  }
}

template <typename T, int V, int L>
__global__ void __launch_bounds__(L < 256 ? 256 : L) ln_bwd_kernel(LnArgs a) {
  constexpr int NC = kElems / V, T_ = L < 256 ? 256 : L, G = T_ / L;
  constexpr int kRed = L > 64 ? 2 * L / 64 : (T_ / 64) * 2 * L * kElems;
  __shared__ float lds[kRed];
  const uint32_t sub = threadIdx.x % L, nch = a.F / V;
  const float inv = 1.0f / (float)a.F;
  float s[NC][V], ds[NC][V], dof[NC][V];
#pragma unroll
  for (int i = 0; i < NC; i++) {
    const uint32_t c = sub + i * L;
#pragma unroll
    for (int j = 0; j < V; j++) { s[i][j] = 1.f; ds[i][j] = 0.f; dof[i][j] = 0.f; }
    if (c < nch && a.scale) ld_weight<T, V>(a.scale, a.w_f32, c * V, s[i]);
  }
  for (uint64_t row = (uint64_t)blockIdx.x * G + threadIdx.x / L; row < a.n; row += (uint64_t)gridDim.x * G) {
    const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.ldx;
    const T *dy = static_cast<const T *>(a.dy) + (int64_t)row * a.lddy;
    float v[NC][V], d[NC][V], c12[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NC; i++) {
      const uint32_t c = sub + i * L;
#pragma unroll
      for (int j = 0; j < V; j++) { v[i][j] = 0.f; d[i][j] = 0.f; }
      if (c < nch) { ldv<T, V>(x + c * V, v[i]); ldv<T, V>(dy + c * V, d[i]); }
    }
    const float mean = a.stats[2 * row], r = a.stats[2 * row + 1];
#pragma unroll
    for (int i = 0; i < NC; i++) {
      const bool in = sub + i * L < nch;   // (columns past the row's end: n = 0, not -mean r)
#pragma unroll
      for (int j = 0; j < V; j++) {
        v[i][j] = in ? (v[i][j] - mean) * r : 0.f;
        dof[i][j] += d[i][j];
        ds[i][j] += d[i][j] * v[i][j];
        d[i][j] *= s[i][j];
        c12[0] += d[i][j];
        c12[1] += d[i][j] * v[i][j];
      }
    }
    row_sum<L>(c12, lds);
    const float c1 = c12[0] * inv, c2 = c12[1] * inv;
    if (a.y) {
      T *dx = static_cast<T *>(a.y) + (int64_t)row * a.ldy;
#pragma unroll
      for (int i = 0; i < NC; i++) {
        const uint32_t c = sub + i * L;
#pragma unroll
        for (int j = 0; j < V; j++) d[i][j] = r * (d[i][j] - c1 - v[i][j] * c2);
        if (c < nch) stv<T, V>(dx + c * V, d[i]);
      }
    }
  }
  if (!a.partial && !a.dscale && !a.doffset) return;
  // one row of partial sums per workgroup: over the row groups of a wavefront, then over its wavefronts, in a fixed order
  auto put = [&](int q, uint32_t f, float t) {
    if (a.partial) {
      a.partial[((uint64_t)blockIdx.x * 2 + q) * a.F + f] = t;
    } else if (void *w = q ? a.doffset : a.dscale) {
      if (a.w_f32) static_cast<float *>(w)[f] = t;
      else static_cast<T *>(w)[f] = (T)t;
    }
  };
  if (L > 64) {
#pragma unroll
    for (int i = 0; i < NC; i++) {
      const uint32_t c = sub + i * L;
      if (c < nch) {
#pragma unroll
        for (int j = 0; j < V; j++) { put(0, c * V + j, ds[i][j]); put(1, c * V + j, dof[i][j]); }
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < NC; i++) {
#pragma unroll
    for (int j = 0; j < V; j++) {
#pragma unroll
      for (int off = L; off < 64; off <<= 1) {
        ds[i][j] += __shfl_xor(ds[i][j], off, 64);
        dof[i][j] += __shfl_xor(dof[i][j], off, 64);
      }
      if (lane_id() < L) {
        const uint32_t f = (sub + i * L) * V + j;
        lds[(wave_id() * 2 + 0) * (L * kElems) + f] = ds[i][j];
        lds[(wave_id() * 2 + 1) * (L * kElems) + f] = dof[i][j];
      }
    }
  }
  __syncthreads();
  for (uint32_t f = threadIdx.x; f < a.F; f += T_) {
#pragma unroll
    for (int q = 0; q < 2; q++) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < T_ / 64; w++) t += lds[(w * 2 + q) * (L * kElems) + f];
      put(q, f, t);
    }
  }
}

// column sums of the partial rows: 32 columns x 32 row slices per workgroup, slices joined in a fixed order
template <typename W>
__global__ void __launch_bounds__(1024) ln_wgrad_kernel(const float *__restrict__ partial, uint32_t rows, uint32_t F, W *__restrict__ dscale,
                                                        W *__restrict__ doffset) {
  __shared__ float lds[32][33];
  const uint32_t c = threadIdx.x & 31, sl = threadIdx.x >> 5, col = blockIdx.x * 32 + c;
  float t = 0.f;
  if (col < 2 * F) {
#pragma unroll 8
    for (uint32_t r = sl; r < rows; r += 32) t += partial[(uint64_t)r * 2 * F + col];
  }
  lds[sl][c] = t;
  __syncthreads();
  if (sl == 0 && col < 2 * F) {
    t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; k++) t += lds[k][c];
    if (col < F) { if (dscale) dscale[col] = (W)t; }
    else if (doffset) doffset[col - F] = (W)t;
  }
}

constexpr uint32_t kMaxF = 1024 * kElems;

// lanes per row: the fewest that hold it at 16 elements each (more rows per wavefront, shorter reductions)
int lanes_of(uint32_t F) {
  for (int L : {8, 16, 32, 64, 256})
    if (F <= (uint32_t)L * kElems) return L;
  return 1024;
}

// up to this many trips one workgroup takes all rows and writes the weight gradient itself: a launch (some 4 us of the host's time)
// less than it costs.  On the GPU one workgroup and several with the second launch take 5.5 and 6.6 us for 32 rows of 256 bf16 (two
// trips), 7.1 and 6.7 for 64 (four), 10 and 6.7 for 128; 20 and 22 for 2 rows of 16384, 24 and 22 for 4.
constexpr uint32_t kAlone = 4;

uint32_t bwd_blocks(uint32_t n, uint32_t F) {
  const int L = lanes_of(F);
  const uint32_t G = L < 256 ? 256 / L : 1, need = (uint32_t)(((uint64_t)n + G - 1) / G);
  const uint32_t most = L == 1024 ? 256u : 1024u;
  return need <= kAlone ? 1u : need < most ? need : most;
}

template <typename T, int V>
int fwd_launch(const LnArgs &a, hipStream_t st) {
  const int L = lanes_of(a.F);
  const uint32_t G = L < 256 ? 256 / L : 1;
  const uint64_t need = ((uint64_t)a.n + G - 1) / G;
  const uint32_t grid = (uint32_t)(need < 2048 ? need : 2048);
#define SHD_LN_FWD(LL) hipLaunchKernelGGL((ln_fwd_kernel<T, V, LL>), dim3(grid), dim3(LL < 256 ? 256 : LL), 0, st, a)
  switch (L) {
    case 8: SHD_LN_FWD(8); break;
    case 16: SHD_LN_FWD(16); break;
    case 32: SHD_LN_FWD(32); break;
    case 64: SHD_LN_FWD(64); break;
    case 256: SHD_LN_FWD(256); break;
    default: SHD_LN_FWD(1024);
  }
#undef SHD_LN_FWD
  return SG_OK;
}

template <typename T, int V>
int bwd_launch(const LnArgs &a, hipStream_t st) {
  const uint32_t grid = bwd_blocks(a.n, a.F);
#define SHD_LN_BWD(LL) hipLaunchKernelGGL((ln_bwd_kernel<T, V, LL>), dim3(grid), dim3(LL < 256 ? 256 : LL), 0, st, a)
  switch (lanes_of(a.F)) {
    case 8: SHD_LN_BWD(8); break;
    case 16: SHD_LN_BWD(16); break;
    case 32: SHD_LN_BWD(32); break;
    case 64: SHD_LN_BWD(64); break;
    case 256: SHD_LN_BWD(256); break;
    default: SHD_LN_BWD(1024);
  }
#undef SHD_LN_BWD
  return SG_OK;
}

int check_shape(const char *who, int dtype, int w_dtype, uint32_t F) {
  if (!elem_dtype_ok(dtype) || !(w_dtype == SL_F32 || w_dtype == dtype))
    return set_error(SG_ERR_INVALID, "%s: types %d / %d", who, dtype, w_dtype);
  if (F < 1 || F > kMaxF) return set_error(SG_ERR_INVALID, "%s: rows of %u elements (1 to %u)", who, F, kMaxF);
  return SG_OK;
}

}  // namespace

extern "C" size_t sl_layer_norm_partial_floats(uint32_t n, uint32_t F) {
  if (F < 1 || F > kMaxF || n == 0) return 0;
  const uint32_t b = bwd_blocks(n, F);
  return b > 1 ? (size_t)b * 2 * F : 0;
}

extern "C" int sl_layer_norm_fwd(int dtype, int w_dtype, const void *d_x, int64_t ldx, const void *d_scale, const void *d_offset, uint32_t n,
                                 uint32_t F, float eps, void *d_y, int64_t ldy, float *d_stats, void *stream) {
  if (const int rc = check_shape("sl_layer_norm_fwd", dtype, w_dtype, F)) return rc;
  if (!(eps >= 0.f)) return set_error(SG_ERR_INVALID, "sl_layer_norm_fwd: eps");
  if (n == 0) return SG_OK;
  if (!d_x || !d_y || ldx < (int64_t)F || ldy < (int64_t)F) return set_error(SG_ERR_INVALID, "sl_layer_norm_fwd: operands");
  hipStream_t st = (hipStream_t)stream;
  LnArgs a = {};
  a.x = d_x; a.scale = d_scale; a.offset = d_offset; a.y = d_y; a.ldx = ldx; a.ldy = ldy; a.stats = d_stats; a.n = n; a.F = F; a.eps = eps;
  a.w_f32 = w_dtype == SL_F32;
  SHD_PROF_FMT((double)2 * n * F * elem_bytes(dtype), 0, st, "layer_norm_fwd_F%u", F);
  const bool words = rows_of_words(d_x, ldx, F, dtype) && rows_of_words(d_y, ldy, F, dtype);
  SHD_DISPATCH_ELEM(dtype, if (words) fwd_launch<T, kVec<T>>(a, st); else fwd_launch<T, 1>(a, st));
  SHD_HIP(hipGetLastError());
  return SG_OK;
}

extern "C" int sl_layer_norm_bwd(int dtype, int w_dtype, const void *d_x, int64_t ldx, const void *d_dy, int64_t lddy, const void *d_scale,
                                 const float *d_stats, uint32_t n, uint32_t F, void *d_dx, int64_t lddx, void *d_dscale, void *d_doffset,
                                 float *d_partial, void *stream) {
  if (const int rc = check_shape("sl_layer_norm_bwd", dtype, w_dtype, F)) return rc;
  const bool weights = d_dscale || d_doffset;
  if (n && (!d_x || !d_dy || !d_stats || ldx < (int64_t)F || lddy < (int64_t)F || (d_dx && lddx < (int64_t)F) || (weights && !d_partial && bwd_blocks(n, F) > 1)))
    return set_error(SG_ERR_INVALID, "sl_layer_norm_bwd: operands");
  hipStream_t st = (hipStream_t)stream;
  const uint32_t grid = n ? bwd_blocks(n, F) : 0;
  const bool alone = grid == 1;
  if (n && (d_dx || weights)) {
    LnArgs a = {};
    a.x = d_x; a.dy = d_dy; a.scale = d_scale; a.y = d_dx; a.ldx = ldx; a.lddy = lddy; a.ldy = lddx; a.stats = const_cast<float *>(d_stats);
    a.n = n; a.F = F; a.w_f32 = w_dtype == SL_F32; a.partial = weights && !alone ? d_partial : nullptr;
    if (alone) { a.dscale = d_dscale; a.doffset = d_doffset; }
    SHD_PROF_FMT((double)3 * n * F * elem_bytes(dtype), 0, st, "layer_norm_bwd_F%u", F);
    const bool words = rows_of_words(d_x, ldx, F, dtype) && rows_of_words(d_dy, lddy, F, dtype) && rows_of_words(d_dx, lddx, F, dtype);
    SHD_DISPATCH_ELEM(dtype, if (words) bwd_launch<T, kVec<T>>(a, st); else bwd_launch<T, 1>(a, st));
    SHD_HIP(hipGetLastError());
  }
  if (weights && !alone) {
    const dim3 g((2 * F + 31) / 32), b(1024);
    SHD_DISPATCH_ELEM(w_dtype, hipLaunchKernelGGL((ln_wgrad_kernel<T>), g, b, 0, st, d_partial, grid, F, (T *)d_dscale, (T *)d_doffset));
    SHD_HIP(hipGetLastError());
  }
  return SG_OK;
}
