// linear16.hip -- the 16-bit Linear (bf16 or fp16 operands, fp32 accumulation on the matrix cores) with bias, activation and residual
// in its epilogue, and its gradients:
//     z = x W^T + b,   y = act(z) + res,   dz = dy act'(z),   dx = dz W,   dW = dz^T x,   db = sum_rows dz
//
// One tile kernel serves x W^T and dz W (the weight transposed once per call, it is small), a second one dz^T x.
// 128 x 128 output tiles, 64 steps of the contraction per stage, two stages in LDS (64 KB: two workgroups share a CU and cover each
// other's barriers), four wavefronts of 64 x 64 on 32x32x16 products.  A tile's rows are 128 bytes of the operand; the 16-byte words of
// row r sit at word ^ ((r >> 1) & 7), so that the 16 lanes that read together hit 16 different bank groups.
// The products are formed as W x^T: a lane then holds four neighbouring output COLUMNS of a row.
// Operands whose rows are whole 16-byte words go to LDS directly (global_load_lds, no registers); any other pitch or width is loaded
// into registers (unaligned 16-byte loads, the last word of a row element by element) and written from there.
#include "elem.h"

using namespace shadow;

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
template <typename T> struct Frag;
template <> struct Frag<bf16_t> { typedef bf16_t v8 __attribute__((ext_vector_type(8))); typedef bf16_t v4 __attribute__((ext_vector_type(4))); };
template <> struct Frag<f16_t> { typedef f16_t v8 __attribute__((ext_vector_type(8))); typedef f16_t v4 __attribute__((ext_vector_type(4))); };

__device__ __forceinline__ f32x16 mma(Frag<bf16_t>::v8 a, Frag<bf16_t>::v8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(Frag<f16_t>::v8 a, Frag<f16_t>::v8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

constexpr int kActGelu = 5, kActSilu = 6, kActs = 7;

// Phi(z) and the density's exp(-z^2 / 2): erfc by Abramowitz & Stegun 7.1.26 (absolute error below 1.5e-7, a hundredth of a bf16 or
// fp16 step of the result), whose exponential is the density's
__device__ __forceinline__ void normal_cdf(float z, float &cdf, float &ex) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(fabsf(z), 0.3275911f * 0.70710678f, 1.f));
  ex = __builtin_amdgcn_exp2f(z * z * (-0.5f * 1.44269504f));
  const float q = 0.5f * ex * t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
  cdf = z > 0.f ? 1.f - q : q;
}
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f)); }
__device__ __forceinline__ float tanh16(float z) {            // exp2 form; near zero, where it cancels, two series terms
  const float s = z * (1.f - z * z * 0.33333333f);
  return fabsf(z) < 0.03f ? s : 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * 2.88539008f));
}

__device__ __forceinline__ float act16(int act, float z) {
  switch (act) {
    case 3: return tanh16(z);
    case kActGelu: { float c, e; normal_cdf(z, c, e); return z == -INFINITY ? 0.f : z * c; }
    case kActSilu: return z == -INFINITY ? 0.f : z * sigmoid(z);
    default: return act_fwd(act, z);
  }
}
__device__ __forceinline__ float slope16(int act, float z) {
  switch (act) {
    case 1: return z > 0.f ? 1.f : 0.f;
    case 2: return z > 0.f ? 1.f : __builtin_amdgcn_exp2f(z * 1.44269504f);
    case 3: { const float h = tanh16(z); return 1.f - h * h; }
    case 4: return z > 0.f ? 1.f : 0.2f;
    case kActGelu: { float c, e; normal_cdf(z, c, e); return fabsf(z) == INFINITY ? c : c + z * e * 0.39894228f; }
    case kActSilu: { const float s = sigmoid(z); return fabsf(z) == INFINITY ? s : s * (1.f + z * (1.f - s)); }
    default: return 1.f;
  }
}
// The pre-activation is kept for the backward pass in fp16 whatever the operands' type: eleven bits keep act'(z) well inside a bf16
// step, and where fp16's range ends every activation's slope has reached its limit.  A tiny positive z keeps its sign (relu's slope).
__device__ __forceinline__ f16_t keep_z(float z) {
  const f16_t h = (f16_t)z;
  return z > 0.f && h == (f16_t)0.f ? (f16_t)5.9604645e-8f : h;
}

constexpr int BM = 128, BN = 128, BK = 64, kThreads = 256;
constexpr int kTileBytes = 128 * BK * 2;                      // one operand's stage
constexpr int kStage = 2 * kTileBytes;

__device__ __attribute__((aligned(16))) const uint32_t g_zero16[4] = {0, 0, 0, 0};

__device__ __forceinline__ uint32_t swz(uint32_t row, uint32_t word) { return word ^ ((row >> 1) & 7); }

// 16 bytes at any alignment; elements at and past `left` read as zero
template <typename T>
__device__ __forceinline__ uint4 load_word(const T *p, int left) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (left >= 8) {
    __builtin_memcpy(&v, p, 16);
  } else if (left > 0) {
    uint16_t h[8];
#pragma unroll
    for (int j = 0; j < 8; j++) h[j] = 0;
#pragma unroll
    for (int j = 0; j < 7; j++)
      if (j < left) __builtin_memcpy(&h[j], p + j, 2);
    __builtin_memcpy(&v, h, 16);
  }
  return v;
}

// everything this wavefront has sent to LDS has arrived, and everybody's has
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
}
// LDS written by a wavefront is read back by other lanes of it (in order in hardware: only the compiler has to keep the order)
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ void lds_dma16(const void *src, void *dst) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src, (__attribute__((address_space(3))) void *)dst, 16, 0, 0);
}

struct GemmArgs {
  const void *A, *B;                        // [M, K], [N, K]
  int64_t lda, ldb;
  uint32_t M, N, K;
  const void *bias;
  int bias_f32;
  const void *res;
  int64_t ldr;
  void *C;
  int64_t ldc;
  f16_t *z;
  int64_t ldz;
  int act;
  uint32_t tiles_m, tiles_n;
};

// the workgroup's tile: consecutive workgroups go to the eight XCDs in turn, so XCD d takes the d-th eighth of the tiles, in groups of
// eight tile rows (the operand tiles that its workgroups share at one time then sit in its L2)
__device__ __forceinline__ void tile_of(uint32_t id, uint32_t tiles_m, uint32_t tiles_n, uint32_t &tm, uint32_t &tn) {
  const uint32_t total = tiles_m * tiles_n, q = total / 8, r = total % 8, d = id % 8, s = id / 8;
  const uint32_t t = d * q + min(d, r) + s;
  const uint32_t per = 8 * tiles_n, g = t / per, in = t % per, rows = min(8u, tiles_m - g * 8);
  tm = g * 8 + in % rows;
  tn = in / rows;
}

// four loads per thread and operand fill a stage; thread t of pass i covers LDS word i * 256 + t, i.e. row (i * 256 + t) / 8
template <typename T, bool DIRECT>
struct Loader {
  const T *base;                             // first row of the tile
  int64_t ld;
  uint32_t rows, K;                          // valid rows of the tile (>= 1), contraction length
  uint4 reg[4];

  __device__ __forceinline__ void start(uint32_t k0, char *lds) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t w = i * kThreads + threadIdx.x, r = w >> 3, k = k0 + swz(r, w & 7) * 8;
      const T *p = base + (int64_t)min(r, rows - 1) * ld + k;          // (rows past the end repeat the last: their products are not stored)
      if (DIRECT) {
        lds_dma16(k < K ? (const void *)p : (const void *)g_zero16, lds + (i * kThreads + (threadIdx.x & ~63u)) * 16);
      } else {
        reg[i] = load_word(p, (int)K - (int)k);
      }
    }
  }
  __device__ __forceinline__ void finish(char *lds) {
    if (!DIRECT) {
#pragma unroll
      for (int i = 0; i < 4; i++) *reinterpret_cast<uint4 *>(lds + (i * kThreads + threadIdx.x) * 16) = reg[i];
    }
  }
};

template <typename T, bool DIRECT>
__global__ void __launch_bounds__(kThreads, 2) nt_kernel(GemmArgs a) {
  typedef typename Frag<T>::v8 v8;
  __shared__ __attribute__((aligned(16))) char lds[2 * kStage];
  uint32_t tm, tn;
  tile_of(blockIdx.x, a.tiles_m, a.tiles_n, tm, tn);
  const uint32_t m0 = tm * BM, n0 = tn * BN, lane = lane_id(), wave = wave_id();
  const uint32_t wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
  Loader<T, DIRECT> la, lb;
  la.base = static_cast<const T *>(a.A) + (int64_t)m0 * a.lda; la.ld = a.lda; la.rows = min((uint32_t)BM, a.M - m0); la.K = a.K;
  lb.base = static_cast<const T *>(a.B) + (int64_t)n0 * a.ldb; lb.ld = a.ldb; lb.rows = min((uint32_t)BN, a.N - n0); lb.K = a.K;
  f32x16 acc[2][2];                          // [n half][m half]
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;
  const uint32_t steps = (a.K + BK - 1) / BK;
  la.start(0, lds); lb.start(0, lds + kTileBytes);
  la.finish(lds); lb.finish(lds + kTileBytes);
  for (uint32_t s = 0; s < steps; s++) {
    char *cur = lds + (s & 1) * kStage, *nxt = lds + ((s + 1) & 1) * kStage;
    stage_barrier();                         // (and everybody has read the other stage)
    v8 fa[2][4], fb[2][4];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const uint32_t rm = wm + h * 32 + (lane & 31), rn = wn + h * 32 + (lane & 31), w = q * 2 + (lane >> 5);
        fa[h][q] = *reinterpret_cast<const v8 *>(cur + rm * 128 + swz(rm, w) * 16);
        fb[h][q] = *reinterpret_cast<const v8 *>(cur + kTileBytes + rn * 128 + swz(rn, w) * 16);
      }
    if (s + 1 < steps) { la.start((s + 1) * BK, nxt); lb.start((s + 1) * BK, nxt + kTileBytes); }
#pragma unroll
    for (int q = 0; q < 4; q++)
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = mma(fb[i][q], fa[j][q], acc[i][j]);
    if (s + 1 < steps) { la.finish(nxt); lb.finish(nxt + kTileBytes); }
  }
  __syncthreads();
  // epilogue: 32 rows x 64 columns of the wavefront at a time through its own corner of LDS, so that a lane handles eight neighbouring
  // columns and eight lanes a 128-byte line of the output
  constexpr int kPitch = 68;                 // floats
  float *mine = reinterpret_cast<float *>(lds) + wave * 32 * kPitch;
#pragma unroll
  for (int j = 0; j < 2; j++) {
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float4 v = make_float4(acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]);
        *reinterpret_cast<float4 *>(mine + (lane & 31) * kPitch + i * 32 + e * 8 + (lane >> 5) * 4) = v;
      }
    wave_order();
#pragma unroll
    for (int p = 0; p < 4; p++) {
      const uint32_t r = p * 8 + (lane >> 3), c = (lane & 7) * 8, m = m0 + wm + j * 32 + r, n = n0 + wn + c;
      if (m < a.M && n < a.N) {
        float v[8];
        *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(mine + r * kPitch + c);
        *reinterpret_cast<float4 *>(v + 4) = *reinterpret_cast<const float4 *>(mine + r * kPitch + c + 4);
        const int left = min(8, (int)(a.N - n));
        if (a.bias) {
#pragma unroll
          for (int e = 0; e < 8; e++)
            if (e < left) v[e] += a.bias_f32 ? static_cast<const float *>(a.bias)[n + e] : (float)static_cast<const T *>(a.bias)[n + e];
        }
        if (a.z) {                           // (rows of z are padded to whole words)
          Vec<f16_t, 8> zz;
#pragma unroll
          for (int e = 0; e < 8; e++) zz.v[e] = keep_z(v[e]);
          *reinterpret_cast<Vec<f16_t, 8> *>(a.z + (int64_t)m * a.ldz + n) = zz;
        }
        if (a.act) {
#pragma unroll
          for (int e = 0; e < 8; e++) v[e] = act16(a.act, v[e]);
        }
        if (a.res) {
          const uint4 w = load_word(static_cast<const T *>(a.res) + (int64_t)m * a.ldr + n, left);
          T rr[8];
          __builtin_memcpy(rr, &w, 16);
#pragma unroll
          for (int e = 0; e < 8; e++) v[e] += (float)rr[e];
        }
        T out[8];
#pragma unroll
        for (int e = 0; e < 8; e++) out[e] = (T)v[e];
        T *dst = static_cast<T *>(a.C) + (int64_t)m * a.ldc + n;
        if (left == 8) __builtin_memcpy(dst, out, 16);
        else {
#pragma unroll
          for (int e = 0; e < 7; e++)
            if (e < left) dst[e] = out[e];
        }
      }
    }
    wave_order();
  }
}

// ------------------------------------------------------------------------------------------------ dz^T x
struct TnArgs {
  const void *A, *B;                        // dz [M, N], x [M, K]
  int64_t lda, ldb;
  uint32_t M, N, K;
  uint32_t tiles_n, tiles_k, slices, per;   // per: rows of a slice, a multiple of BK
  float *part;                              // [slices, N, K] (slices == 1: unused)
  float *part_b;                            // [slices, N]; null: no db
  void *C;
  int64_t ldc;
};

// the LDS image of a stage: 64 rows of the contraction x 128 columns (256 bytes); 16-byte word w of row r sits at w ^ (2 (r & 3) | 8 ((r >> 2) & 1))
__device__ __forceinline__ uint32_t swz_t(uint32_t row, uint32_t word) { return word ^ ((row & 3) * 2 + ((row >> 2) & 1) * 8); }

template <typename T, bool DIRECT>
struct RowLoader {
  const T *base;                             // column c0 of row 0
  int64_t ld;
  int cols;                                  // valid columns from c0 on (>= 1)
  uint4 reg[4];
  __device__ __forceinline__ void start(uint32_t r0, uint32_t r1, char *lds) {       // rows r0 .. r0 + 63, those at and past r1 read as zero
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t w = i * kThreads + threadIdx.x, r = w >> 4, c = swz_t(r, w & 15) * 8;
      const bool in = r0 + r < r1 && (int)c < cols;
      const T *p = base + (int64_t)(r0 + r) * ld + c;
      if (DIRECT) lds_dma16(in ? (const void *)p : (const void *)g_zero16, lds + (i * kThreads + (threadIdx.x & ~63u)) * 16);
      else reg[i] = in ? load_word(p, cols - (int)c) : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void finish(char *lds) {
    if (!DIRECT) {
#pragma unroll
      for (int i = 0; i < 4; i++) *reinterpret_cast<uint4 *>(lds + (i * kThreads + threadIdx.x) * 16) = reg[i];
    }
  }
};

// eight consecutive rows k .. k + 7 of column c0 + (lane & 15), as a product's operand: two transposing reads of four rows each (lane
// 4 q + p of a group of 16 points at 8-byte piece p of row q; it receives column (lane & 15) of the four rows)
template <typename T>
__device__ __forceinline__ typename Frag<T>::v8 read_cols(const char *img, uint32_t k, uint32_t c0) {
  const uint32_t l = lane_id() & 15, r = l >> 2, p = l & 3;
  typedef short s4 __attribute__((ext_vector_type(4)));
  union { s4 h[2]; typename Frag<T>::v8 v; } u;
#pragma unroll
  for (int t = 0; t < 2; t++) {
    const uint32_t row = k + 4 * t + r, word = (c0 >> 3) + (p >> 1);
    const char *at = img + row * 256 + swz_t(row, word) * 16 + (p & 1) * 8;
    u.h[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)at);
  }
  return u.v;
}

template <typename T, bool DA, bool DB>
__global__ void __launch_bounds__(kThreads, 2) tn_kernel(TnArgs a) {
  typedef typename Frag<T>::v8 v8;
  __shared__ __attribute__((aligned(16))) char lds[2 * kStage];
  // the tiles of a row slice are neighbours on one XCD: they read the same rows
  const uint32_t tiles = a.tiles_n * a.tiles_k, total = tiles * a.slices, q8 = total / 8, r8 = total % 8, d = blockIdx.x % 8, s8 = blockIdx.x / 8;
  const uint32_t id = d * q8 + min(d, r8) + s8, slice = id / tiles, tile = id % tiles, tn = tile / a.tiles_k, tk = tile % a.tiles_k;
  const uint32_t n0 = tn * BN, k0 = tk * BM, lane = lane_id(), wave = wave_id();
  const uint32_t wn = (wave >> 1) * 64, wk = (wave & 1) * 64;
  const uint32_t r0 = slice * a.per, r1 = min(a.M, r0 + a.per);
  RowLoader<T, DA> la;
  RowLoader<T, DB> lb;
  la.base = static_cast<const T *>(a.A) + n0; la.ld = a.lda; la.cols = (int)min((uint32_t)BN, a.N - n0);
  lb.base = static_cast<const T *>(a.B) + k0; lb.ld = a.ldb; lb.cols = (int)min((uint32_t)BM, a.K - k0);
  const bool with_b = a.part_b && tk == 0 && (wave & 1) == 0;           // (uniform over the wavefront)
  f32x16 acc[2][2], accb[2];                 // [n half][k half]
#pragma unroll
  for (int e = 0; e < 16; e++) {
    acc[0][0][e] = acc[0][1][e] = acc[1][0][e] = acc[1][1][e] = 0.f;
    accb[0][e] = accb[1][e] = 0.f;
  }
  v8 ones;
#pragma unroll
  for (int j = 0; j < 8; j++) ones[j] = (T)1.0f;
  const uint32_t steps = r1 > r0 ? (r1 - r0 + BK - 1) / BK : 0;
  if (steps) {
    la.start(r0, r1, lds); lb.start(r0, r1, lds + kTileBytes);
    la.finish(lds); lb.finish(lds + kTileBytes);
  }
  for (uint32_t s = 0; s < steps; s++) {
    char *cur = lds + (s & 1) * kStage, *nxt = lds + ((s + 1) & 1) * kStage;
    stage_barrier();
    v8 fa[2][4], fb[2][4];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const uint32_t kk = q * 16 + (lane >> 5) * 8, half = ((lane >> 4) & 1) * 16;
        fa[h][q] = read_cols<T>(cur, kk, wn + h * 32 + half);
        fb[h][q] = read_cols<T>(cur + kTileBytes, kk, wk + h * 32 + half);
      }
    if (s + 1 < steps) { la.start(r0 + (s + 1) * BK, r1, nxt); lb.start(r0 + (s + 1) * BK, r1, nxt + kTileBytes); }
#pragma unroll
    for (int q = 0; q < 4; q++) {
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = mma(fb[j][q], fa[i][q], acc[i][j]);       // rows: k, columns (lanes): n
      if (with_b) {
#pragma unroll
        for (int i = 0; i < 2; i++) accb[i] = mma(ones, fa[i][q], accb[i]);
      }
    }
    if (s + 1 < steps) { la.finish(nxt); lb.finish(nxt + kTileBytes); }
  }
  // a lane holds column n = lane & 31 and four neighbouring k at a time
  float *part = a.part ? a.part + (uint64_t)slice * a.N * a.K : nullptr;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const uint32_t n = n0 + wn + i * 32 + (lane & 31);
    if (n >= a.N) continue;
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const uint32_t k = k0 + wk + j * 32 + (e >> 2) * 8 + (lane >> 5) * 4 + (e & 3);
        if (k >= a.K) continue;
        if (part) part[(uint64_t)n * a.K + k] = acc[i][j][e];
        else static_cast<T *>(a.C)[(int64_t)n * a.ldc + k] = (T)acc[i][j][e];
      }
    if (with_b && lane < 32) a.part_b[(uint64_t)slice * a.N + n] = accb[i][0];
  }
}

// sums of the slices in slice order
template <typename T>
__global__ void __launch_bounds__(256) tn_join_kernel(const float *__restrict__ part, uint32_t slices, uint32_t N, uint32_t K, T *C, int64_t ldc) {
  const uint64_t e = (uint64_t)blockIdx.x * 256 + threadIdx.x, total = (uint64_t)N * K;
  if (e >= total) return;
  float t = 0.f;
#pragma unroll 8
  for (uint32_t s = 0; s < slices; s++) t += part[s * total + e];
  C[(int64_t)(e / K) * ldc + e % K] = (T)t;
}
template <typename T>
__global__ void __launch_bounds__(256) bias_join_kernel(const float *__restrict__ part, uint32_t slices, uint32_t N, void *db, int db_f32) {
  const uint32_t n = blockIdx.x * 256 + threadIdx.x;
  if (n >= N) return;
  float t = 0.f;
#pragma unroll 8
  for (uint32_t s = 0; s < slices; s++) t += part[(uint64_t)s * N + n];
  if (db_f32) static_cast<float *>(db)[n] = t;
  else static_cast<T *>(db)[n] = (T)t;
}

// ------------------------------------------------------------------------------------------------ elementwise pieces
// dz = dy act'(z), rounded to the operands' type (the products need 16-bit operands); pad columns are zero
template <typename T>
__global__ void __launch_bounds__(256) dz_kernel(const T *dy, int64_t lddy, const f16_t *z, T *dz, int64_t ld, uint32_t M, uint32_t N, int act) {
  const uint32_t words = (uint32_t)(ld / 8);
  const uint64_t total = (uint64_t)M * words;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
    const uint64_t m = i / words;
    const uint32_t n = (uint32_t)(i % words) * 8;
    const uint4 w = load_word(dy + (int64_t)m * lddy + n, (int)N - (int)n);
    T g[8];
    __builtin_memcpy(g, &w, 16);
    const Vec<f16_t, 8> zz = *reinterpret_cast<const Vec<f16_t, 8> *>(z + (int64_t)m * ld + n);
    Vec<T, 8> out;
#pragma unroll
    for (int e = 0; e < 8; e++) out.v[e] = n + e < N ? (T)((float)g[e] * slope16(act, (float)zz.v[e])) : (T)0.f;
    *reinterpret_cast<Vec<T, 8> *>(dz + (int64_t)m * ld + n) = out;
  }
}

// W [N, K] -> W^T [K, ld] (ld >= N, pad zero) in 32 x 32 tiles
template <typename T>
__global__ void __launch_bounds__(256) transpose_kernel(const T *W, int64_t ldw, uint32_t N, uint32_t K, T *out, int64_t ld) {
  __shared__ T tile[32][33];
  const uint32_t n0 = blockIdx.y * 32, k0 = blockIdx.x * 32, c = threadIdx.x & 31, r = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    tile[r + i][c] = n0 + r + i < N && k0 + c < K ? W[(int64_t)(n0 + r + i) * ldw + k0 + c] : (T)0.f;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    if (k0 + r + i < K && n0 + c < ld) out[(int64_t)(k0 + r + i) * ld + n0 + c] = tile[c][r + i];
}

inline uint64_t up(uint64_t v, uint64_t m) { return (v + m - 1) / m * m; }

struct BwdPlan {
  uint32_t slices, per;
  uint64_t dz, wt, part, part_b, total;      // byte offsets in the scratch
};

BwdPlan plan_bwd(int act, uint32_t M, uint32_t N, uint32_t K) {
  BwdPlan p;
  const uint32_t tiles = ((N + BN - 1) / BN) * ((K + BM - 1) / BM);
  // row slices of dz^T x: one workgroup per CU, at least four stages each
  uint32_t s = 256 / tiles;
  const uint32_t most = (M + 4 * BK - 1) / (4 * BK);
  s = s < 1 ? 1 : s;
  s = s > most ? most : s;
  s = s < 1 ? 1 : s;
  p.per = (uint32_t)up((M + s - 1) / s, BK);
  p.slices = M ? (M + p.per - 1) / p.per : 1;
  uint64_t at = 0;
  p.dz = at; at += act ? up((uint64_t)M * up(N, 8) * 2, 256) : 0;
  p.wt = at; at += up((uint64_t)K * up(N, 8) * 2, 256);
  p.part = at; at += p.slices > 1 ? up((uint64_t)p.slices * N * K * 4, 256) : 0;
  p.part_b = at; at += up((uint64_t)p.slices * N * 4, 256);
  p.total = at;
  return p;
}

bool dtype16(int d) { return d == SL_BF16 || d == SL_F16; }

template <typename T>
void nt_launch(GemmArgs a, hipStream_t st) {
  a.tiles_m = (a.M + BM - 1) / BM; a.tiles_n = (a.N + BN - 1) / BN;
  const dim3 g(a.tiles_m * a.tiles_n), b(kThreads);
  const bool direct = rows_of_words(a.A, a.lda, a.K, SL_BF16) && rows_of_words(a.B, a.ldb, a.K, SL_BF16);
  if (direct) hipLaunchKernelGGL((nt_kernel<T, true>), g, b, 0, st, a);
  else hipLaunchKernelGGL((nt_kernel<T, false>), g, b, 0, st, a);
}

template <typename T>
void tn_launch(const TnArgs &a, bool da, bool db, hipStream_t st) {
  const dim3 g(a.tiles_n * a.tiles_k * a.slices), b(kThreads);
  if (da && db) hipLaunchKernelGGL((tn_kernel<T, true, true>), g, b, 0, st, a);
  else if (da) hipLaunchKernelGGL((tn_kernel<T, true, false>), g, b, 0, st, a);
  else hipLaunchKernelGGL((tn_kernel<T, false, false>), g, b, 0, st, a);
}

#define SHD_DISPATCH_16(DTYPE, ...)                         \
  if ((DTYPE) == SL_BF16) { using T = bf16_t; __VA_ARGS__; }\
  else { using T = f16_t; __VA_ARGS__; }

constexpr uint64_t kMaxTiles = 0x7FFFFFFFull;

int check_sizes(const char *who, int dtype, int act, uint32_t M, uint32_t N, uint32_t K) {
  if (!dtype16(dtype)) return set_error(SG_ERR_INVALID, "%s: type %d (bf16 or fp16 operands)", who, dtype);
  if (act < 0 || act >= kActs) return set_error(SG_ERR_INVALID, "%s: activation %d", who, act);
  if (M > 0x7FFFFFFFu) return set_error(SG_ERR_INVALID, "%s: %u rows", who, M);
  if (N < 1 || K < 1 || N > (1u << 24) || K > (1u << 24)) return set_error(SG_ERR_INVALID, "%s: weight of %u x %u", who, N, K);
  if ((((uint64_t)M + BM - 1) / BM) * (((uint64_t)N + BN - 1) / BN) > kMaxTiles || (((uint64_t)M + BM - 1) / BM) * (((uint64_t)K + BN - 1) / BN) > kMaxTiles)
    return set_error(SG_ERR_INVALID, "%s: too many tiles", who);
  return SG_OK;
}

}  // namespace

extern "C" int sl_linear16_fwd(int dtype, const void *d_x, int64_t ldx, const void *d_w, int64_t ldw, const void *d_bias, int bias_f32,
                               const void *d_res, int64_t ldr, uint32_t M, uint32_t N, uint32_t K, int act, void *d_y, int64_t ldy,
                               void *d_z, int64_t ldz, void *stream) {
  if (const int rc = check_sizes("sl_linear16_fwd", dtype, act, M, N, K)) return rc;
  if (M == 0) return SG_OK;
  if (!d_x || !d_w || !d_y || ldx < (int64_t)K || ldw < (int64_t)K || ldy < (int64_t)N || (d_res && ldr < (int64_t)N) ||
      (d_z && (ldz < (int64_t)up(N, 8) || ldz % 8 || (reinterpret_cast<uintptr_t>(d_z) & 15))))
    return set_error(SG_ERR_INVALID, "sl_linear16_fwd: operands");
  hipStream_t st = (hipStream_t)stream;
  GemmArgs a = {};
  a.A = d_x; a.lda = ldx; a.B = d_w; a.ldb = ldw; a.M = M; a.N = N; a.K = K; a.bias = d_bias; a.bias_f32 = bias_f32; a.res = d_res; a.ldr = ldr;
  a.C = d_y; a.ldc = ldy; a.z = static_cast<f16_t *>(d_z); a.ldz = ldz; a.act = act;
  SHD_PROF_FMT(2.0 * ((double)M * K + (double)N * K + (double)M * N * (d_res ? 2 : 1)), 2.0 * M * N * K, st, "linear16_fwd_N%u_K%u", N, K);
  SHD_DISPATCH_16(dtype, nt_launch<T>(a, st));
  SHD_HIP(hipGetLastError());
  return SG_OK;
}

extern "C" size_t sl_linear16_bwd_scratch_bytes(int act, uint32_t M, uint32_t N, uint32_t K) { return plan_bwd(act, M, N, K).total; }

extern "C" int sl_linear16_bwd(int dtype, const void *d_x, int64_t ldx, const void *d_w, int64_t ldw, const void *d_dy, int64_t lddy,
                               const void *d_z, int64_t ldz, uint32_t M, uint32_t N, uint32_t K, int act, void *d_dx, int64_t lddx, void *d_dw,
                               int64_t lddw, void *d_db, int db_f32, void *d_scratch, void *stream) {
  if (const int rc = check_sizes("sl_linear16_bwd", dtype, act, M, N, K)) return rc;
  const bool want_w = d_dw || d_db;
  if (!d_scratch || (M && (!d_dy || lddy < (int64_t)N || (act && (!d_z || ldz != (int64_t)up(N, 8) || (reinterpret_cast<uintptr_t>(d_z) & 15))) || (d_dx && (!d_w || ldw < (int64_t)K || lddx < (int64_t)K)) ||
                           (want_w && (!d_x || ldx < (int64_t)K)))) ||
      (d_dw && lddw < (int64_t)K))
    return set_error(SG_ERR_INVALID, "sl_linear16_bwd: operands");
  if (d_db && !d_dw) return set_error(SG_ERR_INVALID, "sl_linear16_bwd: db comes with dW");
  hipStream_t st = (hipStream_t)stream;
  const BwdPlan p = plan_bwd(act, M, N, K);
  char *ws = static_cast<char *>(d_scratch);
  const void *dz = d_dy;
  int64_t lddz = lddy;
  if (act && M) {
    lddz = (int64_t)up(N, 8);
    dz = ws + p.dz;
    const uint64_t need = ((uint64_t)M * (lddz / 8) + 255) / 256;
    const dim3 g((uint32_t)(need < 8192 ? need : 8192)), b(256);
    SHD_PROF_FMT(6.0 * M * N, 0, st, "linear16_dz_N%u", N);
    SHD_DISPATCH_16(dtype, hipLaunchKernelGGL((dz_kernel<T>), g, b, 0, st, (const T *)d_dy, lddy, (const f16_t *)d_z, (T *)(ws + p.dz), lddz, M, N, act));
    SHD_HIP(hipGetLastError());
  }
  if (d_dx && M) {
    const int64_t ldt = (int64_t)up(N, 8);
    GemmArgs a = {};
    a.A = dz; a.lda = lddz; a.B = ws + p.wt; a.ldb = ldt; a.M = M; a.N = K; a.C = d_dx; a.ldc = lddx;
    a.K = act ? (uint32_t)ldt : N;           // (dz of an activation has zero pad columns, as W^T has: whole words)
    SHD_PROF_FMT(2.0 * ((double)M * K + (double)N * K + (double)M * N), 2.0 * M * N * K, st, "linear16_dx_N%u_K%u", N, K);
    SHD_DISPATCH_16(dtype, hipLaunchKernelGGL((transpose_kernel<T>), dim3((K + 31) / 32, (uint32_t)((ldt + 31) / 32)), dim3(256), 0, st, (const T *)d_w, ldw, N, K,
                                              (T *)(ws + p.wt), ldt);
                    nt_launch<T>(a, st));
    SHD_HIP(hipGetLastError());
  }
  if (want_w) {
    TnArgs a = {};
    a.A = dz; a.lda = lddz; a.B = d_x; a.ldb = ldx; a.M = M; a.N = N; a.K = K; a.tiles_n = (N + BN - 1) / BN; a.tiles_k = (K + BM - 1) / BM;
    a.slices = p.slices; a.per = p.per; a.part = p.slices > 1 ? reinterpret_cast<float *>(ws + p.part) : nullptr;
    a.part_b = d_db ? reinterpret_cast<float *>(ws + p.part_b) : nullptr; a.C = d_dw; a.ldc = lddw;
    const bool da = act || rows_of_words(dz, lddz, N, SL_BF16), db = rows_of_words(d_x, ldx, K, SL_BF16);
    SHD_PROF_FMT(2.0 * ((double)M * K + (double)N * K + (double)M * N), 2.0 * M * N * K, st, "linear16_dw_N%u_K%u", N, K);
    SHD_DISPATCH_16(dtype, tn_launch<T>(a, da, db, st);
                    if (p.slices > 1) hipLaunchKernelGGL((tn_join_kernel<T>), dim3((uint32_t)(((uint64_t)N * K + 255) / 256)), dim3(256), 0, st, a.part, p.slices, N, K, (T *)d_dw, lddw);
                    if (d_db) hipLaunchKernelGGL((bias_join_kernel<T>), dim3((N + 255) / 256), dim3(256), 0, st, a.part_b, p.slices, N, d_db, db_f32));
    SHD_HIP(hipGetLastError());
  }
  return SG_OK;
}
