// linear16.hip -- the 16-bit Linear (bf16 or fp16 operands, fp32 accumulation on the matrix cores) with bias, activation and residual
// in its epilogue, and its gradients:
//     z = x W^T + b,   y = act(z) + res,   dz = dy act'(z),   dx = dz W,   dW = dz^T x,   db = sum_rows dz
//
// x W^T and dz W: 256 x 256 tiles for large products, 128 x 128 for the others, 32 x 32 with the contraction cut over wavefronts where
// there are few tiles (nt_launch has the rule), and for tall, narrow operands a kernel that keeps the weight in registers.  dz W reads
// the weight by columns in the last two, and transposed (once per call, it is small) in the others.  dz^T x: 128 x 128 tiles over row
// slices, all of dW at once for narrow operands, 32 x 32 tiles in one launch for few rows.
// Tiles are staged in LDS 64 steps of the contraction at a time -- 128 bytes of every row: with half lines (32 steps) every line
// crossed to the CU twice, 338 instead of 314 us at 32768 x 1024 x 4096 -- and multiplied on 32x32x16 products formed as W x^T: a lane then
// holds four neighbouring output COLUMNS of a row.
// 32768 x 1024 x 4096 fp16 gelu: 352 us, 215 to 226 of them the main loop (1.2 PFLOP/s; the products alone 166, and LDS is busy as long)
// and the rest an epilogue that does not overlap with it (two workgroups per CU of 128 x 256 tiles and half stages, whose would: 412) and
// the wait for its stores: they count in vmcnt, and the first stage after them waits for vmcnt(0).
// 289127 x 256 x 256 bf16 relu with residual: forward 105 us (bound by memory), dx 95 (59 by memory; see narrow_kernel), dW 83 + 12.
// 256 x 256 x 256: 4.8 us.  20011 x 1024 -> 1024 bf16 gelu: forward 80, dx 68 to 95, dz 26, dW 92 + 9 (products: 29 each).
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

// Phi(z) and the density's exp(-z^2 / 2): erfc by Abramowitz & Stegun 7.1.26, whose exponential is the density's.  Its error is an
// absolute one, below 1.5e-7.  Against the result that is next to nothing where |z Phi(z)| is of z's size, but the negative tail is small
// itself: gelu is off by a third of an fp16 step at z = -3.5, half of one at -4, and by 0.3, 0.7 and 1 bf16 step at -5, -6 and -7.
__device__ __forceinline__ void normal_cdf(float z, float &cdf, float &ex) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(fabsf(z), 0.3275911f * 0.70710678f, 1.f));
  ex = __builtin_amdgcn_exp2f(z * z * (-0.5f * 1.44269504f));
  const float q = 0.5f * ex * t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
  cdf = z > 0.f ? 1.f - q : q;
}
// z Phi(z) = max(z, 0) - |z| q, q the tail beyond |z|.  (|z| held below 64, where the tail has long been zero: no 0 * inf; a NaN comes
// through the maximum.)
__device__ __forceinline__ float gelu(float z) {
  const float az = fminf(fabsf(z), 64.f);
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(az, 0.3275911f * 0.70710678f, 1.f));
  const float w = az * 0.84932180f;          // (w^2 = z^2 / 2 log2 e)
  const float q = __builtin_amdgcn_exp2f(-w * w) * t * (0.127414796f + t * (-0.142248368f + t * (0.7107068705f + t * (-0.7265760135f + t * 0.5307027145f))));
  return __builtin_fmaf(-az, q, __builtin_elementwise_maximum(z, 0.f));
}
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f)); }
__device__ __forceinline__ float tanh16(float z) {            // exp2 form; near zero, where it cancels, two series terms
  const float s = z * (1.f - z * z * 0.33333333f);
  return fabsf(z) < 0.03f ? s : 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * 2.88539008f));
}

__device__ __forceinline__ float act16(int act, float z) {
  switch (act) {
    case 3: return tanh16(z);
    case kActGelu: return gelu(z);
    case kActSilu: return z == -INFINITY ? 0.f : z * sigmoid(z);
    default: return act_fwd(act, z);
  }
}
// act'(z) of the activations that keep z (relu and leakyrelu keep a bit of it)
__device__ __forceinline__ float slope16(int act, float z) {
  switch (act) {
    case 2: return z > 0.f ? 1.f : __builtin_amdgcn_exp2f(z * 1.44269504f);
    case 3: { const float h = tanh16(z); return 1.f - h * h; }
    case kActGelu: { float c, e; normal_cdf(z, c, e); return fabsf(z) == INFINITY ? c : c + z * e * 0.39894228f; }
    default: { const float s = sigmoid(z); return fabsf(z) == INFINITY ? s : s * (1.f + z * (1.f - s)); }      // silu
  }
}
// What the forward pass keeps of z for the backward pass.  relu and leakyrelu: one bit (z > 0), a byte per eight columns.  The others:
// z in fp16 whatever the operands' type (half the bytes of fp32; bf16 would keep three bits less).  Rounding z moves act'(z) by at most
// 0.3 x 2^-11 (gelu, silu), 0.36 (elu) or 0.63 (tanh): less than an fp16 step of a slope near 1.  Where the slope is small itself that
// is more of it: 0.4 to 0.8 % of tanh's beyond |z| = 4 (below 1.4e-3), 0.4 % of elu's below -8, 1.6 % and more of gelu's below -4.
// Where fp16's range ends every slope has reached its limit.
__host__ __device__ constexpr bool keeps_bits(int act) { return act == 1 || act == 4; }
__host__ __device__ constexpr uint64_t up(uint64_t v, uint64_t m) { return (v + m - 1) / m * m; }
// bytes of a kept row: whole 16-byte words
__host__ __device__ constexpr uint64_t kept_pitch(int act, uint32_t N) { return keeps_bits(act) ? up((N + 7) / 8, 16) : up(N, 8) * 2; }

// eight elements of dz = dy act'(z), rounded to the operands' type (the products need 16-bit operands; for relu nothing is lost).  db sums
// the same rounded dz on the same products: a sum of its own in fp32 would be another pass over dz.
// z: the word of kept values, or the byte of kept bits in z.x.  A dy of zero is a dz of zero.
template <typename T>
__device__ __forceinline__ uint4 dz_word(int act, const uint4 &dy, const uint4 &z) {
  uint4 out;
  if (act == 1) {
    const uint32_t in[4] = {dy.x, dy.y, dy.z, dy.w};
    uint32_t o[4];
#pragma unroll
    for (int q = 0; q < 4; q++) {            // bits 2 q and 2 q + 1 of the byte as masks of the two halves
      const uint32_t lo = (uint32_t)__builtin_amdgcn_sbfe((int)z.x, 2 * q, 1), hi = (uint32_t)__builtin_amdgcn_sbfe((int)z.x, 2 * q + 1, 1);
      o[q] = in[q] & ((lo & 0xFFFFu) | (hi & 0xFFFF0000u));
    }
    out = make_uint4(o[0], o[1], o[2], o[3]);
  } else {
    T g[8], r[8];
    f16_t zz[8];
    __builtin_memcpy(g, &dy, 16);
    __builtin_memcpy(zz, &z, 16);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float slope = act == 4 ? ((z.x >> e) & 1u ? 1.f : 0.2f) : slope16(act, (float)zz[e]);
      const float v = (float)g[e];
      r[e] = (T)(v == 0.f ? 0.f : v * slope);
    }
    __builtin_memcpy(&out, r, 16);
  }
  return out;
}

constexpr int BM = 128, BN = 128, BK = 64, kThreads = 256;    // tn_kernel's tile
constexpr int kTileBytes = 128 * BK * 2;                      // one operand's stage
constexpr int kStage = 2 * kTileBytes;

__device__ __attribute__((aligned(16))) const uint32_t g_zero16[4] = {0, 0, 0, 0};

// Eight elements from column c of a row of `width`, at any alignment; those past the row's end are zero.
// Rows of eight and more: fetched without a branch -- where the row ends inside the word, as the 16 bytes that end with it -- and shifted
// down when used, so that the loads of a stage are on their way together (behind a branch each, they waited for one another: 25 instead
// of 17 us at 20011 x 500 x 47).  Narrower rows: element by element.
template <typename T>
__device__ __forceinline__ uint4 fetch_word(const T *row, uint32_t c, uint32_t width) {
  uint4 v;
  __builtin_memcpy(&v, row + min(c, width - 8), 16);
  return v;
}
__device__ __forceinline__ uint4 settle_word(const uint4 &v, uint32_t c, uint32_t width) {
  const uint32_t back = c + 8 > width ? c + 8 - width : 0, sh = (back & 3) * 16;
  uint64_t lo = v.x | (uint64_t)v.y << 32, hi = v.z | (uint64_t)v.w << 32;
  lo = back & 4 ? hi : lo;
  hi = back & 4 ? 0 : hi;
  lo = lo >> sh | (hi << 1) << (63 - sh);
  hi >>= sh;
  const uint32_t keep = back >= 8 ? 0u : 0xFFFFFFFFu;
  return make_uint4((uint32_t)lo & keep, (uint32_t)(lo >> 32) & keep, (uint32_t)hi & keep, (uint32_t)(hi >> 32) & keep);
}
template <typename T>
__device__ __forceinline__ uint4 load_elems(const T *row, uint32_t c, uint32_t width) {
  uint4 v;
  uint16_t h[8];
#pragma unroll
  for (uint32_t j = 0; j < 8; j++) {
    h[j] = 0;
    if (c + j < width) __builtin_memcpy(&h[j], row + c + j, 2);
  }
  __builtin_memcpy(&v, h, 16);
  return v;
}
template <typename T>
__device__ __forceinline__ uint4 load_word(const T *row, uint32_t c, uint32_t width) {
  return width < 8 ? load_elems(row, c, width) : settle_word(fetch_word(row, c, width), c, width);
}
// how an operand's rows are read
enum Via { kWords, kRegs, kElems };          // whole 16-byte words; rows of eight elements and more; any rows

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

__device__ __forceinline__ uint32_t lds_addr(const void *p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)p; }

__device__ __forceinline__ void lds_dma16(const void *src, void *dst) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src, (__attribute__((address_space(3))) void *)dst, 16, 0, 0);
}

// The same transfer in inline assembly, for kernels that keep several stages in flight: the compiler would wait for all of them before
// every LDS read.  It has no result register; the kernel counts the transfers itself (wait_vm).  m0 (a register
// the compiler writes in front of each use of its own) needs one wait state before its use.
// First form: an address per lane; second: a uniform base and an offset per lane, nothing to compute from stage to stage.
__device__ __forceinline__ void lds_dma16_async(const void *src, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(__builtin_amdgcn_readfirstlane(dst)) : "memory");
}
__device__ __forceinline__ void lds_dma16_async(const void *base, uint32_t off, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(__builtin_amdgcn_readfirstlane(dst)) : "memory");
}
template <int N>
__device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

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
  char *kept;                                // kept_pitch(act, N) bytes a row; null: nothing is kept
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

// a stage of an operand: ROWS rows of 64 elements (128 bytes: whole lines of the operand, eight 16-byte words); word w of row r sits at
// w ^ ((r >> 1) & 7), so that the 16 lanes that read one word of 16 neighbouring rows hit all 64 banks
__device__ __forceinline__ uint32_t swz(uint32_t row, uint32_t word) { return word ^ ((row >> 1) & 7); }

template <typename T, int ROWS, int THREADS, bool DIRECT>
struct KLoader {
  static constexpr int P = ROWS * 8 / THREADS;
  const char *base;                          // the tile's first row (DIRECT: at the next stage's first column); uniform
  uint32_t off[P];                           // this thread's rows (DIRECT: words) from there, in bytes (the host keeps the pitch below 2^22 elements)
  uint32_t k;                                // the next stage's first column
  uint32_t K;
  uint4 reg[DIRECT ? 1 : P];

  static __device__ __forceinline__ uint32_t col(int i) { const uint32_t w = i * THREADS + threadIdx.x; return swz(w >> 3, w & 7) * 8; }
  __device__ __forceinline__ void init(const void *p, int64_t ld, uint32_t r0, uint32_t rows, uint32_t K_) {
    base = static_cast<const char *>(p) + (int64_t)r0 * ld * 2;
    k = 0; K = K_;
#pragma unroll
    for (int i = 0; i < P; i++) {            // (rows past the end repeat the last one: their products are not stored)
      const uint32_t r = (i * THREADS + threadIdx.x) >> 3;
      off[i] = (min(r0 + r, rows - 1) - r0) * (uint32_t)ld * 2 + (DIRECT ? col(i) * 2 : 0);
    }
  }
  // transfer i of the next stage
  __device__ __forceinline__ void send(int i, uint32_t lds) {
    if (k + 64 <= K) lds_dma16_async(base, off[i], lds + i * THREADS * 16);
    else lds_dma16_async(k + col(i) < K ? (const void *)(base + off[i]) : (const void *)g_zero16, lds + i * THREADS * 16);      // (K % 8 == 0)
  }
  __device__ __forceinline__ void next() {
    if (DIRECT) base += 128;
    k += 64;
  }
  // the next stage into registers (K >= 8), and from there to LDS
  __device__ __forceinline__ void fetch() {
    if constexpr (!DIRECT) {
#pragma unroll
      for (int i = 0; i < P; i++) reg[i] = fetch_word(reinterpret_cast<const T *>(base + off[i]), k + col(i), K);
      next();
    }
  }
  __device__ __forceinline__ void finish(char *lds) {
    if constexpr (!DIRECT) {
      if (k > K) {                           // (k is past the stage that was fetched: it is the last, and the rows end inside it)
#pragma unroll
        for (int i = 0; i < P; i++) reg[i] = settle_word(reg[i], k - 64 + col(i), K);
      }
#pragma unroll
      for (int i = 0; i < P; i++) *reinterpret_cast<uint4 *>(lds + (i * THREADS + threadIdx.x) * 16) = reg[i];
    }
  }
};

// the bias of eight neighbouring columns, `left` of which exist
template <typename T>
__device__ __forceinline__ void load_bias(const GemmArgs &a, uint32_t n, int left, float (&b)[8]) {
#pragma unroll
  for (int e = 0; e < 8; e++) b[e] = 0.f;
  if (!a.bias) return;
#pragma unroll
  for (int e = 0; e < 8; e++)
    if (e < left) b[e] = a.bias_f32 ? static_cast<const float *>(a.bias)[n + e] : (float)static_cast<const T *>(a.bias)[n + e];
}

template <int ACT>
__device__ __forceinline__ void act8(float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = act16(ACT, v[e]);
}

// Eight neighbouring columns of one row: bias, activation, residual, store.  `left` of them exist.  lds_bits: where kept bits are
// gathered instead of stored.
template <typename T>
__device__ __forceinline__ void finish8(const GemmArgs &a, uint32_t m, uint32_t n, int left, float (&v)[8], const float (&b)[8], const uint4 &resw,
                                        uint8_t *lds_bits = nullptr) {
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] += b[e];
  if (a.kept) {
    char *row = a.kept + (uint64_t)m * kept_pitch(a.act, a.N);
    if (keeps_bits(a.act)) {
      uint32_t bits = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) bits |= v[e] > 0.f ? 1u << e : 0u;
      if (left < 8) bits &= (1u << left) - 1u;
      if (lds_bits) *lds_bits = (uint8_t)bits;
      else row[n / 8] = (char)bits;
    } else {
      Vec<f16_t, 8> zz;
#pragma unroll
      for (int e = 0; e < 8; e++) zz.v[e] = (f16_t)v[e];
      *reinterpret_cast<Vec<f16_t, 8> *>(row + n * 2) = zz;
    }
  }
  switch (a.act) {                           // (uniform: one branch per word, not per element)
    case 1: act8<1>(v); break;
    case 2: act8<2>(v); break;
    case 3: act8<3>(v); break;
    case 4: act8<4>(v); break;
    case kActGelu: act8<kActGelu>(v); break;
    case kActSilu: act8<kActSilu>(v); break;
    default: break;
  }
  if (a.res) {
    T rr[8];
    __builtin_memcpy(rr, &resw, 16);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] += (float)rr[e];
  }
  T out[8];
#pragma unroll
  for (int e = 0; e < 8; e++) out[e] = (T)v[e];
  T *dst = static_cast<T *>(a.C) + (int64_t)m * a.ldc + n;
  if (left == 8) {
    __builtin_memcpy(dst, out, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 7; e++)
      if (e < left) dst[e] = out[e];
  }
}

// Workgroups stay and walk tiles (id, id + gridDim.x, ...): the first stages of the next tile are on their way while the epilogue of
// this one runs.
template <typename T, int BM_, int BN_, int WM, int WN, int ST, int OCC, bool DIRECT>
__global__ void __launch_bounds__(WM * WN * 64, OCC) nt_kernel(GemmArgs a) {
  typedef typename Frag<T>::v8 v8;
  constexpr int THREADS = WM * WN * 64, MI = BM_ / WM / 32, NI = BN_ / WN / 32;
  constexpr int kA = BM_ * 128, kBoth = (BM_ + BN_) * 128;    // bytes of a stage
  static_assert(BN_ / WN == 64 && NI == 2, "the epilogue's rows are 64 columns");
  constexpr int kEpi = 16 * 64 * 4;                           // bytes of a wavefront's epilogue corner: 16 rows
  __shared__ __attribute__((aligned(16))) char lds[ST * kBoth + WM * WN * kEpi];
  const uint32_t lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t wm = (wave % WM) * (BM_ / WM), wn = (wave / WM) * 64;
  const uint32_t tiles = a.tiles_m * a.tiles_n, steps = (a.K + 63) / 64;
  KLoader<T, BM_, THREADS, DIRECT> la;
  KLoader<T, BN_, THREADS, DIRECT> lb;
  constexpr int PER = decltype(la)::P + decltype(lb)::P;      // transfers per stage and thread
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(lds)) + wave * 1024;
  v8 fa[2][MI], fb[2][NI];                   // operands of two quarters of a stage
  const uint32_t ra = wm + (lane & 31), rb = wn + (lane & 31);
  auto read_quarter = [&](const char *cur, int q) {
#pragma unroll
    for (int h = 0; h < MI; h++) fa[q & 1][h] = *reinterpret_cast<const v8 *>(cur + (ra + h * 32) * 128 + swz(ra + h * 32, q * 2 + (lane >> 5)) * 16);
#pragma unroll
    for (int h = 0; h < NI; h++) fb[q & 1][h] = *reinterpret_cast<const v8 *>(cur + kA + (rb + h * 32) * 128 + swz(rb + h * 32, q * 2 + (lane >> 5)) * 16);
  };
  // what the loaders fetch next: stage `ls` of tile `lt`
  uint32_t lt = blockIdx.x, ls = 0;
  auto aim = [&]() {
    uint32_t tm, tn;
    tile_of(lt, a.tiles_m, a.tiles_n, tm, tn);
    la.init(a.A, a.lda, tm * BM_, a.M, a.K);
    lb.init(a.B, a.ldb, tn * BN_, a.N, a.K);
  };
  auto advance = [&]() {
    la.next(); lb.next();
    if (++ls == steps) {
      ls = 0; lt += gridDim.x;
      if (lt < tiles) aim();
    }
  };
  // A ring of ST stages in LDS.  A quarter's operands are read while the quarter before it is multiplied.  The one barrier of a stage
  // sits before its last quarter's products, when everybody has read that quarter: the stage's place is free again and the next stage
  // is whole (the younger ones may stay on their way); the transfers of the stage ST ahead go out between the products.
  uint32_t ahead = 0;                        // stages fetched and not yet finished with
  if (lt < tiles) aim();
  if constexpr (DIRECT) {
#pragma unroll
    for (int s = 0; s < ST; s++)
      if (lt < tiles) {
#pragma unroll
        for (int t = 0; t < decltype(la)::P; t++) la.send(t, lds0 + s * kBoth);
#pragma unroll
        for (int t = 0; t < decltype(lb)::P; t++) lb.send(t, lds0 + s * kBoth + kA);
        advance();
        ahead++;
      }
    if (ahead == ST) wait_vm<(ST - 1) * PER>();
    else wait_vm<0>();
    __syncthreads();
    read_quarter(lds, 0);
  }
  uint32_t at = 0;                           // the stage's place in the ring
  for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    uint32_t tm, tn;
    tile_of(tile, a.tiles_m, a.tiles_n, tm, tn);
    const uint32_t m0 = tm * BM_, n0 = tn * BN_;
    f32x16 acc[NI][MI];
#pragma unroll
    for (int i = 0; i < NI; i++)
#pragma unroll
      for (int j = 0; j < MI; j++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;
    if constexpr (!DIRECT) {
      la.init(a.A, a.lda, m0, a.M, a.K);
      lb.init(a.B, a.ldb, n0, a.N, a.K);
      la.fetch(); lb.fetch();
      __syncthreads();                       // (the tile before has been read)
      at = 0;
      la.finish(lds); lb.finish(lds + kA);
      if (steps > 1) { la.fetch(); lb.fetch(); }
      __syncthreads();
      read_quarter(lds, 0);
    }
    for (uint32_t s = 0; s < steps; s++) {
      const uint32_t nx = at + 1 == ST ? 0 : at + 1;
#pragma unroll
      for (int q = 0; q < 3; q++) {
        read_quarter(lds + at * kBoth, q + 1);
        if constexpr (!DIRECT) {
          if (q == 0 && s + 1 < steps) {     // (the next stage's place was last read before the previous barrier)
            la.finish(lds + nx * kBoth); lb.finish(lds + nx * kBoth + kA);
            if (s + 2 < steps) { la.fetch(); lb.fetch(); }
          }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NI; i++)
#pragma unroll
          for (int j = 0; j < MI; j++) acc[i][j] = mma(fb[q & 1][i], fa[q & 1][j], acc[i][j]);
      }
      bool send = false;
      if constexpr (DIRECT) {
        if (ahead > 1) {                     // another stage follows, of this tile or the next
          if (ahead == ST) wait_vm<(ST - 2) * PER>();
          else wait_vm<0>();
          __syncthreads();
          read_quarter(lds + nx * kBoth, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        send = lt < tiles;
      } else if (s + 1 < steps) {
        __syncthreads();
        read_quarter(lds + nx * kBoth, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
      const uint32_t to = lds0 + at * kBoth;
#pragma unroll
      for (int i = 0; i < NI; i++)
#pragma unroll
        for (int j = 0; j < MI; j++) {
          acc[i][j] = mma(fb[1][i], fa[1][j], acc[i][j]);
          if constexpr (DIRECT) {
            if (send) {
              const int x = i * MI + j;
#pragma unroll
              for (int t = x * PER / (NI * MI); t < (x + 1) * PER / (NI * MI); t++) {
                if (t < decltype(la)::P) la.send(t, to);
                else lb.send(t - decltype(la)::P, to + kA);
              }
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        }
      if constexpr (DIRECT) {
        if (send) advance();
        else ahead--;
      }
      at = nx;
    }
    // Epilogue: 16 rows of the wavefront's 64 columns at a time through its own corner of LDS (16-byte word w of row r at w ^ r), so
    // that a lane handles eight neighbouring columns and eight lanes a 128-byte line of the output.  The passes stay a loop: unrolled
    // over passes and activations the epilogue outgrows the instruction cache.
    float *mine = reinterpret_cast<float *>(lds + ST * kBoth) + wave * 16 * 64;
    const uint32_t er = lane >> 3, ec = lane & 7, n = n0 + wn + ec * 8;
    const int left = min(8, (int)a.N - (int)n);
    float b[8];
    load_bias<T>(a, n, left, b);
    uint32_t m = m0 + wm + er;               // this lane's next row
    const T *res = static_cast<const T *>(a.res) + (int64_t)m * a.ldr;
    const bool res_ahead = a.res && a.N >= 8;
    uint4 next = make_uint4(0, 0, 0, 0);
    if (res_ahead && m < a.M) next = fetch_word(res, n, a.N);
#pragma unroll
    for (int j = 0; j < MI; j++) {
#pragma unroll 1
      for (uint32_t half = 0; half < 2; half++) {
        if (((lane >> 4) & 1) == half) {
#pragma unroll
          for (int i = 0; i < NI; i++)
#pragma unroll
            for (int e = 0; e < 4; e++)
              *reinterpret_cast<float4 *>(mine + (lane & 15) * 64 + ((i * 8 + e * 2 + (lane >> 5)) ^ (lane & 15)) * 4) =
                  make_float4(acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]);
        }
        wave_order();
#pragma unroll 1
        for (uint32_t p = 0; p < 16; p += 8, m += 8) {
          const uint4 resw = next;
          const T *here = res;
          res += 8 * a.ldr;
          if (res_ahead && m + 8 < a.M) next = fetch_word(res, n, a.N);      // (a pass ahead; past the wavefront's last row it is not used)
          if (m < a.M && left > 0) {
            const uint32_t r = p + er;
            float v[8];
            *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(mine + r * 64 + ((ec * 2) ^ r) * 4);
            *reinterpret_cast<float4 *>(v + 4) = *reinterpret_cast<const float4 *>(mine + r * 64 + ((ec * 2 + 1) ^ r) * 4);
            finish8<T>(a, m, n, left, v, b, !a.res ? resw : res_ahead ? settle_word(resw, n, a.N) : load_elems(here, n, a.N));
          }
        }
        wave_order();
      }
    }
  }
}

// Few output tiles: 32 x 32 tiles, the contraction cut over the workgroup's eight wavefronts (step 16 w, 16 (w + 8), ...), their
// products joined in LDS in wavefront order.  Operands go from memory to the product's registers: every word is used once.
// COLS (dx = dz W): B is given as [K, N]; A is dy and its words become dz = dy act'(z) on the way (kept_act 0: as they are).
struct FewArgs {
  GemmArgs g;
  const char *kept;
  int kept_act;
};
template <typename T, Via VIA, bool COLS>
__global__ void __launch_bounds__(512) nt_few_kernel(FewArgs f) {
  const GemmArgs &a = f.g;
  typedef typename Frag<T>::v8 v8;
  constexpr int kPitch = 36;
  __shared__ __attribute__((aligned(16))) float part[8][32 * kPitch];
  const uint32_t tm = blockIdx.x % a.tiles_m, tn = blockIdx.x / a.tiles_m, m0 = tm * 32, n0 = tn * 32;
  const uint32_t lane = lane_id(), wave = wave_id(), r = lane & 31;
  const uint32_t row_a = min(m0 + r, a.M - 1), row_b = min(n0 + r, a.N - 1);
  const T *pa = static_cast<const T *>(a.A) + (int64_t)row_a * a.lda;
  const T *pb = static_cast<const T *>(a.B) + (COLS ? (int64_t)row_b : (int64_t)row_b * a.ldb);
  const char *pk = f.kept + (uint64_t)row_a * kept_pitch(f.kept_act, a.K);
  f32x16 acc;
#pragma unroll
  for (int e = 0; e < 16; e++) acc[e] = 0.f;
  constexpr int U = 4;                       // steps whose loads are in flight together
  for (uint32_t k0 = wave * 16; k0 < a.K; k0 += 8 * 16 * U) {
    uint4 wa[U], wb[U], wz[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint32_t k = k0 + u * 128 + (lane >> 5) * 8;
      if (VIA == kWords) wa[u] = k < a.K ? *reinterpret_cast<const uint4 *>(pa + k) : make_uint4(0, 0, 0, 0);
      else if (VIA == kRegs) wa[u] = fetch_word(pa, k, a.K);
      else wa[u] = load_elems(pa, k, a.K);
      if (COLS) {
        T e[8];
#pragma unroll
        for (int j = 0; j < 8; j++) e[j] = pb[(int64_t)min(k + j, a.K - 1) * a.ldb];
        __builtin_memcpy(&wb[u], e, 16);
        wz[u] = make_uint4(0, 0, 0, 0);
        if (f.kept_act && k < a.K) {
          if (keeps_bits(f.kept_act)) wz[u].x = (uint8_t)pk[k / 8];
          else wz[u] = *reinterpret_cast<const uint4 *>(pk + k * 2);
        }
      } else if (VIA == kWords) {
        wb[u] = k < a.K ? *reinterpret_cast<const uint4 *>(pb + k) : make_uint4(0, 0, 0, 0);
      } else if (VIA == kRegs) {
        wb[u] = fetch_word(pb, k, a.K);
      } else {
        wb[u] = load_elems(pb, k, a.K);
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint32_t k = k0 + u * 128 + (lane >> 5) * 8;
      v8 fa, fb;
      if (VIA == kRegs) {
        wa[u] = settle_word(wa[u], k, a.K);
        if (!COLS) wb[u] = settle_word(wb[u], k, a.K);
      }
      if (COLS) {
        if (f.kept_act) wa[u] = dz_word<T>(f.kept_act, wa[u], wz[u]);
        T e[8];
        __builtin_memcpy(e, &wb[u], 16);
#pragma unroll
        for (int j = 0; j < 8; j++) e[j] = k + j < a.K ? e[j] : (T)0.f;
        __builtin_memcpy(&wb[u], e, 16);
      }
      __builtin_memcpy(&fa, &wa[u], 16);
      __builtin_memcpy(&fb, &wb[u], 16);
      acc = mma(fb, fa, acc);
    }
  }
#pragma unroll
  for (int e = 0; e < 4; e++)
    *reinterpret_cast<float4 *>(&part[wave][r * kPitch + e * 8 + (lane >> 5) * 4]) = make_float4(acc[4 * e], acc[4 * e + 1], acc[4 * e + 2], acc[4 * e + 3]);
  __syncthreads();
  if (threadIdx.x >= 128) return;            // 32 rows x four words
  const uint32_t er = threadIdx.x >> 2, ec = (threadIdx.x & 3) * 8, m = m0 + er, n = n0 + ec;
  if (m >= a.M || n >= a.N) return;
  const int left = min(8, (int)a.N - (int)n);
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = 0.f;
#pragma unroll
  for (int w = 0; w < 8; w++)
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] += part[w][er * kPitch + ec + e];
  uint4 resw = make_uint4(0, 0, 0, 0);
  if (a.res) resw = load_word(static_cast<const T *>(a.res) + (int64_t)m * a.ldr, n, a.N);
  float b[8];
  load_bias<T>(a, n, left, b);
  finish8<T>(a, m, n, left, v, b, resw);
}

// dx = dz W of few outputs (N <= 64: a classifier's classes): B is W as it is, [K, N] here.  A wavefront keeps 64 columns of W in
// registers and walks `per` tiles of 32 rows, a tile ahead of its loads; no barriers, no tile of A in LDS (it would be read once), no
// transposed weight.  Wavefronts of one workgroup share rows.  Bound by the loads' latency at a few wavefronts per SIMD: dx of
// 20011 x 64 -> 512 takes 12 us (4 of them the store) and 18 in transposed 128 x 128 tiles, 8192 x 40 -> 1024 10 and 14.
template <typename T>
__global__ void __launch_bounds__(256, 4) nt_short_kernel(GemmArgs a, uint32_t groups, uint32_t per) {
  typedef typename Frag<T>::v8 v8;
  constexpr int Q = 4;
  __shared__ __attribute__((aligned(16))) float corners[4][16 * 64];
  const uint32_t lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), item = blockIdx.x * 4 + wave, n0 = item % groups * 64;
  const uint32_t tile0 = item / groups * per, tiles = (a.M + 31) / 32;
  if (tile0 >= tiles) return;                // (whole wavefronts; no barrier follows)
  const uint32_t tile1 = min(tiles, tile0 + per), kl = (lane >> 5) * 8;
  uint4 wa[Q];
  auto fetch = [&](uint32_t tile) {
    const T *pa = static_cast<const T *>(a.A) + (int64_t)min(tile * 32 + (lane & 31), a.M - 1) * a.lda;
#pragma unroll
    for (int q = 0; q < Q; q++) {
      const uint32_t k = q * 16 + kl;
      wa[q] = *reinterpret_cast<const uint4 *>(pa + (k < a.K ? k : 0));
    }
  };
  v8 fb[2][Q];
#pragma unroll
  for (int h = 0; h < 2; h++) {              // (32-bit offsets: the host keeps the pitch below 2^22 elements)
    const uint32_t col = min(n0 + h * 32 + (lane & 31), a.N - 1);
#pragma unroll
    for (int q = 0; q < Q; q++) {
      T e[8];
#pragma unroll
      for (int j = 0; j < 8; j++)
        e[j] = *reinterpret_cast<const T *>(static_cast<const char *>(a.B) + (min(q * 16 + kl + j, a.K - 1) * (uint32_t)a.ldb + col) * 2);
      __builtin_memcpy(&fb[h][q], e, 16);
    }
  }
  fetch(tile0);
#pragma unroll
  for (int h = 0; h < 2; h++)
#pragma unroll
    for (int q = 0; q < Q; q++)
#pragma unroll
      for (int j = 0; j < 8; j++) fb[h][q][j] = q * 16 + kl + j < a.K ? fb[h][q][j] : (T)0.f;
  float *mine = corners[wave];
  const uint32_t er = lane >> 3, ec = lane & 7, n = n0 + ec * 8;
  const int left = min(8, (int)a.N - (int)n);
  uint32_t m = tile0 * 32 + er;              // this lane's next row
  T *dst = static_cast<T *>(a.C) + (int64_t)m * a.ldc + n;
  const int64_t step = 8 * a.ldc;
  for (uint32_t tile = tile0; tile < tile1; tile++) {
    v8 fa[Q];
#pragma unroll
    for (int q = 0; q < Q; q++) {
      const uint32_t k = q * 16 + kl;
      const uint4 w = k < a.K ? wa[q] : make_uint4(0, 0, 0, 0);
      __builtin_memcpy(&fa[q], &w, 16);
    }
    if (tile + 1 < tile1) fetch(tile + 1);
    f32x16 acc[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
#pragma unroll
      for (int e = 0; e < 16; e++) acc[h][e] = 0.f;
#pragma unroll
      for (int q = 0; q < Q; q++) acc[h] = mma(fb[h][q], fa[q], acc[h]);
    }
#pragma unroll
    for (uint32_t half = 0; half < 2; half++) {               // 16 rows at a time through this wavefront's corner (word w of row r at w ^ r)
      if (((lane >> 4) & 1) == half) {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int e = 0; e < 4; e++)
            *reinterpret_cast<float4 *>(mine + (lane & 15) * 64 + ((h * 8 + e * 2 + (lane >> 5)) ^ (lane & 15)) * 4) =
                make_float4(acc[h][4 * e], acc[h][4 * e + 1], acc[h][4 * e + 2], acc[h][4 * e + 3]);
      }
      wave_order();
#pragma unroll
      for (uint32_t t = 0; t < 16; t += 8, m += 8, dst += step) {
        const uint32_t r = t + er;
        if (m < a.M && left > 0) {
          T out[8];
          float v[8];
          *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(mine + r * 64 + ((ec * 2) ^ r) * 4);
          *reinterpret_cast<float4 *>(v + 4) = *reinterpret_cast<const float4 *>(mine + r * 64 + ((ec * 2 + 1) ^ r) * 4);
#pragma unroll
          for (int e = 0; e < 8; e++) out[e] = (T)v[e];
          if (left == 8) {
            __builtin_memcpy(dst, out, 16);
          } else {
#pragma unroll
            for (int e = 0; e < 7; e++)
              if (e < left) dst[e] = out[e];
          }
        }
      }
      wave_order();
    }
  }
}

// ------------------------------------------------------------------------------------------------ tall, narrow products
// N <= 256 and K <= 256 (the hidden widths of the graph models) over many rows are bound by memory: x, res and y cross it once.  The
// weight stays in the registers of NWC wavefronts (32 output columns each) for the whole launch; four more wavefronts do nothing but
// send 32-row tiles of A, and of what else the rows need (SIDE), to a ring of RS places in LDS.  Transfers are counted together with a
// wavefront's own loads and stores and in order: apart from each other, the senders keep RS - 1 tiles on their way and the multiplying
// wavefronts never wait for their stores (with the residual loaded by them the forward pass took 140, dx 150 us at 289127 x 256 x 256).
// One barrier per tile: the tile is whole, and the one before it has been read.
// SIDE 2 and 3 await a tile one turn earlier, so that it can become dz; there RS - 2 tiles are under way at a wait, which counts as the
// ring's end: everything sent has to arrive, and one tile is on its way beside the products.  dx of 289127 x 256 x 256 takes 95 us of a
// relu or leakyrelu so (59 by memory) and 300 to 370 of gelu, silu, elu and tanh, whose form in addition spills (176 bytes a lane): dz written
// by dz_kernel first and dx through SIDE 0 would take 170 to 177 there, 25 instead of 38 us at 20011 x 256 x 256, 78 instead of 142 at
// 289127 x 128 x 128, with the same bits.
//   SIDE 1: the residual's rows.
//   SIDE 2, 3 (dx = dz W; A is dy): kept fp16 values / kept bits.  The tile becomes dz = dy act'(z) in place, each wavefront a share
//   of it, while the tile before it is multiplied, and is stored for dz^T x if asked for.
// Bits kept by the forward pass are gathered in LDS and leave a tile later as whole words (as bytes they cost 25 us of 140).
struct NarrowArgs {
  GemmArgs g;
  uint32_t b_rows;                           // not 0: B is given as [b_rows, N] (pitch ldb); K may end inside a word of zeros past it
  const char *kept;                          // SIDE 2, 3: kept values of g.K columns
  int kept_act;
  void *dz;                                  // SIDE 2, 3: null, or where dz goes, pitch lddz
  int64_t lddz;
};

template <int W>                             // W 16-byte words per row
__device__ __forceinline__ uint32_t swz_row(uint32_t row, uint32_t word) { return W >= 16 ? word ^ (row & 15) : word ^ ((row >> 1) & 7); }

template <typename T, int NWC, int KS, int RS, int SIDE>
__global__ void __launch_bounds__((NWC + 4) * 64, 3) narrow_kernel(NarrowArgs n) {
  typedef typename Frag<T>::v8 v8;
  constexpr int R = 32, W = KS * 2, WS = SIDE == 1 ? NWC * 4 : SIDE == 2 ? W : 0;      // rows of a tile, words of its rows and of the side's
  constexpr int kA = R * W * 16, kSide = SIDE == 3 ? R * 32 : R * WS * 16, kPlace = kA + kSide;
  constexpr int PA = R * W / 256, PS = SIDE == 3 ? 1 : R * WS / 256, PER = PA + PS;    // transfers per tile and lane
  __shared__ __attribute__((aligned(16))) char lds[RS * kPlace + NWC * 2048 + (SIDE < 2 ? 2 * R * 32 : 0)];
  const GemmArgs &a = n.g;
  const uint32_t lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t tiles = (a.M + R - 1) / R;
  const bool bits_out = SIDE < 2 && a.kept && keeps_bits(a.act);
  if (wave >= NWC) {                         // ---- the sending wavefronts
    const uint32_t me = wave - NWC, lds0 = __builtin_amdgcn_readfirstlane(lds_addr(lds));
    const uint32_t kw = (uint32_t)(kept_pitch(1, a.K) / 16);           // SIDE 3: words of a row of bits (1 or 2)
    auto send = [&](uint32_t tile, uint32_t slot) {
      const uint32_t place = lds0 + slot * kPlace + me * 1024;
#pragma unroll
      for (int i = 0; i < PA; i++) {
        const uint32_t w = (i * 4 + me) * 64 + lane, r = w / W, k = swz_row<W>(r, w % W) * 8, row = min(tile * R + r, a.M - 1);
        const T *p = static_cast<const T *>(a.A) + (int64_t)row * a.lda + k;
        lds_dma16_async(k < a.K ? (const void *)p : (const void *)g_zero16, place + i * 4096);
      }
      if constexpr (SIDE == 1 || SIDE == 2) {
        const char *base = SIDE == 1 ? static_cast<const char *>(a.res) : n.kept;
        const int64_t pitch = SIDE == 1 ? a.ldr * 2 : (int64_t)kept_pitch(5, a.K);
        const uint32_t width = SIDE == 1 ? a.N : a.K;
#pragma unroll
        for (int i = 0; i < PS; i++) {
          const uint32_t w = (i * 4 + me) * 64 + lane, r = w / WS, k = swz_row<WS>(r, w % WS) * 8, row = min(tile * R + r, a.M - 1);
          lds_dma16_async(k < width ? (const void *)(base + row * pitch + k * 2) : (const void *)g_zero16, place + kA + i * 4096);
        }
      }
      if constexpr (SIDE == 3) {
        if (lane < 16) {                     // (64 words, 16 of each sender)
          const uint32_t w = me * 16 + lane, row = min(tile * R + w / kw, a.M - 1);
          lds_dma16_async(w < R * kw ? (const void *)(n.kept + (uint64_t)row * kw * 16 + (w % kw) * 16) : (const void *)g_zero16, lds0 + slot * kPlace + kA + me * 256);
        }
      }
    };
    uint32_t next = blockIdx.x, slot = 0;    // the tile and place sent next
    for (int s = 0; s < RS - 1; s++)
      if (next < tiles) { send(next, slot); next += gridDim.x; slot++; }
    uint32_t left = slot;                    // tiles sent and not yet awaited
    auto await = [&]() {                     // the oldest tile sent is whole
      if (left == RS - 1) wait_vm<(RS - 2) * PER>();
      else wait_vm<0>();
      left--;
    };
    if (SIDE >= 2) { await(); __syncthreads(); }
    for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
      if (SIDE < 2 || tile + gridDim.x < tiles) await();
      __syncthreads();
      if (next < tiles) { send(next, slot); next += gridDim.x; left++; slot = slot + 1 == RS ? 0 : slot + 1; }
    }
    if (bits_out) __syncthreads();
    return;
  }
  // ---- the multiplying wavefronts
  const uint32_t n0 = wave * 32;
  v8 fb[KS];                                 // B's rows n0 + (lane & 31): the step's eight elements of this lane
  {
    // (loads without conditions, so that all are on their way together; K is a multiple of eight: a lane's eight exist or not)
    const uint32_t row = min(n0 + (lane & 31), a.N - 1);
    if (n.b_rows) {
#pragma unroll
      for (int q = 0; q < KS; q++) {
        const uint32_t k = q * 16 + (lane >> 5) * 8;
        const T *p = static_cast<const T *>(a.B) + row;
        T e[8];
#pragma unroll
        for (int j = 0; j < 8; j++) e[j] = p[(int64_t)min(k + j, n.b_rows - 1) * a.ldb];
        __builtin_memcpy(&fb[q], e, 16);
      }
    } else {
#pragma unroll
      for (int q = 0; q < KS; q++) {
        const uint32_t k = q * 16 + (lane >> 5) * 8;
        const uint4 w = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.B) + (int64_t)row * a.ldb + (k < a.K ? k : 0));
        __builtin_memcpy(&fb[q], &w, 16);
      }
    }
#pragma unroll
    for (int q = 0; q < KS; q++)
      if (q * 16 + (lane >> 5) * 8 >= a.K) {
        const uint4 zero = make_uint4(0, 0, 0, 0);
        __builtin_memcpy(&fb[q], &zero, 16);
      } else if (n.b_rows && q * 16 + (lane >> 5) * 8 + 8 > n.b_rows) {
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (q * 16 + (lane >> 5) * 8 + j >= n.b_rows) fb[q][j] = (T)0.f;
      }
  }
  float *mine = reinterpret_cast<float *>(lds + RS * kPlace) + wave * 512;             // 16 rows of 32 columns
  uint8_t *bits = reinterpret_cast<uint8_t *>(lds + RS * kPlace + NWC * 2048);         // two tiles of R rows, 32 bytes each
  const uint32_t er = lane >> 2, ec = lane & 3, col = n0 + ec * 8;
  const int left = min(8, (int)a.N - (int)col);
  float b[8];
  load_bias<T>(a, col, left, b);
  const uint32_t bw = (uint32_t)(kept_pitch(1, a.N) / 16);             // words of an output row of bits (1 or 2)
  auto flush_bits = [&](uint32_t tile, uint32_t which) {               // R rows x bw words, by the first wavefront
    const uint32_t w = threadIdx.x, r = w / bw, m = tile * R + r;
    if (w < R * bw && m < a.M) *reinterpret_cast<uint4 *>(a.kept + ((uint64_t)m * bw + w % bw) * 16) = *reinterpret_cast<const uint4 *>(bits + (which * R + r) * 32 + (w % bw) * 16);
  };
  if (bits_out) {                            // (columns past N: no bits)
    for (uint32_t w = threadIdx.x; w < 2 * R * 8; w += NWC * 64) reinterpret_cast<uint32_t *>(bits)[w] = 0;
  }
  auto form_dz = [&](char *place, uint32_t row0) {
#pragma unroll
    for (int i = 0; i < R * W / (NWC * 64); i++) {
      const uint32_t w = i * NWC * 64 + threadIdx.x, r = w / W, c = w % W;
      uint4 *p = reinterpret_cast<uint4 *>(place + (r * W + swz_row<W>(r, c)) * 16);
      uint4 z = make_uint4(0, 0, 0, 0);
      if constexpr (SIDE == 2) z = *reinterpret_cast<const uint4 *>(place + kA + (r * W + swz_row<W>(r, c)) * 16);
      else if (c * 8 < a.K) z.x = *reinterpret_cast<const uint8_t *>(place + kA + r * (kept_pitch(1, a.K)) + c);
      const uint4 d = dz_word<T>(n.kept_act, *p, z);
      *p = d;
      if (n.dz && row0 + r < a.M && c * 8 < a.K) *reinterpret_cast<uint4 *>(static_cast<T *>(n.dz) + (int64_t)(row0 + r) * n.lddz + c * 8) = d;
    }
  };
  if constexpr (SIDE >= 2) {
    __syncthreads();
    form_dz(lds, blockIdx.x * R);
  }
  uint32_t at = 0, turn = 0;
  for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, turn ^= 1) {
    char *cur = lds + at * kPlace;
    at = at + 1 == RS ? 0 : at + 1;
    __syncthreads();
    const uint32_t m0 = tile * R;
    if (bits_out && tile != blockIdx.x) flush_bits(tile - gridDim.x, turn ^ 1);
    if constexpr (SIDE >= 2) {
      if (tile + gridDim.x < tiles) form_dz(lds + at * kPlace, m0 + gridDim.x * R);
    }
    f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; e++) acc[e] = 0.f;
    // (operands are read eight steps ahead, four at a time: left to itself the compiler reads one ahead and waits for LDS at every product)
    const uint32_t ra = lane & 31;
    v8 fa[8];
#pragma unroll
    for (int q = 0; q < 8; q++) fa[q] = *reinterpret_cast<const v8 *>(cur + (ra * W + swz_row<W>(ra, q * 2 + (lane >> 5))) * 16);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int g = 0; g < KS / 4; g++) {
#pragma unroll
      for (int q = 0; q < 4; q++) acc = mma(fb[g * 4 + q], fa[(g & 1) * 4 + q], acc);
      if (g + 2 < KS / 4) {
#pragma unroll
        for (int q = 0; q < 4; q++) fa[(g & 1) * 4 + q] = *reinterpret_cast<const v8 *>(cur + (ra * W + swz_row<W>(ra, (g * 4 + 8 + q) * 2 + (lane >> 5))) * 16);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (uint32_t h = 0; h < 2; h++) {       // 16 rows at a time through this wavefront's corner (word w of row r at w ^ ((r >> 1) & 7))
      if (((lane >> 4) & 1) == h) {
#pragma unroll
        for (int e = 0; e < 4; e++)
          *reinterpret_cast<float4 *>(mine + (lane & 15) * 32 + swz(lane & 15, e * 2 + (lane >> 5)) * 4) =
              make_float4(acc[4 * e], acc[4 * e + 1], acc[4 * e + 2], acc[4 * e + 3]);
      }
      wave_order();
      const uint32_t r = h * 16 + er, m = m0 + r;
      if (m < a.M && left > 0) {
        float v[8];
        *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(mine + er * 32 + swz(er, ec * 2) * 4);
        *reinterpret_cast<float4 *>(v + 4) = *reinterpret_cast<const float4 *>(mine + er * 32 + swz(er, ec * 2 + 1) * 4);
        uint4 resw = make_uint4(0, 0, 0, 0);
        if constexpr (SIDE == 1) resw = *reinterpret_cast<const uint4 *>(cur + kA + (r * WS + swz_row<WS>(r, wave * 4 + ec)) * 16);
        finish8<T>(a, m, col, left, v, b, resw, bits_out ? bits + (turn * R + r) * 32 + col / 8 : nullptr);
      }
      wave_order();
    }
  }
  if (bits_out) {
    __syncthreads();
    // (the last tile: the largest that this workgroup walks)
    const uint32_t last = blockIdx.x + (tiles - 1 - blockIdx.x) / gridDim.x * gridDim.x;
    flush_bits(last, turn ^ 1);
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

template <typename T, Via VIA>
struct RowLoader {
  const T *base;                             // row 0 of the operand
  int64_t ld;
  uint32_t c0, width;                        // the tile's first column; columns of the operand
  uint32_t past;                             // rows fetched that do not exist (the slice's last stage): from row `past` of the stage on
  uint4 reg[VIA == kWords ? 1 : 4];
  __device__ __forceinline__ void start(uint32_t r0, uint32_t r1, char *lds) {       // rows r0 .. r0 + 63, those at and past r1 read as zero
    past = r1 - r0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t w = i * kThreads + threadIdx.x, r = w >> 4, c = c0 + swz_t(r, w & 15) * 8;
      const T *row = base + (int64_t)min(r0 + r, r1 - 1) * ld;
      if (VIA == kWords) lds_dma16(r0 + r < r1 && c < width ? (const void *)(row + c) : (const void *)g_zero16, lds + (i * kThreads + (threadIdx.x & ~63u)) * 16);
      else if (VIA == kRegs) reg[i] = fetch_word(row, c, width);
      else reg[i] = load_elems(row, c, width);
    }
  }
  __device__ __forceinline__ void finish(char *lds) {
    if (VIA != kWords) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t w = i * kThreads + threadIdx.x, r = w >> 4;
        if (VIA == kRegs && c0 + 128 > width) reg[i] = settle_word(reg[i], c0 + swz_t(r, w & 15) * 8, width);
        *reinterpret_cast<uint4 *>(lds + w * 16) = r < past ? reg[i] : make_uint4(0, 0, 0, 0);
      }
    }
  }
};

// eight consecutive rows k .. k + 7 of column c0 + (lane & 15), as a product's operand: two transposing reads of four rows each (lane
// 4 q + p of a group of 16 points at 8-byte piece p of row q; it receives column (lane & 15) of the four rows)
template <typename T, int W>
__device__ __forceinline__ typename Frag<T>::v8 read_cols(const char *img, uint32_t k, uint32_t c0) {
  const uint32_t l = lane_id() & 15, r = l >> 2, p = l & 3;
  typedef short s4 __attribute__((ext_vector_type(4)));
  union { s4 h[2]; typename Frag<T>::v8 v; } u;
#pragma unroll
  for (int t = 0; t < 2; t++) {
    const uint32_t row = k + 4 * t + r, word = (c0 >> 3) + (p >> 1);
    const char *at = img + (row * W + swz_t(row, word)) * 16 + (p & 1) * 8;
    u.h[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)at);
  }
  return u.v;
}

template <typename T, Via DA, Via DB>
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
  la.base = static_cast<const T *>(a.A); la.ld = a.lda; la.c0 = n0; la.width = a.N;
  lb.base = static_cast<const T *>(a.B); lb.ld = a.ldb; lb.c0 = k0; lb.width = a.K;
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
        fa[h][q] = read_cols<T, 16>(cur, kk, wn + h * 32 + half);
        fb[h][q] = read_cols<T, 16>(cur + kTileBytes, kk, wk + h * 32 + half);
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

// dz^T x of narrow operands (N <= 128 NB, K <= 64 KB): one workgroup holds all of dW -- 128 x 64 per wavefront -- and walks one row
// slice, 32 rows a stage, both operands read once.  BITS: A is dy and its stage is masked in place by relu's (leakyrelu's) kept bits.
// (Two workgroups per slice of 128 columns of dz each halve the partial products but read x twice: 120 + 9 instead of 80 + 15 us at
// 289127 x 256 x 256.)
// db: dz^T 1 on the same products, the 32-column groups of a 128-column block dealt to the block's KB wavefronts.
struct TnNarrowArgs {
  TnArgs t;
  const char *kept;
  int kept_act;
};

template <typename T, int NB, int KB, int RS, bool BITS>
__global__ void __launch_bounds__(NB * KB * 64, 2) tn_narrow_kernel(TnNarrowArgs n) {
  typedef typename Frag<T>::v8 v8;
  constexpr int THREADS = NB * KB * 64, WA = NB * 16, WB = KB * 8;   // words of a row of dz and of x
  constexpr int kA = 32 * WA * 16, kB = 32 * WB * 16, kM = BITS ? 1024 : 0, kBoth = kA + kB + kM;
  constexpr int PA = 32 * WA / THREADS, PB = 32 * WB / THREADS, PER = PA + PB + (BITS ? 1 : 0), NJ = 4 / KB;
  static_assert(PA >= 1 && PB >= 1, "whole transfers");
  __shared__ __attribute__((aligned(16))) char lds[RS * kBoth];
  const TnArgs &a = n.t;
  const uint32_t lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave / KB, wk = wave % KB;
  const uint32_t r0 = blockIdx.x * a.per, r1 = min(a.M, r0 + a.per);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(lds)) + wave * 1024, ldsm = __builtin_amdgcn_readfirstlane(lds_addr(lds)) + kA + kB;
  const uint32_t kw = (uint32_t)(kept_pitch(1, a.N) / 16);           // words of a row of kept bits (1 or 2)
  auto send = [&](uint32_t row, uint32_t slot) {
#pragma unroll
    for (int i = 0; i < PA; i++) {
      const uint32_t w = i * THREADS + threadIdx.x, r = w / WA, c = swz_t(r, w % WA) * 8;
      const T *p = static_cast<const T *>(a.A) + (int64_t)(row + r) * a.lda + c;
      lds_dma16_async(row + r < r1 && c < a.N ? (const void *)p : (const void *)g_zero16, lds0 + slot * kBoth + i * THREADS * 16);
    }
#pragma unroll
    for (int i = 0; i < PB; i++) {
      const uint32_t w = i * THREADS + threadIdx.x, r = w / WB, c = swz_t(r, w % WB) * 8;
      const T *p = static_cast<const T *>(a.B) + (int64_t)(row + r) * a.ldb + c;
      lds_dma16_async(row + r < r1 && c < a.K ? (const void *)p : (const void *)g_zero16, lds0 + slot * kBoth + kA + i * THREADS * 16);
    }
    if constexpr (BITS) {                    // (every wavefront sends the same 64 words: one count of transfers for all)
      const uint32_t r = lane / kw;
      const char *p = n.kept + (uint64_t)(row + r) * kw * 16 + (lane % kw) * 16;
      lds_dma16_async(r < 32 && row + r < r1 ? (const void *)p : (const void *)g_zero16, ldsm + slot * kBoth);
    }
  };
  f32x16 acc[4][2], accb[NJ];                // [n][k] 32 x 32 blocks
#pragma unroll
  for (int e = 0; e < 16; e++) {
#pragma unroll
    for (int i = 0; i < 4; i++) acc[i][0][e] = acc[i][1][e] = 0.f;
#pragma unroll
    for (int i = 0; i < NJ; i++) accb[i][e] = 0.f;
  }
  v8 ones;
#pragma unroll
  for (int j = 0; j < 8; j++) ones[j] = (T)1.0f;
  uint32_t next = r0, slot = 0;
  for (int s = 0; s < RS - 1; s++)
    if (next < r1) { send(next, slot); next += 32; slot++; }
  uint32_t left = slot, at = 0;
  for (uint32_t row = r0; row < r1; row += 32) {
    if (left == RS - 1) wait_vm<(RS - 2) * PER>();
    else wait_vm<0>();
    left--;
    __syncthreads();                         // the stage is whole, the one before it has been read
    char *cur = lds + at * kBoth;
    at = at + 1 == RS ? 0 : at + 1;
    if (next < r1) { send(next, slot); next += 32; left++; slot = slot + 1 == RS ? 0 : slot + 1; }
    if constexpr (BITS) {
#pragma unroll
      for (int i = 0; i < PA; i++) {
        const uint32_t w = i * THREADS + threadIdx.x, r = w / WA, c = w % WA;
        uint4 *p = reinterpret_cast<uint4 *>(cur + (r * WA + swz_t(r, c)) * 16);
        const uint32_t bits = c * 8 < a.N ? *reinterpret_cast<const uint8_t *>(cur + kA + kB + r * kw * 16 + c) : 0u;
        *p = dz_word<T>(n.kept_act, *p, make_uint4(bits, 0, 0, 0));
      }
      __syncthreads();
    }
#pragma unroll
    for (int q = 0; q < 2; q++) {
      const uint32_t kk = q * 16 + (lane >> 5) * 8, half = ((lane >> 4) & 1) * 16;
      v8 fa[4], fb[2];
#pragma unroll
      for (int i = 0; i < 4; i++) fa[i] = read_cols<T, WA>(cur, kk, wn * 128 + i * 32 + half);
#pragma unroll
      for (int j = 0; j < 2; j++) fb[j] = read_cols<T, WB>(cur + kA, kk, wk * 64 + j * 32 + half);
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = mma(fa[i], fb[j], acc[i][j]);
      if (a.part_b) {
#pragma unroll
        for (int i = 0; i < 4; i++)          // (a wavefront-uniform choice among registers: four branches)
          if (wk == (uint32_t)(i % KB)) accb[i / KB] = mma(fa[i], ones, accb[i / KB]);
      }
    }
  }
  // a lane holds column k = lane & 31: 128-byte lines of the partial product
  float *part = a.part + (uint64_t)blockIdx.x * a.N * a.K;
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const uint32_t r = wn * 128 + i * 32 + (e >> 2) * 8 + (lane >> 5) * 4 + (e & 3);
      if (r >= a.N) continue;
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const uint32_t k = wk * 64 + j * 32 + (lane & 31);
        if (k < a.K) part[(uint64_t)r * a.K + k] = acc[i][j][e];
      }
      if (a.part_b && wk == (uint32_t)(i % KB) && (lane & 31) == 0) a.part_b[(uint64_t)blockIdx.x * a.N + r] = accb[i / KB][e];
    }
}

// dz^T x over few rows: 32 x 32 tiles of dW, the rows cut over the workgroup's eight wavefronts (16 at a time) and joined in LDS in
// wavefront order; dz is formed element by element from dy and what was kept.  One launch, no scratch; db from the tiles of the first
// 32 columns of x.
struct TnFewArgs {
  TnArgs t;
  const char *kept;
  int kept_act;                              // 0: A is dz
  void *db;
  int db_f32;
};
template <typename T>
__global__ void __launch_bounds__(512) tn_few_kernel(TnFewArgs f) {
  typedef typename Frag<T>::v8 v8;
  constexpr int kPitch = 33;
  __shared__ float part[8][32 * kPitch], part_b[8][64];
  const TnArgs &a = f.t;
  const uint32_t tn = blockIdx.x / a.tiles_k, tk = blockIdx.x % a.tiles_k, n0 = tn * 32, k0 = tk * 32;
  const uint32_t lane = lane_id(), wave = wave_id(), c = lane & 31;
  const uint32_t n = min(n0 + c, a.N - 1), k = min(k0 + c, a.K - 1);
  const uint64_t pitch = kept_pitch(f.kept_act, a.N);
  f32x16 acc;
#pragma unroll
  for (int e = 0; e < 16; e++) acc[e] = 0.f;
  float sum = 0.f;
  for (uint32_t m0 = wave * 16 + (lane >> 5) * 8; m0 - (lane >> 5) * 8 < a.M; m0 += 128) {
    T ea[8], eb[8];
    float slope[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {            // (rows past the end repeat the last and are cleared below)
      const uint32_t m = min(m0 + j, a.M - 1);
      ea[j] = static_cast<const T *>(a.A)[(int64_t)m * a.lda + n];
      eb[j] = static_cast<const T *>(a.B)[(int64_t)m * a.ldb + k];
      slope[j] = !f.kept_act ? 0.f : keeps_bits(f.kept_act) ? (float)((uint8_t)f.kept[m * pitch + n / 8] >> (n & 7) & 1u)
                                                            : (float)*reinterpret_cast<const f16_t *>(f.kept + m * pitch + n * 2);
    }
    v8 fa, fb;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      float v = (float)ea[j];
      if (f.kept_act) {
        const float s = keeps_bits(f.kept_act) ? (slope[j] != 0.f ? 1.f : f.kept_act == 4 ? 0.2f : 0.f) : slope16(f.kept_act, slope[j]);
        v = v == 0.f || s == 0.f ? 0.f : v * s;
      }
      const bool in = m0 + j < a.M;
      fa[j] = in ? (T)v : (T)0.f;
      fb[j] = in ? eb[j] : (T)0.f;
      sum += (float)fa[j];
    }
    acc = mma(fa, fb, acc);                  // rows: n, columns (lanes): k
  }
#pragma unroll
  for (int e = 0; e < 16; e++) part[wave][((e >> 2) * 8 + (lane >> 5) * 4 + (e & 3)) * kPitch + c] = acc[e];
  part_b[wave][lane] = sum;
  __syncthreads();
  for (uint32_t o = threadIdx.x; o < 1024; o += 512) {
    const uint32_t r = o >> 5, q = o & 31;
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 8; w++) t += part[w][r * kPitch + q];
    if (n0 + r < a.N && k0 + q < a.K) static_cast<T *>(a.C)[(int64_t)(n0 + r) * a.ldc + k0 + q] = (T)t;
  }
  if (f.db && tk == 0 && threadIdx.x < 32 && n0 + threadIdx.x < a.N) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 8; w++) t += part_b[w][threadIdx.x] + part_b[w][32 + threadIdx.x];
    if (f.db_f32) static_cast<float *>(f.db)[n0 + threadIdx.x] = t;
    else static_cast<T *>(f.db)[n0 + threadIdx.x] = (T)t;
  }
}

// Sums of the slices: 64 outputs per workgroup, each of its four wavefronts every fourth slice, joined in wavefront order (always the
// same order).  The first N K outputs are dW (part null: it is written already), N more db (part_b null: not wanted).
template <typename T>
__global__ void __launch_bounds__(256) tn_join_kernel(const float *__restrict__ part, const float *__restrict__ part_b, uint32_t slices, uint32_t N,
                                                      uint32_t K, T *C, int64_t ldc, void *db, int db_f32) {
  __shared__ float sums[4][64];
  const uint64_t total = part ? (uint64_t)N * K : 0;
  const uint64_t o = (uint64_t)blockIdx.x * 64 + lane_id(), e = o < total ? o : o - total;
  const bool in = o < total + (part_b ? N : 0);
  const float *src = o < total ? part : part_b;
  const uint64_t step = o < total ? total : N;
  float t = 0.f;
  if (in) {
#pragma unroll 8
    for (uint32_t s = wave_id(); s < slices; s += 4) t += src[s * step + e];
  }
  sums[wave_id()][lane_id()] = t;
  __syncthreads();
  if (wave_id() != 0 || !in) return;
  t = (sums[0][lane_id()] + sums[1][lane_id()]) + (sums[2][lane_id()] + sums[3][lane_id()]);
  if (o < total) C[(int64_t)(e / K) * ldc + e % K] = (T)t;
  else if (db_f32) static_cast<float *>(db)[e] = t;
  else static_cast<T *>(db)[e] = (T)t;
}

// ------------------------------------------------------------------------------------------------ elementwise pieces
// dz = dy act'(z) (an identity: dy) in rows of whole words, whose pad columns are zero
template <typename T>
__global__ void __launch_bounds__(256) dz_kernel(const T *dy, int64_t lddy, const char *kept, T *dz, int64_t ld, uint32_t M, uint32_t N, int act) {
  const uint32_t words = (uint32_t)(ld / 8);
  const uint64_t total = (uint64_t)M * words, pitch = kept_pitch(act, N);
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
    const uint64_t m = i / words;
    const uint32_t w = (uint32_t)(i % words);
    const uint4 g = load_word(dy + (int64_t)m * lddy, w * 8, N);       // (zero past N)
    uint4 z = make_uint4(0, 0, 0, 0);
    if (act && keeps_bits(act)) z.x = (uint8_t)kept[m * pitch + w];
    else if (act) z = *reinterpret_cast<const uint4 *>(kept + m * pitch + w * 16);
    *reinterpret_cast<uint4 *>(dz + (int64_t)m * ld + w * 8) = act ? dz_word<T>(act, g, z) : g;
  }
}

// W [N, K] -> W^T [K, ld] (ld >= N, pad zero) in 32 x 32 tiles
template <typename T>
__global__ void __launch_bounds__(256) transpose_kernel(const T *W, int64_t ldw, uint32_t N, uint32_t K, T *out, int64_t ld) {
  __shared__ T tile[32][33];
  const uint32_t across = (K + 31) / 32, n0 = blockIdx.x / across * 32, k0 = blockIdx.x % across * 32, c = threadIdx.x & 31, r = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    tile[r + i][c] = n0 + r + i < N && k0 + c < K ? W[(int64_t)(n0 + r + i) * ldw + k0 + c] : (T)0.f;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    if (k0 + r + i < K && n0 + c < ld) out[(int64_t)(k0 + r + i) * ld + n0 + c] = tile[c][r + i];
}

// the tall, narrow form: widths up to 256, the contraction's in whole words (a gradient's dz is: pad columns).  8192 x 256 -> 256 takes 8.4
// us (dx 9.4) so and 10.2 (12.7) in 128 x 128 tiles, 32768 rows 15 (16) and 14 (17), 289127 105 and 140; fewer rows leave CUs idle.
bool narrow_shape(uint32_t M, uint32_t N, uint32_t K) { return N <= 256 && K <= 256 && K % 8 == 0 && M >= 8192; }
// ... of dz^T x, where 128 x 128 tiles would read an operand twice: dx and dW of 131072 x 256 -> 256 relu take 91 us so and 101 in tiles,
// 65536 rows 64 and 58, 131072 x 64 -> 64 (one tile) 55 and 37
bool narrow_dw_shape(uint32_t M, uint32_t N, uint32_t K) { return narrow_shape(M, N, K) && M >= 98304 && (N > 128 || K > 128); }
// dx of so few outputs goes through nt_short_kernel (its wavefronts hold 64 steps of the contraction)
constexpr uint32_t kShort = 64;

inline uint64_t tiles128(uint32_t M, uint32_t N) { return (uint64_t)((M + 127) / 128) * ((N + 127) / 128); }

// dz^T x in one launch of 32 x 32 tiles: 256 rows of 256 x 256 take 8 us so and 17 in slices of 128 x 128 tiles (dz, product, join),
// 1024 rows 24 and 18
bool few_rows(uint32_t M, uint32_t N, uint32_t K) { return M <= 512 && (uint64_t)((N + 31) / 32) * ((K + 31) / 32) <= 1024; }

// Which kernels a backward pass goes through, and what they need in memory.
struct BwdWay {
  bool dy_words, dz_words;                   // rows of whole words: dy's, and those of what dx and dW read
  bool narrow_dx, few_dx, short_dx, narrow_dw, bits_dw, few_dw, tiles_dw;
  bool need_dz, need_wt;                     // dz and the transposed weight in the scratch
};
// small_w: the weight's pitch is below 2^22 elements
BwdWay way_of(int act, uint32_t M, uint32_t N, uint32_t K, bool dy_words, bool x_words, bool small_w, bool want_dx, bool want_dw) {
  BwdWay w;
  w.dy_words = dy_words;
  // a dy of few columns whose rows are not whole words is first laid out in such rows: loads of unaligned rows, many times over, cost
  // more (dx and dW of 20011 x 47 -> 500: 43 us so, 35 with the pass; 289127 x 47 -> 256: 152 and 117; 289127 x 172 -> 128: 120 and 133)
  const bool pad = !act && !dy_words && N <= kShort;
  w.dz_words = act || pad || dy_words;
  w.narrow_dx = want_dx && narrow_shape(M, N, K) && w.dz_words;
  w.few_dx = want_dx && M && !w.narrow_dx && tiles128(M, K) < 64;
  w.short_dx = want_dx && M && !w.narrow_dx && !w.few_dx && N <= kShort && small_w;
  w.narrow_dw = want_dw && narrow_dw_shape(M, N, K) && x_words && w.dz_words;
  w.bits_dw = w.narrow_dw && keeps_bits(act) && dy_words;              // (dz^T x masks dy itself)
  w.few_dw = want_dw && M && !w.narrow_dw && few_rows(M, N, K);
  w.tiles_dw = want_dw && !w.narrow_dw && !w.few_dw;
  // dz in memory, in rows of whole words, unless what reads it forms it itself
  w.need_dz = M && (act || pad) && ((want_dx && !w.few_dx && !(w.narrow_dx && dy_words)) || (want_dw && !w.bits_dw && !w.few_dw));
  w.need_wt = want_dx && M && !w.narrow_dx && !w.few_dx && !w.short_dx;
  return w;
}

struct BwdPlan {
  uint32_t slices, per;                      // of dz^T x
  uint64_t dz, wt, part, part_b, total;      // byte offsets in the scratch
};

BwdPlan plan_bwd(uint32_t M, uint32_t N, uint32_t K, const BwdWay &w) {
  BwdPlan p;
  const uint64_t tiles = (uint64_t)((N + BN - 1) / BN) * ((K + BM - 1) / BM);
  // row slices of dz^T x: one workgroup per CU, at least four stages each
  uint32_t s = w.narrow_dw || tiles == 0 ? 256 : (uint32_t)(256 / tiles);
  const uint32_t most = (M + 4 * BK - 1) / (4 * BK);
  s = s < 1 ? 1 : s;
  s = s > most ? most : s;
  s = s < 1 ? 1 : s;
  p.per = (uint32_t)up((M + s - 1) / s, BK);
  p.slices = M ? (M + p.per - 1) / p.per : 1;
  uint64_t at = 0;
  p.dz = at; at += w.need_dz ? up((uint64_t)M * up(N, 8) * 2, 256) : 0;
  p.wt = at; at += w.need_wt ? up((uint64_t)K * up(N, 8) * 2, 256) : 0;
  p.part = at; at += w.narrow_dw || (w.tiles_dw && p.slices > 1) ? up((uint64_t)p.slices * N * K * 4, 256) : 0;
  p.part_b = at; at += w.narrow_dw || w.tiles_dw ? up((uint64_t)p.slices * N * 4, 256) : 0;
  p.total = at;
  return p;
}

bool dtype16(int d) { return d == SL_BF16 || d == SL_F16; }

template <typename T, int BM_, int BN_, int WM, int WN, int OCC, int PERCU, bool DIRECT>
void nt_tiles(GemmArgs a, hipStream_t st) {
  a.tiles_m = (a.M + BM_ - 1) / BM_; a.tiles_n = (a.N + BN_ - 1) / BN_;
  const uint32_t tiles = a.tiles_m * a.tiles_n, most = 256 * PERCU;       // (a multiple of eight: a workgroup stays on its XCD's tiles)
  // (nothing of the next tile is on its way in the form through registers: a workgroup per tile there)
  hipLaunchKernelGGL((nt_kernel<T, BM_, BN_, WM, WN, 2, OCC, DIRECT>), dim3(DIRECT && tiles > most ? most : tiles), dim3(WM * WN * 64), 0, st, a);
}

template <typename T, int SIDE>
void narrow_launch(const NarrowArgs &n, hipStream_t st) {
  const uint32_t tiles = (n.g.M + 31) / 32;
  // (places of the ring by what LDS holds: 96 to 112 KB on their way on a CU in SIDE 0 and 1)
#define SHD_NARROW(NWC, KS, RS, PERCU)                                                                                                  \
  hipLaunchKernelGGL((narrow_kernel<T, NWC, KS, RS, SIDE>), dim3(tiles < 256 * PERCU ? tiles : 256 * PERCU), dim3((NWC + 4) * 64), 0, st, n)
  if (n.g.N <= 128) {
    if (n.g.K <= 128) SHD_NARROW(4, 8, 4, 2);
    else SHD_NARROW(4, 16, 4, 1);
  } else {
    if (n.g.K <= 128) SHD_NARROW(8, 8, 5, 1);
    else SHD_NARROW(8, 16, (SIDE == 1 || SIDE == 2 ? 4 : 6), 1);
  }
#undef SHD_NARROW
}

template <typename T, bool BITS>
void tn_narrow_launch(const TnNarrowArgs &n, hipStream_t st) {
  const dim3 g(n.t.slices);
  if (n.t.N <= 128) {
    hipLaunchKernelGGL((tn_narrow_kernel<T, 1, 4, 4, BITS>), g, dim3(256), 0, st, n);      // (K > 128)
  } else {
    if (n.t.K <= 128) hipLaunchKernelGGL((tn_narrow_kernel<T, 2, 2, 4, BITS>), g, dim3(256), 0, st, n);
    else hipLaunchKernelGGL((tn_narrow_kernel<T, 2, 4, 4, BITS>), g, dim3(512), 0, st, n);
  }
}

template <typename T, bool COLS>
void few_launch(FewArgs f, bool words, hipStream_t st) {
  f.g.tiles_m = (f.g.M + 31) / 32; f.g.tiles_n = (f.g.N + 31) / 32;
  const dim3 g(f.g.tiles_m * f.g.tiles_n), b(512);
  if (words) hipLaunchKernelGGL((nt_few_kernel<T, kWords, COLS>), g, b, 0, st, f);
  else if (f.g.K >= 8) hipLaunchKernelGGL((nt_few_kernel<T, kRegs, COLS>), g, b, 0, st, f);
  else hipLaunchKernelGGL((nt_few_kernel<T, kElems, COLS>), g, b, 0, st, f);
}

template <typename T>
void short_launch(const GemmArgs &a, hipStream_t st) {
  const uint32_t groups = (a.N + 63) / 64, tiles = (a.M + 31) / 32;
  // (as many tiles per wavefront as leave every SIMD two wavefronts, sixteen at most)
  const uint64_t p = (uint64_t)tiles * groups / 2048;
  const uint32_t per = p < 1 ? 1 : p > 16 ? 16 : (uint32_t)p;
  const uint64_t items = ((uint64_t)tiles + per - 1) / per * groups;
  hipLaunchKernelGGL((nt_short_kernel<T>), dim3((uint32_t)((items + 3) / 4)), dim3(256), 0, st, a, groups, per);
}

// the grid of 32 x 32 tiles: a launch has fewer than 2^32 threads
bool few_fits(uint32_t M, uint32_t N) { return (((uint64_t)M + 31) / 32) * (((uint64_t)N + 31) / 32) < 1u << 23; }
// x W^T in 32 x 32 tiles: fewer than 64 tiles of 128 (1024 x 1024 x 1024, 64 tiles, takes 17.6 us in 32 x 32 tiles and 18.0 in 128 x 128
// ones, twice the rows 32 and 18.5, 1024 x 256 x 256 4.5 and 9.6, one row of 4096 x 4096 11 and 47), fewer than 128 where half of each were
// empty (8192 x 1024 -> 40 9.1 and 17.6, 16000 x 500 -> 48 9.4 to 11.3 and 12.8 to 14.2, but 16000 x 2000 -> 64 37 and 32; above, the
// times cross at about 150 tiles: 16512 x 500 -> 48 12.3 and 13.8, 20011 x 500 -> 47 15.0 and 14.7, 30000 19.6 and 15.4, 50000 30 and 20,
// 20011 x 1000 -> 47 24 and 21, 20011 x 256 -> 47 7.5 and 7.6), any number where three quarters
// were (30000 x 500 -> 16 8.9 and 14.8, 100000 x 600 -> 8 27 and 38, but 60000 x 1000 -> 32 39 and 31); and what the tile kernel does not
// hold: its offsets (256 rows of a pitch below 2^22 elements stay below 2^31 bytes) and contractions of less than eight, both rare
bool takes_few(uint32_t M, uint32_t N, uint32_t K, int64_t lda, int64_t ldb) {
  return tiles128(M, N) < (N <= 64 && K <= 1024 ? 128u : 64u) || (N <= 32 && K <= 640 && few_fits(M, N)) || lda >= (1 << 22) || ldb >= (1 << 22) || K < 8;
}

// 256 x 256 tiles: from 1024 tiles of 128 on (32768 x 1024 -> 1024 82 us in 256 x 256 tiles and 103 in 128 x 128 ones, 8192 x 1024 -> 2048
// 41 and 48, 65536 x 512 -> 256 33 and 39, 4096^3 117 and 143; half as many tiles leave CUs idle: 8192 x 1024 -> 1024 35 and 25, 4096 x 4096
// -> 2048 95 and 72), unless half of each were empty (131072 x 512 -> 128 56 and 47), and of contractions of 512 and more.  (Shorter ones are
// faster so too -- 65536 x 256 -> 1024 76 and 96, 32768 x 256 -> 1024 37 and 42, 65536 x 384 -> 512 49 and 63 -- and still go to 128 x 128.)
template <typename T>
void nt_launch(GemmArgs a, hipStream_t st) {
  const bool direct = rows_of_words(a.A, a.lda, a.K, SL_BF16) && rows_of_words(a.B, a.ldb, a.K, SL_BF16);
  // (what is kept of rows that are not whole words leaves this kernel slowly: 289127 x 256 -> 47 relu takes 66 us here and 57 in tiles,
  //  without it 47 and 51, 128 -> 172 54 and 73)
  if (direct && narrow_shape(a.M, a.N, a.K) && rows_of_words(a.res, a.ldr, a.N, SL_BF16) && (a.N % 8 == 0 || !a.kept)) {
    NarrowArgs n = {};
    n.g = a;
    if (a.res) narrow_launch<T, 1>(n, st);
    else narrow_launch<T, 0>(n, st);
    return;
  }
  const uint64_t tiles = tiles128(a.M, a.N);
  if (takes_few(a.M, a.N, a.K, a.lda, a.ldb)) {
    FewArgs f = {};
    f.g = a;
    few_launch<T, false>(f, direct, st);
  } else if (direct && tiles >= 1024 && a.K >= 512 && a.N >= 256) {
    nt_tiles<T, 256, 256, 2, 4, 2, 1, true>(a, st);
  } else if (direct) {
    nt_tiles<T, 128, 128, 2, 2, 2, 2, true>(a, st);
  } else {
    nt_tiles<T, 128, 128, 2, 2, 2, 2, false>(a, st);
  }
}

template <typename T>
void tn_launch(const TnArgs &a, bool dz_words, bool x_words, hipStream_t st) {
  const dim3 g(a.tiles_n * a.tiles_k * a.slices), b(kThreads);
  if (!dz_words && a.K >= 8) hipLaunchKernelGGL((tn_kernel<T, kRegs, kRegs>), g, b, 0, st, a);       // (more than 64 columns)
  else if (!dz_words) hipLaunchKernelGGL((tn_kernel<T, kRegs, kElems>), g, b, 0, st, a);
  else if (x_words) hipLaunchKernelGGL((tn_kernel<T, kWords, kWords>), g, b, 0, st, a);
  else if (a.K >= 8) hipLaunchKernelGGL((tn_kernel<T, kWords, kRegs>), g, b, 0, st, a);
  else hipLaunchKernelGGL((tn_kernel<T, kWords, kElems>), g, b, 0, st, a);
}

#define SHD_DISPATCH_16(DTYPE, ...)                         \
  if ((DTYPE) == SL_BF16) { using T = bf16_t; __VA_ARGS__; }\
  else { using T = f16_t; __VA_ARGS__; }

constexpr uint64_t kMaxTiles = 0xFFFFFFull;   // of 256 threads each

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
                               void *d_kept, void *stream) {
  if (const int rc = check_sizes("sl_linear16_fwd", dtype, act, M, N, K)) return rc;
  if (M == 0) return SG_OK;
  if (!d_x || !d_w || !d_y || ldx < (int64_t)K || ldw < (int64_t)K || ldy < (int64_t)N || (d_res && ldr < (int64_t)N) ||
      (d_kept && (reinterpret_cast<uintptr_t>(d_kept) & 15)))
    return set_error(SG_ERR_INVALID, "sl_linear16_fwd: operands");
  if (takes_few(M, N, K, ldx, ldw) && !few_fits(M, N)) return set_error(SG_ERR_INVALID, "sl_linear16_fwd: too many tiles");
  hipStream_t st = (hipStream_t)stream;
  GemmArgs a = {};
  a.A = d_x; a.lda = ldx; a.B = d_w; a.ldb = ldw; a.M = M; a.N = N; a.K = K; a.bias = d_bias; a.bias_f32 = bias_f32; a.res = d_res; a.ldr = ldr;
  a.C = d_y; a.ldc = ldy; a.kept = act ? static_cast<char *>(d_kept) : nullptr; a.act = act;
  SHD_PROF_FMT(2.0 * ((double)M * K + (double)N * K + (double)M * N * (d_res ? 2 : 1)), 2.0 * M * N * K, st, "linear16_fwd_N%u_K%u", N, K);
  SHD_DISPATCH_16(dtype, nt_launch<T>(a, st));
  SHD_HIP(hipGetLastError());
  return SG_OK;
}

extern "C" size_t sl_linear16_kept_bytes(int act, uint32_t M, uint32_t N) {
  return act > 0 && act < kActs ? (size_t)M * kept_pitch(act, N) : 0;
}

extern "C" size_t sl_linear16_bwd_scratch_bytes(int act, uint32_t M, uint32_t N, uint32_t K) {
  uint64_t most = 0;                         // over every alignment and pitch; what is not asked for only takes away
  for (int i = 0; i < 8; i++) {
    const bool dy_words = i & 1, x_words = i & 2, small_w = i & 4;
    if ((dy_words && N % 8) || (x_words && K % 8)) continue;
    const uint64_t b = plan_bwd(M, N, K, way_of(act, M, N, K, dy_words, x_words, small_w, true, true)).total;
    most = b > most ? b : most;
  }
  return most;
}

extern "C" size_t sl_linear16_bwd_scratch_bytes_for(int act, const void *d_x, int64_t ldx, int64_t ldw, const void *d_dy, int64_t lddy, uint32_t M,
                                                    uint32_t N, uint32_t K, int want_dx, int want_dw) {
  return plan_bwd(M, N, K, way_of(act, M, N, K, rows_of_words(d_dy, lddy, N, SL_BF16), rows_of_words(d_x, ldx, K, SL_BF16), ldw < (1 << 22), want_dx, want_dw)).total;
}

extern "C" int sl_linear16_bwd(int dtype, const void *d_x, int64_t ldx, const void *d_w, int64_t ldw, const void *d_dy, int64_t lddy,
                               const void *d_kept, uint32_t M, uint32_t N, uint32_t K, int act, void *d_dx, int64_t lddx, void *d_dw,
                               int64_t lddw, void *d_db, int db_f32, void *d_scratch, void *stream) {
  if (const int rc = check_sizes("sl_linear16_bwd", dtype, act, M, N, K)) return rc;
  const bool want_w = d_dw || d_db;
  if (!d_scratch || (reinterpret_cast<uintptr_t>(d_scratch) & 15) || (d_dw && lddw < (int64_t)K) ||
      (M && (!d_dy || lddy < (int64_t)N || (act && (!d_kept || (reinterpret_cast<uintptr_t>(d_kept) & 15))) ||
             (d_dx && (!d_w || ldw < (int64_t)K || lddx < (int64_t)K)) || (want_w && (!d_x || ldx < (int64_t)K)))))
    return set_error(SG_ERR_INVALID, "sl_linear16_bwd: operands");
  if (d_db && !d_dw) return set_error(SG_ERR_INVALID, "sl_linear16_bwd: db comes with dW");
  if (((uint64_t)(K + 31) / 32) * (((uint64_t)N + 31) / 32) > kMaxTiles) return set_error(SG_ERR_INVALID, "sl_linear16_bwd: weight of %u x %u", N, K);
  hipStream_t st = (hipStream_t)stream;
  const bool x_words = rows_of_words(d_x, ldx, K, SL_BF16);
  const BwdWay w = way_of(act, M, N, K, rows_of_words(d_dy, lddy, N, SL_BF16), x_words, ldw < (1 << 22), d_dx != nullptr, want_w);
  const BwdPlan p = plan_bwd(M, N, K, w);
  const bool dy_words = w.dy_words, need_dz = w.need_dz, narrow_dx = w.narrow_dx, narrow_dw = w.narrow_dw;
  if (d_dx && !narrow_dx && !w.short_dx && takes_few(M, K, N, lddy, 0) && !few_fits(M, K)) return set_error(SG_ERR_INVALID, "sl_linear16_bwd: too many tiles");
  char *ws = static_cast<char *>(d_scratch);
  const int64_t ldp = (int64_t)up(N, 8);
  const void *dz = need_dz ? ws + p.dz : d_dy;
  const int64_t lddz = need_dz ? ldp : lddy;
  const double bytes_dx = 2.0 * ((double)M * K + (double)N * K + (double)M * N);
  if (need_dz && !(narrow_dx && dy_words)) {
    const uint64_t need = ((uint64_t)M * (ldp / 8) + 255) / 256;
    const dim3 g((uint32_t)(need < 8192 ? need : 8192)), b(256);
    SHD_PROF_FMT(4.0 * M * N + (act ? (double)M * kept_pitch(act, N) : 0), 0, st, "linear16_dz_N%u", N);
    SHD_DISPATCH_16(dtype, hipLaunchKernelGGL((dz_kernel<T>), g, b, 0, st, (const T *)d_dy, lddy, (const char *)d_kept, (T *)(ws + p.dz), ldp, M, N, act));
    SHD_HIP(hipGetLastError());
  }
  if (narrow_dx) {
    NarrowArgs n = {};
    n.g.A = dy_words ? d_dy : dz; n.g.lda = dy_words ? lddy : lddz; n.g.B = d_w; n.g.ldb = ldw; n.g.M = M; n.g.N = K; n.g.K = (uint32_t)ldp; n.g.C = d_dx;
    n.g.ldc = lddx; n.b_rows = N;
    const int fused = dy_words ? act : 0;
    n.kept = static_cast<const char *>(d_kept); n.kept_act = fused; n.dz = fused && need_dz ? ws + p.dz : nullptr; n.lddz = ldp;
    SHD_PROF_FMT(bytes_dx + (fused ? (double)M * kept_pitch(act, N) : 0), 2.0 * M * N * K, st, "linear16_dx_N%u_K%u", N, K);
    SHD_DISPATCH_16(dtype, if (!fused) narrow_launch<T, 0>(n, st);
                    else if (keeps_bits(act)) narrow_launch<T, 3>(n, st);
                    else narrow_launch<T, 2>(n, st));
    SHD_HIP(hipGetLastError());
  } else if (w.few_dx) {
    FewArgs f = {};
    f.g.A = dz; f.g.lda = lddz; f.g.B = d_w; f.g.ldb = ldw; f.g.M = M; f.g.N = K; f.g.K = N; f.g.C = d_dx; f.g.ldc = lddx;
    f.kept = static_cast<const char *>(d_kept); f.kept_act = need_dz ? 0 : act;
    SHD_PROF_FMT(bytes_dx, 2.0 * M * N * K, st, "linear16_dx_N%u_K%u", N, K);
    SHD_DISPATCH_16(dtype, few_launch<T, true>(f, rows_of_words(dz, lddz, N, SL_BF16), st));
    SHD_HIP(hipGetLastError());
  } else if (w.short_dx) {
    GemmArgs a = {};
    a.A = dz; a.lda = lddz; a.B = d_w; a.ldb = ldw; a.M = M; a.N = K; a.K = N; a.C = d_dx; a.ldc = lddx;
    SHD_PROF_FMT(bytes_dx, 2.0 * M * N * K, st, "linear16_dx_N%u_K%u", N, K);
    SHD_DISPATCH_16(dtype, short_launch<T>(a, st));
    SHD_HIP(hipGetLastError());
  } else if (w.need_wt) {
    GemmArgs a = {};
    a.A = dz; a.lda = lddz; a.B = ws + p.wt; a.ldb = ldp; a.M = M; a.N = K; a.C = d_dx; a.ldc = lddx;
    a.K = need_dz ? (uint32_t)ldp : N;       // (pad columns are zero on both sides: whole words)
    SHD_PROF_FMT(bytes_dx, 2.0 * M * N * K, st, "linear16_dx_N%u_K%u", N, K);
    SHD_DISPATCH_16(dtype, hipLaunchKernelGGL((transpose_kernel<T>), dim3((K + 31) / 32 * (uint32_t)((ldp + 31) / 32)), dim3(256), 0, st, (const T *)d_w, ldw, N, K,
                                              (T *)(ws + p.wt), ldp);
                    nt_launch<T>(a, st));
    SHD_HIP(hipGetLastError());
  }
  if (w.few_dw) {
    TnFewArgs f = {};
    TnArgs &a = f.t;
    a.A = dz; a.lda = lddz; a.B = d_x; a.ldb = ldx; a.M = M; a.N = N; a.K = K; a.tiles_n = (N + 31) / 32; a.tiles_k = (K + 31) / 32; a.C = d_dw; a.ldc = lddw;
    f.kept = static_cast<const char *>(d_kept); f.kept_act = need_dz ? 0 : act; f.db = d_db; f.db_f32 = db_f32;
    SHD_PROF_FMT(bytes_dx, 2.0 * M * N * K, st, "linear16_dw_N%u_K%u", N, K);
    SHD_DISPATCH_16(dtype, hipLaunchKernelGGL((tn_few_kernel<T>), dim3(a.tiles_n * a.tiles_k), dim3(512), 0, st, f));
    SHD_HIP(hipGetLastError());
  } else if (want_w) {
    TnNarrowArgs n = {};
    TnArgs &a = n.t;
    a.A = w.bits_dw ? d_dy : dz; a.lda = w.bits_dw ? lddy : lddz; a.B = d_x; a.ldb = ldx; a.M = M; a.N = N; a.K = K; a.tiles_n = (N + BN - 1) / BN;
    a.tiles_k = (K + BM - 1) / BM; a.slices = p.slices; a.per = p.per; a.C = d_dw; a.ldc = lddw;
    a.part = narrow_dw || p.slices > 1 ? reinterpret_cast<float *>(ws + p.part) : nullptr;
    a.part_b = d_db ? reinterpret_cast<float *>(ws + p.part_b) : nullptr;
    n.kept = static_cast<const char *>(d_kept); n.kept_act = act;
    const uint64_t joined = (a.part ? (uint64_t)N * K : 0) + (d_db ? N : 0);
    SHD_PROF_FMT(bytes_dx, 2.0 * M * N * K, st, "linear16_dw_N%u_K%u", N, K);
    SHD_DISPATCH_16(dtype, if (!narrow_dw) tn_launch<T>(a, w.dz_words, x_words, st);
                    else if (w.bits_dw) tn_narrow_launch<T, true>(n, st);
                    else tn_narrow_launch<T, false>(n, st);
                    if (joined) hipLaunchKernelGGL((tn_join_kernel<T>), dim3((uint32_t)((joined + 63) / 64)), dim3(256), 0, st, a.part, a.part_b, p.slices, N, K,
                                                   (T *)d_dw, lddw, d_db, db_f32));
    SHD_HIP(hipGetLastError());
  }
  return SG_OK;
}
