// Softmax class head over many classes (gfx950): z = (x w^T + b) / T for rows x [n, d] and classes w [V, d],
// in pieces of rows that bound what is held of the n x V scores.
//
//   loss:    per-row targets q_j on classes v_j (one label, or a teacher's k best), lse = log sum_v e^z,
//            loss = g T^2 sum_j q_j (log q_j + lse - z_j);  D = g T (s p - q), s = sum_j q_j, p = e^(z - lse);
//            dx = D w, dw = D^T x, db = sum_i D
//   top k:   the k largest z of each row and lse
//
// Rows are taken in pieces so that at most `piece_bytes` of exponentials (256 rows of them at least) live at a time. Per piece:
//   1. scores_kernel   z by MFMA; per row and group of 64 classes the maximum m and sum s of e^(z - m); with
//                      gradients also E = e^(z - m) (bf16 inputs: as fp16 scaled by 2^15, 11 bits, so that
//                      the one rounding that matters is D's own to bf16; a class more than 20 below its group's maximum
//                      has fewer bits, and from 27 on its p, then below 2 10^-12 of that maximum's, counts as 0 in D, not in lse;
//                      fp32 inputs: fp32); top k: also the largest squared norm of w in each group.
//                      Maxima, and scores that are kept, are those before the division by T. A difference is taken before
//                      it is scaled: the maximum's own exponent is exactly 0 and no other is above it, however large
//                      the scores are (z / T - m / T in one fma keeps the rounding of m / T, 2^-24 of it: unbounded).
//   2. target_kernel   (lists) z of the target classes as plain fp32 dot products
//   3. row_kernel      lse from the groups, loss, and the row's coefficients
//   4. dscore_kernel   E -> D in place (fp32: three bf16 planes), bias gradient partials
//   5. grad kernels    dx = D w, dw = D^T x
// The scores are computed once: 6 n d V operations for a step, against 8 n d V where pieces of the classes compute
// them again for the gradient. (8192 x 4096 x 131072: the D pass over 2 GiB takes 0.86 ms, a fourth product 7.0.)
#include "head_gemm.h"

#include <algorithm>
#include <cstring>

namespace ytk {

constexpr int kGroup = 64;                         // classes per (m, s) pair
constexpr float kLog2e = 1.4426950408889634f;

// ------------------------------------------------------------------ scalar types
template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static __device__ __forceinline__ float get(const float* p, long long i) { return p[i]; }
  static __device__ __forceinline__ void put(float* p, long long i, float v) { p[i] = v; }
};
template <>
struct Elem<__bf16> {
  static __device__ __forceinline__ float get(const __bf16* p, long long i) { return (float)p[i]; }
  static __device__ __forceinline__ void put(__bf16* p, long long i, float v) { p[i] = (__bf16)v; }
};

// fp32 -> hi + mid + lo in bf16 (round to nearest each: |rest| <= 2^-27 of the value). Values that would round up to
// infinity are cut instead; infinities and NaN stay in hi alone.
__device__ __forceinline__ void split3(float v, __bf16& h, __bf16& m, __bf16& l) {
  h = (__bf16)v;
  if (!__builtin_isfinite((float)h)) {
    if (__builtin_isfinite(v)) {
      h = __builtin_bit_cast(__bf16, (unsigned short)(__builtin_bit_cast(unsigned, v) >> 16));
    } else {
      m = l = (__bf16)0.0f;
      return;
    }
  }
  const float r = v - (float)h;
  m = (__bf16)r;
  l = (__bf16)(r - (float)m);
}

// ------------------------------------------------------------------ operand layout
// rows x cols of any strides -> kPlanes bf16 planes [rows][pitch/2], columns padded with zeros. Rows whose
// `coef` is zero are written as zeros (ignored rows must not carry an infinity or NaN into 0 * x).
template <typename T, int kPlanes>
__global__ __launch_bounds__(256) void pack_kernel(const T* __restrict__ src, long long rs, long long cs, long long rows,
                                                   int cols, __bf16* __restrict__ dst, long long ld, long long plane,
                                                   const float* __restrict__ coef) {
  __shared__ float tile[64][65];
  __shared__ int live[64];
  const long long r0 = (long long)blockIdx.y * 64;
  const int c0 = blockIdx.x * 64, t = threadIdx.x;
  const bool by_row = cs == 1 || rs != 1;  // consecutive threads along the dimension that is dense in memory
  if (t < 64) live[t] = r0 + t < rows && (!coef || coef[r0 + t] != 0.0f);
  __syncthreads();
  T v[16];  // loads first, then LDS; places outside read element 0
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    const int i = u * 256 + t, r = by_row ? i >> 6 : i & 63, c = by_row ? i & 63 : i >> 6;
    v[u] = src[r0 + r < rows && c0 + c < cols ? (r0 + r) * rs + (c0 + c) * cs : 0];
  }
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    const int i = u * 256 + t, r = by_row ? i >> 6 : i & 63, c = by_row ? i & 63 : i >> 6;
    tile[r][c] = live[r] && c0 + c < cols ? (float)v[u] : 0.0f;
  }
  __syncthreads();
  for (int i = t; i < 512; i += 256) {
    const int r = i >> 3, c = (i & 7) * 8;
    if (r0 + r >= rows || c0 + c >= ld) continue;
    bf16x8 h, m, l;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      __bf16 a, b, e;
      if (kPlanes == 3) {
        split3(tile[r][c + j], a, b, e);
        h[j] = a, m[j] = b, l[j] = e;
      } else {
        h[j] = (__bf16)tile[r][c + j];
      }
    }
    __bf16* o = dst + (r0 + r) * ld + c0 + c;
    *(bf16x8*)o = h;
    if (kPlanes == 3) {
      *(bf16x8*)(o + plane) = m;
      *(bf16x8*)(o + 2 * plane) = l;
    }
  }
}

// ------------------------------------------------------------------ scores
struct ScoreArgs {
  Operand w, x;
  int kw, kx;         // columns of w and x: K of packed ones, d of those read in place
  int V, n;
  int nm, nn;         // tiles
  const void* bias;   // element type of the inputs
  float inv_t;
  float2* stats;      // [groups][n]: m, s
  void* e;            // E [n][ld] (fp16 or fp32) or null
  float* z;           // scores before the division by T [n][ld], or null
  long long ld;
  const void* label;  // [n] or null: a row's label is left out of its group; its score (before the division) goes to zt
  int idx64;
  float* zt;
  float* norms;       // scores that are kept: [parts][groups] largest squared norm of the group's classes, over each part of d
  int parts;
};

__device__ __forceinline__ long long index_at(const void* p, int is64, long long i) {
  return is64 ? ((const long long*)p)[i] : (long long)((const int*)p)[i];
}
__device__ __forceinline__ int class_at(const void* p, int is64, long long i, int V) {
  const long long v = index_at(p, is64, i);
  return v >= 0 && v < V ? (int)v : -1;
}

// lanes l and l + 32 hold rows 8q .. 8q+3 and 8q+4 .. 8q+7 of a 32-row block: exchange halves so that lane l has
// all 8 values of quad pair 2p and lane l + 32 all 8 of 2p + 1 (16-byte stores of 16-bit values)
__device__ __forceinline__ void swap_quads(unsigned& a0, unsigned& a1, unsigned& b0, unsigned& b1) {
  auto p = __builtin_amdgcn_permlane32_swap(a0, b0, false, false);
  auto q = __builtin_amdgcn_permlane32_swap(a1, b1, false, false);
  a0 = p[0], a1 = q[0], b0 = p[1], b1 = q[1];
}

__device__ __forceinline__ uint4 bits4(float a, float b, float c, float d) {
  return make_uint4(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, c),
                    __builtin_bit_cast(unsigned, d));
}
// the 32 turned rows of 128 bytes to rows of `pitch` bytes, as many as there are
__device__ __forceinline__ void store_rows(const Turn& turn, char* to, long long pitch, int rows) {
  const int l = threadIdx.x & 63, c = l & 7;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = k * 8 + (l >> 3);
    const uint4 v = turn.take(r, c);
    if (r < rows) *(uint4*)(to + r * pitch + c * 16) = v;
  }
}

__device__ __forceinline__ unsigned pack_h2(float a, float b) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  h2 v = {(_Float16)a, (_Float16)b};
  return __builtin_bit_cast(unsigned, v);
}
__device__ __forceinline__ unsigned pack_b2(float a, float b) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  b2 v = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(unsigned, v);
}

// e^v. kFine: the product v log2(e) is kept to twice the precision, since its rounding alone is |v| 2^-24 of the
// result (fp32 inputs, whose gradients are wanted to fp32); bf16 inputs round D to 2^-9 anyway.
template <bool kFine>
__device__ __forceinline__ float exp_of(float v) {
  const float t = v * kLog2e;
  if (!kFine) return __builtin_amdgcn_exp2f(t);
  const float r = fmaf(v, kLog2e, -t) + v * 1.925963033e-8f;  // log2(e) - kLog2e
  const float e = __builtin_amdgcn_exp2f(t);
  return e == 0.0f || v == -INFINITY ? 0.0f : fmaf(e * r, 0.6931471805599453f, e);
}

// what a call keeps of its scores: nothing (bf16, fp32 inputs), E (bf16, fp32), the scores
enum { kStatsOnly = 0, kExpHalf = 1, kExpFloat = 2, kScores = 3, kStatsFloat = 4 };

// bf16 inputs with a loss: the exponential is a difference, an fma and an exp2 from the accumulator (fp32: a finer one)
template <int kMode>
constexpr bool kBase2 = kMode == kStatsOnly || kMode == kExpHalf;

// parts of the squared norms of w: a quarter of the K step each, on two tiles of few rows, or the waves of one
template <class C>
constexpr int kNormParts = C::kWN == 1 ? 2 : C::kBK / 16;

template <class C, int kMode>
__global__ __launch_bounds__(C::kThreads) void scores_kernel(ScoreArgs p) {
  static_assert(C::kFM % 2 == 0, "a wave holds whole groups");
  const int wave = threadIdx.x >> 6, l = threadIdx.x & 63, hi = l >> 5;
  gemm_tiles<C, kKC, kKC, kMode == kExpHalf || kMode == kExpFloat || kMode == kScores, kMode == kScores ? kNormParts<C> : 0>(
      p.w, p.x, p.kw, p.kx,
      [&](int j, int& m0, int& n0, int& kt0, int& nkt) {
        const int id = item_of(j, p.nm * p.nn);
        if (id < 0) return false;
        int tm, tn;
        order_of(id, p.nm, p.nn, tm, tn);
        m0 = tm * C::kBM, n0 = tn * C::kBN, kt0 = 0, nkt = (min(p.kw, p.kx) + C::kBK - 1) / C::kBK;
        return true;
      },
      [&](int, int m0, int n0, f32x16(&acc)[C::kFM][C::kFN], const Turn& turn, const float(&sq)[C::kFM]) {
        const int v0 = m0 + (wave / C::kWN) * C::kFM * 32, i0 = n0 + (wave % C::kWN) * C::kFN * 32;
        int label[C::kFN];
#pragma unroll
        for (int j = 0; j < C::kFN; ++j) {
          const int i = i0 + j * 32 + (l & 31);
          label[j] = kMode != kScores && p.label && i < p.n ? class_at(p.label, p.idx64, i, p.V) : -1;
        }
#pragma unroll
        for (int g = 0; g < C::kFM / 2; ++g) {
          const int vg = v0 + g * kGroup;
          if (vg >= p.V) break;
          const int part = n0 / C::kBN * C::kWN + wave % C::kWN;
          if (kMode == kScores && part < p.parts) {
            float q = fmaxf(sq[2 * g] + __shfl_xor(sq[2 * g], 32, 64), sq[2 * g + 1] + __shfl_xor(sq[2 * g + 1], 32, 64));
#pragma unroll
            for (int o = 16; o; o >>= 1) q = fmaxf(q, __shfl_xor(q, o, 64));
            if (l == 0) p.norms[(long long)part * ((p.V + kGroup - 1) / kGroup) + vg / kGroup] = q;
          }
          if (p.bias) {  // (past the last class: the last one's bias, and -inf below)
            float b[2][16];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                const int v = min(vg + h * 32 + 8 * (r >> 2) + 4 * hi + (r & 3), p.V - 1);
                b[h][r] = C::kPlanes == 3 ? ((const float*)p.bias)[v] : (float)((const __bf16*)p.bias)[v];
              }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int j = 0; j < C::kFN; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[2 * g + h][j][r] += b[h][r];
          }
          if (vg + kGroup > p.V) {  // a class past the end is -inf (its operand rows read as zero)
            const int left = p.V - vg - 4 * hi;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int r = 0; r < 16; ++r)
#pragma unroll
                for (int j = 0; j < C::kFN; ++j)
                  if (h * 32 + 8 * (r >> 2) + (r & 3) >= left) acc[2 * g + h][j][r] = -INFINITY;
          }
          const float c = kBase2<kMode> ? p.inv_t * kLog2e : p.inv_t;
#pragma unroll
          for (int j = 0; j < C::kFN; ++j) {
            const int i = i0 + j * 32 + (l & 31);
            // a row's label is taken out of its group's m and s (row_kernel adds it: a confident row's loss is the log of
            // 1 + what the others sum to, which a sum with the label's 1 in it would round away)
            float zl = 0.0f;
            bool mine = false;
            if (kMode != kScores && __any(label[j] >= vg && label[j] < vg + kGroup)) {
              const int at = label[j] - vg - 4 * hi;
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                  if (at == h * 32 + 8 * (r >> 2) + (r & 3)) zl = acc[2 * g + h][j][r], acc[2 * g + h][j][r] = -INFINITY, mine = true;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int r = 0; r < 16; ++r) mx = fmaxf(mx, acc[2 * g + h][j][r]);
            const float m = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float m0 = m == -INFINITY ? 0.0f : m;
            if (kMode != kScores && mine) p.zt[i] = zl;
            if (kMode == kScores)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const f32x16& t = acc[2 * g + h][j];
#pragma unroll
                for (int q = 0; q < 4; ++q) turn.put(l & 31, 2 * q + hi, bits4(t[4 * q], t[4 * q + 1], t[4 * q + 2], t[4 * q + 3]));
                store_rows(turn, (char*)p.z + (i0 + j * 32) * p.ld * 4 + (vg + h * 32) * 4LL, p.ld * 4, p.n - i0 - j * 32);
              }
            float s = 0.0f, e[2][16];
            const float off = kMode == kExpHalf ? 15.0f : 0.0f;  // E is scaled by 2^15
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                if (kBase2<kMode>)
                  e[h][r] = __builtin_amdgcn_exp2f(fmaf(acc[2 * g + h][j][r] - m0, c, off));
                else
                  e[h][r] = exp_of<kMode == kExpFloat || kMode == kStatsFloat>((acc[2 * g + h][j][r] - m0) * c);
                s += e[h][r];
              }
            s += __shfl_xor(s, 32, 64);
            if (kMode == kExpHalf) s *= 1.0f / 32768.0f;
            if (hi == 0 && i < p.n) p.stats[(long long)(vg / kGroup) * p.n + i] = make_float2(m, s);
            if (kMode == kExpFloat)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int q = 0; q < 4; ++q) turn.put(l & 31, 2 * q + hi, bits4(e[h][4 * q], e[h][4 * q + 1], e[h][4 * q + 2], e[h][4 * q + 3]));
                store_rows(turn, (char*)p.e + (i0 + j * 32) * p.ld * 4 + (vg + h * 32) * 4LL, p.ld * 4, p.n - i0 - j * 32);
              }
            if (kMode == kExpHalf) {
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int q = 0; q < 4; q += 2) {
                  unsigned a0 = pack_h2(e[h][4 * q], e[h][4 * q + 1]), a1 = pack_h2(e[h][4 * q + 2], e[h][4 * q + 3]);
                  unsigned b0 = pack_h2(e[h][4 * q + 4], e[h][4 * q + 5]), b1 = pack_h2(e[h][4 * q + 6], e[h][4 * q + 7]);
                  swap_quads(a0, a1, b0, b1);
                  turn.put(l & 31, h * 4 + q + hi, make_uint4(a0, a1, b0, b1));
                }
              store_rows(turn, (char*)p.e + (i0 + j * 32) * p.ld * 2 + vg * 2LL, p.ld * 2, p.n - i0 - j * 32);
            }
          }
        }
      });
}

// ------------------------------------------------------------------ few fp32 rows
// Up to 128 fp32 rows: reading w is the cost, so w goes from memory to registers as it is (the bf16 planes
// would be another 6 bytes written and read per element) and into the fp32 matrix products, 16 x 16 x 4: lane l holds
// row l % 16 and k = l / 16. A lane loads 16 bytes, whose four elements are four products' k (the order of k is free as
// long as both operands agree).
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4u __attribute__((aligned(4)));  // rows of any float alignment

constexpr int kFewRows = 128;

struct FewArgs {
  const float *w, *x, *bias;
  long long wrs, xrs;
  int V, n, d;
  float inv_t;
  float2* stats;
  float* e;        // E or scores [n][ld], or null
  long long ld;
  const void* label;
  int idx64;
  float *zt, *norms;  // as in ScoreArgs, one part
};

// 4 floats from column c; zero past the end
__device__ __forceinline__ f32x4 row4(const float* row, int c, int d) {
  if (c + 4 <= d) return *(const f32x4u*)(row + c);
  f32x4 v;
#pragma unroll
  for (int u = 0; u < 4; ++u) v[u] = c + u < d ? row[c + u] : 0.0f;
  return v;
}

// Sums over the block's four waves through LDS: wave w returns with the sums of row tile i = w (kNT of them take part).
template <int kNT>
__device__ __forceinline__ bool few_sum(f32x4 (&acc)[4][kNT], f32x4 (&out)[4]) {
  __shared__ f32x4 red[4][4][kNT][64];
  const int l = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int i = 0; i < kNT; ++i) red[wave][t][i][l] = acc[t][i];
  __syncthreads();
  if (wave >= kNT) return false;
#pragma unroll
  for (int t = 0; t < 4; ++t) out[t] = (red[0][t][wave][l] + red[1][t][wave][l]) + (red[2][t][wave][l] + red[3][t][wave][l]);
  return true;
}

// A block takes one group of 64 classes against kNT * 16 rows (more rows are further blocks on the same classes), its
// waves a quarter of the features each: 12 waves a CU at 50000 classes, where a group per wave left one per SIMD.
template <int kNT, int kMode>
__global__ __launch_bounds__(256, 2) void scores_few_kernel(FewArgs p) {
  const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = l & 15, g4 = l >> 4, i0 = blockIdx.y * kNT * 16;
  const int vg = blockIdx.x * kGroup;
  const int per = ((p.d + 63) / 64) * 16, d0 = wave * per, d1 = min(d0 + per, p.d);
  const float *w[4], *x[kNT];
#pragma unroll
  for (int t = 0; t < 4; ++t) w[t] = p.w + (long long)min(vg + t * 16 + r16, p.V - 1) * p.wrs;
#pragma unroll
  for (int t = 0; t < kNT; ++t) x[t] = p.x + (long long)min(i0 + t * 16 + r16, p.n - 1) * p.xrs;
  f32x4 acc[4][kNT] = {};
  float sq[4] = {};  // this lane's part of the squared norms of four classes
  constexpr int kU = kNT > 2 ? 2 : 4;  // steps under way
  auto mma = [&](const f32x4 (&a)[4], const f32x4 (&b)[kNT]) {
    if (kMode == kScores)
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) sq[t] = fmaf(a[t][j], a[t][j], sq[t]);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < kNT; ++i) acc[t][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[t][j], b[i][j], acc[t][i], 0, 0, 0);
  };
  int c = d0;
  for (; c + 16 * kU <= d1; c += 16 * kU) {
    f32x4 a[kU][4], b[kU][kNT];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
#pragma unroll
      for (int t = 0; t < 4; ++t) a[u][t] = *(const f32x4u*)(w[t] + c + g4 * 4 + 16 * u);
#pragma unroll
      for (int i = 0; i < kNT; ++i) b[u][i] = *(const f32x4u*)(x[i] + c + g4 * 4 + 16 * u);
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) mma(a[u], b[u]);
  }
  for (; c < d1; c += 16) {
    f32x4 a[4], b[kNT];
#pragma unroll
    for (int t = 0; t < 4; ++t) a[t] = row4(w[t], c + g4 * 4, d1);
#pragma unroll
    for (int i = 0; i < kNT; ++i) b[i] = row4(x[i], c + g4 * 4, d1);
    mma(a, b);
  }
  __shared__ float part[16][64];  // sums of squares of the 64 classes
  if (kMode == kScores)
#pragma unroll
    for (int t = 0; t < 4; ++t) part[wave * 4 + g4][t * 16 + r16] = sq[t];
  f32x4 sum[4];
  const bool mine_too = few_sum<kNT>(acc, sum);
  if (kMode == kScores && blockIdx.y == 0 && wave == 3) {  // (of up to 32 rows this wave has no scores)
    float q = 0.0f;
#pragma unroll
    for (int u = 0; u < 16; ++u) q += part[u][l];
#pragma unroll
    for (int o = 32; o; o >>= 1) q = fmaxf(q, __shfl_xor(q, o, 64));
    if (l == 0) p.norms[blockIdx.x] = q;
  }
  if (!mine_too) return;
  // lane: row l % 16 of the wave's tile, classes vg + 16 t + 4 (l / 16) + r
  const int row = i0 + wave * 16 + r16;
  const int label = kMode != kScores && p.label && row < p.n ? class_at(p.label, p.idx64, row, p.V) : -1;
  float z[4][4], m = -INFINITY, zl = 0.0f;
  bool mine = false;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int v = vg + t * 16 + g4 * 4 + r;
      const float b = p.bias ? p.bias[min(v, p.V - 1)] : 0.0f;
      z[t][r] = v < p.V ? sum[t][r] + b : -INFINITY;
      if (v == label) zl = z[t][r], z[t][r] = -INFINITY, mine = true;  // as in scores_kernel
      m = fmaxf(m, z[t][r]);
    }
  m = fmaxf(m, __shfl_xor(m, 16, 64));
  m = fmaxf(m, __shfl_xor(m, 32, 64));
  const float m0 = m == -INFINITY ? 0.0f : m;
  if (mine) p.zt[row] = zl;
  float s = 0.0f;
  float* o = p.e + (long long)row * p.ld + vg + g4 * 4;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if (kMode == kScores && row < p.n) *(float4*)(o + t * 16) = make_float4(z[t][0], z[t][1], z[t][2], z[t][3]);
#pragma unroll
    for (int r = 0; r < 4; ++r) s += z[t][r] = exp_of<true>((z[t][r] - m0) * p.inv_t);
    if (kMode == kExpFloat && row < p.n) *(float4*)(o + t * 16) = make_float4(z[t][0], z[t][1], z[t][2], z[t][3]);
  }
  s += __shfl_xor(s, 16, 64);
  s += __shfl_xor(s, 32, 64);
  if (g4 == 0 && row < p.n) p.stats[(long long)(vg / kGroup) * p.n + row] = make_float2(m, s);
}

struct FewGradArgs {
  const float *w, *D;   // D [n][ld], zero from V to ld
  long long wrs, ld;
  int V, n, d, per;     // classes per run, a multiple of 64: 16 per wave and step
  float* acc;           // [runs][n][d]
};

// dx = D w: a block takes 64 columns of one run of classes, its waves every fourth 16 classes; lane l holds columns
// 4 (l % 16) .. + 3 of w's row 4 (l / 16) + j, so that one 16-byte load feeds four products (one per column of the four).
template <int kNT>
__global__ __launch_bounds__(256, 2) void dx_few_kernel(FewGradArgs p) {
  const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = l & 15, g4 = l >> 4, i0 = blockIdx.z * kNT * 16;
  const int d0 = blockIdx.x * 64;
  const int v0 = blockIdx.y * p.per, v1 = min(v0 + p.per, p.V), col = d0 + 4 * r16;
  const float* D[kNT];
#pragma unroll
  for (int i = 0; i < kNT; ++i) D[i] = p.D + (long long)min(i0 + i * 16 + r16, p.n - 1) * p.ld + g4 * 4;
  f32x4 acc[4][kNT] = {};
  auto mma = [&](const f32x4 (&a)[4], const f32x4 (&b)[kNT]) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < kNT; ++i) acc[e][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j][e], b[i][j], acc[e][i], 0, 0, 0);
  };
  constexpr int kU = 2;  // steps under way
  int v = v0 + wave * 16;
  if (d0 + 64 <= p.d || (p.d & 3) == 0) {
    // whole pieces: lanes past the last column read it again, and their results are not stored
    const float* w = p.w + (long long)(g4 * 4) * p.wrs + min(col, p.d - 4);
    for (; v + 64 * (kU - 1) + 16 <= v1; v += 64 * kU) {
      f32x4 a[kU][4], b[kU][kNT];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
#pragma unroll
        for (int j = 0; j < 4; ++j) a[u][j] = *(const f32x4u*)(w + (long long)(v + 64 * u + j) * p.wrs);
#pragma unroll
        for (int i = 0; i < kNT; ++i) b[u][i] = *(const f32x4*)(D[i] + v + 64 * u);
      }
#pragma unroll
      for (int u = 0; u < kU; ++u) mma(a[u], b[u]);
    }
  }
  for (; v < v1; v += 64) {
    f32x4 a[4], b[kNT];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = v + g4 * 4 + j;
      // a class past the run: zero, whatever the next row holds
      a[j] = c < v1 ? row4(p.w + (long long)c * p.wrs, col, p.d) : f32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < kNT; ++i) b[i] = *(const f32x4*)(D[i] + v);
    mma(a, b);
  }
  f32x4 sum[4];
  if (!few_sum<kNT>(acc, sum)) return;
  // product e's row m is column d0 + 4 m + e: lane holds m = 4 (l / 16) + r, so four e make four columns in a row
  const int row = i0 + wave * 16 + r16;
  if (row >= p.n) return;
  float* o = p.acc + ((long long)blockIdx.y * p.n + row) * p.d;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int c = d0 + 16 * g4 + 4 * r;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < p.d) o[c + e] = sum[e][r];
  }
}

struct FewOuterArgs {
  const float *x, *D, *coef;  // D [n][ld]; rows of x without a gradient (coef 0) count as zero
  long long xrs, ld;
  int V, n, d, per;           // classes per block, a multiple of 64
  float* dw;                  // [V][d]
};

// dw = D^T x of at most 16 kK rows: a wave keeps its 64 columns of x in registers and walks over classes, 16 at a time;
// the block's waves are side by side, so that it writes 1 KB pieces of 16 rows (256-byte pieces: 3.0 TB/s of dw).
template <int kK>
__global__ __launch_bounds__(256) void dw_few_kernel(FewOuterArgs p) {
  const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = l & 15, g4 = l >> 4;
  const int d0 = (blockIdx.x * 4 + wave) * 64, col = d0 + 4 * r16;
  const int v0 = blockIdx.y * p.per, v1 = min(v0 + p.per, p.V), steps = (p.n + 3) / 4;
  if (d0 >= p.d) return;
  f32x4 a[4 * kK];
  const float* D[4 * kK];
#pragma unroll
  for (int k = 0; k < 4 * kK; ++k) {
    const int i = k * 4 + g4;
    a[k] = i < p.n && p.coef[min(i, p.n - 1)] != 0.0f ? row4(p.x + (long long)i * p.xrs, col, p.d) : f32x4{0, 0, 0, 0};
    D[k] = p.D + (long long)min(i, p.n - 1) * p.ld + r16;
  }
  const bool vec = (p.d & 3) == 0;
  for (int v = v0; v < v1; v += 16) {
    float b[4 * kK];
#pragma unroll
    for (int k = 0; k < 4 * kK; ++k)
      if (k < steps) b[k] = D[k][v];  // (rows past n: the last one's, against zeros of x)
    f32x4 acc[4] = {};
#pragma unroll
    for (int k = 0; k < 4 * kK; ++k)
      if (k < steps)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[k][e], b[k], acc[e], 0, 0, 0);
    // lane: class v + l % 16, columns d0 + 16 (l / 16) + 4 r + e
    if (v + r16 >= v1) continue;
    float* o = p.dw + (long long)(v + r16) * p.d;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int c = d0 + 16 * g4 + 4 * r;
      if (vec && c + 4 <= p.d) {
        *(float4*)(o + c) = make_float4(acc[0][r], acc[1][r], acc[2][r], acc[3][r]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < p.d) o[c + e] = acc[e][r];
      }
    }
  }
}

// ------------------------------------------------------------------ targets
// Scores (before the division by T) of each row's target classes by plain fp32 dot products.
struct TargetArgs {
  const void *x, *w, *bias;
  long long xrs, xcs, wrs, wcs;
  const void* idx;     // [n][k], int64 or int32
  int idx64, k, n, d, V, vec;
  float* zt;           // [n][k]
};

// 16 bytes of a row as fp32
__device__ __forceinline__ void unpack16(const uint4& u, float (&v)[4]) {
  v[0] = __builtin_bit_cast(float, u.x), v[1] = __builtin_bit_cast(float, u.y);
  v[2] = __builtin_bit_cast(float, u.z), v[3] = __builtin_bit_cast(float, u.w);
}
__device__ __forceinline__ void unpack16(const uint4& u, float (&v)[8]) {
  const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __builtin_bit_cast(float, w[i] << 16);
    v[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xffff0000u);
  }
}

// a wave's dot products of one x row with kW w rows, summed in A (fp32, or fp64 of exact or fp64 products).
// `vec`: rows of whole, aligned 16-byte pieces; otherwise element by element with any stride.
template <typename T, typename A, int kW, int kU>
__device__ __forceinline__ void row_dots(const T* x, long long xcs, const T* const (&w)[kW], long long wcs, int d, bool vec, A (&s)[kW]) {
  const int l = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < kW; ++i) s[i] = 0;
  constexpr int kE = 16 / sizeof(T);
  auto add = [](A& s, float a, float b) {
    if (sizeof(A) == 8 && sizeof(T) == 2)
      s += (A)(a * b);  // exact: 8 x 8 bits
    else
      s = fma((A)a, (A)b, s);
  };
  if (vec) {
    for (int c0 = l * kE; c0 < d; c0 += 64 * kE * kU) {
      uint4 a[kU], b[kU][kW];  // kU (1 + kW) loads under way; pieces past the end are read again from the start and dropped
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int c = c0 + u * 64 * kE < d ? c0 + u * 64 * kE : 0;
        a[u] = *(const uint4*)(x + c);
#pragma unroll
        for (int i = 0; i < kW; ++i) b[u][i] = *(const uint4*)(w[i] + c);
      }
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (c0 + u * 64 * kE >= d) break;
        float f[kE];
        unpack16(a[u], f);
#pragma unroll
        for (int i = 0; i < kW; ++i) {
          float g[kE];
          unpack16(b[u][i], g);
#pragma unroll
          for (int e = 0; e < kE; ++e) add(s[i], f[e], g[e]);
        }
      }
    }
  } else {  // in the same order, so that the result does not depend on the strides
    for (int c = l * kE; c < d; c += 64 * kE)
      for (int e = 0; e < min(kE, d - c); ++e) {
        const float a = Elem<T>::get(x, (c + e) * xcs);
#pragma unroll
        for (int i = 0; i < kW; ++i) add(s[i], a, Elem<T>::get(w[i], (c + e) * wcs));
      }
  }
#pragma unroll
  for (int i = 0; i < kW; ++i)
#pragma unroll
    for (int o = 32; o; o >>= 1) s[i] += __shfl_xor(s[i], o, 64);
}

// kW targets of one row per wave: their loads are in flight together
template <typename T, int kW>
__global__ __launch_bounds__(256) void target_kernel(TargetArgs p) {
  const int l = threadIdx.x & 63, runs = (p.k + kW - 1) / kW;
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= (long long)p.n * runs) return;
  const long long row = item / runs, first = row * p.k + item % runs * kW;
  const int m = min(kW, (int)((row + 1) * p.k - first));
  const T* w[kW];
  long long v[kW];
#pragma unroll
  for (int i = 0; i < kW; ++i) {
    v[i] = i < m ? index_at(p.idx, p.idx64, first + i) : -1;
    if (v[i] >= p.V) v[i] = -1;
    w[i] = (const T*)p.w + (v[i] < 0 ? 0 : v[i]) * p.wrs;  // entries without a class read class 0
  }
  float s[kW];
  row_dots<T, float, kW, kW == 1 ? 4 : 2>((const T*)p.x + row * p.xrs, p.xcs, w, p.wcs, p.d, p.vec, s);
  if (l == 0) {
#pragma unroll
    for (int i = 0; i < kW; ++i)
      if (i < m) p.zt[first + i] = v[i] < 0 ? 0.0f : s[i] + (p.bias ? Elem<T>::get((const T*)p.bias, v[i]) : 0.0f);
  }
}

// ------------------------------------------------------------------ rows
struct RowArgs {
  const float2* stats;  // [groups][n]
  int groups, n, base;  // base: one more class with score 0, index V
  int V, k, mode;       // mode 0: label, 1: teacher list renormalised, 2: teacher list with its normaliser
  const void* idx;
  int idx64;
  long long ignore;
  const float *tl, *tlse, *weight, *zt;
  float temp, inv_t;
  float *lse, *loss;    // outputs
  float* coef;          // [n] g T s  (0: the row has no gradient)
  float2* norm;         // [n] maximum (before the division by T) and 1 / sum: p = e^((z - max) / T) / sum, without the rounding of lse
  float* q;             // [n][k] g T q_j; of a label g (1 - p), all of its D
  int rb;               // rows per block (a power of two, <= 16)
  float* norms;         // [parts][groups] or null: their sums go to the first, the largest sum is that of norm_max [4]
  float* norm_max;
  int parts;
};

// Scores and maxima are those before the division by T. kB2: bf16 inputs, whose exponentials are exp2 alone
template <bool kB2>
__global__ __launch_bounds__(256) void row_kernel(RowArgs p) {
  __shared__ float sm[256], ss[256], sl[16], sg[16];  // sl, sg: loss and -D of a label
  const float unit = kB2 ? p.inv_t * kLog2e : p.inv_t;
  auto ex = [&](float v) { return kB2 ? __builtin_amdgcn_exp2f(v * unit) : exp_of<true>(v * unit); };  // e^(v / T)
  const int t = threadIdx.x, rl = t & (p.rb - 1), strip = t / p.rb, strips = 256 / p.rb;
  const long long row = (long long)blockIdx.x * p.rb + rl;
  if (p.norms && blockIdx.x == gridDim.x - 1) {  // a block of its own, behind those of the rows
    float q = 0.0f;
#pragma unroll 8
    for (int g = t; g < p.groups; g += 256) {
      float sum = p.norms[g];
      for (int u = 1; u < p.parts; ++u) sum += p.norms[(long long)u * p.groups + g];
      if (p.parts > 1) p.norms[g] = sum;
      q = fmaxf(q, sum);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) q = fmaxf(q, __shfl_xor(q, o, 64));
    if ((t & 63) == 0) p.norm_max[t >> 6] = q;
    return;
  }
  // running maximum and sum over this thread's groups
  float m = -INFINITY, s = 0.0f;
  if (row < p.n) {
    // four groups at a time: their loads are in flight together and share one rescaling
    for (int g = strip; g < p.groups; g += 4 * strips) {
      float2 a[4];
      float nm = m;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int gu = g + u * strips;
        a[u] = gu < p.groups ? p.stats[(long long)gu * p.n + row] : make_float2(-INFINITY, 0.0f);
        nm = fmaxf(nm, a[u].x);
      }
      const float n0 = nm == -INFINITY ? 0.0f : nm;  // (groups of NaN scores: the maximum passed over them, s is NaN)
      s *= ex(m - n0);
#pragma unroll
      for (int u = 0; u < 4; ++u) s += a[u].y * (a[u].x == -INFINITY ? 1.0f : ex(a[u].x - n0));
      m = nm;
    }
    if (p.base && strip == 0 && !(p.mode == 0 && p.loss && index_at(p.idx, p.idx64, row) == p.V)) {
      const float nm = fmaxf(m, 0.0f);
      s = (m == -INFINITY ? 0.0f : s * ex(m - nm)) + ex(-nm);
      m = nm;
    }
  }
  sm[t] = m;
  ss[t] = s;
  __syncthreads();
  for (int h = 128; h >= p.rb; h >>= 1) {
    if (t < h) {
      const float m1 = sm[t], m2 = sm[t + h], nm = fmaxf(m1, m2), n0 = nm == -INFINITY ? 0.0f : nm;
      ss[t] = ss[t] * ex(m1 - n0) + ss[t + h] * ex(m2 - n0);
      sm[t] = nm;
    }
    __syncthreads();
  }
  if (t < p.rb && row < p.n) {
    const float m = sm[t];
    float s = ss[t];
    const long long v = p.mode == 0 && p.loss ? index_at(p.idx, p.idx64, row) : -1;
    if (v >= 0 && v < p.V + p.base) {
      // the label's own term: rel = z - m. loss = log(1 + s e^-rel), D = -s / (s + e^rel) without cancellation
      const float z = v < p.V ? p.zt[row] : 0.0f, rel = z - m, nat = rel * p.inv_t;
      if (m == -INFINITY) {  // nothing else
        sl[t] = s;  // 0, or NaN
        sg[t] = s;
        p.lse[row] = z * p.inv_t + s;
        if (p.norm) p.norm[row] = make_float2(z, 1.0f);
      } else if (nat > 60.0f) {  // e^rel does not fit: relative to the label
        const float w = s * ex(-rel);
        sl[t] = log1pf(w);
        sg[t] = w / (1.0f + w);
        p.lse[row] = z * p.inv_t + sl[t];
        if (p.norm) p.norm[row] = make_float2(z, 1.0f / (1.0f + w));
      } else {
        const float e = ex(rel), all = s + e;
        sl[t] = nat > 0.0f ? log1pf(s * ex(-rel)) : logf(all) - nat;
        sg[t] = s / all;
        p.lse[row] = m * p.inv_t + logf(all);
        if (p.norm) p.norm[row] = make_float2(m, 1.0f / all);
      }
    } else {
      if (p.norm) p.norm[row] = make_float2(m, 1.0f / s);
      ss[t] = logf(s);
      p.lse[row] = m * p.inv_t + ss[t];
    }
  }
  __syncthreads();
  if (!p.loss) return;
  // targets: one wave per row in turn
  const int wave = t >> 6, l = t & 63;
  for (int r = wave; r < p.rb; r += 4) {
    const long long i = (long long)blockIdx.x * p.rb + r;
    if (i >= p.n) break;
    const float mx_row = sm[r], log_s = ss[r], g = p.weight ? p.weight[i] : 1.0f;
    float norm = 0.0f, log_e = 0.0f, inv_e = 1.0f;  // q = e^(t - norm) inv_e
    if (p.mode == 1) {  // renormalise the list: log sum e^(t/T) over its entries
      float mx = -INFINITY;
      for (int j = l; j < p.k; j += 64)
        if (index_at(p.idx, p.idx64, i * p.k + j) >= 0) mx = fmaxf(mx, p.tl[i * p.k + j] / p.temp);
#pragma unroll
      for (int o = 32; o; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
      if (mx == -INFINITY) mx = 0.0f;
      float e = 0.0f;
      for (int j = l; j < p.k; j += 64)
        if (index_at(p.idx, p.idx64, i * p.k + j) >= 0) e += expf(p.tl[i * p.k + j] / p.temp - mx);
      e = wave_sumf(e);
      norm = mx;
      if (e != 0.0f) log_e = logf(e), inv_e = 1.0f / e;  // otherwise nothing but -inf: every q_j is 0
    } else if (p.mode == 2) {
      norm = p.tlse[i];
    }
    float sq = 0.0f, ls = 0.0f;
    for (int j = l; j < p.k; j += 64) {
      const long long v = index_at(p.idx, p.idx64, i * p.k + j);
      float q = 0.0f, term = 0.0f;
      const bool skip = p.mode == 0 ? v == p.ignore : v < 0;
      if (!skip) {
        if (v < 0 || v >= p.V + p.base) {
          term = NAN;  // a class that does not exist
        } else {
          const float t = p.mode == 0 ? 0.0f : p.tl[i * p.k + j] / p.temp - norm, lq = t - log_e;
          q = p.mode == 0 ? 1.0f : expf(t) * inv_e;
          if (p.mode == 0) {
            term = sl[r];
          } else if (q > 0.0f || q != q) {
            // log q + lse - z, the maximum's part first: it cancels where z is near the maximum
            const float up = mx_row - p.zt[i * p.k + j];
            term = q * (lq + (up * p.inv_t + log_s));
          }
        }
      }
      if (p.q) p.q[i * p.k + j] = (p.mode == 0 ? q * sg[r] : q) * g * p.temp;
      sq += q;
      ls += term;
    }
    sq = wave_sumf(sq);
    ls = wave_sumf(ls);
    if (l == 0) {
      const float c = g == 0.0f ? 0.0f : g * p.temp * sq;  // (a row without weight: whatever its list holds)
      p.loss[i] = (g == 0.0f || (sq == 0.0f && ls == ls)) ? 0.0f : g * p.temp * p.temp * ls;
      if (p.coef) p.coef[i] = c;
    }
  }
}

// ------------------------------------------------------------------ score gradient
struct DArgs {
  const float2* stats;
  const float2* norm;
  const float *coef, *q, *zt;
  const void* idx;
  int idx64, n, V, k;
  void* e;              // E in; bf16 inputs: D out in place
  __bf16* d;            // fp32 inputs: D planes
  long long ld, plane;
  float* part;          // [row blocks][ld] bias gradient partials, or null
  float unit;           // 1 / T, bf16 inputs: in log2 units
  int rw;               // rows per wave
  int label;            // targets are labels: q is all of D there
  int keep32;           // fp32 inputs: D also in fp32, in place of E
  char* x;              // packed x of these rows, or null: rows without a gradient are cleared in it before they meet D
  long long xpitch, xplane;
  int planes;
};

constexpr int kDRows = 16;    // rows per wave at most, four waves per block
constexpr int kDCols = 512;   // columns per block: one wave = one row's 512 columns, 8 per lane

template <bool kF32>
__global__ __launch_bounds__(256) void dscore_kernel(DArgs p) {
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  constexpr int kB = kF32 ? 2 : 4;  // rows at once: their loads are in flight together
  const int wave = threadIdx.x >> 6, l = threadIdx.x & 63;
  const int c0 = blockIdx.x * kDCols, c = c0 + l * 8;
  const long long r0 = ((long long)blockIdx.y * 4 + wave) * p.rw;
  const int rows = (int)min((long long)p.rw, p.n - r0);  // may be negative
  float db[8] = {};
  const bool live = c < p.ld;
  const long long cl = live ? c : 0;  // lanes past the end read column 0 and write nothing
  const float2* st = p.stats + cl / kGroup * p.n;
  for (int rb = 0; rb < rows; rb += kB) {
    float d[kB][8], m[kB], cw[kB];
    float2 nr[kB];
    long long v[kB];
#pragma unroll
    for (int b = 0; b < kB; ++b) {
      const long long i = min(r0 + rb + b, (long long)p.n - 1);
      cw[b] = rb + b < rows ? p.coef[i] : 0.0f;
      nr[b] = p.norm[i];
      m[b] = st[i].x;
      v[b] = l < p.k ? index_at(p.idx, p.idx64, i * p.k + l) : -1;
      if (kF32) {
        const float4 *e = (const float4*)((const float*)p.e + i * p.ld + cl), x = e[0], y = e[1];
        d[b][0] = x.x, d[b][1] = x.y, d[b][2] = x.z, d[b][3] = x.w;
        d[b][4] = y.x, d[b][5] = y.y, d[b][6] = y.z, d[b][7] = y.w;
      } else {
        const h8 x = *(const h8*)((const _Float16*)p.e + i * p.ld + cl);
#pragma unroll
        for (int j = 0; j < 8; ++j) d[b][j] = (float)x[j];
      }
    }
#pragma unroll
    for (int b = 0; b < kB; ++b) {
      if (rb + b >= rows) break;
      const long long i = r0 + rb + b;
      const float co = cw[b] * nr[b].y;
      if (cw[b] != 0.0f) {
        // (a group that has only -inf, or nothing but the label: E is 0, and m = -inf makes f 0 too. With 0 for its m, f would be
        // e^-max, infinite for a row of low scores, and 0 f NaN)
        const float mg = m[b] - nr[b].x;
        const float f = co * (kF32 ? exp_of<true>(mg * p.unit) : __builtin_amdgcn_exp2f(fmaf(mg, p.unit, -15.0f)));
#pragma unroll
        for (int j = 0; j < 8; ++j) d[b][j] *= f;
        // target classes: every entry of the list on that class is subtracted from p. bf16 lists take p from the fp32
        // score first (E's 11 bits would show where p is near q); fp32 E agrees with the row's sum to the last bit,
        // which the score summed in another order does not, and a label's E is 0
#pragma unroll
        for (int pass = 0; pass < 2; ++pass) {
          if (pass == 0 && (kF32 || p.label)) continue;
          for (int j0 = 0; j0 < p.k; j0 += 64) {
            const long long vv = j0 == 0 ? v[b] : j0 + l < p.k ? index_at(p.idx, p.idx64, i * p.k + j0 + l) : -1;
            const int at = vv >= c0 && vv < c0 + kDCols && vv < p.V ? (int)(vv - c0) : -1;
            for (unsigned long long h = __ballot(at >= 0); h; h &= h - 1) {
              const int bit = __builtin_ctzll(h), vb = __builtin_amdgcn_readlane(at, bit);
              const long long e = i * p.k + j0 + bit;
              const float x = pass != 0 ? p.q[e] : co * __builtin_amdgcn_exp2f((p.zt[e] - nr[b].x) * p.unit);
#pragma unroll
              for (int u = 0; u < 8; ++u)
                if (vb == l * 8 + u) d[b][u] = pass == 0 ? x : d[b][u] - x;
            }
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) d[b][j] = 0.0f;
        // 0 * x must be 0 whatever this x holds
        if (blockIdx.x == 0 && p.x)
          for (int q = 0; q < p.planes; ++q)
            for (long long u = l * 16; u < p.xpitch; u += 1024)
              *(uint4*)(p.x + q * p.xplane + i * p.xpitch + u) = make_uint4(0, 0, 0, 0);
      }
      if (live) {
#pragma unroll
        for (int j = 0; j < 8; ++j) db[j] += d[b][j];
        if (kF32) {
          bf16x8 h, mi, lo;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            __bf16 x, y, z;
            split3(d[b][j], x, y, z);
            h[j] = x, mi[j] = y, lo[j] = z;
          }
          if (p.keep32) {
            float4* e = (float4*)((float*)p.e + i * p.ld + c);
            e[0] = make_float4(d[b][0], d[b][1], d[b][2], d[b][3]);
            e[1] = make_float4(d[b][4], d[b][5], d[b][6], d[b][7]);
          }
          if (!p.d) continue;
          __bf16* o = p.d + i * p.ld + c;
          *(bf16x8*)o = h;
          *(bf16x8*)(o + p.plane) = mi;
          *(bf16x8*)(o + 2 * p.plane) = lo;
        } else {
          *(uint4*)((unsigned short*)p.e + i * p.ld + c) =
              make_uint4(pack_b2(d[b][0], d[b][1]), pack_b2(d[b][2], d[b][3]), pack_b2(d[b][4], d[b][5]), pack_b2(d[b][6], d[b][7]));
        }
      }
    }
  }
  if (!p.part) return;
  __shared__ float sh[4][kDCols];
#pragma unroll
  for (int j = 0; j < 8; ++j) sh[wave][l * 8 + j] = db[j];
  __syncthreads();
  for (int u = threadIdx.x; u < kDCols; u += 256) {
    const int col = blockIdx.x * kDCols + u;
    if (col < p.ld) p.part[(long long)blockIdx.y * p.ld + col] = (sh[0][u] + sh[1][u]) + (sh[2][u] + sh[3][u]);
  }
}

// bias gradient: 64 columns per block, the partials in 16 strips, each in order; `acc` carries pieces of rows (first:
// overwritten)
template <typename T>
__global__ __launch_bounds__(1024) void db_kernel(const float* __restrict__ part, int nb, long long ld, int V,
                                                  float* __restrict__ acc, int first, T* __restrict__ out) {
  __shared__ float sh[16][64];
  const int l = threadIdx.x & 63, strip = threadIdx.x >> 6, v = blockIdx.x * 64 + l;
  float s = 0.0f;
#pragma unroll 8
  for (int b = strip; b < nb; b += 16) s += part[b * ld + v];  // (ld is a multiple of 64)
  sh[strip][l] = s;
  __syncthreads();
  if (strip || v >= V) return;
  s = first ? 0.0f : acc[v];
#pragma unroll
  for (int b = 0; b < 16; ++b) s += sh[b][l];
  if (out)
    Elem<T>::put(out, v, s);
  else
    acc[v] = s;
}

// ------------------------------------------------------------------ gradient products
struct GradArgs {
  Operand a, b;
  long long ka, kb;        // extent of K in each operand's memory
  int K;                   // products run over K (at most ka, kb)
  int M, N, nm, nn;        // result [N][M], M contiguous
  // tiles taken whole; each of the rest is cut along K into ts runs of `per` (a multiple of 64). With runs, whole is
  // a multiple of the grid and the runs are at most one per block.
  int whole, ts, per, grid;
  void* out;               // T [N][ldo]
  long long ldo;
  float* part;             // the runs' sums, a tile each: [tile - whole][ts][kBN][kBM]
  float* acc;              // pieces of rows: [N][M] fp32
  int mode;                // 0: out = C  1: acc = C  2: acc += C  3: out = acc + C
};

// Item of the block's j-th turn: whole tiles first, in full rounds of the grid, then one round of runs.
__device__ __forceinline__ bool grad_item(const GradArgs& p, int j, int& id, int& run) {
  const int rounds = p.ts > 1 ? p.whole / (int)gridDim.x : 1 << 30;
  run = -1;
  if (j < rounds) {
    id = item_of(j, p.whole);
    return id >= 0;
  }
  const int item = j == rounds ? item_of(0, (p.nm * p.nn - p.whole) * p.ts) : -1;
  if (item < 0) return false;
  id = p.whole + item / p.ts;
  run = item % p.ts;
  return true;
}

template <class C, int kLA, int kLB, typename T>
__global__ __launch_bounds__(C::kThreads) void grad_kernel(GradArgs p) {
  const int wave = threadIdx.x >> 6, l = threadIdx.x & 63, hi = l >> 5;
  gemm_tiles<C, kLA, kLB, false>(
      p.a, p.b, p.ka, p.kb,
      [&](int j, int& m0, int& n0, int& kt0, int& nkt) {
        int id, run, tm, tn;
        if (!grad_item(p, j, id, run)) return false;
        order_of(id, p.nm, p.nn, tm, tn);
        const int k0 = run < 0 ? 0 : run * p.per, k1 = run < 0 ? p.K : min(k0 + p.per, p.K);
        m0 = tm * C::kBM, n0 = tn * C::kBN;
        kt0 = k0 / C::kBK, nkt = (k1 - k0 + C::kBK - 1) / C::kBK;
        return true;
      },
      [&](int j, int m0, int n0, f32x16(&acc)[C::kFM][C::kFN], const Turn&, const float(&)[C::kFM]) {
        int id, run;
        grad_item(p, j, id, run);
        const int mw = m0 + (wave / C::kWN) * C::kFM * 32, nw = n0 + (wave % C::kWN) * C::kFN * 32;
        if (run >= 0) {
          float* t = p.part + ((long long)(id - p.whole) * p.ts + run) * (C::kBM * C::kBN);
#pragma unroll
          for (int j = 0; j < C::kFN; ++j)
#pragma unroll
            for (int i = 0; i < C::kFM; ++i)
#pragma unroll
              for (int q = 0; q < 4; ++q)
                *(float4*)(t + (nw - n0 + j * 32 + (l & 31)) * C::kBM + mw - m0 + i * 32 + 8 * q + 4 * hi) =
                    make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
          return;
        }
        const bool vec = (p.ldo & 7) == 0 && ((uintptr_t)p.out & 15) == 0, avec = (p.M & 3) == 0;
        if (sizeof(T) == 2 && p.mode == 0 && vec && (p.M & 7) == 0) {  // 16-byte stores: a lane's 8 values of m
#pragma unroll
          for (int j = 0; j < C::kFN; ++j) {
            const int n = nw + j * 32 + (l & 31);
#pragma unroll
            for (int i = 0; i < C::kFM; ++i)
#pragma unroll
              for (int q = 0; q < 4; q += 2) {
                const f32x16& t = acc[i][j];
                unsigned a0 = pack_b2(t[4 * q], t[4 * q + 1]), a1 = pack_b2(t[4 * q + 2], t[4 * q + 3]);
                unsigned b0 = pack_b2(t[4 * q + 4], t[4 * q + 5]), b1 = pack_b2(t[4 * q + 6], t[4 * q + 7]);
                swap_quads(a0, a1, b0, b1);
                const int m = mw + i * 32 + 8 * q + 8 * hi;
                if (n < p.N && m < p.M) *(uint4*)((T*)p.out + (long long)n * p.ldo + m) = make_uint4(a0, a1, b0, b1);
              }
          }
          return;
        }
#pragma unroll
        for (int j = 0; j < C::kFN; ++j) {
          const int n = nw + j * 32 + (l & 31);
          if (n >= p.N) continue;
#pragma unroll
          for (int i = 0; i < C::kFM; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int m = mw + i * 32 + 8 * q + 4 * hi;
              if (m >= p.M) continue;
              float v[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
              if (p.mode) {
                float* a = p.acc + (long long)n * p.M + m;
                if (avec) {
                  if (p.mode != 1) {
                    const float4 o = *(const float4*)a;
                    v[0] += o.x, v[1] += o.y, v[2] += o.z, v[3] += o.w;
                  }
                  if (p.mode != 3) *(float4*)a = make_float4(v[0], v[1], v[2], v[3]);
                } else {
                  for (int u = 0; u < 4; ++u)
                    if (m + u < p.M) {
                      if (p.mode != 1) v[u] += a[u];
                      if (p.mode != 3) a[u] = v[u];
                    }
                }
              }
              if (p.mode == 0 || p.mode == 3) {
                T* o = (T*)p.out + (long long)n * p.ldo + m;
                if (vec && m + 4 <= p.M) {
                  if (sizeof(T) == 4)
                    *(float4*)o = make_float4(v[0], v[1], v[2], v[3]);
                  else
                    *(uint2*)o = make_uint2(pack_b2(v[0], v[1]), pack_b2(v[2], v[3]));
                } else {
                  for (int u = 0; u < 4; ++u)
                    if (m + u < p.M) Elem<T>::put(o, u, v[u]);
                }
              }
            }
        }
      });
}

// out tile = sum of its runs, in order: 32 result rows of one tile per block
template <int BM, int BN, typename T>
__global__ __launch_bounds__(256) void run_sum_kernel(GradArgs p) {
  int tm, tn;
  order_of(p.whole + (int)blockIdx.x, p.nm, p.nn, tm, tn);
  constexpr int kPer = BM / 4;  // threads per row
  const int m = tm * BM + (int)(threadIdx.x % kPer) * 4;
  if (m >= p.M) return;
  for (int r = threadIdx.x / kPer; r < 32; r += 256 / kPer) {
    const int nl = blockIdx.y * 32 + r, n = tn * BN + nl;
    if (n >= p.N) return;
    const float* t = p.part + (long long)blockIdx.x * p.ts * (BM * BN) + nl * BM + (m - tm * BM);
    float4 s = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int k = 0; k < p.ts; ++k) {
      const float4 v = *(const float4*)(t + (long long)k * (BM * BN));
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    const float v[4] = {s.x, s.y, s.z, s.w};
    T* o = (T*)p.out + (long long)n * p.ldo + m;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (m + u < p.M) Elem<T>::put(o, u, v[u]);
  }
}

// out = sum over splits, in split order
template <typename T>
__global__ __launch_bounds__(256) void split_sum_kernel(const float* __restrict__ acc, int splits, long long rows, int cols,
                                                        T* __restrict__ out, long long ldo) {
  const long long total = rows * cols;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    float s = 0.0f;
    for (int k = 0; k < splits; ++k) s += acc[k * total + i];
    Elem<T>::put(out, i / cols * ldo + i % cols, s);
  }
}

// ------------------------------------------------------------------ top k
// One block per row. Scores are in z [n][ld], group maxima in stats. With kc = k + kSpare candidates:
//   1. a threshold tau that at least kc and (ties aside) few more group maxima reach, found bit by bit with the
//      maxima in registers: every such group holds a score >= tau, so the kc best of all scores are
//      among the scores >= tau, and those are in these groups. Where ties leave more groups, the first kc by
//      (maximum, lower group) do: each of them holds a score that beats everything outside.
//   2. the scores >= tau of those groups, as 64-bit keys (score order, then lower class)
//   3. the kc largest keys
//   4. their scores again as 64-bit sums, and the k largest of them in order
//   5. A class that is no candidate has an fp32 score of at most the candidates' least, `cut`. Where the k-th 64-bit score is
//      above cut by more than fp32 scores are off, no such class belongs to the k best, and the row is done. Otherwise (scores that
//      lie closer together than fp32 tells apart: a common offset, sums that cancel, equal classes) every class whose
//      fp32 score reaches the k-th less that error is scored in 64 bits too, in turns of up to 768 that are merged with
//      the k best so far. So the classes and their order are those of the 64-bit scores for every row.
//      How far an fp32 score may be off: Slack.
constexpr int kSpare = 8, kSlack = 24;
constexpr int kTopMax = 256;       // k at most
constexpr int kTopHold = 8;        // group maxima per thread
constexpr int kTopList = 2048;     // keys held in LDS; where more reach tau (ties), they are read again from memory
constexpr int kTurnList = 768, kTurnAdd = 512;  // classes scored in 64 bits per turn, and added per step at most

struct TopArgs {
  const float2* stats;
  const float* z;
  long long ld;
  int n, V, d, groups, kc, k, vec;
  const void *x, *w, *bias;
  long long xrs, xcs, wrs, wcs;
  double inv_t;
  float* values;
  long long* classes;
  const float *norms, *norm_max;
  float slack;          // Slack::c
};

// What a 32-bit score (before the division by T) of a row with squared norm xx may be off against classes of squared norm <= ww,
// where only scores of magnitude <= z matter: c 2^-24 of sum |x||w| <= |x| |w|, and the rounding of the bias's sum.
// The fp32 matrix product of 4 rounds after every product (c = d), the bf16 one of 16 after every four (against exact sums: at most
// 5.3 units per instruction; c = d / 2 counts 8). Joined accumulators, cut planes and dropped plane pairs take less than 64 units.
// ww is summed in fp32 (fp32 inputs: of the largest planes, at most 2^-8 off): 1.02 + d 2^-23 times it, and squares that underflow
// are below 2^-125 each. The roots are fp32's (a 64-bit root in the way of every row's answer costs 0.3 us), so xx is at least
// 2^-120, and where it has no fp32 value the bound is infinite.
__device__ __forceinline__ float uniform(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}
__device__ __forceinline__ unsigned long long uniform(unsigned long long v) {
  return (unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)v);
}
struct Slack {
  float x, c, d;
  __device__ __forceinline__ Slack(double xx, float c, int d) : x(uniform(__builtin_amdgcn_sqrtf(fmaxf((float)xx, 0x1p-120f)))), c(c), d(d) {}
  __device__ __forceinline__ double operator()(float ww, double z) const {
    const float w = __builtin_amdgcn_sqrtf(ww * (1.02f + d * 0x1p-23f) + d * 0x1p-125f);
    return c * x * w * 0x1.001p-24f + (z * 0x1p-23 + c * 0x1p-125);
  }
};

__device__ __forceinline__ unsigned order_key(float v) {
  if (v != v) return 0xffffffffu;  // NaN above everything
  const unsigned u = __builtin_bit_cast(unsigned, v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long order_key(double v) {
  if (v != v) return ~0ull;
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ float key_value(unsigned key) {
  return __builtin_bit_cast(float, key >> 31 ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ double key_value(unsigned long long key) {
  return __builtin_bit_cast(double, key >> 63 ? key & ~(1ull << 63) : ~key);
}

// k-th largest (k >= 1) of `count` keys; on return `above` keys are larger than the result and `same` equal it. All
// threads call it.
template <typename K, class F>
__device__ K radix_kth(int count, int k, F key, int* hist, int* pick, int& above, int& same) {
  K found = 0, mask = 0;
  above = 0;
  for (int shift = (int)sizeof(K) * 8 - 8; shift >= 0; shift -= 8) {
    for (int b = threadIdx.x; b < 256; b += blockDim.x) hist[b] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < count; i += blockDim.x) {
      const K v = key(i);
      if ((v & mask) == found) atomicAdd(&hist[(int)(v >> shift) & 255], 1);
    }
    __syncthreads();
    if (threadIdx.x < 64) {  // bins from the top, four per lane
      int c[4], sum = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) sum += c[u] = hist[255 - (threadIdx.x * 4 + u)];
      int incl = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(incl, o, 64);
        if ((int)threadIdx.x >= o) incl += t;
      }
      int before = incl - sum;
      const int want = k - above;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (before < want && want <= before + c[u]) {
          pick[0] = 255 - (threadIdx.x * 4 + u);
          pick[1] = before;
          pick[2] = c[u];
        }
        before += c[u];
      }
    }
    __syncthreads();
    found |= (K)pick[0] << shift;
    mask |= (K)255 << shift;
    above += pick[1];
    same = pick[2];
  }
  __syncthreads();
  return found;
}

template <int N>
struct DotTag {
  static constexpr int kW = N;
};

template <typename T>
__global__ __launch_bounds__(1024, sizeof(T) == 4 ? 5 : 4) void topk_kernel(TopArgs p) {
  __shared__ unsigned long long keys[kTopList];
  __shared__ int hist[256], pick[3], cnt, wcnt[2][8][16];
  __shared__ int sel[kTopMax + kSpare + kSlack];
  __shared__ int cls[kTopMax + kSpare];
  __shared__ double xx;
  __shared__ unsigned long long cut;  // the least candidate's key
  // 16 rows share a line of the stats: rows next to each other go to one XCD (4096 rows of 65536 classes 241 -> 234 us)
  const int row = (int)(blockIdx.x & 7) * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3);
  if (row >= p.n) return;
  const int t = threadIdx.x, nt = blockDim.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), waves = nt >> 6, l = t & 63;
  const float2* st = p.stats + row;
  const float* z = p.z + (long long)row * p.ld;
  auto gkey = [&](int g) { return order_key(st[(long long)g * p.n].x); };
  const float4 ww4 = *(const float4*)p.norm_max;
  int nsel = p.groups;
  unsigned tau = 0;
  if (t == 0) cnt = 0, cut = 0;
  const int enough = p.kc + min(kSlack, p.kc >> 2);
  if (p.groups > p.kc) {
    if (p.groups <= nt * kTopHold) {
      unsigned mine[kTopHold];
#pragma unroll
      for (int u = 0; u < kTopHold; ++u) mine[u] = u * nt + t < p.groups ? gkey(u * nt + t) : 0u;
      const int live = (p.groups + nt - 1) / nt;
      // bits that all maxima share
      unsigned hi = 0, lo = ~0u;
#pragma unroll
      for (int u = 0; u < kTopHold; ++u)
        if (u * nt + t < p.groups) hi = max(hi, mine[u]), lo = min(lo, mine[u]);
#pragma unroll
      for (int o = 32; o; o >>= 1) hi = max(hi, (unsigned)__shfl_xor(hi, o, 64)), lo = min(lo, (unsigned)__shfl_xor(lo, o, 64));
      if (l == 0) wcnt[1][0][wave] = (int)hi, wcnt[1][1][wave] = (int)lo;
      __syncthreads();
      hi = (unsigned)wcnt[1][0][l % waves], lo = (unsigned)wcnt[1][1][l % waves];
#pragma unroll
      for (int o = 8; o; o >>= 1) hi = max(hi, (unsigned)__shfl_xor(hi, o, 64)), lo = min(lo, (unsigned)__shfl_xor(lo, o, 64));
      hi = __builtin_amdgcn_readfirstlane(hi), lo = __builtin_amdgcn_readfirstlane(lo);
      int top = hi == lo ? 0 : 32 - __builtin_clz(hi ^ lo);  // bits that differ
      tau = top == 32 ? 0 : lo >> top << top;
      // three bits per step: the highest of the seven thresholds above tau there that enough maxima reach
      for (int step = 0; top > 0 && nsel > enough; ++step) {
        const int bit = max(top - 3, 0), buf = step & 1;  // (the other buffer is written before the next barrier)
        int mineq = 0;                                    // lane q keeps the wave's count for threshold q
#pragma unroll
        for (int q = 1; q < 8; ++q) {
          int c = 0;
#pragma unroll
          for (int u = 0; u < kTopHold; ++u)
            if (u < live) c += __popcll(__ballot(mine[u] >= (tau | (unsigned)q << bit)));
          if (l == q) mineq = c;
        }
        if (l < 8) wcnt[buf][l][wave] = mineq;
        __syncthreads();
        const int w = l & 7;
        int n = (w < waves ? wcnt[buf][l >> 3][w] : 0) + (w + 8 < waves ? wcnt[buf][l >> 3][w + 8] : 0);
#pragma unroll
        for (int o = 4; o; o >>= 1) n += __shfl_xor(n, o, 64);
        const unsigned long long ok = __ballot(n >= p.kc && l >= 8);
        if (ok) {
          const int best = (63 - __builtin_clzll(ok)) >> 3;
          nsel = __builtin_amdgcn_readlane(n, best * 8);
          tau |= (unsigned)best << bit;
        }
        top = bit;
      }
      __syncthreads();
      if (nsel <= enough) {
#pragma unroll
        for (int u = 0; u < kTopHold; ++u)
          if (u * nt + t < p.groups && mine[u] >= tau) sel[atomicAdd(&cnt, 1)] = u * nt + t;
      }
    }
    if (nsel > enough) {  // ties at tau, or more groups than the registers hold
      int above, same;
      __syncthreads();
      tau = radix_kth<unsigned>(p.groups, p.kc, gkey, hist, pick, above, same);
      int seen = 0;
      for (int g0 = 0; g0 < p.groups; g0 += nt) {
        const bool in = g0 + t < p.groups;
        const unsigned key = in ? gkey(g0 + t) : 0u;
        const bool eq = in && key == tau;
        const unsigned long long m = __ballot(eq);
        if (l == 0) wcnt[0][0][wave] = __popcll(m);
        __syncthreads();
        int rank = seen + __popcll(m & ((1ull << l) - 1));
        for (int w = 0; w < waves; ++w) {
          if (w < wave) rank += wcnt[0][0][w];
          seen += wcnt[0][0][w];
        }
        if ((in && key > tau) || (eq && rank < p.kc - above)) sel[atomicAdd(&cnt, 1)] = g0 + t;
        __syncthreads();
      }
      nsel = p.kc;
    }
  }
  __syncthreads();
  if (t == 0) cnt = 0;
  __syncthreads();
  // i-th score of the groups kept
  auto at = [&](int i) { return (p.groups > p.kc ? sel[i >> 6] : i >> 6) * kGroup + (i & 63); };
  auto skey = [&](int i) {
    const int v = at(i);
    return v < p.V ? (unsigned long long)order_key(z[v]) << 32 | (unsigned)~v : 0ull;
  };
  constexpr int kFly = 16;  // groups in flight per wave
  for (int s0 = wave; s0 < nsel; s0 += waves * kFly) {
    float zv[kFly];
    int v[kFly];
#pragma unroll
    for (int u = 0; u < kFly; ++u) {
      v[u] = s0 + u * waves < nsel ? at((s0 + u * waves) * kGroup + l) : p.V;
      zv[u] = z[min(v[u], p.V - 1)];
    }
#pragma unroll
    for (int u = 0; u < kFly; ++u) {
      const unsigned o = order_key(zv[u]);
      const bool take = v[u] < p.V && o >= tau;
      const unsigned long long m = __ballot(take);
      if (!m) continue;
      int base = 0;
      if (l == 0) base = atomicAdd(&cnt, __popcll(m));
      base = __builtin_amdgcn_readfirstlane(base) + __popcll(m & ((1ull << l) - 1));
      if (take && base < kTopList) keys[base] = (unsigned long long)o << 32 | (unsigned)~v[u];
    }
  }
  __syncthreads();
  const int total = cnt;
  __syncthreads();
  if (t == 0) cnt = 0;
  __syncthreads();
  if (total <= 512) {  // (usual) a key is taken if fewer than kc are larger
    for (int i = t; i < total; i += nt) {
      const unsigned long long mine = keys[i];
      int rank = 0;
#pragma unroll 4
      for (int o = 0; o < total; ++o) rank += keys[o] > mine;
      if (rank < p.kc) cls[rank] = (int)~(unsigned)mine;
      if (rank == p.kc - 1) cut = mine;
    }
  } else {
    const bool listed = total <= kTopList;
    const int count = listed ? total : nsel * kGroup;
    auto lkey = [&](int i) { return listed ? keys[i] : skey(i); };
    int above, same;
    const unsigned long long least = radix_kth<unsigned long long>(count, p.kc, lkey, hist, pick, above, same);
    for (int i = t; i < count; i += nt) {
      const unsigned long long key = lkey(i);
      if (key >= least) cls[atomicAdd(&cnt, 1)] = (int)~(unsigned)key;
    }
    if (t == 0) cut = least;
  }
  __syncthreads();
  // 64-bit scores (before the division by T) of `count` classes as keys, a few at a time per wave: two, further ahead, where
  // the waves suffice. The last wave, which has the least to do, also takes the row's own squares.
  auto dots = [&](auto tag, const int* c, int count, unsigned long long* key, bool squares) {
    constexpr int kW = decltype(tag)::kW;
    const T *x = (const T*)p.x + row * p.xrs, *bias = (const T*)p.bias;
    for (int c0 = wave * kW; c0 < count; c0 += waves * kW) {
      const T* w[kW];
#pragma unroll
      for (int u = 0; u < kW; ++u) w[u] = (const T*)p.w + (long long)c[min(c0 + u, count - 1)] * p.wrs;
      double s[kW];
      row_dots<T, double, kW, 8 / kW>(x, p.xcs, w, p.wcs, p.d, p.vec, s);
      if (l == 0)
#pragma unroll
        for (int u = 0; u < kW; ++u)
          if (c0 + u < count) key[c0 + u] = order_key(s[u] + (bias ? (double)Elem<T>::get(bias, c[c0 + u]) : 0.0));
    }
    if (squares && wave == waves - 1) {
      const T* w[1] = {x};
      double s[1];
      row_dots<T, double, 1, 4>(x, p.xcs, w, p.xcs, p.d, p.vec, s);
      if (l == 0) xx = s[0];
    }
  };
  const bool all = p.kc == p.V;  // every class is a candidate
  if (p.kc <= 2 * waves)
    dots(DotTag<2>(), cls, p.kc, keys, !all);
  else
    dots(DotTag<4>(), cls, p.kc, keys, !all);
  __syncthreads();
  // the k best so far (and room for the next), behind the candidates' keys and a turn's classes
  unsigned long long *bkey = &keys[kTurnList + kTurnList / 2], *nkey = bkey + kTopMax + kTopMax / 2;
  int *bcls = (int*)(bkey + kTopMax), *ncls = (int*)(nkey + kTopMax);
  static_assert(kTurnList + kTurnList / 2 + 3 * kTopMax <= kTopList, "");
  for (int c = t; c < p.kc; c += nt) {
    const unsigned long long mine = keys[c];
    const int v = cls[c];
    int rank = 0;
#pragma unroll 4
    for (int o = 0; o < p.kc; ++o) rank += keys[o] > mine || (keys[o] == mine && cls[o] < v);
    if (rank < p.k) bkey[rank] = mine, bcls[rank] = v;
  }
  __syncthreads();
  auto answer = [&]() {
    for (int c = t; c < p.k; c += nt) {
      p.values[(long long)row * p.k + c] = (float)(key_value(bkey[c]) * p.inv_t);
      p.classes[(long long)row * p.k + c] = bcls[c];
    }
  };
  if (all) return answer();
  double zk = key_value(uniform(bkey[p.k - 1]));
  const unsigned long long last = uniform(cut);
  const double zc = key_value((unsigned)(last >> 32));
  const Slack slack(xx, p.slack, p.d);
  // (classes at -inf are switched off, in 64 bits too; comparisons with NaN are false: such a row has some classes)
  const float ww = fmaxf(fmaxf(ww4.x, ww4.y), fmaxf(ww4.z, ww4.w));
  if (!(zk <= zc + slack(ww, fmax(fabs(zk), fabs(zc)))) || zc == -INFINITY) return answer();

  // classes of this turn and their keys
  int* tcls = (int*)&keys[kTurnList];
  unsigned long long* tkey = keys;
  auto reach = [&](int g) { return zk - slack(p.norms[g], fabs(zk)); };  // what a score of group g has to reach
  auto merge = [&]() {  // all threads, with the list written; cnt is 0 afterwards
    const int listed = __builtin_amdgcn_readfirstlane(cnt), total = p.k + listed;
    dots(DotTag<4>(), tcls, listed, tkey, false);
    __syncthreads();
    auto keyed = [&](int e) { return e < p.k ? bkey[e] : tkey[e - p.k]; };
    auto classed = [&](int e) { return e < p.k ? bcls[e] : tcls[e - p.k]; };
    for (int e = t; e < total; e += nt) {
      const unsigned long long mine = keyed(e);
      const int v = classed(e);
      int rank = 0;
      for (int o = 0; o < total; ++o) rank += keyed(o) > mine || (keyed(o) == mine && classed(o) < v);
      if (rank < p.k) nkey[rank] = mine, ncls[rank] = v;
    }
    if (t == 0) cnt = 0;
    __syncthreads();
    unsigned long long* const k = bkey;
    int* const c = bcls;
    bkey = nkey, bcls = ncls, nkey = k, ncls = c;
    zk = key_value(uniform(bkey[p.k - 1]));
  };
  __syncthreads();  // the candidates' keys have been read
  if (t == 0) cnt = 0;
  // groups in pieces of 256, those of a piece that reach far enough in `hist`; eight groups per step
  for (int g0 = 0; g0 < p.groups; g0 += 256) {
    if (t == 0) pick[0] = 0;
    __syncthreads();
    if (t < 256 && g0 + t < p.groups && (double)st[(long long)(g0 + t) * p.n].x >= reach(g0 + t)) hist[atomicAdd(&pick[0], 1)] = g0 + t;
    __syncthreads();
    const int listed = __builtin_amdgcn_readfirstlane(pick[0]);
    for (int s0 = 0; s0 < listed; s0 += kTurnAdd / kGroup) {
      const int have = __builtin_amdgcn_readfirstlane(cnt);
      __syncthreads();  // every wave has read it before one adds to it: all merge or none
      if (have > kTurnList - kTurnAdd) merge();
      for (int u = wave; u < kTurnAdd / kGroup && s0 + u < listed; u += waves) {
        const int g = hist[s0 + u], v = g * kGroup + l;
        const float zv = z[min(v, p.V - 1)];
        const bool take = v < p.V && (double)zv >= reach(g) && ((unsigned long long)order_key(zv) << 32 | (unsigned)~v) < last;
        const unsigned long long m = __ballot(take);
        int base = 0;
        if (l == 0 && m) base = atomicAdd(&cnt, __popcll(m));
        base = __builtin_amdgcn_readfirstlane(base) + __popcll(m & ((1ull << l) - 1));
        if (take) tcls[base] = v;
      }
      __syncthreads();
    }
  }
  merge();
  answer();
}

// ------------------------------------------------------------------ host side
static long long up(long long v, long long m) { return (v + m - 1) / m * m; }

// blocks of a product: what runs at once (each block takes several tiles in turn), a multiple of the 8 XCDs
inline int grid8(long long tiles, int per_cu) { return (int)std::min<long long>((tiles + 7) / 8 * 8, 256 * per_cu); }

// Tiles, with the rate of a long product (32768 x 8192 x 4096 and its two transposes, random data):
typedef TileCfg<256, 256, 2, 4, 32, 5> CfgBig;   // 1.39 PFLOP/s; all 160 KB of LDS, one block per CU
typedef TileCfg<128, 256, 2, 4, 64, 3> CfgWide;  // 1.25 - 1.35
typedef TileCfg<128, 128, 2, 2, 32, 4> CfgMid;   // 0.85 - 1.05 (bound by L2 reads); two blocks per CU in the gradients (188
                                                 // registers) and scores alone (244), one where E or z is kept (268)
typedef TileCfg<128, 128, 2, 2, 32, 10> CfgDeep; // the same tile where one round of blocks does: nine stages under way
typedef TileCfg<128, 128, 2, 4, 32, 3, 3> CfgF32; // three planes
typedef TileCfg<128, 32, 2, 1, 64, 4> CfgSlim;   // few rows: bound by reading w

constexpr int kMostParts = 4;  // of kNormParts

constexpr unsigned kLdsAll = 160 * 1024;

enum { kBig = 0, kWide = 1, kMid = 2, kF32 = 3 };

// How a product is laid over the card, and its estimated time in units of one CU's multiply-adds (2.7e12 a second):
// full rounds of blocks over the 256 CUs at the tile's rate, and about 4 us (10^7) each to start and finish; the
// tiles left over are cut along K into `ts` runs, at most one per block, whose sums are written and read again (4.6
// per value at the card's copy rate).
struct Layout {
  int cfg, whole, ts, per, grid;
  double cost;
};

static Layout layout_of(int cfg, long long m, long long n, long long k, int terms, bool runs) {
  const int bm = cfg == kBig ? 256 : 128, bn = cfg >= kMid ? 128 : 256;
  const double rate = cfg == kMid ? 0.7 : cfg == kWide ? 0.92 : 1.0;
  const long long tiles = (long long)ceil_div(m, bm) * ceil_div(n, bn), grid = cfg == kMid && tiles > 256 ? 512 : 256;
  const long long rounds = tiles / grid, tail = tiles % grid;
  auto one = [&](long long kk, long long blocks) {
    return (double)bm * bn * (double)up(kk, 64) * terms / rate * (double)std::min(grid / 256, (blocks + 255) / 256) + 1e7;
  };
  Layout best = {cfg, (int)tiles, 1, 0, (int)grid, 1e300};
  for (long long ts = 1; ts <= (runs && tail ? std::max(1LL, std::min(grid / tail, k * terms / 512)) : 1); ++ts) {
    const long long per = up((k + ts - 1) / ts, 64);
    if (ceil_div(k, per) != ts) continue;  // an empty run
    const double c = rounds * one(k, grid) + (tail ? one(per, tail * ts) : 0.0) + (ts > 1 ? 8e6 + 4.6 * (double)(tail * ts) * bm * bn : 0.0);
    if (c < best.cost) best = {cfg, (int)(ts > 1 ? tiles - tail : tiles), (int)ts, (int)per, (int)grid, c};
  }
  return best;
}

static Layout pick_layout(long long m, long long n, long long k, int terms, bool runs) {
  Layout best = layout_of(terms == 1 ? kBig : kF32, m, n, k, terms, runs);
  for (int c = kWide; terms == 1 && c <= kMid; ++c) {
    const Layout l = layout_of(c, m, n, k, terms, runs);
    if (l.cost < best.cost) best = l;
  }
  return best;
}

static long long run_bytes(const Layout& l, long long m, long long n) {
  const int bm = l.cfg == kBig ? 256 : 128, bn = l.cfg >= kMid ? 128 : 256;
  return l.ts == 1 ? 0 : ((long long)ceil_div(m, bm) * ceil_div(n, bn) - l.whole) * l.ts * bm * bn * 4;
}

// one round of Mid tiles: a block alone on its CU, so the latency of its K steps counts
static bool use_deep(long long tiles) { return tiles <= 256; }

// returns the parts of the squared norms
template <class C>
int scores_launch(ScoreArgs p, int mode, hipStream_t s) {
  p.nm = ceil_div(p.V, C::kBM);
  p.nn = ceil_div(p.n, C::kBN);
  p.parts = C::kWN * p.nn < kNormParts<C> ? 1 : kNormParts<C>;
  const int g = grid8((long long)p.nm * p.nn, kLdsAll / C::kLds);
#define YTK_SC(M) scores_kernel<C, M><<<g, C::kThreads, C::kLds, s>>>(p)
  if constexpr (C::kPlanes == 3) {
    if (mode == kExpFloat)
      YTK_SC(kExpFloat);
    else if (mode == kStatsFloat)
      YTK_SC(kStatsFloat);
    else
      YTK_SC(kScores);
  } else {
    if (mode == kStatsOnly)
      YTK_SC(kStatsOnly);
    else if (mode == kExpHalf)
      YTK_SC(kExpHalf);
    else
      YTK_SC(kScores);
  }
#undef YTK_SC
  YTK_LAUNCH_CHECK();
  return p.parts;
}

template <class C, int LA, int LB, typename T>
void grad_launch(GradArgs p, hipStream_t s) {
  const long long tiles = (long long)p.nm * p.nn;
  const int g = p.ts > 1 ? p.grid : grid8(tiles, kLdsAll / C::kLds);
  grad_kernel<C, LA, LB, T><<<g, C::kThreads, C::kLds, s>>>(p);
  YTK_LAUNCH_CHECK();
  if (p.ts > 1) {
    run_sum_kernel<C::kBM, C::kBN, T><<<dim3((unsigned)(tiles - p.whole), C::kBN / 32), 256, 0, s>>>(p);
    YTK_LAUNCH_CHECK();
  }
}

}  // namespace ytk

using namespace ytk;

// ------------------------------------------------------------------ plan
// Sizes and workspace of one call. The same code lays the workspace out for the size query and for the call.
struct HeadIn {  // lp of the entry points, in this order
  long long n, d, V, k, f32, xrs, xcs, wrs, wcs, idx64, ignore, base, mode, want_dx, want_dw, has_bias, piece_bytes, x_al, w_al;
};
constexpr int kHeadIn = 19;

static HeadIn head_in(const long long* lp) {
  HeadIn h;
  static_assert(sizeof(HeadIn) == kHeadIn * sizeof(long long), "");
  memcpy(&h, lp, sizeof(h));
  if (h.n < 1 || h.d < 1 || h.V < 1 || h.k < 1) throw std::invalid_argument("class head: empty problem");
  // 256 rows of an operand span less than 2^31 bytes (head_gemm.h)
  if (h.V > (1LL << 21) || h.d > (1LL << 21) || h.n > (1LL << 31) - 65536)
    throw std::invalid_argument("class head: more than 2M classes or features, or 2G rows");
  return h;
}

struct HeadPlan {
  int planes, terms;
  long long kp, ld, groups, piece;
  bool pack_x, pack_w, grads, few, few_dw, planes_d;
  int rw, few_per, few_runs;
  bool many;  // more than one piece of rows
  long long o_x, o_w, o_xg, o_e, o_d, o_stats, o_zt, o_q, o_coef, o_norm, o_part, o_dbacc, o_dwacc, o_split, o_wn, bytes;
};

static HeadPlan head_plan(const HeadIn& h, bool topk) {
  HeadPlan p = {};
  p.planes = h.f32 ? 3 : 1;
  p.terms = h.f32 ? 6 : 1;
  p.kp = up(h.d, 64);
  p.ld = up(h.V, 64);
  p.groups = p.ld / kGroup;
  p.grads = h.want_dx || h.want_dw;
  // few fp32 rows: w is read as it is; the planes of x serve dw alone
  p.few = h.f32 && h.n <= kFewRows;
  if (p.few && (h.xcs != 1 || h.wcs != 1)) throw std::invalid_argument("class head: few fp32 rows need dense columns");
  p.few_dw = p.few && h.n <= 64;  // (more rows: the planes of x and D)
  p.pack_x = p.few ? h.want_dw && !topk && !p.few_dw : h.f32 || !h.x_al;
  p.pack_w = !p.few && (h.f32 || !h.w_al);
  const long long per = topk ? p.ld * 4 : p.grads ? p.ld * (h.f32 ? 10 : 2) : p.groups * 8;
  // (at most 2M rows, fewer of long lists: the grids of the row passes count rows / 64 in 16 bits, and the targets' threads,
  // 16 per list entry, in 32)
  const long long most = topk ? 1LL << 21 : std::min(1LL << 21, (1LL << 25) / ceil_div(h.k, 4) / 256 * 256);
  p.piece = std::min(h.n, std::min(most, std::max(256LL, h.piece_bytes / per / 256 * 256)));
  p.many = p.piece < h.n;
  long long part = 0;
  if (h.want_dx && p.few) {  // runs of classes: about 1024 blocks, at least 128 classes each
    const long long runs = std::max(1LL, std::min<long long>(1024 / (ceil_div(h.d, 64) * ceil_div(h.n, 64)), ceil_div(h.V, 128)));
    p.few_per = (int)up((h.V + runs - 1) / runs, 64);
    p.few_runs = ceil_div(h.V, p.few_per);
    part = p.few_runs > 1 ? p.few_runs * h.n * h.d * 4 : 0;
  } else if (h.want_dx) {
    for (const long long rows : {p.piece, (h.n - 1) % p.piece + 1})
      part = std::max(part, run_bytes(pick_layout(h.d, rows, h.V, p.terms, true), h.d, rows));
  }
  if (h.want_dw && !p.many && !p.few_dw) part = std::max(part, run_bytes(pick_layout(h.d, h.V, h.n, p.terms, true), h.d, h.V));
  long long o = 0;
  auto take = [&](bool want, long long bytes) {
    const long long at = o;
    if (want) o += up(bytes, 256);
    return at;
  };
  p.o_x = take(p.pack_x, h.n * p.kp * 2 * p.planes);
  p.o_w = take(p.pack_w, h.V * p.kp * 2 * p.planes);
  p.o_xg = take(h.want_dw && !p.pack_x, p.piece * p.kp * 2);
  p.o_e = take(p.grads || topk, p.piece * p.ld * (h.f32 || topk ? 4 : 2));
  p.planes_d = p.grads && h.f32 && (!p.few || (h.want_dw && !p.few_dw));
  p.o_d = take(p.planes_d, p.piece * p.ld * 6);
  p.o_stats = take(true, p.groups * p.piece * 8);
  p.o_zt = take(!topk, p.piece * h.k * 4);
  p.o_q = take(p.grads, p.piece * h.k * 4);
  p.o_coef = take(p.grads, p.piece * 4);
  p.o_norm = take(p.grads, p.piece * 8);
  const bool db = h.want_dw && h.has_bias;
  // rows per wave of the D pass: fewer where there would be fewer than about 2048 blocks
  p.rw = kDRows;
  while (p.rw > 1 && ceil_div(p.piece, 4 * p.rw) * ceil_div(p.ld, kDCols) < 2048) p.rw /= 2;
  p.o_part = take(db, ceil_div(p.piece, 4 * p.rw) * p.ld * 4);
  p.o_dbacc = take(db, h.V * 4);
  p.o_dwacc = take(h.want_dw && p.many, h.V * h.d * 4);
  p.o_split = take(part > 0, part);
  p.o_wn = take(topk, (kMostParts * p.groups + 4) * 4);  // four, the largest of which is the largest squared norm of w; that of each group
  p.bytes = o;
  return p;
}

template <typename T>
static void pack(const void* src, long long rs, long long cs, long long rows, long long cols, char* dst, long long ld,
                 const float* coef, hipStream_t s) {
  const dim3 g(ceil_div(ld, 64), ceil_div(rows, 64));
  pack_kernel<T, sizeof(T) == 4 ? 3 : 1><<<g, 256, 0, s>>>((const T*)src, rs, cs, rows, (int)cols, (__bf16*)dst, ld, rows * ld, coef);
  YTK_LAUNCH_CHECK();
}

// grid.y is at most 65535: rows beyond 64 * 65535 go in further launches, planes keep the distance of the whole
template <typename T>
static void pack_rows(const void* src, long long rs, long long cs, long long rows, long long cols, char* dst, long long ld,
                      const float* coef, hipStream_t s) {
  constexpr long long kMost = 64LL * 65535;
  if (rows <= kMost) return pack<T>(src, rs, cs, rows, cols, dst, ld, coef, s);
  for (long long r = 0; r < rows; r += kMost) {
    const long long m = std::min(kMost, rows - r);
    const dim3 g(ceil_div(ld, 64), ceil_div(m, 64));
    pack_kernel<T, sizeof(T) == 4 ? 3 : 1><<<g, 256, 0, s>>>((const T*)src + r * rs, rs, cs, m, (int)cols, (__bf16*)dst + r * ld, ld,
                                                              rows * ld, coef ? coef + r : nullptr);
    YTK_LAUNCH_CHECK();
  }
}

// C = A B^T of g.M x g.N x g.K; `part` has room for the runs of this layout
template <int LA, int LB, typename T>
static void grad_product(GradArgs g, bool runs, hipStream_t s) {
  const Layout l = pick_layout(g.M, g.N, g.K, sizeof(T) == 4 ? 6 : 1, runs);
  g.whole = l.whole, g.ts = l.ts, g.per = l.per, g.grid = l.grid;
  g.nm = ceil_div(g.M, l.cfg == kBig ? 256 : 128);
  g.nn = ceil_div(g.N, l.cfg >= kMid ? 128 : 256);
  if constexpr (sizeof(T) == 4) {
    grad_launch<CfgF32, LA, LB, T>(g, s);
  } else {
    if (l.cfg == kBig)
      grad_launch<CfgBig, LA, LB, T>(g, s);
    else if (l.cfg == kWide)
      grad_launch<CfgWide, LA, LB, T>(g, s);
    else if (use_deep((long long)g.nm * g.nn))
      grad_launch<CfgDeep, LA, LB, T>(g, s);
    else
      grad_launch<CfgMid, LA, LB, T>(g, s);
  }
}

template <typename T>
static void split_sum(const float* acc, int splits, long long rows, long long cols, void* out, hipStream_t s) {
  const int blocks = (int)std::min<long long>((rows * cols + 255) / 256, 4096);
  split_sum_kernel<T><<<blocks, 256, 0, s>>>(acc, splits, rows, (int)cols, (T*)out, cols);
  YTK_LAUNCH_CHECK();
}

struct HeadOps {  // operands of the products for one call
  Operand w, x;
};

static HeadOps head_operands(const HeadIn& h, const HeadPlan& p, const void* x, const void* w, char* ws, hipStream_t s) {
  HeadOps o;
  if (p.pack_x) {
    if (h.f32)
      pack_rows<float>(x, h.xrs, h.xcs, h.n, h.d, ws + p.o_x, p.kp, nullptr, s);
    else
      pack_rows<__bf16>(x, h.xrs, h.xcs, h.n, h.d, ws + p.o_x, p.kp, nullptr, s);
    o.x = {ws + p.o_x, p.kp * 2, h.n * p.kp * 2, (int)h.n};
  } else {
    o.x = {(const char*)x, h.xrs * 2, 0, (int)h.n};
  }
  if (p.pack_w) {
    if (h.f32)
      pack_rows<float>(w, h.wrs, h.wcs, h.V, h.d, ws + p.o_w, p.kp, nullptr, s);
    else
      pack_rows<__bf16>(w, h.wrs, h.wcs, h.V, h.d, ws + p.o_w, p.kp, nullptr, s);
    o.w = {ws + p.o_w, p.kp * 2, h.V * p.kp * 2, (int)h.V};
  } else {
    o.w = {(const char*)w, h.wrs * 2, 0, (int)h.V};
  }
  return o;
}

static Operand rows_from(Operand o, long long r0, long long rows) {
  o.p += r0 * o.pitch;
  o.ext = (int)rows;
  return o;
}

template <int kNT>
static void scores_few_n(const FewArgs& a, int mode, hipStream_t s) {
  const dim3 g(ceil_div(a.V, kGroup), ceil_div(a.n, kNT * 16));
  if (mode == kStatsFloat)
    scores_few_kernel<kNT, kStatsFloat><<<g, 256, 0, s>>>(a);
  else if (mode == kExpFloat)
    scores_few_kernel<kNT, kExpFloat><<<g, 256, 0, s>>>(a);
  else
    scores_few_kernel<kNT, kScores><<<g, 256, 0, s>>>(a);
  YTK_LAUNCH_CHECK();
}

static void scores_few(const HeadIn& h, const HeadPlan& p, const void* x, const void* w, const void* bias, float temp, char* ws, int mode,
                       const void* label, hipStream_t s) {
  FewArgs a = {};
  a.label = label, a.idx64 = (int)h.idx64, a.zt = (float*)(ws + p.o_zt);
  a.w = (const float*)w, a.x = (const float*)x, a.bias = (const float*)bias;
  a.wrs = h.wrs, a.xrs = h.xrs;
  a.V = (int)h.V, a.n = (int)h.n, a.d = (int)h.d;
  a.inv_t = 1.0f / temp;
  a.stats = (float2*)(ws + p.o_stats);
  a.e = (float*)(ws + p.o_e);
  a.ld = p.ld;
  a.norms = (float*)(ws + p.o_wn) + 4;
  if (h.n <= 16)
    scores_few_n<1>(a, mode, s);
  else if (h.n <= 32)
    scores_few_n<2>(a, mode, s);
  else
    scores_few_n<4>(a, mode, s);
}

static void dx_few(const HeadIn& h, const HeadPlan& p, const void* w, char* ws, void* out, hipStream_t s) {
  FewGradArgs a = {};
  a.w = (const float*)w, a.D = (const float*)(ws + p.o_e);
  a.wrs = h.wrs, a.ld = p.ld;
  a.V = (int)h.V, a.n = (int)h.n, a.d = (int)h.d, a.per = p.few_per;
  a.acc = p.few_runs > 1 ? (float*)(ws + p.o_split) : (float*)out;
  const dim3 g(ceil_div(h.d, 64), p.few_runs, h.n <= 64 ? 1 : ceil_div(h.n, 64));
  if (h.n <= 16)
    dx_few_kernel<1><<<g, 256, 0, s>>>(a);
  else if (h.n <= 32)
    dx_few_kernel<2><<<g, 256, 0, s>>>(a);
  else
    dx_few_kernel<4><<<g, 256, 0, s>>>(a);
  YTK_LAUNCH_CHECK();
  if (p.few_runs > 1) split_sum<float>(a.acc, p.few_runs, h.n, h.d, out, s);
}

static void dw_few(const HeadIn& h, const HeadPlan& p, const void* x, char* ws, void* out, hipStream_t s) {
  FewOuterArgs a = {};
  a.x = (const float*)x, a.D = (const float*)(ws + p.o_e), a.coef = (const float*)(ws + p.o_coef);
  a.xrs = h.xrs, a.ld = p.ld;
  a.V = (int)h.V, a.n = (int)h.n, a.d = (int)h.d;
  // about 4096 blocks, each with its x loaded once
  const long long runs = std::max(1LL, std::min<long long>(4096 / ceil_div(h.d, 256), ceil_div(h.V, 64)));
  a.per = (int)up((h.V + runs - 1) / runs, 64);
  a.dw = (float*)out;
  const dim3 g(ceil_div(h.d, 256), ceil_div(h.V, a.per));
  if (h.n <= 16)
    dw_few_kernel<1><<<g, 256, 0, s>>>(a);
  else if (h.n <= 32)
    dw_few_kernel<2><<<g, 256, 0, s>>>(a);
  else
    dw_few_kernel<4><<<g, 256, 0, s>>>(a);
  YTK_LAUNCH_CHECK();
}

// returns the parts of the squared norms of w (scores that are kept)
static int scores(const HeadIn& h, const HeadPlan& p, const HeadOps& o, long long r0, long long rows, const void* bias, float temp,
                   char* ws, int mode, const void* label, hipStream_t s) {
  ScoreArgs a = {};
  a.label = label, a.idx64 = (int)h.idx64, a.zt = (float*)(ws + p.o_zt);
  a.w = o.w;
  a.x = rows_from(o.x, r0, rows);
  a.kw = (int)(p.pack_w ? p.kp : h.d);
  a.kx = (int)(p.pack_x ? p.kp : h.d);
  a.V = (int)h.V;
  a.n = (int)rows;
  a.bias = bias;
  a.inv_t = 1.0f / temp;
  a.stats = (float2*)(ws + p.o_stats);
  a.e = ws + p.o_e;
  a.z = (float*)(ws + p.o_e);
  a.ld = p.ld;
  a.norms = (float*)(ws + p.o_wn) + 4;
  const int tile = pick_layout(h.V, rows, p.kp, p.terms, false).cfg;
  if (h.f32)
    return scores_launch<CfgF32>(a, mode, s);
  if (rows <= 64)
    return scores_launch<CfgSlim>(a, mode, s);
  if (tile == kBig)
    return scores_launch<CfgBig>(a, mode, s);
  if (tile == kWide)
    return scores_launch<CfgWide>(a, mode, s);
  if (use_deep((long long)ceil_div(h.V, 128) * ceil_div(rows, 128)))
    return scores_launch<CfgDeep>(a, mode, s);
  return scores_launch<CfgMid>(a, mode, s);
}

// whole, aligned 16-byte pieces in the rows of x and w
static int dots_vec(const HeadIn& h, const void* x, const void* w) {
  const long long e = h.f32 ? 4 : 8;
  return h.xcs == 1 && h.wcs == 1 && h.d % e == 0 && h.xrs % e == 0 && h.wrs % e == 0 && ((uintptr_t)x & 15) == 0 && ((uintptr_t)w & 15) == 0;
}

template <typename T>
static void targets(const TargetArgs& t, hipStream_t s) {
  if (t.k == 1)
    target_kernel<T, 1><<<ceil_div(t.n, 4), 256, 0, s>>>(t);
  else
    target_kernel<T, 4><<<ceil_div((long long)t.n * ceil_div(t.k, 4), 4), 256, 0, s>>>(t);
  YTK_LAUNCH_CHECK();
}

static void rows_pass(RowArgs a, bool base2, hipStream_t s) {
  // 16 rows share the lines of the group statistics, unless that leaves CUs without a block
  a.rb = 1;
  while (a.rb < 16 && a.rb * 512 <= a.n) a.rb *= 2;
  if (base2)
    row_kernel<true><<<ceil_div(a.n, a.rb), 256, 0, s>>>(a);
  else
    row_kernel<false><<<ceil_div(a.n, a.rb) + (a.norms ? 1 : 0), 256, 0, s>>>(a);
  YTK_LAUNCH_CHECK();
}

extern "C" long long ytk_head_loss_ws(const long long* lp) { return head_plan(head_in(lp), false).bytes; }

// ptrs: x, w, bias, idx, tl, tlse, weight, ws, loss, lse, dx, dw, db
extern "C" void ytk_head_loss(const uintptr_t* ptrs, const long long* lp, double temp_, uintptr_t stream) {
  const HeadIn h = head_in(lp);
  const HeadPlan p = head_plan(h, false);
  hipStream_t s = (hipStream_t)stream;
  const float temp = (float)temp_;
  const char *x = (const char*)ptrs[0], *idx = (const char*)ptrs[3];
  const void *w = (const void*)ptrs[1], *bias = (const void*)ptrs[2];
  const float *tl = (const float*)ptrs[4], *tlse = (const float*)ptrs[5], *weight = (const float*)ptrs[6];
  char* ws = (char*)ptrs[7];
  float *loss = (float*)ptrs[8], *lse = (float*)ptrs[9];
  const int el = h.f32 ? 4 : 2;
  const HeadOps o = head_operands(h, p, x, w, ws, s);
  for (long long r0 = 0; r0 < h.n; r0 += p.piece) {
    const long long rows = std::min(p.piece, h.n - r0);
    const bool first = r0 == 0, last = r0 + rows == h.n;
    TargetArgs t = {};
    t.x = x + r0 * h.xrs * el;
    t.w = w;
    t.bias = bias;
    t.xrs = h.xrs, t.xcs = h.xcs, t.wrs = h.wrs, t.wcs = h.wcs;
    t.idx = idx + r0 * h.k * (h.idx64 ? 8 : 4);
    t.idx64 = (int)h.idx64;
    t.k = (int)h.k, t.n = (int)rows, t.d = (int)h.d, t.V = (int)h.V, t.vec = dots_vec(h, x, w);
    t.zt = (float*)(ws + p.o_zt);
    const void* label = h.mode == 0 ? t.idx : nullptr;
    if (p.few)
      scores_few(h, p, x, w, bias, temp, ws, p.grads ? kExpFloat : kStatsFloat, label, s);
    else
      scores(h, p, o, r0, rows, bias, temp, ws, h.f32 ? (p.grads ? kExpFloat : kStatsFloat) : p.grads ? kExpHalf : kStatsOnly, label, s);
    if (h.mode != 0) {  // (a label's score comes from the products)
      if (h.f32)
        targets<float>(t, s);
      else
        targets<__bf16>(t, s);
    }
    RowArgs r = {};
    r.stats = (const float2*)(ws + p.o_stats);
    r.groups = (int)p.groups, r.n = (int)rows, r.base = (int)h.base;
    r.V = (int)h.V, r.k = (int)h.k, r.mode = (int)h.mode;
    r.idx = t.idx, r.idx64 = t.idx64, r.ignore = h.ignore;
    r.tl = tl ? tl + r0 * h.k : nullptr, r.tlse = tlse ? tlse + r0 : nullptr;
    r.weight = weight ? weight + r0 : nullptr;
    r.zt = t.zt, r.temp = temp, r.inv_t = 1.0f / temp;
    r.lse = lse + r0, r.loss = loss + r0;
    r.coef = p.grads ? (float*)(ws + p.o_coef) : nullptr;
    r.q = p.grads ? (float*)(ws + p.o_q) : nullptr;
    r.norm = p.grads ? (float2*)(ws + p.o_norm) : nullptr;
    rows_pass(r, !h.f32, s);
    if (!p.grads) continue;

    const bool db = h.want_dw && h.has_bias;
    DArgs d = {};
    d.stats = r.stats, d.norm = r.norm, d.coef = r.coef, d.q = r.q, d.zt = r.zt;
    d.idx = t.idx, d.idx64 = t.idx64, d.n = (int)rows, d.V = (int)h.V, d.k = (int)h.k;
    d.e = ws + p.o_e, d.d = (__bf16*)(ws + p.o_d), d.ld = p.ld, d.plane = rows * p.ld;
    d.part = db ? (float*)(ws + p.o_part) : nullptr;
    d.unit = h.f32 ? 1.0f / temp : 1.0f / temp * kLog2e;
    d.rw = p.rw;
    d.label = h.mode == 0;
    d.keep32 = p.few;
    if (h.f32 && !p.planes_d) d.d = nullptr;
    if (h.want_dw && p.pack_x) {
      d.x = ws + p.o_x + r0 * p.kp * 2;
      d.xpitch = p.kp * 2, d.xplane = h.n * p.kp * 2, d.planes = p.planes;
    }
    const dim3 dg(ceil_div(p.ld, kDCols), ceil_div(rows, 4 * p.rw));
    if (h.f32)
      dscore_kernel<true><<<dg, 256, 0, s>>>(d);
    else
      dscore_kernel<false><<<dg, 256, 0, s>>>(d);
    YTK_LAUNCH_CHECK();
    if (db) {
      float* acc = (float*)(ws + p.o_dbacc);
      if (h.f32)
        db_kernel<float><<<ceil_div(h.V, 64), 1024, 0, s>>>(d.part, (int)dg.y, p.ld, (int)h.V, acc, first, last ? (float*)ptrs[12] : nullptr);
      else
        db_kernel<__bf16><<<ceil_div(h.V, 64), 1024, 0, s>>>(d.part, (int)dg.y, p.ld, (int)h.V, acc, first, last ? (__bf16*)ptrs[12] : nullptr);
      YTK_LAUNCH_CHECK();
    }
    // D as an operand: rows = score rows, K contiguous for dx, K strided for dw
    const Operand D = {h.f32 ? ws + p.o_d : ws + p.o_e, p.ld * 2, rows * p.ld * 2, (int)rows};
    if (h.want_dx && p.few) {
      dx_few(h, p, w, ws, (void*)ptrs[10], s);
    } else if (h.want_dx) {
      GradArgs g = {};
      g.a = o.w;
      g.a.ext = (int)(p.pack_w ? p.kp : h.d);
      g.b = D;
      g.ka = h.V, g.kb = p.ld;
      g.K = (int)h.V;
      g.M = (int)h.d, g.N = (int)rows;
      g.out = (char*)ptrs[10] + r0 * h.d * el, g.ldo = h.d;
      g.part = (float*)(ws + p.o_split);
      if (h.f32)
        grad_product<kKS, kKC, float>(g, true, s);
      else
        grad_product<kKS, kKC, __bf16>(g, true, s);
    }
    if (h.want_dw && p.few_dw) {
      dw_few(h, p, x, ws, (void*)ptrs[11], s);
    } else if (h.want_dw) {
      GradArgs g = {};
      if (p.pack_x) {
        g.a = rows_from(o.x, r0, rows);
      } else {
        pack_rows<__bf16>(x + r0 * h.xrs * el, h.xrs, h.xcs, rows, h.d, ws + p.o_xg, p.kp, r.coef, s);
        g.a = {ws + p.o_xg, p.kp * 2, 0, 0};
      }
      g.a.ext = (int)p.kp;
      g.b = D;
      g.b.ext = (int)p.ld;
      g.ka = g.kb = rows;
      g.K = (int)rows;
      g.M = (int)h.d, g.N = (int)h.V;
      g.out = (void*)ptrs[11], g.ldo = h.d;
      g.part = (float*)(ws + p.o_split);
      g.acc = (float*)(ws + p.o_dwacc);
      g.mode = !p.many ? 0 : first ? 1 : last ? 3 : 2;
      if (h.f32)
        grad_product<kKS, kKS, float>(g, !p.many, s);
      else
        grad_product<kKS, kKS, __bf16>(g, !p.many, s);
    }
  }
}

extern "C" long long ytk_head_topk_ws(const long long* lp) { return head_plan(head_in(lp), true).bytes; }

// ptrs: x, w, bias, ws, values, classes, lse
extern "C" void ytk_head_topk(const uintptr_t* ptrs, const long long* lp, double temp_, uintptr_t stream) {
  const HeadIn h = head_in(lp);
  if (h.k > kTopMax || h.k > h.V) throw std::invalid_argument("head_topk: k is at most 256 and at most the number of classes");
  const HeadPlan p = head_plan(h, true);
  hipStream_t s = (hipStream_t)stream;
  const char* x = (const char*)ptrs[0];
  const void *w = (const void*)ptrs[1], *bias = (const void*)ptrs[2];
  char* ws = (char*)ptrs[3];
  const int el = h.f32 ? 4 : 2;
  const HeadOps o = head_operands(h, p, x, w, ws, s);
  for (long long r0 = 0; r0 < h.n; r0 += p.piece) {
    const long long rows = std::min(p.piece, h.n - r0);
    int parts = 1;
    if (p.few)
      scores_few(h, p, x, w, bias, (float)temp_, ws, kScores, nullptr, s);
    else
      parts = scores(h, p, o, r0, rows, bias, (float)temp_, ws, kScores, nullptr, s);
    RowArgs r = {};
    r.parts = parts;
    r.stats = (const float2*)(ws + p.o_stats);
    r.groups = (int)p.groups, r.n = (int)rows, r.V = (int)h.V;
    r.inv_t = 1.0f / (float)temp_;
    r.norm_max = (float*)(ws + p.o_wn), r.norms = r.norm_max + 4;
    r.lse = (float*)ptrs[6] + r0;
    rows_pass(r, false, s);
    TopArgs t = {};
    t.stats = r.stats;
    t.z = (const float*)(ws + p.o_e);
    t.ld = p.ld;
    t.n = (int)rows, t.V = (int)h.V, t.d = (int)h.d, t.groups = (int)p.groups;
    t.vec = dots_vec(h, x, w);
    t.k = (int)h.k, t.kc = (int)std::min(h.k + kSpare, h.V);
    t.x = x + r0 * h.xrs * el, t.w = w, t.bias = bias;
    t.xrs = h.xrs, t.xcs = h.xcs, t.wrs = h.wrs, t.wcs = h.wcs;
    t.inv_t = 1.0 / temp_;
    t.norms = r.norms, t.norm_max = r.norm_max;
    t.slack = (p.few ? 1.0f : 0.5f) * (float)h.d + 64.0f;
    t.values = (float*)ptrs[4] + r0 * h.k;
    t.classes = (long long*)ptrs[5] + r0 * h.k;
    const int threads = rows < 256 ? 1024 : 256;  // fewer rows than CUs: more waves for each
    if (h.f32)
      topk_kernel<float><<<(int)up(rows, 8), threads, 0, s>>>(t);
    else
      topk_kernel<__bf16><<<(int)up(rows, 8), threads, 0, s>>>(t);
    YTK_LAUNCH_CHECK();
  }
}
