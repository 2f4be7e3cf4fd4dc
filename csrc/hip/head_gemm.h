// Matrix-product core of the class head (head.hip): C[m][n] = sum_k A[m][k] B[n][k] in bf16 on the
// matrix cores, fp32 accumulators, gfx950 only.
//
// One block computes a kBM x kBN tile in K steps of kBK = 64 or 32. An operand lies in memory either with K
// contiguous (kKC: row r holds its K values) or with K strided (kKS: row k holds the values of all m or n);
// the three products of a softmax head need all of them from the same row-major x, w and D:
//   scores  z^T[v][i] = sum_d w[v][d] x[i][d]   A = w (KC)  B = x (KC)
//   dx^T[d][i]        = sum_v w[v][d] D[i][v]   A = w (KS)  B = D (KC)
//   dw^T[d][v]        = sum_i x[i][d] D[i][v]   A = x (KS)  B = D (KS)
// M is always the dimension that is contiguous in the result, because a 32x32 accumulator holds four
// consecutive m per lane.
//
// Tiles go from global memory straight into LDS (buffer_load ... lds, 16 B a lane). The buffer descriptor ends at
// the operand's last byte, so rows past the end (of M, N or K) read as zero and need no branch.
// The DMA writes LDS linearly, so the bank swizzle is applied to the SOURCE address: a KC row is eight or four 16-B
// chunks, chunk c of row r sits at c ^ swc(r); a KS row is cut into 64-B units, unit u of row k sits at u ^ swz(k). KC fragments are ds_read_b128; KS fragments are read transposed
// (ds_read_b64_tr_b16: 16 lanes exchange a 4 x 16 block).
#pragma once
#include "common.h"

namespace ytk {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

enum { kKC = 0, kKS = 1 };

// fp32 operands are three bf16 planes (hi, mid, lo: 24 bits); a product takes the six plane pairs whose weight is
// above 2^-24. A stage then holds all planes of its K step: each is read once
// from memory and from LDS for the products it is part of.
__device__ constexpr int kPairA[6] = {2, 0, 1, 1, 0, 0}, kPairB[6] = {0, 2, 1, 0, 1, 0};

struct Operand {
  const char* p;    // plane 0
  long long pitch;  // bytes per memory row
  long long plane;  // bytes from plane to plane
  int ext;          // extent of M (or N)
};

// m0 holds the LDS address. It is declared as written, although the compiler gives it to no value, so that a setting of its own
// for an instruction that reads m0 is not carried across (the compiler warns of any such register on a list).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16(unsigned voff, i32x4 rsrc, unsigned soff, unsigned lds) {
  asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voff), "s"(rsrc), "s"(soff),
               "s"(lds)
               : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lgkm() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// one operand's side of the tile: kT = tile extent, kNW waves load it, kFB 32-wide fragments per wave
template <int kL, int kT, int kNW, int kFB, int kBK>
struct Side {
  static constexpr int kBytes = kT * kBK * 2;       // per stage
  static constexpr int kLoads = kBytes / 1024 / kNW;  // DMA instructions per wave and stage
  static_assert(kBytes % (1024 * kNW) == 0, "tile not divisible among the waves");
  static constexpr int kCh = kBK / 8, kRpi = 64 / kCh;  // KC: 16-B chunks per row, rows per DMA instruction
  static_assert(kBK == 32 || kBK == 64, "");
  // KC swizzle: a ds_read_b128 serves rows {0-3, 12-15, 20-23, 24-27} of a fragment (or 16 in a row) together
  static __device__ __forceinline__ int swc(int row) { return kBK == 64 ? (row >> 1) & 7 : (row >> 2) & 3; }
  static constexpr int kRow = kT * 2;          // KS: LDS bytes per k row
  static constexpr int kUnits = kRow / 64;
  unsigned voff[kLoads];
  unsigned lds0;                // wave's first LDS byte of a stage
  unsigned rd[kL == kKC ? kBK / 16 : kFB];
  const char* base;
  long long rem;                // bytes to the operand's end
  unsigned koff;                // KC: bytes along K
  unsigned tail;                // KC: what puts this lane's piece of the last K step out of bounds if it lies past K
  long long step, plane;

  static __device__ __forceinline__ int swz(int row) { return ((row & 3) | (((row >> 3) & 1) << 2)) & (kUnits - 1); }

  // lane constants
  __device__ __forceinline__ void init(const Operand& o, long long K, int wave, int frag0, unsigned lds) {
    const int l = threadIdx.x & 63;
    tail = 0;
    if (kL == kKC) {
      // (the chunk a lane takes of its row is the same in all its loads: their rows differ by multiples of 16)
      static_assert((kNW * kRpi) % 16 == 0, "");
      const int last = (int)(K % kBK), c = (l & (kCh - 1)) ^ swc(wave * kRpi + l / kCh);
      if (last && c * 8 >= last) tail = 0x80000000u;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int row = (i * kNW + wave) * kRpi + l / kCh;
        voff[i] = (unsigned)(row * o.pitch) + (((l & (kCh - 1)) ^ swc(row)) << 4);
      }
#pragma unroll
      for (int s = 0; s < kBK / 16; ++s) {
        const int row = frag0 * 32 + (l & 31);
        rd[s] = lds + row * kBK * 2 + (((s * 2 + (l >> 5)) ^ swc(row)) << 4);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int byte = (i * kNW + wave) * 1024 + l * 16;
        const int row = byte / kRow, chunk = (byte % kRow) / 16;
        voff[i] = (unsigned)(row * o.pitch) + ((((chunk >> 2) ^ swz(row)) << 2 | (chunk & 3)) << 4);
      }
      const int g = l >> 4, i16 = l & 15, row = (g >> 1) * 8 + (i16 >> 2);
#pragma unroll
      for (int b = 0; b < kFB; ++b)
        rd[b] = lds + row * kRow + (((frag0 + b) ^ swz(row)) << 6) + (g & 1) * 32 + (i16 & 3) * 8;
    }
    lds0 = lds + wave * 1024;
  }
  // first row (or column) and K step of a tile
  __device__ __forceinline__ void at(const Operand& o, int t0, long long K, int kt0) {
    if (kL == kKC) {
      base = o.p + (long long)t0 * o.pitch + kt0 * (kBK * 2LL);
      rem = (long long)(o.ext - t0 - 1) * o.pitch + (K - kt0 * (long long)kBK) * 2;
      step = kBK * 2;
    } else {
      base = o.p + kt0 * (long long)kBK * o.pitch + t0 * 2LL;
      rem = (K - kt0 * (long long)kBK - 1) * o.pitch + (long long)(o.ext - t0) * 2;
      step = kBK * o.pitch;
    }
    plane = o.plane;
    koff = 0;
  }

  // Buffer descriptor and scalar offset of the stage to issue. A KC tile spans less than 2^31 bytes (checked by
  // the host), so K is the scalar offset; a KS operand may be longer than 2^32 bytes, so K moves the base.
  struct Src {
    i32x4 d;
    unsigned soff, past;
  };
  // the next K step
  __device__ __forceinline__ void advance() {
    if (kL == kKC) {
      koff += kBK * 2;
    } else {
      base += step;
      rem -= step;
    }
  }
  __device__ __forceinline__ Src src(int pl, bool some, bool last) const {
    const unsigned long long a = (unsigned long long)(base + pl * plane);
    const unsigned hi = (unsigned)((unsigned long long)rem >> 32), lo = (unsigned)rem;
    Src s;
    s.d[0] = __builtin_amdgcn_readfirstlane((int)(unsigned)a);
    s.d[1] = __builtin_amdgcn_readfirstlane((int)((a >> 32) & 0xffff));
    // past the last stage, and at or past the operand's end: no records, zeros
    s.d[2] = __builtin_amdgcn_readfirstlane(!some || (int)hi < 0 ? 0 : hi || lo > 0x7fffffffu ? 0x7fffffff : (int)lo);
    s.d[3] = 0x00020000;
    s.soff = kL == kKC ? __builtin_amdgcn_readfirstlane(koff) : 0u;
    s.past = last ? tail : 0u;
    return s;
  }
  // this wave's i-th piece of the stage at LDS offset `so`
  __device__ __forceinline__ void issue(int i, const Src& s, unsigned so) const {
    dma16(kL == kKC ? voff[i] + s.past : voff[i], s.d, s.soff, __builtin_amdgcn_readfirstlane(lds0 + so + i * kNW * 1024));
  }

  __device__ __forceinline__ bf16x8 frag(int b, int s, unsigned so) const {
    typedef __attribute__((address_space(3))) char lc;
    typedef __attribute__((address_space(3))) bf16x8 l8;
    typedef __attribute__((address_space(3))) bf16x4 l4;
    // constant parts as pointer arithmetic: they become the instruction's offset
    if (kL == kKC) return *(const l8*)((const lc*)(uintptr_t)(rd[s] + so) + b * 64 * kBK);
    const lc* q = (const lc*)(uintptr_t)(rd[b] + so) + s * 16 * kRow;
    const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((l4*)q);
    const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((l4*)(q + 4 * kRow));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

template <int BM, int BN, int WM, int WN, int BK, int S, int P = 1>
struct TileCfg {
  static constexpr int kPlanes = P, kBM = BM, kBN = BN, kWM = WM, kWN = WN, kBK = BK, kStages = S;
  static constexpr int kNW = WM * WN, kThreads = 64 * kNW;
  static constexpr int kFM = BM / WM / 32, kFN = BN / WN / 32;  // 32x32 blocks per wave
  static constexpr unsigned kStageBytes = (BM + BN) * BK * 2 * P;
  static constexpr unsigned kLds = S * kStageBytes;
};

// A wave's 4 KB of LDS to turn 32 rows of 128 bytes: lanes put 16-byte chunk c of their row, then take whole rows, eight
// per step, so that a store instruction covers full 128-byte lines. Against 32-byte pieces straight from the accumulators:
// fp32 scores of 4096 x 65536 at K = 1024 735 -> 668 us, E of 8192 x 131072 at K = 4096 -0.8 %; the gradients' bf16 stores
// did not gain (dw of 131072 x 4096 7.03 -> 7.17 ms) and stay direct.
struct Turn {
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) u32x4 l16;
  unsigned at;
  __device__ __forceinline__ void put(int row, int c, uint4 v) const {
    *(l16*)(uintptr_t)(at + row * 128 + ((c ^ (row & 7)) << 4)) = u32x4{v.x, v.y, v.z, v.w};
  }
  __device__ __forceinline__ uint4 take(int row, int c) const {
    const u32x4 v = *(const l16*)(uintptr_t)(at + row * 128 + ((c ^ (row & 7)) << 4));
    return make_uint4(v.x, v.y, v.z, v.w);
  }
};

// The squared norms of A's rows, as the products run: quarter q of a K step is taken by part q % kOf, and the waves that share A's
// rows, in one tile or in tiles side by side, take a part each (kOf = 0: none). Taken whole by every wave they cost 78 us of
// 650 (4096 x 65536, K = 1024); by one wave of the first tile, whose steps the others wait for, 13 there and 10 of 85 at
// 300 x 32003, K = 2048; in parts 0 and 6.
template <int kOf, int kIs>
struct Part {
  static constexpr bool takes(int q) { return kOf > 0 && q % (kOf > 0 ? kOf : 1) == kIs; }
};

// One block's tiles, one after the other: tile(j, m0, n0, kt0, nkt) tells its j-th (false: no more; nkt >= 1 steps
// of kBK from step kt0), done(j, m0, n0, acc, turn, sq) takes the accumulators, with a free stage to turn them in
// where kTurn, and with kParts > 0 the lane's part of the squared norms of A's rows: of row l % 32 of fragment i, half of the elements
// (lane l + 32 has the others) of its part, three planes by the largest. Wave wn of the t-th tile along n has part
// t kWN + wn, if that is below `parts` (kParts, or 1 where there are fewer such waves than kParts). The DMA runs S - 1 stages ahead across
// the border of two tiles, so only the epilogue's own instructions stand between their products. (Its stores share the
// counter of the DMA, which counts down in the order of issue.)
// ka, kb: extent of K in each operand's memory, a multiple of 8 for a KC operand; both reach every step:
// (kt0 + nkt - 1) * kBK < min(ka, kb). Past it an operand counts as zero, whatever its memory holds there (a KC operand
// whose K is no multiple of kBK: in the last step of every tile, so its tiles all run to the end of K).
template <class C, int kLA, int kLB, bool kTurn, int kParts = 0, class FTile, class FDone>
__device__ __forceinline__ void gemm_tiles(const Operand& A, const Operand& B, long long ka, long long kb, FTile tile,
                                           FDone done, int parts = kParts) {
  extern __shared__ __align__(1024) char head_smem[];
  typedef __attribute__((address_space(3))) char lc;
  const unsigned lds = (unsigned)(uintptr_t)(lc*)head_smem;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / C::kWN, wn = wave % C::kWN;
  typedef Side<kLA, C::kBM, C::kNW, C::kFM, C::kBK> SideA;
  typedef Side<kLB, C::kBN, C::kNW, C::kFN, C::kBK> SideB;
  SideA a;
  SideB b;
  a.init(A, ka, wave, wm * C::kFM, lds);
  constexpr int P = C::kPlanes, kTerms = P == 1 ? 1 : 6;
  static_assert(P == 1 || P == 3, "");
  b.init(B, kb, wave, wn * C::kFN, lds + P * SideA::kBytes);
  constexpr int kPlaneLoads = SideA::kLoads + SideB::kLoads, kLoads = P * kPlaneLoads;

  // the DMA's place in the stream of stages
  int ij = 0, ikt = 0, inkt = 0;
  bool some;
  auto begin = [&]() {
    int m0 = 0, n0 = 0, kt0 = 0;
    some = tile(ij, m0, n0, kt0, inkt);
    if (some) {
      a.at(A, m0, ka, kt0);
      b.at(B, n0, kb, kt0);
    } else {
      inkt = 1 << 30;
    }
    ikt = 0;
  };
  begin();
  if (!some) return;
  typename SideA::Src da[P];
  typename SideB::Src db[P];
  auto next = [&]() {  // (past the last stage: zeros that nothing reads, so that every step issues the same loads)
#pragma unroll
    for (int p = 0; p < P; ++p) {
      da[p] = a.src(p, some, ikt + 1 == inkt);
      db[p] = b.src(p, some, ikt + 1 == inkt);
    }
    a.advance();
    b.advance();
    if (++ikt == inkt) {
      ++ij;
      begin();
    }
  };
  auto piece = [&](int i, unsigned so) {
    const int p = i / kPlaneLoads, u = i % kPlaneLoads;
    if (u < SideA::kLoads)
      a.issue(u, da[p], so + p * SideA::kBytes);
    else
      b.issue(u - SideA::kLoads, db[p], so + p * SideB::kBytes);
  };
  constexpr int S = C::kStages;
  static_assert(S >= 3, "");
#pragma unroll
  for (int s = 0; s < S - 1; ++s) {
    next();
#pragma unroll
    for (int i = 0; i < kLoads; ++i) piece(i, s * C::kStageBytes);
  }
  wait_vm<(S - 2) * kLoads>();
  __builtin_amdgcn_s_barrier();

  bf16x8 fa[2][P][C::kFM], fb[2][P][C::kFN];
  auto read = [&](int r, int set, int q, unsigned so) {
    const int p = r % P, f = r / P;
    if (f < C::kFN)
      fb[set][p][f] = b.frag(f, q, so + p * SideB::kBytes);
    else
      fa[set][p][f - C::kFN] = a.frag(f - C::kFN, q, so + p * SideA::kBytes);
  };
  // kQ quarters per K step, each kFM rows of products. The next quarter's kR fragments are read during the first
  // half of a quarter (they have returned by its end), the DMA is issued in the second half: in one
  // burst, the loads stall every wave at the memory unit (1.20 -> 1.34 PFLOP/s at 32768 x 8192 x 4096).
  constexpr int kQ = C::kBK / 16, kR = P * (C::kFM + C::kFN), kHalf = C::kFM / 2, kSlots = kQ * (C::kFM - kHalf);
  // DMA instructions that may still be under way when the next stage has landed
  constexpr int kAhead = (S - 3) * kLoads + (kQ - 1) * (C::kFM - kHalf) * kLoads / kSlots;
  unsigned so = 0, fill = (S - 1) * C::kStageBytes;  // stage being read, stage being filled
#pragma unroll
  for (int r = 0; r < kR; ++r) read(r, 0, 0, 0);
  int m0, n0, kt0, nkt;
  for (int j = 0; tile(j, m0, n0, kt0, nkt); ++j) {
    // three planes: the five small pairs have sums of their own and the large one has two, so that these are rounded
    // less often and at a smaller size
    f32x16 acc[C::kFM][C::kFN] = {}, odd[C::kFM][C::kFN] = {}, low[C::kFM][C::kFN] = {};
    float sq[C::kFM] = {};
    auto steps = [&](auto part) {
    for (int left = nkt; left > 0; --left) {
      const unsigned after = so + C::kStageBytes == C::kLds ? 0u : so + C::kStageBytes;
#pragma unroll
      for (int q = 0; q < kQ; ++q) {
        if (q == kQ - 1) {
          // every read of this stage has returned and the next stage has landed: one barrier hands this buffer
          // to the DMA of the next step, while the products of the last quarter, already in registers, follow
          wait_lgkm();
          wait_vm<kAhead>();
          __builtin_amdgcn_s_barrier();
        }
#pragma unroll
        for (int i = 0; i < C::kFM; ++i) {
#pragma unroll
          for (int t = 0; t < kTerms; ++t)
#pragma unroll
            for (int j = 0; j < C::kFN; ++j) {
              f32x16& to = P == 1 ? acc[i][j] : t < 5 ? low[i][j] : q & 1 ? odd[i][j] : acc[i][j];
              to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[q & 1][P == 1 ? 0 : kPairA[t]][i], fb[q & 1][P == 1 ? 0 : kPairB[t]][j],
                                                           to, 0, 0, 0);
            }
          if (q == 0 && i == 0) next();  // scalar work, while the first products run
          if (i < kHalf) {
            // (the next step's are the next tile's after a tile's last step)
#pragma unroll
            for (int r = i * kR / kHalf; r < (i + 1) * kR / kHalf; ++r)
              read(r, (q + 1) & 1, (q + 1) % kQ, q == kQ - 1 ? after : so);
          } else {
            const int slot = q * (C::kFM - kHalf) + i - kHalf;
#pragma unroll
            for (int u = slot * kLoads / kSlots; u < (slot + 1) * kLoads / kSlots; ++u) piece(u, fill);
          }
          if (decltype(part)::takes(q)) {
            typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
            const bf16x8 f = fa[q & 1][0][i];
#pragma unroll
            for (int u = 0; u < 8; u += 2) {
              const bf16x2 v = {f[u], f[u + 1]};
              sq[i] = __builtin_amdgcn_fdot2_f32_bf16(v, v, sq[i], false);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      so = after;
      fill = fill + C::kStageBytes == C::kLds ? 0u : fill + C::kStageBytes;
    }
    };
    const int part = n0 / C::kBN * C::kWN + wn;
    if constexpr (kParts == 0) {
      steps(Part<0, 0>());
    } else if (part >= parts) {
      steps(Part<0, 0>());
    } else if (C::kWN < kParts && parts == 1) {
      steps(Part<C::kWN < kParts ? 1 : 0, 0>());
    } else if (part == 0) {
      steps(Part<kParts, 0>());
    } else if (kParts == 2 || part == 1) {
      steps(Part<kParts, 1>());
    } else if (part == 2) {
      steps(Part<kParts, kParts == 4 ? 2 : 0>());
    } else {
      steps(Part<kParts, kParts == 4 ? 3 : 0>());
    }
    if (P == 3)
#pragma unroll
      for (int i = 0; i < C::kFM; ++i)
#pragma unroll
        for (int j = 0; j < C::kFN; ++j) acc[i][j] += odd[i][j] + low[i][j];
    // the stage to be filled next is free: every wave has read it (last barrier), and none fills it before the next one
    static_assert(C::kStageBytes >= 4096u * C::kNW, "");
    done(j, m0, n0, acc, Turn{lds + fill + wave * 4096u}, sq);
    if (kTurn) {
      wait_lgkm();
      __builtin_amdgcn_s_barrier();
    }
  }
  wait_vm<0>();  // no DMA outlives the block
}

// Tile order: 8 m tiles before the next n tile, so that tiles next to each other share their panels.
__device__ __forceinline__ void order_of(int id, int nm, int nn, int& tm, int& tn) {
  const int gsz = 8 * nn, g = id / gsz, r = id % gsz, gm = nm - g * 8 < 8 ? nm - g * 8 : 8;
  tm = g * 8 + r % gm;
  tn = r / gm;
}

// j-th of the `count` items of this block: each XCD (blocks go to them round robin) works through a contiguous run of
// them, its blocks side by side, so the 32 CUs behind one L2 share what they read. The grid is a multiple of 8. -1: no more.
__device__ __forceinline__ int item_of(int j, int count) {
  const int chunk = (count + 7) / 8, at = (int)(blockIdx.x >> 3) + j * (int)(gridDim.x >> 3);
  const int id = (int)(blockIdx.x & 7) * chunk + at;
  return at < chunk && id < count ? id : -1;
}

}  // namespace ytk
