// Grouped products of few rows (single tokens, small serving batches): bound
// by reading the matrices once.
//
// A workgroup makes 16 columns of 16 MT rows; its waves take K tiles of 128
// bytes in turn and join their sums through LDS. 16 columns a workgroup rather
// than 64 or more: one token's 4096 columns then already make 256 workgroups.
//
// Rows that begin on 16 bytes come through LDS, though nothing is shared: a
// fragment read straight from memory takes 64 bytes of each of 16 rows, and
// such pieces reach 4.2 TB/s here where whole 128-byte lines reach 5.7. Every
// wave has a ring of its own and waits only for its own copies: no barriers.
// Other rows are loaded into registers, from any byte.
#pragma once
#include "grouped_core.h"

#include <algorithm>

// A chunk of 16 bytes from element k on; zeros from klim on.
template <int TY>
__device__ __forceinline__ i32x4 chunk_at(const typename Elt<TY>::T* row,
                                          int k, int klim) {
  constexpr int ES = Elt<TY>::ES, EPC = 16 / ES;
  i32x4 w = {0, 0, 0, 0};
  if (k + EPC <= klim) {
    __builtin_memcpy(&w, row + k, 16);
  } else {
#pragma unroll
    for (int j = 0; j < EPC; ++j)
      if (k + j < klim)
        w[j * ES / 4] |= (int)((u32)row[k + j] << (j * ES % 4 * 8));
  }
  return w;
}

template <int N> struct Count { static constexpr int n = N; };

// ROWS rows of a K tile, copied to LDS by one wave, 1 KB at a time.
template <int ROWS> struct WaveSide {
  static constexpr int N = ROWS / 8;
  u32 at[N];
  static __device__ __forceinline__ int swz(int c, int row) {
    return c ^ (row >> 1 & 7);
  }
  // last: the last row that may be read, from the side's first one
  __device__ __forceinline__ void init(u32 ld_bytes, int last) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = i * 8 + (lane >> 3);
      at[i] = (u32)min(row, last) * ld_bytes + swz(lane & 7, row) * 16;
    }
  }
  template <int COUNT = N>
  __device__ __forceinline__ void copy(const char* tile, char* lds) const {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
      glds16(tile + at[i], lds + (i * 64 + lane) * 16);
  }
  static __device__ __forceinline__ i32x4 chunk(const char* lds, int row,
                                                int c) {
    return *(const i32x4*)(lds + row * 128 + swz(c, row) * 16);
  }
};

template <int TY, int MT, int NB, int W, bool FAST>
__global__ void __launch_bounds__(64 * W) grouped_skinny_k(const GroupedArgs p) {
  constexpr int ES = Elt<TY>::ES, EPC = 16 / ES, BKE = 128 / ES;
  constexpr int U = MT == 1 ? 4 : 2;  // K tiles at a time
  typedef typename Elt<TY>::T E;
  typedef WaveSide<16> SX;
  typedef WaveSide<16 * MT> SY;
  constexpr int SCALES = TY == GT_FP8 ? 256 : 0;
  constexpr int STAGE = 2048 + 16 * MT * 128 + SCALES;
  constexpr int D = 3;  // 4 and 5 stages a wave measured the same
  static_assert((D - 1) * (SX::N + SY::N + 1) < 64, "counted by vmcnt");
  constexpr int RING = FAST ? W * D * STAGE : 0, SUMS = W * NB * MT * 64 * 16;
  __shared__ __attribute__((aligned(16))) char smem[RING > SUMS ? RING : SUMS];
  f32x4 (*sums)[NB * MT][64] = (f32x4 (*)[NB * MT][64])smem;

  const int ntn = (p.N + 16 * NB - 1) / (16 * NB);
  RowTile t;
  if (!find_row_tile<16 * MT>(p, ntn, &t)) return;
  const int g = __builtin_amdgcn_readfirstlane(t.g);
  const int m0 = __builtin_amdgcn_readfirstlane(t.m0);
  const int mend = __builtin_amdgcn_readfirstlane(t.mend);
  const int n0 = __builtin_amdgcn_readfirstlane(t.nt) * (16 * NB);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;

  f32x4 acc[NB][MT];
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[j][i] = f32x4{0, 0, 0, 0};

  if (g < p.E) {
    const E* a[MT];
    int row[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      row[i] = min(m0 + i * 16 + r, mend - 1);
      a[i] = (const E*)p.a + (long)row[i] * p.lda;
    }
    const int tiles = (p.K + BKE - 1) / BKE;
    const float* bsc = nullptr;
    int nb = 0;
    if constexpr (TY == GT_FP8) {
      nb = (p.N + 127) / 128;
      bsc = p.bsc + (long)g * tiles * nb + n0 / 128;
    }
    int first = wave;  // the first tile that registers take
    if constexpr (FAST) {
      SX sx;
      SY sy;
      sx.init((u32)p.ldb * ES, few_rows_row(p.N, n0, 15));
      sy.init((u32)p.lda * ES, mend - 1 - m0);
      const char* xb = (const char*)((const E*)p.b + (long)g * p.gsb +
                                     (long)n0 * p.ldb);
      const char* yb = (const char*)((const E*)p.a + (long)m0 * p.lda);
      char* ring = smem + wave * (D * STAGE);
      const int whole = p.K / BKE;
      const int mine = whole > wave ? (whole - wave + W - 1) / W : 0;
      // the ring runs on over the NB blocks of 16 columns
      const int all = mine * NB;
      int ci = 0, cslot = 0, cblock = 0;
      const char* cx = xb;
      // ny: copies of a's rows a stage; up to 8 rows need the first only (what
      // LDS holds in place of the others makes results that are not stored)
      auto copy = [&](auto ny) {
        const long tile = wave + (long)ci * W;
        const int slot = cslot;
        cslot = cslot == D - 1 ? 0 : cslot + 1;
        char* lds = ring + slot * STAGE;
        if constexpr (SCALES) {  // of the rows; behind them, of the columns
          const float* s = bsc + tile * nb;
          if (lane < 16 * MT)
            s = p.asc + tile * p.T + min(m0 + lane, mend - 1);
          glds4(s, lds + 2048 + 16 * MT * 128 + lane * 4);
        }
        sx.copy(cx + tile * 128, lds);
        sy.template copy<ny.n>(yb + tile * 128, lds + 2048);
        if (++ci == mine) {
          ci = 0;
          if constexpr (NB > 1) {  // the next block, which can end earlier
            const int at = few_rows_block(p.N, n0, ++cblock);
            cx = xb + (long)(at - n0) * p.ldb * ES;
            sx.init((u32)p.ldb * ES, few_rows_row(p.N, at, 15));
          }
        }
      };
      auto product = [&](int slot, f32x4 (&acc)[MT]) {
        const char* lds = ring + slot * STAGE;
        const float* sc = (const float*)(lds + 2048 + 16 * MT * 128);
        i32x4 x[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) x[h] = SX::chunk(lds, r, h * 4 + q);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          i32x4 y[2];
          float sa = 0;
#pragma unroll
          for (int h = 0; h < 2; ++h)
            y[h] = SY::chunk(lds + 2048, i * 16 + r, h * 4 + q);
          if constexpr (TY == GT_FP8) sa = sc[i * 16 + r];
          if constexpr (TY == GT_FP8) {
            const float s = sa * sc[16 * MT];
            const f32x4 d = mma_fp8(join8(x[0], x[1]), join8(y[0], y[1]),
                                    f32x4{0, 0, 0, 0});
#pragma unroll
            for (int j = 0; j < 4; ++j)
              acc[i][j] = __builtin_fmaf(d[j], s, acc[i][j]);
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) acc[i] = mma<TY>(x[h], y[h], acc[i]);
          }
        }
      };
      auto run = [&](auto ny) {
        constexpr int OPS = SX::N + ny.n + (SCALES ? 1 : 0);
        int left = all;  // tiles that are not yet on their way
        for (int i = 0; i < min(D - 1, all); ++i, --left) copy(ny);
        int slot = 0;
#pragma unroll
        for (int j = 0; j < NB; ++j)
          for (int i = 0; i < mine; ++i) {
            if (left > 0) {
              copy(ny);
              --left;
              asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 1) * OPS)
                           : "memory");
            } else {
              asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            product(slot, acc[j]);
            // read to the end, before the slot is copied into
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            slot = slot == D - 1 ? 0 : slot + 1;
          }
      };
      if (MT == 1 && mend - m0 <= 8) run(Count<1>{});
      else run(Count<SY::N>{});
      first = wave + mine * W;  // at most one tile is left, and ends early
    }
    if (first < tiles)
#pragma unroll
    for (int nbk = 0; nbk < NB; ++nbk)
    for (int t0 = first; t0 < tiles; t0 += W * U) {
      const E* b = (const E*)p.b + (long)g * p.gsb +
                   (long)min(n0 + nbk * 16 + r, p.N - 1) * p.ldb;
      i32x4 x[U][2], y[U][MT][2];
      float sa[U][MT], sb[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int tile = t0 + u * W;  // past the end: all zeros
        const int k = tile * BKE;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          x[u][h] = chunk_at<TY>(b, k + (h * 4 + q) * EPC, p.K);
        if constexpr (TY == GT_FP8) sb[u] = tile < tiles ? bsc[(long)tile * nb] : 0;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            y[u][i][h] = chunk_at<TY>(a[i], k + (h * 4 + q) * EPC, p.K);
          if constexpr (TY == GT_FP8)
            sa[u][i] = tile < tiles ? p.asc[(long)tile * p.T + row[i]] : 0;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          if constexpr (TY == GT_FP8) {
            const f32x4 d = mma_fp8(join8(x[u][0], x[u][1]),
                                    join8(y[u][i][0], y[u][i][1]),
                                    f32x4{0, 0, 0, 0});
            const float s = t0 + u * W < tiles ? sa[u][i] * sb[u] : 0;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              acc[nbk][i][j] = __builtin_fmaf(d[j], s, acc[nbk][i][j]);
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              acc[nbk][i] = mma<TY>(x[u][h], y[u][i][h], acc[nbk][i]);
          }
        }
      }
    }
  }

  if constexpr (FAST) __syncthreads();  // the rings are read to the end
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) sums[wave][j * MT + i][lane] = acc[j][i];
  __syncthreads();
  // a wave adds up a 16 x 16 block at a time, in the order of the waves
  const bool vec = p.N % 4 == 0 && (u64)p.c % 16 == 0;
  for (int f = wave; f < NB * MT; f += W) {
    f32x4 sum = sums[0][f][lane];
#pragma unroll
    for (int i = 1; i < W; ++i) sum += sums[i][f][lane];
    const int at = m0 + f % MT * 16 + r, n = n0 + f / MT * 16 + q * 4;
    if (at >= mend || n >= p.N) continue;
    if constexpr (TY == GT_FP8)
      if (zero4(sum) != 0) sum = fp8_again(p, g, at, n, 0, p.K, sum);
    const int have = min(4, p.N - n);
    if (p.accum) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < have) sum[j] += ((const float*)p.c)[(long)at * p.N + n + j];
    }
    store4(p.c, (long)at * p.N + n, p.out, sum, have, vec);
  }
}

template <int TY, int MT, int NB>
static void grouped_skinny_nb(const GroupedArgs& p, bool fast, bool eight,
                              hipStream_t s) {
  const long wgs =
      grouped_row_tiles(p, 16 * MT) * ((p.N + 16 * NB - 1) / (16 * NB));
#define GO(W, FAST)                                                         \
  hipLaunchKernelGGL((grouped_skinny_k<TY, MT, NB, W, FAST>),          \
                     dim3((unsigned)wgs), dim3(64 * W), 0, s, p)
  if constexpr (NB == 1)
    if (eight) {
      if (fast) GO(8, true);
      else GO(8, false);
      return;
    }
  if (fast) GO(4, true);
  else GO(4, false);
#undef GO
}

// Blocks of 16 columns a workgroup, by how many blocks there are: a workgroup
// costs about 2 us beside its reading, but the chip has to be filled. bf16,
// 64 rows in 8 groups of 4096 x 4096 (12 x 256 by this count), 1 / 2 / 4
// blocks: 73 / 52 / 61 us; one row, 4096 x 4096 (256): 8.5 / 11.1 / 15.3 us;
// fp8, 64 rows in 32 groups of 4096 x 2048 (9216): 43 / 34 / 31 us. With few
// blocks and a long sum, eight waves share it instead of four.
template <int TY, int MT>
static void grouped_skinny_go(const GroupedArgs& p, bool fast,
                              hipStream_t s) {
  const long blocks =
      ((long)p.T / (16 * MT) + std::min(p.E, p.T)) * ((p.N + 15) / 16);
  const int tiles = (p.K + 128 / Elt<TY>::ES - 1) / (128 / Elt<TY>::ES);
  if (blocks >= 8192)
    grouped_skinny_nb<TY, MT, 4>(p, fast, false, s);
  else if (blocks >= 512)
    grouped_skinny_nb<TY, MT, 2>(p, fast, false, s);
  else
    grouped_skinny_nb<TY, MT, 1>(p, fast, tiles >= 64 && blocks <= 256,
                                      s);
}
