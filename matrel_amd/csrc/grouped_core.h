// Matrix products of many row groups in one launch (gfx950).
//
//   rows:    C[t, n] = sum_k A[t, k] * B[g(t)](n, k)      t in group g(t)
//   weights: C[g][m, n] = sum_{t in group g} A[t, m] * B[t, n]
//
// Group g is the rows [offs[g], offs[g + 1]); the offsets stay on the device,
// so a launch covers the most tiles that T rows in E groups can make and every
// workgroup finds its own tile from the offsets by a wave-wide prefix sum.
// Rows in no group (before offs[0], behind offs[E]) count as two more groups
// with an empty sum: their outputs are zeros.
//
// All types share one tile shape in bytes: a K tile is 128 bytes of a row
// (128 e4m3, 64 bf16/fp16, 32 f32), cut into 16-byte chunks. An operand lies in
// memory either with k along its rows ("K" side: the chunk holds consecutive
// k of one row) or with rows along its k ("R" side: the chunk holds
// consecutive rows at one k). Both are copied to LDS as they lie, 16 bytes a
// lane, with the chunk index XOR-swizzled so that fragment reads meet no bank
// twice: the K side is read by ds_read_b128, the R side by the transposing
// ds_read_b64_tr_b16 (16-bit types) or by single words (f32).
//
// The right operand is the matrix instruction's first one, so that a lane's
// four results are four neighbouring n of one row: stores are vectors, and a
// scale of a row is one register.
#pragma once
#include "common.h"
#include "grouped_args.h"

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// ---- arithmetic by type ----------------------------------------------------

template <int TY> struct Elt;
template <> struct Elt<GT_BF16> { typedef unsigned short T; enum { ES = 2 }; };
template <> struct Elt<GT_F16> { typedef unsigned short T; enum { ES = 2 }; };
template <> struct Elt<GT_F32> { typedef unsigned int T; enum { ES = 4 }; };
template <> struct Elt<GT_FP8> { typedef unsigned char T; enum { ES = 1 }; };

// One 16-byte chunk of each operand: 8 products deep in 16 bits, 4 in f32.
template <int TY>
__device__ __forceinline__ f32x4 mma(i32x4 x, i32x4 y, f32x4 c) {
  if constexpr (TY == GT_BF16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
        __builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0,
        0);
  } else if constexpr (TY == GT_F16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(
        __builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0,
        0);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__int_as_float(x[i]),
                                               __int_as_float(y[i]), c, 0, 0,
                                               0);
    return c;
  }
}

// e4m3, 128 products deep, no hardware scale: both operands take any order
// of k that is the same for the two.
__device__ __forceinline__ f32x4 mma_fp8(i32x8 x, i32x8 y, f32x4 c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 0, 0, 0, 0,
                                                          0, 0);
}

__device__ __forceinline__ i32x8 join8(i32x4 lo, i32x4 hi) {
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

__device__ __forceinline__ unsigned short f32_to_bits16(float x, int ty) {
  // to nearest, ties to even: the one rounding of a 16-bit result
  if (ty == GT_BF16) return __builtin_bit_cast(unsigned short, (__bf16)x);
  return __builtin_bit_cast(unsigned short, (_Float16)x);
}

// Four neighbouring results of one row; `have` of them lie inside.
__device__ __forceinline__ void store4(void* base, long at, int ty, f32x4 v,
                                       int have, bool vec) {
  if (ty == GT_F32) {
    float* o = (float*)base + at;
    if (vec && have == 4) {
      *(f32x4*)o = v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < have) o[i] = v[i];
    }
  } else {
    unsigned short* o = (unsigned short*)base + at;
    unsigned short q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = f32_to_bits16(v[i], ty);
    if (vec && have == 4) {
      *(uint2*)o = make_uint2(q[0] | (u32)q[1] << 16, q[2] | (u32)q[3] << 16);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < have) o[i] = q[i];
    }
  }
}

// ---- groups ----------------------------------------------------------------

// The i-th boundary of the E + 2 row ranges (head, groups, tail). Offsets are
// held to [0, T] and each range to a length of zero or more, so that offsets
// which break their order still address nothing outside.
__device__ __forceinline__ int bound_at(const GroupedArgs& p, int i) {
  if (i <= 0) return 0;
  if (i > p.E + 1) return p.T;
  if (!p.offs) return i == 1 ? 0 : p.T;
  long v = p.off64 ? ((const long*)p.offs)[i - 1]
                   : (long)((const int*)p.offs)[i - 1];
  return (int)(v < 0 ? 0 : v > p.T ? p.T : v);
}

struct RowTile {
  int g;     // group, -1 or E: rows of no group
  int m0;    // first row
  int mend;  // end of the group's rows
  int nt;    // tile along n
};

// Tile `id` of the tiles of all ranges, each cut into BM rows x ntn tiles.
// Neighbouring ids are kept within an 8-row-tile wide band of one group, so
// that the workgroups of one XCD share both operands in its L2.
template <int BM>
__device__ __forceinline__ bool find_row_tile(const GroupedArgs& p, int ntn,
                                              RowTile* out) {
  const int lane = threadIdx.x & 63;
  const int nv = p.E + 2;
  int total = 0, inc = 0, cnt = 0, lo = 0, hi = 0;
  auto scan = [&](int base) {
    const int v = base + lane;
    lo = hi = 0;
    if (v < nv) {
      lo = bound_at(p, v);
      hi = bound_at(p, v + 1);
      if (hi < lo) hi = lo;
    }
    cnt = (hi - lo + BM - 1) / BM * ntn;
    inc = cnt;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      int t = __shfl_up(inc, d);
      if (lane >= d) inc += t;
    }
  };
  for (int base = 0; base < nv; base += 64) {
    scan(base);
    total += __shfl(inc, 63);
  }
  if ((int)blockIdx.x >= total) return false;
  const int id = (int)xcd_swizzle(blockIdx.x, (u32)total);
  int before = 0;
  for (int base = 0; base < nv; base += 64) {
    if (nv > 64) scan(base);  // one step's sums are still at hand
    const u64 m = __ballot(before + inc > id);
    if (m) {
      const int at = __ffsll((unsigned long long)m) - 1;
      const int first = before + __shfl(inc, at) - __shfl(cnt, at);
      const int s = __shfl(lo, at), e = __shfl(hi, at);
      const int rem = id - first, mtc = (e - s + BM - 1) / BM;
      const int band = rem / (8 * ntn), r = rem - band * 8 * ntn;
      const int wide = min(8, mtc - band * 8);
      out->g = base + at - 1;
      out->m0 = s + (band * 8 + r % wide) * BM;
      out->mend = e;
      out->nt = r / wide;
      return true;
    }
    before += __shfl(inc, 63);
  }
  return false;
}

// ---- operands --------------------------------------------------------------

// An operand's tile of R rows x 128 bytes of k in LDS, filled by NT threads.
template <int TY, int R, int NT, bool KROWS>
struct Side {
  typedef typename Elt<TY>::T E;
  static constexpr int ES = Elt<TY>::ES;
  static constexpr int EPC = 16 / ES;          // elements of a chunk
  static constexpr int BKE = 128 / ES;         // k of a tile
  static constexpr int IT = R * 8 / NT;        // chunks of a thread
  static constexpr int CPR = R * ES / 16;      // R side: chunks of one k
  static_assert(R * 8 % NT == 0, "whole chunks for every thread");

  const char* at[IT];  // where this thread's chunks of the first tile begin
  const E* base;
  long ld;
  int row0, rlim, k0;

  // R side, swizzled chunk c at k <-> the chunk as it lies in memory.
  // 16 bits: the 16 lanes of a transposing read take 32 bytes at each of 4 k,
  // and 4 such groups run at once (k = 8g + j): 32-byte slots are permuted by
  // j and g's low bit. f32: 64-byte slots by k / 4.
  static __device__ __forceinline__ int swz(int c, int k) {
    if constexpr (ES == 2) {
      return c ^ (((k & 3) | (k >> 3 & 1) << 2) << 1);
    } else {
      return c ^ (k >> 2 & 3) << 2;
    }
  }

  // Rows [row0, row0 + R) of which those below rlim exist (at least one).
  __device__ __forceinline__ void init(const void* b, long ld_, int row0_,
                                       int rlim_, int k0_, bool fast) {
    base = (const E*)b;
    ld = ld_;
    row0 = row0_;
    rlim = rlim_;
    k0 = k0_;
    if (!fast) return;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int id = i * NT + (int)threadIdx.x;
      long e;
      if constexpr (KROWS) {
        const int row = id >> 3, c = (id & 7) ^ (row >> 1 & 7);
        e = (long)min(row0 + row, rlim - 1) * ld + k0 + c * EPC;
      } else {
        const int k = id / CPR, c = swz(id % CPR, k);
        e = (long)(k0 + k) * ld + min(row0 + c * EPC, rlim - EPC);
      }
      at[i] = (const char*)base + e * ES;
    }
  }

  // Whole tiles of operands whose rows begin on 16 bytes: straight to LDS.
  // A row (R side: a chunk of rows) past the end reads the last one again;
  // what it makes is never stored.
  __device__ __forceinline__ void copy(char* lds, int tile) const {
    const long step = (long)tile * (KROWS ? 128 : (long)BKE * ld * ES);
#pragma unroll
    for (int i = 0; i < IT; ++i)
      glds16(at[i] + step, lds + (i * NT + threadIdx.x) * 16);
  }

  // Any tile: through registers, zeros outside of the rows and of k < klim.
  __device__ __forceinline__ void gather(char* lds, int tile, int klim,
                                         bool aligned) const {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int id = i * NT + (int)threadIdx.x;
      E v[EPC];
#pragma unroll
      for (int j = 0; j < EPC; ++j) v[j] = 0;
      i32x4 w = {0, 0, 0, 0};
      bool whole = false;
      if constexpr (KROWS) {
        const int row = row0 + (id >> 3);
        const int k = k0 + tile * BKE + ((id & 7) ^ ((id >> 3) >> 1 & 7)) * EPC;
        const E* s = base + (long)row * ld + k;
        if (row < rlim && k < klim) {
          if (aligned && k + EPC <= klim) {
            w = *(const i32x4*)s;
            whole = true;
          } else {
#pragma unroll
            for (int j = 0; j < EPC; ++j)
              if (k + j < klim) v[j] = s[j];
          }
        }
      } else {
        const int kk = id / CPR, k = k0 + tile * BKE + kk;
        const int row = row0 + swz(id % CPR, kk) * EPC;
        const E* s = base + (long)k * ld + row;
        if (k < klim && row < rlim) {
          if (aligned && row + EPC <= rlim) {
            w = *(const i32x4*)s;
            whole = true;
          } else {
#pragma unroll
            for (int j = 0; j < EPC; ++j)
              if (row + j < rlim) v[j] = s[j];
          }
        }
      }
      if (!whole) {
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          u32 x = 0;
#pragma unroll
          for (int j = 0; j < 4 / ES; ++j)
            x |= (u32)v[d * (4 / ES) + j] << (8 * ES * j);
          w[d] = (int)x;
        }
      }
      *(i32x4*)(lds + id * 16) = w;
    }
  }

  // The chunk of the fragment of rows [row, row + 16) (row: a multiple of 16)
  // in half kk of the tile: lane l holds row l & 15, its k group l >> 4.
  static __device__ __forceinline__ i32x4 frag(const char* lds, int row,
                                               int kk) {
    const int l = threadIdx.x & 63, r = l & 15, g = l >> 4;
    if constexpr (KROWS) {
      const int rr = row + r;
      return *(const i32x4*)(lds + rr * 128 +
                             (((kk * 4 + g) ^ (r >> 1)) << 4));
    } else if constexpr (ES == 2) {
      i32x4 out;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = kk * 32 + g * 8 + h * 4 + (r >> 2);
        const int c = swz(row / 8 + (r >> 1 & 1), k);
        const char* s = lds + k * (R * 2) + c * 16 + (r & 1) * 8;
        const i16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) i16x4*)s);
        const int2 d = __builtin_bit_cast(int2, v);
        out[2 * h] = d.x;
        out[2 * h + 1] = d.y;
      }
      return out;
    } else {
      i32x4 out;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = kk * 16 + g * 4 + i;
        const int c = swz((row + r) >> 2, k);
        out[i] = *(const int*)(lds + k * (R * 4) + c * 16 + (r & 3) * 4);
      }
      return out;
    }
  }
};

// ---- the kernel ------------------------------------------------------------

// BM x BN results a workgroup, its waves WM x WN. AK/BK: the operand has k
// along its rows. WEIGHTS: the sum runs over a group's rows. FAST: rows (and
// for an R side its length) are multiples of 16 bytes.
//
// Two LDS buffers: the copy of the next K tile runs under the products of
// this one, with one barrier a tile.
template <int TY, int BM, int BN, int WM, int WN, bool AK, bool BK,
          bool WEIGHTS, bool FAST>
__global__ void __launch_bounds__(64 * WM * WN)
grouped_k(const GroupedArgs p) {
  constexpr int NT = 64 * WM * WN;
  constexpr int ES = Elt<TY>::ES, BKE = 128 / ES;
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  typedef Side<TY, BM, NT, AK> SA;
  typedef Side<TY, BN, NT, BK> SB;
  constexpr int BUF = (BM + BN) * 128;
  extern __shared__ __attribute__((aligned(16))) char smem[];

  const int ntn = (p.N + BN - 1) / BN;
  int g, m0, mend, n0, kbeg, kend;
  if constexpr (WEIGHTS) {
    const int ntm = (p.M + BM - 1) / BM;
    const int id = (int)xcd_swizzle(blockIdx.x, gridDim.x);
    g = id / (ntm * ntn);
    const int rem = id - g * ntm * ntn;
    const int band = rem / (8 * ntn), r = rem - band * 8 * ntn;
    const int wide = min(8, ntm - band * 8);
    m0 = (band * 8 + r % wide) * BM;
    n0 = r / wide * BN;
    mend = p.M;
    kbeg = bound_at(p, g + 1);
    kend = max(kbeg, bound_at(p, g + 2));
  } else {
    RowTile t;
    if (!find_row_tile<BM>(p, ntn, &t)) return;
    g = t.g;
    m0 = t.m0;
    mend = t.mend;
    n0 = t.nt * BN;
    kbeg = 0;
    kend = g < 0 || g >= p.E ? 0 : p.K;
  }
  const int split = blockIdx.y;
  if (p.splits > 1) {  // an equal share of whole K tiles for each
    const int tiles = (kend - kbeg + BKE - 1) / BKE;
    const int share = (tiles + p.splits - 1) / p.splits;
    const int lo = min(kend, kbeg + split * share * BKE);
    kend = min(kend, lo + share * BKE);
    kbeg = lo;
  }

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);

  f32x4 acc[FN][FM];
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int i = 0; i < FM; ++i) acc[j][i] = f32x4{0, 0, 0, 0};

  SA sa;
  SB sb;
  const int depth = kend - kbeg;
  const int whole = depth / BKE, tiles = (depth + BKE - 1) / BKE;

  const float* asc = nullptr;
  const float* bsc = nullptr;
  int nb = 0;
  if constexpr (TY == GT_FP8) {
    nb = (p.N + 127) / 128;
    asc = p.asc + (long)(kbeg / 128) * p.T;
    bsc = p.bsc + ((long)g * ((p.K + 127) / 128) + kbeg / 128) * nb +
          (n0 + wn) / 128;
    if (n0 + wn >= p.N) bsc = p.bsc;  // a wave past the end: stores nothing
  }

  auto products = [&](const char* lds, int tile) {
    const char* la = lds;
    const char* lb = lds + BM * 128;
    if constexpr (TY == GT_FP8) {
      // a K tile is one block of scales: its products are summed apart and
      // join the f32 sum with one multiply-add
      const float s = bsc[(long)tile * nb];
      float sc[FM];
      i32x8 y[FM];
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int row = min(m0 + wm + i * 16 + (lane & 15), p.T - 1);
        sc[i] = asc[(long)tile * p.T + row] * s;
        y[i] = join8(SA::frag(la, wm + i * 16, 0),
                     SA::frag(la, wm + i * 16, 1));
      }
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const i32x8 x = join8(SB::frag(lb, wn + j * 16, 0),
                              SB::frag(lb, wn + j * 16, 1));
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          const f32x4 d = mma_fp8(x, y[i], f32x4{0, 0, 0, 0});
#pragma unroll
          for (int q = 0; q < 4; ++q)
            acc[j][i][q] = __builtin_fmaf(d[q], sc[i], acc[j][i][q]);
        }
      }
    } else {
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        i32x4 y[FM];
#pragma unroll
        for (int i = 0; i < FM; ++i) y[i] = SA::frag(la, wm + i * 16, kk);
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const i32x4 x = SB::frag(lb, wn + j * 16, kk);
#pragma unroll
          for (int i = 0; i < FM; ++i)
            acc[j][i] = mma<TY>(x, y[i], acc[j][i]);
        }
      }
    }
  };

  if (tiles > 0) {
    const char* bbase = (const char*)p.b +
                        (WEIGHTS ? 0 : (long)g * p.gsb * ES);
    sa.init(p.a, p.lda, m0, mend, kbeg, FAST && whole > 0);
    sb.init(bbase, p.ldb, n0, p.N, kbeg, FAST && whole > 0);
    auto fill = [&](int tile) {
      char* lds = smem + (tile & 1) * BUF;
      if (FAST && tile < whole) {
        sa.copy(lds, tile);
        sb.copy(lds + BM * 128, tile);
      } else {
        sa.gather(lds, tile, kend, FAST);
        sb.gather(lds + BM * 128, tile, kend, FAST);
      }
    };
    fill(0);
    for (int t = 0; t < tiles; ++t) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (t + 1 < tiles) fill(t + 1);
      products(smem + (t & 1) * BUF, t);
    }
  }

  // results: lane l holds row l & 15, columns 4 (l >> 4) + 0..3
  const long rows = WEIGHTS ? (long)p.E * p.M : p.T;
  const long first = WEIGHTS ? (long)g * p.M : 0;
  void* c = p.part ? (void*)(p.part + split * rows * p.N) : p.c;
  const int ty = p.part ? (int)GT_F32 : p.out;
  const bool vec = p.N % 4 == 0 && (u64)c % 16 == 0;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int row = m0 + wm + i * 16 + (lane & 15);
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = n0 + wn + j * 16 + (lane >> 4) * 4;
      if (row < mend && n < p.N) {
        const long at = (first + row) * p.N + n;
        const int have = min(4, p.N - n);
        f32x4 v = acc[j][i];
        if (p.accum) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (q < have) v[q] += ((const float*)c)[at + q];
        }
        store4(c, at, ty, v, have, vec);
      }
    }
  }
}
