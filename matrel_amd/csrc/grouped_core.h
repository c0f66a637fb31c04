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
// of k that is the same for the two, by 8 neighbours.
//
// The unit adds the products of 8 neighbours with 13 bits behind the largest
// one's power of two (what is smaller is cut off) and these sums in f32: up to
// 7 * 2^-13 of the largest product of a group, where its operands are off by
// 2^-4. The 32-deep instruction does the same and takes 1.4 times as long
// (16384 x 8192 x 8192: 1403 against 1013 us); 16-bit instructions have half
// the rate. It is the rounding that 8-bit speed costs here.
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
  int g;     // group, E or more: rows of no group
  int m0;    // first row
  int mend;  // end of the group's rows
  int nt;    // tile along n
};

// Inclusive prefix sum over the wave.
__device__ __forceinline__ int wave_sum(int x) {
#define STEP(ctrl, rows) \
  x += __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xf, false)
  STEP(0x111, 0xf);  // from 1, 2, 4, 8 lanes before, within 16
  STEP(0x112, 0xf);
  STEP(0x114, 0xf);
  STEP(0x118, 0xf);
  STEP(0x142, 0xa);  // lane 15 to the next 16, lane 31 to the next 32
  STEP(0x143, 0xc);
#undef STEP
  return x;
}

// Tile `id` of the tiles of all ranges, each cut into BM rows x ntn tiles:
// the groups', then those of the head and the tail. Neighbouring ids are kept
// within an 8-row-tile wide band of one group, so that the workgroups of one
// XCD share both operands in its L2.
template <int BM>
__device__ __forceinline__ bool find_row_tile(const GroupedArgs& p, int ntn,
                                              RowTile* out) {
  const int lane = threadIdx.x & 63;
  int inc = 0, cnt = 0, lo = 0, hi = 0;
  auto scan = [&](int base) {  // groups, or (E, E + 1): head and tail
    const int v = base + lane;
    lo = hi = 0;
    if (v < p.E) {
      lo = bound_at(p, v + 1);
      hi = bound_at(p, v + 2);
    } else if (v < p.E + 2) {
      lo = v == p.E ? 0 : bound_at(p, p.E + 1);
      hi = v == p.E ? bound_at(p, 1) : p.T;
    }
    if (hi < lo) hi = lo;
    cnt = (hi - lo + BM - 1) / BM * ntn;
    inc = wave_sum(cnt);
  };
  const int nv = p.E + 2;
  int total = 0;
  for (int base = 0; base < nv; base += 64) {
    scan(base);
    total += __builtin_amdgcn_readlane(inc, 63);
  }
  if ((int)blockIdx.x >= total) return false;
  const int id = (int)xcd_swizzle(blockIdx.x, (u32)total);
  int before = 0;
  for (int base = 0; base < nv; base += 64) {
    if (nv > 64) scan(base);  // one step's sums are still at hand
    const u64 m = __ballot(before + inc > id);
    if (m) {
      const int at = __ffsll((unsigned long long)m) - 1;
      const int first = before + __builtin_amdgcn_readlane(inc, at) -
                        __builtin_amdgcn_readlane(cnt, at);
      const int s = __builtin_amdgcn_readlane(lo, at);
      const int e = __builtin_amdgcn_readlane(hi, at);
      const int rem = id - first, mtc = (e - s + BM - 1) / BM;
      const int band = rem / (8 * ntn), r = rem - band * 8 * ntn;
      const int wide = min(8, mtc - band * 8);
      out->g = base + at;
      out->m0 = s + (band * 8 + r % wide) * BM;
      out->mend = e;
      out->nt = r / wide;
      return true;
    }
    before += __builtin_amdgcn_readlane(inc, 63);
  }
  return false;
}

// The group with the n-th longest range and that range, for up to 64 groups:
// long sums begin first and short ones fill what they leave (f32, 8192 rows
// in 4 uneven groups, 2048 x 2048: 1061 -> 503 us). It takes a microsecond,
// which sums over few rows do not repay.
__device__ __forceinline__ void by_length(const GroupedArgs& p, int n,
                                          int* g, int* lo, int* hi) {
  const int lane = threadIdx.x & 63;
  const int a = bound_at(p, lane + 1), b = max(a, bound_at(p, lane + 2));
  const int len = lane < p.E ? b - a : -1;
  int rank = 0;
  for (int j = 0; j < p.E; ++j) {
    const int other = __builtin_amdgcn_readlane(len, j);
    rank += other > len || (other == len && j < lane);
  }
  const int at =
      __ffsll((unsigned long long)__ballot(rank == n && lane < p.E)) - 1;
  *g = at;
  *lo = __builtin_amdgcn_readlane(a, at);
  *hi = __builtin_amdgcn_readlane(b, at);
}

// ---- operands --------------------------------------------------------------

// An operand's tile of R rows x 128 bytes of k in LDS, filled by NT threads.
template <int TY, int R, int NT, bool KROWS>
struct Side {
  typedef typename Elt<TY>::T E;
  typedef i32x4 Regs[R * 8 / NT];
  static constexpr int ES = Elt<TY>::ES;
  static constexpr int EPC = 16 / ES;          // elements of a chunk
  static constexpr int BKE = 128 / ES;         // k of a tile
  static constexpr int IT = R * 8 / NT;        // chunks of a thread
  static constexpr int CPR = R * ES / 16;      // R side: chunks of one k
  static_assert(R * 8 % NT == 0, "whole chunks for every thread");

  int at[IT];        // this thread's chunks of a tile, bytes from `base`
  const char* base;  // the operand's first row (R side: column) and k
  long ld;
  int row0, rlim, k0;

  // R side, swizzled chunk c at k <-> the chunk as it lies in memory.
  // 16 bits: the 16 lanes of a transposing read take 32 bytes at each of 4 k,
  // and 4 such groups run at once (k = 8g + j): 32-byte slots are permuted by
  // j and g's low bit; of 64 rows two k share the 256 bytes of all banks, and
  // there are 4 slots. f32: 64-byte slots by k / 4.
  static_assert(KROWS || R >= 64, "R side: at least 4 slots");
  static __device__ __forceinline__ int swz(int c, int k) {
    if constexpr (ES == 2 && R == 64) {
      return c ^ ((k >> 1 & 1) | (k >> 3 & 1) << 1) << 1;
    } else if constexpr (ES == 2) {
      return c ^ (((k & 3) | (k >> 3 & 1) << 2) << 1);
    } else {
      return c ^ (k >> 2 & 3) << 2;
    }
  }

  // Rows [row0, row0 + R), of which those below rlim exist (at least one),
  // from k0 on. A row (R side: a chunk of rows) past the end reads the last
  // one again; what it makes is never stored.
  __device__ __forceinline__ void init(const void* b, long ld_, int row0_,
                                       int rlim_, int k0_) {
    ld = ld_;
    row0 = row0_;
    rlim = rlim_;
    k0 = k0_;
    base = (const char*)b +
           (KROWS ? (long)row0 * ld + k0 : (long)k0 * ld + row0) * ES;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int id = i * NT + (int)threadIdx.x;
      if constexpr (KROWS) {
        const int row = id >> 3, c = (id & 7) ^ (row >> 1 & 7);
        at[i] = min(row, rlim - 1 - row0) * (int)ld * ES + c * 16;
      } else {
        const int k = id / CPR, c = swz(id % CPR, k);
        // below zero where the last tile is narrower than a chunk
        at[i] = k * (int)ld * ES + min(c * EPC, rlim - EPC - row0) * ES;
      }
    }
  }

  // Whole tiles of operands whose rows begin on 16 bytes: straight to LDS.
  // `lds`: an offset from smem.
  __device__ __forceinline__ void copy(char* smem, u32 lds, int tile) const {
    const char* s = base + (long)tile * (KROWS ? 128 : (long)BKE * ld * ES);
    if constexpr (ES != 1) {
      const u64 v = (u64)s;
      s = (const char*)((u64)(u32)__builtin_amdgcn_readfirstlane((u32)v) |
                        (u64)(u32)__builtin_amdgcn_readfirstlane(
                            (u32)(v >> 32)) << 32);
    }
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      if constexpr (ES == 1) {
        glds16(s + at[i], smem + lds + (i * NT + threadIdx.x) * 16);
      } else {
        // the same instruction by hand: the compiler, which knows these
        // copies, waits for all of them before each transposing read. What it
        // writes to LDS is not declared for that reason: every read of it
        // stands behind a wait for its count that clobbers memory
        const u32 to = __builtin_amdgcn_readfirstlane(
            (u32)(uintptr_t)(__attribute__((address_space(3))) char*)smem +
            lds + (i * NT + (threadIdx.x & ~63u)) * 16);
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\t"
                     "global_load_lds_dwordx4 %0, %1"
                     :: "v"(at[i]), "s"(s), "s"(to) : "m0");
      }
    }
  }

  // Any tile, any alignment: through registers. Nothing in load() depends on
  // what it loads or branches, so that loads stay on their way: a chunk that
  // ends early is read from further in front, and put() shifts it.
  __device__ __forceinline__ void load(i32x4 (&w)[IT], int tile,
                                       int klim) const {
    const int k1 = klim - k0 - tile * BKE;  // k of the tile that exist
    const char* s = base + (long)tile * (KROWS ? 128 : (long)BKE * ld * ES);
#pragma unroll
    for (int i = 0; i < IT; ++i)  // global loads need no alignment
      __builtin_memcpy(&w[i], s + ((long)at[i] - back(i, k1)), 16);
  }

  __device__ __forceinline__ int back(int i, int k1) const {
    const int id = i * NT + (int)threadIdx.x;
    if constexpr (KROWS)
      return max(0, (((id & 7) ^ (id >> 4 & 7)) + 1) * EPC - k1) * ES;
    else
      return max(0, id / CPR + 1 - k1) * (int)ld * ES;
  }

  // Zeros for k >= klim. PARTS: the last chunk of an R side's rows may be a
  // part of one.
  template <bool PARTS>
  __device__ __forceinline__ void put(char* lds, i32x4 (&w)[IT], int tile,
                                      int klim) const {
    const int k1 = klim - k0 - tile * BKE;
    if (k1 < BKE) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        if constexpr (KROWS) w[i] = shifted(w[i], back(i, k1));
        else if ((i * NT + (int)threadIdx.x) / CPR >= k1)
          w[i] = i32x4{0, 0, 0, 0};
      }
    }
    if constexpr (!KROWS && PARTS) {
      if (row0 + R > rlim) {
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const int id = i * NT + (int)threadIdx.x;
          const int c = swz(id % CPR, id / CPR) * EPC;
          w[i] = shifted(w[i], max(0, c - (rlim - EPC - row0)) * ES);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < IT; ++i)
      *(i32x4*)(lds + (i * NT + threadIdx.x) * 16) = w[i];
  }

  // The chunk without its first n bytes, zeros behind.
  static __device__ __forceinline__ i32x4 shifted(i32x4 v, int n) {
    u64 lo = (u32)v[0] | (u64)(u32)v[1] << 32;
    u64 hi = (u32)v[2] | (u64)(u32)v[3] << 32;
    if (n >= 16) lo = hi = 0;
    if (n >= 8) {
      lo = hi;
      hi = 0;
      n -= 8;
    }
    if (n > 0 && n < 8) {
      lo = lo >> 8 * n | hi << (64 - 8 * n);
      hi >>= 8 * n;
    }
    return i32x4{(int)lo, (int)(lo >> 32), (int)hi, (int)(hi >> 32)};
  }

  // Rows shorter than a chunk or further apart than 31 bits: element by
  // element, straight to LDS.
  __device__ __forceinline__ void gather(char* lds, int tile, int klim) const {
#pragma unroll 1
    for (int id = threadIdx.x; id < IT * NT; id += NT) {
      int n;  // elements of the chunk that exist
      const E* s;
      if constexpr (KROWS) {
        const int row = id >> 3;
        const int k = tile * BKE + ((id & 7) ^ (row >> 1 & 7)) * EPC;
        n = row0 + row < rlim ? klim - k0 - k : 0;
        s = (const E*)base + (long)row * ld + k;
      } else {
        const int k = tile * BKE + id / CPR;
        const int row = swz(id % CPR, id / CPR) * EPC;
        n = k0 + k < klim ? rlim - row0 - row : 0;
        s = (const E*)base + (long)k * ld + row;
      }
#pragma unroll 1
      for (int j = 0; j < EPC; ++j)
        ((E*)(lds + id * 16))[j] = j < n ? s[j] : (E)0;
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

// ---- what a workgroup computes ---------------------------------------------

struct Work {
  int g;           // group (rows: E or more for rows of no group)
  int m0, mend;    // first row and the end of the rows
  int n0;
  int kbeg, kend;  // what is summed
};

template <int TY, int BM, int BN, bool WEIGHTS>
__device__ __forceinline__ bool locate(const GroupedArgs& p, Work* w) {
  constexpr int BKE = 128 / Elt<TY>::ES;
  const int ntn = (p.N + BN - 1) / BN;
  if constexpr (WEIGHTS) {
    // every XCD takes a share of every group: groups differ in length
    const int ntm = (p.M + BM - 1) / BM, per = ntm * ntn;
    w->g = blockIdx.x / per;
    const int rem = (int)xcd_swizzle(blockIdx.x - w->g * per, per);
    if (p.E > 1 && p.E <= 64 && p.T >= 256 * p.E) {
      by_length(p, w->g, &w->g, &w->kbeg, &w->kend);
    } else {
      w->kbeg = bound_at(p, w->g + 1);
      w->kend = max(w->kbeg, bound_at(p, w->g + 2));
    }
    const int band = rem / (8 * ntn), r = rem - band * 8 * ntn;
    const int wide = min(8, ntm - band * 8);
    w->m0 = (band * 8 + r % wide) * BM;
    w->n0 = r / wide * BN;
    w->mend = p.M;
  } else {
    RowTile t;
    if (!find_row_tile<BM>(p, ntn, &t)) return false;
    w->g = t.g;
    w->m0 = t.m0;
    w->mend = t.mend;
    w->n0 = t.nt * BN;
    w->kbeg = 0;
    w->kend = t.g >= p.E ? 0 : p.K;
  }
  if (p.splits > 1) {  // an equal share of whole K tiles for each
    const int tiles = (w->kend - w->kbeg + BKE - 1) / BKE;
    const int share = (tiles + p.splits - 1) / p.splits;
    const int lo = min(w->kend, w->kbeg + (int)blockIdx.y * share * BKE);
    w->kend = min(w->kend, lo + share * BKE);
    w->kbeg = lo;
  }
  // the same for all lanes, which only their owner can know
  w->g = __builtin_amdgcn_readfirstlane(w->g);
  w->m0 = __builtin_amdgcn_readfirstlane(w->m0);
  w->mend = __builtin_amdgcn_readfirstlane(w->mend);
  w->n0 = __builtin_amdgcn_readfirstlane(w->n0);
  w->kbeg = __builtin_amdgcn_readfirstlane(w->kbeg);
  w->kend = __builtin_amdgcn_readfirstlane(w->kend);
  return true;
}

// Where results go. A lane holds four neighbouring n of one row.
template <bool WEIGHTS> struct Results {
  void* c;
  int ty;
  bool vec, accum;
  long first;
  int mend, n;

  __device__ __forceinline__ Results(const GroupedArgs& p, const Work& w) {
    const long rows = WEIGHTS ? (long)p.E * p.M : p.T;
    c = p.part ? (void*)(p.part + blockIdx.y * rows * p.N) : p.c;
    ty = p.part ? (int)GT_F32 : p.out;
    vec = p.N % 4 == 0 && (u64)c % 16 == 0;
    accum = p.accum;
    first = WEIGHTS ? (long)w.g * p.M : 0;
    mend = w.mend;
    n = p.N;
  }

  // A 16 x 16 fragment at (row, col): lane l has row l & 15 and columns
  // 4 (l >> 4) + 0..3.
  __device__ __forceinline__ void put(int row, int col, f32x4 v) const {
    const int lane = threadIdx.x & 63;
    row += lane & 15;
    col += (lane >> 4) * 4;
    if (row >= mend || col >= n) return;
    const long at = (first + row) * n + col;
    const int have = min(4, n - col);
    if (accum) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (q < have) v[q] += ((const float*)c)[at + q];
    }
    store4(c, at, ty, v, have, vec);
  }
};

// ---- scales whose product overflows -----------------------------------------

// Zero where all four are finite, else NaN.
__device__ __forceinline__ float zero4(f32x4 v) {
  return (v[0] - v[0]) + (v[1] - v[1]) + (v[2] - v[2]) + (v[3] - v[3]);
}

// fp8: a lane's four sums over [kbeg, kend) at (row, col). A block pair whose
// scales are finite and their product is not makes infinities, or NaN of a
// payload sum of 0, where the values' own products can be finite. Such sums
// are taken again, one value at a time, each scaled before it is multiplied.
// Where all results are finite this costs two operations each.
__device__ __forceinline__ f32x4 fp8_again(const GroupedArgs& p, int g,
                                           int row, int col, int kbeg,
                                           int kend, f32x4 v) {
  const int nb = (p.N + 127) / 128, kbs = (p.K + 127) / 128;
  const float* xs = p.asc + row;
  const float* ys = p.bsc + (long)g * kbs * nb + col / 128;
  bool over = false;
#pragma unroll 1
  for (int kb = kbeg / 128; kb * 128 < kend; ++kb) {
    const float x = xs[(long)kb * p.T], y = ys[(long)kb * nb];
    if (x - x != 0 || y - y != 0) return v;  // not a number by its values
    over |= x * y - x * y != 0;
  }
  if (!over) return v;
  const unsigned char* a = (const unsigned char*)p.a + (long)row * p.lda;
  const unsigned char* b = (const unsigned char*)p.b + (long)g * p.gsb;
  f32x4 sum = {0, 0, 0, 0};
  bool any = true;  // what has become infinite or NaN stays so
#pragma unroll 1
  for (int k = kbeg; k < kend && any; ++k) {
    const float x = __builtin_amdgcn_cvt_f32_fp8(a[k], 0) *
                    xs[(long)(k / 128) * p.T];
    any = false;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int n = min(col + q, p.N - 1);
      const float y = __builtin_amdgcn_cvt_f32_fp8(b[(long)n * p.ldb + k], 0) *
                      ys[(long)(k / 128) * nb];
      sum[q] = __builtin_fmaf(x, y, sum[q]);
      any |= sum[q] - sum[q] == 0;
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) v[q] = v[q] - v[q] == 0 ? v[q] : sum[q];
  return v;
}

// ---- small and middle tiles ------------------------------------------------

// BM x BN results a workgroup, its waves WM x WN. AK/BK: the operand has k
// along its rows. WEIGHTS: the sum runs over a group's rows.
//
// D LDS stages: the copies of D - 1 K tiles are on their way at a time, since
// a tile's products are shorter than the way to memory; one barrier a tile.
// ALIGNED: rows (and for an R side its length) are multiples of 16 bytes, and
// whole tiles are copied to LDS; a last tile that ends early, and all tiles of
// ANY rows, go through registers. SLOW: rows shorter than that.
enum RowsPath { ALIGNED, ANY, SLOW };

template <int TY, int BM, int BN, int WM, int WN, int D, bool AK, bool BK,
          bool WEIGHTS, RowsPath PATH>
__global__ void __launch_bounds__(64 * WM * WN, 2)  // waves a SIMD
grouped_k(const GroupedArgs p) {
  constexpr int NT = 64 * WM * WN;
  constexpr int ES = Elt<TY>::ES, BKE = 128 / ES;
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  typedef Side<TY, BM, NT, AK> SA;
  typedef Side<TY, BN, NT, BK> SB;
  // fp8: scales of BM rows, then of the columns, 64 a wave
  constexpr int SCALES = TY == GT_FP8 ? NT * 4 : 0;
  static_assert(!SCALES || BM + 64 <= NT, "a wave is left for the columns");
  constexpr int STAGE = (BM + BN) * 128 + SCALES;
  constexpr int OPS = SA::IT + SB::IT + (SCALES ? 1 : 0);  // copies a stage
  extern __shared__ __attribute__((aligned(16))) char smem[];

  Work w;
  if (!locate<TY, BM, BN, WEIGHTS>(p, &w)) return;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);

  f32x4 acc[FN][FM];
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int i = 0; i < FM; ++i) acc[j][i] = f32x4{0, 0, 0, 0};

  const int depth = w.kend - w.kbeg;
  const int whole = depth / BKE, tiles = (depth + BKE - 1) / BKE;

  const float* scale = nullptr;  // this thread's, of the first tile
  int scale_step = 0;
  if constexpr (TY == GT_FP8) {
    const int nb = (p.N + 127) / 128;
    const long kb = w.kbeg / 128;
    const bool rows = tid < BM;
    scale = rows ? p.asc + kb * p.T + min(w.m0 + tid, p.T - 1)
                 : p.bsc + ((long)min(w.g, p.E - 1) * ((p.K + 127) / 128) +
                            kb) * nb + w.n0 / 128;
    scale_step = rows ? p.T : nb;
  }

  auto products = [&](const char* lds) {
    const char* la = lds;
    const char* lb = lds + BM * 128;
    if constexpr (TY == GT_FP8) {
      // a K tile is one block of scales: its products are summed apart and
      // join the f32 sum with one multiply-add. BN <= 128: one block of b
      const float* sc = (const float*)(lds + (BM + BN) * 128);
      float s[FM];
      i32x8 y[FM];
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        s[i] = sc[wm + i * 16 + (lane & 15)] * sc[BM];
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
            acc[j][i][q] = __builtin_fmaf(d[q], s[i], acc[j][i][q]);
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
    SA sa;
    SB sb;
    sa.init(p.a, p.lda, w.m0, w.mend, w.kbeg);
    sb.init((const char*)p.b + (WEIGHTS ? 0 : (long)w.g * p.gsb * ES), p.ldb,
            w.n0, p.N, w.kbeg);
    struct Held {  // a tile on its way through registers
      typename SA::Regs a;
      typename SB::Regs b;
      float scale;
    };
    auto load = [&](Held& h, int tile) {
      if constexpr (SCALES) h.scale = scale[(long)tile * scale_step];
      sa.load(h.a, tile, w.kend);
      sb.load(h.b, tile, w.kend);
    };
    auto put = [&](Held& h, int tile, int stage) {
      char* lds = smem + stage * STAGE;
      sa.template put<PATH != ALIGNED>(lds, h.a, tile, w.kend);
      sb.template put<PATH != ALIGNED>(lds + BM * 128, h.b, tile, w.kend);
      if constexpr (SCALES) ((float*)(lds + (BM + BN) * 128))[tid] = h.scale;
    };
    if constexpr (PATH == ALIGNED) {
      int next = 0, to = 0;  // the next copy and its stage
      auto copy = [&]() {
        const u32 lds = to * STAGE;
        if constexpr (SCALES)
          glds4(scale + (long)next * scale_step,
                smem + lds + (BM + BN) * 128 + tid * 4);
        sa.copy(smem, lds, next);
        sb.copy(smem, lds + BM * 128, next);
        ++next;
        to = to == D - 1 ? 0 : to + 1;
      };
      Held h;
      for (int i = 0; i < D - 1 && i < whole; ++i) copy();
      int stage = 0;
      for (int t = 0; t < whole; ++t) {
        // tile t is there when no more than the D - 2 behind it are missing
        if (next < whole)
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 2) * OPS) : "memory");
        else
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        if (next < whole) copy();
        if (t + 1 == whole && whole < tiles) load(h, whole);
        products(smem + stage * STAGE);
        stage = stage == D - 1 ? 0 : stage + 1;
      }
      if (whole < tiles) {  // behind D - 1 others, its stage is free
        if (whole == 0) load(h, 0);
        put(h, whole, stage);
        __syncthreads();
        products(smem + stage * STAGE);
      }
    } else if constexpr (PATH == ANY) {
      // two stages in LDS and two tiles in registers: a load has the time of
      // two tiles' products
      Held h0, h1;
      load(h0, 0);
      if (tiles > 1) load(h1, 1);
      put(h0, 0, 0);
      auto step = [&](int t, int stage, Held& free, Held& next) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        if (t + 2 < tiles) load(free, t + 2);
        products(smem + stage * STAGE);
        if (t + 1 < tiles) put(next, t + 1, stage ^ 1);
      };
      for (int t = 0; t < tiles; t += 2) {
        step(t, 0, h0, h1);
        if (t + 1 < tiles) step(t + 1, 1, h1, h0);
      }
    } else {
      for (int t = 0; t < tiles; ++t) {
        sa.gather(smem, t, w.kend);
        sb.gather(smem + BM * 128, t, w.kend);
        if constexpr (SCALES)
          ((float*)(smem + (BM + BN) * 128))[tid] =
              scale[(long)t * scale_step];
        __syncthreads();
        products(smem);
        __syncthreads();
      }
    }
  }

  const Results<WEIGHTS> out(p, w);
  if constexpr (TY == GT_FP8) {
    float z = 0;
#pragma unroll
    for (int i = 0; i < FM * FN; ++i) z += zero4(((f32x4*)acc)[i]);
    if (z != 0) {
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const int row = w.m0 + wm + i * 16 + (lane & 15);
          const int col = w.n0 + wn + j * 16 + (lane >> 4) * 4;
          if (row < w.mend && col < p.N && zero4(acc[j][i]) != 0)
            acc[j][i] = fp8_again(p, w.g, row, col, w.kbeg, w.kend, acc[j][i]);
        }
    }
  }
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
      out.put(w.m0 + wm + i * 16, w.n0 + wn + j * 16, acc[j][i]);
}

// ---- the large tile --------------------------------------------------------

// 256 x 256 results, 8 waves, operands whose rows begin on 16 bytes. A K tile
// is four halves of 16 KB: A0, A1 (rows), B0, B1 (columns). In each of four
// phases all waves work on one 128 x 128 quarter, a 32 x 64 slice each, in the
// order A0B0, A0B1, A1B1, A1B0, so that the halves are needed one after
// another: while a tile is multiplied the next one's halves are copied in
// that order, one a phase, and a phase ends with a wait that leaves the
// younger copies in flight. The copies are never waited for to the last one
// inside the loop. The second four waves have the higher priority: two waves
// of a SIMD then take turns at the matrix unit instead of reading LDS at once.
// A tile whose group ends within its first 128 rows does the first two phases
// only.
template <int TY, bool AK, bool BK, bool WEIGHTS>
__global__ void __launch_bounds__(512) grouped_big_k(const GroupedArgs p) {
  constexpr int ES = Elt<TY>::ES, BKE = 128 / ES;
  typedef Side<TY, 128, 512, AK> SA;
  typedef Side<TY, 128, 512, BK> SB;
  constexpr int HALF = 128 * 128, BUF = 4 * HALF;
  extern __shared__ __attribute__((aligned(16))) char smem[];

  Work w;
  if (!locate<TY, 256, 256, WEIGHTS>(p, &w)) return;

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int qr = (wave & 3) * 32, qc = (wave >> 2) * 64;

  f32x4 acc[2][2][4][2];  // [row half][column half][columns][rows]
#pragma unroll
  for (int i = 0; i < 32; ++i) ((f32x4*)acc)[i] = f32x4{0, 0, 0, 0};

  const int depth = w.kend - w.kbeg;
  const int whole = depth / BKE;

  // fp8: the scales of a K tile go through LDS as well, a word a lane: of 256
  // rows by the first four waves, of the two column blocks by the others.
  // (Loaded into registers, they would be waited for together with all copies
  // behind them.)
  constexpr int SCALES = TY == GT_FP8 ? 2048 : 0;
  const float* scale = nullptr;
  int scale_step = 0;
  if constexpr (TY == GT_FP8) {
    const int nb = (p.N + 127) / 128, tid = threadIdx.x;
    const long kb = w.kbeg / 128;
    scale = tid < 256
                ? p.asc + kb * p.T + min(w.m0 + tid, p.T - 1)
                : p.bsc + ((long)min(w.g, p.E - 1) * ((p.K + 127) / 128) +
                           kb) * nb + min(w.n0 / 128 + (tid & 1), nb - 1);
    scale_step = tid < 256 ? p.T : nb;
  }
  auto copy_scales = [&](int stage, int tile) {
    if constexpr (SCALES)
      glds4(scale + (long)tile * scale_step,
            smem + 2 * BUF + stage * SCALES + threadIdx.x * 4);
  };

  i32x4 y[2][2], x[2][4];  // [half of k][fragments]
  auto read_a = [&](const char* buf, int h) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        y[kk][i] = SA::frag(buf + h * HALF, qr + i * 16, kk);
  };
  auto read_b = [&](const char* buf, int h) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[kk][j] = SB::frag(buf + (2 + h) * HALF, qc + j * 16, kk);
  };
  float sa[2][2], sb[2];  // the scales of the tile that is multiplied
  auto quarter = [&](int hm, int hn) {
    if constexpr (TY == GT_FP8) {
      float sc[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) sc[i] = sa[hm][i] * sb[hn];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const f32x4 d = mma_fp8(join8(x[0][j], x[1][j]),
                                  join8(y[0][i], y[1][i]),
                                  f32x4{0, 0, 0, 0});
#pragma unroll
          for (int q = 0; q < 4; ++q)
            acc[hm][hn][j][i][q] =
                __builtin_fmaf(d[q], sc[i], acc[hm][hn][j][i][q]);
        }
    } else {
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            acc[hm][hn][j][i] =
                mma<TY>(x[kk][j], y[kk][i], acc[hm][hn][j][i]);
    }
  };
  auto read_scales = [&](int stage) {
    if constexpr (SCALES) {
      const float* v = (const float*)(smem + 2 * BUF + stage * SCALES);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          sa[h][i] = v[h * 128 + qr + i * 16 + (lane & 15)];
        sb[h] = v[256 + h];
      }
    }
  };

  if (depth > 0) {
    const char* b = (const char*)p.b +
                    (WEIGHTS ? 0 : (long)w.g * p.gsb * ES);
    SA a0, a1;
    SB b0, b1;
    // a half past the end takes its row from inside
    a0.init(p.a, p.lda, w.m0, w.mend, w.kbeg);
    b0.init(b, p.ldb, w.n0, p.N, w.kbeg);
    a1.init(p.a, p.lda, w.m0 + 128 < w.mend ? w.m0 + 128 : w.m0, w.mend,
            w.kbeg);
    b1.init(b, p.ldb, w.n0 + 128 < p.N ? w.n0 + 128 : w.n0, p.N, w.kbeg);

    // Groups start at different K tiles: rows of many kilobytes lie a power of
    // two apart, and all XCDs, each in its own group, would read the same
    // columns, hence the same memory channels, at the same time. The order of
    // a sum depends on its group alone.
    const int turn = WEIGHTS ? 0 : (int)((long)whole * (w.g & 7) / 8);
    auto at = [&](int t) {
      t += turn;
      return t >= whole ? t - whole : t;
    };

    // vector memory operations of a lane in flight at each wait, oldest
    // first (2 a half; S: the scales of fp8, 1; ' = next tile):
    //   end of phase 1: B1 A1 S' A0'        B1 has to be there
    //   end of phase 2: A1 S' A0' B0'       A1 has to be there
    //   end of phase 4: S' A0' B0' B1' A1'  A0' and B0' have to be there
#define GB_WAIT(n) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory")
    // with the first rows alone:
    //   end of phase 1: B1 S' A0'           B1 has to be there
    //   end of phase 2: S' A0' B0' B1'      A0' and B0' have to be there
    auto step = [&](auto more, auto both, int t) {
      const char* cur = smem + (t & 1) * BUF;
      const u32 nxt = (~t & 1) * BUF;
      read_scales(t & 1);
      read_a(cur, 0);
      read_b(cur, 0);
      if constexpr (more) {
        copy_scales(~t & 1, at(t + 1));
        a0.copy(smem, nxt, at(t + 1));
      }
      quarter(0, 0);
      if constexpr (!more) GB_WAIT(both ? 2 : 0);
      else GB_WAIT((both ? 4 : 2) + (SCALES ? 1 : 0));
      __builtin_amdgcn_s_barrier();
      read_b(cur, 1);
      if constexpr (more) b0.copy(smem, nxt + 2 * HALF, at(t + 1));
      if constexpr (more && !both) b1.copy(smem, nxt + 3 * HALF, at(t + 1));
      quarter(0, 1);
      if constexpr (both) {
        if constexpr (!more) GB_WAIT(0);
        else GB_WAIT(4 + (SCALES ? 1 : 0));
        __builtin_amdgcn_s_barrier();
        read_a(cur, 1);
        if constexpr (more) b1.copy(smem, nxt + 3 * HALF, at(t + 1));
        quarter(1, 1);
        read_b(cur, 0);
        if constexpr (more) a1.copy(smem, nxt + HALF, at(t + 1));
        quarter(1, 0);
      }
      // every read of this buffer is back too, before it is copied into
      if constexpr (more) GB_WAIT(both ? 4 : 2);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
    };
    struct Yes { constexpr operator bool() const { return true; } };
    struct No { constexpr operator bool() const { return false; } };

    if (__builtin_amdgcn_readfirstlane(threadIdx.x) >= 256)
      __builtin_amdgcn_s_setprio(1);
    const bool lower = w.m0 + 128 < w.mend;
    auto all = [&](auto both) {
      copy_scales(0, at(0));
      a0.copy(smem, 0, at(0));
      b0.copy(smem, 2 * HALF, at(0));
      b1.copy(smem, 3 * HALF, at(0));
      if constexpr (both) a1.copy(smem, HALF, at(0));
      GB_WAIT(both ? 4 : 2);
      __builtin_amdgcn_s_barrier();
      for (int t = 0; t + 1 < whole; ++t) step(Yes{}, both, t);
      step(No{}, both, whole - 1);
    };
    if (whole > 0) {
      if (lower) all(Yes{});
      else all(No{});
    }
#undef GB_WAIT
    if (whole * BKE < depth) {  // what is left of k
      __syncthreads();
      typename SA::Regs r, r1;
      typename SB::Regs s, s1;
      a0.load(r, whole, w.kend);
      a1.load(r1, whole, w.kend);
      b0.load(s, whole, w.kend);
      b1.load(s1, whole, w.kend);
      a0.template put<false>(smem, r, whole, w.kend);
      a1.template put<false>(smem + HALF, r1, whole, w.kend);
      b0.template put<false>(smem + 2 * HALF, s, whole, w.kend);
      b1.template put<false>(smem + 3 * HALF, s1, whole, w.kend);
      if constexpr (SCALES)
        *(float*)(smem + 2 * BUF + threadIdx.x * 4) =
            scale[(long)whole * scale_step];
      __syncthreads();
      read_scales(0);
      read_a(smem, 0);
      read_b(smem, 0);
      quarter(0, 0);
      read_b(smem, 1);
      quarter(0, 1);
      read_a(smem, 1);
      quarter(1, 1);
      read_b(smem, 0);
      quarter(1, 0);
    }
    __builtin_amdgcn_s_setprio(0);
  }

  if constexpr (TY == GT_FP8) {
    float z = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) z += zero4(((f32x4*)acc)[i]);
    if (z != 0) {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        f32x4& v = ((f32x4*)acc)[i];
        const int row = w.m0 + (i >> 4) * 128 + qr + (i & 1) * 16 + (lane & 15);
        const int col = w.n0 + (i >> 3 & 1) * 128 + qc + (i >> 1 & 3) * 16 +
                        (lane >> 4) * 4;
        if (row < w.mend && col < p.N && zero4(v) != 0)
          v = fp8_again(p, w.g, row, col, w.kbeg, w.kend, v);
      }
    }
  }
  const Results<WEIGHTS> out(p, w);
  if (out.ty != GT_F32 && out.n % 8 == 0 && (u64)out.c % 16 == 0) {
    // 16-bit results turn round in LDS, so that 32 lanes store 512 bytes of
    // a row: 4 KB rows x 8-byte pieces from registers reach half the rate
    __syncthreads();
#pragma unroll
    for (int hm = 0; hm < 2; ++hm)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = hm * 128 + qr + i * 16 + (lane & 15);
#pragma unroll
        for (int hn = 0; hn < 2; ++hn)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int c8 = (hn * 128 + qc + j * 16 + (lane >> 4) * 4) / 4;
            const f32x4 v = acc[hm][hn][j][i];
            const u32 lo = f32_to_bits16(v[0], out.ty) |
                           (u32)f32_to_bits16(v[1], out.ty) << 16;
            const u32 hi = f32_to_bits16(v[2], out.ty) |
                           (u32)f32_to_bits16(v[3], out.ty) << 16;
            *(uint2*)(smem + row * 512 +
                      ((c8 ^ (row & 15) << 1) << 3)) = make_uint2(lo, hi);
          }
      }
    __syncthreads();
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
      const int row = i * 16 + (threadIdx.x >> 5), c = threadIdx.x & 31;
      const i32x4 v =
          *(const i32x4*)(smem + row * 512 + ((c ^ (row & 15)) << 4));
      const int r = w.m0 + row, n = w.n0 + c * 8;
      if (r < out.mend && n < out.n)
        *(i32x4*)((unsigned short*)out.c + (out.first + r) * out.n + n) = v;
    }
    return;
  }
#pragma unroll
  for (int hm = 0; hm < 2; ++hm)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int hn = 0; hn < 2; ++hn)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          out.put(w.m0 + hm * 128 + qr + i * 16, w.n0 + hn * 128 + qc + j * 16,
                  acc[hm][hn][j][i]);
}
