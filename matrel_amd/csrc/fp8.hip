// Values to e4m3 with a float32 scale for each block of 128:
//   top = max(max |x|, 2^-100),  scale = top / 448,  q = e4m3(x * (448 / top))
// in float32, every step rounded to nearest. A block is 128 values along a row
// ("row") or 128 x 128 ("tile"). A NaN or an infinity makes its block's scale
// NaN or infinite, and the values that it stands for NaN.
//
// Bound by memory: each value is read once, kept in registers between the
// maximum and the conversion, and written once.
#include "grouped_core.h"

// |x| as bits: their order as integers is the order of the values, with NaN
// above infinity, so that one integer maximum carries both.
__device__ __forceinline__ u32 abs_bits(float x) {
  return __float_as_uint(x) & 0x7fffffffu;
}

template <int TY> __device__ __forceinline__ float load1(const void* x, long i) {
  if constexpr (TY == GT_F32) return ((const float*)x)[i];
  if constexpr (TY == GT_BF16) return (float)((const __bf16*)x)[i];
  return (float)((const _Float16*)x)[i];
}

// Eight neighbouring values from any address, zeros from `have` on.
template <int TY>
__device__ __forceinline__ void load8(const void* x, long i, int have,
                                      float* v) {
  if (have >= 8) {
    if constexpr (TY == GT_F32) {
      f32x4 lo, hi;
      __builtin_memcpy(&lo, (const float*)x + i, 16);
      __builtin_memcpy(&hi, (const float*)x + i + 4, 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = lo[j];
        v[4 + j] = hi[j];
      }
    } else if constexpr (TY == GT_BF16) {
      bf16x8 q;
      __builtin_memcpy(&q, (const __bf16*)x + i, 16);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (float)q[j];
    } else {
      f16x8 q;
      __builtin_memcpy(&q, (const _Float16*)x + i, 16);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (float)q[j];
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = j < have ? load1<TY>(x, i + j) : 0.0f;
}

__device__ __forceinline__ uint2 pack8(const float* v, float up) {
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * up, v[1] * up, lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * up, v[3] * up, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * up, v[5] * up, hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * up, v[7] * up, hi, true);
  return make_uint2((u32)lo, (u32)hi);
}

__device__ __forceinline__ void put8(unsigned char* o, uint2 q, int have) {
  if (have >= 8) {
    __builtin_memcpy(o, &q, 8);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < have) o[j] = (unsigned char)((j < 4 ? q.x : q.y) >> (8 * (j & 3)));
}

#define TOP_MIN 0x0d800000u  // 2^-100

// Where rows are not whole lines, neighbouring blocks share lines: they go to
// one XCD, whose L2 joins them (f32 8 x 2000 x 5000: 94 -> 81 us).
__device__ __forceinline__ u32 place(long cols) {
  return cols % 128 ? xcd_swizzle(blockIdx.x, gridDim.x) : blockIdx.x;
}

// 16 lanes take a block of a row, 8 values each; a workgroup 16 rows of one
// column block, whose scales are neighbours.
template <int TY>
__global__ void __launch_bounds__(256)
quantize_row_k(const void* __restrict__ x, long ld, long rows, long cols,
               unsigned char* __restrict__ q, float* __restrict__ scale) {
  const u32 id = place(cols);
  const long ncb = (cols + 127) / 128, cb = id % ncb;
  const long row = id / ncb * 16 + (threadIdx.x >> 4);
  const long col = cb * 128 + (threadIdx.x & 15) * 8;
  const bool in = row < rows && col < cols;
  const int have = in ? (int)min(8L, cols - col) : 0;
  float v[8];
  load8<TY>(x, in ? row * ld + col : 0, have, v);
  u32 top = TOP_MIN;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, abs_bits(v[j]));
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) top = max(top, (u32)__shfl_xor((int)top, d));
  const float t = __uint_as_float(top);
  if (!in) return;
  put8(q + row * cols + col, pack8(v, 448.0f / t), have);
  if ((threadIdx.x & 15) == 0) scale[cb * rows + row] = t / 448.0f;
}

// A tile of 128 x 128 bytes in LDS, to its place in the transposed matrix: a
// thread gathers 8 rows of one column, 16 lanes write its 128 rows.
__device__ __forceinline__ void put_turned(const unsigned char (*turn)[132],
                                           unsigned char* qt, long rows,
                                           long cols, long rb, long cb) {
  const long r8 = rb * 128 + (threadIdx.x & 15) * 8;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = (threadIdx.x >> 4) + i * 16;
    u32 w[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      w[j >> 2] |= (u32)turn[(threadIdx.x & 15) * 8 + j][c] << (8 * (j & 3));
    if (cb * 128 + c < cols && r8 < rows)
      put8(qt + (cb * 128 + c) * rows + r8, make_uint2(w[0], w[1]),
           (int)min(8L, rows - r8));
  }
}

// A workgroup takes a tile of 128 x 128, 64 values a thread. With `qt` it also
// writes the tile transposed (through LDS), for products along the other axis.
template <int TY>
__global__ void __launch_bounds__(256)
quantize_tile_k(const void* __restrict__ x, long ld, long batch_ld, long rows,
                long cols, unsigned char* __restrict__ q,
                unsigned char* __restrict__ qt, float* __restrict__ scale,
                float* __restrict__ scale_t) {
  __shared__ u32 tops[4];
  __shared__ unsigned char turn[128][132];
  const long nrb = (rows + 127) / 128, ncb = (cols + 127) / 128;
  const u32 id = place(cols);
  const long cb = id % ncb, rb = id / ncb, e = blockIdx.y;
  const char* base = (const char*)x + e * batch_ld * (TY == GT_F32 ? 4 : 2);
  const long col = cb * 128 + (threadIdx.x & 15) * 8;
  const long row0 = rb * 128 + (threadIdx.x >> 4);
  float v[8][8];
  u32 top = TOP_MIN;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long row = row0 + i * 16;
    const bool in = row < rows && col < cols;
    load8<TY>(base, in ? row * ld + col : 0, in ? (int)min(8L, cols - col) : 0,
              v[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, abs_bits(v[i][j]));
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = max(top, (u32)__shfl_xor((int)top, d));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
  const float t = __uint_as_float(top), up = 448.0f / t;
  if (threadIdx.x == 0) {
    scale[(e * ncb + cb) * nrb + rb] = t / 448.0f;
    if (scale_t) scale_t[(e * nrb + rb) * ncb + cb] = t / 448.0f;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long row = row0 + i * 16;
    const uint2 w = pack8(v[i], up);
    if (row < rows && col < cols)
      put8(q + (e * rows + row) * cols + col, w, (int)min(8L, cols - col));
    if (qt) {
      u32* s = (u32*)&turn[(threadIdx.x >> 4) + i * 16][(threadIdx.x & 15) * 8];
      s[0] = w.x;
      s[1] = w.y;
    }
  }
  if (!qt) return;
  __syncthreads();
  put_turned(turn, qt + e * rows * cols, rows, cols, rb, cb);
}

// e4m3 matrices transposed, where a program keeps blocks of one side only.
// Bound by memory: 8 x 4096 x 2048 in 30 us, 4.4 TB/s read + written.
__global__ void __launch_bounds__(256)
turn_k(const unsigned char* __restrict__ q, long rows, long cols,
       unsigned char* __restrict__ qt) {
  __shared__ unsigned char turn[128][132];
  const long nrb = (rows + 127) / 128, ncb = (cols + 127) / 128;
  const u32 id = xcd_swizzle(blockIdx.x, (u32)(nrb * ncb));
  const long cb = id % ncb, rb = id / ncb, e = blockIdx.y;
  const long col = cb * 128 + (threadIdx.x & 15) * 8;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = (threadIdx.x >> 4) + i * 16;
    const long row = rb * 128 + r;
    uint2 w = {0, 0};
    if (row < rows && col < cols) {
      const unsigned char* x = q + (e * rows + row) * cols + col;
      if (col + 8 <= cols) {
        __builtin_memcpy(&w, x, 8);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col + j < cols)
            (j < 4 ? w.x : w.y) |= (u32)x[j] << (8 * (j & 3));
      }
    }
    u32* s = (u32*)&turn[r][(threadIdx.x & 15) * 8];
    s[0] = w.x;
    s[1] = w.y;
  }
  __syncthreads();
  put_turned(turn, qt + e * rows * cols, rows, cols, rb, cb);
}

extern "C" void launch_fp8_quantize_row(const void* x, int ty, long ld,
                                        long rows, long cols, void* q,
                                        float* scale, hipStream_t s) {
  const dim3 grid((unsigned)((cols + 127) / 128 * ((rows + 15) / 16)));
#define GO(TY)                                                              \
  hipLaunchKernelGGL(quantize_row_k<TY>, grid, dim3(256), 0, s, x, ld, rows, \
                     cols, (unsigned char*)q, scale)
  if (ty == GT_F32) GO(GT_F32);
  else if (ty == GT_BF16) GO(GT_BF16);
  else GO(GT_F16);
#undef GO
}

extern "C" void launch_fp8_quantize_tile(const void* x, int ty, long ld,
                                         long batch_ld, long batch, long rows,
                                         long cols, void* q, void* qt,
                                         float* scale, float* scale_t,
                                         hipStream_t s) {
  const dim3 grid((unsigned)(((cols + 127) / 128) * ((rows + 127) / 128)),
                  (unsigned)batch);
#define GO(TY)                                                               \
  hipLaunchKernelGGL(quantize_tile_k<TY>, grid, dim3(256), 0, s, x, ld,      \
                     batch_ld, rows, cols, (unsigned char*)q,                \
                     (unsigned char*)qt, scale, scale_t)
  if (ty == GT_F32) GO(GT_F32);
  else if (ty == GT_BF16) GO(GT_BF16);
  else GO(GT_F16);
#undef GO
}

extern "C" void launch_fp8_turn(const void* q, long batch, long rows,
                                long cols, void* qt, hipStream_t s) {
  const dim3 grid((unsigned)(((cols + 127) / 128) * ((rows + 127) / 128)),
                  (unsigned)batch);
  hipLaunchKernelGGL(turn_k, grid, dim3(256), 0, s, (const unsigned char*)q,
                     rows, cols, (unsigned char*)qt);
}
