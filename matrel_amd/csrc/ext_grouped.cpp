// Python bindings of the grouped products and of the 8-bit block conversion.
// Host-side only: what the kernels assume of shapes, strides and alignment is
// checked or chosen here.
#include <torch/extension.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <tuple>
#include <unordered_set>
#include <vector>

#include "grouped_args.h"

extern "C" {
void launch_grouped_bf16(const GroupedArgs*, int, int, int, int, hipStream_t);
void launch_grouped_f16(const GroupedArgs*, int, int, int, int, hipStream_t);
void launch_grouped_f32(const GroupedArgs*, int, int, int, int, hipStream_t);
void launch_grouped_fp8(const GroupedArgs*, int, int, hipStream_t);
void launch_grouped_join(const float*, void*, long, int, int, hipStream_t);
void launch_fp8_quantize_row(const void*, int, long, long, long, void*,
                             float*, hipStream_t);
void launch_fp8_quantize_tile(const void*, int, long, long, long, long, long,
                              void*, void*, float*, float*, hipStream_t);
void launch_fp8_turn(const void*, long, long, long, void*, hipStream_t);
}

namespace {

using torch::Tensor;

int type_of(at::ScalarType t) {
  switch (t) {
    case torch::kBFloat16: return GT_BF16;
    case torch::kFloat16: return GT_F16;
    case torch::kFloat32: return GT_F32;
    case torch::kFloat8_e4m3fn: return GT_FP8;
    default: TORCH_CHECK(false, "unsupported type ", t);
  }
}

hipStream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

void check_launch() {
  const hipError_t e = hipGetLastError();
  TORCH_CHECK(e == hipSuccess, "HIP error: ", hipGetErrorString(e));
}

// Kernels count in 32 bits, up to 16 parts of whole tiles or 32 K tiles of 128
// bytes past the end.
int dim32(int64_t n, const char* what) {
  TORCH_CHECK(n >= 0 && n < (int64_t(1) << 31) - (1 << 16), what,
              " is too large");
  return (int)n;
}

// Rows (or k) of `ld` elements that begin on 16 bytes.
bool aligned(const Tensor& t, int64_t ld, int64_t count) {
  const int64_t es = t.element_size();
  return (uintptr_t)t.data_ptr() % 16 == 0 &&
         (count <= 1 || ld * es % 16 == 0);
}

// A row of `len` elements holds 16 bytes, and a tile's 256 rows lie within 31
// bits of its first one.
// Neither alignment (path 1) nor that (path 2) is asked of the operands.
bool near_rows(const Tensor& t, int64_t ld, int64_t len) {
  return len * t.element_size() >= 16 &&
         ld * t.element_size() < (1 << 23);
}

// t as the kernels can read it: what torch only marks as negated or as zeros
// is written out, and a tensor without memory (a fake one) refused.
Tensor readable(const Tensor& t) {
  if (t.is_neg() || t._is_zerotensor()) return t.clone();
  TORCH_CHECK(t.numel() == 0 || t.const_data_ptr() != nullptr,
              "operands must have memory");
  return t;
}

// t, or a copy whose last dimension is contiguous.
Tensor rows_contiguous(const Tensor& t) {
  return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

void set_offsets(GroupedArgs& p, c10::optional<Tensor>& offs,
                 const Tensor& a, int64_t groups) {
  if (!offs.has_value()) {
    TORCH_CHECK(groups == 1, "several groups need offsets");
    return;
  }
  offs = readable(*offs).contiguous();
  TORCH_CHECK(offs->device() == a.device() && offs->dim() == 1 &&
                  offs->numel() == groups + 1 &&
                  (offs->scalar_type() == torch::kInt32 ||
                   offs->scalar_type() == torch::kInt64),
              "offsets must be groups + 1 integers on the operands' device");
  p.offs = offs->data_ptr();
  p.off64 = offs->scalar_type() == torch::kInt64;
}

struct Plan {
  int tile, splits;
};

// A launch holds fewer than 2^32 threads. For row tiles of 16 or 32 the grid
// is counted in blocks of 64 columns, which is what so many get.
void check_grid(const GroupedArgs& p, int tile, int path, bool weights) {
  const int bm = tile == -1 ? 16 : tile == -2 || tile == 0 ? 32
                 : path == 2 || tile == 1 ? 64 : tile == 2 ? 128 : 256;
  const int bn = tile == 0 ? 128 : std::max(bm, 64);
  const int64_t rows = weights ? (int64_t)p.E * ((p.M + bm - 1) / bm)
                               : grouped_row_tiles(p, bm);
  TORCH_CHECK(rows * ((p.N + bn - 1) / bn) <
                  (int64_t(1) << 32) / (bm == 256 ? 512 : 256),
              "product has too many tiles");
}

// Into how many parts long sums are split where even small tiles do not fill
// the chip.
int choose_splits(int64_t tiles, int64_t k_tiles) {
  // the join is a launch and a pass over the parts: not for short sums
  if (tiles >= 192 || k_tiles < 16) return 1;
  return (int)std::min<int64_t>({k_tiles / 4, (383 + tiles) / tiles, 16});
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tiles (codes: grouped_launch.h). Measured, us, 64 x 64 / 128 x 128 / 256 x
// 256, behind the number of 256 x 256 ones that the host counts:
//   rows, bf16 8192 rows, 8 groups, 1112 x 776 (190): 39 / 36 / 27
//   rows, bf16 8192 rows, 32 groups, 1536 x 1032 (280): 57 / 48 / 71
//   rows, fp8 16384 rows, 8192 x 8192 (2048): the large one 1.2 x the middle
//   rows, bf16 913 rows, 24 groups, 1344 x 2904: 39 / 44 / 64
//   d_b, bf16 8192 rows, 32 groups, 1536 x 1032 (960): 109 / 71 / 62
//   d_b, bf16 8192 rows, 8 groups, 2048 x 2048 (512): 123 / 84 / 104
//   d_b, bf16 8192 rows, 8 groups, 1112 x 776 (160): 42 / 61 / 97
//   d_b, bf16 10641 rows, 3 groups, 2232 x 1632 (189): 158 / 104 / 87
//   rows, f32 4096 rows, 12 groups, 1024 x 1000: 106 / 138 / -
//   d_b, fp16 unaligned, 3001 rows, 10 groups, 1111 x 777: 36 / 50 / -
// Over 38 other shapes drawn at random the choice takes 1.02 - 1.05 of the
// best tile's time on average.

// Whether 256 x 256 tiles take less time in rounds over the chip's 256 CUs,
// one on each, than 128 x 128 ones, two on each: a round of large tiles takes
// 3/2 of the time of one of small ones, which are half as much work.
bool large_pays(int64_t large, int64_t middle) {
  return 3 * ceil_div(large, 256) <= 2 * ceil_div(middle, 512);
}

// large: whether 256 x 256 tiles pay; enough: 128 x 128 tiles that do.
template <class F>
Plan choose(int ty, bool fast, bool large, int64_t enough, int64_t k_tiles,
            F count) {
  Plan p = {1, 1};
  const bool free = fast && ty != GT_F32;
  if (free && large) p.tile = 3;
  else if (count(128, 128) >= (free ? enough : 1024)) p.tile = 2;
  if (p.tile == 1) p.splits = choose_splits(count(64, 64), k_tiles);
  return p;
}

// Tiles of the rows of E groups, each of which can end inside a tile.
int64_t row_tiles(int64_t T, int64_t E, int64_t bm) {
  return E == 1 ? ceil_div(T, bm) : T / bm + std::min(E, T);
}

Plan choose_rows(int ty, bool bk, bool fast, int64_t T, int64_t E, int64_t K,
                 int64_t N) {
  const int64_t each = ceil_div(T, E);
  const int64_t k_tiles = ceil_div(K, ty == GT_FP8 ? 128
                                      : ty == GT_F32 ? 32 : 64);
  if (bk && each <= 32) return {each <= 16 ? -1 : -2, 1};
  if (fast && each <= 32)
    return {0, choose_splits(row_tiles(T, E, 32) * ceil_div(N, 128), k_tiles)};
  // a group ends inside a tile by half of it on average, short ones by more
  const auto met = [&](int64_t b) {
    return (E == 1 ? ceil_div(T, b) : T / b + std::min(E, T) * 3 / 4) *
           ceil_div(N, b);
  };
  // and where all are short, a large tile is mostly empty
  const bool large = each >= 128 && large_pays(met(256), met(128));
  return choose(ty, fast, large, 250, k_tiles,
                [&](int64_t bm, int64_t bn) {
                  return row_tiles(T, E, bm) * ceil_div(N, bn);
                });
}

// Where the kernel writes: c, or partial sums that finish() joins.
Tensor begin(GroupedArgs& p, Tensor& c, int splits) {
  Tensor part;
  p.splits = splits;
  if (splits > 1) {
    part = torch::empty({splits, c.numel()},
                        c.options().dtype(torch::kFloat32));
    p.part = part.data_ptr<float>();
  }
  return part;
}

void finish(const GroupedArgs& p, Tensor& c, hipStream_t s) {
  if (p.splits > 1)
    launch_grouped_join(p.part, p.c, c.numel(), p.splits, p.out, s);
  check_launch();
}

void launch_rows(const GroupedArgs& p, int ty, int tile, bool bk, int path,
                 hipStream_t s) {
  if (ty == GT_FP8) launch_grouped_fp8(&p, tile, path, s);
  else if (ty == GT_BF16) launch_grouped_bf16(&p, tile, bk, 0, path, s);
  else if (ty == GT_F16) launch_grouped_f16(&p, tile, bk, 0, path, s);
  else launch_grouped_f32(&p, tile, bk, 0, path, s);
}

// c[t, :] = a[t, :] @ b[group of t], zeros for rows of no group.
// a [T, K], b [E, K, N]; k or n of b contiguous, or it is copied.
Tensor grouped_rows(Tensor a, Tensor b, c10::optional<Tensor> offs,
                    at::ScalarType out) {
  TORCH_CHECK(a.is_cuda() && b.device() == a.device(),
              "operands must be on one GPU");
  TORCH_CHECK(a.dim() == 2 && b.dim() == 3 && a.size(1) == b.size(1) &&
              a.scalar_type() == b.scalar_type(), "operands do not match");
  const c10::hip::HIPGuard guard(a.device().index());
  const int64_t T = a.size(0), K = a.size(1), N = b.size(2), E = b.size(0);
  GroupedArgs p = {};
  p.T = dim32(T, "rows");
  p.K = dim32(K, "inner size");
  p.N = dim32(N, "columns");
  p.E = dim32(E, "groups");
  const int ty = type_of(a.scalar_type());
  TORCH_CHECK(ty != GT_FP8);
  set_offsets(p, offs, a, E);
  a = readable(a);
  b = readable(b);
  Tensor c = torch::empty({T, N}, a.options().dtype(out));
  if (c.numel() == 0) return c;
  if (E == 0 || K == 0) return c.zero_();
  a = rows_contiguous(a);
  bool bk = K == 1 || b.stride(1) == 1;
  if (!bk && N > 1 && b.stride(2) != 1) b = b.contiguous();
  const int64_t epc = 16 / a.element_size();
  p.a = a.data_ptr();
  p.b = b.data_ptr();
  p.c = c.data_ptr();
  p.lda = T > 1 ? a.stride(0) : 0;
  p.ldb = bk ? (N > 1 ? b.stride(2) : 0) : b.stride(1);
  p.gsb = E > 1 ? b.stride(0) : 0;
  p.out = type_of(out);
  const int path = !near_rows(a, p.lda, K) ||
                           !near_rows(b, p.ldb, bk ? K : N) ? 2
                   : aligned(a, p.lda, T) && aligned(b, p.ldb, bk ? N : K) &&
                           aligned(b, p.gsb, E) && (bk || N % epc == 0) ? 0
                   : 1;
  const Plan plan = choose_rows(ty, bk, path == 0, T, E, K, N);
  const hipStream_t s = stream_of(a);
  check_grid(p, plan.tile, path, false);
  const Tensor part = begin(p, c, plan.splits);
  launch_rows(p, ty, plan.tile, bk, path, s);
  finish(p, c, s);
  return c;
}

// c[g] = a_g^T @ b_g over the rows of each group, zeros for an empty one.
// a [T, M], b [T, N].
Tensor grouped_weights(Tensor a, Tensor b, c10::optional<Tensor> offs,
                       int64_t E, at::ScalarType out) {
  TORCH_CHECK(a.is_cuda() && b.device() == a.device(),
              "operands must be on one GPU");
  TORCH_CHECK(a.dim() == 2 && b.dim() == 2 && a.size(0) == b.size(0) &&
              a.scalar_type() == b.scalar_type(), "operands do not match");
  const c10::hip::HIPGuard guard(a.device().index());
  const int64_t T = a.size(0), M = a.size(1), N = b.size(1);
  GroupedArgs p = {};
  p.T = dim32(T, "rows");
  p.M = dim32(M, "columns of a");
  p.N = dim32(N, "columns of b");
  p.K = p.T;
  p.E = dim32(E, "groups");
  const int ty = type_of(a.scalar_type());
  TORCH_CHECK(ty != GT_FP8);
  set_offsets(p, offs, a, E);
  a = readable(a);
  b = readable(b);
  Tensor c = torch::empty({E, M, N}, a.options().dtype(out));
  if (c.numel() == 0) return c;
  if (T == 0) return c.zero_();
  a = rows_contiguous(a);
  b = rows_contiguous(b);
  const int64_t epc = 16 / a.element_size();
  p.a = a.data_ptr();
  p.b = b.data_ptr();
  p.c = c.data_ptr();
  p.lda = T > 1 ? a.stride(0) : 0;
  p.ldb = T > 1 ? b.stride(0) : 0;
  p.out = type_of(out);
  const int path = !near_rows(a, p.lda, M) || !near_rows(b, p.ldb, N) ? 2
                   : aligned(a, p.lda, T) && aligned(b, p.ldb, T) &&
                           M % epc == 0 && N % epc == 0 ? 0
                   : 1;
  const int64_t k_tiles = T / E / (ty == GT_F32 ? 32 : 64);
  const auto count = [&](int64_t bm, int64_t bn) {
    return E * ceil_div(M, bm) * ceil_div(N, bn);
  };
  // the sums of several groups have uneven lengths, which many tiles even out,
  // unless they are short beside the writing of the results
  const bool even = E <= 4 || T / E <= 128;
  const Plan plan =
      choose(ty, path == 0,
             even ? large_pays(count(256, 256), count(128, 128))
                  : count(256, 256) >= 800,
             even ? 250 : 640, k_tiles, count);
  const int tile = plan.tile;
  const hipStream_t s = stream_of(a);
  check_grid(p, tile, path, true);
  const Tensor part = begin(p, c, plan.splits);
  if (ty == GT_BF16) launch_grouped_bf16(&p, tile, 0, 1, path, s);
  else if (ty == GT_F16) launch_grouped_f16(&p, tile, 0, 1, path, s);
  else launch_grouped_f32(&p, tile, 0, 1, path, s);
  finish(p, c, s);
  return c;
}

std::tuple<Tensor, Tensor> fp8_quantize_row(Tensor x);

// c = a @ bt[group]^T of e4m3 operands: a [T, K] with scales [kb][T], or a
// wider a without scales that is quantized by rows, bt [E, N, K] with scales
// [E][kb][nb], or one matrix. With `into` (f32, contiguous), the product is
// written there, or added where `accum` is set.
Tensor grouped_rows_fp8(Tensor a, c10::optional<Tensor> a_scales, Tensor bt,
                        Tensor bsc, c10::optional<Tensor> offs,
                        at::ScalarType out, c10::optional<Tensor> into,
                        bool accum) {
  TORCH_CHECK(a.is_cuda() && bt.device() == a.device() &&
              bsc.device() == a.device(), "operands must be on one GPU");
  if (bt.dim() == 2) {
    bt = bt.unsqueeze(0);
    bsc = bsc.unsqueeze(0);
  }
  TORCH_CHECK(a.dim() == 2 && bt.dim() == 3 && a.size(1) == bt.size(2) &&
              bt.scalar_type() == torch::kFloat8_e4m3fn && bt.is_contiguous(),
              "operands do not match");
  const c10::hip::HIPGuard guard(a.device().index());
  a = readable(a);
  bt = readable(bt);
  bsc = readable(bsc);
  const int64_t T = a.size(0), K = a.size(1), N = bt.size(1), E = bt.size(0);
  const int64_t kb = (K + 127) / 128, nb = (N + 127) / 128;
  Tensor asc;
  if (a_scales.has_value()) {
    asc = readable(*a_scales);
    TORCH_CHECK(a.scalar_type() == torch::kFloat8_e4m3fn &&
                a.is_contiguous(), "a with scales must be contiguous e4m3");
    TORCH_CHECK(asc.device() == a.device() &&
                asc.scalar_type() == torch::kFloat32 && asc.is_contiguous() &&
                asc.dim() == 2 && asc.size(0) == kb && asc.size(1) == T,
                "scales of a must be float32 [ceil(K/128), rows]");
  } else {
    std::tie(a, asc) = fp8_quantize_row(a);
  }
  TORCH_CHECK(bsc.scalar_type() == torch::kFloat32 && bsc.is_contiguous() &&
              bsc.dim() == 3 && bsc.size(0) == E && bsc.size(1) == kb &&
              bsc.size(2) == nb,
              "scales of bt must be float32 [groups, ceil(K/128), "
              "ceil(N/128)]");
  GroupedArgs p = {};
  p.T = dim32(T, "rows");
  p.K = dim32(K, "inner size");
  p.N = dim32(N, "columns");
  p.E = dim32(E, "groups");
  set_offsets(p, offs, a, E);
  Tensor c;
  if (into.has_value()) {
    c = *into;
    TORCH_CHECK(!c.is_neg() && !c._is_zerotensor() &&
                c.scalar_type() == torch::kFloat32 && c.is_contiguous() &&
                c.device() == a.device() && c.dim() == 2 && c.size(0) == T &&
                c.size(1) == N, "the result must be float32 [rows, columns]");
  } else {
    c = torch::empty({T, N}, a.options().dtype(out));
  }
  if (c.numel() == 0) return c;
  if (E == 0 || K == 0) return accum ? c : c.zero_();
  p.a = a.data_ptr();
  p.b = bt.data_ptr();
  p.c = c.data_ptr();
  p.asc = asc.data_ptr<float>();
  p.bsc = bsc.data_ptr<float>();
  p.lda = T > 1 ? K : 0;
  p.ldb = N > 1 ? K : 0;
  p.gsb = E > 1 ? N * K : 0;
  p.out = type_of(c.scalar_type());
  p.accum = accum;
  const int path = !near_rows(a, p.lda, K) || !near_rows(bt, p.ldb, K) ? 2
                   : aligned(a, p.lda, T) && aligned(bt, p.ldb, N) &&
                           aligned(bt, p.gsb, E) ? 0
                   : 1;
  const Plan plan = choose_rows(GT_FP8, true, path == 0, T, E, K, N);
  const hipStream_t s = stream_of(a);
  check_grid(p, plan.tile, path, false);
  const Tensor part = begin(p, c, accum ? 1 : plan.splits);
  launch_rows(p, GT_FP8, plan.tile, true, path, s);
  finish(p, c, s);
  return c;
}

// [R, C] -> (e4m3 [R, C], scales [ceil(C/128), R])
std::tuple<Tensor, Tensor> fp8_quantize_row(Tensor x) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2);
  const c10::hip::HIPGuard guard(x.device().index());
  const int64_t R = x.size(0), C = x.size(1);
  x = rows_contiguous(readable(x));
  const int ty = type_of(x.scalar_type());
  TORCH_CHECK(ty != GT_FP8);
  Tensor q = torch::empty({R, C}, x.options().dtype(torch::kFloat8_e4m3fn));
  Tensor s = torch::empty({(C + 127) / 128, R},
                          x.options().dtype(torch::kFloat32));
  if (q.numel() == 0) return {q, s};
  // a launch holds fewer than 2^32 threads
  TORCH_CHECK((C + 127) / 128 * ((R + 15) / 16) < (int64_t(1) << 24),
              "matrix is too large");
  const int64_t ld = R > 1 ? x.stride(0) : 0;
  launch_fp8_quantize_row(x.data_ptr(), ty, ld, R, C, q.data_ptr(),
                          s.data_ptr<float>(), stream_of(x));
  check_launch();
  return {q, s};
}

// [E, R, C] -> (e4m3 [E, R, C], scales [E, ceil(C/128), ceil(R/128)]), and
// with `both` the same for the transposed matrices.
std::tuple<Tensor, Tensor, Tensor, Tensor> fp8_quantize_tile(Tensor x,
                                                             bool both) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 3);
  const c10::hip::HIPGuard guard(x.device().index());
  const int64_t E = x.size(0), R = x.size(1), C = x.size(2);
  x = rows_contiguous(readable(x));
  const int ty = type_of(x.scalar_type());
  TORCH_CHECK(ty != GT_FP8);
  const int64_t rb = (R + 127) / 128, cb = (C + 127) / 128;
  const auto o8 = x.options().dtype(torch::kFloat8_e4m3fn);
  const auto of = x.options().dtype(torch::kFloat32);
  Tensor q = torch::empty({E, R, C}, o8), s = torch::empty({E, cb, rb}, of);
  Tensor qt, st;
  if (both) {
    qt = torch::empty({E, C, R}, o8);
    st = torch::empty({E, rb, cb}, of);
  } else {
    qt = torch::empty({0}, o8);
    st = torch::empty({0}, of);
  }
  if (q.numel() == 0) return {q, s, qt, st};
  TORCH_CHECK(rb * cb < (int64_t(1) << 24), "matrix is too large");
  const int64_t ld = R > 1 ? x.stride(1) : 0, bld = E > 1 ? x.stride(0) : 0;
  const auto at = [](const Tensor& t, int64_t i) {
    return (char*)t.data_ptr() + i * t.element_size();
  };
  for (int64_t e = 0; e < E; e += 65535)  // what a launch's grid holds
    launch_fp8_quantize_tile(
        at(x, e * bld), ty, ld, bld, std::min<int64_t>(E - e, 65535), R, C,
        at(q, e * R * C), both ? at(qt, e * R * C) : nullptr,
        (float*)at(s, e * rb * cb),
        both ? (float*)at(st, e * rb * cb) : nullptr, stream_of(x));
  check_launch();
  return {q, s, qt, st};
}

// e4m3 [E, R, C] -> [E, C, R]
Tensor fp8_turn(Tensor q) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 3 && q.is_contiguous() &&
              q.scalar_type() == torch::kFloat8_e4m3fn,
              "needs contiguous e4m3 matrices");
  const c10::hip::HIPGuard guard(q.device().index());
  const int64_t E = q.size(0), R = q.size(1), C = q.size(2);
  q = readable(q);
  Tensor qt = torch::empty({E, C, R}, q.options());
  if (q.numel() == 0) return qt;
  TORCH_CHECK((R + 127) / 128 * ((C + 127) / 128) < (int64_t(1) << 24),
              "matrix is too large");
  for (int64_t e = 0; e < E; e += 65535)  // what a launch's grid holds
    launch_fp8_turn((const char*)q.data_ptr() + e * R * C,
                    std::min<int64_t>(E - e, 65535), R, C,
                    (char*)qt.data_ptr() + e * R * C, stream_of(q));
  check_launch();
  return qt;
}

// ---- autograd --------------------------------------------------------------

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Gradients that were computed outside of autograd: they say so when they are
// differentiated once more.
variable_list once(variable_list grads, bool create_graph) {
  if (!create_graph) return grads;
  for (auto& g : grads)
    if (g.defined()) g = g.detach().requires_grad_();
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "grouped and 8-bit products are differentiable once only",
      (int64_t)grads.size());
  return (*error)(std::move(grads));
}

c10::optional<Tensor> given(const Tensor& offs) {
  return offs.defined() ? c10::optional<Tensor>(offs) : c10::nullopt;
}

// The one type of a gradient's product: the operands', to which the gradient of
// a wider result is rounded. It can lie outside of fp16's range (the products
// of 1e5 and 1e-4 are not infinite): all is multiplied in float32 there.
at::ScalarType product_type(const Tensor& grad, at::ScalarType ty) {
  return ty == torch::kFloat16 && grad.scalar_type() != ty ? torch::kFloat32
                                                           : ty;
}

Tensor grad_a(const Tensor& grad, const Tensor& b,
              const c10::optional<Tensor>& offs) {
  return grouped_rows(grad, b.to(grad.scalar_type()).transpose(1, 2), offs,
                      b.scalar_type());
}

// In the memory order of b, so that an optimizer walks both alike.
Tensor grad_b(const Tensor& grad, const Tensor& a, const Tensor& b,
              const c10::optional<Tensor>& offs) {
  const Tensor x = a.to(grad.scalar_type());
  if (b.stride(1) == 1 && b.size(1) > 1)
    return grouped_weights(grad, x, offs, b.size(0), b.scalar_type())
        .transpose(1, 2);
  return grouped_weights(x, grad, offs, b.size(0), b.scalar_type());
}

struct GroupedMatmul : torch::autograd::Function<GroupedMatmul> {
  static Tensor forward(AutogradContext* ctx, const Tensor& a,
                        const Tensor& b, const Tensor& offs, int64_t out) {
    ctx->save_for_backward({a, b, offs});
    return grouped_rows(a, b, offs, (at::ScalarType)out);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool again = at::GradMode::is_enabled();
    const at::NoGradGuard guard;
    const auto saved = ctx->get_saved_variables();
    const Tensor &a = saved[0], &b = saved[1], &offs = saved[2];
    const Tensor grad = rows_contiguous(
        grads[0].to(product_type(grads[0], a.scalar_type())));
    Tensor da, db;
    if (ctx->needs_input_grad(0)) da = grad_a(grad, b, offs);
    if (ctx->needs_input_grad(1)) db = grad_b(grad, a, b, offs);
    auto r = once({da, db}, again);
    return {r[0], r[1], Tensor(), Tensor()};
  }
};

Tensor grouped_matmul(Tensor a, Tensor b, Tensor offs, at::ScalarType out) {
  return GroupedMatmul::apply(a, b, offs, (int64_t)out);
}

// w [N, K] or [E, N, K], quantized here; or already quantized in q and s.
struct Fp8Matmul : torch::autograd::Function<Fp8Matmul> {
  typedef std::optional<Tensor> Maybe;
  static Tensor forward(AutogradContext* ctx, const Tensor& a, const Maybe& w,
                        const Maybe& q, const Maybe& s, const Maybe& offs,
                        int64_t out) {
    Tensor bt, bsc, turned, turned_sc;
    ctx->saved_data["frozen"] = !w.has_value();
    ctx->saved_data["a_type"] = (int64_t)a.scalar_type();
    bool keep = false;
    if (w.has_value()) {
      std::tie(bt, bsc, turned, turned_sc) = fp8_quantize_tile(
          w->dim() == 3 ? *w : w->unsqueeze(0), a.requires_grad());
      ctx->saved_data["w_type"] = (int64_t)w->scalar_type();
      ctx->saved_data["w_shape"] = w->sizes().vec();
      keep = w->requires_grad();
    } else {  // turned when the gradient is wanted
      turned = bt = *q;
      turned_sc = bsc = *s;
    }
    ctx->save_for_backward({keep ? a : Tensor(), turned, turned_sc,
                            offs.has_value() ? *offs : Tensor()});
    return grouped_rows_fp8(a, c10::nullopt, bt, bsc, offs,
                            (at::ScalarType)out, c10::nullopt, false);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool again = at::GradMode::is_enabled();
    const at::NoGradGuard guard;
    const auto saved = ctx->get_saved_variables();
    const auto a_type = (at::ScalarType)ctx->saved_data["a_type"].toInt();
    const c10::optional<Tensor> offs = given(saved[3]);
    const Tensor grad = rows_contiguous(grads[0]);
    Tensor da, dw;
    if (ctx->needs_input_grad(0)) {
      Tensor bt = saved[1], bsc = saved[2];
      if (ctx->saved_data["frozen"].toBool()) {
        bt = fp8_turn(bt.dim() == 3 ? bt : bt.unsqueeze(0));
        if (bsc.dim() == 2) bsc = bsc.unsqueeze(0);
        bsc = bsc.transpose(-1, -2).contiguous();
      }
      da = grouped_rows_fp8(grad, c10::nullopt, bt, bsc, offs, a_type,
                            c10::nullopt, false);
    }
    if (!ctx->saved_data["frozen"].toBool() && ctx->needs_input_grad(1)) {
      // in the operands' own type: the sum runs over rows, along which
      // neither has its scales
      const auto shape = ctx->saved_data["w_shape"].toIntVector();
      const auto ty = product_type(grad, a_type);
      dw = grouped_weights(rows_contiguous(grad.to(ty)), saved[0].to(ty), offs,
                           shape.size() == 2 ? 1 : shape[0],
                           (at::ScalarType)ctx->saved_data["w_type"].toInt())
               .reshape(shape);
    }
    auto r = once({da, dw}, again);
    return {r[0], r[1], Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor fp8_matmul(Tensor a, c10::optional<Tensor> w, c10::optional<Tensor> q,
                  c10::optional<Tensor> s, c10::optional<Tensor> offs,
                  at::ScalarType out) {
  TORCH_CHECK(w.has_value() || (q.has_value() && s.has_value()));
  return Fp8Matmul::apply(a, w, q, s, offs, (int64_t)out);
}

// Whether a stream is being captured. The default stream (id 0) never is, and
// must not be asked while another thread captures.
bool is_captured(const c10::hip::HIPStream& s) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (s.id() == 0) return false;
  const hipError_t e = hipStreamIsCapturing(s.stream(), &status);
  TORCH_CHECK(e == hipSuccess, "HIP error: ", hipGetErrorString(e));
  return status != hipStreamCaptureStatusNone;
}

bool capturing(const Tensor& t) {
  return is_captured(c10::hip::getCurrentHIPStream(t.device().index()));
}

// Whether the backward pass behind t, a leaf or not, would run nodes on a
// stream that is neither the current one nor captured with it: those of a
// leaf that an autograd graph from there still holds, or of what was computed
// there.
bool held_by_other_stream(const Tensor& t) {
  using torch::autograd::Node;
  if (!t.requires_grad()) return false;
  std::vector<std::shared_ptr<Node>> left = {
      t.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(t)
                  : t.grad_fn()};
  std::unordered_set<Node*> met;
  while (!left.empty()) {
    const std::shared_ptr<Node> node = std::move(left.back());
    left.pop_back();
    if (!node || !met.insert(node.get()).second) continue;
    if (const auto s = node->stream()) {
      // by id: the one is of device type "cuda", the other "hip"
      if (s->id() != c10::hip::getCurrentHIPStream(s->device_index()).id() &&
          !is_captured(c10::hip::HIPStream(c10::hip::HIPStream::UNCHECKED, *s)))
        return true;
    }
    for (const auto& edge : node->next_edges()) left.push_back(edge.function);
  }
  return false;
}

}  // namespace

void bind_grouped(pybind11::module& m) {
  m.def("grouped_rows", &grouped_rows,
        "rows of each group times the group's matrix");
  m.def("grouped_weights", &grouped_weights,
        "each group's a^T @ b over its rows");
  m.def("grouped_rows_fp8", &grouped_rows_fp8,
        "grouped product of e4m3 operands with block scales");
  m.def("fp8_quantize_row", &fp8_quantize_row,
        "e4m3 with a scale for each 128 of a row");
  m.def("fp8_quantize_tile", &fp8_quantize_tile,
        "e4m3 with a scale for each 128 x 128 tile");
  m.def("fp8_turn", &fp8_turn, "e4m3 matrices transposed");
  m.def("grouped_matmul", &grouped_matmul, "differentiable grouped_rows");
  m.def("fp8_matmul", &fp8_matmul, "differentiable grouped_rows_fp8");
  m.def("capturing", &capturing,
        "whether the current stream of a tensor's device is captured");
  m.def("held_by_other_stream", &held_by_other_stream,
        "whether a tensor's backward pass would run on another stream");
}
