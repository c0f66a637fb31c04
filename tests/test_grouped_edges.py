"""Grouped and 8-bit products where operands, sizes and modes end: column
blocks past the last column, captures beside eager graphs, forward mode,
scales and gradients near the ends of a type's range.

Tolerances as in test_grouped_fp8.py."""

import os
import subprocess

import pytest
import torch
import torch.autograd.forward_ad as fwd

import matrel_amd as ma
from test_grouped_fp8 import (DEVICES, assert_near, fp8_cut, offsets_of,
                              plain_rows, plain_weights, randn, values_of)

CSRC = os.path.join(os.path.dirname(os.path.abspath(ma.__file__)), "csrc")

# Every row of b that the few-rows kernel's ring reads: block j of the NB of a
# workgroup, its 16 rows, for all workgroups of n columns.
FEW_ROWS = r"""
#include "grouped_args.h"
#include <cstdio>
int main() {
  for (int nb : {1, 2, 4})
    for (int n = 1; n <= 300; ++n)
      for (int n0 = 0; n0 < n; n0 += 16 * nb)
        for (int j = 0; j <= nb; ++j)  // the ring steps on once too often
          for (int i = 0; i < 16; ++i) {
            const int block = few_rows_block(n, n0, j);
            const int last = few_rows_row(n, block, 15);
            const int row = block + (i < last ? i : last);
            const int want = n0 + j * 16 + i;
            if (row < 0 || row >= n || row != block + few_rows_row(n, block, i)
                || (want < n && j < nb && row != want)) {
              std::printf("nb %d n %d n0 %d block %d row %d reads %d\n", nb, n,
                          n0, j, i, row);
              return 1;
            }
          }
}
"""


def test_few_rows_reads_rows_that_exist(tmp_path):
    src, exe = tmp_path / "few.cpp", tmp_path / "few"
    src.write_text(FEW_ROWS)
    subprocess.run(["g++", "-std=c++17", "-I", CSRC, str(src), "-o",
                    str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16,
                                   torch.float32])
@pytest.mark.parametrize("sizes,k,n", [
    ([1] * 64, 256, 1400),       # 16 rows, two blocks, 24 columns left
    ([3] * 16, 256, 4120),       # the same, 24 left
    ([2] * 140, 128, 1000),      # four blocks, 40 left
    ([20] * 12, 256, 1400),      # 32 rows, two blocks
    ([20] * 140, 128, 1000)])    # 32 rows, four blocks
def test_few_rows_last_columns(sizes, k, n, dtype):
    """Column blocks that end early behind others of their workgroup."""
    off = offsets_of(sizes, "cuda")
    a = randn(sum(sizes), k, seed=1, dtype=dtype, device="cuda")
    w = randn(len(sizes), n, k, seed=2, dtype=dtype, device="cuda")
    b = w.transpose(1, 2)
    assert_near(ma.grouped_matmul(a, b, off), *plain_rows(a, b, off), k)
    qa, qw = ma.quantize_fp8(a), ma.quantize_fp8(w, "tile")
    assert_near(ma.fp8_matmul(qa, qw, off, out_dtype=dtype),
                *plain_rows(values_of(qa), values_of(qw).transpose(1, 2), off),
                k, fp8_cut(qa, qw, off))


@pytest.mark.parametrize("device", DEVICES)
def test_forward_mode(device):
    """A tangent is carried in full or refused, never dropped."""
    off = offsets_of([3, 5], device)
    a = randn(8, 136, seed=3, device=device)
    w = randn(2, 24, 136, seed=4, device=device)
    ta, tw = randn(8, 136, seed=5, device=device), \
        randn(2, 24, 136, seed=6, device=device)
    gy = randn(8, 24, seed=7, device=device)
    qa, qw = ma.quantize_fp8(a), ma.quantize_fp8(w, "tile")
    with fwd.dual_level():
        da, dw = fwd.make_dual(a, ta), fwd.make_dual(w, tw)
        # with and without a backward pass beside it
        for x in (da, fwd.make_dual(a.clone().requires_grad_(), ta)):
            for f in (lambda: ma.fp8_matmul(x, w, off),
                      lambda: ma.fp8_matmul(x, qw, off)):
                with pytest.raises(NotImplementedError):
                    f()
        for f in (lambda: ma.fp8_matmul(a, dw, off),
                  lambda: ma.fp8_matmul(qa, dw, off)):
            with pytest.raises(NotImplementedError):
                f()
        b = w.transpose(1, 2)
        calls = ((da, b), (a, dw.transpose(1, 2)), (da, dw.transpose(1, 2)))
        for x, y in calls:
            if device == "cuda":
                with pytest.raises(NotImplementedError):
                    ma.grouped_matmul(x, y, off)
                with pytest.raises(NotImplementedError):
                    ma.grouped_matmul_grads(gy, x, y, off)
                continue
            got = fwd.unpack_dual(ma.grouped_matmul(x, y, off)).tangent
            want = torch.zeros(8, 24, dtype=torch.float64)
            size = torch.zeros_like(want)
            if x is da:
                p = plain_rows(ta, b, off)
                want, size = want + p[0], size + p[1]
            if y is not b:
                p = plain_rows(a, tw.transpose(1, 2), off)
                want, size = want + p[0], size + p[1]
            assert_near(got, want, size, 2 * 136)
        # no tangent: as ever, also inside of a level
        assert torch.equal(ma.fp8_matmul(a, w, off),
                           ma.fp8_matmul(qa, qw, off, torch.float32))
        assert fwd.unpack_dual(ma.grouped_matmul(a, b, off)).tangent is None
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: ma.fp8_matmul(x, w, off), (a,), (ta,))


@pytest.mark.gpu
def test_capture_guard_sees_through_views():
    """What a graph of another stream holds, behind views and casts too."""
    from matrel_amd.ops.backend import require_ext
    held = require_ext().held_by_other_stream
    w = randn(2, 64, 64, seed=8, device="cuda").requires_grad_()
    x = randn(9, 64, seed=9, device="cuda").requires_grad_()
    forms = (lambda: w, lambda: w.transpose(1, 2),
             lambda: w.to(torch.bfloat16), lambda: (w * 2)[:, :8],
             lambda: w[0].expand(3, 64, 64))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    assert not any(held(f()) for f in forms)
    with torch.cuda.stream(side):  # no graph lives: nothing is held
        assert not any(held(f()) for f in forms)
        assert not held(w.detach()) and not held(torch.ones(3, device="cuda"))
    torch.cuda.synchronize()
    alive = w * 1
    outside = x * 1
    assert not any(held(f()) for f in forms)
    with torch.cuda.stream(side):
        assert all(held(f()) for f in forms)
        assert held(outside) and held(outside[:4]) and not held(w.detach())
    del alive, outside
    with torch.cuda.stream(side):
        assert not any(held(f()) for f in forms) and not held(x)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_capture_beside_a_living_graph_of_a_view():
    """A captured forward pass is refused for views of held leaves and for
    operands that were computed outside, and for nothing else."""
    bf = dict(dtype=torch.bfloat16, device="cuda")
    a = randn(64, 64, seed=10, **bf)
    w = randn(2, 64, 64, seed=11, **bf).requires_grad_()
    free = randn(2, 64, 64, seed=12, **bf).requires_grad_()
    off = offsets_of([30, 34], "cuda")
    alive = ma.grouped_matmul(a, w.transpose(1, 2), off)
    outside = randn(64, 64, seed=13, **bf).requires_grad_() * 2
    want = ma.grouped_matmul(a, free.transpose(1, 2), off).detach()
    torch.cuda.synchronize()
    refused, taken = 0, []
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for f in (lambda: ma.grouped_matmul(a, w.transpose(1, 2), off),
                  lambda: ma.fp8_matmul(a, w.reshape(2, 64, 64), off),
                  lambda: ma.grouped_matmul(outside, free, off),
                  lambda: ma.fp8_matmul(outside, free, off)):
            try:
                f()
            except RuntimeError as e:
                refused += "outside of this capture" in str(e)
        taken.append(ma.grouped_matmul(a, free.transpose(1, 2), off))
        taken.append(ma.grouped_matmul(a, w.detach().transpose(1, 2), off))
        # a stream that the capture itself forks is inside
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            forked = free.transpose(1, 2) * 1
        torch.cuda.current_stream().wait_stream(side)
        taken.append(ma.grouped_matmul(a, forked, off))
    assert refused == 4 and len(taken) == 3
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(taken[0], want) and torch.equal(taken[2], want)
        assert torch.equal(taken[1], alive)


def far_scales(sizes, k, n, meet):
    """Operands with a block pair whose scales' product passes float32 while
    the values' products do not: 0 everywhere, or 2^119 at one k. Also the
    operands without that pair."""
    a = randn(sum(sizes), k, seed=14, dtype=torch.bfloat16)
    w = randn(len(sizes), n, k, seed=15, dtype=torch.bfloat16)
    at = 128 if k > 256 else 0
    a[:, at:at + 128], w[..., at:at + 128] = 0, 0
    a0, w0 = a.clone(), w.clone()
    a[:, at + 1], w[..., at + 2] = 2.0 ** 75, 2.0 ** 72
    if meet:  # 1.75 * 2^-6 in both payloads
        a[:, at + 5], w[..., at + 5] = 2.0 ** 61, 2.0 ** 58
    return a, w, a0, w0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("meet", [False, True])
@pytest.mark.parametrize("sizes,k,n", [
    ([3], 384, 200), ([2, 3], 389, 200), ([20, 9], 384, 72),  # few rows
    ([70], 4096, 200),                                        # split sums
    ([70, 1, 60], 384, 136), ([70, 1, 60], 389, 136),
    ([100, 100], 7, 40),
    ([2000, 1, 2099], 320, 1032), ([1300, 1, 1299], 320, 4104)])
def test_fp8_scales_beyond_float32(sizes, k, n, meet, device):
    """Sums are taken again by values there, without the matrix unit: nothing
    is cut off but in the other blocks of a split sum."""
    a, w, a0, w0 = (t.to(device) for t in far_scales(sizes, k, n, meet))
    off = offsets_of(sizes, device)
    qa, qw = ma.quantize_fp8(a), ma.quantize_fp8(w, "tile")
    want = plain_rows(values_of(qa), values_of(qw).transpose(1, 2), off)
    cut = fp8_cut(ma.quantize_fp8(a0), ma.quantize_fp8(w0, "tile"), off)
    for dtype in (torch.float32, torch.bfloat16):
        y = ma.fp8_matmul(qa, qw, off, dtype)
        assert_near(y, *want, k, cut)
    # what is not finite by its values stays so, and in its place
    a[1, 0] = float("inf")
    y = ma.fp8_matmul(a, qw, off, torch.float32)
    assert torch.isnan(y[1]).all()
    y[1] = 0
    assert torch.isfinite(y).all()


@pytest.mark.gpu
def test_fp8_scales_beyond_float32_accumulate():
    from matrel_amd.ops import blockops
    a, w, _, _ = (t.cuda() for t in far_scales([90], 384, 72, False))
    qa, sa = blockops.to_fp8(a, "row")
    qb, sb = blockops.to_fp8(w[0], "tile")
    acc = torch.full((90, 72), 3.0, device="cuda")
    blockops.gemm_bt_fp8_acc(acc, qa, sa, qb, sb, beta0=True)
    one = acc.clone()
    assert torch.isfinite(one).all()
    blockops.gemm_bt_fp8_acc(acc, qa, sa, qb, sb)
    assert torch.equal(acc, 2 * one)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e5, 1e-9])
@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_wide_gradient_of_half_operands(layout, size, out, device):
    """Gradients that float16 does not hold, of products that it does."""
    hf = dict(dtype=torch.float16, device=device)
    off = offsets_of([20, 0, 45], device)
    unit = 1e-4 if size > 1 else 1e3
    a = randn(65, 72, seed=16, scale=unit, **hf).requires_grad_()
    w = randn(3, 40, 72, seed=17, scale=unit, **hf)
    if layout == "kn":
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    w.requires_grad_()
    gy = randn(65, 40, seed=18, dtype=out, device=device, scale=size)
    want_a = plain_rows(gy, w, off)
    want_w = plain_weights(gy, a, off)
    y = ma.grouped_matmul(a, w.transpose(1, 2), off, out)
    da, dw = torch.autograd.grad(y, (a, w), gy)
    assert da.dtype == dw.dtype == torch.float16
    assert_near(da, *want_a, 40)
    assert_near(dw, *want_w, 45)
    da2, db2 = ma.grouped_matmul_grads(gy, a, w.transpose(1, 2), off)
    assert torch.equal(da, da2) and torch.equal(dw, db2.transpose(1, 2))
    y = ma.fp8_matmul(a, w, off, out)
    da, dw = torch.autograd.grad(y, (a, w), gy)
    assert_near(dw, *want_w, 45)
    qg, qw = ma.quantize_fp8(gy), ma.quantize_fp8(w, "tile")
    assert_near(da, *plain_rows(values_of(qg), values_of(qw), off), 40,
                fp8_cut(qg, qw.transpose(), off))


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [200, 100, 72, 33])
def test_engine_fp8_any_block_size(bs, monkeypatch):
    """gemm_precision="fp8" multiplies 8-bit blocks of any size, local and by
    SUMMA's panels (over RCCL with one rank)."""
    import torch.distributed as dist
    from matrel_amd.exec import runtime, summa
    old = ma.get_config()
    runtime.reset_runtime()
    os.environ.setdefault("MASTER_ADDR", "127.0.0.1")
    os.environ.setdefault("MASTER_PORT", "29419")
    dist.init_process_group("nccl", rank=0, world_size=1)
    try:
        s = ma.MatrelSession(ma.MatrelConfig(block_size=bs,
                                             gemm_precision="fp8"))
        m, k, n = 300, 250, 210
        ta = randn(m, k, seed=19, dtype=torch.bfloat16, device="cuda")
        tb = randn(k, n, seed=20, dtype=torch.bfloat16, device="cuda")
        local = (s.from_dense(ta) @ s.from_dense(tb)).to_tensor()
        a, b = s.from_dense(ta).plan.data, s.from_dense(tb).plan.data
        out = ma.BlockMatrix(m, n, block_size=bs)
        rt = runtime.get_runtime()
        monkeypatch.setattr(type(rt), "is_distributed", True)
        monkeypatch.setattr(type(rt), "row_group",
                            lambda self, p: dist.group.WORLD)
        monkeypatch.setattr(type(rt), "col_group",
                            lambda self, q: dist.group.WORLD)
        summa.summa_matmul(a, b, out)
        panels = torch.cat([torch.cat([out.blocks[i, j] for j in
                                       range(-(-n // bs))], 1)
                            for i in range(-(-m // bs))])
        exact = torch.zeros(m, n, dtype=torch.float64)
        size, cut = torch.zeros_like(exact), torch.zeros_like(exact)
        for p in range(0, k, bs):
            qa = ma.quantize_fp8(ta[:, p:p + bs])
            for j in range(0, n, bs):
                qb = ma.quantize_fp8(tb[p:p + bs, j:j + bs].t()[None], "tile")
                off = offsets_of([m], "cuda")
                y, z = plain_rows(values_of(qa), values_of(qb).transpose(1, 2),
                                  off)
                exact[:, j:j + bs] += y
                size[:, j:j + bs] += z
                cut[:, j:j + bs] += fp8_cut(qa, qb, off)
        for got in (local, panels):
            assert got.shape == (m, n)
            assert_near(got.to(torch.bfloat16), exact, size, k, cut)
    finally:
        monkeypatch.undo()
        dist.destroy_process_group()
        ma.set_config(old)
        runtime.reset_runtime()


@pytest.mark.gpu
def test_quantize_many_matrices():
    """More matrices than a launch's grid holds, and their product's step."""
    x = randn(70000, 3, 5, seed=21, device="cuda")
    r = ma.quantize_fp8(x, "tile")
    want = ma.quantize_fp8(x.cpu(), "tile")
    assert torch.equal(r.scale.cpu(), want.scale)
    assert torch.equal(r.data.cpu().float(), want.data.float())
    a = randn(70000, 5, seed=22, device="cuda").requires_grad_()
    w = x.requires_grad_()
    off = torch.arange(70001, device="cuda", dtype=torch.int32)
    gy = randn(70000, 3, seed=23, device="cuda")
    y = ma.fp8_matmul(a, w, off)
    da, dw = torch.autograd.grad(y, (a, w), gy)
    qa, qg = ma.quantize_fp8(a), ma.quantize_fp8(gy)
    v = values_of(r)

    def rows(p, m):  # one row a group
        p = p[:, None, :]
        return [torch.bmm(f(p), f(m).contiguous())[:, 0]
                for f in (lambda t: t, torch.abs)]

    # 5 and 3 products of one group of 8 neighbours
    for got, q, m in ((y, qa, v.transpose(1, 2)), (da, qg, v)):
        exact, size = rows(values_of(q), m)
        top = (q.data.cpu().float().abs().amax(1).clamp(min=2.0 ** -6)
               .double() * q.scale.cpu()[0].double())
        wtop = (r.data.cpu().float().abs().amax((1, 2)).clamp(min=2.0 ** -6)
                .double() * r.scale.cpu().reshape(-1).double())
        cut = 7 * 2.0 ** -13 * (top * wtop)[:, None].expand_as(exact)
        assert_near(got, exact, size, 8, cut)
    p = gy.detach().cpu().double()[:, :, None] * a.detach().cpu().double()[
        :, None, :]
    assert_near(dw, p, p.abs(), 1)


def test_cpu_forms_under_other_defaults():
    """Sums of CPU tensors are float32 ones on the CPU, whatever torch makes
    tensors of by default."""
    a, w = randn(40, 300, seed=24), randn(2, 24, 300, seed=25)
    gy = randn(40, 24, seed=26)
    off = offsets_of([15, 25], "cpu")

    def step():
        x, m = a.clone().requires_grad_(), w.clone().requires_grad_()
        out = []
        for y in (ma.grouped_matmul(x, m.transpose(1, 2), off),
                  ma.fp8_matmul(x, m, off)):
            out += [y.detach(), *torch.autograd.grad(y, (x, m), gy)]
        return out

    want = step()
    for dtype in (torch.bfloat16, torch.float64):
        torch.set_default_dtype(dtype)
        try:
            got = step()
        finally:
            torch.set_default_dtype(torch.float32)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    with torch.device("meta"):
        got = step()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_bench_names_the_precision():
    import sys
    sys.path.insert(0, os.path.dirname(os.path.dirname(
        os.path.abspath(__file__))))
    import bench
    assert bench.DTYPES["bf16"] == "bf16"
    assert len(set(bench.DTYPES.values())) == len(bench.DTYPES)
    assert "fp8" in bench.DTYPES["fp8"]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("sizes,k,n", [
    ([1], 8192, 1000), ([3], 8200, 200), ([3], 8195, 200),  # eight waves
    ([3] * 20, 144, 6400), ([3] * 20, 145, 1400), ([20] * 20, 392, 1000),
    ([20, 40], 4096, 300), ([70], 4096, 200), ([70], 4100, 333),
    ([100, 100], 7, 140), ([33, 0, 129, 1, 62], 1000, 264),
    ([33, 0, 129, 1, 62], 1001, 263), ([2000, 1, 2099], 392, 1032),
    ([1300, 1, 1299], 392, 4104), ([2000, 1, 2099], 131, 4099)])
def test_fp8_exact_sums(sizes, k, n, device):
    """Payloads of -1, 0, 1 and scales of powers of two: every sum is a whole
    number below 2^24 of its unit, no step rounds or cuts anything, and one
    value, scale or tail off is a wrong result. 7 bits of 128 products, up to
    7 of the scales and 7 of 65 K tiles make 21; the gradients' payloads, 448
    = 7 * 2^6, make 24 with a factor that is a power of two."""
    off = offsets_of(sizes, device)
    g = torch.Generator().manual_seed(27)
    t, e, kb, nb = sum(sizes), len(sizes), -(-k // 128), -(-n // 128)

    def ints(*shape):
        return torch.randint(-1, 2, shape, generator=g).float()

    def powers(most, *shape):
        return 2.0 ** torch.randint(0, most + 1, shape, generator=g)

    f8 = torch.float8_e4m3fn
    qa = ma.Fp8Blocks(ints(t, k).to(f8).to(device),
                      powers(3, kb, t).to(device), "row")
    qw = ma.Fp8Blocks(ints(e, n, k).to(f8).to(device),
                      powers(4, e, kb, nb).to(device), "tile")
    want = plain_rows(values_of(qa), values_of(qw).transpose(1, 2), off)
    assert want[1].max() < 2.0 ** 24
    y = ma.fp8_matmul(qa, qw, off, torch.float32)
    assert torch.equal(y.cpu().double(), want[0])
    # 448 is the largest value of a block: payloads of 448, scales as given
    gy = ints(t, n) * 448 * powers(3, nb, t).repeat_interleave(
        128, 0)[:n].t()
    a = torch.zeros(t, k, device=device, requires_grad=True)
    da, = torch.autograd.grad(ma.fp8_matmul(a, qw, off), a, gy.to(device))
    want = plain_rows(gy, values_of(qw), off)
    assert (want[1] / 448).max() < 2.0 ** 21
    assert torch.equal(da.cpu().double(), want[0])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape", [
    (1, 1), (1, 300), (300, 1), (128, 128), (130, 257), (3, 136, 264),
    (2, 77, 111), (2, 3, 40, 9), (0, 4, 8), (2, 0, 8), (70000, 3, 5)])
def test_transposed_blocks(shape, device):
    """Bit for bit, every payload among them."""
    g = torch.Generator().manual_seed(28)
    d = torch.randint(0, 256, shape, generator=g, dtype=torch.uint8)
    s = torch.rand(*shape[:-2], -(-shape[-1] // 128), -(-shape[-2] // 128),
                   generator=g)
    q = ma.Fp8Blocks(d.to(device).view(torch.float8_e4m3fn), s.to(device),
                     "tile").transpose()
    assert torch.equal(q.data.view(torch.uint8).cpu(), d.transpose(-1, -2))
    assert torch.equal(q.scale.cpu(), s.transpose(-1, -2))
    assert q.kind == "tile"


@pytest.mark.gpu
@pytest.mark.parametrize("k", [(1 << 31) - (1 << 16), (1 << 31) - 600])
def test_refuses_sizes_near_2_31(k):
    """The last K tiles would be counted past 31 bits. (Nothing is allocated:
    refused before the expanded operands are copied.)"""
    one = torch.zeros(1, dtype=torch.bfloat16, device="cuda")
    off = offsets_of([1], "cuda")
    for a, b in ((one.expand(1, k), one.expand(1, k, 1)),
                 (one.expand(k, 1), one.expand(1, 1, 1)),
                 (one.expand(1, 1), one.expand(1, 1, k))):
        with pytest.raises(RuntimeError, match="too large"):
            ma.grouped_matmul(a, b, off)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("t", [5, 700])
def test_fp8_results_beyond_float32(t, device):
    """What is infinite by its values stays infinite, with its sign."""
    k, n = 520, 300
    a = torch.full((t, k), 2.0 ** 80, device=device)
    w = torch.full((n, k), 2.0 ** 70, device=device)
    w[1::2] *= -1
    y = ma.fp8_matmul(a, w)
    assert (y[:, ::2] == float("inf")).all()
    assert (y[:, 1::2] == -float("inf")).all()
    w[3, 400] = float("nan")
    y = ma.fp8_matmul(a, w)  # its tile: columns 0 .. 127
    assert torch.isnan(y[:, :128]).all()
    assert torch.isinf(y[:, 128:]).all()


@pytest.mark.gpu
def test_operands_without_memory():
    """What torch only marks as negated or zero is read as such; fake tensors
    are refused before anything is launched."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    a = randn(9, 72, seed=31, device="cuda")
    w = randn(2, 40, 72, seed=32, device="cuda")
    off = offsets_of([4, 5], "cuda")
    b = w.transpose(1, 2)
    zero = torch._efficientzerotensor
    for x, m in ((torch._neg_view(a), w), (a, torch._neg_view(w)),
                 (zero(a.shape, device="cuda"), w),
                 (a, zero(w.shape, device="cuda"))):
        assert x.is_neg() or m.is_neg() or x._is_zerotensor() \
            or m._is_zerotensor()
        y, z = x.clone(), m.clone()
        assert torch.equal(ma.grouped_matmul(x, m.transpose(1, 2), off),
                           ma.grouped_matmul(y, z.transpose(1, 2), off))
        assert torch.equal(ma.fp8_matmul(x, m, off), ma.fp8_matmul(y, z, off))
    gy = zero((9, 40), device="cuda")
    assert all((g == 0).all() for g in ma.grouped_matmul_grads(gy, a, b, off))
    with FakeTensorMode(allow_non_fake_inputs=True):
        x = torch.empty(9, 72, device="cuda")
        for f in (lambda: ma.grouped_matmul(x, b, off),
                  lambda: ma.fp8_matmul(x, w, off),
                  lambda: ma.quantize_fp8(x),
                  lambda: ma.quantize_fp8(x, "tile"),
                  lambda: ma.grouped_matmul(a, b, torch.empty(
                      3, dtype=torch.int32, device="cuda"))):
            with pytest.raises(RuntimeError, match="must have memory"):
                f()
