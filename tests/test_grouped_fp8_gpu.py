"""Grouped and 8-bit products on the GPU: every tile of the kernels, the
engine's fp8 tier, graphs, streams and large tensors.

References are float64 products on the GPU. Tolerances as in
test_grouped_fp8.py: (K + 8) * 2^-23 * sum |a b| for a float32 sum, what the
8-bit matrix unit cuts off (fp8_cut), half a step of the result's type for its
rounding."""

import pytest
import torch

import matrel_amd as ma
from test_grouped_fp8 import fp8_cut

pytestmark = pytest.mark.gpu

BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


def randn(*shape, seed, dtype=BF, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda")
            * scale).to(dtype)


def offsets_of(sizes, head=0):
    v = [head]
    for s in sizes:
        v.append(v[-1] + s)
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def assert_near(got, exact, size, depth, cut=0.0):
    if torch.is_tensor(cut):
        cut = cut.to(size.device)
    err = (depth + 8) * 2.0 ** -23 * size + cut
    tol = err + torch.finfo(got.dtype).eps / 2 * (exact.abs() + err)
    if got.dtype == HF:
        tol = tol + 2.0 ** -25
    off = (got.detach().double() - exact).abs()
    assert torch.isfinite(off).all()
    worst = (off / tol.clamp(min=1e-300)).max().item() if off.numel() else 0
    assert worst <= 1, f"{worst:.3g} x tol"


def rows(a, b, off):
    """(a @ b by groups, |a| @ |b|) in float64; a, b in float64."""
    y = torch.zeros(a.shape[0], b.shape[2], dtype=torch.float64,
                    device="cuda")
    s = torch.zeros_like(y)
    v = off.tolist()
    for g, (lo, hi) in enumerate(zip(v, v[1:])):
        if hi > lo:
            y[lo:hi] = a[lo:hi] @ b[g]
            s[lo:hi] = a[lo:hi].abs() @ b[g].abs()
    return y, s


def check_grouped(sizes, k, n, dtype, layout, seed=1):
    off = offsets_of(sizes)
    t, e = sum(sizes), len(sizes)
    a = randn(t, k, seed=seed, dtype=dtype).requires_grad_()
    if layout == "kn":
        b = randn(e, k, n, seed=seed + 1, dtype=dtype)
    else:
        b = randn(e, n, k, seed=seed + 1, dtype=dtype).transpose(1, 2)
    b.requires_grad_()
    gy = randn(t, n, seed=seed + 2, dtype=dtype)
    y = ma.grouped_matmul(a, b, off)
    da, db = torch.autograd.grad(y, (a, b), gy)
    ad, bd, gd = a.detach().double(), b.detach().double(), gy.double()
    assert_near(y, *rows(ad, bd, off), k)
    assert_near(da, *rows(gd, bd.transpose(1, 2).contiguous(), off), n)
    v = off.tolist()
    for g, (lo, hi) in enumerate(zip(v, v[1:])):
        x, z = ad[lo:hi], gd[lo:hi]
        assert_near(db[g], x.t() @ z, x.abs().t() @ z.abs(), hi - lo)
    # no atomics, no race: the same bits again
    y2 = ma.grouped_matmul(a, b, off)
    da2, db2 = torch.autograd.grad(y2, (a, b), gy)
    assert torch.equal(y, y2) and torch.equal(da, da2)
    assert torch.equal(db, db2)


UNEVEN = [3, 0, 700, 88, 130, 1, 256, 40, 0, 17, 60, 5]


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("sizes,k,n", [
    (UNEVEN, 1544, 1544),                    # 256 x 256, whole and half
    ([100, 2500, 0, 900, 1, 499], 840, 840),  # 128 x 128
    (UNEVEN, 1543, 1541),                    # unaligned
])
def test_tiles(sizes, k, n, dtype, layout):
    check_grouped(sizes, k, n, dtype, layout)


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("dtype", [BF, FF])
def test_tiles_many_rows(dtype, layout):
    """128 x 128 of float32 and of unaligned rows: above 1024 tiles."""
    sizes = [8700 // 12] * 11 + [8700 - 8700 // 12 * 11]
    check_grouped(sizes, 1543 if dtype == BF else 1544, 1541 if dtype == BF
                  else 1544, dtype, layout)


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("dtype", [BF, FF])
@pytest.mark.parametrize("sizes,k,n", [
    ([70], 4096, 200),          # sums split, one group
    ([3, 2], 4096, 200),        # few rows, sums split with k across rows
    ([5000], 104, 96),          # gradients of matrices split over rows
    ([3] * 20, 136, 6400),      # few rows, four column blocks a workgroup
    ([20, 40], 136, 5000),      # 32 rows, two column blocks
    ([1], 4096, 1000),          # eight waves
])
def test_splits_and_few_rows(sizes, k, n, dtype, layout):
    check_grouped(sizes, k, n, dtype, layout)


@pytest.mark.parametrize("sizes,k,n", [
    (UNEVEN, 1544, 1544), (UNEVEN, 1552, 1552),
    ([100, 2500, 0, 900, 1, 499], 840, 848), (UNEVEN, 1543, 1541),
    ([70], 4096, 200), ([3] * 20, 144, 6400), ([20, 40], 144, 5000),
    ([1], 8192, 1000), ([3], 8200, 77)])
@pytest.mark.parametrize("dtype", [BF, FF])
def test_fp8_tiles(sizes, k, n, dtype):
    off = offsets_of(sizes)
    t, e = sum(sizes), len(sizes)
    a = randn(t, k, seed=5, dtype=dtype).requires_grad_()
    w = randn(e, n, k, seed=6, dtype=dtype).requires_grad_()
    gy = randn(t, n, seed=7, dtype=dtype)
    y = ma.fp8_matmul(a, w, off)
    da, dw = torch.autograd.grad(y, (a, w), gy)
    qa, qw, qg = ma.quantize_fp8(a), ma.quantize_fp8(w, "tile"), \
        ma.quantize_fp8(gy)

    def values(q):  # e4m3 times a float32 scale is exact in float64
        s = q.scale.double().transpose(-1, -2)
        s = s.repeat_interleave(128, -1)[..., :q.shape[-1]]
        if q.kind == "tile":
            s = s.repeat_interleave(128, -2)[..., :q.shape[-2], :]
        return q.data.double() * s

    assert_near(y, *rows(values(qa), values(qw).transpose(1, 2).contiguous(),
                         off), k, fp8_cut(qa, qw, off))
    assert_near(da, *rows(values(qg), values(qw), off), n,
                fp8_cut(qg, qw.transpose(), off))
    v, ad, gd = off.tolist(), a.detach().double(), gy.double()
    for g, (lo, hi) in enumerate(zip(v, v[1:])):
        x, z = gd[lo:hi], ad[lo:hi]
        assert_near(dw[g], x.t() @ z, x.abs().t() @ z.abs(), hi - lo)
    assert torch.equal(y, ma.fp8_matmul(a, w, off))
    assert torch.equal(y, ma.fp8_matmul(qa, qw, off, out_dtype=dtype))


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("sizes,k,n", [
    ([1300, 1, 1299], 200, 4104),    # the product
    ([1300, 0, 1300], 4104, 200),    # the gradient of a
    ([130, 1, 70], 1032, 3080),      # the gradient of b, few groups
    ([300] * 32, 1032, 1544),        # the same, many
])
def test_large_tile(sizes, k, n, dtype, layout):
    """256 x 256, with ends of groups, columns and sums inside a tile."""
    check_grouped(sizes, k, n, dtype, layout)


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("dtype", [HF, FF])
@pytest.mark.parametrize("sizes,k,n", [
    ([2000, 1, 2099], 17, 4099),     # the product
    ([33, 7, 60], 2305, 1545),       # the gradient of b
])
def test_middle_tile_unaligned(sizes, k, n, dtype, layout):
    check_grouped(sizes, k, n, dtype, layout)


FEW = [([3] * 20, 6400), ([3, 3], 6400), ([3], 1000),      # 16 rows: 4, 2, 1
       ([20] * 20, 6400), ([20, 40], 5000), ([20], 1000)]  # 32 rows


@pytest.mark.parametrize("k", [136, 137, 4096, 4099])
@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("sizes,n", FEW)
def test_few_rows(sizes, n, k, dtype):
    """Blocks of columns a workgroup, four waves or (long sums) eight."""
    if k < 4096 or n == 1000:
        check_grouped(sizes, k, n, dtype, "nk")


@pytest.mark.parametrize("sizes,k,n", [
    ([1300, 1, 1299], 208, 4104), ([2000, 1, 2099], 131, 4099),  # large tiles
    ([100, 100], 7, 40)] +                                 # rows of a few bytes
    [(s, k, n) for s, n in FEW for k in (144, 145)] +
    [(s, k, 1000) for s, n in FEW if n == 1000 for k in (8192, 8195)])
def test_fp8_variants(sizes, k, n):
    test_fp8_tiles(sizes, k, n, BF)


def test_far_rows():
    """Rows 8 MB apart: offsets within a tile pass 31 bits."""
    off = offsets_of([2, 1])
    a = randn(3, 1 << 22, seed=8)[:, :64]
    b = randn(2, 64, 40, seed=9)
    assert_near(ma.grouped_matmul(a, b, off),
                *rows(a.double(), b.double(), off), 64)
    w = randn(64, 1 << 22, seed=10)[:, :40]
    b = w.expand(2, 64, 40)
    assert_near(ma.grouped_matmul(a.contiguous(), b, off),
                *rows(a.double(), b.double(), off), 64)


def test_large_tensors():
    """Weights and results of more than 2^31 elements."""
    b = torch.zeros(3, 32768, 32768, dtype=BF, device="cuda")
    b[2] = randn(32768, 32768, seed=11, scale=0.01)
    a = randn(5, 32768, seed=12)
    off = offsets_of([0, 1, 4])
    for w in (b, b.transpose(1, 2)):
        y = ma.grouped_matmul(a, w, off)
        assert (y[0] == 0).all()
        for cols in (slice(0, 300), slice(32768 - 300, 32768)):
            x = w[2][:, cols].double()
            assert_near(y[1:, cols], a[1:].double() @ x,
                        a[1:].double().abs() @ x.abs(), 32768)
    del b, w, y
    a = randn(70000, 64, seed=13)
    w = randn(1, 64, 32768, seed=14)
    y = ma.grouped_matmul(a, w, offsets_of([70000]))
    x, z = a[-300:].double(), w[0].double()
    assert_near(y[-300:], x @ z, x.abs() @ z.abs(), 64)
    q = ma.fp8_matmul(a, w[0].t().contiguous(), out_dtype=BF)
    assert q.shape == y.shape
    full = ma.fp8_matmul(a[-300:].contiguous(), w[0].t().contiguous())
    assert torch.equal(q[-300:], full)


# ------------------------------------------------- engine, graphs, streams --

def test_engine_fp8_tier():
    """MatMul at gemm_precision="fp8", ragged blocks: the product of what the
    blocks stand for."""
    from matrel_amd.exec.runtime import reset_runtime
    old = ma.get_config()
    reset_runtime()
    try:
        s = ma.MatrelSession(ma.MatrelConfig(block_size=512,
                                             gemm_precision="fp8"))
        ta, tb = randn(700, 900, seed=15), randn(900, 650, seed=16)
        c = (s.from_dense(ta) @ s.from_dense(tb)).to_tensor()
        # 512 is a multiple of 128: blocks quantize as the whole does
        fa, fb = ma.quantize_fp8(ta), ma.quantize_fp8(tb.t()[None], "tile")
        qa = fa.dequantize().double()
        qb = fb.dequantize()[0].double().t()
        assert c.shape == (700, 650)
        assert torch.equal(c, c.to(BF).float())  # as the engine stores it
        assert_near(c.to(BF), qa @ qb, qa.abs() @ qb.abs(), 900,
                    fp8_cut(fa, fb, offsets_of([700])))
    finally:
        ma.set_config(old)
        reset_runtime()


def test_engine_fp8_summa_panels(monkeypatch):
    """The panels that SUMMA broadcasts at gemm_precision="fp8" (payloads and
    float32 scales of both kinds, ragged edges), over RCCL with one rank."""
    import os

    import torch.distributed as dist
    from matrel_amd.exec import runtime, summa
    old = ma.get_config()
    runtime.reset_runtime()
    os.environ.setdefault("MASTER_ADDR", "127.0.0.1")
    os.environ.setdefault("MASTER_PORT", "29418")
    dist.init_process_group("nccl", rank=0, world_size=1)
    try:
        s = ma.MatrelSession(ma.MatrelConfig(block_size=256,
                                             gemm_precision="fp8"))
        ta, tb = randn(600, 500, seed=15), randn(500, 300, seed=16)
        a, b = s.from_dense(ta).plan.data, s.from_dense(tb).plan.data
        want = (s.from_dense(ta) @ s.from_dense(tb)).compute().blocks
        out = ma.BlockMatrix(600, 300, block_size=256)
        rt = runtime.get_runtime()
        monkeypatch.setattr(type(rt), "is_distributed", True)
        monkeypatch.setattr(type(rt), "row_group",
                            lambda self, p: dist.group.WORLD)
        monkeypatch.setattr(type(rt), "col_group",
                            lambda self, q: dist.group.WORLD)
        summa.summa_matmul(a, b, out)
        assert set(out.blocks) == set(want.blocks)
        for k, t in out.blocks.items():
            assert torch.equal(t, want.blocks[k])
    finally:
        monkeypatch.undo()
        dist.destroy_process_group()
        ma.set_config(old)
        runtime.reset_runtime()


def test_block_accumulate():
    from matrel_amd.ops import blockops
    a, bt = randn(130, 260, seed=17), randn(70, 260, seed=18)
    qa, sa = blockops.to_fp8(a, "row")
    qb, sb = blockops.to_fp8(bt, "tile")
    acc = torch.empty(130, 70, device="cuda")
    blockops.gemm_bt_fp8_acc(acc, qa, sa, qb, sb, beta0=True)
    one = acc.clone()
    blockops.gemm_bt_fp8_acc(acc, qa, sa, qb, sb)
    assert torch.equal(acc, 2 * one)
    fa, fb = ma.quantize_fp8(a), ma.quantize_fp8(bt[None], "tile")
    x, y = fa.dequantize().double(), fb.dequantize()[0].double()
    assert_near(one, x @ y.t(), x.abs() @ y.abs().t(), 260,
                fp8_cut(fa, fb, offsets_of([130])))


def serve(x, w1, w2, off):
    """Two layers by experts, 16 and 8 bits."""
    h = ma.grouped_matmul(x, w1, off)
    return ma.fp8_matmul(torch.relu(h), w2, off)


def test_layers_together_in_a_graph():
    """Captured once, replayed with other inputs and other group sizes."""
    w1 = randn(6, 256, 512, seed=19, scale=0.06)
    w2 = ma.quantize_fp8(randn(6, 256, 512, seed=20, scale=0.05), "tile")
    x = randn(48, 256, seed=21)
    off = offsets_of([8] * 6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        serve(x, w1, w2, off)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = serve(x, w1, w2, off)
    for i, sizes in enumerate(([8] * 6, [0, 48, 0, 0, 0, 0],
                               [1, 2, 3, 4, 5, 6], [40, 0, 0, 0, 7, 1])):
        x.copy_(randn(48, 256, seed=30 + i))
        off.copy_(offsets_of(sizes))
        graph.replay()
        eager = serve(x, w1, w2, off)
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


def test_two_graphs_share_nothing():
    """Split sums have a workspace: graphs replayed at once, on two streams,
    keep their own."""
    w = randn(1, 4096, 200, seed=22)
    xs = [randn(70, 4096, seed=23 + i) for i in range(2)]
    off = offsets_of([70])
    want = [ma.grouped_matmul(x, w, off) for x in xs]
    graphs, ys = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ys.append(ma.grouped_matmul(x, w, off))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for y, z in zip(ys, want):
            assert torch.equal(y, z)


def test_training_step_in_a_graph():
    a = randn(300, 256, seed=25).requires_grad_()
    w = randn(4, 128, 256, seed=26).requires_grad_()
    gy = randn(300, 128, seed=27)
    off = offsets_of([100, 0, 150, 50])

    def step():
        y = ma.grouped_matmul(a, w.transpose(1, 2), off)
        z = ma.fp8_matmul(a, w, off)
        return torch.autograd.grad(y + z, (a, w), gy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        with torch.no_grad():
            a.copy_(randn(300, 256, seed=40 + i))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_capture_beside_a_living_graph():
    """Leaves that an eager autograd graph still holds: a captured forward
    pass is refused, grouped_matmul_grads is not."""
    a = randn(64, 64, seed=28).requires_grad_()
    w = randn(2, 64, 64, seed=29).requires_grad_()
    gy = randn(64, 64, seed=30)
    off = offsets_of([30, 34])
    alive = ma.grouped_matmul(a, w, off)
    want = ma.grouped_matmul_grads(gy, a, w, off)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    refused = 0
    with torch.cuda.graph(graph):
        for f in (lambda: ma.grouped_matmul(a, w, off),
                  lambda: ma.fp8_matmul(a, w, off)):
            try:
                f()
            except RuntimeError as e:
                refused += "outside of this capture" in str(e)
        got = ma.grouped_matmul_grads(gy, a, w, off)
    assert refused == 2
    for _ in range(3):
        for g in got:
            g.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    alive.sum().backward()
    assert a.grad is not None


def test_other_streams():
    """Calls on two streams at once, and a backward pass on the stream of its
    forward pass."""
    off = offsets_of([20, 0, 50])
    xs = [randn(70, 2048, seed=31 + i) for i in range(2)]
    w = randn(3, 2048, 320, seed=33)
    want = [ma.grouped_matmul(x, w, off) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(4):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(ma.grouped_matmul(x, w, off))
        torch.cuda.synchronize()
        assert all(torch.equal(y, z) for y, z in zip(got, want))
    x = xs[0].requires_grad_()
    with torch.cuda.stream(streams[0]):
        y = ma.grouped_matmul(x, w, off)
        g, = torch.autograd.grad(y, x, torch.ones_like(y))
    torch.cuda.synchronize()
    assert_near(g, *rows(torch.ones(70, 320, dtype=torch.float64,
                                    device="cuda"),
                         w.double().transpose(1, 2).contiguous(), off), 320)


def test_refuses_more_tiles_than_a_launch_holds():
    """As many groups as rows: a tile for every row, 2^32 threads and more."""
    t, k, n = 1 << 17, 16, 8192
    a = torch.zeros(t, k, dtype=BF, device="cuda")
    b = torch.zeros(1, n, k, dtype=BF, device="cuda").expand(t, n, k)
    off = torch.arange(t + 1, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="too many tiles"):
        ma.grouped_matmul(a, b.transpose(1, 2), off)
