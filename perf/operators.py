"""Cases for the 8-bit block-scaled product and the ragged grouped product.

Three operators are measured:

* ``quantize``  - values to e4m3 with a float32 scale for each 128 along a row
  (``row``) or for each 128 x 128 tile (``tile``);
* ``fp8``       - a @ bt^T with a quantized by rows and bt by tiles, for one
  right operand or for one per group of rows; with ``grad`` a training step;
* ``grouped``   - the rows of group g times b[g], groups of any size; with
  ``grad`` a training step.

``run`` computes them from elementary torch operations in float32, or, where
``own`` is true, through matrel_amd.
"""

import math

import torch

own = False

BLOCK = 128
FP8_MAX = 448.0
TINY = 2.0 ** -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16,
          "fp32": torch.float32}


# ---------------------------------------------------------------- cases ----

def listed():
    return [
        # one token's activations on their way into an 8-bit layer: latency
        dict(name="quantize one token", op="quantize", kind="row", groups=1,
             rows=1, cols=4096, dtype="bf16"),
        # the activations of a long prompt or a training batch
        dict(name="quantize a batch", op="quantize", kind="row", groups=1,
             rows=16384, cols=8192, dtype="bf16"),
        # the master weights of some experts, edges that end inside a tile
        dict(name="quantize weights", op="quantize", kind="tile", groups=8,
             rows=2000, cols=5000, dtype="fp32"),
        # one token through one layer while serving
        dict(name="fp8 one token", op="fp8", tokens=1, groups=0, n=4096,
             k=4096, dtype="bf16", grad=False, seen=1.0),
        # a serving batch routed to experts, a few rows for each
        dict(name="fp8 serving experts", op="fp8", tokens=64, groups=32,
             n=4096, k=2048, dtype="bf16", grad=False, seen=0.9),
        # ragged in every direction
        dict(name="fp8 ragged", op="fp8", tokens=5003, groups=24, n=1500,
             k=2500, dtype="fp16", grad=False, seen=0.8),
        # a prompt or batch through one large layer
        dict(name="fp8 large", op="fp8", tokens=16384, groups=0, n=8192,
             k=8192, dtype="bf16", grad=False, seen=1.0),
        # a training step of an 8-bit expert layer
        dict(name="fp8 step", op="fp8", tokens=8192, groups=8, n=4096,
             k=2048, dtype="bf16", grad=True, seen=1.0),
        # a serving batch routed to 16-bit experts
        dict(name="grouped serving", op="grouped", tokens=32, groups=64,
             n=1024, k=4096, dtype="bf16", layout="nk", grad=False,
             seen=0.5),
        # odd sizes, so that no row starts on 16 bytes
        dict(name="grouped odd", op="grouped", tokens=3001, groups=10,
             n=1111, k=777, dtype="fp16", layout="kn", grad=False,
             seen=0.9),
        # a training step of an expert layer
        dict(name="grouped step", op="grouped", tokens=16384, groups=16,
             n=4096, k=4096, dtype="bf16", layout="nk", grad=True,
             seen=1.0),
        # per-key linear maps in exact float32, with their gradients
        dict(name="grouped fp32 step", op="grouped", tokens=4096, groups=12,
             n=1024, k=1000, dtype="fp32", layout="kn", grad=True,
             seen=0.9),
    ]


def _size(rng, lo, hi):
    """A size spread over the logarithm; multiples of 128, of 8, or odd."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    step = rng.choice((128, 8, 1))
    return min(hi, max(lo, v // step * step + (step == 1 and v % 2 == 0)))


def draw(rng):
    op = rng.choice(("quantize", "fp8", "grouped"))
    if op == "quantize":
        kind = rng.choice(("row", "tile"))
        groups = 1 if kind == "row" else rng.choice((1, 2, 5, 8))
        cols = _size(rng, 64, 8192)
        rows = _size(rng, 1, 16384 // groups)
        return dict(op=op, kind=kind, groups=groups, rows=rows, cols=cols,
                    dtype=rng.choice(("bf16", "fp16", "fp32")))
    dtypes = ("bf16", "fp16") if op == "fp8" else ("bf16", "fp16", "fp32")
    c = dict(op=op, tokens=_size(rng, 1, 16384),
             groups=rng.choice((0, 1)) if op == "fp8" and rng.random() < .4
             else int(round(math.exp(rng.uniform(0, math.log(64))))),
             n=_size(rng, 64, 8192), k=_size(rng, 64, 8192),
             dtype=rng.choice(dtypes), grad=rng.random() < 0.35,
             seen=rng.choice((0.5, 0.8, 1.0)))
    if op == "grouped":
        c["layout"] = rng.choice(("nk", "kn"))
    # no more work than the largest listed cases: 2.2e12 flops at 8 bits,
    # 1.7e12 in a 16-bit step, 5e10 in a float32 one; 6e8 weights
    most = {"fp8": 1e12, "grouped": 2.5e11}[op]
    if c["dtype"] == "fp32":
        most = 8e9
    while c["tokens"] * c["n"] * c["k"] > most / (3 if c["grad"] else 1):
        c["tokens"] = c["tokens"] * 2 // 3
    while max(1, c["groups"]) * c["n"] * c["k"] > 3e8:
        c["groups"] = c["groups"] * 2 // 3
        if c["groups"] <= 1:
            c["n"] = c["n"] * 2 // 3
    c["tokens"] = max(1, c["tokens"])
    return c


# --------------------------------------------------------------- inputs ----

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _activations(rows, cols, g):
    """Near-normal values with a few channels that are much larger."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    loud = torch.rand(cols, device="cuda", generator=g) < 0.01
    return x * torch.where(loud, 20.0, 1.0)


def _sizes(tokens, groups, seen, seed):
    """Rows of each group: skewed, and some groups see none at all."""
    g = torch.Generator()
    g.manual_seed(int(seed) * 7 + 1)
    p = torch.softmax(torch.randn(groups, generator=g), 0)
    p = p * (torch.rand(groups, generator=g) < seen)
    p[int(torch.randint(groups, (1,), generator=g))] += 0.1
    pick = torch.multinomial(p, tokens, replacement=True, generator=g)
    return torch.bincount(pick, minlength=groups).tolist()


def prepare(case, seed):
    c, g = case, _gen(seed)
    dt = DTYPES[c["dtype"]]
    s = dict(case=c)
    if c["op"] == "quantize":
        if c["kind"] == "row":
            s["x"] = _activations(c["rows"], c["cols"], g).to(dt)
        else:
            s["x"] = (torch.randn(c["groups"], c["rows"], c["cols"],
                                  device="cuda", generator=g) * 0.02).to(dt)
        return s
    t, n, k = c["tokens"], c["n"], c["k"]
    dense = c["groups"] == 0
    s["sizes"] = [t] if dense else _sizes(t, c["groups"], c["seen"], seed)
    starts = [0]
    for v in s["sizes"]:
        starts.append(starts[-1] + v)
    s["offsets"] = None if dense else torch.tensor(
        starts, dtype=torch.int32, device="cuda")
    s["x"] = _activations(t, k, g).to(dt)
    # weights as they are stored: [n, k] for each group, or [k, n]
    shape = (max(1, c["groups"]),) + (
        (k, n) if c.get("layout") == "kn" else (n, k))
    w = torch.randn(shape, device="cuda", generator=g) / math.sqrt(k)
    if dense:
        w = w[0]
    if c["grad"]:
        s["w"] = w.to(dt).requires_grad_()
        s["x"].requires_grad_()
        s["gy"] = (torch.randn(t, n, device="cuda", generator=g)
                   * 0.01).to(dt)
    elif c["op"] == "fp8":
        s["wq"], s["ws"] = _quantize(w.to(dt), "tile")
    else:
        s["w"] = w.to(dt)
    return s


# ---------------------------------------------------------- plain forms ----

def _blocks(x, kind):
    """x in float32, padded with zeros and cut into its blocks: [..., row
    blocks, rows of one, column blocks, 128]."""
    r, c = x.shape[-2:]
    h = 1 if kind == "row" else BLOCK
    x = torch.nn.functional.pad(x.float(), (0, -c % BLOCK, 0, -r % h))
    return x.reshape(*x.shape[:-2], x.shape[-2] // h, h,
                     x.shape[-1] // BLOCK, BLOCK)


def _quantize(x, kind):
    """(e4m3 of x's shape, scales [..., column blocks, row blocks])."""
    r, c = x.shape[-2:]
    b = _blocks(x, kind)
    top = b.abs().amax(dim=(-3, -1), keepdim=True)
    top = torch.maximum(top, torch.full_like(top, TINY))
    # both divisions are of tensors: of a number, torch multiplies by the
    # other side's rounded reciprocal instead
    most = torch.full_like(top, FP8_MAX)
    q = (b * (most / top)).to(torch.float8_e4m3fn)
    q = q.reshape(*q.shape[:-4], q.shape[-4] * q.shape[-3], -1)[..., :r, :c]
    scale = (top / most).squeeze(-1).squeeze(-2)
    return q.contiguous(), scale.transpose(-1, -2).contiguous()


def _values(q, scale, kind, dtype=torch.float32):
    """What a quantized matrix stands for."""
    r, c = q.shape[-2:]
    s = scale.transpose(-1, -2).to(dtype)
    s = s.repeat_interleave(BLOCK, -1)[..., :c]
    if kind == "tile":
        s = s.repeat_interleave(BLOCK, -2)[..., :r, :]
    return q.to(dtype) * s


def _by_group(rows, weights, sizes):
    """Each group's rows times its weights [k, n]."""
    parts = torch.split(rows, sizes)
    return torch.cat([p @ w for p, w in zip(parts, weights)])


def _weight_grads(rows, grads, sizes):
    """Each group's rows^T @ its gradient's rows, [groups, k, n]."""
    return torch.stack([a.t() @ b for a, b in
                        zip(torch.split(rows, sizes),
                            torch.split(grads, sizes))])


def _plain(s):
    c = s["case"]
    if c["op"] == "quantize":
        return dict(zip(("q", "scale"), _quantize(s["x"], c["kind"])))
    dt, sizes = s["x"].dtype, s["sizes"]
    x = s["x"].detach()
    if c["op"] == "fp8":
        xv = _values(*_quantize(x, "row"), "row")
        if c["grad"]:
            w = s["w"].detach()
            wv = _values(*_quantize(w, "tile"), "tile")
        else:
            wv = _values(s["wq"], s["ws"], "tile")
        wv = wv.reshape(-1, c["n"], c["k"])
        out = dict(y=_by_group(xv, wv.transpose(1, 2), sizes).to(dt))
        if c["grad"]:
            gv = _values(*_quantize(s["gy"], "row"), "row")
            out["dx"] = _by_group(gv, wv, sizes).to(dt)
            dw = _weight_grads(s["gy"].float(), x.float(), sizes)
            out["dw"] = dw.reshape(w.shape).to(dt)
        return out
    w = s["w"].detach().float()
    if c["layout"] == "nk":
        w = w.transpose(1, 2)
    out = dict(y=_by_group(x.float(), w, sizes).to(dt))
    if c["grad"]:
        gy = s["gy"].float()
        out["dx"] = _by_group(gy, w.transpose(1, 2), sizes).to(dt)
        if c["layout"] == "nk":
            out["dw"] = _weight_grads(gy, x.float(), sizes).to(dt)
        else:
            out["dw"] = _weight_grads(x.float(), gy, sizes).to(dt)
    return out


# -------------------------------------------------------- the framework ----

def _own(s):
    import matrel_amd as ma
    c = s["case"]
    if c["op"] == "quantize":
        r = ma.quantize_fp8(s["x"], c["kind"])
        return dict(q=r.data, scale=r.scale)
    x = s["x"]
    if c["op"] == "fp8":
        bt = s["w"] if c["grad"] else ma.Fp8Blocks(s["wq"], s["ws"], "tile")
        y = ma.fp8_matmul(x, bt, s["offsets"])
    else:
        b = s["w"].transpose(1, 2) if c["layout"] == "nk" else s["w"]
        y = ma.grouped_matmul(x, b, s["offsets"])
    if not c["grad"]:
        return dict(y=y)
    dx, dw = torch.autograd.grad(y, (x, s["w"]), s["gy"])
    return dict(y=y.detach(), dx=dx, dw=dw)


def run(state):
    return _own(state) if own else _plain(state)


# ----------------------------------------------------------- the counts ----

def work(case):
    c = case
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[c["dtype"]]
    if c["op"] == "quantize":
        n = c["groups"] * c["rows"] * c["cols"]
        blocks = (c["groups"] * math.ceil(c["cols"] / BLOCK)
                  * math.ceil(c["rows"] / (1 if c["kind"] == "row"
                                           else BLOCK)))
        return dict(bytes=n * (size + 1) + 4 * blocks, flops=2 * n)
    t, n, k, e = c["tokens"], c["n"], c["k"], max(1, c["groups"])
    # groups that have rows, as a mean: the others' weights are not needed
    met = 1 if c["groups"] == 0 else sum(
        1 for seed in range(8)
        for v in _sizes(t, e, c["seen"], seed) if v) / 8
    flops = 2 * t * n * k
    if c["grad"]:  # x, gy, w read; y, dx, dw written
        return dict(bytes=size * (2 * t * (k + n) + (met + e) * n * k),
                    flops=3 * flops)
    wsize = 1 if c["op"] == "fp8" else size
    return dict(bytes=size * t * (k + n) + wsize * met * n * k, flops=flops)


def _exact_e4m3(x, scale_up):
    """The e4m3 value next to x * scale_up (one float32 product, as the
    definition has it), ties to even, worked out in float64."""
    v = (x.float() * scale_up).double()
    e = torch.frexp(v.abs())[1].clamp(min=-5) - 4  # spacing of 3 bits
    step = ((e.long() + 1023) << 52).view(torch.float64)  # 2 ** e exactly
    return torch.round(v / step) * step


def _exact_quantized(x, kind):
    """(values of the payload, scales, both float64) block by block."""
    r, c = x.shape[-2:]
    h = 1 if kind == "row" else BLOCK
    cb, rb = math.ceil(c / BLOCK), math.ceil(r / h)
    cols = torch.arange(c, device=x.device) // BLOCK
    rows = torch.arange(r, device=x.device) // h
    top = torch.zeros(*x.shape[:-2], r, cb, dtype=torch.float64,
                      device=x.device)
    top.scatter_reduce_(-1, cols.expand(x.shape), x.double().abs(), "amax")
    tops = torch.zeros(*x.shape[:-2], rb, cb, dtype=torch.float64,
                       device=x.device)
    tops.scatter_reduce_(-2, rows[:, None].expand(top.shape), top, "amax")
    tops = tops.clamp(min=TINY)
    up = torch.full_like(tops, FP8_MAX).float() / tops.float()
    up = up[..., rows, :][..., cols]
    return _exact_e4m3(x, up), (tops / FP8_MAX)


def _exact_values(x, kind):
    q, s = _exact_quantized(x, kind)
    h = 1 if kind == "row" else BLOCK
    rows = torch.arange(x.shape[-2], device=x.device) // h
    cols = torch.arange(x.shape[-1], device=x.device) // BLOCK
    return q * s[..., rows, :][..., cols]


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    x = s["x"].detach()
    if c["op"] == "quantize":
        q, scale = _exact_quantized(x, c["kind"])
        return dict(q=q, scale=scale.transpose(-1, -2))
    t, n, k = c["tokens"], c["n"], c["k"]
    w = s["w"].detach() if "w" in s else None
    if c["op"] == "fp8":
        xv = _exact_values(x, "row")
        if w is not None:
            wv = _exact_values(w, "tile")
        else:
            up = torch.arange(n, device=x.device) // BLOCK
            left = torch.arange(k, device=x.device) // BLOCK
            wv = s["wq"].double() * s["ws"].double().transpose(
                -1, -2)[..., up, :][..., left]
        wv = wv.reshape(-1, n, k).transpose(1, 2)
    else:
        xv, wv = x.double(), w.double()
        if c["layout"] == "nk":
            wv = wv.transpose(1, 2)
    y = torch.empty(t, n, dtype=torch.float64, device=x.device)
    out = dict(y=y)
    if c["grad"]:
        g = s["gy"]
        gv = _exact_values(g, "row") if c["op"] == "fp8" else g.double()
        out["dx"] = torch.empty(t, k, dtype=torch.float64, device=x.device)
        out["dw"] = torch.empty(w.shape, dtype=torch.float64,
                                device=x.device)
        dw = out["dw"].reshape(-1, *w.shape[-2:])
    at = 0
    for e, m in enumerate(s["sizes"]):
        here = slice(at, at + m)
        y[here] = xv[here] @ wv[e]
        if c["grad"]:
            out["dx"][here] = gv[here] @ wv[e].t()
            d = x[here].double().t() @ g[here].double()
            dw[e] = d if c.get("layout") == "kn" else d.t()
        at += m
    return out
