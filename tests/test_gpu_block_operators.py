"""Block-scaled 8-bit quantization and products, the norms around a block and rotary positions on the GPU, against
their formulas in 64 bits.  Bounds count roundings: half a step is 2^-24 of the value for fp32, 2^-11 for fp16, 2^-8 for
bf16 and 2^-4 for e4m3 (2^-10 below its smallest normal number)."""

import math

import pytest

import sam3cpp_b200 as s3t

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
KINDS = {"f32": (s3t.TYPE_F32, "float32", 2.0 ** -24), "f16": (s3t.TYPE_F16, "float16", 2.0 ** -11),
         "bf16": (s3t.TYPE_BF16, "bfloat16", 2.0 ** -8)}


@pytest.fixture(scope="module")
def torch(request):
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    yield torch
    torch.cuda.synchronize()
    s3t.check(s3t.lib().s3t_device_status(0))


def up(n, m):
    return -(-n // m) * m


def rows_of(torch, values, dtype, pad, fill=float("nan")):
    """The values as rows of a wider buffer whose other elements must not matter."""
    wide = torch.full((values.shape[0], values.shape[1] + pad), fill, device="cuda", dtype=dtype)
    wide[:, : values.shape[1]] = values
    return wide


class Eight:
    """An 8-bit matrix with sentinels behind its rows, columns and scales."""

    def __init__(self, torch, rows, cols, block_rows=1, extra=16):
        self.rows, self.cols, self.block_rows = rows, cols, block_rows
        self.groups, self.blocks = up(cols, 128) // 128, up(rows, block_rows) // block_rows
        self.q = torch.full((rows + 1, up(cols, 16) + extra), 0x55, device="cuda", dtype=torch.uint8)
        self.scale = torch.full((self.groups + 1, self.blocks + 3), -7.0, device="cuda")

    @property
    def matrix(self):
        return s3t.Matrix(self.q.data_ptr(), self.q.stride(0), self.scale.data_ptr(), self.scale.stride(0))

    def codes(self, torch):
        return self.q[: self.rows, : self.cols].view(torch.float8_e4m3fn)

    def scales(self):
        return self.scale[: self.groups, : self.blocks]

    def spans(self):
        s = self.scales().t().double().repeat_interleave(self.block_rows, 0)[: self.rows]
        return s.repeat_interleave(128, 1)[:, : self.cols]

    def values(self, torch):
        return self.codes(torch).double() * self.spans()

    def untouched(self):
        return bool((self.q[self.rows:] == 0x55).all() and (self.q[:, self.cols:] == 0x55).all()
                    and (self.scale[self.groups:] == -7).all() and (self.scale[:, self.blocks:] == -7).all())


def random_eight(torch, g, rows, cols, block_rows):
    m = Eight(torch, rows, cols, block_rows)
    codes = (torch.randn(rows, cols, generator=g, device="cuda") * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
    m.q[:rows, :cols] = codes.view(torch.uint8)
    m.q[:, cols:] = 0x7F     # NaN behind the columns: never read
    m.q[rows:] = 0x7F
    m.scale[: m.groups, : m.blocks] = torch.exp(torch.randn(m.groups, m.blocks, generator=g, device="cuda"))
    m.scale[:, m.blocks:] = float("nan")
    return m


def quantized(torch, x, block_rows):
    """The defined codes and scales of fp32 values, each operation in fp32."""
    rows, cols = x.shape
    wide = torch.zeros(up(rows, block_rows), up(cols, 128), device=x.device)
    wide[:rows, :cols] = x
    b = wide.view(wide.shape[0] // block_rows, block_rows, -1, 128)
    a = b.abs().amax((1, 3)).clamp(min=2.0 ** -100)
    top = torch.full_like(a, 448.0)      # tensor by tensor: torch divides by a number through its reciprocal
    q = (b * (top / a)[:, None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return q.view(wide.shape)[:rows, :cols], (a / top).t()


# ------------------------------------------------------------ quantization ---

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows, cols, pad", [(1, 1, 0), (3, 127, 0), (33, 256, 0), (129, 300, 0), (40, 264, 8), (130, 257, 3),
                                             (1, 4736, 0), (257, 128, 1)])
def test_quantize_equals_its_definition(torch, kind, block_rows, rows, cols, pad):
    code, dtype, _ = KINDS[kind]
    g = torch.Generator("cuda").manual_seed(rows * 1000 + cols)
    x = torch.randn(rows, cols, generator=g, device="cuda") * torch.exp(torch.randn(rows, 1, generator=g, device="cuda") * 2)
    x[rows // 2] = 0
    x = rows_of(torch, x, getattr(torch, dtype), pad)
    m = Eight(torch, rows, cols, block_rows)
    s3t.quantize_fp8(0, code, x.data_ptr(), rows, cols, x.stride(0), block_rows, m.matrix)
    q, scale = quantized(torch, x[:, :cols].float(), block_rows)
    assert torch.equal(m.scales(), scale)
    assert torch.equal(m.codes(torch).float(), q.float())
    assert m.untouched()
    # and what it stands for is x within half a step and the roundings of 448 / a, x * (448 / a) and a / 448
    v, x64, s = m.values(torch), x[:, :cols].double(), m.spans()
    assert ((v - x64).abs() <= x64.abs() * (2.0 ** -4 + 4 * U) + s * 2.0 ** -10).all()


def test_quantize_extremes(torch):
    x = torch.zeros(6, 256, device="cuda")
    x[0, 3] = 3e38
    x[1] = 1e-42                       # below the floor: codes 0, a finite scale
    x[2, 200] = float("inf")
    x[3, 5] = float("nan")
    x[4, 130] = -float("inf")
    x[5] = -2.5
    m = Eight(torch, 6, 256)
    s3t.quantize_fp8(0, s3t.TYPE_F32, x.data_ptr(), 6, 256, 256, 1, m.matrix)
    v = m.values(torch)
    assert float(v[0, 3]) == pytest.approx(3e38, rel=1e-6) and (v[0, 4:] == 0).all()
    assert (m.codes(torch)[1].float() == 0).all() and torch.isfinite(m.scales()[:, 1]).all()
    for row, group in ((2, 1), (3, 0), (4, 1)):    # the whole group stands for NaN, the other one for zeros
        here = v[row, 128 * group: 128 * group + 128]
        there = v[row, 128 * (1 - group): 128 * (1 - group) + 128]
        assert torch.isnan(here).all() and (there == 0).all()
    assert torch.allclose(v[5], torch.full_like(v[5], -2.5), rtol=1e-6)


# ---------------------------------------------------------------- products ---

def product_reference(torch, x, w, bias, gelu):
    """(y, bound of the fp32 arithmetic's error) in 64 bits: every partial sum of a group's 128 products and of the
    groups is rounded (or truncated) once, by at most 2^-23 of the sum of magnitudes."""
    xv, wv = x.values(torch), w.values(torch)
    y, mag = xv @ wv.t(), xv.abs() @ wv.abs().t()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    e = mag * (128 + x.groups + 8) * 2 * U
    if gelu:
        # |gelu'| < 1.13; the error function's formula is good to 1.5e-7, the hardware 2^x and 1/x to 2^-21
        e = 1.13 * e + y.abs() * 4e-7 + 1e-30
        y = 0.5 * y * torch.special.erfc(-y * math.sqrt(0.5))
    return y, e


def call_product(torch, x, w, bias, gelu, out, pad=0, stream=0):
    m, n, k = x.rows, w.rows, x.cols
    b = bias.data_ptr() if bias is not None else None
    if out == "e4m3":
        y = Eight(torch, m, n)
        s3t.gemm_fp8(0, x.matrix, w.matrix, b, m, n, k, int(gelu), s3t.TYPE_E4M3, y.matrix, stream)
        return y
    code, dtype, _ = KINDS[out]
    y = torch.full((m + 1, n + pad), -9.0, device="cuda", dtype=getattr(torch, dtype))
    s3t.gemm_fp8(0, x.matrix, w.matrix, b, m, n, k, int(gelu), code, s3t.Matrix(y.data_ptr(), y.stride(0)), stream)
    return y


def check_product(torch, x, w, bias, gelu, out, y):
    m, n = x.rows, w.rows
    want, e = product_reference(torch, x, w, bias, gelu)
    if out == "e4m3":
        scale_e = torch.zeros(m, up(n, 128), device="cuda", dtype=torch.float64)
        scale_e[:, :n] = e
        top = torch.zeros_like(scale_e)
        top[:, :n] = want.abs()
        top = top.view(m, -1, 128).amax(2).clamp(min=2.0 ** -100) / 448
        err = (y.scales().t().double() - top).abs()
        assert (err <= scale_e.view(m, -1, 128).amax(2) / 448 + top * 3 * U).all()
        assert ((y.values(torch) - want).abs() <= (want.abs() + e) * (2.0 ** -4 + 4 * U) + y.spans() * 2.0 ** -10 + e).all()
        assert y.untouched()
        return
    half = KINDS[out][2]
    err = (y[:m, :n].double() - want).abs()
    tiny = 2.0 ** -25 if out == "f16" else 0.0     # half the smallest step of fp16
    assert (err <= e + (want.abs() + e) * half + tiny).all(), float((err - e - want.abs() * half).max())
    assert (y[m:] == -9).all() and (y[:, n:] == -9).all()


SHAPES = [(1, 1, 1), (1, 128, 128), (2, 130, 129), (16, 256, 384), (17, 100, 40), (31, 257, 1000), (33, 384, 512), (64, 1000, 130),
          (65, 129, 257), (128, 256, 1024), (129, 5, 2000), (201, 2053, 1000), (300, 513, 640), (1000, 260, 300)]


@pytest.mark.parametrize("m, n, k", SHAPES)
def test_product_against_64_bits(torch, m, n, k):
    g = torch.Generator("cuda").manual_seed(m * 7 + n * 3 + k)
    x, w = random_eight(torch, g, m, k, 1), random_eight(torch, g, n, k, 128)
    bias = torch.randn(n, generator=g, device="cuda") * 100
    for out in ("f32", "f16", "bf16", "e4m3"):
        if out == "f16":           # keep the products inside fp16
            w.scale[: w.groups, : w.blocks] *= 1e-3 / k
        check_product(torch, x, w, bias, False, out, call_product(torch, x, w, bias, False, out))
    check_product(torch, x, w, None, False, "f32", call_product(torch, x, w, None, False, "f32", pad=3))
    check_product(torch, x, w, bias, False, "bf16", call_product(torch, x, w, bias, False, "bf16", pad=1))


@pytest.mark.parametrize("m", [5, 200, 700])
@pytest.mark.parametrize("out", ["f32", "f16", "e4m3"])
def test_product_gelu(torch, m, out):
    g = torch.Generator("cuda").manual_seed(m)
    x, w = random_eight(torch, g, m, 384, 1), random_eight(torch, g, 300, 384, 128)
    w.scale[: w.groups, : w.blocks] *= 1e-3 / math.sqrt(384)
    bias = torch.randn(300, generator=g, device="cuda")
    check_product(torch, x, w, bias, True, out, call_product(torch, x, w, bias, True, out))


@pytest.mark.parametrize("m", [3, 100, 2600])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16", "e4m3"])
def test_product_gelu_by_its_argument(torch, m, out):
    """Zero products: y is GELU(bias), from the flat tail to the linear end.  The kernel takes |b| to at most 6 and
    Q = erfc(|b| / sqrt 2) / 2 as 2^P: a polynomial within 6.5e-8 of Q (8 bits: 3.2e-7), eight roundings of partial sums
    no larger than 1 + |P|, a 2^x within 2^-22 and the rounding of the last sum."""
    n = 640
    x, w = Eight(torch, m, 130), Eight(torch, n, 130, 128)
    for t in (x, w):
        t.q[:] = 0
        t.scale[:] = 1
    b = torch.linspace(-8, 8, n, device="cuda")
    if out != "e4m3":
        b[[0, 1, 2]] = torch.tensor([float("nan"), float("inf"), -float("inf")], device="cuda")
        b[[3, 4, 5]] = torch.tensor([3e4, -3e4, -0.0], device="cuda")
    y = call_product(torch, x, w, b, True, out)
    if out != "e4m3":
        assert torch.isnan(y[:m, 0]).all() and (y[:m, 1] == float("inf")).all() and (y[:m, 2].float().abs() < 1e-8).all()
        b[[0, 1, 2]] = 1.0
    v = b.double()
    a, q = v.abs().clamp(max=6), torch.special.erfc(v.abs().clamp(max=6) * math.sqrt(0.5)) / 2
    want = 0.5 * v * torch.special.erfc(-v * math.sqrt(0.5))
    poly = 3.2e-7 if out == "e4m3" else 6.5e-8
    e = a * (poly + q * (2.0 ** -22 + 2.0 ** -21 * (1 + q.log2().abs()))) + want.abs() * U + 6e-9
    if out == "e4m3":
        err = (y.values(torch) - want).abs()
        assert (err <= (want.abs() + e) * (2.0 ** -4 + 4 * U) + y.spans() * 2.0 ** -10 + e).all()
        return
    got = y[:m].double()
    err = (got - want).abs()[:, 3:]
    half, tiny = KINDS[out][2], 2.0 ** -25 if out == "f16" else 0.0
    assert (err <= (e + (want.abs() + e) * half + tiny)[3:]).all(), float((err - e[3:]).max())


@pytest.mark.parametrize("m", [3, 100, 2600])
@pytest.mark.parametrize("n", [129, 256, 300])
@pytest.mark.parametrize("low, high", [(-5.0, -2.0), (-6.0, -4.5), (-3.0, 3.0), (-1e-3, 1e-3), (-40.0, -9.0)])
def test_product_gelu_block_scales(torch, m, n, low, high):
    """Zero products: a block's 8 bits are GELU(bias) as the same call answers it in fp32, quantized, and its scale is
    the block's largest GELU / 448, also where all of a block lies in GELU's tail (or the last block is one column).
    GELU is within 2.3e-4 of its value down to -6, by at most 2.3e-4 + 2^-22 + eight roundings of partial sums no
    larger than 1 + |log2 Q| of the exponent, each worth ln 2 of it."""
    x, w = Eight(torch, m, 130), Eight(torch, n, 130, 128)
    for t in (x, w):
        t.q[:] = 0
        t.scale[:] = 1
    b = torch.linspace(low, high, n, device="cuda")
    y8, y = call_product(torch, x, w, b, True, "e4m3"), call_product(torch, x, w, b, True, "f32")[:m]
    codes, scales = quantized(torch, y, 1)
    assert torch.equal(y8.scales(), scales)
    assert torch.equal(y8.codes(torch).float(), codes.float())
    v = b.double()
    q = torch.special.erfc(v.abs() * math.sqrt(0.5)) / 2
    want = 0.5 * v * torch.special.erfc(-v * math.sqrt(0.5))
    if low < -6:                    # tiny, and never above what is left at -9
        assert (y <= 0).all() and (y.abs() <= 1.1e-18).all()
        return
    rel = 2.3e-4 + 2.0 ** -22 + 8 * U * math.log(2) * (1 + q.log2().abs()) + 3 * U
    assert ((y.double() - want).abs() <= want.abs() * rel).all()
    top = torch.zeros(up(n, 128), device="cuda", dtype=torch.float64)
    top[:n] = want.abs()
    top = top.view(-1, 128).amax(1) / 448
    assert ((y8.scales().double() / top[:, None] - 1).abs() <= float(rel.max()) + 4 * U).all()


LARGE = [(2048, 1024, 1024), (2500, 4736, 1024), (5184, 1000, 4736), (4097, 129, 100), (20000, 512, 100), (3000, 257, 4000),
         (30011, 11, 500), (9000, 1, 1)]


@pytest.mark.parametrize("m, n, k", LARGE)
@pytest.mark.parametrize("out, gelu", [("f32", False), ("f16", True), ("e4m3", True)])
def test_product_many_rows(torch, m, n, k, out, gelu):
    g = torch.Generator("cuda").manual_seed(m + n + k)
    x, w = random_eight(torch, g, m, k, 1), random_eight(torch, g, n, k, 128)
    w.scale[: w.groups, : w.blocks] *= 1e-3 / math.sqrt(k)
    bias = torch.randn(n, generator=g, device="cuda")
    check_product(torch, x, w, bias, gelu, out, call_product(torch, x, w, bias, gelu, out))
    if out == "f32":
        check_product(torch, x, w, None, gelu, "bf16", call_product(torch, x, w, None, gelu, "bf16", pad=5))


@pytest.mark.parametrize("m", [4, 150, 2600])
def test_product_nonfinite_rows_stay_apart(torch, m):
    """A NaN value, a NaN scale and an infinite scale reach their own rows and columns only."""
    g = torch.Generator("cuda").manual_seed(3)
    n, k = 200, 300
    x, w = random_eight(torch, g, m, k, 1), random_eight(torch, g, n, k, 128)
    x.q[1, 5] = 0x7F
    x.scale[1, 2] = float("nan")
    w.q[7, 290] = 0x7F
    y = call_product(torch, x, w, None, False, "f32")[:m]
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    bad[1] = bad[2] = True
    bad[:, 7] = True
    assert torch.equal(torch.isnan(y), bad)


@pytest.mark.parametrize("m", [4, 150, 2600])
@pytest.mark.parametrize("out", ["f32", "e4m3"])
@pytest.mark.parametrize("gelu", [False, True])
def test_product_infinite_scales(torch, m, out, gelu):
    """What a quantized block with an infinity leaves as its scale: its row (or its block of columns) becomes infinite,
    which 8 bits hold as an infinite scale, also where the block ends before 128 columns; all else stays as it was."""
    g = torch.Generator("cuda").manual_seed(3)
    n, k = 200, 300
    x, w = random_eight(torch, g, m, k, 1), random_eight(torch, g, n, k, 128)
    x.q &= 0x7F                     # no sum of a group is 0: even columns are positive, odd ones negative
    w.q &= 0x7F
    w.q[1:n:2] |= 0x80
    inf = float("inf")
    ends = torch.tensor([inf, 0.0 if gelu else -inf], device="cuda").repeat(n // 2)

    def call():
        y = call_product(torch, x, w, None, gelu, out)
        return (y.codes(torch).float(), y.scales().t()) if out == "e4m3" else (y[:m].clone(), None)

    before, before_scale = call()
    kept = float(x.scale[1, 3])
    x.scale[1, 3] = inf
    y, scale = call()
    others = torch.arange(m, device="cuda") != 3
    assert torch.equal(y[others], before[others])
    if out == "e4m3":
        assert (scale[3] == inf).all() and torch.equal(scale[others], before_scale[others])
    else:
        assert torch.equal(y[3], ends)
    x.scale[1, 3] = kept
    w.scale[2, 1] = inf
    y, scale = call()
    assert torch.equal(y[:, :128], before[:, :128])
    if out == "e4m3":
        assert torch.equal(scale[:, 0], before_scale[:, 0]) and (scale[:, 1] == inf).all()
    else:
        assert torch.equal(y[:, 128:], ends[128:].expand(m, -1))


@pytest.mark.parametrize("m, n, k", [(1, 4736, 1024), (100, 1024, 4736), (2600, 1024, 512)])
def test_product_repeats_on_streams_and_in_graphs(torch, m, n, k):
    g = torch.Generator("cuda").manual_seed(11)
    x, w = random_eight(torch, g, m, k, 1), random_eight(torch, g, n, k, 128)
    first = call_product(torch, x, w, None, False, "f32").clone()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [torch.full_like(first, -9.0) for _ in range(6)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for i, y in enumerate(outs):               # calls that overlap on three streams
        s3t.gemm_fp8(0, x.matrix, w.matrix, None, m, n, k, 0, s3t.TYPE_F32, s3t.Matrix(y.data_ptr(), n),
                     streams[i % 3].cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(y, first) for y in outs)
    graph, y = torch.cuda.CUDAGraph(), torch.full_like(first, -9.0)
    with torch.cuda.graph(graph):
        for _ in range(2):
            s3t.gemm_fp8(0, x.matrix, w.matrix, None, m, n, k, 0, s3t.TYPE_F32, s3t.Matrix(y.data_ptr(), n),
                         torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        y.fill_(-9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, first)


# ------------------------------------------------------------------- norms ---

def norm64(torch, v, e, weight, bias, layer, eps):
    """(norm, bound) of values v known to within e.  Sums take at most 64 fp32 roundings a term; an error d of the
    values moves the mean by mean(d), the root mean square by at most rms(d)."""
    mean = v.mean(1, keepdim=True) if layer else torch.zeros_like(v[:, :1])
    c = v - mean
    rstd = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
    w = 1.0 if weight is None else weight.double()
    out = c * rstd * w
    mean_e = (64 * U * v.abs().mean(1, keepdim=True) + e.mean(1, keepdim=True)) if layer else 0.0
    each = e + mean_e + U * (v.abs() + mean.abs())
    spread = torch.sqrt((each * each).mean(1, keepdim=True))
    bound = rstd * (each + c.abs() * rstd * spread) * (w if weight is None else w.abs()) + out.abs() * 50 * U
    if bias is not None:
        out = out + bias.double()
    return out, bound + out.abs() * 2 * U


def run_norm(torch, seed, rows, dim, kind, resid, layer=False, post=True, gate="none", gate_rows=1, channel=True, eight=False,
             pad=0, weights=True, branch=True, resid_scale=1.0, branch_scale=1.0, in_place=False, shift=0.0, write_x=True,
             write_u=True, stream=0):
    g = torch.Generator("cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    code, dtype, half = KINDS[kind]
    rcode, rdtype, rhalf = KINDS[resid]
    tdtype, trdtype = getattr(torch, dtype), getattr(torch, rdtype)
    x = rows_of(torch, rnd(rows, dim) * 2 + shift, trdtype, pad)
    y = rows_of(torch, rnd(rows, dim) + shift, tdtype, pad)
    y[rows // 2, :dim] = 0
    gates = up(rows, gate_rows) // gate_rows
    gt = rows_of(torch, rnd(gates, dim), tdtype, pad) if gate != "none" else None
    ch = rnd(dim) if channel and branch else None
    pw, pb, qw, qb = (rnd(dim) if weights else None for _ in range(4))
    x_in = x.clone()
    x_out = x if in_place else torch.full((rows + 1, dim + pad), -9.0, device="cuda", dtype=trdtype)
    u8 = Eight(torch, rows, dim) if eight else None
    u = torch.full((rows + 1, dim + pad), -9.0, device="cuda", dtype=tdtype)
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    flags = ((s3t.NORM_LAYER if layer else 0) | (s3t.NORM_POST if post and branch else 0)
             | {"sigmoid": s3t.NORM_GATE_SIGMOID, "tanh": s3t.NORM_GATE_TANH}.get(gate, 0))
    eps = 1e-5
    args = s3t.NormArgs(rows=rows, dim=dim, type=code, resid_type=rcode, u_type=s3t.TYPE_E4M3 if eight else code, flags=flags,
                        eps=eps, resid_scale=resid_scale, branch_scale=branch_scale, y=ptr(y) if branch else None,
                        y_stride=y.stride(0), post_weight=ptr(pw), post_bias=ptr(pb), gate=ptr(gt),
                        gate_stride=dim + pad, gate_rows=gate_rows, channel_scale=ptr(ch), x=ptr(x), x_stride=x.stride(0),
                        x_out=ptr(x_out) if write_x else None, x_out_stride=x_out.stride(0), pre_weight=ptr(qw),
                        pre_bias=ptr(qb),
                        u=(u8.matrix if eight else s3t.Matrix(u.data_ptr(), u.stride(0))) if write_u else s3t.Matrix())
    s3t.norm_residual(0, args, stream)
    torch.cuda.synchronize()
    # the formula in 64 bits
    want = resid_scale * x_in[:, :dim].double()
    e = want.abs() * U
    if branch:
        h = y[:, :dim].double()
        he = torch.zeros_like(h)
        if post:
            h, he = norm64(torch, h, he, pw, pb, layer, eps)
        if gt is not None:
            gv = gt[:, :dim].double()
            gv = torch.sigmoid(gv) if gate == "sigmoid" else torch.tanh(gv) if gate == "tanh" else gv
            gv = gv.repeat_interleave(gate_rows, 0)[:rows]
            h, he = h * gv, he * gv.abs() + (h * gv).abs() * 10 * U
        scale = branch_scale * (ch.double() if ch is not None else 1.0)
        h, he = h * scale, he * abs(scale) + (h * scale).abs() * 3 * U
        want = want + h
        e = e + he + want.abs() * U
    if write_x:
        err = (x_out[:rows, :dim].double() - want).abs()
        assert (err <= e + (want.abs() + e) * rhalf + (2.0 ** -25 if resid == "f16" else 0)).all(), float(err.max())
        if not in_place:
            assert (x_out[rows:] == -9).all() and (x_out[:, dim:] == -9).all()
    if write_u:
        un, ue = norm64(torch, want, e, qw, qb, layer, eps)
        if eight:
            assert ((u8.values(torch) - un).abs()
                    <= (un.abs() + ue) * (2.0 ** -4 + 4 * U) + u8.spans() * 2.0 ** -10 + ue).all()
            top = torch.zeros(rows, up(dim, 128), device="cuda", dtype=torch.float64)
            top[:, :dim] = un.abs()
            tope = torch.zeros_like(top)
            tope[:, :dim] = ue
            top, tope = (t.view(rows, -1, 128).amax(2) for t in (top, tope))
            top = top.clamp(min=2.0 ** -100) / 448
            assert ((u8.scales().t().double() - top).abs() <= tope / 448 + top * 3 * U).all()
            assert u8.untouched()
        else:
            err = (u[:rows, :dim].double() - un).abs()
            assert (err <= ue + (un.abs() + ue) * half + (2.0 ** -25 if kind == "f16" else 0)).all(), float(err.max())
            assert (u[rows:] == -9).all() and (u[:, dim:] == -9).all()
    return x_out, u


TYPE_PAIRS = [("f32", "f32"), ("f16", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16")]


@pytest.mark.parametrize("kind, resid", TYPE_PAIRS)
@pytest.mark.parametrize("rows, dim, pad", [(1, 1024, 0), (3, 1, 0), (5, 8, 0), (2, 255, 0), (201, 1001, 5), (33, 256, 8), (7, 2050, 0),
                                            (4, 4736, 0), (2, 16384, 0), (3, 16383, 1)])
@pytest.mark.parametrize("layer", [False, True])
def test_norm_sizes_and_types(torch, kind, resid, rows, dim, pad, layer):
    run_norm(torch, dim + rows, rows, dim, kind, resid, layer=layer, gate="plain", pad=pad)
    run_norm(torch, dim + rows, rows, dim, kind, resid, layer=layer, eight=True, pad=pad)


@pytest.mark.parametrize("gate", ["plain", "sigmoid", "tanh"])
@pytest.mark.parametrize("gate_rows", [1, 7, 1000])
def test_norm_gates(torch, gate, gate_rows):
    run_norm(torch, 5, 40, 264, "bf16", "f32", layer=True, gate=gate, gate_rows=gate_rows)
    run_norm(torch, 6, 40, 1021, "f16", "f16", post=False, gate=gate, gate_rows=gate_rows)


@pytest.mark.parametrize("rows, dim", [(2048, 1024), (2500, 264), (2051, 1001), (2049, 4736)])
def test_norm_many_rows(torch, rows, dim):
    run_norm(torch, 9, rows, dim, "f16", "f32", layer=True, gate="plain", gate_rows=500, eight=True)
    run_norm(torch, 9, rows, dim, "bf16", "bf16", gate="none")


@pytest.mark.parametrize("kind, resid", TYPE_PAIRS)
@pytest.mark.parametrize("rows, dim, pad", [(5000, 1024, 0), (4800, 264, 0), (4741, 1001, 0), (4740, 515, 3), (2400, 2050, 1),
                                            (1300, 4735, 0), (4739, 257, 16), (4745, 130, 0), (4737, 7, 1), (4800, 256, 0),
                                            (4736, 500, 4)])
def test_norm_streams_of_rows(torch, kind, resid, rows, dim, pad):
    """Enough rows for the persistent kernel (two a team), aligned and at any address."""
    run_norm(torch, 10, rows, dim, kind, resid, layer=True, gate="plain", gate_rows=7, eight=True, pad=pad)
    run_norm(torch, 11, rows, dim, kind, resid, gate="tanh", gate_rows=1000, pad=pad, in_place=True, resid_scale=0.5)
    run_norm(torch, 12, rows, dim, kind, resid, branch=False, layer=True, weights=False, pad=pad, write_x=False)


@pytest.mark.parametrize("kind, resid", TYPE_PAIRS)
@pytest.mark.parametrize("rows, dim, pad", [(1, 128, 0), (6, 127, 0), (1, 1, 0), (131, 64, 0), (67, 65, 3), (300, 32, 8), (129, 33, 1),
                                            (30001, 31, 0), (40007, 128, 0), (30003, 80, 1), (60005, 16, 0),
                                            (1184, 129, 0), (9001, 256, 0), (5003, 200, 8), (7001, 255, 1)])
def test_norm_narrow_rows(torch, kind, resid, rows, dim, pad):
    """Several rows a warp: whole and ragged warps, more rows than the grid takes at once."""
    run_norm(torch, 13, rows, dim, kind, resid, layer=True, gate="sigmoid", gate_rows=5, eight=True, pad=pad)
    run_norm(torch, 14, rows, dim, kind, resid, gate="tanh", gate_rows=1000, pad=pad, in_place=True, branch_scale=0.25)
    run_norm(torch, 15, rows, dim, kind, resid, branch=False, weights=False, pad=pad, write_x=False)
    run_norm(torch, 16, rows, dim, kind, resid, post=False, channel=False, layer=True, write_u=False, pad=pad)


def test_norm_narrow_nonfinite_rows_stay_apart(torch):
    rows, dim = 70, 64
    x = torch.randn(rows, dim, device="cuda")
    x[9, 3], x[34, 4] = float("nan"), -float("inf")
    u = Eight(torch, rows, dim)
    s3t.norm_residual(0, s3t.NormArgs(rows=rows, dim=dim, type=0, resid_type=0, u_type=s3t.TYPE_E4M3, flags=s3t.NORM_LAYER,
                                      eps=1e-5, resid_scale=1.0, x=x.data_ptr(), x_stride=dim, u=u.matrix))
    bad = torch.isnan(u.values(torch))
    assert bad[9].all() and bad[34].all() and int(bad.any(1).sum()) == 2 and u.untouched()


@pytest.mark.parametrize("kind, resid", TYPE_PAIRS)
@pytest.mark.parametrize("rows, dim, pad", [(5, 4097, 0), (9, 8192, 0), (3, 8193, 3), (620, 5120, 0), (310, 7001, 1), (300, 8200, 0),
                                            (301, 9024, 0), (299, 12289, 0), (330, 16384, 0)])
def test_norm_wide_rows(torch, kind, resid, rows, dim, pad):
    """Rows of 5 to 16 streaming warps, and those that one CTA a row takes."""
    run_norm(torch, 17, rows, dim, kind, resid, layer=True, gate="sigmoid", gate_rows=3, eight=True, pad=pad)
    run_norm(torch, 18, rows, dim, kind, resid, weights=False, pad=pad, in_place=True)
    run_norm(torch, 19, rows, dim, kind, resid, branch=False, pad=pad, write_x=False)
    run_norm(torch, 20, rows, dim, kind, resid, post=False, weights=False, gate="plain", write_u=False, pad=pad)


@pytest.mark.parametrize("kind, resid", TYPE_PAIRS)
@pytest.mark.parametrize("rows, dim, pad", [(900, 6144, 0), (1790, 8192, 0), (1490, 9024, 0), (1481, 7070, 3), (4450, 5111, 0)])
def test_norm_streams_of_wide_rows(torch, kind, resid, rows, dim, pad):
    """Rows enough for teams of 5 to 9 warps, one to three an SM, to stream rows of more than 4096 columns."""
    run_norm(torch, 21, rows, dim, kind, resid, layer=True, gate="plain", gate_rows=500, pad=pad)
    run_norm(torch, 22, rows, dim, kind, resid, eight=True, pad=pad, in_place=True)


@pytest.mark.parametrize("kind, resid, rows, dim", [("f32", "f32", 4445, 9024), ("f16", "f32", 2371, 12288), ("f16", "f16", 2371, 10001),
                                                    ("bf16", "bf16", 2370, 16384), ("bf16", "f32", 2370, 13000)])
def test_norm_streams_of_the_widest_rows(torch, kind, resid, rows, dim):
    """One team of 9 to 16 warps an SM."""
    run_norm(torch, 23, rows, dim, kind, resid)


def test_norm_parts_that_are_left_out(torch):
    for dim in (256, 515):
        run_norm(torch, 1, 9, dim, "f16", "f32", branch=False)                                  # a pre-norm alone
        run_norm(torch, 2, 9, dim, "f16", "f32", branch=False, write_x=False, layer=True, weights=False, channel=False,
                 resid_scale=0.5)
        run_norm(torch, 3, 9, dim, "f32", "f32", write_u=False)                                 # a post-norm alone
        run_norm(torch, 4, 9, dim, "bf16", "f32", post=False, channel=False, weights=False, resid_scale=0.7,
                 branch_scale=-1.5)
        run_norm(torch, 5, 9, dim, "f16", "f16", in_place=True, eight=True)


def test_norm_far_from_zero(torch):
    """A mean a thousand times the spread: the variance must not come from a difference of squares."""
    for dim in (1024, 4736, 1003):
        run_norm(torch, 8, 6, dim, "f32", "f32", layer=True, shift=2000.0, post=True, channel=False)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows, dim, pad", [(131, 7, 0), (300, 32, 0), (300, 64, 0), (300, 128, 0), (67, 65, 3), (30001, 31, 0),
                                            (1200, 130, 0), (1200, 256, 0), (1201, 255, 1), (5000, 512, 0), (5000, 1024, 0),
                                            (4741, 1001, 0), (2400, 2050, 1), (700, 4096, 0), (900, 6144, 0)])
def test_norm_far_from_zero_by_the_width_of_a_row(torch, kind, rows, dim, pad):
    """As above for every lane count of the narrow kernel, and streaming teams of one and of several warps: y and x a
    thousand spreads from zero (16-bit values of them: the spread is their rounding's)."""
    shift = 2000.0 if kind == "f32" else 500.0
    run_norm(torch, 24, rows, dim, kind, kind, layer=True, shift=shift, post=True, channel=False, pad=pad)
    run_norm(torch, 25, rows, dim, kind, "f32", layer=True, shift=shift, branch=False, pad=pad)


def test_norm_nonfinite_rows_stay_apart(torch):
    for rows, dim in ((5, 1024), (2100, 512), (5, 301), (5000, 512), (5000, 1003)):
        x = torch.randn(rows, dim, device="cuda")
        x[1, 3], x[2, 4] = float("nan"), float("inf")
        u = torch.empty(rows, dim, device="cuda")
        s3t.norm_residual(0, s3t.NormArgs(rows=rows, dim=dim, type=0, resid_type=0, u_type=0, flags=s3t.NORM_LAYER, eps=1e-5,
                                          resid_scale=1.0, x=x.data_ptr(), x_stride=dim, u=s3t.Matrix(u.data_ptr(), dim)))
        bad = torch.isnan(u).any(1)
        assert bad[1] and bad[2] and int(bad.sum()) == 2


# ------------------------------------------------------------------ rotary ---

def turned64(torch, x, positions, freq, rot, magnitude, interleaved, inverse):
    angle = positions.double()[:, None] * freq
    c, s = torch.cos(angle)[:, None] * magnitude, torch.sin(angle)[:, None] * magnitude
    if inverse:
        s = -s
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., : rot // 2], x[..., rot // 2: rot])
    out, mag = x.clone(), torch.zeros_like(x)
    size = (a.abs() + b.abs()) * magnitude
    if interleaved:
        out[..., 0:rot:2], out[..., 1:rot:2] = a * c - b * s, a * s + b * c
        mag[..., 0:rot:2] = mag[..., 1:rot:2] = size
    else:
        out[..., : rot // 2], out[..., rot // 2: rot] = a * c - b * s, a * s + b * c
        mag[..., : rot // 2] = mag[..., rot // 2: rot] = size
    return out, mag * 8 * U      # the turn to 2^-26, sincospif to 2 steps, magnitude, two products and a sum


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens, heads, kheads, dim, rot", [(1, 1, 0, 2, 2), (8, 16, 4, 64, 64), (5, 3, 1, 80, 32), (700, 4, 4, 128, 96),
                                                             (3, 2, 2, 37, 10), (2, 1, 1, 256, 64), (4, 2, 0, 1024, 1024),
                                                             (1300, 1, 1, 66, 66)])
def test_rotary_against_64_bits(torch, kind, interleaved, tokens, heads, kheads, dim, rot):
    code, dtype, half = KINDS[kind]
    g = torch.Generator("cuda").manual_seed(tokens + dim)
    freq, magnitude = s3t.rotary_frequencies(rot, 10000.0, s3t.ROTARY_BY_PARTS, 8.0, 4096.0)
    freq = torch.from_numpy(freq).cuda()
    positions = torch.randint(0, 1 << 27, (tokens,), generator=g, device="cuda")
    positions[0] = 0
    if tokens > 2:
        positions[2] = -1
    # a packed projection: q heads, k heads, and columns that belong to v
    x = torch.randn(tokens, (heads + kheads) * dim + 16, generator=g, device="cuda").to(getattr(torch, dtype))
    size, width = x.element_size(), x.stride(0)
    for inverse in (False, True):
        q = torch.full((heads, tokens, dim), 5.0, device="cuda", dtype=x.dtype)      # head-major out
        packed = x.clone()
        kview = s3t.RotaryView(packed.data_ptr() + heads * dim * size, packed.data_ptr() + heads * dim * size, kheads, width, dim,
                               width, dim) if kheads else None                       # in place
        s3t.rotary(0, freq.data_ptr(), rot, magnitude, positions.data_ptr(), tokens, code, dim,
                   s3t.RotaryView(packed.data_ptr(), q.data_ptr(), heads, width, dim, dim, tokens * dim), kview,
                   (s3t.ROTARY_INTERLEAVED if interleaved else 0) | (s3t.ROTARY_INVERSE if inverse else 0))
        x64 = x[:, : (heads + kheads) * dim].double().view(tokens, heads + kheads, dim)
        want, e = turned64(torch, x64, positions, freq, rot, magnitude, interleaved, inverse)
        there = positions >= 0
        e = e + want.abs() * half + (2.0 ** -25 if kind == "f16" else 0)
        got = q.permute(1, 0, 2)
        assert ((got[there].double() - want[there][:, :heads]).abs() <= e[there][:, :heads]).all()
        assert (got[~there] == 5).all()
        assert torch.equal(packed[:, (heads + kheads) * dim:], x[:, (heads + kheads) * dim:])
        assert torch.equal(packed[:, : heads * dim], x[:, : heads * dim])
        if kheads:
            k = packed[:, heads * dim: (heads + kheads) * dim].view(tokens, kheads, dim)
            assert ((k[there].double() - want[there][:, heads:]).abs() <= e[there][:, heads:]).all()
            assert torch.equal(k[~there], x[:, heads * dim: (heads + kheads) * dim].view(tokens, kheads, dim)[~there])
        assert torch.equal(got[there][..., rot:], x[:, : heads * dim].view(tokens, heads, dim)[there][..., rot:])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("quarter", [0, 1, 2, 3])
def test_rotary_next_to_quarter_turns(torch, interleaved, quarter):
    """Heads of pairs (1, 0) answer with the cosine and sine themselves.  Next to a quarter turn one of them is small and
    as exact as its type: sincospif to a step (2^-23), one sum's rounding (2^-24), and 1e-13 for the 64-bit angle."""
    n, tokens = 256, 5
    away = torch.exp(torch.linspace(math.log(1e-5), math.log(1e-2), n, dtype=torch.float64)) * (-1) ** torch.arange(n)
    freq = (2 * math.pi * (quarter / 4 + 1 + away)).cuda()
    positions = torch.tensor([1, 5, -1, 9, 13], device="cuda")       # whole quarter turns away from one another
    x = torch.zeros(tokens, 2 * n, device="cuda")
    if interleaved:
        x[:, ::2] = 1
    else:
        x[:, :n] = 1
    y = torch.full_like(x, 5.0)
    s3t.rotary(0, freq.data_ptr(), 2 * n, 1.0, positions.data_ptr(), tokens, s3t.TYPE_F32, 2 * n,
               s3t.RotaryView(x.data_ptr(), y.data_ptr(), 1, 2 * n, 2 * n, 2 * n, 2 * n), None,
               s3t.ROTARY_INTERLEAVED if interleaved else 0)
    got = y.view(tokens, n, 2) if interleaved else y.view(tokens, 2, n).transpose(1, 2)
    angle = positions.double()[:, None] * freq
    want = torch.stack((angle.cos(), angle.sin()), -1)
    there = positions >= 0
    assert ((got.double() - want).abs() <= want.abs() * (2.0 ** -23 + 2.0 ** -24) * 1.01 + 1e-13)[there].all()
    assert (got[~there] == 5).all()


@pytest.mark.parametrize("tokens, heads, token, head", [(5, 3, 192, 256), (9, 2, 160, 640 + 80), (1, 4, 0, 64), (6, 1, 64, 0)])
def test_rotary_layouts_that_interleave(torch, tokens, heads, token, head):
    """Heads of out between one another's tokens, neither token- nor head-major, and strides that nothing uses; every
    head of x the same one (strides of 0)."""
    dim = 64
    x = torch.randn(dim, device="cuda")
    freq, _ = s3t.rotary_frequencies(dim)
    freq, positions = torch.from_numpy(freq).cuda(), torch.arange(tokens, device="cuda") * 17
    at = torch.arange(tokens)[:, None] * token + torch.arange(heads) * head
    out = torch.full((int(at.max()) + dim + 8,), 5.0, device="cuda")
    s3t.rotary(0, freq.data_ptr(), dim, 1.0, positions.data_ptr(), tokens, s3t.TYPE_F32, dim,
               s3t.RotaryView(x.data_ptr(), out.data_ptr(), heads, 0, 0, token, head))
    want, e = turned64(torch, x.double().expand(tokens, heads, dim), positions, freq, dim, 1.0, False, False)
    places = (at[..., None] + torch.arange(dim)).cuda()
    assert ((out[places].double() - want).abs() <= e + want.abs() * U).all()
    out[places] = 5.0
    assert (out == 5.0).all()


def test_rotary_offsets_past_32_bits(torch):
    """Token strides that put the last token over 2^32 elements away (a slot of a long cache)."""
    stride, tokens, dim = (1 << 31) + 64, 3, 64
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 18 GB of free device memory")
    cache = torch.empty(2 * stride + dim, device="cuda", dtype=torch.float16)
    x = torch.randn(tokens, dim, device="cuda").half()
    freq, _ = s3t.rotary_frequencies(dim)
    freq, positions = torch.from_numpy(freq).cuda(), torch.tensor([5, 70000, 123], device="cuda")
    s3t.rotary(0, freq.data_ptr(), dim, 1.0, positions.data_ptr(), tokens, s3t.TYPE_F16, dim,
               s3t.RotaryView(x.data_ptr(), cache.data_ptr(), 1, dim, dim, stride, dim))
    want, e = turned64(torch, x.double()[:, None], positions, freq, dim, 1.0, False, False)
    for t in range(tokens):
        got = cache[t * stride: t * stride + dim].double()
        assert ((got - want[t, 0]).abs() <= e[t, 0] + want[t, 0].abs() * 2.0 ** -11 + 2.0 ** -25).all()


def test_quantize_and_product_past_32_bits(torch):
    """Rows of x, q and y that lie more than 2^32 elements apart, for both product kernels."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 50 GB of free device memory")
    g = torch.Generator("cuda").manual_seed(2)
    for m, n, k, stride in ((3, 130, 200, (1 << 31) + 16), (161, 4736, 1024, (1 << 26) + 16)):
        w = random_eight(torch, g, n, k, 128)
        w.scale[: w.groups, : w.blocks] *= 1e-3
        x = torch.randn(m, k, generator=g, device="cuda").half()
        q = torch.empty((m - 1) * stride + k, device="cuda", dtype=torch.uint8)
        scale = torch.empty(up(k, 128) // 128, m, device="cuda")
        s3t.quantize_fp8(0, s3t.TYPE_F16, x.data_ptr(), m, k, k, 1, s3t.Matrix(q.data_ptr(), stride, scale.data_ptr(), m))
        codes, want_scale = quantized(torch, x.float(), 1)
        rows = torch.stack([q[i * stride: i * stride + k] for i in range(m)]).view(torch.float8_e4m3fn)
        assert torch.equal(rows.float(), codes.float()) and torch.equal(scale, want_scale)
        y = torch.empty((m - 1) * stride + n, device="cuda", dtype=torch.float16)
        xm = s3t.Matrix(q.data_ptr(), stride, scale.data_ptr(), m)
        s3t.gemm_fp8(0, xm, w.matrix, None, m, n, k, 0, s3t.TYPE_F16, s3t.Matrix(y.data_ptr(), stride))
        near = torch.empty(m, n, device="cuda", dtype=torch.float16)
        s3t.gemm_fp8(0, xm, w.matrix, None, m, n, k, 0, s3t.TYPE_F16, s3t.Matrix(near.data_ptr(), n))
        assert torch.equal(torch.stack([y[i * stride: i * stride + n] for i in range(m)]), near)
        xv = rows.double() * scale.t().double().repeat_interleave(128, 1)[:, :k]
        want, mag = xv @ w.values(torch).t(), xv.abs() @ w.values(torch).abs().t()
        e = mag * (128 + up(k, 128) // 128 + 8) * 2 * U
        assert ((near.double() - want).abs() <= e + (want.abs() + e) * 2.0 ** -11 + 2.0 ** -25).all()
        del q, y


def test_calls_from_two_threads(torch):
    """Two host threads, a stream each, every operator: the same results as one after the other."""
    import threading
    dim, rows = 512, 300
    g = torch.Generator("cuda").manual_seed(4)
    w = random_eight(torch, g, 384, dim, 128)

    def work(seed, stream, out):
        gg = torch.Generator("cuda").manual_seed(seed)
        x = torch.randn(rows, dim, generator=gg, device="cuda")
        u = Eight(torch, rows, dim)
        y = torch.empty(rows, 384, device="cuda", dtype=torch.float16)
        q8 = Eight(torch, rows, 384)
        torch.cuda.synchronize()
        st = stream.cuda_stream
        for _ in range(20):
            s3t.norm_residual(0, s3t.NormArgs(rows=rows, dim=dim, type=1, resid_type=0, u_type=s3t.TYPE_E4M3, eps=1e-6,
                                              resid_scale=1.0, x=x.data_ptr(), x_stride=dim, u=u.matrix), st)
            s3t.gemm_fp8(0, u.matrix, w.matrix, None, rows, 384, dim, 1, s3t.TYPE_F16, s3t.Matrix(y.data_ptr(), 384), st)
            s3t.quantize_fp8(0, s3t.TYPE_F16, y.data_ptr(), rows, 384, 384, 1, q8.matrix, st)
        stream.synchronize()
        out[seed] = (y.clone(), q8.q.clone(), q8.scale.clone())

    alone, together = {}, {}
    streams = [torch.cuda.Stream() for _ in range(2)]
    for seed in (1, 2):
        work(seed, streams[0], alone)
    threads = [threading.Thread(target=work, args=(seed, streams[seed - 1], together)) for seed in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for seed in (1, 2):
        assert all(torch.equal(a, b) for a, b in zip(alone[seed], together[seed]))


def test_errors_stay_with_their_callers(torch):
    """A refused device leaves no error in the runtime for the next check of the caller's (torch makes one after every
    launch), and a call does not report an error that was there before it."""
    import ctypes
    runtime = ctypes.CDLL("libcudart.so.12")
    x, w = Eight(torch, 4, 256), Eight(torch, 256, 256, 128)
    for t in (x, w):
        t.q[:] = 0
        t.scale[:] = 1
    v, y = torch.ones(4, 256, device="cuda"), torch.zeros(4, 256, device="cuda")
    wide, wide_y = torch.ones(2, 8192, device="cuda"), torch.zeros(2, 8192, device="cuda")
    many, many_y = torch.ones(5000, 512, device="cuda"), torch.zeros(5000, 512, device="cuda")
    many8, many8_y = Eight(torch, 2600, 256), torch.zeros(2600, 256, device="cuda")
    freq, positions = torch.ones(32, device="cuda", dtype=torch.float64), torch.zeros(4, device="cuda", dtype=torch.int64)
    view = s3t.RotaryView(v.data_ptr(), y.data_ptr(), 4, 256, 64, 256, 64)

    def norm(device, rows, dim, x, u):
        s3t.norm_residual(device, s3t.NormArgs(rows=rows, dim=dim, eps=1e-5, resid_scale=1.0, x=x.data_ptr(), x_stride=dim,
                                               u=s3t.Matrix(u.data_ptr(), dim)))

    calls = [
        lambda d: s3t.quantize_fp8(d, s3t.TYPE_F32, v.data_ptr(), 4, 256, 256, 1, x.matrix),
        lambda d: s3t.quantize_fp8(d, s3t.TYPE_F32, v.data_ptr(), 4, 256, 256, 128, w.matrix),
        lambda d: s3t.gemm_fp8(d, x.matrix, w.matrix, None, 4, 256, 256, 0, s3t.TYPE_F32, s3t.Matrix(y.data_ptr(), 256)),
        lambda d: s3t.gemm_fp8(d, many8.matrix, w.matrix, None, 2600, 256, 256, 0, s3t.TYPE_F32,
                               s3t.Matrix(many8_y.data_ptr(), 256)),
        lambda d: norm(d, 4, 256, v, y),
        lambda d: norm(d, 16, 64, v, y),
        lambda d: norm(d, 2, 8192, wide, wide_y),
        lambda d: norm(d, 5000, 512, many, many_y),
        lambda d: s3t.rotary(d, freq.data_ptr(), 64, 1.0, positions.data_ptr(), 4, s3t.TYPE_F32, 64, view),
    ]
    torch.cuda.synchronize()
    for call in calls:
        assert runtime.cudaPeekAtLastError() == 0
        with pytest.raises(s3t.S3TError):
            call(4096)
        assert runtime.cudaPeekAtLastError() == 0
        error = runtime.cudaSetDevice(4096)             # the caller's own, on the host only
        assert error != 0 and runtime.cudaPeekAtLastError() == error
        call(0)
        assert runtime.cudaGetLastError() == error
    torch.cuda.synchronize()


def test_small_operators_in_a_graph(torch):
    """Quantization, the norms and rotary captured once and replayed on new values in the same buffers."""
    rows, dim = 9, 256
    x, y = torch.empty(rows, dim, device="cuda"), torch.empty(rows, dim, device="cuda", dtype=torch.float16)
    xo, u8, q = torch.empty_like(x), Eight(torch, rows, dim), torch.empty_like(y)
    freq, _ = s3t.rotary_frequencies(32)
    freq, positions = torch.from_numpy(freq).cuda(), torch.arange(rows, device="cuda")

    def step():
        st = torch.cuda.current_stream().cuda_stream
        s3t.norm_residual(0, s3t.NormArgs(rows=rows, dim=dim, type=1, resid_type=0, u_type=s3t.TYPE_E4M3, flags=s3t.NORM_POST,
                                          eps=1e-5, resid_scale=1.0, branch_scale=1.0, y=y.data_ptr(), y_stride=dim,
                                          x=x.data_ptr(), x_stride=dim, x_out=xo.data_ptr(), x_out_stride=dim, u=u8.matrix), st)
        s3t.rotary(0, freq.data_ptr(), 32, 1.0, positions.data_ptr(), rows, s3t.TYPE_F16, 32,
                   s3t.RotaryView(y.data_ptr(), q.data_ptr(), 8, dim, 32, dim, 32), None, 0, st)

    def fill(seed):
        g = torch.Generator("cuda").manual_seed(seed)
        x.copy_(torch.randn(rows, dim, generator=g, device="cuda"))
        y.copy_(torch.randn(rows, dim, generator=g, device="cuda"))

    graph = torch.cuda.CUDAGraph()
    fill(0)
    with torch.cuda.graph(graph):
        step()
    for seed in (1, 2):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [xo.clone(), u8.q.clone(), u8.scale.clone(), q.clone()]
        for t in (xo, u8.q, u8.scale, q):
            t.zero_()
        step()
        torch.cuda.synchronize()
        u8_rows = [xo, u8.q, u8.scale, q]
        assert torch.equal(got[0], xo) and torch.equal(got[3], q)
        assert torch.equal(got[1][:rows, :dim], u8_rows[1][:rows, :dim])
        assert torch.equal(got[2][:2, :rows], u8_rows[2][:2, :rows])


# ---------------------------------------------------------------- together ---

@pytest.mark.parametrize("tokens", [1, 201, 2100])
def test_an_attention_block_in_8_bits(torch, tokens):
    """The operators as a block runs them: pre-norm to 8 bits, q and k products, rotary positions, the d = 32
    attention, the output product, and the closing post-norm, gate and residual, against the same steps in 64 bits
    with their roundings to 8 and 16 bits.  A value within an fp16 rounding (2^-11, twice) of an e4m3 boundary may fall on
    its other side: about 2 * 2^-11 / 2^-4 of the values move by 2^-3.5, an rms change of 2^-3.5 * sqrt(2^-6) = 1.1e-2
    of the operand; three such operands in a row and the attention's own 2e-3 stay below 2.5e-2."""
    dim, heads = 256, 8
    g = torch.Generator("cuda").manual_seed(tokens)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x = rnd(tokens, dim)
    weights = [rnd(2 * dim, dim) / 16, rnd(dim, dim) / 16, rnd(dim, dim) / 16]
    w8 = []
    for w in weights:
        m = Eight(torch, w.shape[0], dim, 128)
        s3t.quantize_fp8(0, s3t.TYPE_F32, w.data_ptr(), w.shape[0], dim, dim, 128, m.matrix)
        w8.append(m)
    ls, gate = rnd(dim), rnd(1, dim).half()
    freq, magnitude = s3t.rotary_frequencies(32, 10000.0, s3t.ROTARY_LINEAR, 2.0)
    freq, positions = torch.from_numpy(freq).cuda(), torch.arange(tokens, device="cuda") + 1000
    half = lambda n: torch.empty(tokens, n, device="cuda", dtype=torch.float16)  # noqa: E731
    u, a8, qk, q, k, v, attn, y = Eight(torch, tokens, dim), Eight(torch, tokens, dim), half(512), half(256), half(256), half(256), \
        half(256), half(256)
    out = torch.empty_like(x)
    mat = lambda t: s3t.Matrix(t.data_ptr(), t.stride(0))  # noqa: E731
    s3t.norm_residual(0, s3t.NormArgs(rows=tokens, dim=dim, type=1, resid_type=0, u_type=s3t.TYPE_E4M3, eps=1e-6, resid_scale=1.0,
                                      x=x.data_ptr(), x_stride=dim, u=u.matrix))
    s3t.gemm_fp8(0, u.matrix, w8[0].matrix, None, tokens, 512, dim, 0, s3t.TYPE_F16, mat(qk))
    s3t.gemm_fp8(0, u.matrix, w8[1].matrix, None, tokens, 256, dim, 0, s3t.TYPE_F16, mat(v))
    s3t.rotary(0, freq.data_ptr(), 32, magnitude, positions.data_ptr(), tokens, s3t.TYPE_F16, 32,
               s3t.RotaryView(qk.data_ptr(), q.data_ptr(), heads, 512, 32, 256, 32),
               s3t.RotaryView(qk.data_ptr() + 512, k.data_ptr(), heads, 512, 32, 256, 32))
    s3t.mha_d32(0, q.data_ptr(), k.data_ptr(), v.data_ptr(), 1, tokens, tokens, None, attn.data_ptr(), s3t.MHA_OUT_F16)
    s3t.quantize_fp8(0, s3t.TYPE_F16, attn.data_ptr(), tokens, dim, dim, 1, a8.matrix)
    s3t.gemm_fp8(0, a8.matrix, w8[2].matrix, None, tokens, 256, dim, 0, s3t.TYPE_F16, mat(y))
    s3t.norm_residual(0, s3t.NormArgs(rows=tokens, dim=dim, type=1, resid_type=0, u_type=1, eps=1e-6, resid_scale=1.0, branch_scale=1.0,
                                      flags=s3t.NORM_POST | s3t.NORM_GATE_SIGMOID, y=y.data_ptr(), y_stride=dim,
                                      gate=gate.data_ptr(), gate_stride=0, gate_rows=tokens, channel_scale=ls.data_ptr(),
                                      x=x.data_ptr(), x_stride=dim, x_out=out.data_ptr(), x_out_stride=dim))
    torch.cuda.synchronize()

    def eighth(t):
        c, s = quantized(torch, t.float(), 1)
        return c.double() * s.t().double().repeat_interleave(128, 1)

    rms = lambda t: t / torch.sqrt((t * t).mean(1, keepdim=True) + 1e-6)  # noqa: E731
    r16 = lambda t: t.half().double()  # noqa: E731
    u64 = eighth(rms(x.double()))
    qk64, v64 = r16(u64 @ w8[0].values(torch).t()), r16(u64 @ w8[1].values(torch).t())
    turned, _ = turned64(torch, qk64.view(tokens, 16, 32), positions, freq, 32, magnitude, False, False)
    q64, k64 = r16(turned[:, :8]).permute(1, 0, 2), r16(turned[:, 8:]).permute(1, 0, 2)
    p = torch.softmax(q64 @ k64.transpose(1, 2) / math.sqrt(32.0), -1)
    attn64 = r16((p @ v64.view(tokens, 8, 32).permute(1, 0, 2)).permute(1, 0, 2).reshape(tokens, 256))
    y64 = r16(eighth(attn64) @ w8[2].values(torch).t())
    branch = torch.sigmoid(gate.double()) * ls.double() * rms(y64)
    got = out.double() - x.double()
    rel = float((got - branch).norm() / branch.norm())
    assert rel < 2.5e-2, rel
