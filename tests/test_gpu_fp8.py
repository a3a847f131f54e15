"""The 8-bit row operators and projections against their plain forms in 64 bits."""
import pytest
import torch

from hashattention import _ops
from tests import fp8_util as ref

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def noise(*shape, seed=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float64) * scale


def rows(m, k):
    """Output rows filled with a pattern, so that what a kernel does not write shows."""
    q, s = _ops.fp8_rows(m, k, DEV)
    q.view(torch.uint8).fill_(0x5a)
    s.fill_(-7.0)
    return q, s


# ------------------------------------------------------------------------------------------ rows as they are

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 127), (2, 129), (17, 100), (5, 4096), (33, 1003), (16, 14336), (301, 640)])
def test_quantize_rows(dtype, m, k):
    x = (noise(m, k, seed=m + k) * torch.exp(2 * noise(1, k, seed=1))).to(dtype)
    q, s = rows(m, k)
    _ops.quantize_rows_fp8(x, q, s)
    ref.assert_rows(q, s, x.double(), 0.0)
    assert torch.allclose(_ops.fp8_values(q, s, k).double(), x.double(), rtol=0, atol=float(x.double().abs().max()) * 2.0 ** -4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,stride", [(0, 200), (8, 304), (1, 201), (3, 300)])
def test_quantize_rows_strided_and_unaligned(dtype, offset, stride):
    m, k = 9, 199
    wide = noise(m * stride + 16, seed=5).to(dtype)
    x = wide[offset:offset + m * stride].view(m, stride)[:, :k]
    big_q = torch.full((m + 1, 3 * 128), 0x5a, dtype=torch.uint8, device=DEV)
    big_s = torch.full((m + 1, 5), -7.0, device=DEV)
    _ops.quantize_rows_fp8(x, big_q[:m, :256].view(torch.float8_e4m3fn), big_s[:m, :2])
    ref.assert_rows(big_q[:m, :256].view(torch.float8_e4m3fn), big_s[:m, :2], x.double(), 0.0)
    assert (big_q[:, 256:] == 0x5a).all() and (big_q[m] == 0x5a).all(), "behind a row's blocks and behind the last row: as it was"
    assert (big_s[:, 2:] == -7.0).all() and (big_s[m] == -7.0).all()


def test_every_e4m3_number_and_the_ties_between_them():
    """A block whose largest magnitude is 448 has scale 1: every e4m3 number comes back as itself, every midpoint goes to the
    even neighbour, and what lies a bf16 step off a midpoint to the nearer one."""
    grid = torch.arange(0, 0x7f, dtype=torch.uint8).view(torch.float8_e4m3fn).double()       # 0 .. 448
    mid = (grid[1:] + grid[:-1]) / 2
    values = torch.cat([grid, -grid, mid, -mid, mid * (1 + 2.0 ** -12), mid * (1 - 2.0 ** -12)])
    n = ref.blocks(values.numel() + 1)
    x = torch.zeros(n, 128, dtype=torch.float64)
    x.view(-1)[torch.arange(values.numel()) + torch.arange(values.numel()) // 127] = values   # every block keeps a place for its 448
    x[:, 127] = 448.0
    x = x.float().to(DEV)
    q, s = rows(n, 128)
    _ops.quantize_rows_fp8(x, q, s)
    assert (s == 1.0).all()
    assert torch.equal(q.double(), ref.round_e4m3(x.double()))
    assert torch.equal(q.float(), x.to(torch.float8_e4m3fn).float())


@pytest.mark.parametrize("dtype", DTYPES)
def test_zero_tiny_and_non_finite_blocks(dtype):
    x = noise(6, 384, seed=9).to(dtype)
    x[0] = 0
    x[1, 128:256] = 0
    x[2, 130] = float("inf")
    x[3, 5] = float("nan")
    x[4, 300] = float("-inf")
    x[4, 301] = float("nan")
    x[5] = 0
    x[5, 7] = torch.finfo(dtype).tiny
    q, s = rows(6, 384)
    _ops.quantize_rows_fp8(x, q, s)
    v = _ops.fp8_values(q, s, 384)
    assert (v[0] == 0).all() and (s[0] == 1).all() and (v[1, 128:256] == 0).all() and s[1, 1] == 1
    assert v[2, 128:256].isnan().all() and v[2, :128].isfinite().all() and v[2, 256:].isfinite().all()
    assert v[3, :128].isnan().all() and v[3, 128:].isfinite().all()
    assert v[4, 256:].isnan().all() and v[4, :256].isfinite().all()
    ref.assert_rows(q[:2], s[:2], x[:2].double(), 0.0)
    ref.assert_rows(q[5:], s[5:], x[5:].double(), 0.0)


# ------------------------------------------------------------------------------------------ SwiGLU

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,f", [(1, 1), (4, 14336), (3, 129), (16, 128), (67, 1001), (2, 4100)])
def test_swiglu(dtype, m, f):
    x = noise(m, 2 * f, seed=m + f, scale=3.0).to(dtype)
    q, s = rows(m, f)
    _ops.swiglu_fp8(x, q, s)
    g, u = x[:, :f].double(), x[:, f:].double()
    # exponential to 2 ulp, sum, quotient (2.5 ulp), product: below 2^-20
    ref.assert_rows(q, s, g * torch.sigmoid(g) * u, 2.0 ** -20)


def test_swiglu_far_gates():
    """Gates far out: silu(-200) is 0 (the exponential overflows, the quotient is 0), silu(200) is 200; a NaN stays in its block."""
    f = 256
    x = noise(3, 2 * f, seed=3)
    x[0, :f] = -200.0
    x[1, :f] = 200.0
    x[2, 3] = float("nan")
    q, s = rows(3, f)
    _ops.swiglu_fp8(x.float(), q, s)
    v = _ops.fp8_values(q, s, f)
    assert (v[0] == 0).all() and (s[0] == 1).all()
    ref.assert_rows(q[1:2], s[1:2], 200.0 * x[1:2, f:].float().double(), 2.0 ** -20)
    assert v[2, :128].isnan().all() and v[2, 128:].isfinite().all()


@pytest.mark.parametrize("gate", [88.0, -86.0, 1e4, 2.0e38, 2.4e38, 3.4e38])
def test_swiglu_gates_up_to_the_largest_number(gate):
    """silu(g) = g up to the largest fp32 number, whose product with log2(e) overflows."""
    x = torch.zeros(2, 2 * 128, device=DEV)
    x[:, :128] = gate
    x[:, 128:] = torch.linspace(0.5, 1.0, 128, device=DEV) * (1e-35 if gate > 1e30 else 1.0)
    q, s = rows(2, 128)
    _ops.swiglu_fp8(x, q, s)
    g, u = x[:, :128].double(), x[:, 128:].double()
    ref.assert_rows(q, s, g * torch.sigmoid(g) * u, 2.0 ** -20)


# ------------------------------------------------------------------------------------------ norm

# sum of squares: at most 64 additions in a thread, 6 + 16 across them, each 2^-24 of a positive total; the root halves that;
# mean, eps, root, reciprocal and two products round once each: 43 + 6 roundings of 2^-24 < 2^-18
NORM_DELTA = 2.0 ** -18


def norm_reference(x, w, eps, residual=None):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    hd = h.double()
    return h, hd / torch.sqrt(hd.square().mean(-1, keepdim=True) + eps) * w.double()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (4, 4096), (3, 500), (2, 513), (5, 2049), (7, 5000), (2, 8200), (2, 16385), (1, 65536), (600, 256)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_rmsnorm(dtype, m, k, with_residual):
    x = noise(m, k, seed=k).to(dtype)
    w = (1 + 0.3 * noise(k, seed=2)).to(dtype)
    r = noise(m, k, seed=7, scale=2.0).to(dtype) if with_residual else None
    h = torch.full((m, k), 9.0, dtype=dtype, device=DEV) if with_residual else None
    q, s = rows(m, k)
    _ops.rmsnorm_fp8(x, w, 1e-5, q, s, residual=r, sum_out=h)
    hr, y = norm_reference(x, w, 1e-5, r)
    ref.assert_rows(q, s, y, NORM_DELTA)
    if with_residual:
        assert torch.equal(h, hr)


@pytest.mark.parametrize("where", ["x", "residual"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rmsnorm_sum_over_its_inputs(where, dtype):
    m, k = 6, 1500
    x, r, w = noise(m, k, seed=1).to(dtype), noise(m, k, seed=2).to(dtype), noise(k, seed=3).to(dtype)
    hr, y = norm_reference(x, w, 1e-6, r)
    q, s = rows(m, k)
    target = x if where == "x" else r
    _ops.rmsnorm_fp8(x, w, 1e-6, q, s, residual=r, sum_out=target)
    assert torch.equal(target, hr)
    ref.assert_rows(q, s, y, NORM_DELTA)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rmsnorm_unaligned_rows_and_a_copy_without_residual(dtype):
    m, k, stride = 5, 333, 335
    wide = noise(m * stride + 4, seed=4).to(dtype)
    x = wide[1:1 + m * stride].view(m, stride)[:, :k]
    w = noise(k + 1, seed=5).to(dtype)[1:]
    out = torch.full((m, stride), 9.0, dtype=dtype, device=DEV)
    q, s = rows(m, k)
    _ops.rmsnorm_fp8(x, w, 1e-5, q, s, sum_out=out[:, :k])
    assert torch.equal(out[:, :k], x) and (out[:, k:] == 9.0).all()
    ref.assert_rows(q, s, norm_reference(x, w, 1e-5)[1], NORM_DELTA)


def test_rmsnorm_rows_keep_their_non_finite_values_to_themselves():
    x = noise(4, 512, seed=6).bfloat16()
    x[1, 3], x[2, 400] = float("nan"), float("inf")
    x[3] = 0
    w = torch.ones(512, dtype=torch.bfloat16, device=DEV)
    q, s = rows(4, 512)
    _ops.rmsnorm_fp8(x, w, 1e-5, q, s)
    v = _ops.fp8_values(q, s, 512)
    assert v[1].isnan().all() and v[2, 384:].isnan().all() and (v[3] == 0).all()
    ref.assert_rows(q[:1], s[:1], norm_reference(x[:1], w, 1e-5)[1], NORM_DELTA)


# ------------------------------------------------------------------------------------------ the product

def make_linear(m, n, k, seed=0, glu=False, outlier=True):
    x = noise(m, k, seed=seed) * (torch.exp(noise(1, k, seed=seed + 1)) if outlier else 1.0)
    q, s = ref.quantise(x)
    if glu:
        parts = [ref.quantise_weight(noise(n // 2, k, seed=seed + 2 + i, scale=k ** -0.5)) for i in range(2)]
        wq = torch.cat([p[0].view(torch.uint8) for p in parts]).view(torch.float8_e4m3fn)
        ws = torch.cat([p[1] for p in parts])
    else:
        wq, ws = ref.quantise_weight(noise(n, k, seed=seed + 2, scale=k ** -0.5))
    return q, s, wq, ws


def eight_bit_sums(m, out_dtype):
    """16-bit results of more than 16 rows run on the 8-bit matrix instructions."""
    return m > 16 and out_dtype != torch.float32


LINEAR_SIZES = [(1, 1, 1), (1, 16, 128), (2, 17, 129), (4, 6144, 4096), (4, 4096, 14336), (15, 100, 300), (16, 256, 1111), (17, 130, 257),
                (31, 48, 1000), (33, 1000, 127), (64, 512, 4096), (65, 257, 640), (100, 1000, 1111), (128, 512, 1024), (200, 640, 384),
                (256, 256, 2048), (300, 129, 2000), (513, 384, 512), (1000, 1030, 900), (2048, 1024, 512),
                (20, 130, 4200), (40, 300, 14336), (90, 1000, 2200), (130, 2000, 4000), (257, 700, 1100), (700, 3000, 640),
                (3000, 5000, 300),
                # rows in registers over several groups of rows and rounds of tiles, on both sides of every length they are cut at
                (24, 6200, 1000), (48, 9000, 1024), (130, 4200, 1025), (192, 6144, 2048), (200, 5000, 2049), (500, 1700, 4096), (17, 8200, 4000),
                # K cut, and whole tiles of both sizes
                (17, 64, 4097), (300, 515, 8192), (1000, 300, 5000), (900, 2000, 4200), (28, 17000, 4200), (50, 17000, 4200), (1030, 1600, 700), (4200, 3300, 257)]


@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", LINEAR_SIZES)
def test_linear(m, n, k, out_dtype):
    q, s, wq, ws = make_linear(m, n, k, seed=m + n + k)
    w = _ops.pack_weight_fp8(wq, scales=ws)
    out = torch.full((m, n), 77.0, dtype=out_dtype, device=DEV)
    assert _ops.linear_fp8(q, s, w, out) is out
    ref.assert_linear(out, *ref.linear(q, s, wq, ws, k, eight_bit_sums=eight_bit_sums(m, out_dtype)))
    again = torch.empty_like(out)
    assert torch.equal(_ops.linear_fp8(q, s, w, again), out), "the same bits on every run"


@pytest.mark.parametrize("m,n,k", [(1, 33, 100), (4, 4096, 1024), (20, 200, 300), (48, 300, 1111), (130, 384, 640), (512, 512, 256), (700, 1000, 384),
                                   (50, 260, 4300), (300, 515, 1200), (2100, 6000, 200), (300, 515, 4900), (700, 2700, 300)])
@pytest.mark.parametrize("out_dtype", DTYPES)
def test_linear_residual(m, n, k, out_dtype):
    q, s, wq, ws = make_linear(m, n, k, seed=1)
    w = _ops.pack_weight_fp8(wq, scales=ws)
    r = noise(m, n, seed=8).to(out_dtype)
    want = ref.linear(q, s, wq, ws, k, residual=r, eight_bit_sums=eight_bit_sums(m, out_dtype))
    out = torch.empty_like(r)
    _ops.linear_fp8(q, s, w, out, residual=r)
    ref.assert_linear(out, *want)
    _ops.linear_fp8(q, s, w, r, residual=r)
    assert torch.equal(r, out), "the residual's own memory as the output"


@pytest.mark.parametrize("m,n,k", [(1, 2, 128), (4, 28672, 512), (16, 2 * 37, 300), (17, 2 * 130, 257), (40, 2 * 200, 1000), (129, 2 * 256, 384),
                                   (520, 2 * 384, 256), (600, 2 * 333, 500), (60, 2 * 1001, 4096), (150, 2 * 515, 1500), (2100, 2 * 3001, 200),
                                   (150, 2 * 515, 4900), (700, 2 * 1351, 300), (200, 2 * 3100, 2500)])
@pytest.mark.parametrize("out_dtype", DTYPES)
def test_linear_swiglu(m, n, k, out_dtype):
    q, s, wq, ws = make_linear(m, n, k, seed=3, glu=True)
    w = _ops.pack_weight_fp8(wq, scales=ws, glu=True)
    out = torch.full((m, n // 2), 77.0, dtype=out_dtype, device=DEV)
    _ops.linear_fp8(q, s, w, out, swiglu=True)
    ref.assert_linear(out, *ref.linear(q, s, wq, ws, k, glu=True, eight_bit_sums=eight_bit_sums(m, out_dtype)))


@pytest.mark.parametrize("m,n,k", [(3, 200, 300), (40, 200, 300), (300, 200, 300), (700, 2600, 300), (2100, 6000, 300), (300, 200, 4300), (5, 200, 4300)])
def test_linear_strides(m, n, k):
    """Rows of x, scales, residual and out that are parts of wider ones; what lies beside them stays."""
    kb = ref.blocks(k)
    q, s, wq, ws = make_linear(m, n, k, seed=4)
    w = _ops.pack_weight_fp8(wq, scales=ws)
    wide_q = torch.full((m, 128 * (kb + 1)), 0x7f, dtype=torch.uint8, device=DEV)          # NaN beside the rows
    wide_q[:, 64:64 + 128 * kb] = q.view(torch.uint8)
    wide_s = torch.full((m, kb + 4), float("nan"), device=DEV)
    wide_s[:, 2:2 + kb] = s
    wide_r = torch.full((m, n + 3), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide_r[:, 1:n + 1] = noise(m, n, seed=5).bfloat16()
    wide_o = torch.full((m + 1, n + 5), 9.0, dtype=torch.bfloat16, device=DEV)
    _ops.linear_fp8(wide_q[:, 64:64 + 128 * kb].view(torch.float8_e4m3fn), wide_s[:, 2:2 + kb], w, wide_o[:m, 3:n + 3], residual=wide_r[:, 1:n + 1])
    ref.assert_linear(wide_o[:m, 3:n + 3], *ref.linear(q, s, wq, ws, k, residual=wide_r[:, 1:n + 1], eight_bit_sums=eight_bit_sums(m, torch.bfloat16)))
    assert (wide_o[:, :3] == 9.0).all() and (wide_o[:, n + 3:] == 9.0).all() and (wide_o[m] == 9.0).all()


@pytest.mark.parametrize("m,n,k", [(3, 100, 300), (40, 100, 300), (40, 300, 4300), (150, 300, 4300)])
def test_linear_rows_far_apart(m, n, k):
    """Rows of x four MiB and more apart: positions within a group of rows pass 32 bits."""
    q, s, wq, ws = make_linear(m, n, k, seed=14)
    w = _ops.pack_weight_fp8(wq, scales=ws)
    far = torch.empty(m, (1 << 24) // (2 if m > 100 else 1), dtype=torch.uint8, device=DEV)[:, 32:32 + q.shape[1]]
    far.copy_(q.view(torch.uint8))
    out = _ops.linear_fp8(far.view(torch.float8_e4m3fn), s, w, torch.empty(m, n, dtype=torch.bfloat16, device=DEV))
    ref.assert_linear(out, *ref.linear(q, s, wq, ws, k, eight_bit_sums=eight_bit_sums(m, torch.bfloat16)))


@pytest.mark.parametrize("m,n,k", [(5, 384, 512), (30, 384, 512), (64, 384, 512), (300, 384, 512), (600, 384, 512), (1100, 1500, 512), (64, 384, 4224),
                                   (6, 384, 4224), (100, 384, 4096)])
def test_linear_rows_keep_their_nan_to_themselves(m, n, k):
    q, s, wq, ws = make_linear(m, n, k, seed=6)
    w = _ops.pack_weight_fp8(wq, scales=ws)
    clean = _ops.linear_fp8(q, s, w, torch.empty(m, n, device=DEV))
    q.view(torch.uint8)[m // 2, 77] = 0x7f
    s[m // 2, 0] = float("inf")
    out = _ops.linear_fp8(q, s, w, torch.empty(m, n, device=DEV))
    assert out[m // 2].isnan().all()
    others = torch.arange(m, device=DEV) != m // 2
    assert torch.equal(out[others], clean[others])


@pytest.mark.parametrize("n,k,glu", [(1, 1, False), (16, 128, False), (200, 300, False), (129, 1111, False), (2 * 130, 257, True), (2 * 8, 128, True),
                                     (2 * 5, 100, True)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_weights_quantised_while_packing(n, k, glu, dtype):
    """Multiplying with the rows of the identity gives the packed matrix back: each weight within half a step of its block's
    scale, as `assert_rows` has it, and the same as packing the numbers that 64 bits give where those are no near ties."""
    wide = noise(n, k + 3, seed=n + k).to(dtype)
    w = wide[:, 1:k + 1]
    pack = _ops.pack_weight_fp8(w, glu=glu)
    eye = torch.eye(k, dtype=torch.float32, device=DEV)
    q, s = rows(k, k)
    _ops.quantize_rows_fp8(eye, q, s)           # 448 * (1 / 448): fp32 rounds the product, below
    if glu:                                     # the sums themselves: pack each half as a plain matrix of its own
        halves = [_ops.pack_weight_fp8(w[:n // 2]), _ops.pack_weight_fp8(w[n // 2:])]
        got = torch.cat([_ops.linear_fp8(q, s, h, torch.empty(k, n // 2, device=DEV)) for h in halves], dim=1).t().double()
        f = n // 2
        act = _ops.linear_fp8(q, s, pack, torch.empty(k, f, device=DEV), swiglu=True).t().double()
        want = got[:f] * torch.sigmoid(got[:f]) * got[f:]
        assert ((act - want).abs() <= want.abs() * 2.0 ** -19).all()
        parts = [w[:f].double(), w[f:].double()]
    else:
        got = _ops.linear_fp8(q, s, pack, torch.empty(k, n, device=DEV)).t().double()
        parts = [w.double()]
    at = 0
    for part in parts:
        _, ws = ref.quantise_weight(part)
        sc = ref.weight_spread(ws, *part.shape)
        v = part / sc
        mine = got[at:at + part.shape[0]] / sc
        assert ((mine - v).abs() <= ref.half_step(v) + v.abs() * 2.0 ** -20).all()
        at += part.shape[0]


@pytest.mark.parametrize("m,n,k", [(200, 512, 4096), (640, 1024, 1024)])
@pytest.mark.parametrize("out_dtype", DTYPES)
def test_linear_error_as_a_whole(m, n, k, out_dtype):
    """2-norm of the error against 64 bits on normally distributed numbers.  Rounding to the output type is off by at most eps / 2
    of each value; the 8-bit matrix instructions add 1.5e-5 on such numbers (measured on one block of 128), taken twice here; fp32
    results have only their own sums."""
    q, s, wq, ws = make_linear(m, n, k, seed=12, outlier=False)
    out = _ops.linear_fp8(q, s, _ops.pack_weight_fp8(wq, scales=ws), torch.empty(m, n, dtype=out_dtype, device=DEV))
    y, _ = ref.linear(q, s, wq, ws, k)
    most = 1e-6 if out_dtype == torch.float32 else torch.finfo(out_dtype).eps / 2 + 3e-5
    assert float((out.double() - y).norm() / y.norm()) <= most


def test_packing_takes_numbers_and_scales_over_as_they_are():
    n, k = 200, 300
    q, s, wq, ws = make_linear(4, n, k, seed=11)
    ws = ws * torch.linspace(0.5, 3.0, ws.numel(), device=DEV).view_as(ws)      # any scales, not this library's own
    wide = torch.zeros(n, k + 7, dtype=torch.uint8, device=DEV)
    wide[:, 3:k + 3] = wq.view(torch.uint8)
    w = _ops.pack_weight_fp8(wide[:, 3:k + 3].view(torch.float8_e4m3fn), scales=ws)
    out = _ops.linear_fp8(q, s, w, torch.empty(4, n, device=DEV))
    ref.assert_linear(out, *ref.linear(q, s, wq, ws, k))


@pytest.mark.parametrize("m,n,k", [(40, 300, 4300), (300, 512, 8192)])
def test_linear_with_a_workspace_of_the_callers(m, n, k):
    """The same bits from the caller's scratch as from the allocator's; what lies behind the bytes asked for stays; too little is refused."""
    q, s, wq, ws = make_linear(m, n, k, seed=21)
    w = _ops.pack_weight_fp8(wq, scales=ws)
    need = _ops.linear_fp8_workspace_bytes(m, w)
    assert need > 0
    mem = torch.full((need + 256,), 0x5a, dtype=torch.uint8, device=DEV)
    a = _ops.linear_fp8(q, s, w, torch.empty(m, n, dtype=torch.bfloat16, device=DEV))
    b = _ops.linear_fp8(q, s, w, torch.empty(m, n, dtype=torch.bfloat16, device=DEV), ws=mem[:need])
    assert torch.equal(a, b) and (mem[need:] == 0x5a).all()
    ref.assert_linear(a, *ref.linear(q, s, wq, ws, k, eight_bit_sums=True))
    with pytest.raises(_ops.HashAttnError):
        _ops.linear_fp8(q, s, w, b, ws=mem[:need - 16])


def test_no_rows_is_no_work():
    x = torch.empty(0, 300, dtype=torch.bfloat16, device=DEV)
    q, s = _ops.fp8_rows(0, 300, DEV)
    _ops.quantize_rows_fp8(x, q, s)
    _ops.rmsnorm_fp8(x, torch.ones(300, dtype=torch.bfloat16, device=DEV), 1e-5, q, s, residual=x, sum_out=torch.empty_like(x))
    _ops.swiglu_fp8(torch.empty(0, 600, dtype=torch.bfloat16, device=DEV), q, s)
    w = _ops.pack_weight_fp8(noise(40, 300).bfloat16())
    assert _ops.linear_fp8(q, s, w, torch.empty(0, 40, device=DEV)).shape == (0, 40)


# ------------------------------------------------------------------------------------------ together

def mlp(x, r, norm_w, gate_up, down, buffers):
    """A layer's feed-forward half: the addition and its norm, gate/up, SwiGLU in 8 bits, the down projection with its residual."""
    m, hidden = x.shape
    f = gate_up.N // 2
    h, q1, s1, gu, q2, s2, out = buffers
    _ops.rmsnorm_fp8(x, norm_w, 1e-5, q1, s1, residual=r, sum_out=h)
    _ops.linear_fp8(q1, s1, gate_up, gu)
    _ops.swiglu_fp8(gu, q2, s2)
    return _ops.linear_fp8(q2, s2, down, out, residual=h)


def mlp_buffers(m, hidden, f):
    return (torch.empty(m, hidden, dtype=torch.bfloat16, device=DEV), *_ops.fp8_rows(m, hidden, DEV),
            torch.empty(m, 2 * f, dtype=torch.bfloat16, device=DEV), *_ops.fp8_rows(m, f, DEV),
            torch.empty(m, hidden, dtype=torch.bfloat16, device=DEV))


@pytest.mark.parametrize("m", [1, 4, 24, 100, 600])
def test_feed_forward_half_of_a_layer(m):
    """Every operator on the others' outputs: each step against the plain form on the very numbers the step before it left."""
    hidden, f = 512, 1100
    x, r = noise(m, hidden, seed=1).bfloat16(), noise(m, hidden, seed=2).bfloat16()
    nw = (1 + 0.1 * noise(hidden, seed=3)).bfloat16()
    wgu, wd = noise(2 * f, hidden, seed=4, scale=hidden ** -0.5), noise(hidden, f, seed=5, scale=f ** -0.5)
    (gq, gs), (dq, ds) = ref.quantise_weight(wgu), ref.quantise_weight(wd)
    bufs = mlp_buffers(m, hidden, f)
    out = mlp(x, r, nw, _ops.pack_weight_fp8(gq, scales=gs), _ops.pack_weight_fp8(dq, scales=ds), bufs)
    h, q1, s1, gu, q2, s2, _ = bufs
    hr, y = norm_reference(x, nw, 1e-5, r)
    assert torch.equal(h, hr)
    ref.assert_rows(q1, s1, y, NORM_DELTA)
    ref.assert_linear(gu, *ref.linear(q1, s1, gq, gs, hidden, eight_bit_sums=eight_bit_sums(m, gu.dtype)))
    g, u = gu[:, :f].double(), gu[:, f:].double()
    ref.assert_rows(q2, s2, g * torch.sigmoid(g) * u, 2.0 ** -20)
    ref.assert_linear(out, *ref.linear(q2, s2, dq, ds, f, residual=h, eight_bit_sums=eight_bit_sums(m, out.dtype)))


@pytest.mark.parametrize("m", [4, 200])
def test_in_a_graph_and_on_another_stream(m):
    """Captured once, replayed on new inputs with eager work in between: the eager results every time, also from a second graph
    over the same weights, and on a stream that is not the current one's default."""
    hidden, f = 512, 640
    nw = torch.ones(hidden, dtype=torch.bfloat16, device=DEV)
    gu_w = _ops.pack_weight_fp8(noise(2 * f, hidden, seed=4, scale=hidden ** -0.5).bfloat16())
    d_w = _ops.pack_weight_fp8(noise(hidden, f, seed=5, scale=f ** -0.5).bfloat16())
    x, r = torch.zeros(m, hidden, dtype=torch.bfloat16, device=DEV), torch.zeros(m, hidden, dtype=torch.bfloat16, device=DEV)
    bufs = [mlp_buffers(m, hidden, f) for _ in range(3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mlp(x, r, nw, gu_w, d_w, bufs[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            mlp(x, r, nw, gu_w, d_w, bufs[i])
        graphs.append(g)
    for step in range(4):
        x.copy_(noise(m, hidden, seed=20 + step).bfloat16())
        r.copy_(noise(m, hidden, seed=40 + step).bfloat16())
        graphs[0].replay()
        graphs[1].replay()
        want = mlp(x, r, nw, gu_w, d_w, bufs[2])
        torch.cuda.synchronize()
        assert torch.equal(bufs[0][-1], want) and torch.equal(bufs[1][-1], want)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            bufs[2][-1].zero_()
            on_side = mlp(x, r, nw, gu_w, d_w, bufs[2])
        side.synchronize()
        assert torch.equal(on_side, bufs[0][-1])


@pytest.mark.parametrize("m,n,k,glu", [(300, 2000, 2200, False), (2100, 6200, 1000, False), (2100, 6200, 4096, True), (700, 300, 4000, True),
                                       (4096, 4096, 128, False), (2048, 8192, 300, False), (700, 300, 5000, True), (1000, 3000, 2200, False)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_counted_waits_and_full_waits_give_the_same_bits(m, n, k, glu, out_dtype):
    """The staged kernels wait for counted requests; the library's twin waits for all of them."""
    q, s, wq, ws = make_linear(m, n, k, seed=31, glu=glu)
    w = _ops.pack_weight_fp8(wq, scales=ws, glu=glu)
    main, twin = _ops.load_library(), _ops.load_wait_all_variant()
    outs = []
    for lib in (main, twin, main):
        _ops._lib = lib
        try:
            outs.append(_ops.linear_fp8(q, s, w, torch.empty(m, n // 2 if glu else n, dtype=out_dtype, device=DEV), swiglu=glu))
            torch.cuda.synchronize()
        finally:
            _ops._lib = main
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_refusals_of_the_bindings():
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device=DEV)
    q, s = _ops.fp8_rows(4, 256, DEV)
    w = _ops.pack_weight_fp8(torch.ones(32, 256, device=DEV))
    glu = _ops.pack_weight_fp8(torch.ones(32, 256, device=DEV), glu=True)
    out = torch.empty(4, 32, device=DEV)
    bad = [
        lambda: _ops.quantize_rows_fp8(x.cpu(), q, s),
        lambda: _ops.quantize_rows_fp8(x.double(), q, s),
        lambda: _ops.quantize_rows_fp8(x.t(), q, s),
        lambda: _ops.quantize_rows_fp8(x, q[:3], s),
        lambda: _ops.quantize_rows_fp8(x, q, s[:, :1]),
        lambda: _ops.quantize_rows_fp8(x, q.view(torch.uint8), s),
        lambda: _ops.swiglu_fp8(x, q, s),                                       # rows of 128 do not fit rows of 256
        lambda: _ops.swiglu_fp8(x[:, :255], q, s),
        lambda: _ops.rmsnorm_fp8(x, torch.ones(256, device=DEV), 1e-5, q, s),   # weight of another type
        lambda: _ops.rmsnorm_fp8(x, x[0], 1e-5, q, s, residual=x[:2]),
        lambda: _ops.rmsnorm_fp8(x, x[0], 1e-5, q, s, sum_out=x.float()),
        lambda: _ops.pack_weight_fp8(torch.ones(33, 256, device=DEV), glu=True),
        lambda: _ops.pack_weight_fp8(torch.ones(32, 256, device=DEV), scales=torch.ones(1, 2, device=DEV)),
        lambda: _ops.pack_weight_fp8(torch.ones(32, 256, device=DEV).to(torch.float8_e4m3fn)),
        lambda: _ops.pack_weight_fp8(torch.ones(32, 256, device=DEV).to(torch.float8_e4m3fn), scales=torch.ones(2, 1, device=DEV)),
        lambda: _ops.pack_weight_fp8(torch.ones(32, 256, dtype=torch.int32, device=DEV)),
        lambda: _ops.linear_fp8(q, s, w, out, swiglu=True),
        lambda: _ops.linear_fp8(q, s, glu, out),
        lambda: _ops.linear_fp8(q, s, glu, out[:, :16], swiglu=True, residual=out),
        lambda: _ops.linear_fp8(q, s, w, out[:, :16]),
        lambda: _ops.linear_fp8(q, s, w, out.double()),
        lambda: _ops.linear_fp8(q, s, w, out, residual=out.bfloat16()),
        lambda: _ops.linear_fp8(q[:, :128], s[:, :1], w, out),
        # weights that are not as they were packed
        lambda: _ops.linear_fp8(q, s, w._replace(scales=w.scales.bfloat16()), out),
        lambda: _ops.linear_fp8(q, s, w._replace(scales=w.scales[1:]), out),
        lambda: _ops.linear_fp8(q, s, w._replace(tiles=w.tiles[:2048]), out),
        lambda: _ops.linear_fp8(q, s, w._replace(tiles=w.tiles.float()), out),
        lambda: _ops.linear_fp8(q, s, w._replace(N=64), torch.empty(4, 64, device=DEV)),
        lambda: _ops.linear_fp8(q, s, w._replace(tiles=w.tiles.expand(2, -1)[:, ::2]), out),
        lambda: _ops.linear_fp8(q, s, w, out, ws=torch.empty(64, dtype=torch.uint8, device=DEV)[::2]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(_ops.HashAttnError):     # the library's own limit
        k = 65537
        _ops.rmsnorm_fp8(torch.zeros(1, k, device=DEV), torch.ones(k, device=DEV), 1e-5, *_ops.fp8_rows(1, k, DEV))
    with pytest.raises(_ops.HashAttnError):     # rows of 8-bit numbers off their 16-byte boundary
        wide = torch.zeros(4, 300, dtype=torch.uint8, device=DEV)
        _ops.quantize_rows_fp8(x, wide[:, 8:264].view(torch.float8_e4m3fn), s)
