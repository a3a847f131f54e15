"""Plain 64-bit forms of the 8-bit operators, for the tests."""
import torch

BLOCK = 128
FLOOR = 2.0 ** -96


def blocks(k):
    return -(-k // BLOCK)


def half_step(v):
    """Half the distance of neighbouring e4m3 numbers around v (fp64): 3 mantissa bits, subnormal below 2^-6."""
    e = (torch.frexp(v)[1].long() - 1).clamp(min=-6) - 4
    return ((e + 1023) << 52).view(torch.float64)          # 2^e exactly (torch.ldexp goes through pow)


def round_e4m3(v):
    """fp64 -> nearest e4m3, ties to even."""
    step = 2 * half_step(v)
    return torch.round(v / step) * step


def block_scales(y):
    """y fp64 [m, k] -> scales fp64 [m, blocks]."""
    m, k = y.shape
    t = torch.nn.functional.pad(y, (0, blocks(k) * BLOCK - k)).view(m, -1, BLOCK).abs().amax(-1)
    return torch.where(t > 0, t.clamp(min=FLOOR) / 448, torch.ones_like(t))


def spread(scales, k):
    return scales.double().repeat_interleave(BLOCK, dim=1)[:, :k]


def assert_rows(q, scales, y, delta):
    """q, scales (as the kernels leave them) against y fp64 [m, k], which the kernel computed to a relative `delta`.  Scale: one
    more rounding (2^-24).  Number: v = y / scale carries delta twice (y's own, the scale's) and three roundings of 2^-24; the
    nearest e4m3 of it is then within half a step of v plus that."""
    m, k = y.shape
    assert q.dtype == torch.float8_e4m3fn and q.shape == (m, blocks(k) * BLOCK) and scales.shape == (m, blocks(k))
    exact = block_scales(y)
    assert ((scales.double() - exact).abs() <= exact * (delta + 2.0 ** -23)).all()
    assert (q[:, k:].view(torch.uint8) == 0).all(), "zero beyond the row"
    v = y / spread(exact, k)
    err = (q[:, :k].double() - v).abs()
    bound = half_step(v) + v.abs() * (2 * delta + 2.0 ** -21)
    assert (err <= bound).all(), float((err / bound).max())


def quantise(y):
    """y fp64 [m, k] -> (q float8_e4m3fn [m, padded], scales fp32), rounded from 64 bits."""
    m, k = y.shape
    s = block_scales(y).float()
    q = round_e4m3(y / spread(s, k)).clamp(-448, 448)
    return torch.nn.functional.pad(q, (0, blocks(k) * BLOCK - k)).float().to(torch.float8_e4m3fn), s


def quantise_weight(w):
    """w fp64 [n, k] -> (q float8_e4m3fn [n, k], scales fp32 [row blocks, column blocks])."""
    n, k = w.shape
    t = torch.nn.functional.pad(w, (0, blocks(k) * BLOCK - k, 0, blocks(n) * BLOCK - n)).view(blocks(n), BLOCK, blocks(k), BLOCK)
    top = t.abs().amax(dim=(1, 3))
    s = torch.where(top > 0, top.clamp(min=FLOOR) / 448, torch.ones_like(top)).float()
    return round_e4m3(w / weight_spread(s, n, k)).clamp(-448, 448).float().to(torch.float8_e4m3fn), s


def weight_spread(s, n, k):
    return s.double().repeat_interleave(BLOCK, dim=0)[:n].repeat_interleave(BLOCK, dim=1)[:, :k]


def linear(q, s, wq, ws, k, residual=None, glu=False, eight_bit_sums=False):
    """(y, b): the product in fp64 and what its fp32 form may be off by (fp64, same shape), before any rounding of the result.
    wq [n, k]; ws: per matrix for glu (gate's rows of blocks, then up's).  Products of e4m3 numbers are exact (8 bits of mantissa).
    Every output is a sum of k products, scaled per block: at most 128 additions inside a block, one multiply-add per block, two
    roundings of the scale, and up to 64 partial sums joined.  Each addition is taken at 2^-23 of the sum of magnitudes (the
    matrix instruction may truncate where an FMA rounds).
    eight_bit_sums: the 8-bit matrix instructions add eight neighbouring products at a time on a grid whose step is 2^-13 of
    the largest product's power of two (measured: 2^3 beside 2^16 is kept, 2^2 is dropped).  Each of the eight loses less than
    that step, which is at most 2^-13 of the largest magnitude: together less than 8 * 2^-13 = 2^-10 of the eight magnitudes' sum,
    and over all groups 2^-10 of the sum of all magnitudes."""
    n = wq.shape[0]
    x = q[:, :k].double() * spread(s, k)
    if glu:
        f = n // 2
        w = torch.cat([wq[:f].double() * weight_spread(ws[:blocks(f)], f, k), wq[f:].double() * weight_spread(ws[blocks(f):], f, k)])
    else:
        w = wq.double() * weight_spread(ws, n, k)
    y = x @ w.t()
    off = (x.abs() @ w.abs().t()) * ((min(k, 128) + blocks(k) + 66) * 2.0 ** -23 + (2.0 ** -10 if eight_bit_sums else 0.0))
    if glu:
        # the exponential to 2 ulp of fp32, sum, quotient and product rounded; |d silu| <= 1.1 |d gate|
        gate, up, dg, du = y[:, :f], y[:, f:], off[:, :f], off[:, f:]
        silu = gate * torch.sigmoid(gate)
        y = silu * up
        off = 1.1 * dg * (up.abs() + du) + silu.abs() * du + y.abs() * 2.0 ** -20
    elif residual is not None:
        y = y + residual.double()
        off = off + y.abs() * 2.0 ** -24
    return y, off


def assert_linear(out, y, off):
    """One rounding to out's type on top: half a step relative, and the smallest number of fp16 where it is subnormal."""
    fi = torch.finfo(out.dtype)
    bound = off + (y.abs() + off) * fi.eps / 2 + (2.0 ** -25 if out.dtype == torch.float16 else 0.0)
    err = (out.double() - y).abs()
    assert (err <= bound).all(), float((err / bound).max())
