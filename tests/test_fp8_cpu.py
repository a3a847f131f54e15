"""Host side of the 8-bit entry points, without a GPU: sizes, and refusals before any device work (host buffers stand in for device
pointers; nothing is launched).  The 64-bit helper of the GPU tests against torch's own e4m3."""
import ctypes as C
import os
import re
import subprocess

import pytest
import torch

from hashattention import _ops
from tests import fp8_util as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "hashattention-1.0_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
NULL, SHAPE, DTYPE, ALIGN, WS, NODEV = -1, -2, -3, -4, -5, -6
BF16, F32, E4M3 = _ops.HA_BF16, _ops.HA_F32, _ops.HA_FP8_E4M3


@pytest.fixture(scope="module")
def lib():
    return _ops.load_library()


@pytest.fixture(scope="module")
def mem():
    buf = (C.c_char * (1 << 16))()
    mem.keep = buf
    return (C.addressof(buf) + 255) // 256 * 256


def test_sizes(lib):
    assert [lib.ha_fp8_row_bytes(k) for k in (-1, 0, 1, 128, 129, 4096)] == [0, 0, 128, 128, 256, 4096]
    assert lib.ha_weight_fp8_bytes(16, 128, 0) == 2048 and lib.ha_weight_fp8_scales(16, 128, 0) == 2
    assert lib.ha_weight_fp8_bytes(17, 129, 0) == 2 * 2 * 2048 and lib.ha_weight_fp8_scales(17, 129, 0) == 8
    assert lib.ha_weight_fp8_bytes(18, 128, 1) == 2 * 2048                  # 9 columns: two tiles of 8 gate and 8 up rows
    assert lib.ha_weight_fp8_bytes(17, 128, 1) == 0 and lib.ha_weight_fp8_bytes(0, 128, 0) == 0 and lib.ha_weight_fp8_bytes(16, 0, 0) == 0
    assert lib.ha_weight_fp8_bytes(2 ** 31 - 1, 2 ** 31 - 1, 0) == 2 ** 62   # no overflow
    assert _ops.fp8_blocks(1) == 1 and _ops.fp8_blocks(128) == 1 and _ops.fp8_blocks(129) == 2


def test_row_operators_refuse(lib, mem):
    ok = dict(x=mem, xs=256, dt=BF16, M=4, K=256, q=mem, qs=256, s=mem, ss=2)

    def rows(**kw):
        a = {**ok, **kw}
        return lib.ha_quantize_rows_fp8(a["x"], a["xs"], a["dt"], a["M"], a["K"], a["q"], a["qs"], a["s"], a["ss"], None)

    def norm(w=mem, r=None, rs=0, eps=1e-5, h=None, hs=0, **kw):
        a = {**ok, **kw}
        return lib.ha_rmsnorm_fp8(a["x"], a["xs"], r, rs, w, a["dt"], a["M"], a["K"], eps, h, hs, a["q"], a["qs"], a["s"], a["ss"], None)

    def glu(**kw):
        a = {**ok, "xs": 512, **kw}
        return lib.ha_swiglu_fp8(a["x"], a["xs"], a["dt"], a["M"], a["K"], a["q"], a["qs"], a["s"], a["ss"], None)

    for f in (rows, norm, glu):
        assert f(x=None) == NULL and f(q=None) == NULL and f(s=None) == NULL
        assert f(dt=E4M3) == DTYPE and f(dt=-1) == DTYPE
        assert f(M=-1) == SHAPE and f(K=0) == SHAPE and f(xs=255) == SHAPE and f(qs=255) == SHAPE and f(ss=1) == SHAPE
        assert f(K=2 ** 31 - 1, xs=2 ** 33, qs=2 ** 31, ss=2 ** 24, M=2 ** 10) == SHAPE            # more blocks than a launch takes
        assert f(q=mem + 8) == ALIGN and f(qs=264) == ALIGN and f(s=mem + 2) == ALIGN and f(x=mem + 1) == ALIGN
        # a launch holds fewer than 2^32 threads: 2^28 - 16 blocks of 128, 2^26 - 1 narrow rows to normalise
        assert f(K=128, qs=128, ss=1, M=2 ** 28 + 1) == SHAPE and f(K=2 ** 31 - 1, xs=2 ** 33, qs=2 ** 31, ss=2 ** 24, M=1) == SHAPE
    if lib.ha_device_count() == 0:
        assert rows(K=128, qs=128, ss=1, M=2 ** 28 - 16) == NODEV and glu(K=128, qs=128, ss=1, M=2 ** 28 - 16) == NODEV
        assert norm(K=128, qs=128, ss=1, M=2 ** 26 - 1) == NODEV
        assert rows(K=2 ** 31 - 129, xs=2 ** 33, qs=2 ** 31, ss=2 ** 24, M=1) == NODEV
    assert norm(K=128, qs=128, ss=1, M=2 ** 26) == SHAPE and norm(K=4096, xs=4096, qs=4096, ss=32, M=2 ** 24) == SHAPE
    assert norm(w=None) == NULL and norm(r=mem, rs=255) == SHAPE and norm(h=mem, hs=255) == SHAPE and norm(eps=-1.0) == SHAPE
    assert norm(K=65537, xs=65537, qs=65664, ss=513) == SHAPE
    assert norm(w=mem + 1) == ALIGN and norm(r=mem + 1, rs=256) == ALIGN and norm(h=mem + 1, hs=256) == ALIGN
    if lib.ha_device_count() == 0:
        assert rows() == NODEV and norm() == NODEV and glu() == NODEV


def test_pack_and_linear_refuse(lib, mem):
    def pack(w=mem, sn=256, dt=BF16, ws=None, wss=0, N=32, K=256, glu=0, t=mem, ts=mem):
        return lib.ha_pack_weight_fp8(w, sn, dt, ws, wss, N, K, glu, t, ts, None)

    assert pack(w=None) == NULL and pack(t=None) == NULL and pack(ts=None) == NULL
    assert pack(dt=7) == DTYPE
    assert pack(dt=E4M3) == NULL and pack(ws=mem, wss=2) == NULL        # e4m3 comes with scales, nothing else does
    assert pack(N=0) == SHAPE and pack(K=0) == SHAPE and pack(sn=255) == SHAPE and pack(N=33, glu=1) == SHAPE and pack(glu=2) == SHAPE
    assert pack(dt=E4M3, ws=mem, wss=1) == SHAPE and pack(N=2 ** 31 - 1) == SHAPE
    assert pack(w=mem + 1) == ALIGN and pack(t=mem + 8) == ALIGN and pack(ts=mem + 4) == ALIGN

    def lin(x=mem, xs=256, s=mem, ss=2, t=mem, ts=mem, r=None, rs=0, act=0, o=mem, os=32, dt=BF16, M=4, N=32, K=256, ws=None, wsb=0):
        return lib.ha_linear_fp8(x, xs, s, ss, t, ts, r, rs, act, o, os, dt, M, N, K, ws, wsb, None)

    for k in ("x", "s", "t", "ts", "o"):
        assert lin(**{k: None}) == NULL
    assert lin(dt=E4M3) == DTYPE
    assert lin(M=-1) == SHAPE and lin(N=0) == SHAPE and lin(K=0) == SHAPE and lin(act=2) == SHAPE and lin(act=1, N=33) == SHAPE
    assert lin(act=1, r=mem, rs=32) == SHAPE and lin(xs=255) == SHAPE and lin(ss=1) == SHAPE and lin(os=31) == SHAPE and lin(r=mem, rs=31) == SHAPE
    assert lin(x=mem + 8) == ALIGN and lin(xs=264) == ALIGN and lin(t=mem + 8) == ALIGN and lin(ts=mem + 4) == ALIGN
    assert lin(s=mem + 2) == ALIGN and lin(o=mem + 1) == ALIGN and lin(r=mem + 1, rs=32) == ALIGN
    assert lin(M=2 ** 31 - 1, N=2 ** 31 - 1, os=2 ** 31) == SHAPE
    # positions in a row and threads in a launch are 32-bit
    huge = dict(K=2 ** 31 - 1, xs=2 ** 31, ss=2 ** 24)
    assert lin(**huge) == SHAPE and pack(K=2 ** 31 - 1, sn=2 ** 31) == SHAPE
    assert lin(N=2 ** 27, os=2 ** 27) == SHAPE and lin(M=300, xs=2 ** 62, ss=2 ** 62, N=2 ** 31 - 1, os=2 ** 31) == SHAPE
    if lib.ha_device_count() == 0:
        assert lin(N=2 ** 25, os=2 ** 25) == NODEV and lin(M=2 ** 19, N=2 ** 18, os=2 ** 18) == NODEV
        assert lin(M=300, xs=2 ** 62, ss=2 ** 62) == NODEV                  # strides whose products leave 64 bits
    # sizes whose sums go through a workspace: missing, too small, misaligned
    big = dict(M=300, N=32, K=8192, xs=8192, ss=64)
    need = lib.ha_linear_fp8_workspace_bytes(300, 32, 8192, 0)
    assert need == 16 * 300 * 32 * 4
    assert lin(**big) == WS and lin(**big, ws=mem, wsb=need - 1) == WS and lin(**big, ws=mem + 8, wsb=need) == ALIGN
    for m, n, k, act in ((4, 32, 4096, 0), (16, 4096, 14336, 0), (64, 6144, 4096, 0), (4096, 28672, 4096, 0), (0, 32, 8192, 0), (300, 33, 8192, 1), (300, 32, 4096, 0)):
        assert lib.ha_linear_fp8_workspace_bytes(m, n, k, act) == 0
    assert lib.ha_linear_fp8_workspace_bytes(300, 33, 8192, 0) > 0
    assert _ops.LINEAR_FP8_UNSPLIT_ROWS == 16 and lib.ha_linear_fp8_workspace_bytes(17, 32, 14336, 0) > 0
    if lib.ha_device_count() == 0:
        assert pack() == NODEV and lin() == NODEV and lin(**big, ws=mem, wsb=need) == NODEV


def test_bindings_take_gpu_tensors_only():
    x = torch.zeros(2, 128)
    q, s = _ops.fp8_rows(2, 128, "cpu")
    with pytest.raises(ValueError):
        _ops.quantize_rows_fp8(x, q, s)
    with pytest.raises(ValueError):
        _ops.pack_weight_fp8(x)


def test_the_64_bit_helper_rounds_as_torch_does():
    """All midpoints, their neighbours and a sweep: the helper the GPU tests lean on against torch's cast."""
    grid = torch.arange(0, 0x7f, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (grid[1:] + grid[:-1]) / 2
    v = torch.cat([grid, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20), torch.rand(4096, dtype=torch.float64) * 448])
    v = torch.cat([v, -v])
    assert torch.equal(ref.round_e4m3(v), v.float().to(torch.float8_e4m3fn).double())
    y = torch.randn(3, 300, dtype=torch.float64)
    q, s = ref.quantise(y)
    assert torch.allclose(_ops.fp8_values(q, s, 300).double(), y, rtol=2.0 ** -4 * 1.01, atol=float(s.max()) * 2.0 ** -10)


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")
def test_what_the_counted_waits_rely_on():
    """The staged kernels count their own requests: in the loops around their matrix instructions there is no other vector memory
    access (a spilled register would be one), and nothing but the requests writes M0."""
    from importlib import util
    spec = util.spec_from_file_location("hashattn_build", os.path.join(ROOT, "hashattention-1.0_amd", "build.py"))
    mod = util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    flags = [f for f in mod.FLAGS if f != "-shared"]
    r = subprocess.run([HIPCC, *flags, "-S", "--cuda-device-only", "-I", os.path.join(ROOT, "include"), "-I", CSRC,
                        os.path.join(CSRC, "ha_linear_fp8.hip"), "-o", "-"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    scratch = dict(re.findall(r"\.name:\s+(\S+)\n\s+\.private_segment_fixed_size: (\d+)", r.stdout))
    assert scratch and not {n: b for n, b in scratch.items() if b != "0"}
    staged = [n for n in scratch if "tiled_kernel" in n]
    assert len(staged) >= 6
    for name in staged:
        body = r.stdout[r.stdout.index("\n" + name + ":"):]
        lines = body[:body.index("s_endpgm")].splitlines()
        mfma = [i for i, line in enumerate(lines) if "v_mfma" in line]
        inside = [line.strip() for line in lines[mfma[0]:mfma[-1]]]
        foreign = [line for line in inside if re.match(r"(global_|flat_|scratch_|buffer_)", line) and not line.endswith(" lds")]
        assert not foreign, (name, foreign[:3])
        assert not [line for line in lines if re.search(r"\bm0\b", line) and not line.strip().startswith(("s_mov_b32 m0,", ";"))], name
