"""GPU tests of the decoder operators (e4m3 linear layers, norm and rotation
of queries and keys, cross attention) against plain float64 forms on the CPU.

Tolerances are bounds on the arithmetic the entry points document, with
u(t) = half a step of type t relative to the value (finfo(t).eps / 2) and
U = 2^-24, every f32 operation being off by at most U of its result (2 U
where an instruction may truncate):
  - e4m3 quantization is exact: bytes and scales have to be equal;
  - a product of K terms, summed within blocks of 128 and then over blocks:
    (2 * 128 + K / 128 + 4) * U * sum |terms|, the bias and GELU a few U of
    their operands, then u(output) of the value. For 16-bit outputs the
    8-bit MFMA cuts the products of each group of 8 consecutive k off at
    2^-13 of the group's largest exponent (at most its largest term): 7
    terms lose less than that each, the largest nothing;
  - norm: the mean of D squares is off by at most (D + 2) U, its root by
    half of it; a turn adds products and one sum: (D / 2 + 16) U of
    (|a| + |b|) amp, then u of the value;
  - attention: a score is off by (D + 4) U * scale * sum |q k|, a weight by
    twice that and the exponent's rounding (U * |score| log2 e), the sums
    over n keys by n U, and 16-bit weights by u each, twice (numerator and
    their sum): all of sum p |v|; then u of the value. v_exp_f32 is within
    2 U.
Smallest outputs of f16 also round to a subnormal step (2^-25).
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from gpu_util import require_gpu
from sam3_amd import abi, hip

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TT = {abi.F32: torch.float32, abi.F16: torch.float16, abi.BF16: torch.bfloat16}
IDS = {abi.F32: "f32", abi.F16: "f16", abi.BF16: "bf16"}
DTYPES = [abi.F32, abi.F16, abi.BF16]


def u_of(dt):
    return torch.finfo(TT[dt]).eps / 2


def tiny(dt):
    return {abi.F32: 2.0 ** -149, abi.F16: 2.0 ** -25, abi.BF16: 2.0 ** -134}[dt]


@pytest.fixture(scope="module", autouse=True)
def gpu():
    require_gpu()


def rng(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def stream():
    return torch.cuda.current_stream().cuda_stream


def within(got, ref, tol, what=""):
    """|got - ref| <= tol elementwise; NaN where the reference has NaN."""
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, (got.shape, ref.shape)
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN in other places"
    err = (got - ref).abs()
    bad = (err > tol) & ~nan
    if bad.any():
        i = int(torch.argmax(torch.where(bad, err / torch.as_tensor(tol), torch.zeros_like(err))))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {got.flatten()[i]} for "
                             f"{ref.flatten()[i]}")


# ------------------------------------------------------------------- e4m3
def e4m3_groups(x, rows_per, K):
    """float64 [rows, K] -> (e4m3 values, scales) with groups of rows_per x
    128, values on [rows, KB * 128]."""
    rows, kb = x.shape[0], -(-K // 128)
    rb = -(-rows // rows_per)
    full = torch.zeros(rb * rows_per, kb * 128, dtype=torch.float64)
    full[:rows, :K] = x
    g = full.view(rb, rows_per, kb, 128).transpose(1, 2)
    mag = torch.where(g.isfinite(), g.abs(), torch.zeros_like(g)).amax((2, 3), keepdim=True)
    e = torch.full_like(mag, -126.0)
    while True:
        up = mag > 448.0 * torch.exp2(e)
        if not up.any():
            break
        e = torch.where(up, e + 1.0, e)
    y = g * torch.exp2(-e)
    _, ex = torch.frexp(y)
    step = torch.exp2((torch.clamp(ex - 1, min=-6) - 3).double())
    y = torch.where(g.isfinite(), torch.round(y / step) * step, torch.full_like(y, math.nan))
    return y.transpose(1, 2).reshape(rb * rows_per, kb * 128)[:rows], torch.exp2(e[:, :, 0, 0]), mag[:, :, 0, 0]


def bytes_value(q):
    return q.cpu().view(torch.float8_e4m3fn).float().double()


def special(x):
    """Values where a group's scale and rounding can go wrong."""
    x = x.clone()
    n = x.shape[0]
    x[0 % n, : min(5, x.shape[1])] = 448.0
    if n > 4:
        x[1] = 0.0
        x[2] *= 2.0 ** -20
        x[3] = x[3].sign() * 17.0                       # ties: 17 = 16 + 1 of a step of 2
        x[4] *= 2.0 ** 10
    return x


@pytest.mark.parametrize("dt", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("rows,K,ld", [(1, 1, 1), (1, 128, 128), (7, 129, 133), (33, 1000, 1000),
                                       (130, 256, 264), (5, 4096, 4096)])
def test_fp8_quantize_rows(dt, rows, K, ld):
    x = special(torch.randn(rows, K, generator=rng(rows + K)))
    xd = torch.full((rows, ld), 1e4, dtype=TT[dt], device="cuda")
    xd[:, :K] = x.to(TT[dt])
    kb = -(-K // 128)
    q = torch.full((rows + 1, kb * 128), 99, dtype=torch.uint8, device="cuda")
    s = torch.full((kb * rows + 3,), -1.0, device="cuda")
    hip.fp8_quantize_dev(dt, xd.data_ptr(), rows, K, q.data_ptr(), s.data_ptr(), ldx=ld, stream=stream())
    ref, sc, mag = e4m3_groups(xd[:, :K].cpu().double(), 1, K)
    got = s[:kb * rows].view(kb, rows).t().cpu().double()
    assert torch.equal(got[mag > 0], sc[mag > 0])
    assert torch.equal(torch.frexp(got)[0], torch.full_like(got, 0.5))  # powers of two everywhere
    assert torch.equal(bytes_value(q[:rows]), ref)
    assert (q[rows] == 99).all() and (s[kb * rows:] == -1).all()  # what lies behind stays


@pytest.mark.parametrize("dt", DTYPES, ids=IDS.get)
def test_fp8_quantize_extremes(dt):
    x = torch.zeros(8, 128)
    big = torch.finfo(TT[dt]).max
    x[0, 3], x[0, 4] = math.inf, 1.0
    x[1, 5], x[1, 6] = math.nan, 448.0
    x[2, 0], x[2, 1], x[2, 2] = big, -big, 1.0
    x[3, 0] = torch.finfo(TT[dt]).tiny
    x[4, 7] = {abi.F32: 2.0 ** -149, abi.F16: 2.0 ** -24, abi.BF16: 2.0 ** -133}[dt]
    x[5, :] = -math.inf
    x[6, 1], x[6, 2] = 448.5 if dt == abi.F32 else 450.0, 1.0
    x = x.to(TT[dt])
    xd = x.cuda()
    q = torch.zeros(8, 128, dtype=torch.uint8, device="cuda")
    s = torch.zeros(1, 8, device="cuda")
    hip.fp8_quantize_dev(dt, xd.data_ptr(), 8, 128, q.data_ptr(), s.data_ptr(), stream=stream())
    ref, sc, mag = e4m3_groups(x.double(), 1, 128)
    got = s.t().cpu().double()
    assert torch.equal(got[mag > 0], sc[mag > 0])
    assert (got > 0).all() and got.isfinite().all()
    v = bytes_value(q)
    assert torch.equal(torch.isnan(v), torch.isnan(ref))
    assert torch.equal(torch.nan_to_num(v), torch.nan_to_num(ref))


@pytest.mark.parametrize("dt", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("N,K,ld", [(1, 1, 3), (128, 128, 128), (129, 257, 300), (300, 1000, 1000)])
def test_fp8_quantize_weight(dt, N, K, ld):
    w = torch.randn(N, K, generator=rng(N + K)) * 0.03
    w[N // 2] *= 40.0
    wd = torch.full((N, ld), 1e4, dtype=TT[dt], device="cuda")
    wd[:, :K] = w.to(TT[dt])
    kb, nb = -(-K // 128), -(-N // 128)
    q = torch.full((N + 1, kb * 128), 99, dtype=torch.uint8, device="cuda")
    s = torch.zeros(nb, kb, device="cuda")
    hip.fp8_quantize_dev(dt, wd.data_ptr(), N, K, q.data_ptr(), s.data_ptr(), ldx=ld, stream=stream(),
                         weight=True)
    ref, sc, mag = e4m3_groups(wd[:, :K].cpu().double(), 128, K)
    assert torch.equal(s.cpu().double(), sc)
    assert torch.equal(bytes_value(q[:N]), ref)
    assert (q[N] == 99).all()


def gelu64(y):
    return 0.5 * y * (1.0 + torch.tanh(0.7978845608 * (y + 0.044715 * y ** 3)))


def product64(av, sa, wv, sw, N, K, bias, gelu, c_dt):
    """float64 result and its bound for values av [M, Kp], scales sa [KB, M],
    wv [N, Kp], sw [NB, KB]."""
    M, kb = av.shape[0], av.shape[1] // 128
    y, mag, cut = (torch.zeros(M, N, dtype=torch.float64, device=av.device) for _ in range(3))
    for b in range(kb):
        a, w = av[:, 128 * b:128 * b + 128], wv[:, 128 * b:128 * b + 128]
        s = sa[b][:, None] * sw[:, b].repeat_interleave(128)[:N]
        y += (a @ w.t()) * s
        mag += (a.abs() @ w.abs().t()) * s.abs()
        if c_dt != abi.F32:
            for k in range(0, 128, 8):
                top = (a[:, None, k:k + 8] * w[None, :, k:k + 8]).abs().amax(-1)
                cut += 7 * 2.0 ** -13 * top * s.abs()
    tol = (2 * 128 + kb + 4) * U * mag + cut
    if bias is not None:
        y = y + bias
        tol = tol + U * y.abs()
    if gelu:
        # slope of GELU at most 1.13; its own evaluation within 16 U of
        # the value, or of the argument times the logistic's steepness
        tol = 1.13 * tol + 16 * U * y.abs()
        y = gelu64(y)
    return y, tol + u_of(c_dt) * (y.abs() + tol) + tiny(c_dt)


def weights(g, N, K):
    kb, nb = -(-K // 128), -(-N // 128)
    wv = torch.zeros(N, kb * 128)
    wv[:, :K] = torch.randn(N, K, generator=g) * 60.0
    w8 = wv.clamp(-448, 448).to(torch.float8_e4m3fn)
    sw = torch.rand(nb, kb, generator=g) * 1e-3 + 1e-5  # any f32 scales, not powers of two
    return w8, sw


@pytest.mark.parametrize("c_dt", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("M,N,K,flags", [
    (1, 1, 1, 0), (1, 130, 128, hip.BIAS), (5, 64, 129, hip.BIAS | hip.GELU), (16, 48, 1000, 0),
    (33, 33, 384, hip.GELU), (64, 64, 256, 0), (65, 127, 500, hip.BIAS), (100, 300, 1544, 0),
    (257, 520, 640, hip.BIAS | hip.GELU), (300, 1001, 128, hip.BIAS), (513, 257, 130, 0)])
def test_matmul_fp8(c_dt, M, N, K, flags):
    g = rng(M * 1000 + N)
    kb = -(-K // 128)
    av = torch.zeros(M, kb * 128)
    av[:, :K] = torch.randn(M, K, generator=g) * 60.0
    a8 = av.clamp(-448, 448).to(torch.float8_e4m3fn)
    sa = torch.rand(kb, M, generator=g) * 0.02 + 1e-4
    w8, sw = weights(g, N, K)
    bias = torch.randn(N, generator=g).to(TT[c_dt])
    d = [t.cuda() for t in (a8, sa, w8, sw, bias)]
    c = torch.full((M + 1, N), 7.0, dtype=TT[c_dt], device="cuda")
    hip.matmul_fp8_dev(d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(), d[3].data_ptr(), c_dt,
                       c.data_ptr(), M, N, K, d[4].data_ptr() if flags & hip.BIAS else None, flags,
                       stream())
    ref, tol = product64(a8.float().double(), sa.double(), w8.float().double(), sw.double(), N, K,
                         bias.double() if flags & hip.BIAS else None, bool(flags & hip.GELU), c_dt)
    within(c[:M], ref, tol, f"{M}x{N}x{K}")
    assert (c[M] == 7.0).all()


@pytest.mark.parametrize("c_dt", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("M,N,K,flags", [
    (300, 702, 4100, hip.BIAS), (900, 1500, 300, 0), (700, 3001, 200, hip.BIAS), (390, 1001, 4000, 0),
    (390, 1004, 4000, hip.BIAS | hip.GELU), (400, 900, 2000, 0), (400, 905, 2000, hip.GELU),
    (1500, 3100, 700, hip.BIAS | hip.GELU), (1500, 3101, 700, 0), (2500, 4000, 260, hip.BIAS | hip.GELU),
    (2491, 4003, 260, hip.BIAS), (3000, 5000, 1100, hip.BIAS | hip.GELU), (2990, 4999, 1100, 0),
    (2990, 4996, 1100, hip.BIAS)])
def test_matmul_fp8_large(c_dt, M, N, K, flags):
    """Every tile size and both splits of k, with ends inside tiles and rows
    of whole 16 bytes, 8 and neither. The float64 form runs on the GPU."""
    g = rng(M + N)
    kb = -(-K // 128)
    av = torch.zeros(M, kb * 128)
    av[:, :K] = torch.randn(M, K, generator=g) * 60.0
    a8 = av.clamp(-448, 448).to(torch.float8_e4m3fn).cuda()
    sa = (torch.rand(kb, M, generator=g) * 0.02 + 1e-4).cuda()
    w8, sw = (t.cuda() for t in weights(g, N, K))
    bias = torch.randn(N, generator=g).to(TT[c_dt]).cuda()
    c = torch.full((M + 1, N), 7.0, dtype=TT[c_dt], device="cuda")
    hip.matmul_fp8_dev(a8.data_ptr(), sa.data_ptr(), w8.data_ptr(), sw.data_ptr(), c_dt, c.data_ptr(), M, N, K,
                       bias.data_ptr() if flags & hip.BIAS else None, flags, stream())
    ref, tol = product64(a8.float().double(), sa.double(), w8.float().double(), sw.double(), N, K,
                         bias.double() if flags & hip.BIAS else None, bool(flags & hip.GELU), c_dt)
    within(c[:M], ref.cpu(), tol.cpu(), f"{M}x{N}x{K}")
    assert (c[M] == 7.0).all()


@pytest.mark.parametrize("c_dt", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("M,N,K,flags", [
    (4400, 5003, 1100, hip.BIAS), (5600, 4104, 1100, hip.BIAS | hip.GELU), (4700, 5400, 1030, 0),
    (5000, 5003, 1100, hip.BIAS | hip.GELU), (5600, 6000, 390, hip.BIAS), (333, 2004, 700, hip.BIAS),
    (500, 1001, 700, hip.GELU), (2000, 3001, 300, hip.BIAS), (77, 1000, 4096, 0)])
def test_matmul_fp8_many_tiles(c_dt, M, N, K, flags):
    """More tiles than CUs, so that a workgroup takes several, with odd and
    even numbers of blocks and ends inside tiles; and sizes between those
    of the other tests, where the kernel changes."""
    test_matmul_fp8_large(c_dt, M, N, K, flags)


def test_matmul_fp8_k0_and_nan():
    c = torch.full((40, 9), 7.0, device="cuda")
    bias = torch.arange(9.0, device="cuda")
    hip.matmul_fp8_dev(None, None, None, None, abi.F32, c.data_ptr(), 40, 9, 0, bias.data_ptr(), hip.BIAS,
                       stream())
    assert torch.equal(c, bias.expand(40, 9))
    # a NaN byte reaches its row alone
    a = torch.full((40, 128), 0x38, dtype=torch.uint8, device="cuda")
    a[3, 5] = 0x7F
    w = torch.full((9, 128), 0x38, dtype=torch.uint8, device="cuda")
    one = torch.ones(1, 40, device="cuda")
    hip.matmul_fp8_dev(a.data_ptr(), one.data_ptr(), w.data_ptr(), one.data_ptr(), abi.F32, c.data_ptr(),
                       40, 9, 128, None, 0, stream())
    assert c[3].isnan().all()
    c[3] = 128.0
    assert (c == 128.0).all()


def linear(dt, c_dt, x, w8, sw, N, K, bias, flags, ldx=None, work=None, work_bytes=0, st=None):
    M = x.shape[0]
    c = torch.full((M, N), 7.0, dtype=TT[c_dt], device="cuda")
    hip.linear_fp8_dev(dt, x.data_ptr(), w8.data_ptr(), sw.data_ptr(), c_dt, c.data_ptr(), M, N, K,
                       bias.data_ptr() if bias is not None else None, flags, ldx=ldx, work=work,
                       work_bytes=work_bytes, stream=st or stream())
    return c


@pytest.mark.parametrize("dt", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("M,N,K,pad,flags", [
    (1, 4096, 1024, 0, hip.BIAS | hip.GELU), (1, 5, 1, 0, 0), (2, 100, 200, 3, hip.BIAS), (16, 1000, 515, 0, 0),
    (17, 96, 2048, 8, hip.BIAS), (31, 64, 128, 0, hip.GELU), (32, 1024, 4096, 0, hip.BIAS),
    (33, 200, 129, 1, 0), (77, 256, 1000, 0, hip.BIAS), (200, 130, 384, 8, hip.GELU)])
def test_linear_fp8(dt, M, N, K, pad, flags):
    g = rng(M + 7 * N + K)
    x = torch.randn(M, K, generator=g)
    x[M // 2] *= 100.0
    xd = torch.full((M, K + pad), 1e4, dtype=TT[dt], device="cuda")
    xd[:, :K] = x.to(TT[dt])
    w8, sw = weights(g, N, K)
    bias = torch.randn(N, generator=g).to(TT[dt]) if flags & hip.BIAS else None
    c = linear(dt, dt, xd, w8.cuda(), sw.cuda(), N, K, bias.cuda() if bias is not None else None, flags,
               ldx=K + pad)
    av, sa, _ = e4m3_groups(xd[:, :K].cpu().double(), 1, K)
    ref, tol = product64(av, sa.t(), w8.float().double(), sw.double(), N, K,
                         bias.double() if bias is not None else None, bool(flags & hip.GELU), dt)
    within(c, ref, tol, f"{M}x{N}x{K}")


@pytest.mark.parametrize("dt", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("M,pad", [(1, 0), (16, 1), (5, 3), (17, 0), (33, 5), (64, 1), (65, 0)])
@pytest.mark.parametrize("K", [1, 7, 8, 9, 12, 15, 23, 127, 129, 135, 250, 1029, 4097])
def test_linear_fp8_few_rows_of_any_length(dt, M, pad, K):
    """Few rows whose last values fill no eight of them, at odd addresses,
    large values between the rows."""
    test_linear_fp8(dt, M, 40, K, pad, hip.BIAS)


@pytest.mark.parametrize("dt", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("c_dt", [abi.F32, abi.BF16], ids=["to-f32", "to-bf16"])
@pytest.mark.parametrize("M", [2, 16, 40, 700])
def test_linear_fp8_nan_and_infinity(dt, c_dt, M):
    """An infinity or NaN makes its row NaN and no other."""
    g = rng(70 + M)
    N, K = 70, 264
    x = torch.randn(M, K, generator=g)
    x[0, 5], x[M - 1, 263] = math.inf, math.nan
    x = x.to(TT[dt])
    w8, sw = weights(g, N, K)
    c = linear(dt, c_dt, x.cuda(), w8.cuda(), sw.cuda(), N, K, None, 0)
    assert c[0].isnan().all() and c[M - 1].isnan().all()
    if M > 2:
        av, sa, _ = e4m3_groups(x[1:M - 1].double(), 1, K)
        ref, tol = product64(av, sa.t(), w8.float().double(), sw.double(), N, K, None, False, c_dt)
        within(c[1:M - 1], ref, tol, "other rows")


def test_linear_fp8_is_quantize_and_matmul():
    """Beyond the fused rows: the same bits as the two calls, from the
    library's scratch as from the caller's work space; x 2 bytes off."""
    g = rng(3)
    M, N, K = 150, 200, 700
    flat = torch.randn(M * K + 1, generator=g).to(torch.bfloat16).cuda()
    x = flat[1:].view(M, K)
    w8, sw = (t.cuda() for t in weights(g, N, K))
    q = torch.empty(M, 768, dtype=torch.uint8, device="cuda")
    s = torch.empty(6, M, device="cuda")
    c = torch.empty(M, N, device="cuda")
    hip.fp8_quantize_dev(abi.BF16, x.data_ptr(), M, K, q.data_ptr(), s.data_ptr(), stream=stream())
    hip.matmul_fp8_dev(q.data_ptr(), s.data_ptr(), w8.data_ptr(), sw.data_ptr(), abi.F32, c.data_ptr(), M, N,
                       K, stream=stream())
    assert torch.equal(c, linear(abi.BF16, abi.F32, x, w8, sw, N, K, None, 0))
    need = hip.linear_fp8_work(M, N, K)
    work = torch.full((need + 64,), 55, dtype=torch.uint8, device="cuda")
    assert torch.equal(c, linear(abi.BF16, abi.F32, x, w8, sw, N, K, None, 0, work=work.data_ptr(),
                                 work_bytes=need))
    assert (work[need:] == 55).all()


def test_linear_fp8_captured(env):
    """Few rows and rows with the caller's work space can be captured and
    replayed; without it a call that needs some is refused."""
    env.set("SAM3_HIP_QUIET", "1")
    g = rng(4)
    for M, N, K in ((3, 300, 520), (90, 300, 520), (50, 200, 2001), (16, 100, 4104), (5, 100, 515), (5, 100, 7)):
        w8, sw = (t.cuda() for t in weights(g, N, K))
        xs = [torch.randn(M, K, generator=g).cuda() for _ in range(3)]
        x, c = xs[0].clone(), torch.empty(M, N, device="cuda")
        need = hip.linear_fp8_work(M, N, K)
        work = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        eager = [linear(abi.F32, abi.F32, t, w8, sw, N, K, None, 0) for t in xs]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            st = stream()
            if M > 64 or K < 8:
                with pytest.raises(hip.HipError):
                    hip.linear_fp8_dev(abi.F32, x.data_ptr(), w8.data_ptr(), sw.data_ptr(), abi.F32,
                                       c.data_ptr(), M, N, K, stream=st)
            hip.linear_fp8_dev(abi.F32, x.data_ptr(), w8.data_ptr(), sw.data_ptr(), abi.F32, c.data_ptr(), M,
                               N, K, work=work.data_ptr(), work_bytes=need, stream=st)
            if M == 16:  # few rows need no space, if it comes to that
                c2 = torch.empty_like(c)
                hip.linear_fp8_dev(abi.F32, x.data_ptr(), w8.data_ptr(), sw.data_ptr(), abi.F32, c2.data_ptr(), M,
                                   N, K, stream=st)
        for t, e in zip(xs, eager):
            x.copy_(t)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(c, e)
            if M == 16:
                assert torch.allclose(c2, c, rtol=1e-4, atol=1e-4 * float(c.abs().max()))
            linear(abi.F32, abi.F32, t, w8, sw, N, K, None, 0)  # eager work between the replays


# ------------------------------------------------------- norm and rotation
def rope64(x, w, pos, freq, amp, rot, half, norm, eps, dt):
    """float64 result and bound; x [B, S, H, D], pos [B, S]."""
    D = x.shape[-1]
    if norm:
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w
    out, mag = x.clone(), x.abs()
    if rot:
        ang = pos.double()[:, :, None, None] * freq
        c, s = torch.cos(ang) * amp, torch.sin(ang) * amp
        ia = torch.arange(rot // 2) if half else torch.arange(0, rot, 2)
        ib = ia + (rot // 2 if half else 1)
        a, b = x[..., ia], x[..., ib]
        out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
        # an angle's own rounding in 64 bits: 2^-51 of it, on both sides
        both = (a.abs() + b.abs()) * amp * (1.0 + ang.abs() * 2.0 ** -51 / U)
        mag[..., ia], mag[..., ib] = both, both
    tol = ((D / 2 if norm else 0) + 16) * U * mag
    return out, tol + u_of(dt) * (out.abs() + tol) + tiny(dt)


def run_rope(dt, qkv, hq, hk, D, rot, half, norm, pos=None, freq=None, amp=1.0, wq=None, wk=None, eps=1e-6,
             inplace=False):
    """qkv [B, S, H, D] on the GPU, its first hq heads queries, the next hk
    keys; returns both (copies of their places when in place)."""
    B, S, Hn, _ = qkv.shape
    es = qkv.element_size()
    sb, ss, sh = qkv.stride()[:3]
    if inplace:
        q, k = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
    else:
        q = torch.full((B, S, hq, D), 7.0, dtype=qkv.dtype, device="cuda")
        k = torch.full((B, S, hk, D), 7.0, dtype=qkv.dtype, device="cuda")
    ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
    hip.norm_rope_dev(
        dt, B, S, D, rot, hip.ROPE_HALF if half else hip.ROPE_INTERLEAVED,
        hip.Heads(qkv.data_ptr(), q.data_ptr(), hq, sb, ss, sh, *q.stride()[:3], ptr(wq)),
        hip.Heads(qkv.data_ptr() + hq * sh * es, k.data_ptr(), hk, sb, ss, sh, *k.stride()[:3], ptr(wk)),
        pos=ptr(pos), pos_stride=S if pos is not None else 0, freq=ptr(freq), amp=amp, norm=norm, eps=eps,
        stream=stream())
    return q, k


@pytest.mark.parametrize("dt", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("norm", [False, True], ids=["turn", "norm"])
@pytest.mark.parametrize("half", [False, True], ids=["pairs", "half"])
@pytest.mark.parametrize("B,S,hq,hk,D,rot", [
    (1, 1, 1, 0, 2, 2), (4, 1, 16, 4, 128, 128), (1, 77, 3, 3, 64, 64), (2, 130, 8, 2, 80, 20),
    (1, 5, 2, 1, 96, 26), (1, 1100, 2, 1, 32, 0), (3, 33, 5, 1, 256, 64), (2, 9, 1, 1, 512, 512),
    (1, 7, 2, 2, 510, 250), (1, 4100, 2, 1, 64, 32), (2, 3, 300, 1, 16, 16)])
def test_norm_rope(dt, norm, half, B, S, hq, hk, D, rot):
    g = rng(B + S + D + rot)
    qkv = torch.randn(B, S, hq + 2 * hk, D, generator=g).to(TT[dt])
    pos = torch.randint(-50, 5000, (B, S), generator=g).to(torch.int32)
    freq = torch.from_numpy(hip.rope_frequencies(rot, 10000.0)[0])
    amp = 1.25
    wq, wk = ((1.0 + 0.3 * torch.randn(D, generator=g)).to(TT[dt]) for _ in range(2))
    x = qkv.cuda()
    before = x.clone()
    dev = [t.cuda() for t in (pos, freq, wq, wk)]
    q, k = run_rope(dt, x, hq, hk, D, rot, half, norm, dev[0], dev[1] if rot else None, amp, dev[2], dev[3])
    assert torch.equal(x, before)
    for got, src, w in ((q, qkv[:, :, :hq], wq), (k, qkv[:, :, hq:hq + hk], wk)):
        if got.numel():
            ref, tol = rope64(src.double(), w.double(), pos, freq, amp, rot, half, norm, 1e-6, dt)
            within(got, ref, tol, f"{IDS[dt]} D={D} rot={rot}")
            if not norm:  # what is not turned is copied
                assert torch.equal(got[..., rot:].cpu(), src[..., rot:])
    # in place: the same bits, and the values behind the keys stay
    q2, k2 = run_rope(dt, x, hq, hk, D, rot, half, norm, dev[0], dev[1] if rot else None, amp, dev[2], dev[3],
                      inplace=True)
    assert torch.equal(q2, q) and torch.equal(k2, k)
    assert torch.equal(x[:, :, hq + hk:], before[:, :, hq + hk:])


@pytest.mark.parametrize("dt", DTYPES, ids=IDS.get)
def test_norm_rope_far_and_default_positions(dt):
    g = rng(11)
    D = 64
    freq = torch.from_numpy(hip.rope_frequencies(D, 1e6)[0])
    x = torch.randn(1, 40, 2, D, generator=g).to(TT[dt])
    far = torch.randint(2 ** 30, 2 ** 31 - 1, (1, 40), generator=g).to(torch.int32)
    far[0, :3] = torch.tensor([-2 ** 31, 2 ** 31 - 1, 0], dtype=torch.int64).to(torch.int32)
    for pos in (far, None):
        q, _ = run_rope(dt, x.cuda(), 2, 0, D, D, True, False, pos.cuda() if pos is not None else None,
                        freq.cuda())
        ref, tol = rope64(x.double(), None, torch.arange(40)[None] if pos is None else pos, freq, 1.0, D, True,
                          False, 0.0, dt)
        within(q, ref, tol, "far" if pos is not None else "default")


@pytest.mark.parametrize("dt", DTYPES, ids=IDS.get)
def test_norm_rope_unaligned_and_transposed(dt):
    """Bases one element off, heads before positions, no weights."""
    g = rng(12)
    B, S, H, D, rot = 2, 11, 3, 48, 16
    flat = torch.randn(B * H * S * D + 1, generator=g).to(TT[dt]).cuda()
    x = flat[1:].view(B, H, S, D).transpose(1, 2)
    freq = torch.from_numpy(hip.rope_frequencies(rot)[0])
    pos = torch.arange(S).expand(B, S).to(torch.int32).contiguous()
    for half in (False, True):
        q, _ = run_rope(dt, x, H, 0, D, rot, half, True, pos.cuda(), freq.cuda(), eps=0.5)
        ref, tol = rope64(x.cpu().double(), torch.ones(D, dtype=torch.float64), pos, freq, 1.0, rot, half, True,
                          0.5, dt)
        within(q, ref, tol, f"half={half}")


def test_norm_rope_rows_do_not_mix():
    """A NaN or infinity stays in its head; a head of zeros gives zeros."""
    x = torch.randn(1, 6, 4, 64, generator=rng(13))
    x[0, 1, 2, 5], x[0, 3, 0, 9], x[0, 4] = math.nan, math.inf, 0.0
    freq = torch.from_numpy(hip.rope_frequencies(64)[0]).cuda()
    q, _ = run_rope(abi.F32, x.cuda(), 4, 0, 64, 64, True, True, None, freq)
    q = q.cpu()
    hit = torch.zeros(6, 4, dtype=torch.bool)
    hit[1, 2] = hit[3, 0] = True
    assert torch.equal(q[0].isnan().any(-1), hit)
    assert (q[0, 4] == 0).all()


# --------------------------------------------------------- cross attention
def cross64(q, k, v, qn, kn, scale, dt):
    """float64 result [B, Sq, H, D] and bound; rows past qn are NaN."""
    B, Sq, H, D = q.shape
    Hkv = k.shape[2]
    out = torch.full((B, Sq, H, D), math.nan, dtype=torch.float64)
    tol = torch.zeros_like(out)
    p_u = 0.0 if dt == abi.F32 else 2 * u_of(dt)
    for b in range(B):
        n, m = kn[b], qn[b]
        for h in range(H):
            if n == 0:
                out[b, :m, h] = 0.0
                continue
            qq, kk, vv = q[b, :m, h], k[b, :n, h * Hkv // H], v[b, :n, h * Hkv // H]
            s = qq @ kk.t() * scale
            es = (D + 4) * U * scale * (qq.abs() @ kk.abs().t()) + 4 * U * s.abs()
            es = torch.where(s.isfinite(), es, torch.zeros_like(es))  # no weight, or NaN all over
            top = s.amax(-1, keepdim=True)
            empty = (top == -math.inf)
            p = torch.where(empty, torch.zeros_like(s), torch.exp(s - torch.where(empty, torch.zeros_like(top), top)))
            l = p.sum(-1, keepdim=True)
            p = p / torch.where(l == 0, torch.ones_like(l), l)
            out[b, :m, h] = p @ vv
            w = 2 * es.amax(-1, keepdim=True) + (n + 16) * U + p_u
            tol[b, :m, h] = w * (p @ vv.abs())
    return out, tol + u_of(dt) * (out.abs() + tol) + tiny(dt)


def desc(dt, q, k, v, out, qn=None, kn=None, scale=0.0):
    B, Sq, H, D = q.shape
    return hip.CrossAttention(
        dtype=dt, B=B, H=H, Hkv=k.shape[2], Sq=Sq, Sk=k.shape[1], D=D, scale=scale, q=q.data_ptr(),
        k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(),
        **{f"{n}_{a}": t.stride(i) for n, t in (("q", q), ("k", k), ("v", v), ("o", out))
           for i, a in enumerate("bsh")},
        q_len=qn.data_ptr() if qn is not None else None, k_len=kn.data_ptr() if kn is not None else None)


def check_cross(dt, q, k, v, qn=None, kn=None, scale=0.0, path=0, out=None, what=""):
    """q, k, v on the GPU in any strides; lengths as lists."""
    B, Sq, H, D = q.shape
    Sk = k.shape[1]
    if out is None:
        out = torch.empty(B, Sq, H, D, dtype=TT[dt], device="cuda")
    out.fill_(7.0)
    lens = [torch.tensor(n, dtype=torch.int32, device="cuda") if n is not None else None for n in (qn, kn)]
    hip.cross_attention_dev(desc(dt, q, k, v, out, *lens, scale=scale), stream=stream(), path=path)
    clamp = lambda ns, most: [min(max(n, 0), most) for n in ns] if ns is not None else [most] * B  # noqa: E731
    qc, kc = clamp(qn, Sq), clamp(kn, Sk)
    ref, tol = cross64(q.cpu().double(), k.cpu().double(), v.cpu().double(), qc, kc,
                       scale if scale else D ** -0.5, dt)
    for b in range(B):
        within(out[b, :qc[b]], ref[b, :qc[b]], tol[b, :qc[b]], f"{what} b={b}")
        assert (out[b, qc[b]:] == 7.0).all(), f"{what}: rows past the length of {b}"
    return out


def qkv(seed, dt, B, H, Hkv, Sq, Sk, D, qs=1.0):
    g = rng(seed)
    return [(a * torch.randn(B, s, h, D, generator=g)).to(TT[dt]).cuda()
            for s, h, a in ((Sq, H, qs), (Sk, Hkv, 1.0), (Sk, Hkv, 1.0))]


@pytest.mark.parametrize("dt", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("B,H,Hkv,Sq,Sk,D", [
    (1, 1, 1, 1, 1, 8), (2, 4, 4, 1, 100, 64), (1, 8, 2, 1, 5000, 128), (3, 2, 1, 7, 65, 16),
    (1, 4, 1, 40, 33, 32), (2, 2, 2, 129, 200, 64), (1, 6, 2, 50, 127, 80), (1, 1, 1, 33, 64, 256),
    (1, 2, 2, 260, 1000, 128), (2, 1, 1, 200, 3000, 256), (1, 16, 4, 1, 31, 256), (1, 3, 3, 1000, 77, 32),
    (1, 32, 1, 1, 700, 64), (1, 33, 1, 1, 300, 24), (1, 2, 2, 200, 500, 72), (1, 2, 1, 40, 300, 88),
    (1, 2, 2, 200, 300, 96), (2, 2, 1, 150, 200, 104), (1, 4, 4, 5, 90, 68), (4, 8, 8, 9, 2500, 16)])
def test_cross_attention(dt, B, H, Hkv, Sq, Sk, D):
    q, k, v = qkv(B + H + Sq + Sk + D, dt, B, H, Hkv, Sq, Sk, D, 1.5)
    check_cross(dt, q, k, v)


@pytest.mark.parametrize("dt", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("path", [0, 3])
@pytest.mark.parametrize("Sq,Sk,D", [(1, 900, 64), (5, 70, 32), (70, 130, 128), (130, 300, 64), (40, 200, 256)])
def test_cross_attention_lengths(dt, path, Sq, Sk, D):
    """Lengths of zero, one, one past a tile, past the tensor, negative;
    what lies behind them holds NaN and infinities and is not read."""
    kn = [0, 1, 33, 64, 65, Sk - 1, Sk + 9, -3]
    qn = [Sq, Sq, 1, Sq // 2, Sq + 5, 0, Sq - 1, Sq]
    B = len(kn)
    q, k, v = qkv(Sq + Sk, dt, B, 4, 2, Sq, Sk, D)
    for b in range(B):
        k[b, max(kn[b], 0):], v[b, max(kn[b], 0):] = math.nan, math.inf
        q[b, max(qn[b], 0):] = math.nan
    check_cross(dt, q, k, v, qn, kn, path=path)
    check_cross(dt, q[:, :, :, :], k, v, qn, [0] * B, path=path)


@pytest.mark.parametrize("dt", DTYPES, ids=IDS.get)
def test_cross_attention_layouts(dt):
    """Heads before positions, keys and values fused in one row, rows with
    gaps, an output of its own strides, one k for all sequences."""
    g = rng(21)
    B, H, Hkv, Sq, Sk, D = 2, 4, 2, 45, 150, 64
    q = torch.randn(B, H, Sq, D, generator=g).to(TT[dt]).cuda().transpose(1, 2)
    kv = torch.randn(B, Sk, 3 * Hkv, D + 8, generator=g).to(TT[dt]).cuda()
    k, v = kv[:, :, :Hkv, :D], kv[:, :, Hkv:2 * Hkv, 8:]
    out = torch.empty(B, H, Sq, D, dtype=TT[dt], device="cuda").transpose(1, 2)
    check_cross(dt, q, k, v, kn=[149, 65], out=out, what="heads first")
    one = kv[:1, :, :Hkv, :D].expand(B, Sk, Hkv, D)
    check_cross(dt, q, one, v, kn=[150, 3], what="broadcast keys")
    shared = kv[:, :, :1, :D].expand(B, Sk, Hkv, D)
    check_cross(dt, q, shared, v, what="broadcast key head")
    wide = torch.full((B, Sq, H, D + 1), 5.0, dtype=TT[dt], device="cuda")
    check_cross(dt, q, k, v, out=wide[..., 1:], what="unaligned output")
    assert (wide[..., 0] == 5.0).all()


@pytest.mark.parametrize("dt", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("D,off", [(5, 0), (1, 0), (30, 0), (64, 1), (250, 0), (66, 0)])
def test_cross_attention_any_alignment(dt, D, off):
    g = rng(D)
    B, H, Hkv, Sq, Sk = 1, 4, 2, 9, 140
    ts = [torch.randn(B * s * h * D + off, generator=g).to(TT[dt]).cuda()[off:].view(B, s, h, D)
          for s, h in ((Sq, H), (Sk, Hkv), (Sk, Hkv))]
    p = desc(dt, *ts, ts[0])
    assert hip.load().sam3_hip_cross_attention_path(C.byref(p)) == 3
    check_cross(dt, *ts, kn=[139])


@pytest.mark.parametrize("dt", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("Sq", [1, 40, 300])
def test_cross_attention_scores_of_all_sizes(dt, Sq):
    """Sharp and flat softmax, maxima that grow from tile to tile or sit at
    the end, equal scores far from zero."""
    B, H, Sk, D = 1, 2, 700, 64
    q, k, v = qkv(5, dt, B, H, H, Sq, Sk, D)
    check_cross(dt, q, k, v, scale=3.0, what="sharp")
    check_cross(dt, q, k, v, scale=1e-6, what="flat")
    ramp = torch.linspace(-4, 4, Sk, device="cuda").view(1, Sk, 1, 1)
    one = torch.ones_like(q) * 2.0
    check_cross(dt, one, (ramp * torch.ones_like(k)).to(TT[dt]), v, what="growing")
    check_cross(dt, one, (-ramp * torch.ones_like(k)).to(TT[dt]), v, what="falling")
    check_cross(dt, one, torch.full_like(k, -30.0), v, scale=1.0, what="far below zero")
    spike = k * 0.01
    spike[:, Sk - 1] = 20.0
    check_cross(dt, one, spike, v, scale=1.0, what="last key")


@pytest.mark.parametrize("dt", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("path", [0, 3])
def test_cross_attention_infinite_scores(dt, path):
    """A key whose scores are -inf has no weight; a row of such keys alone
    gives zeros; NaN in a query or a valid key reaches its rows only."""
    B, H, Sq, Sk, D = 1, 1, 40, 70, 32
    q, k, v = qkv(6, dt, B, H, H, Sq, Sk, D)
    q = q.abs() + 0.1
    k[0, 3], k[0, 66] = -math.inf, -math.inf
    out = check_cross(dt, q, k, v, path=path, what="two")
    k2 = torch.full_like(k, -math.inf)
    out = torch.empty_like(q)
    hip.cross_attention_dev(desc(dt, q, k2, v, out), stream=stream(), path=path)
    assert (out == 0).all()
    q2 = q.clone()
    q2[0, 7, 0, 4] = math.nan
    k[0, 3], k[0, 66] = 0.5, 0.25
    check_cross(dt, q2, k, v, path=path, what="nan query")


@pytest.mark.parametrize("dt", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("B,H,Hkv,Sq,Sk,D", [
    (1, 1, 1, 1100, 3000, 64), (1, 2, 1, 1100, 2600, 256), (1, 1, 1, 1030, 2100, 16), (1, 1, 1, 2100, 1100, 64),
    (2, 4, 2, 1, 3000, 80), (1, 1, 1, 300, 2900, 72), (1, 4, 1, 300, 1700, 96),
    (1, 1, 1, 1, 40000, 64), (1, 3, 3, 2, 9000, 24), (1, 1, 1, 1, 20001, 200)])
def test_cross_attention_parts(dt, B, H, Hkv, Sq, Sk, D):
    """Keys shared out: many rows and few, as many parts as are ever made,
    and lengths that leave most parts without a key."""
    q, k, v = qkv(B + H + Sq + Sk + D, dt, B, H, Hkv, Sq, Sk, D, 1.5)
    assert hip.cross_attention_work(desc(dt, q, k, v, q)) > 0
    check_cross(dt, q, k, v)
    check_cross(dt, q, k, v, qn=[Sq - 1] * B, kn=[70] * B, what="short")
    check_cross(dt, q, k, v, kn=[0] * B, what="none")


@pytest.mark.parametrize("dt", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("B,H,Hkv,Sq,D", [(3, 8, 8, 1500, 32), (17, 4, 2, 330, 64), (64, 2, 2, 260, 16), (65, 2, 2, 260, 16)])
def test_cross_attention_many_sequences(dt, B, H, Hkv, Sq, D):
    """Many workgroups over sequences of unlike lengths, equal ones and empty
    ones among them, whichever is taken first."""
    Sk = 1100
    q, k, v = qkv(B + Sq, dt, B, H, Hkv, Sq, Sk, D)
    g = rng(B)
    kn = torch.randint(1, Sk + 1, (B,), generator=g).tolist()
    kn[0], kn[1], kn[B - 1] = 0, Sk, Sk
    check_cross(dt, q, k, v, kn=kn)
    check_cross(dt, q, k, v, qn=[Sq - b for b in range(B)], kn=[700] * B, what="equal")


@pytest.mark.parametrize("dt", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("path", [0, 3])
@pytest.mark.parametrize("Sq,Sk", [(1, 90), (1, 6000), (40, 90), (200, 2000)])
def test_cross_attention_no_weights_over_infinite_values(dt, path, Sq, Sk):
    """Rows whose scores are all -inf are zeros whatever the values hold."""
    q = torch.ones(1, Sq, 2, 64, dtype=TT[dt], device="cuda")
    k = torch.full((1, Sk, 2, 64), -math.inf, dtype=TT[dt], device="cuda")
    v = torch.full((1, Sk, 2, 64), math.inf, dtype=TT[dt], device="cuda")
    v[:, ::2] = math.nan
    out = torch.full_like(q, 7.0)
    hip.cross_attention_dev(desc(dt, q, k, v, out), stream=stream(), path=path)
    assert (out == 0).all()


def test_cross_attention_long_cache():
    """Keys and values more than 2^32 bytes from their first one."""
    Sk, D, row = 600, 64, 1 << 22
    for dt in (abi.BF16, abi.F32):
        # what is read lies in Sk rows of 2 D; the rest is never touched
        big = torch.empty(Sk * row, dtype=TT[dt], device="cuda")
        kv = big.view(Sk, row)
        kv[:, :2 * D] = torch.randn(Sk, 2 * D, generator=rng(8)).cuda().to(TT[dt])
        k = kv[:, :D].view(1, Sk, 1, D)
        v = kv[:, D:2 * D].view(1, Sk, 1, D)
        assert k.stride(1) == row
        for Sq, path in ((1, 0), (140, 0), (3, 3)):
            q = torch.randn(1, Sq, 1, D, generator=rng(9)).to(TT[dt]).cuda()
            check_cross(dt, q, k, v, kn=[599], path=path, what=f"{IDS[dt]} {Sq}")
        del big, kv, k, v


def test_cross_attention_work_space_and_graphs():
    """Parts in the caller's space, in the library's scratch, or none (a
    captured call without space); two graphs replayed on two streams."""
    dt, B, H, Sq, Sk, D = abi.BF16, 2, 4, 1, 6000, 64
    q, k, v = qkv(31, dt, B, H, H, Sq, Sk, D)
    kn = torch.tensor([6000, 3001], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    p = desc(dt, q, k, v, out, kn=kn)
    need = hip.cross_attention_work(p)
    assert need > 0
    hip.cross_attention_dev(p, stream=stream())
    eager = out.clone()
    ref, tol = cross64(q.cpu().double(), k.cpu().double(), v.cpu().double(), [1, 1], [6000, 3001], D ** -0.5, dt)
    within(eager, ref, tol, "scratch")
    work = torch.full((need + 64,), 55, dtype=torch.uint8, device="cuda")
    out.zero_()
    hip.cross_attention_dev(p, work.data_ptr(), need, stream=stream())
    assert torch.equal(out, eager) and (work[need:] == 55).all()
    torch.cuda.synchronize()

    graphs = []
    for with_work in (True, False):
        o = torch.empty_like(q)
        w = torch.empty(need, dtype=torch.uint8, device="cuda")
        gr = torch.cuda.CUDAGraph()
        d = desc(dt, q, k, v, o, kn=kn)
        with torch.cuda.graph(gr):
            hip.cross_attention_dev(d, w.data_ptr() if with_work else None, need if with_work else 0,
                                    stream=stream())
        graphs.append((gr, o, w, torch.cuda.Stream()))
    for n in range(4):
        q.copy_(torch.randn(q.shape, generator=rng(40 + n)).to(q.dtype))
        torch.cuda.synchronize()
        for gr, o, _, st in graphs:
            o.zero_()
        torch.cuda.synchronize()
        for gr, o, _, st in graphs:
            with torch.cuda.stream(st):
                gr.replay()
        hip.cross_attention_dev(p, stream=stream())
        torch.cuda.synchronize()
        ref, tol = cross64(q.cpu().double(), k.cpu().double(), v.cpu().double(), [1, 1], [6000, 3001], D ** -0.5, dt)
        assert torch.equal(graphs[0][1], out)
        within(graphs[1][1], ref, tol, f"captured without space, replay {n}")


def test_cross_attention_same_bits_every_time():
    for dt, Sq in ((abi.BF16, 1), (abi.F32, 3), (abi.F16, 200)):
        q, k, v = qkv(50, dt, 2, 4, 2, Sq, 5000, 64)
        out = torch.empty_like(q)
        p = desc(dt, q, k, v, out)
        hip.cross_attention_dev(p, stream=stream())
        first = out.clone()
        for _ in range(5):
            out.zero_()
            hip.cross_attention_dev(p, stream=stream())
            assert torch.equal(out, first)


# ------------------------------------------------------- calls side by side
def test_calls_of_several_threads():
    """Threads on streams of their own, all with the library's scratch, get
    the results of calls one after the other."""
    import threading

    M, N, K = 90, 260, 900
    jobs = []
    for n in range(4):
        g = rng(70 + n)
        w8, sw = (t.cuda() for t in weights(g, N, K))
        x = torch.randn(M, K, generator=g).to(torch.bfloat16).cuda()
        att = qkv(80 + n, abi.F16, 1, 4, 2, 1 + n, 5000, 64)
        rot = torch.randn(1, 30, 2, 64, generator=g).cuda()
        freq = torch.tensor([10000.0 ** (-i / 32) for i in range(32)], dtype=torch.float64, device="cuda")
        jobs.append((x, w8, sw, att, rot, freq, torch.cuda.Stream()))

    def run(job, st):
        x, w8, sw, (q, k, v), rot, freq, _ = job
        c = torch.empty(M, N, device="cuda")
        o, r = torch.empty_like(q), torch.empty_like(rot)
        hip.linear_fp8_dev(abi.BF16, x.data_ptr(), w8.data_ptr(), sw.data_ptr(), abi.F32, c.data_ptr(), M, N, K,
                           stream=st)
        hip.cross_attention_dev(desc(abi.F16, q, k, v, o), stream=st)
        hip.norm_rope_dev(abi.F32, 1, 30, 64, 64, hip.ROPE_HALF,
                          hip.Heads(rot.data_ptr(), r.data_ptr(), 2, 3840, 128, 64, 3840, 128, 64),
                          freq=freq.data_ptr(), norm=True, stream=st)
        return c, o, r

    alone = [run(j, stream()) for j in jobs]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(n):
        try:
            with torch.cuda.stream(jobs[n][-1]):
                got[n] = [run(jobs[n], jobs[n][-1].cuda_stream) for _ in range(20)]
                jobs[n][-1].synchronize()
        except Exception as e:  # noqa: BLE001 - handed to the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for n in range(4):
        for res in got[n]:
            for a, b in zip(res, alone[n]):
                assert torch.equal(a, b)


# ------------------------------------------------------------- as one layer
def test_decoder_layer_over_encoder_states():
    """A decoder's cross attention layer end to end: e4m3 projections of its
    tokens and of an encoder's states, norm and rotation, attention over
    states of another length, the output projection. Each step is held to
    float64 on the values it was given."""
    dt, B, Sq, Sk, E, H, Hkv, D = abi.BF16, 2, 37, 300, 256, 4, 2, 64
    g = rng(60)
    x = torch.randn(B * Sq, E, generator=g).to(TT[dt]).cuda()
    states = torch.randn(B * Sk, E, generator=g).to(TT[dt]).cuda()
    kn = [300, 123]
    lens = torch.tensor(kn, dtype=torch.int32, device="cuda")

    def made(n, k):
        w = (torch.randn(n, k, generator=g) * k ** -0.5).cuda()
        q = torch.empty(n, -(-k // 128) * 128, dtype=torch.uint8, device="cuda")
        s = torch.empty(-(-n // 128), -(-k // 128), device="cuda")
        hip.fp8_quantize_dev(abi.F32, w.data_ptr(), n, k, q.data_ptr(), s.data_ptr(), stream=stream(),
                             weight=True)
        return q, s

    def held(y, inp, w8, sw, n, k):
        av, sa, _ = e4m3_groups(inp.cpu().double(), 1, k)
        ref, tol = product64(av, sa.t(), bytes_value(w8), sw.cpu().double(), n, k, None, False, dt)
        within(y, ref, tol, "projection")

    wq, wkv, wo = made(H * D, E), made(2 * Hkv * D, E), made(E, H * D)
    q = linear(dt, dt, x, *wq, H * D, E, None, 0)
    held(q, x, *wq, H * D, E)
    kv = linear(dt, dt, states, *wkv, 2 * Hkv * D, E, None, 0)
    held(kv, states, *wkv, 2 * Hkv * D, E)
    q, kv = q.view(B, Sq, H, D), kv.view(B, Sk, 2 * Hkv, D)
    q0, kv0 = q.cpu().double(), kv.cpu().double()

    freq = torch.from_numpy(hip.rope_frequencies(D)[0])
    w = (1.0 + 0.1 * torch.randn(D, generator=g)).to(TT[dt])
    fd, wd = freq.cuda(), w.cuda()
    qp = (torch.arange(Sq) + 100).expand(B, Sq).to(torch.int32).contiguous()
    for t, heads, src, pos in ((q, H, q0, qp), (kv, Hkv, kv0[:, :, :Hkv], None)):
        n = t.shape[1]
        pd = pos.cuda() if pos is not None else None
        hd = hip.Heads(t.data_ptr(), t.data_ptr(), heads, *t.stride()[:3], *t.stride()[:3], wd.data_ptr())
        hip.norm_rope_dev(dt, B, n, D, D, hip.ROPE_HALF, hd, pos=pd.data_ptr() if pos is not None else None,
                          pos_stride=n, freq=fd.data_ptr(), norm=True, stream=stream())
        ref, tol = rope64(src, w.double(), pos if pos is not None else torch.arange(n)[None].expand(B, n), freq,
                          1.0, D, True, True, 1e-6, dt)
        within(t[:, :, :heads], ref, tol, "norm and turn")
    assert torch.equal(kv[:, :, Hkv:].cpu().double(), kv0[:, :, Hkv:])

    o = check_cross(dt, q, kv[:, :, :Hkv], kv[:, :, Hkv:], kn=kn)
    del lens
    y = linear(dt, dt, o.view(B * Sq, H * D), *wo, E, H * D, None, 0)
    held(y, o.view(B * Sq, H * D), *wo, E, H * D)
    assert np.isfinite(y.float().cpu().numpy()).all()
