"""CPU-side checks of the decoder operators (e4m3 linear layers, norm and
rotation, cross attention): refusals, work sizes, kernel choice and the
rotation's frequencies. Every call here returns before any device call."""
import ctypes as C
import math

import numpy as np
import pytest

from sam3_amd import abi, hip

OK = 64  # a non-NULL, aligned address that is never touched


@pytest.fixture(autouse=True)
def quiet(env):
    env.set("SAM3_HIP_QUIET", "1")


def test_fp8_refusals():
    lib = hip.load()
    q = lib.sam3_hip_fp8_quantize
    for fn in (q, lib.sam3_hip_fp8_quantize_weight):
        assert fn(abi.I8, OK, 8, 4, 8, OK, OK, None) == abi.EDTYPE
        assert fn(abi.F32, OK, 7, 4, 8, OK, OK, None) == abi.EINVAL     # rows overlap
        assert fn(abi.F32, OK, 8, -1, 8, OK, OK, None) == abi.EINVAL
        assert fn(abi.F32, OK, 8, 4, -1, OK, OK, None) == abi.EINVAL
        assert fn(abi.F32, OK, 1 << 30, 4, (1 << 22) + 1, OK, OK, None) == abi.EINVAL
        assert fn(abi.F32, None, 8, 4, 8, OK, OK, None) == abi.EINVAL
        assert fn(abi.F32, OK, 8, 4, 8, None, OK, None) == abi.EINVAL
        assert fn(abi.F32, OK, 8, 4, 8, OK, None, None) == abi.EINVAL
        assert fn(abi.F32, OK + 2, 8, 4, 8, OK, OK, None) == abi.EINVAL
        assert fn(abi.F16, OK, 8, 4, 8, OK + 8, OK, None) == abi.EINVAL
        assert fn(abi.F16, OK, 8, 4, 8, OK, OK + 2, None) == abi.EINVAL
        assert fn(abi.F16, None, 8, 0, 8, None, None, None) == abi.OK
        assert fn(abi.F16, None, 8, 4, 0, None, None, None) == abi.OK
    mm = lib.sam3_hip_matmul_fp8
    assert mm(OK, OK, OK, OK, abi.Q8_0, OK, 4, 4, 8, None, 0, None) == abi.EDTYPE
    assert mm(OK, OK, OK, OK, abi.F32, OK, -4, 4, 8, None, 0, None) == abi.EINVAL
    assert mm(OK, OK, OK, OK, abi.F32, OK, 4, 4, 8, None, hip.BIAS, None) == abi.EINVAL
    assert mm(OK, OK, OK, OK, abi.F32, OK, 4, 4, 8, None, hip.B_NT, None) == abi.EINVAL
    for i in range(4):
        args = [OK] * 4
        args[i] = None
        assert mm(*args, abi.F32, OK, 4, 4, 8, None, 0, None) == abi.EINVAL
    assert mm(OK, OK, OK, OK, abi.F32, None, 4, 4, 8, None, 0, None) == abi.EINVAL
    assert mm(OK + 8, OK, OK, OK, abi.F32, OK, 4, 4, 8, None, 0, None) == abi.EINVAL
    assert mm(OK, OK, OK + 8, OK, abi.F32, OK, 4, 4, 8, None, 0, None) == abi.EINVAL
    assert mm(OK, OK, OK, OK, abi.F32, OK + 2, 4, 4, 8, None, 0, None) == abi.EINVAL
    assert mm(None, None, None, None, abi.F32, None, 0, 4, 8, None, 0, None) == abi.OK
    lin = lib.sam3_hip_linear_fp8
    assert lin(abi.I32, OK, 8, OK, OK, abi.F32, OK, 4, 4, 8, None, 0, None, 0, None) == abi.EDTYPE
    assert lin(abi.F32, OK, 8, OK, OK, abi.I32, OK, 4, 4, 8, None, 0, None, 0, None) == abi.EDTYPE
    assert lin(abi.F32, OK, 7, OK, OK, abi.F32, OK, 4, 4, 8, None, 0, None, 0, None) == abi.EINVAL
    assert lin(abi.F32, None, 8, OK, OK, abi.F32, OK, 4, 4, 8, None, 0, None, 0, None) == abi.EINVAL
    need = hip.linear_fp8_work(1000, 4, 130)
    assert need >= 1000 * 256 + 1000 * 2 * 4
    for work, n in ((OK, need - 1), (OK + 8, need)):
        assert lin(abi.F32, OK, 130, OK, OK, abi.F32, OK, 1000, 4, 130, None, 0, work, n,
                   None) == abi.EINVAL
    assert hip.linear_fp8_work(1, 4096, 4096) == 4096 + 32 * 4
    assert hip.linear_fp8_work(1000, 0, 128) == 0 and hip.linear_fp8_work(1000, 8, 0) == 0


def heads(n=4, at=OK, out=2 * OK, **kw):
    d = dict(inp=at, out=out, heads=n, in_b=256, in_s=256, in_h=64, out_b=256, out_s=256, out_h=64,
             weight=None)
    d.update(kw)
    return hip.Heads(**d)


def norm_rope(**kw):
    d = dict(dtype=abi.F32, B=1, S=4, D=64, rot=64, layout=hip.ROPE_HALF, q=heads(), k=hip.Heads(),
             pos=None, pos_b=0, freq=OK, amp=1.0, norm=1, eps=1e-6)
    d.update(kw)
    p = hip.NormRope(**d)
    return hip.load().sam3_hip_norm_rope(C.byref(p), None)


def test_norm_rope_refusals():
    assert hip.load().sam3_hip_norm_rope(None, None) == abi.EINVAL
    assert norm_rope(dtype=abi.Q8_0) == abi.EDTYPE
    for bad in (dict(D=63), dict(D=0), dict(D=514), dict(rot=66), dict(rot=7), dict(rot=-2), dict(B=-1),
                dict(S=-1), dict(layout=2), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf),
                dict(freq=None), dict(freq=OK + 4), dict(pos=OK + 2), dict(pos=OK, pos_b=-1),
                dict(q=heads(-1)), dict(q=heads(at=None)), dict(q=heads(out=None)),
                dict(q=heads(at=OK + 2)), dict(q=heads(out=OK + 1)), dict(q=heads(weight=OK + 1)),
                dict(q=heads(in_s=-64)), dict(q=heads(out_h=-64)), dict(q=heads(out_h=0)),
                dict(q=heads(out_s=0)), dict(B=2, q=heads(out_b=0)),
                dict(q=heads(out=OK, out_s=512)),           # in place with other strides
                dict(k=heads(at=None)), dict(k=heads(out_s=0))):
        assert norm_rope(**bad) == abi.EINVAL, bad
    assert norm_rope(B=0) == abi.OK
    assert norm_rope(S=0) == abi.OK
    assert norm_rope(q=heads(0)) == abi.OK


def test_rope_frequencies():
    f, amp = hip.rope_frequencies(128, 10000.0)
    i = np.arange(64)
    assert amp == 1.0
    np.testing.assert_allclose(f, 10000.0 ** (-2.0 * i / 128), rtol=1e-14)
    g, amp = hip.rope_frequencies(128, 10000.0, hip.ROPE_LINEAR, 4.0)
    assert amp == 1.0
    np.testing.assert_allclose(g, f / 4.0, rtol=1e-15)
    g, amp = hip.rope_frequencies(128, 10000.0, hip.ROPE_PARTS, 8.0, 8192.0, 32.0, 1.0)
    keep = np.clip((8192.0 * f / (2.0 * np.pi) - 1.0) / 31.0, 0.0, 1.0)
    np.testing.assert_allclose(g, f * keep + f / 8.0 * (1.0 - keep), rtol=1e-14)
    assert amp == np.float32(0.1 * math.log(8.0) + 1.0)
    assert g[0] == f[0] and abs(g[-1] - f[-1] / 8.0) < 1e-18
    f, amp = hip.rope_frequencies(0)
    assert f.size == 0
    # factor 1 leaves them as they are
    np.testing.assert_allclose(hip.rope_frequencies(64, 1e6, hip.ROPE_PARTS, 1.0, 4096.0)[0],
                               hip.rope_frequencies(64, 1e6)[0], rtol=1e-15)
    buf, a = np.zeros(64), C.c_float()
    fn = hip.load().sam3_hip_rope_frequencies
    at = buf.ctypes.data
    for bad in ((7, 1e4, 0, 1, 1, 2, 1, at, C.byref(a)), (-2, 1e4, 0, 1, 1, 2, 1, at, C.byref(a)),
                (8, 0.0, 0, 1, 1, 2, 1, at, C.byref(a)), (8, math.nan, 0, 1, 1, 2, 1, at, C.byref(a)),
                (8, 1e4, 3, 1, 1, 2, 1, at, C.byref(a)), (8, 1e4, 1, 0.5, 1, 2, 1, at, C.byref(a)),
                (8, 1e4, 1, math.inf, 1, 2, 1, at, C.byref(a)),
                (8, 1e4, 2, 4, 0.5, 2, 1, at, C.byref(a)), (8, 1e4, 2, 4, 10, 1, 1, at, C.byref(a)),
                (8, 1e4, 2, 4, 10, 4, -math.inf, at, C.byref(a)), (8, 1e4, 2, 4, 10, math.inf, 1, at, C.byref(a)),
                (8, math.inf, 0, 1, 1, 2, 1, at, C.byref(a)),
                (8, 1e4, 0, 1, 1, 2, 1, None, C.byref(a)), (8, 1e4, 0, 1, 1, 2, 1, at, None)):
        assert fn(*bad) == abi.EINVAL, bad


def cross(**kw):
    B, H, Hkv, Sq, Sk, D = (kw.get(n, v) for n, v in (("B", 2), ("H", 8), ("Hkv", 4), ("Sq", 5),
                                                      ("Sk", 20000), ("D", 64)))
    d = dict(dtype=abi.BF16, B=B, H=H, Hkv=Hkv, Sq=Sq, Sk=Sk, D=D, scale=0.125,
             q=OK, k=OK, v=OK, out=OK, q_b=Sq * H * D, q_s=H * D, q_h=D, k_b=Sk * Hkv * D, k_s=Hkv * D,
             k_h=D, v_b=Sk * Hkv * D, v_s=Hkv * D, v_h=D, o_b=Sq * H * D, o_s=H * D, o_h=D)
    d.update(kw)
    return hip.CrossAttention(**d)


def test_cross_attention_refusals():
    lib = hip.load()

    def run(work=None, n=0, path=0, **kw):
        p = cross(**kw)
        return lib.sam3_hip_cross_attention_on_path(path, C.byref(p), work, n, None)

    assert lib.sam3_hip_cross_attention(None, None, 0, None) == abi.EINVAL
    assert run(dtype=abi.I32) == abi.EDTYPE
    for bad in (dict(B=-1), dict(H=-8), dict(Hkv=0), dict(Hkv=3), dict(Sq=-1), dict(Sk=-1), dict(D=0),
                dict(D=257), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf),
                dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(q=OK + 1), dict(k=OK + 1),
                dict(v=OK + 1), dict(out=OK + 1), dict(q_len=OK + 2), dict(k_len=OK + 1), dict(q_b=-8),
                dict(k_s=-8), dict(v_h=-8), dict(o_b=-8), dict(o_s=0), dict(o_h=0), dict(o_b=0),
                dict(Sq=1 << 30), dict(Sk=1 << 30), dict(path=4), dict(path=2),
                dict(path=1, D=60), dict(path=1, k=OK + 2), dict(path=1, q_s=12)):
        assert run(**bad) == abi.EINVAL, bad
    need = hip.cross_attention_work(cross())
    assert need > 0  # five queries over 20000 keys are shared out
    assert run(work=OK, n=need - 1) == abi.EINVAL
    assert run(work=OK + 8, n=need) == abi.EINVAL
    for nothing in (dict(B=0), dict(H=0), dict(Sq=0)):
        assert run(**nothing) == abi.OK
        assert hip.cross_attention_work(cross(**nothing)) == 0


@pytest.mark.parametrize("kw,path", [
    (dict(), 1), (dict(dtype=abi.F16, D=8), 1), (dict(D=256), 1), (dict(D=60), 3), (dict(k=OK + 2), 3),
    (dict(q_s=4), 3), (dict(dtype=abi.F32), 2), (dict(dtype=abi.F32, D=20), 2),
    (dict(dtype=abi.F32, D=18), 3), (dict(dtype=abi.F32, v=OK + 4), 3), (dict(k_s=(1 << 23) + 8), 3),
    (dict(out=OK + 2), 1), (dict(H=0), 0), (dict(D=300), 0)])
def test_cross_attention_path(kw, path):
    assert hip.load().sam3_hip_cross_attention_path(C.byref(cross(**kw))) == path


def test_too_large_for_a_launch():
    """More work-items than one launch takes, and more rows than the kernels
    count, are refused before any launch."""
    lib = hip.load()
    big, over = 1 << 30, (1 << 30) + 1
    for fn in (lib.sam3_hip_fp8_quantize, lib.sam3_hip_fp8_quantize_weight):
        assert fn(abi.BF16, OK, 8, over, 8, OK, OK, None) == abi.EINVAL
    assert lib.sam3_hip_fp8_quantize(abi.BF16, OK, 128, big, 128, OK, OK, None) == abi.EINVAL
    assert lib.sam3_hip_fp8_quantize_weight(abi.BF16, OK, 1 << 22, big, 1 << 22, OK, OK, None) == abi.EINVAL
    mm = lib.sam3_hip_matmul_fp8
    for M, N in ((over, 8), (8, over), (big, big)):
        for c in (abi.F32, abi.BF16):
            assert mm(OK, OK, OK, OK, c, OK, M, N, 8, None, 0, None) == abi.EINVAL, (M, N, c)
    lin = lib.sam3_hip_linear_fp8
    assert lin(abi.BF16, OK, 8, OK, OK, abi.BF16, OK, 1, big, 8, None, 0, None, 0, None) == abi.EINVAL
    assert norm_rope(B=1 << 16, S=1 << 16) == abi.EINVAL
    p = cross(H=1 << 20, Hkv=1 << 20, Sq=1000, D=7)
    assert lib.sam3_hip_cross_attention(C.byref(p), None, 0, None) == abi.EINVAL
