"""Operators of a decoder that reads an encoder's states, as measured cases: the
8-bit floating point linear layer with scales for blocks of 128, the norm and
rotation of queries and keys, and cross attention to states of another length.

Kinds:
  fp8    y = x W^T: x quantized by groups of 128 along k (e4m3, power-of-two
         scales), W e4m3 with an f32 scale for each 128 x 128 block
  rope   queries and keys of a fused projection: RMS norm of each head (or
         none), then the rotation by position (both layouts, part of the head)
  cross  attention of queries to an encoder's keys and values, lengths per
         sequence, grouped heads

`own` chooses between the plain torch form and the framework's calls.
"""
import math
import os
import sys

import torch

# the package lies in a folder whose name is no module name
sys.path.insert(0, os.path.join(os.getcwd(), "sam3.c_amd"))

own = False

DEV = "cuda"
TT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ES = {"f32": 4, "bf16": 2, "f16": 2}
BLK = 128


def listed():
    return [
        # one token through an MLP's first layer: the latency-bound end
        {"name": "fp8_token", "kind": "fp8", "m": 1, "n": 4096, "k": 1024, "x": "bf16",
         "bias": True, "gelu": True},
        # a text prompt through an MLP's second layer: few rows, long sums
        {"name": "fp8_prompt", "kind": "fp8", "m": 32, "n": 1024, "k": 4096, "x": "bf16",
         "bias": True, "gelu": False},
        # four images' tokens through an image encoder's MLP
        {"name": "fp8_images_fc1", "kind": "fp8", "m": 20736, "n": 4096, "k": 1024, "x": "bf16",
         "bias": True, "gelu": True},
        # a cropped image's tokens, sizes that divide by no tile and end inside a block
        {"name": "fp8_ragged", "kind": "fp8", "m": 1369, "n": 1000, "k": 1544, "x": "f16",
         "bias": False, "gelu": False},
        # one new token for each of four sequences, far into a long context
        {"name": "qk_norm_token", "kind": "rope", "b": 4, "s": 1, "hq": 16, "hk": 4, "d": 128,
         "rot": 128, "half": True, "norm": True, "x": "bf16", "pos0": 70001, "scaling": "parts"},
        # the queries and keys of one image's tokens
        {"name": "qk_norm_image", "kind": "rope", "b": 1, "s": 5184, "hq": 16, "hk": 16, "d": 64,
         "rot": 64, "half": False, "norm": True, "x": "f32", "pos0": 0, "scaling": "none"},
        # a long prompt, half of each head rotated, no norm
        {"name": "rope_part_long", "kind": "rope", "b": 2, "s": 16383, "hq": 32, "hk": 8, "d": 128,
         "rot": 64, "half": True, "norm": False, "x": "f16", "pos0": 0, "scaling": "linear"},
        # one decoder token of each of eight sequences over an image's tokens
        {"name": "cross_token", "kind": "cross", "b": 8, "h": 16, "hkv": 16, "sq": 1, "sk": 5184,
         "d": 64, "x": "bf16", "lens": True},
        # prompt tokens of sixteen objects over an image, narrow heads, f32
        {"name": "cross_prompts", "kind": "cross", "b": 16, "h": 8, "hkv": 8, "sq": 9, "sk": 5184,
         "d": 16, "x": "f32", "lens": False},
        # an image's tokens over a text's tokens
        {"name": "cross_text", "kind": "cross", "b": 4, "h": 8, "hkv": 8, "sq": 5184, "sk": 77,
         "d": 32, "x": "bf16", "lens": True},
        # odd lengths, grouped heads
        {"name": "cross_grouped", "kind": "cross", "b": 3, "h": 32, "hkv": 8, "sq": 1031, "sk": 1369,
         "d": 128, "x": "f16", "lens": True},
        # a video frame's tokens over the memory of seven earlier frames, one wide head
        {"name": "cross_memory", "kind": "cross", "b": 1, "h": 1, "hkv": 1, "sq": 5184, "sk": 36288,
         "d": 256, "x": "bf16", "lens": False},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["fp8", "rope", "cross"])
    x = rng.choice(["bf16", "f16", "f32"])
    if kind == "fp8":
        n, k = _log(rng, 64, 8192), _log(rng, 64, 8192)
        return {"kind": kind, "m": _log(rng, 1, max(2, min(20736, 20736 * 4096 * 1024 // (n * k)))),
                "n": n, "k": k, "x": x, "bias": rng.random() < 0.5, "gelu": rng.random() < 0.3}
    if kind == "rope":
        d = rng.choice([32, 64, 80, 128, 256])
        hk = rng.choice([1, 2, 4, 8, 16])
        hq = hk * rng.choice([1, 1, 2, 4, 8])
        b = _log(rng, 1, 32)
        most = 2 * 16383 * 40 * 128 // (b * (hq + hk) * d * (2 if x == "f32" else 1))
        return {"kind": kind, "b": b, "s": _log(rng, 1, max(1, min(32768, most))), "hq": hq, "hk": hk,
                "d": d, "rot": rng.choice([d, d, d // 2, d // 4 // 2 * 2]), "half": rng.random() < 0.5,
                "norm": rng.random() < 0.6, "x": x, "pos0": rng.choice([0, 0, _log(rng, 1, 1 << 20)]),
                "scaling": rng.choice(["none", "linear", "parts"])}
    d = rng.choice([16, 32, 64, 64, 80, 128, 128, 256])
    hkv = rng.choice([1, 2, 4, 8])
    h = hkv * rng.choice([1, 1, 2, 4])
    b = _log(rng, 1, 32)
    sk = _log(rng, 1, 36288)
    # keys and values of at most 1 GiB; the work of the longest listed case (f32 is dearer)
    sk = max(1, min(sk, (1 << 29) // (b * hkv * d * ES[x])))
    sq = 1 if rng.random() < 0.3 else _log(rng, 1, 8192)
    sq = max(1, min(sq, 5184 * 36288 * 256 // (8 if x == "f32" else 1) // (b * h * sk * d),
                    (1 << 28) // (b * h * sk)))
    return {"kind": kind, "b": b, "h": h, "hkv": hkv, "sq": sq, "sk": sk, "d": d, "x": x,
            "lens": rng.random() < 0.6}


# ------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _frequencies(rot, scaling):
    """Radians per position of each pair, float64, and the factor on the
    rotated values, as a model's configuration gives them."""
    half = rot // 2
    f = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))
    if scaling == "linear":  # positions compressed fourfold
        return f / 4.0, 1.0
    if scaling == "parts":
        # an eightfold context: long waves compressed, short ones kept, a ramp between
        turns = 8192.0 * f / (2.0 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        return f * keep + f / 8.0 * (1.0 - keep), 0.1 * math.log(8.0) + 1.0
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) & 0x7FFFFFFFFFFFFFFF)
    t = TT[case["x"]]
    st = {"case": case}
    if case["kind"] == "fp8":
        m, n, k = case["m"], case["n"], case["k"]
        x = _randn(g, m, k)
        x *= torch.exp(0.5 * _randn(g, k))  # channels of unlike size, as activations have them
        # the checkpoint's form of the weight: e4m3 rows of whole blocks, f32 scales
        nb, kb = -(-n // BLK), -(-k // BLK)
        w = torch.zeros(nb * BLK, kb * BLK, device=DEV)
        w[:n, :k] = _randn(g, n, k) * k ** -0.5
        blocks = w.view(nb, BLK, kb, BLK)
        scale = (blocks.abs().amax((1, 3)) / 448.0).clamp_min(1e-30)
        w8 = (blocks / scale[:, None, :, None]).to(torch.float8_e4m3fn).view(nb * BLK, kb * BLK)
        st.update(x=x.to(t), w=w8[:n].contiguous(), ws=scale.contiguous(),
                  bias=_randn(g, n).to(t) if case["bias"] else None)
    elif case["kind"] == "rope":
        b, s, hq, hk, d = (case[i] for i in ("b", "s", "hq", "hk", "d"))
        qkv = _randn(g, b, s, hq + 2 * hk, d).to(t)  # a fused projection's rows
        f, amp = _frequencies(case["rot"], case["scaling"])
        start = torch.randint(0, 100, (b, 1), generator=g, device=DEV)
        pos = (torch.arange(s, device=DEV)[None] + case["pos0"] + start).to(torch.int32)
        st.update(qkv=qkv, pos=pos.contiguous(), freq=f.to(DEV), amp=amp,
                  wq=(1.0 + 0.2 * _randn(g, d)).to(t), wk=(1.0 + 0.2 * _randn(g, d)).to(t))
    else:
        b, h, hkv, sq, sk, d = (case[i] for i in ("b", "h", "hkv", "sq", "sk", "d"))
        lens = None
        if case["lens"]:
            lens = torch.randint(max(1, sk // 2), sk + 1, (b,), generator=g, device=DEV).to(torch.int32)
        st.update(q=(1.5 * _randn(g, b, sq, h, d)).to(t), kv=_randn(g, b, sk, 2 * hkv, d).to(t), lens=lens)
    return st


# ------------------------------------------------------------------- plain
def _quantized(x):
    """x [M, K] -> the values its e4m3 groups of 128 stand for, f32."""
    m, k = x.shape
    kb = -(-k // BLK)
    g = torch.nn.functional.pad(x.float(), (0, kb * BLK - k)).view(m, kb, BLK)
    mant, ex = torch.frexp(g.abs().amax(-1, keepdim=True))
    e = (ex - 9 + (mant > 0.875)).clamp_min(-126)  # least e with amax <= 448 * 2^e
    down = ((127 - e) << 23).view(torch.float32)
    up = ((127 + e) << 23).view(torch.float32)
    return ((g * down).to(torch.float8_e4m3fn).float() * up).view(m, kb * BLK)


def _plain_fp8(st):
    c = st["case"]
    n = c["n"]
    ws = st["ws"].repeat_interleave(BLK, 0)[:n].repeat_interleave(BLK, 1)
    y = _quantized(st["x"]) @ (st["w"].float() * ws).t()
    if st["bias"] is not None:
        y = y + st["bias"].float()
    if c["gelu"]:
        y = 0.5 * y * (1.0 + torch.tanh(0.7978845608 * (y + 0.044715 * y * y * y)))
    return y.to(st["x"].dtype)


def _plain_turn(x, w, cos, sin, c):
    x = x.float()
    if c["norm"]:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()
    rot = c["rot"]
    r = x[..., :rot]
    if c["half"]:
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        r = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    return torch.cat((r, x[..., rot:]), -1)


def _plain_rope(st):
    c = st["case"]
    hq, hk, t = c["hq"], c["hk"], st["qkv"].dtype
    angle = st["pos"].double()[..., None] * st["freq"]
    cos = (torch.cos(angle) * st["amp"]).float()[:, :, None]
    sin = (torch.sin(angle) * st["amp"]).float()[:, :, None]
    return (_plain_turn(st["qkv"][:, :, :hq], st["wq"], cos, sin, c).to(t),
            _plain_turn(st["qkv"][:, :, hq:hq + hk], st["wk"], cos, sin, c).to(t))


def _plain_cross(st):
    c = st["case"]
    b, h, hkv, sq, sk, d = (c[i] for i in ("b", "h", "hkv", "sq", "sk", "d"))
    q = st["q"].float().view(b, sq, hkv, h // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    k = st["kv"][:, :, :hkv].float().transpose(1, 2).contiguous()
    v = st["kv"][:, :, hkv:].float().transpose(1, 2).contiguous()
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * d ** -0.5
    if st["lens"] is not None:
        s.masked_fill_(torch.arange(sk, device=DEV) >= st["lens"].view(b, 1, 1, 1), -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return o.view(b, hkv, h // hkv, sq, d).permute(0, 3, 1, 2, 4).reshape(b, sq, h, d).to(st["q"].dtype)


# --------------------------------------------------------- the framework's
def _own(st):
    from sam3_amd import abi, hip

    c = st["case"]
    dt = {"f32": abi.F32, "bf16": abi.BF16, "f16": abi.F16}[c["x"]]
    stream = torch.cuda.current_stream().cuda_stream
    if c["kind"] == "fp8":
        x, bias = st["x"], st["bias"]
        y = torch.empty(c["m"], c["n"], dtype=x.dtype, device=DEV)
        flags = (hip.BIAS if c["bias"] else 0) | (hip.GELU if c["gelu"] else 0)
        hip.linear_fp8_dev(dt, x.data_ptr(), st["w"].data_ptr(), st["ws"].data_ptr(), dt, y.data_ptr(),
                           c["m"], c["n"], c["k"], bias.data_ptr() if bias is not None else None,
                           flags, stream=stream)
        return y
    if c["kind"] == "rope":
        b, s, hq, hk, d = (c[i] for i in ("b", "s", "hq", "hk", "d"))
        qkv, row = st["qkv"], (hq + 2 * hk) * d
        es = qkv.element_size()
        q = torch.empty(b, s, hq, d, dtype=qkv.dtype, device=DEV)
        k = torch.empty(b, s, hk, d, dtype=qkv.dtype, device=DEV)
        norm = c["norm"]
        hip.norm_rope_dev(
            dt, b, s, d, c["rot"], hip.ROPE_HALF if c["half"] else hip.ROPE_INTERLEAVED,
            hip.Heads(qkv.data_ptr(), q.data_ptr(), hq, s * row, row, d, s * hq * d, hq * d, d,
                      st["wq"].data_ptr() if norm else None),
            hip.Heads(qkv.data_ptr() + hq * d * es, k.data_ptr(), hk, s * row, row, d, s * hk * d, hk * d, d,
                      st["wk"].data_ptr() if norm else None),
            pos=st["pos"].data_ptr(), pos_stride=s, freq=st["freq"].data_ptr(), amp=st["amp"],
            norm=norm, eps=1e-6, stream=stream)
        return q, k
    b, h, hkv, sq, sk, d = (c[i] for i in ("b", "h", "hkv", "sq", "sk", "d"))
    q, kv = st["q"], st["kv"]
    row = 2 * hkv * d
    out = torch.empty(b, sq, h, d, dtype=q.dtype, device=DEV)
    hip.cross_attention_dev(hip.CrossAttention(
        dtype=dt, B=b, H=h, Hkv=hkv, Sq=sq, Sk=sk, D=d, scale=d ** -0.5,
        q=q.data_ptr(), k=kv.data_ptr(), v=kv.data_ptr() + hkv * d * kv.element_size(), out=out.data_ptr(),
        q_b=sq * h * d, q_s=h * d, q_h=d, k_b=sk * row, k_s=row, k_h=d, v_b=sk * row, v_s=row, v_h=d,
        o_b=sq * h * d, o_s=h * d, o_h=d,
        k_len=st["lens"].data_ptr() if st["lens"] is not None else None), stream=stream)
    return out


def run(state):
    if own:
        return _own(state)
    return {"fp8": _plain_fp8, "rope": _plain_rope, "cross": _plain_cross}[state["case"]["kind"]](state)


def work(case):
    es = ES[case["x"]]
    if case["kind"] == "fp8":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k * es + n * k + 4 * (-(-n // BLK)) * (-(-k // BLK)) + m * n * es
                + (n * es if case["bias"] else 0), "flops": 2 * m * n * k}
    if case["kind"] == "rope":
        vals = case["b"] * case["s"] * (case["hq"] + case["hk"]) * case["d"]
        return {"bytes": 2 * vals * es + 4 * case["b"] * case["s"], "flops": vals * (7 if case["norm"] else 3)}
    b, h, hkv, sq, sk, d = (case[i] for i in ("b", "h", "hkv", "sq", "sk", "d"))
    # lengths lie between half of sk and sk
    keys = b * sk * (3 if case["lens"] else 4) / 4
    return {"bytes": int((2 * b * sq * h * d + 2 * keys * hkv * d) * es), "flops": int(4 * keys * h * sq * d)}


# ------------------------------------------------------------------- exact
def _e4m3_64(x):
    """The nearest e4m3 value (4 significant bits, least exponent -6, ties to
    even) of float64 values of at most 448."""
    _, ex = torch.frexp(x)
    step = torch.exp2((torch.clamp(ex - 1, min=-6) - 3).double())
    return torch.round(x / step) * step


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "fp8":
        m, n, k = case["m"], case["n"], case["k"]
        x = st["x"].double()
        w = st["w"].float().double()
        y = torch.zeros(m, n, dtype=torch.float64, device=DEV)
        for kb in range(-(-k // BLK)):
            xs = x[:, kb * BLK:(kb + 1) * BLK]
            top = xs.abs().amax(1, keepdim=True)
            e = torch.clamp(torch.ceil(torch.log2(top / 448.0)), min=-126.0)
            # the logarithm may round over a power of two: settle it exactly
            e = torch.where(top > 448.0 * torch.exp2(e), e + 1.0, e)
            e = torch.where((top <= 448.0 * torch.exp2(e - 1.0)) & (e > -126.0), e - 1.0, e)
            qs = _e4m3_64(xs * torch.exp2(-e)) * torch.exp2(e)
            ws = st["ws"][:, kb].double().repeat_interleave(BLK)[:n]
            y += (qs @ w[:, kb * BLK:kb * BLK + xs.shape[1]].t()) * ws
        if case["bias"]:
            y += st["bias"].double()
        if case["gelu"]:
            y = 0.5 * y * (1.0 + torch.tanh(0.7978845608 * (y + 0.044715 * y ** 3)))
        return y
    if case["kind"] == "rope":
        hq, hk, rot = case["hq"], case["hk"], case["rot"]
        turn = torch.polar(torch.full((), st["amp"], dtype=torch.float64, device=DEV),
                           st["pos"].double()[:, :, None, None] * st["freq"])
        outs = []
        for lo, n, w in ((0, hq, st["wq"]), (hq, hk, st["wk"])):
            x = st["qkv"][:, :, lo:lo + n].double()
            if case["norm"]:
                x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6) * w.double()
            pairs = x[..., :rot].unflatten(-1, (2, rot // 2)).transpose(-1, -2) if case["half"] \
                else x[..., :rot].unflatten(-1, (rot // 2, 2))
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            x[..., :rot] = (z.transpose(-1, -2) if case["half"] else z).flatten(-2)
            outs.append(x)
        return tuple(outs)
    b, h, hkv, sq, sk, d = (case[i] for i in ("b", "h", "hkv", "sq", "sk", "d"))
    out = torch.zeros(b, sq, h, d, dtype=torch.float64, device=DEV)
    for i in range(b):
        n = int(st["lens"][i]) if st["lens"] is not None else sk
        for j in range(h):
            k = st["kv"][i, :n, j * hkv // h].double()
            v = st["kv"][i, :n, hkv + j * hkv // h].double()
            p = torch.softmax(st["q"][i, :, j].double() @ k.t() * d ** -0.5, -1)
            out[i, :, j] = p @ v
    return out
