"""The dense feed-forward operators: residual addition + RMS norm + MXFP8 codes, quantization to MXFP4 and back, products with MXFP4
weights, the gated product with its quantized output, and a run of them as a block uses them.  References are plain float64
evaluations of the documented definitions (numpy / torch on the CPU), written here; tolerances are counted in rounding steps."""
import ctypes

import numpy as np
import pytest
import torch

from helpers import geometry, native, synth

EPS = 1e-6
LIMIT = 10.0
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
TYPES = {0: torch.bfloat16, 1: torch.float16, 2: torch.float32}


# ---- references ----------------------------------------------------------------------------------------------------------

def nearest(y, mantissa, least, most):
    """Nearest value of a float type with `mantissa` bits behind the point and least exponent `least` (float64, ties to even)."""
    a = np.abs(y)
    e = np.maximum(np.frexp(np.maximum(a, 1e-300))[1] - 1, least)
    return np.clip(np.round(np.ldexp(y, mantissa - e)) * np.ldexp(1.0, e - mantissa), -most, most)


def quant4(x):
    """float32 [rows][cols] -> (values of the codes, scale bytes): floor(log2(amax)) - 2, NaN blocks 255."""
    b = np.asarray(x, dtype=np.float64).reshape(x.shape[0], -1, 32)
    bad = ~np.isfinite(b).all(axis=2)
    amax = np.abs(np.where(np.isfinite(b), b, 0.0)).max(axis=2)
    zero = amax < 2.0 ** -126
    e = np.where(zero, 0, np.clip(np.frexp(np.maximum(amax, 2.0 ** -126))[1] - 3, -126, 120))
    with np.errstate(invalid="ignore"):
        codes = nearest(np.ldexp(np.where(np.isfinite(b), b, 0.0), -e[..., None]), 1, 0, 6.0)
    codes[zero | bad] = 0.0
    return codes, np.where(bad, 255, e + 127).astype(np.uint8)


def quant8(x, block, floor=0.0):
    """float64 [rows][cols] holding BF16 values -> (code values, scale bytes): amax / 448 in FP32, rounded up to a power of two."""
    b = np.asarray(x).reshape(x.shape[0], -1, block)
    amax = np.maximum(np.abs(b).max(axis=2), np.float64(np.float32(floor))).astype(np.float32) * np.float32(1.0 / 448.0)
    m, e = np.frexp(amax)
    e = np.where(m == 0.5, e - 1, e)
    codes = nearest(np.ldexp(b, -e[..., None]), 3, -6, 448.0)
    codes[amax == 0] = 0.0
    return codes.reshape(x.shape), np.where(amax == 0, 0, e + 127).astype(np.uint8)


def values4(words, scales):
    """Float64 values of canonical words [n][k / 2] and scales [n][k / 32] (torch uint8)."""
    w = words.cpu().numpy()
    codes = np.stack([w & 15, w >> 4], axis=2).reshape(w.shape[0], -1)
    v = E2M1[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = scales.cpu().numpy().astype(np.int64)
    power = np.where(s == 255, np.nan, np.ldexp(1.0, s - 127))
    return (v.reshape(w.shape[0], -1, 32) * power[..., None]).reshape(w.shape[0], -1)


def values8(codes, scales, block):
    c = codes.cpu().view(torch.float8_e4m3fn).to(torch.float64).numpy()
    s = scales.cpu().numpy().astype(np.int64)
    power = np.where(s == 0, 0.0, np.ldexp(1.0, s - 127))
    return (c.reshape(c.shape[0], -1, block) * power[..., None]).reshape(c.shape)


def f64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def bf16(v):
    return f64(torch.from_numpy(np.asarray(v)).to(torch.float32).to(torch.bfloat16))


def normal(name, *shape, std=1.0):
    return synth.normal("dense/" + name, shape, std=std)


def mxfp4(name, n, k, std=0.02):
    return synth.quantize_mxfp4(normal(name, n, k, std=std))


# ---- on the CPU ----------------------------------------------------------------------------------------------------------

def test_the_reference_quantizer_is_the_generators():
    """The numpy quantizer above against the package's own generator (written from comparisons), ties and saturation included."""
    grid = torch.tensor([0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.96875, 0.2509765625, 0.7470703125, 4.0, -0.25, -5.0])
    x = torch.cat([grid, torch.ones(16) * 4.0]).reshape(1, 32) * torch.tensor([[1.0], [2.0 ** -20], [2.0 ** 30]])
    x = torch.cat([x, normal("generator", 61, 32), torch.zeros(1, 32)])
    words, scales = synth.quantize_mxfp4(x)
    codes, bytes_ = quant4(x.numpy())
    assert np.array_equal(bytes_, scales.numpy())
    assert np.array_equal((codes * np.ldexp(1.0, bytes_.astype(int) - 127)[..., None]).reshape(x.shape), values4(words, scales))


def fake_context(block=32):
    """Memory that begins as a context does, for calls that are refused before anything else of it is read."""
    g = geometry(1024, 16, 2, 512, 512, "benchmark" if block == 128 else "reference")
    memory = ctypes.create_string_buffer(4096)
    ctypes.memmove(memory, ctypes.byref(g), ctypes.sizeof(g))
    return memory


def refusals(ctx, block=32):
    """(status wanted, function, arguments): every documented refusal.  Addresses are never followed."""
    P, Q = 1 << 20, 1 << 21          # aligned addresses
    i64 = ctypes.c_int64
    norm = dict(context=ctx, rows=2, cols=256, x=P, xs=i64(256), r=Q, rs=i64(256), w=P, eps=1e-6, ro=Q, ros=i64(256), n=P, c=P, s=P, cm=None, sm=None, stream=None)
    quant = dict(context=ctx, rows=2, cols=64, x=P, xs=i64(64), t=0, w=P, s=P, stream=None)
    dequant = dict(context=ctx, rows=2, cols=64, w=P, s=P, o=P, os=i64(64), t=0, stream=None)
    prep = dict(context=ctx, n=16, k=64, w=P, s=P, pw=Q, ps=Q, stream=None)
    linear = dict(context=ctx, rows=2, n=16, k=256, a=P, s=P, t=0, w=P, ws=P, o=P, os=i64(16), stream=None)
    swiglu = dict(context=ctx, rows=2, inter=256, k=256, a=P, s=P, t=0, u=P, us=P, g=P, gs=P, act=P, c=P, cs=P, ot=0, stream=None)
    out = []
    for name, base, changes in [
        ("ca_ffn_add_norm_quant", norm, [dict(context=None), dict(rows=-1), dict(rows=(1 << 22) + 1), dict(x=None), dict(w=None), dict(c=None), dict(s=None), dict(cm=P), dict(sm=P), dict(eps=-1.0),
                                         dict(eps=float("nan")), dict(xs=i64(248)), dict(xs=i64(260)), dict(rs=i64(255)), dict(rs=i64(12)), dict(ros=i64(1)), dict(ros=i64(257)),
                                         dict(x=P + 2), dict(r=Q + 8), dict(w=P + 4), dict(ro=P + 1), dict(n=P + 8), dict(c=P + 4), dict(cm=P + 4, sm=P),
                                         dict(n=None, c=None, s=None, ro=None)]),
        ("ca_mxfp4_quant", quant, [dict(context=None), dict(rows=-1), dict(cols=0), dict(cols=-32), dict(cols=48), dict(t=3), dict(t=-1), dict(x=None), dict(w=None), dict(s=None),
                                   dict(xs=i64(63)), dict(xs=i64(68)), dict(x=P + 8), dict(w=P + 2), dict(xs=i64(66), t=2), dict(rows=2 ** 31 - 1, cols=64)]),
        ("ca_mxfp4_dequant", dequant, [dict(context=None), dict(rows=-1), dict(cols=0), dict(cols=33), dict(t=3), dict(t=-1), dict(o=None), dict(w=None), dict(s=None),
                                       dict(os=i64(32)), dict(os=i64(65)), dict(o=P + 8), dict(w=P + 1), dict(rows=2 ** 31 - 1)]),
        ("ca_mxfp4_prepare", prep, [dict(context=None), dict(n=0), dict(n=-1), dict(k=0), dict(k=48), dict(k=65568), dict(n=(1 << 20) + 1, k=65536), dict(w=None), dict(s=None), dict(pw=None), dict(ps=None),
                                    dict(pw=P), dict(ps=P), dict(w=P + 8), dict(pw=Q + 8), dict(ps=Q + 2)]),
        ("ca_mxfp4_linear", linear, [dict(context=None), dict(rows=-1), dict(rows=(1 << 22) + 1), dict(n=0), dict(k=0), dict(k=16), dict(k=65568), dict(t=2), dict(t=-1), dict(a=None),
                                     dict(s=None), dict(w=None), dict(ws=None), dict(o=None), dict(os=i64(15)), dict(a=P + 8), dict(w=P + 8), dict(ws=P + 2), dict(o=P + 1)]
         + ([dict(k=160)] if block == 128 else [])),
        ("ca_mxfp4_swiglu", swiglu, [dict(context=None), dict(rows=-1), dict(inter=0), dict(inter=272), dict(k=0), dict(k=40), dict(t=2), dict(ot=2), dict(ot=-1), dict(a=None), dict(s=None),
                                     dict(u=None), dict(us=None), dict(g=None), dict(gs=None), dict(c=None), dict(cs=None), dict(act=None, c=None, cs=None), dict(a=P + 8), dict(u=P + 8),
                                     dict(g=P + 8), dict(us=P + 2), dict(gs=P + 1), dict(act=P + 8), dict(c=P + 4)]
         + ([dict(inter=160)] if block == 128 else [])),
    ]:
        out += [(-1, name, list({**base, **change}.values())) for change in changes]
    out += [(-4, "ca_ffn_add_norm_quant", list({**norm, **change}.values())) for change in
            [dict(cols=0), dict(cols=block // 2), dict(cols=256 + block // 2), dict(cols=8192 + block, xs=i64(16384), rs=i64(16384), ros=i64(16384))]]
    return out


@pytest.mark.parametrize("block", [32, 128])
def test_refusals_come_before_the_device(block):
    lib = native.load()
    memory = fake_context(block)
    ctx = ctypes.addressof(memory)
    for want, name, args in refusals(ctx, block):
        assert getattr(lib, name)(*args) == want, (name, args)
    assert lib.ca_mxfp4_words_bytes(0, 32) == -1 and lib.ca_mxfp4_scales_bytes(16, 48) == -1 and lib.ca_mxfp4_words_bytes(16, 65568) == -1
    # no rows: nothing is enqueued, no operand is looked at
    i64 = ctypes.c_int64
    assert lib.ca_ffn_add_norm_quant(ctx, 0, 256, None, i64(0), None, i64(0), None, 0.0, None, i64(0), None, None, None, None, None, None) == 0
    assert lib.ca_mxfp4_quant(ctx, 0, 32, None, i64(0), 0, None, None, None) == 0
    assert lib.ca_mxfp4_dequant(ctx, 0, 32, None, None, None, i64(0), 0, None) == 0
    assert lib.ca_mxfp4_linear(ctx, 0, 1, 128, None, None, 0, None, None, None, i64(0), None) == 0
    assert lib.ca_mxfp4_swiglu(ctx, 0, 128, 128, None, None, 1, None, None, None, None, None, None, None, 0, None) == 0


def test_prepared_sizes():
    lib = native.load()
    for n, k in [(1, 32), (16, 128), (17, 160), (2304, 576), (4096, 4096), (1000, 8192)]:
        tiles = -(-n // 16)
        assert lib.ca_mxfp4_words_bytes(n, k) == tiles * -(-k // 128) * 1024
        assert lib.ca_mxfp4_scales_bytes(n, k) == tiles * -(-k // 512) * 256
    assert lib.ca_mxfp4_words_bytes((1 << 20) + 1, 65536) == -1 and lib.ca_mxfp4_scales_bytes((1 << 20) + 1, 65536) == -1
    # above 2^31 bytes
    assert lib.ca_mxfp4_words_bytes(1 << 20, 65536) == 65536 * 512 * 1024


# ---- on the GPU ----------------------------------------------------------------------------------------------------------

class Gpu:
    """A context and the calls, with outputs allocated and their surroundings filled, so that a write outside shows."""

    def __init__(self, block=32):
        self.lib, self.block = native.load(), block
        g = geometry(1024, 16, 2, 512, 512, "benchmark" if block == 128 else "reference")
        self.handle = native.open_context(g)
        self.ctx = ctypes.c_void_p(self.handle)

    def stream(self):
        return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    @staticmethod
    def guarded(*shape, dtype=torch.uint8):
        """A tensor inside a larger buffer; check() sees that the bytes either side are as they were."""
        n = 1
        for s in shape:
            n *= s
        n *= torch.empty(0, dtype=dtype).element_size()
        whole = torch.full((n + 512 + (-n) % 16,), 0xA5, dtype=torch.uint8, device="cuda")
        part = whole[256:256 + n].view(dtype).reshape(shape)
        part.guard = (whole, n)
        return part

    @staticmethod
    def check(*tensors):
        for t in tensors:
            whole, n = t.guard
            assert bool((whole[:256] == 0xA5).all()) and bool((whole[256 + n:] == 0xA5).all())

    def norm(self, x, residual, weight, eps=EPS, minimum=True, out=None):
        rows, cols = x.shape
        p, B = native.ptr, self.block
        r = out if out is not None else self.guarded(rows, cols, dtype=torch.bfloat16)
        n = self.guarded(rows, cols, dtype=torch.bfloat16)
        c, s = self.guarded(rows, cols), self.guarded(rows, cols // B)
        cm, sm = (self.guarded(rows, cols), self.guarded(rows, cols // B)) if minimum else (None, None)
        status = self.lib.ca_ffn_add_norm_quant(self.ctx, rows, cols, p(x), x.stride(0), p(residual), 0 if residual is None else residual.stride(0), p(weight), eps,
                                                p(r), r.stride(0), p(n), p(c), p(s), p(cm), p(sm), self.stream())
        assert status == 0, status
        torch.cuda.synchronize()
        self.check(*[t for t in (n, c, s, cm, sm) if t is not None])
        return r, n, c, s, cm, sm

    def quant(self, x):
        rows, cols = x.shape
        w, s = self.guarded(rows, cols // 2), self.guarded(rows, cols // 32)
        kind = {v: k for k, v in TYPES.items()}[x.dtype]
        assert self.lib.ca_mxfp4_quant(self.ctx, rows, cols, native.ptr(x), x.stride(0), kind, native.ptr(w), native.ptr(s), self.stream()) == 0
        torch.cuda.synchronize()
        self.check(w, s)
        return w, s

    def dequant(self, words, scales, kind, pad=0):
        rows, cols = words.shape[0], words.shape[1] * 2
        out = self.guarded(rows, cols + pad, dtype=TYPES[kind])
        assert self.lib.ca_mxfp4_dequant(self.ctx, rows, cols, native.ptr(words), native.ptr(scales), native.ptr(out), cols + pad, kind, self.stream()) == 0
        torch.cuda.synchronize()
        self.check(out)
        return out

    def prepare(self, words, scales):
        n, k = words.shape[0], words.shape[1] * 2
        w, s = self.guarded(self.lib.ca_mxfp4_words_bytes(n, k)), self.guarded(self.lib.ca_mxfp4_scales_bytes(n, k))
        words, scales = words.cuda(), scales.cuda()
        assert self.lib.ca_mxfp4_prepare(self.ctx, n, k, native.ptr(words), native.ptr(scales), native.ptr(w), native.ptr(s), self.stream()) == 0
        torch.cuda.synchronize()
        self.check(w, s)
        return w, s

    def linear(self, rows, n, k, a, a_scales, kind, w, out=None):
        out = self.guarded(rows, n, dtype=torch.bfloat16) if out is None else out
        status = self.lib.ca_mxfp4_linear(self.ctx, rows, n, k, native.ptr(a), native.ptr(a_scales), kind, native.ptr(w[0]), native.ptr(w[1]), native.ptr(out),
                                          out.stride(0), self.stream())
        assert status == 0, status
        torch.cuda.synchronize()
        if hasattr(out, "guard"):
            self.check(out)
        return out

    def swiglu(self, rows, inter, k, a, a_scales, kind, up, gate, out_kind=0, act=True, codes=True):
        h = self.guarded(rows, inter, dtype=torch.bfloat16) if act else None
        block = self.block if out_kind == 0 else 32
        c = self.guarded(rows, inter if out_kind == 0 else inter // 2) if codes else None
        s = self.guarded(rows, inter // block) if codes else None
        p = native.ptr
        status = self.lib.ca_mxfp4_swiglu(self.ctx, rows, inter, k, p(a), p(a_scales), kind, p(up[0]), p(up[1]), p(gate[0]), p(gate[1]), p(h), p(c), p(s), out_kind, self.stream())
        assert status == 0, status
        torch.cuda.synchronize()
        self.check(*[t for t in (h, c, s) if t is not None])
        return h, c, s


@pytest.fixture(scope="module")
def gpu():
    made = {}

    def get(block=32):
        if block not in made:
            made[block] = Gpu(block)
        return made[block]
    yield get
    for g in made.values():
        g.lib.ca_primitives_close(g.ctx)


# -- quantization

@pytest.mark.gpu
def test_quant_every_bf16_value(gpu):
    """Every one of the 2^16 BF16 values in a block with every neighbour size: the device's codes, scales and what they stand for."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = torch.zeros(65536, 32, dtype=torch.bfloat16)
    x[:, 7] = bits                                            # alone in its block: the largest magnitude
    x2 = torch.zeros(65536, 32, dtype=torch.bfloat16)
    x2[:, 31], x2[:, 2] = bits, 1.0                           # beside 1: its code goes through every rounding border
    both = torch.cat([x, x2], dim=1).cuda()
    words, scales = gpu().quant(both)
    codes, want = quant4(both.cpu().float().numpy())
    assert np.array_equal(scales.cpu().numpy(), want)
    with np.errstate(invalid="ignore"):
        values = (codes * np.where(want == 255, np.nan, np.ldexp(1.0, want.astype(int) - 127))[..., None]).reshape(both.shape)
    assert np.array_equal(values4(words, scales), values, equal_nan=True)
    back = gpu().dequant(words, scales, 2)
    assert np.array_equal(f64(back), values, equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("rows,cols,pad", [(1, 32, 0), (3, 96, 8), (37, 576, 64), (130, 4096, 0), (5, 16384, 32)])
def test_quant_and_back(gpu, kind, rows, cols, pad):
    x = normal("quant", rows, cols + pad, std=0.05)
    x[0, :32] = 0.0
    if rows > 2:
        x[2, 5] = float("nan")
        x[1, cols - 1] = float("inf")
        x[2, cols - 2] = -float("inf") if cols > 32 else 0.0
    x = x.to(TYPES[kind]).cuda()[:, :cols]
    words, scales = gpu().quant(x)
    codes, want = quant4(f64(x).astype(np.float32))
    assert np.array_equal(scales.cpu().numpy(), want)
    with np.errstate(invalid="ignore"):
        values = (codes * np.where(want == 255, np.nan, np.ldexp(1.0, want.astype(int) - 127))[..., None]).reshape(rows, cols)
    for out in (0, 2):                                # BF16 and FP32 hold every value
        back = gpu().dequant(words, scales, out, pad)
        assert np.array_equal(f64(back[:, :cols]), values, equal_nan=True)
        assert back[:, cols:].numel() == 0 or bool((back[:, cols:].contiguous().view(torch.uint8) == 0xA5).all())     # between the rows: as it was
    back = gpu().dequant(words, scales, 1)            # FP16: one rounding
    want16 = f64(torch.from_numpy(values).to(torch.float32).to(torch.float16))
    assert np.array_equal(f64(back), want16, equal_nan=True)


@pytest.mark.gpu
def test_quant_fp32_extremes(gpu):
    """Scale bytes at both ends of their range, subnormal blocks, dequantization of every scale byte."""
    x = torch.zeros(8, 32)
    x[0, 0], x[1, 0], x[2, 0], x[3, 0] = 3.4e38, 2.0 ** -126, 2.0 ** -127, 2.0 ** -124
    x[4], x[5, 3], x[6, 3], x[7] = 2.0 ** 120, 1.9999999 * 2 ** 121, -(2.0 ** 122) * 1.75, -1e-38
    words, scales = gpu().quant(x.cuda())
    codes, want = quant4(x.numpy())
    assert np.array_equal(scales.cpu().numpy(), want) and want.max() == 247 and 1 in want and 127 in want
    assert np.array_equal(values4(words, scales), (codes * np.ldexp(1.0, want.astype(int) - 127)[..., None]).reshape(8, 32))
    words = torch.randint(0, 256, (256, 16), dtype=torch.uint8, generator=torch.Generator().manual_seed(1)).cuda()
    scales = torch.arange(256, dtype=torch.uint8).reshape(256, 1).cuda()
    back = f64(gpu().dequant(words, scales, 2))
    want = values4(words, scales)
    want[np.abs(want) > 3.4028235677973366e38] = np.inf * np.sign(want[np.abs(want) > 3.4028235677973366e38])
    assert np.array_equal(back, want, equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("n,k", [(1, 32), (16, 128), (17, 160), (50, 576), (512, 1024), (33, 4096)])
def test_prepared_layout(gpu, n, k):
    words, scales = mxfp4("prepare", n, k)
    w, s = gpu().prepare(words, scales)
    ks, kq, tiles = -(-k // 128), -(-k // 512), -(-n // 16)
    full = np.zeros((tiles * 16, ks * 4, 16), np.uint8)
    full[:n, :k // 32] = words.numpy().reshape(n, k // 32, 16)
    want = full.reshape(tiles, 16, ks, 4, 16).transpose(0, 2, 3, 1, 4)           # [tile][ks][g][r][16]
    assert np.array_equal(w.cpu().numpy().reshape(want.shape), want)
    full = np.zeros((tiles * 16, kq * 16), np.uint8)
    full[:n, :k // 32] = scales.numpy()
    want = full.reshape(tiles, 16, kq, 4, 4).transpose(0, 2, 4, 1, 3)            # [tile][kq][g][r][q]
    assert np.array_equal(s.cpu().numpy().reshape(want.shape), want)
    if n % 512 == 0 and k % 512 == 0:                                            # the experts' layout
        out, outs = torch.empty_like(w), torch.empty_like(s)
        native.launch("ca_expert_compact_words", -(-n * k // 32 // 256), 256, [words.cuda(), out, n, k, n])
        native.launch("ca_expert_compact_scales", -(-n * k // 32 // 256), 256, [scales.cuda(), outs, n, k, n])
        torch.cuda.synchronize()
        assert torch.equal(out, w) and torch.equal(outs, s)


# -- residual addition + norm

def norm_want(x, residual, weight, eps):
    r = f64(x) if residual is None else bf16((f64(x) + f64(residual)).astype(np.float32))      # FP32 sums of two BF16 values of like size are exact or rounded once more
    return r, r / np.sqrt((r * r).mean(axis=1, keepdims=True) + eps) * f64(weight)


@pytest.mark.gpu
@pytest.mark.parametrize("block", [32, 128])
@pytest.mark.parametrize("rows,cols,pad,residual", [(1, 128, 0, True), (3, 384, 8, True), (5, 512, 0, False), (9, 640, 64, True), (7, 1024, 0, True), (6, 1152, 8, True),
                                                    (5, 2048, 0, True), (4, 2176, 0, True), (33, 4096, 0, True), (3, 4224, 128, True), (17, 5120, 0, True), (2, 8192, 8, True),
                                                    # many rows
                                                    (515, 640, 8, True), (514, 1024, 0, False), (530, 1152, 0, True), (600, 2048, 0, True), (515, 2176, 64, True),
                                                    (513, 4096, 0, True), (530, 4224, 0, True), (520, 8192, 0, True)])
def test_add_norm_quant(gpu, block, rows, cols, pad, residual):
    g = gpu(block)
    x = normal("norm/x", rows, cols + pad).to(torch.bfloat16).cuda()[:, :cols]
    res = normal("norm/r", rows, cols + pad, std=2.0).to(torch.bfloat16).cuda()[:, :cols] if residual else None
    if rows > 2:
        x[1] = 0.0                                # a zero row: zero blocks in one flavour, floored ones in the other
        if residual:
            res[1] = 0.0
        x[2, 3] = 200.0
    w = (1.0 + normal("norm/w", cols, std=0.2)).to(torch.bfloat16).cuda()
    r, n, c, s, cm, sm = g.norm(x, res, w)
    want_r, want = norm_want(x, res, w, EPS)
    assert np.array_equal(f64(r), want_r)
    # half a BF16 step and the FP32 chain: a sum of cols terms in lanes of at most 32 and 8 exchanges (40 steps of 2^-24), root, division, two products
    assert np.all(np.abs(f64(n) - want) <= np.abs(want) * (2.0 ** -8 + 48 * 2.0 ** -24))
    for got, scales, floor in ((c, s, 0.0), (cm, sm, 1e-4)):
        codes, bytes_ = quant8(f64(n), block, floor)        # of the normalized row that the kernel stored
        assert np.array_equal(scales.cpu().numpy(), bytes_)
        assert np.array_equal(got.cpu().view(torch.float8_e4m3fn).to(torch.float64).numpy(), codes)
    # the codes alone, and in place: the same bits
    p = native.ptr
    c2, s2 = g.guarded(rows, cols), g.guarded(rows, cols // block)
    assert g.lib.ca_ffn_add_norm_quant(g.ctx, rows, cols, p(x), x.stride(0), p(res), 0 if res is None else res.stride(0), p(w), EPS, None, 0, None, p(c2), p(s2), None, None, g.stream()) == 0
    torch.cuda.synchronize()
    assert torch.equal(c, c2) and torch.equal(s, s2)
    if residual:
        again = res.clone() if pad == 0 else torch.nn.functional.pad(res, (0, pad))[:, :cols]
        g.norm(x, again, w, out=again, minimum=False)
        assert torch.equal(again, r)
        again = x.clone() if pad == 0 else torch.nn.functional.pad(x, (0, pad))[:, :cols]
        g.norm(again, res, w, out=again, minimum=False)
        assert torch.equal(again, r)


@pytest.mark.gpu
def test_add_norm_quant_is_the_norm_of_the_sum_and_keeps_rows_apart(gpu):
    """Beside ca_ffn_norm_quant on the same rows (another order of the same sum: half a step and the chain apart), NaN and infinite rows,
    and a row's result alone or among others."""
    g = gpu(32)
    rows, cols = 64, 1024
    x = normal("norm/apart", rows, cols).to(torch.bfloat16).cuda()
    res = normal("norm/apart-r", rows, cols).to(torch.bfloat16).cuda()
    w = (1.0 + normal("norm/w", cols, std=0.2)).to(torch.bfloat16).cuda()
    r, n, c, s, _, _ = g.norm(x, res, w, minimum=False)
    normed, codes, scales = torch.empty_like(n), torch.empty_like(c), torch.empty_like(s)
    p = native.ptr
    assert g.lib.ca_ffn_norm_quant(g.ctx, rows, p(r), p(w), EPS, p(normed), p(codes), p(scales), None, None, g.stream()) == 0
    torch.cuda.synchronize()
    a, b = f64(n), f64(normed)
    assert np.all(np.abs(a - b) <= np.abs(a) * 2.0 ** -7) and np.mean(a != b) < 1e-3
    bad = x.clone()
    bad[3, 10], bad[8, 0] = float("nan"), float("inf")
    r2, n2, c2, s2, _, _ = g.norm(bad, res, w, minimum=False)
    keep = [i for i in range(rows) if i not in (3, 8)]
    assert torch.equal(n2[keep], n[keep]) and torch.equal(c2[keep], c[keep]) and torch.equal(s2[keep], s[keep])
    assert bool(torch.isnan(n2[3]).all()) and bool(torch.isnan(n2[8, 0]))
    one = g.norm(x[5:6], res[5:6], w, minimum=False)
    assert torch.equal(one[1][0], n[5]) and torch.equal(one[2][0], c[5])


# -- products

def activations(g, kind, rows, k, name="a", std=1.0):
    """(codes or words, scales, float64 values) of normal rows with an outlier and a zero row."""
    x = normal(name, rows, k, std=std)
    x[0, 0] = 30.0
    if rows > 4:
        x[3] = 0.0
    if kind == native.MX_E2M1:
        words, scales = synth.quantize_mxfp4(x)
        return words.cuda(), scales.cuda(), values4(words, scales)
    codes, scales = quant8(bf16(x.numpy()), g.block)
    codes = torch.from_numpy(codes).to(torch.float8_e4m3fn).view(torch.uint8)
    scales = torch.from_numpy(scales)
    return codes.cuda(), scales.cuda(), values8(codes, scales, g.block)


def product_error(a, w, kind):
    """What the matrix core's sums may be off by.  MXFP8 x MXFP4: the instruction first adds groups of eight products of consecutive columns,
    each cut off below 2^-13 of the power of two of the group's largest (measured on one product beside a large one: 2^-13 of it is kept, 2^-14
    is lost; 1.875 * 2^-11 of it comes back as 1.75 * 2^-11); the largest itself has six significant bits and loses nothing.  So seven products
    a group lose less than 2^-13 of max|a| max|w| each.  MXFP4 products span nine bits and lose nothing there.  The groups' sums and the
    steps' meet in FP32; an addition is off by at most 2^-23 of its result (cut off): four levels of the instruction's 16 groups, at most eight
    additions where waves join, and the steps of 128 columns one after the other, whose partial sums grow from nothing to the
    sum of magnitudes: half of k / 128 times it.  Together (16 + k / 256) 2^-23 of the sum of magnitudes."""
    e = (np.abs(a) @ np.abs(w).T) * ((16 + a.shape[1] / 256) * 2.0 ** -23)
    if kind == native.MX_E4M3:
        most = lambda v: np.abs(v).reshape(v.shape[0], -1, 8).max(axis=2)
        e += (most(a) @ most(w).T) * (7 * 2.0 ** -13)
    return e


SHAPES = [(1, 16, 32), (1, 1, 128), (2, 50, 160), (5, 257, 576), (16, 64, 512), (17, 100, 1056), (31, 304, 2048), (33, 48, 4096), (64, 513, 1152), (65, 96, 640),
          (127, 320, 2176), (128, 256, 512), (257, 515, 1600), (300, 1024, 1024), (531, 130, 576), (1025, 777, 384)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,block", [(0, 32), (0, 128), (1, 32)])
@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_linear(gpu, kind, block, rows, n, k):
    g = gpu(block)
    if block == 128:
        k = -(-k // 128) * 128
    a, a_scales, av = activations(g, kind, rows, k)
    words, scales = mxfp4("w", n, k)
    wv = values4(words, scales)
    w = g.prepare(words, scales)
    out = g.linear(rows, n, k, a, a_scales, kind, w)
    want = av @ wv.T
    assert np.all(np.abs(f64(out) - want) <= np.abs(want) * 2.0 ** -8 + product_error(av, wv, kind))
    # rows further apart, at an odd distance (two-byte stores) and a multiple of four: the same bits, nothing between the rows written
    for stride in (n + 1, n + (-n) % 4 + 4):
        wide = g.guarded(rows, stride, dtype=torch.bfloat16)
        g.linear(rows, n, k, a, a_scales, kind, w, out=wide[:, :n])
        g.check(wide)
        assert torch.equal(wide[:, :n], out) and bool((wide[:, n:].contiguous().view(torch.uint8) == 0xA5).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind,block", [(0, 32), (0, 128), (1, 32)])
@pytest.mark.parametrize("rows,n,k", [(1090, 2100, 416), (1090, 2100, 640), (1025, 2304, 512), (4090, 4090, 512), (4090, 4090, 640), (4090, 4084, 544),
                                       (4090, 4088, 512), (8190, 4088, 640), (8190, 4088, 1536)])
def test_linear_large_tiles(gpu, kind, block, rows, n, k):
    """Enough tiles that the larger ones are chosen, and more than one a compute unit, ragged in both directions.  The reference runs on the
    device in float64."""
    g = gpu(block)
    if block == 128:
        k = -(-k // 128) * 128
    a, a_scales, av = activations(g, kind, rows, k)
    words, scales = mxfp4("w", n, k)
    wv = values4(words, scales)
    out = g.linear(rows, n, k, a, a_scales, kind, g.prepare(words, scales)).double()
    want, bound = device_product(av, wv, kind)
    assert bool(((out - want).abs() <= want.abs() * 2.0 ** -8 + bound).all())
    # rows further apart: the same bits, nothing between the rows written
    wide = g.guarded(rows, n + 8, dtype=torch.bfloat16)
    g.linear(rows, n, k, a, a_scales, kind, g.prepare(words, scales), out=wide[:, :n])
    g.check(wide)
    assert torch.equal(wide[:, :n].double(), out) and bool((wide[:, n:].contiguous().view(torch.uint8) == 0xA5).all())


def device_product(av, wv, kind):
    """The product and product_error() on the device, in float64."""
    a, w = torch.from_numpy(av).cuda(), torch.from_numpy(wv).cuda()
    e = (a.abs() @ w.abs().t().contiguous()) * ((16 + av.shape[1] / 256) * 2.0 ** -23)
    if kind == native.MX_E4M3:
        most = lambda v: v.abs().reshape(v.shape[0], -1, 8).amax(dim=2)
        e += (most(a) @ most(w).t().contiguous()) * (7 * 2.0 ** -13)
    return a @ w.t().contiguous(), e


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [0, 1])
def test_linear_exact_small_whole_numbers(gpu, kind):
    """Whole-number operands whose sums every format holds: no rounding anywhere, so every index of the product is checked exactly."""
    g = gpu(32)
    gen = torch.Generator().manual_seed(7)
    for rows, n, k in [(3, 40, 96), (70, 272, 1120), (260, 512, 512)]:
        grid = torch.tensor([-1.0, 0.0, 0.0, 0.0, 0.0, 1.0])
        a = grid[torch.randint(0, 6, (rows, k), generator=gen)]
        w = grid[torch.randint(0, 6, (n, k), generator=gen)]
        a[:, ::32], w[:, ::32] = 4.0, 4.0                   # every block's scale is 1 (MXFP4: floor(log2 4) - 2 = 0)
        a[:, 32::64] = -4.0
        words, scales = synth.quantize_mxfp4(w)
        assert np.array_equal(values4(words, scales), w.numpy())
        if kind == 1:
            ac, asc = synth.quantize_mxfp4(a)
        else:
            ac, asc = a.to(torch.float8_e4m3fn).view(torch.uint8), torch.full((rows, k // 32), 127, dtype=torch.uint8)
        out = g.linear(rows, n, k, ac.cuda(), asc.cuda(), kind, g.prepare(words, scales))
        want = a.double() @ w.double().T
        assert float(want.abs().max()) <= 256 * 4
        assert np.array_equal(f64(out), bf16(want.numpy()))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("rows", [5, 200])
def test_linear_rows_do_not_touch_each_other(gpu, kind, rows):
    """A NaN in one row stays there, whatever tile it shares (k no multiple of 128: the next row's bytes lie where the last step's columns
    would be); a block whose scale is NaN is one too."""
    g = gpu(32)
    n, k = 80, 288
    a, a_scales, _ = activations(g, kind, rows, k)
    words, scales = mxfp4("w", n, k)
    w = g.prepare(words, scales)
    clean = g.linear(rows, n, k, a, a_scales, kind, w)
    bad = a_scales.clone()
    bad[2, 0], bad[4, k // 32 - 1] = 255, 255
    codes = a.clone()
    if kind == 0:
        codes[1, 0] = 0x7f
    out = g.linear(rows, n, k, codes, bad, kind, w)
    hit = [2, 4] + ([1] if kind == 0 else [])
    keep = [i for i in range(rows) if i not in hit]
    assert torch.equal(out[keep], clean[keep]) and bool(torch.isnan(out[hit]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("rows", [7, 300])
def test_linear_scale_range(gpu, kind, rows):
    """Scales from 2^-60 to 2^60 a block, the weights' opposite: sums stay of ordinary size."""
    g = gpu(32)
    n, k = 96, 768
    gen = torch.Generator().manual_seed(3)
    shift = torch.randint(-60, 61, (k // 32,), generator=gen)
    a, a_scales, _ = activations(g, kind, rows, k)
    a_scales = (a_scales.cpu().int().clamp(min=64) + shift).to(torch.uint8).cuda()
    words, scales = mxfp4("w", n, k)
    scales = (scales.int() - shift).to(torch.uint8)
    av = values4(a, a_scales) if kind else values8(a, a_scales, 32)
    wv = values4(words, scales)
    out = g.linear(rows, n, k, a, a_scales, kind, g.prepare(words, scales))
    want = av @ wv.T
    assert np.all(np.abs(f64(out) - want) <= np.abs(want) * 2.0 ** -8 + product_error(av, wv, kind))


def swiglu_want(av, up, gate, kind):
    """The activation in float64, and what an error of the two sums moves it by: |d(silu)| <= 1.1 |dg|, |u| <= L."""
    g, u = av @ gate.T, av @ up.T
    eg, eu = product_error(av, gate, kind), product_error(av, up, kind)
    gc, uc = np.minimum(g, LIMIT), np.clip(u, -LIMIT, LIMIT)
    sig = 1.0 / (1.0 + np.exp(-gc))
    silu = gc * sig
    # the fast logistic: the hardware's exponential and reciprocal, one unit of FP32 each, and the exponent's rounding times its size
    return silu * uc, 1.1 * eg * (np.abs(uc) + eu) + np.abs(silu) * eu + np.abs(silu * uc) * (np.abs(gc) + 4) * 2.0 ** -23


@pytest.mark.gpu
@pytest.mark.parametrize("kind,block", [(0, 32), (0, 128), (1, 32), (1, 128)])
@pytest.mark.parametrize("rows,inter,k", [(1, 128, 128), (4, 640, 512), (16, 256, 1152), (17, 384, 2048), (45, 2304, 640), (64, 128, 4096), (65, 256, 512), (130, 512, 768), (300, 1152, 512),
                                          (515, 384, 1664)])
def test_swiglu(gpu, kind, block, rows, inter, k):
    g = gpu(block)
    a, a_scales, av = activations(g, kind, rows, k, std=2.0)
    ups, gates = mxfp4("up", inter, k, std=0.1), mxfp4("gate", inter, k, std=0.1)
    up, gate = g.prepare(*ups), g.prepare(*gates)
    h, c, s = g.swiglu(rows, inter, k, a, a_scales, kind, up, gate)
    want, moved = swiglu_want(av, values4(*ups), values4(*gates), kind)
    assert k < 512 or np.abs(av @ values4(*gates).T).max() > LIMIT           # the clip is in play
    assert np.all(np.abs(f64(h) - want) <= np.abs(want) * 2.0 ** -8 + moved)
    codes, bytes_ = quant8(f64(h), block)                          # of the activation that the kernel stored
    assert np.array_equal(s.cpu().numpy(), bytes_)
    assert np.array_equal(c.cpu().view(torch.float8_e4m3fn).to(torch.float64).numpy(), codes)
    if rows > 4:
        assert not bool(s[3].any()) and not bool(c[3].view(torch.float8_e4m3fn).float().any())     # a zero row: zero blocks
    # each output alone: the same bits
    h2, _, _ = g.swiglu(rows, inter, k, a, a_scales, kind, up, gate, codes=False)
    _, c2, s2 = g.swiglu(rows, inter, k, a, a_scales, kind, up, gate, act=False)
    assert torch.equal(h, h2) and torch.equal(c, c2) and torch.equal(s, s2)
    # 4-bit codes: what the quantizer makes of the stored activation
    h4, w4, s4 = g.swiglu(rows, inter, k, a, a_scales, kind, up, gate, out_kind=native.MX_E2M1)
    words, scales = g.quant(h4)
    assert torch.equal(h4, h) and torch.equal(w4, words) and torch.equal(s4, scales)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,block", [(0, 32), (0, 128), (1, 32), (1, 128)])
@pytest.mark.parametrize("rows,inter,k", [(1090, 1152, 640), (4090, 2016, 512), (4090, 2016, 416)])
def test_swiglu_large_tiles(gpu, kind, block, rows, inter, k):
    g = gpu(block)
    if block == 128:
        inter, k = -(-inter // 128) * 128, -(-k // 128) * 128
    a, a_scales, av = activations(g, kind, rows, k, std=2.0)
    ups, gates = mxfp4("up", inter, k, std=0.1), mxfp4("gate", inter, k, std=0.1)
    up, gate = g.prepare(*ups), g.prepare(*gates)
    h, c, s = g.swiglu(rows, inter, k, a, a_scales, kind, up, gate)
    (gv, eg), (uv, eu) = device_product(av, values4(*gates), kind), device_product(av, values4(*ups), kind)
    gc, uc = gv.clamp(max=LIMIT), uv.clamp(-LIMIT, LIMIT)
    silu = gc / (1.0 + torch.exp(-gc))
    want = silu * uc
    moved = 1.1 * eg * (uc.abs() + eu) + silu.abs() * eu + want.abs() * (gc.abs() + 4) * 2.0 ** -23        # as swiglu_want()
    assert bool(((h.double() - want).abs() <= want.abs() * 2.0 ** -8 + moved).all())
    codes, bytes_ = quant8(f64(h), block)
    assert np.array_equal(s.cpu().numpy(), bytes_)
    assert np.array_equal(c.cpu().view(torch.float8_e4m3fn).to(torch.float64).numpy(), codes)
    h2, w4, s4 = g.swiglu(rows, inter, k, a, a_scales, kind, up, gate, out_kind=native.MX_E2M1)
    words, scales = g.quant(h2)
    assert torch.equal(h2, h) and torch.equal(w4, words) and torch.equal(s4, scales)
    _, c3, s3 = g.swiglu(rows, inter, k, a, a_scales, kind, up, gate, act=False)
    assert torch.equal(c3, c) and torch.equal(s3, s)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 150])
def test_swiglu_odd_widths_and_nan(gpu, rows):
    """A width that is a multiple of the code blocks alone (96), a contraction of 32 and of 1,056, and a NaN row that stays one."""
    g = gpu(32)
    for inter, k in [(96, 32), (32, 1056), (160, 544)]:
        a, a_scales, av = activations(g, 0, rows, k)
        ups, gates = mxfp4("up", inter, k, std=0.2), mxfp4("gate", inter, k, std=0.2)
        up, gate = g.prepare(*ups), g.prepare(*gates)
        h, c, s = g.swiglu(rows, inter, k, a, a_scales, 0, up, gate)
        want, moved = swiglu_want(av, values4(*ups), values4(*gates), 0)
        assert np.all(np.abs(f64(h) - want) <= np.abs(want) * 2.0 ** -8 + moved)
        codes, bytes_ = quant8(f64(h), 32)
        assert np.array_equal(s.cpu().numpy(), bytes_) and np.array_equal(c.cpu().view(torch.float8_e4m3fn).to(torch.float64).numpy(), codes)
        bad = a.clone()
        bad[1, k - 1] = 0x7f
        h2, c2, _ = g.swiglu(rows, inter, k, bad, a_scales, 0, up, gate)
        keep = [i for i in range(rows) if i != 1]
        assert torch.equal(h2[keep], h[keep]) and torch.equal(c2[keep], c[keep])
        assert bool(torch.isnan(h2[1]).all()) and bool(((c2[1] & 0x7f) == 0x7f).all())
        _, w4, s4 = g.swiglu(rows, inter, k, bad, a_scales, 0, up, gate, out_kind=1)
        assert bool((s4[1] == 255).all()) and not bool(w4[1].any())


# -- as a block uses them

def block_pass(g, kind, weights, x, residual, norm_w, inter, buffers):
    """norm -> gated product -> down projection, all enqueued on the current stream; returns (residual, output)."""
    rows, cols = x.shape
    lib, p, B = g.lib, native.ptr, g.block
    r, n, c, s, h, hc, hs, y = buffers
    up, gate, down = weights
    assert lib.ca_ffn_add_norm_quant(g.ctx, rows, cols, p(x), cols, p(residual), cols, p(norm_w), EPS, p(r), cols, p(n), p(c) if kind == 0 else None,
                                     p(s) if kind == 0 else None, None, None, g.stream()) == 0
    if kind == 1:
        assert lib.ca_mxfp4_quant(g.ctx, rows, cols, p(n), cols, 0, p(c), p(s), g.stream()) == 0
    assert lib.ca_mxfp4_swiglu(g.ctx, rows, inter, cols, p(c), p(s), kind, p(up[0]), p(up[1]), p(gate[0]), p(gate[1]), p(h), p(hc), p(hs), kind, g.stream()) == 0
    assert lib.ca_mxfp4_linear(g.ctx, rows, cols, inter, p(hc), p(hs), kind, p(down[0]), p(down[1]), p(y), cols, g.stream()) == 0
    return r, y


def block_buffers(g, kind, rows, cols, inter):
    e = lambda *shape, dtype=torch.uint8: torch.empty(shape, dtype=dtype, device="cuda")
    block, half = (32, 2) if kind == 1 else (g.block, 1)
    return (e(rows, cols, dtype=torch.bfloat16), e(rows, cols, dtype=torch.bfloat16), e(rows, cols // half), e(rows, cols // block),
            e(rows, inter, dtype=torch.bfloat16), e(rows, inter // half), e(rows, inter // block), e(rows, cols, dtype=torch.bfloat16))


def block_case(g, rows, cols, inter):
    x, res = normal("block/x", rows, cols).to(torch.bfloat16).cuda(), normal("block/r", rows, cols).to(torch.bfloat16).cuda()
    w = (1.0 + normal("block/w", cols, std=0.1)).to(torch.bfloat16).cuda()
    # the weights come from BF16 masters through the device's own quantizer
    masters = [normal("block/" + name, *shape, std=0.05).to(torch.bfloat16).cuda() for name, shape in
               (("up", (inter, cols)), ("gate", (inter, cols)), ("down", (cols, inter)))]
    canonical = [g.quant(m) for m in masters]
    return x, res, w, canonical, [g.prepare(*c) for c in canonical]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,block", [(0, 32), (0, 128), (1, 32)])
@pytest.mark.parametrize("rows", [1, 4, 33, 300])
def test_a_block_of_them(gpu, kind, block, rows):
    g = gpu(block)
    cols, inter = 512, 1152
    x, res, w, canonical, weights = block_case(g, rows, cols, inter)
    buffers = block_buffers(g, kind, rows, cols, inter)
    r, y = block_pass(g, kind, weights, x, res, w, inter, buffers)
    torch.cuda.synchronize()
    # each step against float64 from the step before it as the device stored it
    up, gate, down = (values4(*c) for c in canonical)
    _, n, c, s, h, hc, hs, _ = buffers
    read = values4 if kind == 1 else lambda a, b: values8(a, b, block)
    want, moved = swiglu_want(read(c, s), up, gate, kind)
    assert np.all(np.abs(f64(h) - want) <= np.abs(want) * 2.0 ** -8 + moved)
    hv = read(hc, hs)
    want = hv @ down.T
    assert np.all(np.abs(f64(y) - want) <= np.abs(want) * 2.0 ** -8 + product_error(hv, down, kind))
    want_r, want_n = norm_want(x, res, w, EPS)
    assert np.array_equal(f64(r), want_r) and np.all(np.abs(f64(n) - want_n) <= np.abs(want_n) * (2.0 ** -8 + 48 * 2.0 ** -24))
    # end to end against the same block without any quantization of its activations: 8 bits cost 3 % of the output's size, 4 bits 20 %.
    # E4M3 keeps each value to 2^-4 (uniform in a step: 2^-4 / sqrt 3 / 1.4 ~ 2.6 %), twice; E2M1 to a quarter (~ 12 %), twice.
    g0, u0 = want_n @ gate.T, want_n @ up.T
    h0 = np.minimum(g0, LIMIT) / (1.0 + np.exp(-np.minimum(g0, LIMIT))) * np.clip(u0, -LIMIT, LIMIT)
    plain = h0 @ down.T
    off = np.linalg.norm(f64(y) - plain) / np.linalg.norm(plain)
    assert off < (0.06 if kind == 0 else 0.3), off


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("rows", [3, 200])
def test_a_block_captured_and_replayed(gpu, kind, rows):
    """The block in a graph on a stream of its own: replays with new inputs, eager work and other calls between them, give the eager bits."""
    g = gpu(32)
    cols, inter = 512, 640
    x, res, w, _, weights = block_case(g, rows, cols, inter)
    buffers, eager = block_buffers(g, kind, rows, cols, inter), block_buffers(g, kind, rows, cols, inter)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        block_pass(g, kind, weights, x, res, w, inter, buffers)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        block_pass(g, kind, weights, x, res, w, inter, buffers)
    for i in range(4):
        x.copy_(normal("block/replay%d" % i, rows, cols).to(torch.bfloat16))
        for b in buffers:
            b.view(torch.uint8).fill_(0x11)
        graph.replay()
        block_pass(g, kind, weights, x, res, w, inter, eager)
        torch.cuda.synchronize()
        for a, b in zip(buffers, eager):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.gpu
def test_two_streams_at_once(gpu):
    """Passes on two streams that overlap share nothing: each gives what it gives alone."""
    g = gpu(32)
    cases = [(96, 512, 640), (300, 256, 512)]
    made = [block_case(g, *c) for c in cases]
    alone = []
    for (rows, cols, inter), (x, res, w, _, weights) in zip(cases, made):
        buffers = block_buffers(g, 0, rows, cols, inter)
        block_pass(g, 0, weights, x, res, w, inter, buffers)
        torch.cuda.synchronize()
        alone.append([b.clone() for b in buffers])
    streams = [torch.cuda.Stream() for _ in cases]
    both = [block_buffers(g, 0, *c) for c in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for (rows, cols, inter), (x, res, w, _, weights), stream, buffers in zip(cases, made, streams, both):
            with torch.cuda.stream(stream):
                block_pass(g, 0, weights, x, res, w, inter, buffers)
    torch.cuda.synchronize()
    for a, b in zip(alone, both):
        assert all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("block", [32, 128])
def test_refusals_on_a_real_context(gpu, block):
    g = gpu(block)
    for want, name, args in refusals(g.handle, block):
        assert getattr(g.lib, name)(*args) == want, (name, args)
    assert torch.cuda.is_available() and int(torch.ones(3, device="cuda").sum()) == 3      # no error was left behind


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("rows,n", [(3, 5), (300, 72)])
def test_the_longest_contraction(gpu, kind, rows, n):
    g = gpu(32)
    k = 65536
    a, a_scales, av = activations(g, kind, rows, k)
    words, scales = mxfp4("long", n, k)
    wv = values4(words, scales)
    out = g.linear(rows, n, k, a, a_scales, kind, g.prepare(words, scales))
    want = av @ wv.T
    assert np.all(np.abs(f64(out) - want) <= np.abs(want) * 2.0 ** -8 + product_error(av, wv, kind))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(1, 1 << 24), (33, 1 << 24), (1 << 22, 16)])
def test_the_largest_counts(gpu, rows, n):
    """As many output columns, and rows, as a call may have: sampled ones against float64."""
    g, k = gpu(32), 32
    gen = torch.Generator(device="cuda").manual_seed(5)
    words = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=gen)
    scales = torch.randint(120, 124, (n, 1), dtype=torch.uint8, device="cuda", generator=gen)
    a = torch.randint(0, 0x70, (rows, k), dtype=torch.uint8, device="cuda", generator=gen)          # finite E4M3 codes
    a_scales = torch.full((rows, 1), 120, dtype=torch.uint8, device="cuda")
    w, ws = (torch.empty(size, dtype=torch.uint8, device="cuda") for size in (g.lib.ca_mxfp4_words_bytes(n, k), g.lib.ca_mxfp4_scales_bytes(n, k)))
    p = native.ptr
    assert g.lib.ca_mxfp4_prepare(g.ctx, n, k, p(words), p(scales), p(w), p(ws), g.stream()) == 0
    out = torch.empty((rows, n), dtype=torch.bfloat16, device="cuda")
    g.linear(rows, n, k, a, a_scales, 0, (w, ws), out=out)
    r = torch.tensor(sorted({0, 1, rows // 2, rows - 2, rows - 1} & set(range(rows))))
    c = torch.cat([torch.arange(min(n, 40)), torch.randint(0, n, (200,), generator=torch.Generator().manual_seed(1)), torch.arange(n - min(n, 40), n)])
    av, wv = values8(a[r.cuda()], a_scales[r.cuda()], 32), values4(words[c.cuda()], scales[c.cuda()])
    got, want = f64(out[r.cuda()][:, c.cuda()]), av @ wv.T
    assert np.all(np.abs(got - want) <= np.abs(want) * 2.0 ** -8 + product_error(av, wv, 0))


@pytest.mark.gpu
def test_long_offsets(gpu):
    """Outputs past 2^32 bytes: the last rows of a wide activation buffer equal the same rows computed alone."""
    g = gpu(32)
    rows, n, k = 70000, 32768, 32
    a, a_scales, _ = activations(g, 0, 512, k)
    a, a_scales = a.repeat(137, 1)[:rows].contiguous(), a_scales.repeat(137, 1)[:rows].contiguous()
    w = g.prepare(*mxfp4("w", n, k, std=0.5))
    out = torch.empty((rows, n), dtype=torch.bfloat16, device="cuda")
    g.linear(rows, n, k, a, a_scales, 0, w, out=out)
    few = g.linear(100, n, k, a[-100:].contiguous(), a_scales[-100:].contiguous(), 0, w)
    assert rows * n * 2 > 2 ** 32 and torch.equal(out[-100:], few)
