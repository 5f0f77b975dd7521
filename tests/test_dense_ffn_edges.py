"""The dense feed-forward operators at the ends of what their calls allow: alignment, the range of the norm's statistics, kernels that only some
sizes reach, results of a row in calls of different row counts.  References as in test_dense_ffn.py."""
import ctypes

import numpy as np
import pytest
import torch

from helpers import native, synth
from test_dense_ffn import Gpu, activations, f64, fake_context, mxfp4, norm_want, normal, product_error, quant8, swiglu_want, values4


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


def test_scales_of_prepared_weights_lie_at_16_bytes():
    """The many-row products copy them into LDS sixteen bytes a lane, so every call that writes or reads them asks for that alignment.  Addresses
    are never followed."""
    lib, memory = native.load(), fake_context()
    ctx, P, Q, i64 = ctypes.addressof(memory), 1 << 20, 1 << 21, ctypes.c_int64
    for off in (4, 8, 12):
        assert lib.ca_mxfp4_prepare(ctx, 16, 64, P, P, Q, Q + off, None) == -1
        assert lib.ca_mxfp4_linear(ctx, 64, 16, 256, P, P, 0, P, P + off, P, i64(16), None) == -1
        assert lib.ca_mxfp4_swiglu(ctx, 64, 256, 256, P, P, 0, P, P + off, P, P, P, P, P, 0, None) == -1
        assert lib.ca_mxfp4_swiglu(ctx, 64, 256, 256, P, P, 0, P, P, P, P + off, P, P, P, 0, None) == -1


# ---- the norm's statistics --------------------------------------------------------------------------------------------------

# every variant of waves and pieces a row, few rows and many
NORM_SHAPES = [(9, 384), (9, 1024), (9, 2048), (9, 4096), (9, 8192), (520, 1024), (520, 4096), (520, 8192)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
@pytest.mark.parametrize("eps", [0.0, 1e-38, 1e-6, 1e30])
def test_norm_of_rows_whose_squares_leave_fp32(gpu, rows, cols, eps):
    """Rows of every size that BF16 has: the squares of the large ones pass FP32's range, those of the small ones vanish in it (which shows where
    eps is as small).  Each is the formula's value; the rows between are what they are alone."""
    g = gpu(32)
    x = normal("edges/norm", rows, cols).to(torch.float64)
    sizes = [2.0 ** 125, 2.0 ** 100, 2.0 ** 66, 2.0 ** 61, 2.0 ** -40, 2.0 ** -62, 2.0 ** -80, 2.0 ** -110, 1.0]
    x *= torch.tensor([sizes[i % len(sizes)] for i in range(rows)], dtype=torch.float64)[:, None]
    x[0, 5], x[1, 7], x[1, 8] = 2.0 ** 127 * 1.5, 2.0 ** -126, 2.0 ** -60
    x = x.to(torch.bfloat16).cuda()
    w = (1.0 + normal("edges/norm-w", cols, std=0.2)).to(torch.bfloat16).cuda()
    r, n, c, s, _, _ = g.norm(x, None, w, eps=eps, minimum=False)
    assert torch.equal(r, x)
    want = norm_want(x, None, w, float(np.float32(eps)))[1]
    # Half a BF16 step (2^-134 where the result is subnormal) beside the FP32 chain of test_add_norm_quant, to which subnormal products add half of
    # FP32's least value, 2^-150, each: the first times a weight below 2, and the second, less than 2^-148 in all.  The two add up: a value
    # of 2^-134 (1 + 5.8e-6) comes out of the chain as the tie 2^-134, within 2^-149 of it, and goes to the even zero.
    assert float(w.abs().max()) < 2
    chain = np.abs(want) * (48 * 2.0 ** -24) + np.where(np.abs(want) < 2.0 ** -124, 2.0 ** -148, 0.0)
    assert np.all(np.abs(f64(n) - want) <= np.maximum(np.abs(want) * 2.0 ** -8, 2.0 ** -134) + chain)
    ordinary = np.abs(f64(n)).reshape(rows, -1, 32).max(axis=2).min(axis=1) > 2.0 ** -100      # (blocks below E4M3's scales have codes of their own)
    codes, bytes_ = quant8(f64(n)[ordinary], 32)
    assert ordinary[0] and np.array_equal(s.cpu().numpy()[ordinary], bytes_)
    assert np.array_equal(c.cpu().view(torch.float8_e4m3fn).to(torch.float64).numpy()[ordinary], codes)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_norm_of_rows_that_are_not_finite(gpu, rows, cols):
    """A NaN anywhere and an infinity at its own place stay NaN, and nothing else of the call changes; a sum past BF16's range is an infinity."""
    g = gpu(32)
    x = normal("edges/norm", rows, cols).to(torch.bfloat16).cuda()
    res = normal("edges/norm-r", rows, cols).to(torch.bfloat16).cuda()
    w = torch.ones(cols, dtype=torch.bfloat16, device="cuda")
    clean = g.norm(x, res, w, minimum=False)
    bad, other = x.clone(), res.clone()
    bad[2, cols - 1], bad[4, 3], bad[6, 9], other[6, 9] = float("nan"), -float("inf"), 3e38, 3e38
    r, n, c, s, _, _ = g.norm(bad, other, w, minimum=False)
    keep = [i for i in range(rows) if i not in (2, 4, 6)]
    assert all(torch.equal(a[keep], b[keep]) for a, b in zip(clean[:4], (r, n, c, s)))
    assert bool(torch.isnan(n[2]).all()) and bool(torch.isnan(n[4, 3])) and bool(torch.isinf(r[6, 9])) and bool(torch.isnan(n[6, 9]))


# ---- the ends of the quantizer's range ----------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_blocks_at_the_ends_of_the_range(gpu, dtype):
    """As the header has it, and the generator of the experts' weights: a block below 2^-126 is a zero block, one past 2^123 saturates."""
    g = gpu(32)
    largest = [2.0 ** -133, 2.0 ** -128, 2.0 ** -127, 2.0 ** -126 * (1 - 2.0 ** -7), 2.0 ** -126, 2.0 ** -125, 2.0 ** -124, 2.0 ** 122 * 1.75, 2.0 ** 123, 2.0 ** 127 * 1.5]
    x = torch.zeros(len(largest), 32, dtype=torch.float64)
    x[:, 3] = torch.tensor(largest, dtype=torch.float64)
    x[:, 20], x[:, 21] = -x[:, 3], x[:, 3] / 2
    x = x.to(dtype)
    words, scales = g.quant(x.cuda())
    assert scales.flatten().tolist() == [127, 127, 127, 127, 1, 1, 1, 247, 247, 247]
    back = f64(g.dequant(words, scales, 2))
    assert not back[:4].any()
    assert back[4:7, 3].tolist() == largest[4:7]
    assert np.array_equal(back[7:, 3], [6 * 2.0 ** 120] * 3) and np.array_equal(back[:, 20], -back[:, 3])
    generated = synth.quantize_mxfp4(x.float())                      # (whose zero blocks keep the signs of their zeros)
    assert np.array_equal(values4(words, scales), values4(*generated)) and torch.equal(scales.cpu(), generated[1]) and not bool(words[:4].any())


# ---- a row in calls of different row counts ------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("cols", [384, 1024, 2048, 4096, 8192])
def test_a_row_alone_and_among_many(gpu, cols):
    """Few rows and many are summed in different orders, so a row's BF16 values may differ by a rounding (never its residual): each is within half a
    step and the chain of the formula's, so they are within two of that of each other."""
    g = gpu(32)
    rows = 600
    x, res = normal("edges/x", rows, cols).to(torch.bfloat16).cuda(), normal("edges/r", rows, cols).to(torch.bfloat16).cuda()
    w = (1.0 + normal("edges/norm-w", cols, std=0.2)).to(torch.bfloat16).cuda()
    many = g.norm(x, res, w, minimum=False)
    for at in (0, 7, rows - 1):
        one = g.norm(x[at:at + 1], res[at:at + 1], w, minimum=False)
        assert torch.equal(one[0][0], many[0][at])
        a, b = f64(one[1][0]), f64(many[1][at])
        assert np.all(np.abs(a - b) <= np.abs(b) * (1 + 2.0 ** -7) * 2 * (2.0 ** -8 + 48 * 2.0 ** -24)) and np.mean(a != b) < 1e-2


@pytest.mark.gpu
@pytest.mark.parametrize("kind,block", [(0, 32), (0, 128), (1, 32)])
def test_a_token_in_a_small_and_a_large_batch(gpu, kind, block):
    """The same row through every regime of the products: the streaming kernels, and each size of tile."""
    g = gpu(block)
    n, k = 1152, 1664
    a, a_scales, av = activations(g, kind, 4500, k, std=2.0)
    ups, gates = mxfp4("up", n, k, std=0.1), mxfp4("gate", n, k, std=0.1)
    up, gate = g.prepare(*ups), g.prepare(*gates)
    uv, gv = values4(*ups), values4(*gates)
    want, bound = av[:4] @ uv.T, product_error(av[:4], uv, kind)
    h_want, h_bound = swiglu_want(av[:4], uv, gv, kind)
    for rows in (4, 16, 30, 60, 400, 1100, 4500):
        out = f64(g.linear(rows, n, k, a[:rows], a_scales[:rows], kind, up)[:4])
        assert np.all(np.abs(out - want) <= np.abs(want) * 2.0 ** -8 + bound), rows
        h = f64(g.swiglu(rows, n, k, a[:rows], a_scales[:rows], kind, up, gate)[0][:4])
        assert np.all(np.abs(h - h_want) <= np.abs(h_want) * 2.0 ** -8 + h_bound), rows


# ---- captured, beside other work ---------------------------------------------------------------------------------------------

@pytest.mark.gpu
def test_two_launches_and_persistent_workgroups_captured_beside_each_other(gpu):
    """A gated product whose codes are a launch of their own, and a product of several tiles a workgroup, in graphs on two streams that run at once: every
    replay gives the eager bits of its new rows."""
    g, p = gpu(128), native.ptr
    n, k, rows, wide, many = 1152, 640, 60, 4088, 8190
    up, gate = g.prepare(*mxfp4("up", n, k, std=0.1)), g.prepare(*mxfp4("gate", n, k, std=0.1))
    w = g.prepare(*mxfp4("w", wide, 512))
    a, a_scales, _ = activations(g, 0, rows, k, std=2.0)
    b, b_scales, _ = activations(g, 1, many, 512)
    e = lambda *shape, dtype=torch.uint8: torch.empty(shape, dtype=dtype, device="cuda")
    sets = [(e(rows, n, dtype=torch.bfloat16), e(rows, n), e(rows, n // 128), e(many, wide, dtype=torch.bfloat16)) for _ in range(2)]

    def gated(out):
        assert g.lib.ca_mxfp4_swiglu(g.ctx, rows, n, k, p(a), p(a_scales), 0, p(up[0]), p(up[1]), p(gate[0]), p(gate[1]), p(out[0]), p(out[1]), p(out[2]), 0, g.stream()) == 0

    def product(out):
        assert g.lib.ca_mxfp4_linear(g.ctx, many, wide, 512, p(b), p(b_scales), 1, p(w[0]), p(w[1]), p(out[3]), wide, g.stream()) == 0

    streams, graphs = [torch.cuda.Stream() for _ in range(2)], [torch.cuda.CUDAGraph() for _ in range(2)]
    torch.cuda.synchronize()
    for call, stream, graph in zip((gated, product), streams, graphs):
        with torch.cuda.graph(graph, stream=stream):
            for _ in range(3):
                call(sets[0])
    for i in range(4):
        a.copy_(a.roll(7 * i + 1, 0).clone())
        b.copy_(b.roll(13 * i + 1, 0).clone())
        for t in sets[0]:
            t.view(torch.uint8).fill_(0x11)
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        gated(sets[1])
        product(sets[1])
        torch.cuda.synchronize()
        for got, want in zip(*sets):
            assert torch.equal(got.view(torch.uint8), want.view(torch.uint8)), i
