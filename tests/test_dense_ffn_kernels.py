"""Every kernel of the products with MXFP4 weights runs here: one call at least for each instantiation in the built library, its operands whole numbers
times powers of two whose sums FP32 holds exactly, so that each row, column, block scale and k-step shows in the result.

Which kernel a call runs is asked of the rule that the library itself goes by (csrc/mxfp4_choice.hpp)."""
import ctypes
import importlib
import os
import re
import subprocess

import numpy as np
import pytest
import torch

from helpers import native
from test_dense_ffn import LIMIT, Gpu, f64, quant8

listing = importlib.import_module("titanic-flash-41_amd.listing")
CSRC = os.path.join(os.path.dirname(native.KERNEL_LIB), "csrc")
CUS = 256

FEW = {0: (1, 1), 1: (2, 1), 2: (2, 4)}                                                 # MX_FEW_*: CT, NW
TILES = {3: (1, 2, 2, 2), 4: (1, 4, 4, 1), 5: (4, 4, 2, 2), 6: (8, 8, 2, 2), 7: (4, 4, 1, 4)}      # MX_TILE_*: FM, FT, WM, WN

# Rows and output columns that reach each size of kernel, ragged both ways.  Columns of a gated product with codes are a multiple of their block.
LINEAR_SIZES = [(1, 100), (16, 4204), (32, 100), (29, 4203), (40, 101), (531, 2300), (1090, 2100), (3490, 3490), (3490, 3488)]
GATED_SIZES = [(3, 128), (16, 4224), (40, 128), (531, 1152), (1090, 1152), (3490, 1792)]
# A whole number of rounds of four k-steps, of k-steps, neither; long and within a round.
LENGTHS = {32: [1536, 512, 1664, 384, 1568, 96], 128: [1536, 512, 1664, 384]}
OUTPUTS = [("act",), ("codes",), ("act", "codes"), ("act", "e2m1"), ("e2m1",)]


# (kind, block, rows, n) and the k each runs with; several tiles a persistent workgroup come last, whose first round of k-steps may be its last
LINEAR = [(kind, block, rows, n, LENGTHS[block]) for kind, block in ((0, 32), (0, 128), (1, 32)) for rows, n in LINEAR_SIZES] + [(1, 32, 8190, 4088, [512, 384, 640])]
GATED = [(kind, block, rows, n, LENGTHS[block if kind == 0 else 32]) for kind, block in ((0, 32), (0, 128), (1, 32), (1, 128)) for rows, n in GATED_SIZES]


def outputs_at(i):
    """Every form of the outputs at a group's long k, one at its short ones."""
    return OUTPUTS if i % 2 == 0 else OUTPUTS[2:3]


def calls():
    for gated, groups in ((False, LINEAR), (True, GATED)):
        for kind, block, rows, n, lengths in groups:
            for i, k in enumerate(lengths):
                for outputs in outputs_at(i) if gated else [()]:
                    yield dict(kind=kind, block=block, rows=rows, n=n, k=k, gated=gated, outputs=outputs)


class Call(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_int), ("n", ctypes.c_int), ("k", ctypes.c_int), ("cus", ctypes.c_int), ("fp4_rows", ctypes.c_bool), ("gated", ctypes.c_bool),
                ("block_shift", ctypes.c_int), ("a_scales", ctypes.c_size_t), ("wide", ctypes.c_int), ("out_stride", ctypes.c_longlong), ("act", ctypes.c_bool),
                ("codes", ctypes.c_bool), ("out_block", ctypes.c_int)]


class Choice(ctypes.Structure):
    _fields_ = [("kernel", ctypes.c_int), ("scales", ctypes.c_int), ("codes_apart", ctypes.c_bool)]


@pytest.fixture(scope="module")
def choose(tmp_path_factory):
    folder = tmp_path_factory.mktemp("choice")
    (folder / "choice.cpp").write_text('#include "mxfp4_choice.hpp"\nextern "C" MxChoice choose(MxCall c) { return tf_mx_choose(c); }\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, str(folder / "choice.cpp"), "-o", str(folder / "choice.so")], check=True)
    lib = ctypes.CDLL(str(folder / "choice.so"))
    lib.choose.argtypes, lib.choose.restype = [Call], Choice

    def ask(kind, block, rows, n, k, gated, outputs, misaligned=0):
        codes = "codes" in outputs or "e2m1" in outputs
        return lib.choose(Call(rows, n, k, CUS, kind == 1, gated, 7 if kind == 0 and block == 128 else 5, 4096 + misaligned, 2 if n % 8 == 0 else 1 if n % 4 == 0 else 0, n,
                               "act" in outputs, codes, (32 if "e2m1" in outputs else block) if codes else 0))
    return ask


def kernel_of(call, choice):
    flags = (call["kind"] == 1, call["gated"])
    if choice.kernel in FEW:
        ct, nw = FEW[choice.kernel]
        return ("tf_mx_stream", *map(int, flags), ct, 2 if not call["gated"] and call["rows"] > 16 else 1, nw)
    return ("tf_mx_gemm", *map(int, flags), choice.scales, *TILES[choice.kernel])


def built_kernels():
    found = set()
    for image in listing.device_images(native.KERNEL_LIB):
        for symbol in re.findall(r"_Z\d+tf_mx_(?:gemm|stream)I\w+", image.decode("latin-1")):
            name, values = re.match(r"_Z\d+(tf_mx_(?:gemm|stream))I((?:L[bi]\d+E)+)E", symbol).groups()
            values = [int(v) for v in re.findall(r"L[bi](\d+)E", values)]
            found.add((name, *(values[:7] if name == "tf_mx_gemm" else values[:5])))
    return found


def test_every_kernel_in_the_library_is_run_below(choose):
    """And no kernel is there that no call reaches."""
    run = {kernel_of(c, choose(**c)) for c in calls()}
    built = built_kernels()
    assert len(built) == 65 + 14 and run == built, (sorted(built - run), sorted(run - built))


def test_alignment_of_the_rows_scales_chooses_how_they_come(choose):
    def scales(block, k, off):
        return choose(0, block, 64, 64, k, False, (), off).scales
    assert [scales(32, 512, off) for off in (0, 4, 1)] == [0, 2, 4] and [scales(32, 128, off) for off in (0, 2)] == [2, 4]
    assert [scales(128, 512, off) for off in (0, 4, 2)] == [1, 1, 3] and scales(128, 128, 0) == 3 and scales(32, 96, 0) == 4


# ---- on the GPU ----------------------------------------------------------------------------------------------------------

GRID = [-1.0, 0.0, 0.0, 0.0, 1.0, 0.5, -2.0, 0.0]
E2M1_CODES = [10, 0, 0, 0, 2, 1, 12, 0]


def whole(kind, block, rows, k, seed, shift=0):
    """Codes (or words), scale bytes and float64 values: -2 .. 1 times 2^0 .. 2^3 a block, times 2^shift.  Products of two such are multiples of 2^-2
    of magnitude 2^8 at most: 1,664 of them sum to less than 2^19, so FP32 holds every partial sum."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pick = torch.randint(0, len(GRID), (rows, k), generator=gen, device="cuda")
    values = torch.tensor(GRID, device="cuda")[pick]
    if kind == 1:
        codes = torch.tensor(E2M1_CODES, dtype=torch.uint8, device="cuda")[pick]
        codes = codes[:, 0::2] | (codes[:, 1::2] << 4)
    else:
        codes = values.to(torch.float8_e4m3fn).view(torch.uint8)
    scales = 127 + torch.randint(0, 4, (rows, k // block), generator=gen, device="cuda")
    power = ((scales - 127 + shift + 1023) << 52).view(torch.float64)          # by its bits: the device's pow is not exact
    values = values.double() * power.repeat_interleave(block, dim=1)
    return codes.contiguous(), (scales + shift).to(torch.uint8), values


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


def rounded(v):
    return v.to(torch.float32).to(torch.bfloat16)          # (the float64 values here are FP32 values)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,block,rows,n,lengths", LINEAR)
def test_linear_is_exact(gpu, kind, block, rows, n, lengths):
    g = gpu(block)
    for k in lengths:
        a, a_scales, av = whole(kind, block if kind == 0 else 32, rows, k, 1)
        words, scales, wv = whole(1, 32, n, k, 2)
        out = g.linear(rows, n, k, a, a_scales, kind, g.prepare(words, scales))
        assert torch.equal(out, rounded(av @ wv.t().contiguous())), k


@pytest.mark.gpu
@pytest.mark.parametrize("kind,block,rows,n,lengths", GATED)
def test_swiglu_is_exact_but_for_its_function(gpu, kind, block, rows, n, lengths):
    """The two sums are exact; what is left is the activation's own FP32 chain (swiglu_want in test_dense_ffn.py), one rounding, and the codes of the
    rounded value, whichever outputs are asked for."""
    g = gpu(block)
    for i, k in enumerate(lengths):
        a, a_scales, av = whole(kind, block if kind == 0 else 32, rows, k, 3)
        (uw, us, uv), (gw, gs, gv) = whole(1, 32, n, k, 4, shift=-7), whole(1, 32, n, k, 5, shift=-7)
        up, gate = g.prepare(uw, us), g.prepare(gw, gs)
        gc, uc = (av @ gv.t().contiguous()).clamp(max=LIMIT), (av @ uv.t().contiguous()).clamp(-LIMIT, LIMIT)
        want = gc / (1.0 + torch.exp(-gc)) * uc
        act = g.swiglu(rows, n, k, a, a_scales, kind, up, gate, codes=False)[0]
        assert bool(((act.double() - want).abs() <= want.abs() * (2.0 ** -8 + (gc.abs() + 4) * 2.0 ** -23)).all()), k
        codes, bytes_ = quant8(f64(act), block)
        codes, bytes_ = torch.from_numpy(codes).to(torch.float8_e4m3fn).view(torch.uint8).cuda(), torch.from_numpy(bytes_).cuda()
        words, word_scales = g.quant(act)
        for outputs in outputs_at(i):
            e2m1 = "e2m1" in outputs
            h, c, s = g.swiglu(rows, n, k, a, a_scales, kind, up, gate, out_kind=int(e2m1), act="act" in outputs, codes=e2m1 or "codes" in outputs)
            assert h is None or torch.equal(h, act), (k, outputs)
            if e2m1:
                assert torch.equal(c, words) and torch.equal(s, word_scales), (k, outputs)
            elif c is not None:
                assert torch.equal(s, bytes_) and torch.equal(c.view(torch.float8_e4m3fn).float(), codes.view(torch.float8_e4m3fn).float()), (k, outputs)


@pytest.mark.gpu
@pytest.mark.parametrize("block,off,k", [(32, 4, 1536), (32, 1, 1536), (32, 2, 384), (128, 1, 1536), (128, 4, 1536)])
@pytest.mark.parametrize("rows", [5, 70])
def test_rows_scales_at_any_address(gpu, block, off, k, rows):
    g, n = gpu(block), 100
    a, a_scales, av = whole(0, block, rows, k, 6)
    words, scales, wv = whole(1, 32, n, k, 7)
    buffer = torch.full((a_scales.numel() + off + 64,), 255, dtype=torch.uint8, device="cuda")       # NaN scales either side
    moved = buffer[off:off + a_scales.numel()].view_as(a_scales)
    moved.copy_(a_scales)
    assert moved.data_ptr() % 16 == off
    out = g.linear(rows, n, k, a, moved, 0, g.prepare(words, scales))
    assert torch.equal(out, rounded(av @ wv.t().contiguous()))
