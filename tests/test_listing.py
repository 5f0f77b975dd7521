"""The check of the many-row products' machine code: the built library passes it, and a listing that breaks a rule does not."""
import importlib

import pytest

from helpers import native

listing = importlib.import_module("titanic-flash-41_amd.listing")

PRODUCT = "v_mfma_scale_f32_16x16x128_f8f6f4 a[%d:%d], v[0:3], v[4:7], a[%d:%d], v8, v9 op_sel_hi:[0,0,0] cbsz:4 blgp:4"


def product(acc):
    return PRODUCT % (acc, acc + 3, acc, acc + 3)


def code_of(*lines):
    """A kernel of these instructions, four bytes each; a branch names the place of its target."""
    text = ["0000000000001000 <_Z10tf_mx_gemm_x>:"]
    for i, line in enumerate(lines):
        target = " <_Z10tf_mx_gemm_x+0x%x>" % (4 * int(line.split()[1])) if line.startswith(("s_branch", "s_cbranch")) else ""
        text.append("\t%s // %012X: 00000000%s" % (line, 0x1000 + 4 * i, target))
    (code,) = listing.kernels("\n".join(text)).values()
    assert len(code) == len(lines)
    return listing.faults(code)


def test_the_built_library_keeps_the_rules():
    images = [listing.kernels(listing.disassemble(i)) for i in listing.device_images(native.KERNEL_LIB)]
    found = {name: code for image in images for name, code in image.items()}
    assert len(found) > 60 and listing.check(native.KERNEL_LIB) == len(found)
    for name, code in found.items():
        # a round of four k-steps: products, requests and waits are recognised
        assert sum(c.product for c in code) % 8 == 0 and any(c.product for c in code), name
        assert sum(c.request for c in code) >= 10 and any("m0" in c.operands[0] for c in code if c.operands), name


CLEAN = ["s_mov_b32 m0, s4", "s_nop 0", "global_load_lds_dwordx4 v1, s[6:7] offset:1024", product(0), product(4), "s_nop 15", "v_accvgpr_read_b32 v20, a0", "s_endpgm"]


def test_a_clean_listing():
    assert code_of(*CLEAN) == []
    assert code_of(product(0), "s_nop 11", "v_accvgpr_read_b32 v20, a3") == []
    assert code_of("v_mov_b32_e32 v4, v5", "s_nop 1", product(0)) == []
    assert code_of(product(0), "v_accvgpr_read_b32 v20, a4") == []                       # another sum
    assert code_of("v_readfirstlane_b32 s6, v0", "s_nop 4", "global_load_lds_dwordx4 v1, s[6:7]") == []


@pytest.mark.parametrize("rule,lines", [
    ("sums", [product(0), "s_nop 10", "v_accvgpr_read_b32 v20, a3"]),
    ("sums", [product(0), product(4), "v_accvgpr_write_b32 a2, v20"]),
    ("sums", [product(0), "s_nop 7", "v_accvgpr_mov_b32 a9, a1"]),
    ("sums", [product(0), "global_store_dwordx4 v[0:1], a[0:3], off"]),
    # around a loop: the product at its end, the copy at its top
    ("sums", ["v_accvgpr_read_b32 v20, a0", "s_nop 3", product(0), "s_nop 5", "s_cbranch_scc1 0", "s_endpgm"]),
    ("operands", ["v_mov_b32_e32 v5, v50", "s_nop 0", product(0)]),
    ("operands", ["v_perm_b32 v8, v20, v21, v22", product(0)]),
    ("operands", ["v_accvgpr_write_b32 a0, 0", product(0)]),
    ("operands", ["v_permlane32_swap_b32_e32 v60, v8", product(0)]),
    ("requests", ["v_readfirstlane_b32 s7, v0", "s_nop 3", "global_load_lds_dwordx4 v1, s[6:7]"]),
    ("requests", ["s_mov_b32 m0, s4", "global_load_lds_dwordx4 v1, s[6:7]"]),
    ("requests", ["s_add_i32 m0, s4, 16", "s_nop 0", "global_load_lds_dwordx4 v1, s[6:7]"]),
    ("counting", ["global_load_dword v1, v[2:3], off"]),
    ("counting", ["scratch_store_dword off, v1, s32"]),
    ("counting", ["buffer_load_dword v1, off, s[0:3], 0"]),
    ("stores", ["buffer_store_dwordx4 v[0:3], v4, s[0:3], 0 offen"] * 31),
    ("stores", ["buffer_store_dwordx4 v[0:3], v4, s[0:3], 0 offen"] * 32 + ["global_store_dword v[0:1], v2, off"]),
])
def test_what_breaks_a_rule(rule, lines):
    found = code_of(*lines)
    assert found and all(f.startswith(rule + ":") for f in found), found
