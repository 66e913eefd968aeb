"""The build's check of kernels with LDS reads and matrix products by inline assembly: on written-out assembly, right
and wrong."""
import re

import pytest

from pytorch_distributed_amd import _build
from pytorch_distributed_amd._asm_check import WAIT_STATES, early_products, kernels_with_lds_reads, unawaited_reads


def kernel(*lines, name="_Zkernel"):
    return "\t.text\n" + f"{name}: ; @{name}\n" + "\n".join(l if l.endswith(":") else "\t" + l for l in lines) + "\n.Lfunc_end0:\n\t.size x, 1\n"


READ = "ds_read_b128 v[4:7], v20 offset:16"
USE = "v_mfma_f32_32x32x16_bf16 a[0:15], v[4:7], v[8:11], a[0:15]"


def test_awaited_reads_pass():
    assert unawaited_reads(kernel(READ, "s_waitcnt lgkmcnt(0)", USE, "s_endpgm")) == []
    # two younger reads may stay in flight
    assert unawaited_reads(kernel(READ, "ds_read_b64 v[30:31], v20", "ds_read_u8 v32, v21", "s_waitcnt vmcnt(3) lgkmcnt(2)", USE, "s_endpgm")) == []
    # a read may overwrite its own address
    assert unawaited_reads(kernel("ds_read_b128 v[4:7], v6", "s_waitcnt lgkmcnt(0)", USE, "s_endpgm")) == []
    # a scalar load in between only makes the wait stricter
    assert unawaited_reads(kernel(READ, "s_load_dword s4, s[0:1], 0x0", "ds_read_b64 v[30:31], v20", "s_waitcnt lgkmcnt(1)", USE, "s_endpgm")) == []


@pytest.mark.parametrize("touch", [USE, "v_mov_b32_e32 v40, v7", "v_accvgpr_write_b32 a3, v4", "scratch_store_dwordx4 off, v[4:7], off",
                                   "v_mov_b32_e32 v5, 0", "ds_write_b128 v20, v[4:7]", "global_load_dword v6, v[50:51], off",
                                   "ds_read_b128 v[40:43], v5"])
def test_a_touch_before_the_wait_is_found(touch):
    bad = unawaited_reads(kernel(READ, touch, "s_waitcnt lgkmcnt(0)", USE, "s_endpgm"))
    assert len(bad) == 1 and bad[0].startswith("_Zkernel:4: " + touch.split()[0])
    assert unawaited_reads(kernel(READ, "s_waitcnt lgkmcnt(0)", touch, "s_endpgm")) == []


def test_a_wait_that_is_too_weak_is_found():
    younger = ["ds_read_b64 v[30:31], v20"]
    assert unawaited_reads(kernel(READ, *younger, "s_waitcnt lgkmcnt(2)", USE, "s_endpgm"))
    assert unawaited_reads(kernel(READ, *younger, "s_waitcnt vmcnt(0)", USE, "s_endpgm"))
    assert unawaited_reads(kernel(READ, "s_waitcnt lgkmcnt(15)", USE, "s_endpgm"))
    assert unawaited_reads(kernel(READ, *["ds_write_b32 v1, v2"] * 20, "s_waitcnt lgkmcnt(15)", USE, "s_endpgm")) == []


def test_every_path_counts():
    # awaited on one side of a branch only
    assert unawaited_reads(kernel(READ, "s_cbranch_scc1 .L1", "s_waitcnt lgkmcnt(0)", ".L1:", USE, "s_endpgm"))
    assert unawaited_reads(kernel(READ, "s_cbranch_scc1 .L1", "s_waitcnt lgkmcnt(0)", "s_branch .L2", ".L1:", "s_waitcnt lgkmcnt(0)", ".L2:", USE, "s_endpgm")) == []
    # around a loop: the read at its end is used at its start
    loop = lambda wait: kernel(READ, "s_waitcnt lgkmcnt(0)", ".L1:", *wait, USE, READ, "s_cbranch_scc1 .L1", "s_endpgm")  # noqa: E731
    assert unawaited_reads(loop([])) and unawaited_reads(loop(["s_waitcnt lgkmcnt(0)"])) == []
    # the other way round a loop has fewer younger operations behind the read
    assert unawaited_reads(kernel(READ, "ds_write_b32 v1, v2", ".L1:", "s_waitcnt lgkmcnt(1)", USE, READ, "s_cbranch_scc1 .L1", "s_endpgm"))


def test_kernels_are_told_apart():
    two = kernel(READ, USE, "s_endpgm", name="_Za") + kernel("v_mov_b32_e32 v4, 0", "s_endpgm", name="_Zb")
    assert [f.split(":")[0] for f in unawaited_reads(two)] == ["_Za"] and kernels_with_lds_reads(two) == ["_Za"]


def test_the_build_refuses():
    fine = kernel(READ, "s_waitcnt lgkmcnt(0)", USE, "s_endpgm")
    remark = "a.hip:3:1: remark: Function Name: _Zkernel [x]\na.hip:3:1: remark:     VGPRs Spill: {} [x]\na.hip:3:1: remark:     ScratchSize [bytes/lane]: 0 [x]\n"
    _build.check_hand_reads("fp8_gemm.hip", remark.format(0), fine)
    with pytest.raises(RuntimeError, match="spill registers do: _Zkernel"):  # into accumulator registers: no scratch
        _build.check_hand_reads("fp8_gemm.hip", remark.format(3), fine)
    with pytest.raises(RuntimeError, match="no kernel named"):
        _build.check_hand_reads("fp8_gemm.hip", "", fine)
    with pytest.raises(RuntimeError, match="no kernel with LDS reads"):
        _build.check_hand_reads("gemm_fused.hip", "", "")
    with pytest.raises(RuntimeError, match="before the LDS read of them is awaited"):
        _build.check_hand_reads("gemm_fused.hip", "", kernel(READ, USE, "s_endpgm"))
    with pytest.raises(RuntimeError, match="before the matrix product into them is done"):
        _build.check_hand_reads("gemm_fused.hip", "", kernel(READ, "s_waitcnt lgkmcnt(0)", *INLINE, "v_accvgpr_read_b32 v2, a15", "s_endpgm"))


INLINE = [";;#ASMSTART", "v_mfma_f32_32x32x16_bf16 a[0:15], v[4:7], v[8:11], a[0:15]", ";;#ASMEND"]


@pytest.mark.parametrize("touch", ["v_accvgpr_read_b32 v2, a15", "v_accvgpr_mov_b32 a40, a3", "v_accvgpr_write_b32 a0, 0", "buffer_store_dwordx4 a[12:15], v0, s[0:3], 0 offen",
                                   "v_mfma_f32_32x32x16_bf16 a[16:31], a[0:3], v[8:11], a[16:31]"])
def test_a_product_touched_too_early_is_found(touch):
    fill = ["v_add_u32_e32 v40, v41, v42"] * (WAIT_STATES - 17)
    assert len(early_products(kernel(*INLINE, "s_nop 15", *fill[:-1], touch, "s_endpgm"))) == 1
    assert early_products(kernel(*INLINE, "s_nop 15", *fill, "s_nop 0", touch, "s_endpgm")) == []
    # on one path
    assert len(early_products(kernel(*INLINE, "s_cbranch_scc1 .L1", "s_nop 15", "s_nop 15", ".L1:", touch, "s_endpgm"))) == 1
    # around a loop
    assert len(early_products(kernel(".L1:", touch, *INLINE, "s_cbranch_scc1 .L1", "s_endpgm"))) == 1


def test_products_into_one_accumulator_follow_each_other():
    assert early_products(kernel(*INLINE, *INLINE, "s_nop 15", "s_nop 15", "v_accvgpr_read_b32 v2, a15", "s_endpgm")) == []
    # a product that the compiler issued itself is its own business
    assert early_products(kernel(INLINE[1], "v_accvgpr_read_b32 v2, a15", "s_endpgm")) == []


def test_every_source_with_such_assembly_is_checked():
    read = re.compile(r'asm volatile\("[^"]*(ds_(read|load|bpermute)|v_mfma)')
    kernels = _build.CSRC / "kernels"
    headers = [h.name for h in kernels.glob("*.h") if read.search(h.read_text())]
    for src in sorted(kernels.glob("*.hip")):
        text = src.read_text()
        if read.search(text) or any(f'#include "{h}"' in text for h in headers):
            assert src.name in _build.HAND_READS, src.name
