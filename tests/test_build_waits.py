"""The build's check of waits around MFMAs of inline asm (build.check_waits), on short
listings and on the assembly of the kernels that it covers."""
import pytest
from test_build_checks import build  # noqa: F401  (the fixture)

M = "v_mfma_f32_32x32x16_f16 v[0:15], v[16:19], v[20:23], v[0:15]"
ACC = "v_mfma_f32_32x32x16_f16 a[0x10:0x1f], v[16:19], v[20:23], a[0x10:0x1f]"
OTHER = "v_mfma_f32_32x32x16_f16 v[40:55], v[16:19], v[20:23], 0"


@pytest.mark.parametrize("code", [
    [M, "v_mov_b32_e32 v60, v3"],                                    # read at once
    [M, "v_mov_b32_e32 v3, 0"],                                      # overwritten
    [M, "s_nop 15", "s_nop 1", "ds_write_b128 v60, v[12:15]"],       # 18 states
    [M, OTHER, OTHER, "s_nop 1", "v_max_f32_e32 v60, v0, v1"],       # 8 + 8 + 2
    [M, "s_cbranch_scc1 .LBB0_2", "s_nop 15", "s_nop 7", ".LBB0_2:", "v_mov_b32_e32 v60, v3"],
    [M, "s_branch .LBB0_3", ".LBB0_2:", "s_endpgm", ".LBB0_3:", "v_mov_b32_e32 v60, v3"],
    [ACC, "v_accvgpr_read_b32 v60, a17"],
    [M, "v_mfma_f32_32x32x16_f16 v[40:55], v[0:3], v[20:23], 0"],    # as an operand
    ["v_mov_b32_e32 v17, 0", M],                                     # written at once before
    ["v_mov_b32_e32 v17, 0", "s_nop 0", M],
    ["v_accvgpr_write_b32 a20, 0", ACC],
])
def test_too_close(build, code):  # noqa: F811
    with pytest.raises(RuntimeError, match="no wait between"):
        build.check_waits(code + ["s_endpgm"], "k")


@pytest.mark.parametrize("code", [
    [M, M, "s_nop 15", "s_nop 7", "v_mov_b32_e32 v60, v3"],
    [M, "s_nop 15", "s_nop 2", "ds_write_b128 v60, v[12:15]"],       # 19 states
    [M, OTHER, OTHER, OTHER, "v_max_f32_e32 v60, v0, v1"],
    [M, "s_cbranch_scc1 .LBB0_2", "s_nop 15", "s_nop 7", "v_mov_b32_e32 v60, v3", ".LBB0_2:",
     "s_endpgm"],
    [ACC, ACC, "v_mov_b32_e32 v60, v3"],
    ["v_mov_b32_e32 v17, 0", "s_nop 1", M],
    ["v_mov_b32_e32 v60, 0", M],
    [".LBB0_1:", M, "s_nop 15", "s_nop 2", "v_mov_b32_e32 v60, v3", "s_cbranch_scc1 .LBB0_1"],
])
def test_far_enough(build, code):  # noqa: F811
    build.check_waits(code + ["s_endpgm"], "k")


def test_the_tree_attention_kernels(build):  # noqa: F811
    import os

    name = "mla_tree.hip"
    src, path = os.path.join(build.CSRC, name), build.asm_path(name)
    if not os.path.exists(path) or os.path.getmtime(path) < os.path.getmtime(src):
        os.makedirs(build.BUILD_DIR, exist_ok=True)
        build._compile(src)
    asm = open(path).read()
    # the settling waits taken out of the listing, some read comes too early
    for kernel in build.OWN_AGPRS[name]:
        build.check_waits(build._body(asm, kernel)[1], kernel)
        lines = [x for x in build._body(asm, kernel)[1] if not x.strip().startswith("s_nop 15")
                 and not x.strip().startswith("s_nop 7")]
        with pytest.raises(RuntimeError, match="no wait between"):
            build.check_waits(lines, kernel)
