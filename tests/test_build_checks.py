"""The build's check of kernels that hold sums in accumulator registers by name: what it finds in assembly, that this tree's
has none of it, and that a source that keeps a value of the compiler's in one does not build."""
import shutil

import pytest

from xgen_amd import _build

OWN = """
	.amdhsa_accum_offset 256
_ZN4xgen6kernelE:                       ; a[0:3] in a comment
	v_mfma_scale_f32_32x32x64_f8f6f4 a[0:15], v[0:3], v[4:7], a[0:15], v8, v9 op_sel_hi:[0,0,0] cbsz:4 blgp:4
	;;#ASMSTART
	v_accvgpr_read_b32 v12, a[3]
	v_accvgpr_read_b32 v13, a4
	s_add_u32 s0, s1, alpha@rel32@lo+4
	v_add_f32_e32 v12, v12, v13
	s_cbranch_scc1 .LBB0_a1
"""


def test_the_statements_own_uses():
    assert _build.foreign_accumulators(OWN) == []


@pytest.mark.parametrize("line", ["v_accvgpr_write_b32 a7, v3", "v_accvgpr_mov_b32 a1, a2", "ds_read_b128 a[4:7], v1", "buffer_load_dword a255, v1, s[0:3], 0 offen",
                                  "global_store_dwordx4 v[0:1], a[8:11], off", "scratch_store_dword off, v1, s32", "v_mov_b32_e32\tv1, a9"])
def test_foreign_uses(line):
    assert _build.foreign_accumulators(OWN + "\t" + line + "\n") == [line]


needs_hipcc = pytest.mark.skipif(shutil.which("hipcc") is None, reason="needs hipcc")


@needs_hipcc
def test_sources_of_this_tree(tmp_path, monkeypatch):
    monkeypatch.setattr(_build, "OBJ_DIR", tmp_path)
    names = {p.stem for p in _build.CSRC.glob("*.hip")}
    assert _build.NAMED_ACCUMULATORS <= names
    for stem in _build.NAMED_ACCUMULATORS:
        _build._check_accumulators(_build.CSRC / f"{stem}.hip")


@needs_hipcc
def test_a_source_whose_values_share_them_does_not_build(tmp_path, monkeypatch):
    """More values than the vector registers hold: the compiler keeps some in accumulators."""
    monkeypatch.setattr(_build, "OBJ_DIR", tmp_path)
    src = tmp_path / "crowded.hip"
    src.write_text("""#include <hip/hip_runtime.h>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(1, 1))) void k(float *p, const int *at) {
  float v[300];
#pragma unroll
  for (int i = 0; i < 300; ++i) v[i] = p[at[i] + threadIdx.x];
  asm volatile("v_mfma_f32_32x32x2_f32 a[0:15], %0, %1, 0" :: "v"(v[0]), "v"(v[1]));
#pragma unroll
  for (int i = 0; i < 300; ++i) p[at[299 - i] + threadIdx.x] = v[i] * v[(i * 7 + 3) % 300];
}
""")
    with pytest.raises(RuntimeError, match="crowded.hip: the compiler uses accumulator registers"):
        _build._check_accumulators(src)
