"""The MFMA distances of the 2 x 2-wave tiles (test_mfma_hazards_host.py) in the objects with gated epilogues and with
the rows' adapters, whose low-rank MFMAs are assembly as well."""
import subprocess

import pytest

from test_mfma_hazards_host import LLVM, ROOT, _scan


@pytest.mark.parametrize("stem", ["gemm_tile_gated", "gemm_tile_gated_grad", "gemm_tile_adapters"])
def test_built_tiles_keep_the_distances(stem, tmp_path):
    obj = ROOT / "vllm-mach_amd" / "_build" / f"{stem}.o"
    if not obj.exists() or not (LLVM / "clang-offload-bundler").exists():
        pytest.skip("no built object (run __graft_entry__.build() first) or no disassembler")
    code, fatbin = tmp_path / f"{stem}.co", tmp_path / f"{stem}.fatbin"
    subprocess.run([LLVM / "llvm-objcopy", f"--dump-section=.hip_fatbin={fatbin}", obj], check=True)
    subprocess.run([LLVM / "clang-offload-bundler", "--unbundle", "--type=o", f"--input={fatbin}", f"--output={code}",
                    "--targets=hipv4-amdgcn-amd-amdhsa--gfx950"], check=True)
    text = subprocess.run([LLVM / "llvm-objdump", "-d", "--no-show-raw-insn", code], check=True, capture_output=True,
                          text=True).stdout
    mfmas, faults = _scan(text.splitlines())
    assert mfmas >= 480
    assert not faults, faults[:10]
