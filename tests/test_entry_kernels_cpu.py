"""The kernels that leave entries out put no registers off to memory, and their workgroups fit a compute unit more than once. Read from the
notes the compiler leaves in the library built here, which has a bundle of device code for each of its sources."""
import os
import re
import subprocess

import pytest

from vet_amd import build

LLVM = "/opt/rocm/llvm/bin"
TOOLS = [os.path.join(LLVM, t) for t in ("llvm-objcopy", "clang-offload-bundler", "llvm-readelf")]
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


@pytest.mark.skipif(not all(map(os.path.exists, TOOLS)), reason="no LLVM tools")
def test_registers_and_shared_memory(tmp_path):
    if not os.path.exists(build.LIB_PATH):
        build.build_library(verbose=False)
    objcopy, bundler, readelf = TOOLS
    fat = tmp_path / "fat.bin"
    subprocess.run([objcopy, "--dump-section", f".hip_fatbin={fat}", build.LIB_PATH, str(tmp_path / "rest.so")], check=True)
    bundles = fat.read_bytes().split(MAGIC)[1:]
    assert len(bundles) == len(build.SOURCES)
    found = {}
    for k, bundle in enumerate(bundles):
        one, code = tmp_path / f"{k}.bin", tmp_path / f"{k}.elf"
        one.write_bytes(MAGIC + bundle)
        subprocess.run([bundler, "--unbundle", "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", f"--input={one}", f"--output={code}"], check=True)
        notes = subprocess.run([readelf, "--notes", str(code)], check=True, capture_output=True, text=True).stdout
        for kernel in notes.split("- .agpr_count:")[1:]:
            number = {n: int(re.search(rf"\.{n}:\s+(\d+)", kernel).group(1)) for n in ("private_segment_fixed_size", "group_segment_fixed_size")}
            found[re.search(r"\.name:\s+(\S+)", kernel).group(1)] = number
    own = {k: v for k, v in found.items() if re.search(r"dropout_kernel|select_|keep_rows_kernel|weights_|clear_slots", k)}
    assert len(own) >= 20, sorted(own)
    for name, number in own.items():
        assert number["private_segment_fixed_size"] == 0 and number["group_segment_fixed_size"] <= 80 * 1024, (name, number)
