"""What the compiled kernels of the paged cache must hold and no run can be relied on to show, looked at in the code object that was
built (no GPU)."""
import re
import subprocess
from pathlib import Path

import pytest

from bigger_bird_amd import _lib

OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{mangled name: its instructions, labels among them} of the kernels with `paged_` in their names."""
    if not OBJDUMP.exists():
        pytest.skip("no llvm-objdump")
    at = tmp_path_factory.mktemp("code")
    lib = at / "lib.so"
    lib.write_bytes(_lib.library_path().read_bytes())
    subprocess.run([OBJDUMP, "--offloading", lib.name], cwd=at, check=True, capture_output=True)
    found = {}
    for obj in sorted(at.glob("*gfx950")):
        if b"paged_tile_kernel" not in obj.read_bytes():
            continue
        text = subprocess.run([OBJDUMP, "-d", "--symbolize-operands", "--no-show-raw-insn", obj.name], cwd=at, check=True,
                              capture_output=True, text=True).stdout
        for line in text.splitlines():
            m = re.match(r"[0-9a-f]+ <(.*)>:$", line)
            if m and not re.fullmatch(r"L\d+", m[1]):
                body = found.setdefault(m[1], [])
            elif m:
                body.append(m[1] + ":")
            elif line.startswith("\t"):
                body.append(line.split("//")[0].strip())
    assert len([k for k in found if "paged_tile_kernel" in k]) == 8
    return found


def test_flags_are_stored_before_the_barrier_that_publishes_them(kernels):
    """paged_tile_kernel's barriers wait for nothing, so that its loads stay in flight: a store to LDS (the flags of tiles that hold
    values that are not finite) is waited for where it is made."""
    for name, code in kernels.items():
        if "paged_tile_kernel" not in name:
            continue
        stores = [i for i, x in enumerate(code) if x.startswith("ds_write")]
        assert stores, name
        for i in stores:
            for x in code[i + 1:]:
                if re.match(r"s_waitcnt .*lgkmcnt\(0\)", x):
                    break
                assert not re.match(r"s_barrier|s_c?branch|s_endpgm|L\d+:", x), f"{name}: `{code[i]}` is not waited for before `{x}`"
