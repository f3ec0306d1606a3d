"""What the built kernels do around copies from memory into LDS (their listing; no GPU needed)."""
import os
import re
import shutil
import subprocess

import pytest

import f2cgt_amd

LLVM = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin")


def _listing(tmp_path, kernel):
    """{name: instructions} of the kernels whose name holds `kernel`."""
    objdump = os.path.join(LLVM, "llvm-objdump")
    if not os.path.exists(objdump):
        pytest.skip("no llvm-objdump")
    library = shutil.copy(f2cgt_amd.capi_path(), tmp_path)
    subprocess.run([objdump, "--offloading", os.path.basename(library)], cwd=tmp_path, check=True, capture_output=True)
    found = {}
    for name in sorted(os.listdir(tmp_path)):
        if not name.endswith("gfx950"):
            continue
        names = subprocess.run([objdump, "-t", name], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        symbols = [line.split()[-1] for line in names.splitlines() if kernel in line and ".text" in line]
        if not symbols:
            continue
        text = subprocess.run([objdump, "-d", "--no-show-raw-insn", "--disassemble-symbols=" + ",".join(symbols), name],
                              cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        for part in re.split(r"^(?=[0-9a-f]+ <\w+>:$)", text, flags=re.M)[1:]:
            symbol = re.search(r"<(\w+)>", part).group(1)
            found[symbol] = [line.split("//")[0].strip() for line in part.splitlines()[1:] if line.strip()]
    return found


def test_few_columns_wait_for_the_weights(tmp_path):
    """Each wave waits for its own copies in front of the barrier behind which the others read them: there, not where the loads of the
    tokens, which come after them, happen to be used."""
    listing = _listing(tmp_path, "int8_rows_kernel")
    assert len(listing) == 6
    for name, lines in listing.items():
        copies = [i for i, text in enumerate(lines) if "_lds_" in text]
        barrier = next(i for i, text in enumerate(lines) if text.startswith("s_barrier"))
        assert copies and copies[-1] < barrier, name
        waits = [text for text in lines[barrier - 8:barrier] if text.startswith("s_waitcnt")]
        assert any("vmcnt(0)" in text for text in waits), (name, waits)
