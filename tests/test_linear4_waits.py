"""The wait states between the global -> LDS copies of the 4-bit products and the writes of
the scalar registers they read, in the compiled device code. CPU only (hipcc)."""
import os
import subprocess

import pytest

from hy3_amd import build
from test_copy_waits import short_waits


@pytest.mark.parametrize("src", [s for s in build.sources() if "linear4_" in os.path.basename(s)],
                         ids=os.path.basename)
def test_copies_wait_for_their_scalar_registers(src):
    asm = subprocess.run([*build.compile_command(src), "-S", "--cuda-device-only", "-o", "-"],
                         check=True, capture_output=True, text=True).stdout
    copies, bad = short_waits(asm)
    assert not bad, bad[:5]
    assert copies or "f32" in src  # fp32 goes by way of registers
