"""The wait states of the direct LDS loads (see test_attention_wait_states.py) in the paged cache's kernels, whose loads' bases come
from page numbers."""
import subprocess

from test_attention_wait_states import hazards
from transformer_amd import build


def test_direct_lds_loads_wait(tmp_path):
    out = tmp_path / "paged.s"
    flags = [f for f in build.HIPCC_FLAGS if f != "-shared"]
    subprocess.run([build.hipcc(), *flags, "--cuda-device-only", "-S", f"{build.HERE}/csrc/paged.hip", "-o", str(out)], check=True)
    loads, lacks = hazards(out.read_text())
    assert loads > 100 and not lacks, lacks[:4]
