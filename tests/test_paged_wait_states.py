"""The wait states of the direct LDS loads (see test_attention_wait_states.py) in the paged cache's kernels, whose loads' bases come
from page numbers."""
import re
import subprocess

import pytest

from test_attention_wait_states import hazards
from transformer_amd import build


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    out = tmp_path_factory.mktemp("paged") / "paged.s"
    flags = [f for f in build.HIPCC_FLAGS if f != "-shared"]
    subprocess.run([build.hipcc(), *flags, "--cuda-device-only", "-S", f"{build.HERE}/csrc/paged.hip", "-o", str(out)], check=True)
    return out.read_text()


def test_direct_lds_loads_wait(assembly):
    loads, lacks = hazards(assembly)
    assert loads > 100 and not lacks, lacks[:4]


@pytest.mark.parametrize("DP,loads", [(32, 4), (64, 4), (96, 8), (128, 8)])
def test_a_tile_of_values_is_waited_for_past_the_scores_stores(assembly, DP, loads):
    """A wave that stores scores waits for all but the next tile's loads and four stores: four there must be, before the wait."""
    body = re.search(rf"^_ZN3msp9paged_fewILi{DP}E.*?:\n(.*?)s_endpgm\n\s*\.section", assembly, re.S | re.M).group(1).split("\n")
    waits = [i for i, x in enumerate(body) if re.search(rf"s_waitcnt vmcnt\({2 * loads + 4}\)", x)]
    stores = []
    for i in waits:
        last = max(k for k in range(i) if re.search(r"buffer_load_dwordx4 .* lds", body[k]))
        stores.append(sum("global_store_dwordx4" in x for x in body[last:i]))
    # (3 * 4 is 2 * 4 + 4: the wait for the keys, with no stores behind the loads yet)
    assert stores == ([0, 4] if loads == 4 else [4])
