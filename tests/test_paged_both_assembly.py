"""The kernel of tokens and chunks in one launch has an instance of the tokens' code of its own, by two of its four waves where heads
are wide: what is counted by hand there, and that all of a workgroup's waves reach its barriers."""
import re

import pytest

from test_paged_wait_states import assembly  # noqa: F401 (a fixture)


def bodies(text):
    return {m.group(1): m.group(2).split("\n") for m in re.finditer(r"^(_ZN3msp\w+):.*?\n(.*?)s_endpgm\n\s*\.section", text, re.S | re.M)}


def test_barriers_are_reached_by_all_waves(assembly):  # noqa: F811
    """No barrier lies between a branch that waves without lanes left take and where it leads: waves that others wait for cannot have gone
    another way.  (The branch on lanes that there are is also what the compiler makes of some plain jumps.)"""
    kernels, barriers = bodies(assembly), 0
    for name, body in kernels.items():
        labels = {x.split(":")[0]: i for i, x in enumerate(body) if re.match(r"\.LBB\w+:", x)}
        at = [i for i, x in enumerate(body) if "s_barrier" in x]
        barriers += len(at)
        for i, x in enumerate(body):
            b = re.search(r"s_cbranch_execz\s+(\.LBB\w+)", x)
            if b:
                lo, hi = sorted((i, labels.get(b.group(1), len(body))))
                assert not any(lo < k < hi for k in at), (name, i, x.strip())
    assert sum("paged_both" in k for k in kernels) == 4 and barriers > 100


@pytest.mark.parametrize("DP,loads", [(32, 4), (64, 4), (96, 8), (128, 8)])
def test_a_tile_of_values_is_waited_for_past_the_scores_stores(assembly, DP, loads):  # noqa: F811
    """As in the tokens' own kernel: the wait that leaves the next tile's loads and four stores follows four stores."""
    body = next(b for name, b in bodies(assembly).items() if f"paged_bothILi{DP}E" in name)
    stores = []
    for i, x in enumerate(body):
        if re.search(rf"s_waitcnt vmcnt\({2 * loads + 4}\)", x):
            last = max(k for k in range(i) if re.search(r"buffer_load_dwordx4 .* lds", body[k]))
            stores.append(sum("global_store_dwordx4" in y for y in body[last:i]))
    # (3 * 4 is 2 * 4 + 4: the wait for the keys, with no stores behind the loads yet)
    assert stores == ([0, 4] if loads == 4 else [4])
