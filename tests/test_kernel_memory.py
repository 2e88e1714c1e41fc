"""The kernels of the verifier and of the logits head keep nothing in private memory, whatever their types, groups and
numbers of rows: their tiles are meant to stay in registers."""
import re

from test_build_hygiene import resources


def test_operators_keep_nothing_in_private_memory():
    seen = {}
    for name, v in resources().items():
        m = re.search(r"(verify_(?:stats|decide|greedy|rest|finish)_kernel|head_(?:stream|rows|tile)_kernel)", name)
        if m:
            assert v["ScratchSize"] == 0 and v["VGPRs Spill"] == 0, (name, v)
            seen[m.group(1)] = seen.get(m.group(1), 0) + 1
    assert len(seen) == 8 and all(n >= 3 for n in seen.values()), seen
