"""The workspace of attention over the paged cache: one made for some sizes serves
every smaller call, whichever of its forms that takes."""
import itertools

import pytest

from moe_infer_amd import _lib


def size(batch, n, max_q, max_len, H=16, G=2):
    return _lib.lib().mi_attn_paged_workspace_size(batch, n, max_q, max_len, H, G)


@pytest.mark.parametrize("H,G", [(16, 2), (4, 4), (15, 3), (16, 1), (2048, 2048)])
def test_a_larger_workspace_serves_smaller_calls(H, G):
    steps = {"batch": [1, 3, 64, 300, 65535], "tokens": [1, 2, 5, 40, 3000], "max_len": [0, 512, 1025, 2049, 5000, 200000]}
    if G == 2048:
        steps["max_len"] = [0, 512]
    last = {}
    for b, q, length in itertools.product(*steps.values()):
        now = size(b, b * q if b * q < 2 ** 31 else 2 ** 31 - 1, q, length, H, G)
        if not now:
            continue  # refused: too many tiles for one call
        last[b, q, length] = now
    assert len(last) > 20
    for (b, q, length), now in last.items():
        for (b2, q2, l2), smaller in last.items():
            if b2 <= b and q2 <= q and l2 <= length:
                assert smaller <= now, ((b, q, length), (b2, q2, l2))


def test_sizes():
    assert size(1, 1 << 20, 1 << 20, 1 << 20) > 0, "a prompt of a million tokens"
    assert size(65535, 65535, 1, 1 << 24) == 0, "more tiles than a decode step counts"
    assert size(0, 1, 1, 1) == 0 and size(1, 0, 1, 1) == 0 and size(1, 1, 0, 1) == 0 and size(1, 1, 1, -1) == 0
    assert size(1, 1, 1, 1, 16, 3) == 0 and size(1, 1, 1, 1, 34, 2) == 0
