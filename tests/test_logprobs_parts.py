"""Which rows ``bfly_token_logprobs`` takes in parts, told by its workspace: no GPU."""
from __future__ import annotations

import pytest

from butterfly_amd import _native


@pytest.mark.parametrize("rows,vocab,parts", [
    (1, 8192, 1), (1, 8193, 1), (32, 12000, 1), (1, 16383, 1), (1, 16384, 2), (1, 16385, 3), (32, 32003, 4), (1, 151936, 19),
    (200, 151936, 5), (1, 1 << 29, 32), (513, 151936, 1), (5000, 151936, 1),
])
def test_rows_below_16384_are_whole(rows, vocab, parts):
    need = _native.lib().bfly_token_logprobs_workspace_bytes
    for top in (0, 7):
        assert need(rows, vocab, top) == (rows * parts * (16 + 8 * top) if parts > 1 else 0)
