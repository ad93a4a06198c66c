"""Windows of any size over a paged cache: what a call needs and takes, at the C entries; nothing runs on a GPU."""
import sys

import pytest

from tests.test_paged_refusals import attend


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("left", [sys.maxsize, sys.maxsize - 1, 1 << 62, 1 << 32, (1 << 29) + 1, 1 << 29])
def test_a_window_beyond_all_keys_is_none(lib, left, bits):
    """The room that a call is told and the room that it asks for are the same."""
    for n, width in ((48, 512), (2, 8192), (2, 3), (64, 40)):
        size = lambda w: lib.trx_attn_paged_bytes(n, 1, 4, 2, 128, 16 * width, w, int(bits == 4))  # noqa: E731
        assert size(left) == size(-1)
        if size(-1):
            assert attend(lib, bits, n=n, width=width, left=left, pb=size(left) - 1) == -9
