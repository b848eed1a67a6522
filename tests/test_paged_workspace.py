"""The workspace that lowbit_attention_paged has use for: none where nothing is split or the sizes are refused, never more than
every tile's parts twice over, and no more with bounds that the sizes do not reach (on the CPU: of sizes alone)."""
import itertools

import pytest

from lowbit import _native


def size(t, b, hq, hkv, d, width, page, new, keys):
    return _native.lib().lowbit_attention_paged_workspace(t, b, hq, hkv, d, width, page, new, keys)


def test_calls_that_split_nothing_need_none():
    assert size(1, 1, 16, 2, 128, 100, 16, 1, 1) == 0
    assert size(500, 3, 28, 4, 128, 100, 16, 400, 256) == 0            # no part has fewer keys
    assert size(2000, 5, 28, 4, 128, 64, 16, 500, 1000) == 0           # many tiles of not many keys


@pytest.mark.parametrize("sizes", [(0, 1, 16, 2, 128, 9, 64, 1, 500), (1, 0, 16, 2, 128, 9, 64, 1, 500), (1, 1, 16, 3, 128, 9, 64, 1, 500),
                                   (1, 1, 16, 2, 96, 9, 64, 1, 500), (1, 1, 16, 2, 128, 0, 64, 1, 500), (1, 1, 16, 2, 128, 9, 48, 1, 500),
                                   (1, 1, 16, 2, 128, 9, 64, 0, 500), (1, 1, 16, 2, 128, 9, 64, 1, 0), (1 << 40, 1, 16, 2, 128, 9, 64, 1, 1)])
def test_refused_sizes_need_none(sizes):
    assert size(*sizes) == 0


def test_sizes():
    for (hq, hkv, d), t, b, new, keys in itertools.product(((28, 4, 128), (32, 8, 128), (14, 2, 64), (40, 1, 64)), (1, 3, 64, 500, 9000),
                                                           (1, 3, 64), (1, 2, 40, 9000), (300, 700, 1000, 9000, 70000)):
        got = size(t, b, hq, hkv, d, 5000, 16, new, keys)
        for rows in (32, 64, 128):                                     # a record: 32, 64 or 128 rows of d + 4 floats
            if got % (rows * (d + 4) * 4) == 0 and got // (rows * (d + 4) * 4) <= (2048 if rows == 128 else 1024):
                break
        else:
            raise AssertionError((hq, hkv, d, t, b, new, keys, got))
        tiles = (-(-t * (hq // hkv) // 32) + min(t, b)) * hkv          # of 32 rows: the most there can be
        assert got <= 2 * tiles * -(-keys // 256) * 128 * (d + 4) * 4
        assert got == size(t, b, hq, hkv, d, 5000, 16, min(new, t), keys)         # at most t tokens are new
        assert size(t, b, hq, hkv, d, 5000, 16, new, 1 << 40) == size(t, b, hq, hkv, d, 5000, 16, new, 80000)


def test_batches_whose_lengths_take_too_long_to_walk_are_refused():
    from test_paged_refusals import attend
    assert attend(b=65537, t=65537, hq=2, hkv=1) == 3
    assert "B 65536" in _native.lib().lowbit_last_error().decode()
    assert size(65537, 65537, 2, 1, 128, 9, 64, 1, 500) == 0 and size(1, 65536, 2, 1, 128, 99, 64, 1, 5000) > 0
