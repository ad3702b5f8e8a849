"""The size of the int8 attention's workspace: one made for the largest sizes has
room for every call of smaller ones."""
import importlib
import itertools

import pytest

L = importlib.import_module("truellm-engine_b200._lib")


def size(b, hq, h, d, mq, ml):
    return L.lib().tkv_int8_attend_workspace_bytes(b, hq, h, d, mq, ml)


@pytest.mark.parametrize("heads,d", [((8, 32), 128), ((2, 8), 64), ((1, 40), 128), ((4, 4), 64)])
def test_the_size_never_falls_as_a_size_grows(heads, d):
    h, hq = heads
    grid = ((1, 2, 7, 8, 18, 37, 63, 64, 75, 148, 500), (1, 2, 4, 5, 17, 33, 64, 128, 256, 512, 600),
            (0, 1, 64, 200, 511, 512, 513, 2000, 8192, 60000))
    need = {at: size(at[0], hq, h, d, at[1], at[2]) for at in itertools.product(*grid)}
    assert min(need.values()) > 0
    for at, n in need.items():
        for axis in range(3):  # the next larger value of one size
            i = grid[axis].index(at[axis]) + 1
            if i < len(grid[axis]):
                up = at[:axis] + (grid[axis][i],) + at[axis + 1:]
                assert n <= need[up], (at, n, up, need[up])


def test_every_smaller_batch_and_chunk_fits():
    """64 sequences, chunks of 512, contexts of 8192, 32 q heads on 8 kv heads."""
    most = size(64, 32, 8, 128, 512, 8192)
    for b in range(1, 65):
        assert size(b, 32, 8, 128, 512, 8192) <= most, b
    for mq in range(1, 513):
        for b in (1, 3, 8, 37, 64):
            assert size(b, 32, 8, 128, mq, 8192) <= most, (b, mq)
    for ml in range(0, 8193, 64):
        assert size(8, 32, 8, 128, 512, ml) <= most, ml
    for hq in (8, 16, 24):
        assert size(8, hq, 8, 128, 512, 8192) <= most, hq
    # the partials of one round of the SMs, not of the batch
    assert most < 32 << 20 and size(4096, 32, 8, 128, 512, 8192) < 32 << 20


@pytest.mark.parametrize("at", range(6))
@pytest.mark.parametrize("over", [2 ** 32, 2 ** 31, -2 ** 32])
def test_sizes_past_32_bits_are_refused(ops, at, over):
    """(and not taken for what their low 32 bits say)"""
    sizes = [2, 8, 2, 128, 1, 64]
    assert ops.int8_workspace_bytes(*sizes) > 0
    sizes[at] += over
    with pytest.raises(ValueError, match="32 bits"):
        ops.int8_workspace_bytes(*sizes)


def test_sections_past_32_bits_are_refused(ops):
    for sections in ((64 + 2 ** 32,), (2 ** 32, 64), (64 + 2 ** 32, -2 ** 32)):
        with pytest.raises(ValueError, match="32 bits"):
            ops._rope_plan(2 * sum(sections), sections, 1e4, "blocks", "halves")
