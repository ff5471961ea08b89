"""How much room the weight gradient's partial sums get: enough for whatever start indices the device may hold, and no more than rows
that exist can need.  Host arithmetic; no device needed."""
import itertools
import random

import pytest

from ops3d_b200 import capi

F32, BF16 = 0, 2
BLOCK = {F32: 256, BF16: 64}            # rows of a block
LEAST_PIECE = {F32: 1, BF16: 8}         # blocks of the shortest piece


def ceil_div(a, b):
    return -(-a // b)


def piece_of(batch, rows, groups, dtype, tiles, workers):
    """Blocks of a piece: enough pieces for the workers over the weight's tiles, or of twice a group's mean where groups are many."""
    block = BLOCK[dtype]
    blocks = max(1, batch * min(rows, rows // block + groups))
    wanted = max(1, workers // tiles)
    length = ceil_div(blocks, wanted - (groups - 1)) if wanted >= 2 * groups else 2 * ceil_div(blocks, groups)
    return blocks if blocks <= 2 * LEAST_PIECE[dtype] else max(LEAST_PIECE[dtype], length)


def slots_needed(sizes, batch, dtype, piece):
    pieces = [ceil_div(batch * ceil_div(n, BLOCK[dtype]), piece) for n in sizes]
    return sum(n for n in pieces if n > 1)


def slots_reserved(batch, rows, groups, inputs, outputs, dtype):
    assert inputs * outputs % 64 == 0 and outputs % 64 == 0 and inputs % 8 == 0    # nothing but slots, nothing rounded up
    reserved = capi.load().fda_linear_backward_workspace_bytes(batch, rows, groups, inputs, outputs, 0, dtype)
    assert reserved % (4 * outputs * (inputs + 1)) == 0
    return reserved // (4 * outputs * (inputs + 1))


# inputs, outputs, type, tiles of the weight, workers
SHAPES = [(64, 64, BF16, 1, 148), (64, 64, F32, 1, 148), (256, 256, F32, 16, 148), (1024, 4096, BF16, 64, 74)]


@pytest.mark.parametrize("batch,rows,groups", [(16, 12, 4), (40, 9, 3), (5, 15, 5), (200, 7, 7), (64, 1, 3), (65, 1, 3)])
def test_every_cut_of_a_few_rows_fits(batch, rows, groups):
    """Elements of so few rows that each group of a single row has pieces: all sizes that the groups can have."""
    for inputs, outputs, dtype, tiles, workers in SHAPES[:2]:
        piece, room = piece_of(batch, rows, groups, dtype, tiles, workers), slots_reserved(batch, rows, groups, inputs, outputs, dtype)
        if batch * rows <= 64:
            assert room == 0                                # kernels for few rows, which cut nothing
            continue
        worst = max(slots_needed(sizes, batch, dtype, piece)
                    for sizes in itertools.product(range(rows + 1), repeat=groups) if sum(sizes) <= rows)
        assert worst <= room


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_uneven_groups_fit(shape):
    """Long and short batches, few and many groups: random sizes, and as many groups as rows allow that just need n slots."""
    inputs, outputs, dtype, tiles, workers = shape
    rng = random.Random(1)
    for _ in range(400):
        batch, groups = rng.choice([1, 1, 2, 3, 17, 300]), int(2 ** rng.uniform(0, 10))
        rows = int(2 ** rng.uniform(0, 17 - batch.bit_length()))
        if batch * rows <= 64:
            continue
        if (inputs, outputs) == (1024, 4096) and 64 * ceil_div(batch * min(rows, rows // 64 + groups), 16) < 74:
            continue                                        # (too short for the tile that the list names)
        piece, room = piece_of(batch, rows, groups, dtype, tiles, workers), slots_reserved(batch, rows, groups, inputs, outputs, dtype)
        cuts = sorted(rng.randint(0, rows) for _ in range(groups))
        assert slots_needed([b - a for a, b in zip(cuts, cuts[1:])], batch, dtype, piece) <= room
        assert slots_needed([rows], batch, dtype, piece) <= room
        for n in (2, 3, 5):
            least = BLOCK[dtype] * ((n - 1) * piece // batch) + 1       # the fewest rows an element with which a group has n pieces
            sizes = [least] * min(groups, rows // least)
            if sizes:
                sizes[0] += rows - sum(sizes)
            assert slots_needed(sizes, batch, dtype, piece) <= room


def test_experts_do_not_reserve_what_their_rows_cannot_need():
    """2048 rows in pieces of at least 512: three groups can be longer than a piece, with two slots each, however many groups there are."""
    assert slots_reserved(1, 2048, 256, 1024, 4096, BF16) <= 6
    assert slots_reserved(1, 2048, 1024, 1024, 1024, BF16) <= 6
    assert slots_reserved(1, 500, 1024, 1024, 1024, BF16) == 0
    assert slots_reserved(1, 100000, 1, 1024, 1024, BF16) <= 74 // 16 + 1
