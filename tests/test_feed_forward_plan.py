"""How the gated block's products are launched, by the library's own arithmetic on the host (no GPU needed)."""
import random

import pytest

pytest.importorskip("torch")    # first: the library then shares its HIP runtime

from ffn_plan import D_W, D_X, FORWARD, plan    # noqa: E402

# rows, d, f and strides: dp of millions of features, whose rows lie further apart than 2^32 bytes over a tile of 128 or 256 of them, or over 32;
# rows of x and of the weights that far apart, as they are and as copies
WIDE = [(128, 64, 9_000_000), (300, 64, 4_200_000), (256, 8, 4_194_304), (2, 8, 40_000_000), (64, 8, 80_000_000), (33, 8, 1 << 21), (200, 3, 9_000_000),
        (300, (1 << 23) + 8, 64), (300, (1 << 23) + 1, 64), (257, (1 << 22) - 8, 64), (257, (1 << 22) - 7, 64), (40, (1 << 27) + 1, 64)]


@pytest.mark.parametrize("product", [FORWARD, D_X, D_W])
@pytest.mark.parametrize("shape", WIDE, ids=lambda s: "x".join(map(str, s)))
def test_offsets_of_32_bits_stay_inside_them(product, shape):
    p = plan(product, *shape)
    assert p is not None and 0 <= p.span < 1 << 32


def test_offsets_of_32_bits_over_random_sizes():
    rng, seen = random.Random(1), 0
    size = lambda most: int(2 ** rng.uniform(0, most))  # noqa: E731
    for _ in range(4000):
        rows, d, f, gap = size(14), size(24), size(28), rng.choice((0, 0, 8, size(30)))
        for product in (FORWARD, D_X, D_W):
            p = plan(product, rows, d, f, (d + gap, d + gap, f + gap), at=rng.choice((4096, 4096, 4098)))
            if p is not None:
                seen += p.span > 1 << 30
                assert 0 <= p.span < 1 << 32, (product, rows, d, f, gap, p)
    assert seen > 20


def test_ordinary_sizes_go_straight_into_lds():
    """rows that are whole pieces, up to where their distance ends that"""
    for product in (FORWARD, D_X, D_W):
        assert plan(product, 4096, 2048, 8192).direct == 1
        assert plan(product, 300, 64, (1 << 21) - 128).direct == 1
    assert plan(D_X, 300, 64, 1 << 21).direct == 0 and plan(D_W, 300, 64, 1 << 21).direct == 0
    assert plan(FORWARD, 300, 64, 1 << 21).direct == 1    # (dp is none of its operands)
