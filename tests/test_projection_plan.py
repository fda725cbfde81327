"""Which kernel the linear layer in 8 bits takes: the sizes that the GPU tests use reach every one of them, split and whole, and a call that is refused has none."""
import pytest

pytest.importorskip("torch")
import test_gpu_linear_int8 as sizes  # noqa: E402
import test_gpu_projection_use as use  # noqa: E402
from projection_plan import plan  # noqa: E402


def test_every_kernel_is_reached():
    seen = {(p.tile, p.features, p.splits > 1) for p in (plan(*s) for s in sizes.FEW + sizes.MANY + use.FORMS)}
    assert seen == {(0, 16, False), (0, 16, True), (64, 64, False), (64, 64, True), (128, 64, False), (128, 128, False), (128, 256, False), (256, 256, False)}


@pytest.mark.parametrize("shape,tile,features,split", use.KINDS_OF_FORMS)
def test_forms(shape, tile, features, split):
    p = plan(*shape)
    assert (p.tile, p.features) == (tile, features) and (p.splits > 1) == split


def test_rows_that_lie_far_apart_are_no_tiles():
    """offsets over a tile are held in 32 bits"""
    assert plan(3000, 3000, 64, ld_x=(1 << 23) - 16).tile > 0
    assert plan(3000, 3000, 64, ld_x=1 << 23).tile == plan(3000, 3000, 64, ld_w=1 << 23).tile == 0


def test_few_rows_are_no_large_tiles():
    for n in (1, 16, 100, 4096, 100000):
        for k in (1, 64, 1000, 16384, 131071):
            for m in (1, 16, 33):
                p = plan(m, n, k)
                assert p.tile < 256 and 1 <= p.splits <= 16
            assert plan(m, n, 0) == (0, 16, 1)


def test_none_where_the_call_is_refused():
    assert plan(-1, 3, 4) is None and plan(1, 3, 131072) is None and plan(1, 3, 40, ld_x=40) is None and plan(1, (1 << 25) + 1, 40) is None
    assert plan(1, 1 << 25, 40).tile == 0
