"""The plan's size, which the kernels' library tells the host."""
import pytest

from system_lab_b200.ops import cuda, packed


@pytest.mark.parametrize("rows", [1, 127, 128, 129, 256, 257, 8191, 2 ** 20 + 1, packed.MAX_ROWS])
def test_words_of_a_plan(rows):
    """Two words a row, four a tile of 128 and one a pair of tiles (packed_attention.cuh)."""
    try:
        words = cuda.lib().slab_packed_plan_words
    except Exception as e:
        pytest.skip(f"kernel library not built: {e}")
    tiles = -(-rows // packed.TILE)
    assert words(rows) == 2 * rows + 4 * tiles + -(-tiles // 2)
    assert words(0) < 0 and words(packed.MAX_ROWS + 1) < 0
