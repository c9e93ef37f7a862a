"""Which calls on rows of class scores need a workspace (no GPU)."""
import pytest


@pytest.mark.parametrize("score_type,classes", [(0, 32768), (0, 1 << 20), (1, 65536), (2, 65537), (1, 1 << 30)])
@pytest.mark.parametrize("n", [1, 7, 64])
def test_few_long_rows_need_one_that_grows_with_the_alternatives(score_type, classes, n):
    from cutdet._lib import lib
    sizes = [lib.cd_rows_workspace(n, classes, score_type, top) for top in (0, 1, 20, 64)]
    assert 0 < sizes[0] < sizes[1] < sizes[2] < sizes[3]
    # statistics (16 bytes) and alternatives (8 bytes each) of 2 to 64 parts of a row, the student's scores of 256 entries
    assert n * (2 * 16 + 1024) <= sizes[0] <= n * (64 * 16 + 1024) and sizes[3] <= n * (64 * (16 + 8 * 64) + 1024)


@pytest.mark.parametrize("n,classes,score_type", [(200000, 3, 0), (1, 32767, 0), (1, 65535, 1), (4096, 131072, 1)])
def test_short_or_many_rows_need_none(n, classes, score_type):
    from cutdet._lib import lib
    assert lib.cd_rows_workspace(n, classes, score_type, 0) == lib.cd_rows_workspace(n, classes, score_type, 20) == 0
