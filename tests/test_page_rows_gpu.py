"""Pages of fewer rows than a wave loads at a time, in every form of the paged attention."""
import pytest

torch = pytest.importorskip("torch")

from cachecase import E4M3  # noqa: E402
from test_cache_gpu import attend  # noqa: E402

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("page", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("dtype,cache", [(BF, BF), (HF, HF), (BF, E4M3)])
@pytest.mark.parametrize("D", [64, 128, 144, 256])
@pytest.mark.parametrize("n,G", [(1, 4), (2, 10), (30, 5)])  # units of 16, 32 and 128 rows
def test_small_pages(gpu, n, G, D, dtype, cache, page):
    for layout in ("nhd", "hnd"):
        attend(gpu, [n] * 3, [n + 1, n + 62, 333], 2 * G, 2, D, page, dtype, cache, layout=layout)


@pytest.mark.parametrize("n,G", [(1, 4), (2, 10), (30, 5)])
def test_small_pages_with_holes(gpu, n, G):
    """Pages of 4 next to ones that are not there."""
    holes = [(0, e, -1) for e in (1, 2, 9)] + [(1, e, 10 ** 6) for e in (0, 4, 7)]
    attend(gpu, [n] * 2, [140, 131], 2 * G, 2, 256, 4, HF, HF, holes=holes, window=100)
