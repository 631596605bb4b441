"""Books of pools that were filled in ascending order, as page_reserve itself fills them, at the
sizes where a launch has more workgroups than the table's rows keep busy."""
import pytest

torch = pytest.importorskip("torch")

import triton_ext_amd as tx  # noqa: E402
from dotcase import say  # noqa: E402
from test_cache_gpu import Books, same  # noqa: E402

pytestmark = pytest.mark.gpu


def ascending(S, W, P, page, held):
    """Books of S sequences that hold the first `held` pages, in equal parts, in order."""
    b = Books(0, 0, W, P, page)
    b.table = [[-1] * W for _ in range(S)]
    b.len = [0] * S
    at = 0
    for s in range(S):
        k = held // S + (s < held % S)
        b.table[s][:k] = range(at, at + k)
        b.len[s] = k * page
        b.refs[at:at + k] = [1] * k
        at += k
    return b


@pytest.mark.parametrize("S,W,P,held", [
    (1, 1024, 8192, 512), (3, 1024, 16384, 1536), (8, 8192, 65536, 5000), (5, 2048, 32768, 3000),
    (257, 2048, 100000, 80000), (2, 3, 300000, 6), (1, 4097, 4097, 4097), (1, 16384, 65536, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_no_page_is_given_twice(gpu, S, W, P, held, in_place):
    say("reserve", S, W, P, held, in_place)
    page = 4
    b = ascending(S, W, P, page, held)
    t, n, r = b.to(gpu)
    for more in (1, 3 * page, 0, 7):  # one call after another on what the last one wrote
        new = [x + more for x in b.len]
        out = (t, n, r) if in_place else None
        t, n, r, missing = tx.page_reserve(t, n, r, torch.tensor(new, dtype=torch.int32, device=gpu),
                                           page, out=out)
        assert int(missing) == b.reserve(new)
        same(b, t, n, r)
    given = t[t >= 0]
    assert given.unique().numel() == given.numel()
    assert int((r > 0).sum()) == given.numel()
