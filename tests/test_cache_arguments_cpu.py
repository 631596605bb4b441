"""Whole numbers of other types than int, as page sizes."""
import numpy as np
import pytest

import triton_ext_amd as tx

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("number", [int, np.int32, np.int64, torch.tensor])
def test_page_sizes_of_any_whole_type(number):
    t, n, r = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(8, dtype=torch.int32)
    for call in (lambda p: tx.page_reserve(t, n, r, n, p), lambda p: tx.page_free(t, n, r, n > 0, p)):
        with pytest.raises(tx.TxError) as e:  # it comes as far as the check of its value
            call(number(12))
        assert e.value.code == tx.ERR_UNSUPPORTED and "power of two" in str(e.value)
        with pytest.raises(Exception) as e:  # (16 is fine; then there is no device for host tensors)
            call(number(16))
        assert "power of two" not in str(e.value)
        with pytest.raises(tx.TxError) as e:  # and its value counts, not its type and shape
            call(number(24))
        assert "power of two" in str(e.value)
        for bad in (16.0, "16", None):
            with pytest.raises(TypeError):
                call(bad)
