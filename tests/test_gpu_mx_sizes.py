"""Sizes over what the entry points count in."""
import pytest
import torch

from test_gpu_mx import DEV, K

pytestmark = pytest.mark.gpu


def test_more_columns_than_an_int_counts_are_refused():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    k = K()
    x = torch.empty(1, 2 ** 32 + 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="2\\^31"):
        k.mx_quantize(x, "e2m1")
