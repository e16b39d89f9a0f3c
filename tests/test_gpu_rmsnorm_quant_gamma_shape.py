"""A gamma without dimensions, which no row length makes a row of, is refused like any other wrong shape."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H", [1, 8])
def test_a_gamma_without_dimensions_is_refused(H):
    from nkilib.core.rmsnorm import rmsnorm_quant_rows, rmsnorm_quant_rows_bwd

    x = torch.zeros((4, H), device="cuda", dtype=torch.bfloat16)
    g = torch.ones((), device="cuda", dtype=torch.bfloat16)
    for call in (lambda: rmsnorm_quant_rows(x, g), lambda: rmsnorm_quant_rows_bwd(x, x, g)):
        with pytest.raises(AssertionError, match="gamma must hold"):
            call()
    codes, scales = rmsnorm_quant_rows(x, g.view(1).expand(H).contiguous())
    assert codes.shape == (4, H) and scales.shape == (4,)
