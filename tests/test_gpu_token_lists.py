"""Tables without slots (operators and tolerances: test_gpu_token_permute)."""

import pytest

pytestmark = pytest.mark.gpu


def test_no_slots_and_no_table():
    """Without slots there is no table to hand over, and every sum is zero whatever the scratch memory holds."""
    import torch
    from nkilib import _native as nv

    L = nv.lib()
    y = torch.ones((1, 16), device="cuda")
    aff, be = torch.ones((4, 3), device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    for T in (1, 4, 600):
        for fill in (0, 2, 10**6, -1):
            slots = torch.full((T, 3), fill, dtype=torch.int32, device="cuda")
            out = torch.full((T, 16), 7.0, device="cuda")
            rc = L.moe_combine_tokens(y.data_ptr(), nv.DT_FP32, None, 0, 0, 0, None, None, 0, 0, slots.data_ptr(), 2, 1, 0, T, 16,
                                      out.data_ptr(), nv.stream_ptr(y.device))
            assert rc == 0 and not out.any(), (T, fill)
            if T <= 4:
                out.fill_(7.0)
                rc = L.moe_combine_tokens(y.data_ptr(), nv.DT_FP32, aff.data_ptr(), nv.DT_FP32, 4, 3, None, be.data_ptr(), 4, 0,
                                          slots.data_ptr(), 2, 1, 0, T, 16, out.data_ptr(), nv.stream_ptr(y.device))
                assert rc == 0 and not out.any(), (T, fill)
