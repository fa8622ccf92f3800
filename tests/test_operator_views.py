"""Views whose memory does not hold their values (torch keeps a sign, or that all are zero, beside it): refused, never read as they lie."""
import pytest

from hugectr_backend_amd import hps


def test_views_whose_memory_holds_other_values_are_refused():
    import torch
    from hugectr_backend_amd.quantized_rows import calls
    c, ids = calls(), torch.zeros(4, dtype=torch.int32)
    rows = torch.zeros(4, 4, dtype=torch.float16)
    for f in (lambda: c.group_rows(torch._neg_view(ids), 2), lambda: c.rows_read(0, 0, 4, torch._neg_view(ids.long()), None, 0, 0.0),
              lambda: c.linear_forward(0, 0, 1, 4, 4, 1, torch._neg_view(rows), None, None, None, None, None, None, 1),
              lambda: c.linear_forward(0, 0, 1, 4, 4, 1, torch._efficientzerotensor((4, 4), dtype=torch.float16), None, None, None, None, None, None, 1)):
        with pytest.raises(hps.HpsError, match="holds its values") as e:
            f()
        assert e.value.code == hps.ERR_INVALID_ARG
