"""Broadcast operands: rows expanded from one (stride 0) reach the library as rows of their own."""
import pytest
import torch

import swvr_b200 as swvr
from tests.helpers import rel_err

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,tol", [(torch.float64, 1e-10), (torch.float32, 1e-4), (torch.bfloat16, 2e-2)])
def test_readout_of_broadcast_rows_is_the_readout_of_their_copies(dtype, tol):
    g = torch.Generator().manual_seed(0)
    t = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype).cuda()  # noqa: E731
    h, W, E = t(64), t(300, 64), t(16)
    rows, table = h.expand(40, 64), E.expand(300, 16)
    O, lse = swvr.softmax_readout(rows, W, table)
    O2, lse2 = swvr.softmax_readout(rows.contiguous(), W, table.contiguous())
    assert torch.equal(O, O2) and torch.equal(lse, lse2)
    ref, lse_ref = swvr.softmax_readout_reference(rows.double(), W.double(), table.double())
    assert rel_err(O, ref) < tol and rel_err(lse, lse_ref) < tol
