"""Verification of drafted tokens with weights whose sum passes fp32's range: against the plain loop in 64 bits, equal or wrong."""
import pytest
import torch

from test_gpu_verify import plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R,V,dt", [(1, 50257, torch.float32), (60, 4097, torch.float32), (120, 50257, torch.bfloat16), (3, 33, torch.float32)])
@pytest.mark.parametrize("draft", [True, False])
def test_weights_whose_sum_passes_fp32(R, V, dt, draft):
    """Rows of a few huge entries (in one lane's reach: 32 apart) or of nothing but huge ones, behind a rejected draft and behind none."""
    from mathbrain_b200.verify import verify_drafts
    G = 1
    g = torch.Generator().manual_seed(R + V)
    p = torch.rand(R, G + 1, V, generator=g)
    p[::2, :, ::32] = 2.0 ** 127
    p[1::2] = 2.0 ** 126 * (1 + torch.randint(0, 4, (len(p[1::2]), G + 1, V), generator=g) / 4)
    p = p.to(dt)
    q = torch.rand(R, G, V, generator=g).to(dt)
    q[:, :, ::64] = 2.0 ** 125
    x = torch.randint(0, V, (R, G), generator=g)
    u = torch.rand(R, G + 1, generator=g)
    q.scatter_(2, x[..., None], torch.finfo(torch.float32).max / 2)         # the draft is rejected in many rows
    p[::3].scatter_(2, x[::3, None].expand(-1, G + 1, -1), 0.0)
    n, t = verify_drafts(p.cuda(), x.cuda(), u.cuda(), p_draft=q.cuda() if draft else None)
    n_ref, t_ref = plain(p, x, u, q if draft else None)
    assert torch.equal(n.cpu(), n_ref) and torch.equal(t.cpu(), t_ref)
