"""Verification of drafted tokens against a plain loop in 64 bits; whole numbers, so equal or wrong."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def plain(p, drafted, u, q=None):
    R, G1, V = p.shape
    G = G1 - 1
    p, u, drafted = p.double().cpu().numpy(), u.double().cpu().numpy(), drafted.cpu().numpy()
    q = None if q is None else q.double().cpu().numpy()

    def clean(w):
        return np.where(np.isfinite(w) & (w > 0), w, 0.0)

    n, tokens = np.zeros(R, np.int64), np.full((R, G1), -1, np.int64)
    for r in range(R):
        a, w = 0, None
        while a < G:
            x = drafted[r, a]
            if x < 0 or x >= V:
                break
            qx = 1.0 if q is None else q[r, a, x]
            if not u[r, a] * qx < p[r, a, x]:
                qrow = np.zeros(V) if q is None else q[r, a]
                if q is None:
                    qrow[x] = 1.0
                with np.errstate(invalid="ignore"):
                    w = clean(p[r, a] - qrow)
                if w.sum() == 0:
                    w = None
                break
            tokens[r, a] = x
            a += 1
        if w is None:
            w = clean(p[r, a])
        n[r] = a
        run = np.cumsum(w)
        if run[-1] > 0:
            i = int(np.searchsorted(run, u[r, G] * run[-1], side="right"))
            tokens[r, a] = i if i < V else np.nonzero(w)[0][-1]
    return torch.from_numpy(n), torch.from_numpy(tokens)


def _case(R, G, V, dt, draft, seed, sharp=1.5):
    g = torch.Generator().manual_seed(seed)
    base = torch.randn(R, G + 1, V, generator=g) * sharp
    p = (base + 0.3 * torch.randn(R, G + 1, V, generator=g)).softmax(-1).to(dt)
    q = (base[:, :G] + 0.6 * torch.randn(R, G, V, generator=g)).softmax(-1).to(dt)
    x = torch.multinomial(q.float().view(R * G, V), 1, generator=g).view(R, G) if G else torch.zeros(R, 0, dtype=torch.long)
    return p, x, torch.rand(R, G + 1, generator=g), q if draft else None


@pytest.mark.parametrize("R,G,V,dt,draft", [
    (1, 1, 1, torch.float32, True), (3, 2, 2, torch.float32, False), (5, 3, 31, torch.bfloat16, True), (4, 0, 1000, torch.float32, False),
    (40, 4, 127, torch.float32, True), (40, 7, 128, torch.bfloat16, False), (17, 40, 129, torch.float32, True),
    (64, 5, 4097, torch.float32, True), (9, 3, 50257, torch.float32, True), (9, 3, 50257, torch.bfloat16, True), (300, 2, 513, torch.bfloat16, True),
    (2, 65, 77, torch.float32, False)])
def test_matches_the_plain_loop(R, G, V, dt, draft):
    from mathbrain_b200.verify import verify_drafts
    for seed in (1, 2):
        p, x, u, q = _case(R, G, V, dt, draft, 100 * R + G + seed)
        n, t = verify_drafts(p.cuda(), x.cuda(), u.cuda(), p_draft=None if q is None else q.cuda())
        n_ref, t_ref = plain(p, x, u, q)
        assert torch.equal(n.cpu(), n_ref) and torch.equal(t.cpu(), t_ref), seed


def test_borders_ties_and_rows_without_mass():
    from mathbrain_b200.verify import verify_drafts
    V, G = 300, 2
    flat = torch.full((V,), 1.0 / 256)                       # sums without rounding: 300 / 256
    spike = torch.zeros(V)
    spike[37] = 1.0
    last = torch.zeros(V)
    last[V - 1] = 0.5
    zero = torch.zeros(V)
    bad = flat.clone()
    bad[::7] = float("nan")
    bad[1::7] = float("inf")
    bad[2::7] = -1.0
    rows, drafts, us, qs = [], [], [], []
    for first, x, u, q in [
            (flat, 5, 0.0, flat), (flat, 5, 1.0 - 2 ** -24, flat),             # p = q: stands whatever u
            (zero, 5, 0.0, flat),                                              # p = 0: 0 < 0 is false
            (spike, 37, 0.5, spike), (spike, 36, 0.0, flat), (spike, 36, 0.9, flat * 2),
            (flat * 0.5, 9, 0.75, flat),                                       # rejected with p <= q everywhere: from p
            (zero, 9, 0.5, flat),                                              # rejected without any mass: -1
            (flat, -1, 0.0, flat), (flat, V, 0.0, flat), (flat, 2 ** 40, 0.0, flat), (flat, -2 ** 40, 0.0, flat),   # the drafts end
            (bad, 0, 0.5, flat * 0.5), (bad, 1, 0.5, flat), (bad, 2, 0.0, flat), (bad, 3, 0.3, flat * 0.5), (last, 3, 0.2, flat)]:
        for second in (flat, spike, last, zero, bad):
            for u2 in (0.0, 0.25, 0.5, 1.0 - 2 ** -24, 128.0 / 300, 1.0, float("nan")):
                rows.append(torch.stack([first, second, second]))
                drafts.append([x, 11])
                us.append([u, 0.4, u2])
                qs.append(torch.stack([q, flat]))
    p, x, u, q = torch.stack(rows), torch.tensor(drafts), torch.tensor(us), torch.stack(qs)
    for dt in (torch.float32, torch.bfloat16):
        for qq in (q, None):
            n, t = verify_drafts(p.to(dt).cuda(), x.cuda(), u.cuda(), p_draft=None if qq is None else qq.to(dt).cuda())
            n_ref, t_ref = plain(p.to(dt), x, u, None if qq is None else qq.to(dt))
            assert torch.equal(n.cpu(), n_ref)
            wrong = (t.cpu() != t_ref).any(1).nonzero().flatten().tolist()
            assert not wrong, (wrong[:5], t.cpu()[wrong[:5]], t_ref[wrong[:5]])


def test_strided_rows_and_other_layouts():
    from mathbrain_b200.verify import verify_drafts
    R, G, V = 6, 3, 1001
    p, x, u, q = _case(R, G, V, torch.float32, True, 5)
    n_ref, t_ref = plain(p, x, u, q)
    wide = torch.full((R, G + 1, V + 13), 9.0)
    wide[:, :, 5:5 + V] = p
    pos_first = p.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    vocab_first = p.permute(2, 0, 1).contiguous().cuda().permute(1, 2, 0)
    for pp in (wide.cuda()[:, :, 5:5 + V], pos_first, vocab_first):
        for qq in (q.cuda(), q.permute(2, 0, 1).contiguous().cuda().permute(1, 2, 0)):
            n, t = verify_drafts(pp, x.t().contiguous().cuda().t(), u.cuda(), p_draft=qq)
            assert torch.equal(n.cpu(), n_ref) and torch.equal(t.cpu(), t_ref)
    one = p[:1, :1].cuda()
    n, t = verify_drafts(one.expand(R, G + 1, V), x.cuda(), u.cuda())
    n_ref, t_ref = plain(p[:1, :1].expand(R, G + 1, V), x, u)
    assert torch.equal(n.cpu(), n_ref) and torch.equal(t.cpu(), t_ref)
    empty = verify_drafts(torch.zeros(0, 3, 9).cuda(), torch.zeros(0, 2, dtype=torch.long).cuda(), torch.zeros(0, 3).cuda())
    assert empty[0].shape == (0,) and empty[1].shape == (0, 3)


def test_frequencies_are_the_targets():
    """The next token after one draft has the target's distribution, whatever the draft's: 40 000 draws of a 12-token target
    (the largest of 12 deviations from n p, in units of sqrt(n p), stays below 5)."""
    from mathbrain_b200.verify import verify_drafts
    g = torch.Generator().manual_seed(2)
    R, V = 40000, 12
    p = torch.randn(V, generator=g).softmax(0)
    q = (2.0 * torch.randn(V, generator=g)).softmax(0)
    x = torch.multinomial(q, R, replacement=True, generator=g)[:, None]
    u = torch.rand(R, 2, generator=g)
    _, t = verify_drafts(p.cuda().expand(R, 2, V), x.cuda(), u.cuda(), p_draft=q.cuda().expand(R, 1, V))
    got = torch.bincount(t[:, 0].cpu(), minlength=V).double()
    assert float(((got - R * p.double()).abs() / (R * p.double()).sqrt()).max()) < 5.0


def test_captured_in_a_graph_and_on_a_side_stream():
    from mathbrain_b200.verify import verify_drafts
    p, x, u, q = (t.cuda() for t in _case(5, 3, 777, torch.float32, True, 9))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        n1, t1 = verify_drafts(p, x, u, p_draft=q)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n, t = verify_drafts(p, x, u, p_draft=q)
    graph.replay()
    assert torch.equal(n, n1) and torch.equal(t, t1)
    u.copy_(torch.rand(5, 4, generator=torch.Generator().manual_seed(4)))
    graph.replay()
    n_ref, t_ref = plain(p, x, u, q)
    assert torch.equal(n.cpu(), n_ref) and torch.equal(t.cpu(), t_ref)


def test_refusals():
    from mathbrain_b200 import _lib
    from mathbrain_b200.verify import verify_drafts
    E = _lib.MbemaError
    p, x, u, q = (t.cuda() for t in _case(2, 3, 50, torch.float32, True, 1))
    for bad in (dict(p_target=p[0]), dict(p_target=p[:, :3]), dict(p_target=p.half()), dict(p_target=p.double()), dict(drafted=x.int()),
                dict(drafted=x[:1]), dict(uniforms=u[:, :3]), dict(uniforms=u.double()), dict(p_draft=q[:, :2]), dict(p_draft=q.bfloat16()),
                dict(p_draft=q[:, :, :40]), dict(p_target=p[:, :, :0], p_draft=None), dict(drafted=x.cpu()), dict(p_target=p.cpu())):
        with pytest.raises(E):
            verify_drafts(**{**dict(p_target=p, drafted=x, uniforms=u, p_draft=q), **bad})
