"""Branches of a decode state against the dense decode loop in 64 bits: every branch as a sequence of its own.

Tolerances (norm-wise, rel_err), from half a rounding step a value: fp32 arithmetic 1e-4 (dot products of up to 128 and 64 terms, each
2^-24, into an exponent of scores of a few units); bf16 2e-2 (2^-8 each for the output, the values and the weights, and the scores'
16-bit operands); states 1e-5 (a rounding of 2^-24 for every kept token of a slot)."""
import numpy as np
import pytest
import torch

from oracle import ema_oracle as orc
from helpers import rel_err

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 1e-4, torch.bfloat16: 2e-2}


def _setup(B, V, N, H, prefix, dt, seed, hl=(2.0, 64.0), cap=None, scale=0.2):
    """A decode state after `prefix` steps, its dense double, tables."""
    from mathbrain_b200 import synth
    from mathbrain_b200.decode import DecodeState
    g = torch.Generator().manual_seed(seed)
    rhos = synth.make_rhos(N, *hl)
    D = 64 * H
    E_k, E_v = ((torch.randn(V, D, generator=g) * scale).to(dt) for _ in range(2))
    W = torch.randn(N, D, generator=g) * 0.1
    st = DecodeState(B, V, rhos.cuda(), capacity=cap or V)
    state, last = torch.zeros(B, V, N, dtype=torch.float64), torch.full((B, V), -1, dtype=torch.long)
    q = torch.zeros(B, 1, 64, dtype=torch.float64)
    for t in range(prefix):
        tok = torch.randint(0, V, (B,), generator=g)
        tok = torch.where(torch.rand(B, generator=g) < 0.3, tok % 7, tok)        # some tokens again and again
        st.update(tok.cuda(), t)
        orc.decode_step(state, last, t, tok, q, E_k[:, :64].double(), E_v[:, :64].double(), W[:, :64].double(), rhos, V,
                        dtype=torch.float64)
    return g, rhos, E_k, E_v, W, st, state, last


def _rows(state, last, t, tok, q, E_k, E_v, W, rhos, V, **kw):
    """n steps of a batch of dense sequences: (O [R, n, H, 64], C_q [R, n, N]); state and last move on.  tok -1: no token."""
    outs, cqs = [], []
    listed_only = kw.pop("listed_only", False)
    for j in range(tok.shape[1]):
        v = tok[:, j]
        keep = state[torch.arange(len(v)), v.clamp_min(0)].clone(), last[torch.arange(len(v)), v.clamp_min(0)].clone()
        if listed_only:
            O = _listed_only(state, last, t[:, None] + j, q[:, j], E_k, E_v, W, rhos, **kw)
        O_all, C_all = [], []
        for r in range(len(v)):                                          # rows may stand at different steps
            sr, lr = state[r:r + 1], last[r:r + 1]
            o, c = orc.decode_step(sr, lr, int(t[r]) + j, v[r:r + 1].clamp_min(0), q[r:r + 1, j], E_k, E_v, W, rhos, V,
                                   dtype=torch.float64, **kw)
            O_all.append(o)
            C_all.append(c)
        idle = v < 0
        rows = torch.arange(len(v))[idle]
        state[rows, 0], last[rows, 0] = keep[0][idle], keep[1][idle]
        C = torch.cat(C_all)
        C[idle] = 0
        outs.append(O if listed_only else torch.cat(O_all))
        cqs.append(C)
    return torch.stack(outs, 1), torch.stack(cqs, 1)


def _listed_only(state, last, t, q, E_k, E_v, W, rhos, use_silu=True):
    R, V, N = state.shape
    H = q.shape[1]
    M = state * rhos.double() ** (t - last).clamp_min(0)[..., None].double()
    x = M @ W
    g = x * torch.sigmoid(x) if use_silu else x
    K, U = ((E.view(1, V, H, 64) * g.view(R, V, H, 64)) for E in (E_k, E_v))
    s = torch.einsum("rhd,rvhd->rhv", q, K) / 8.0
    s = s.masked_fill((last < 0)[:, None], -float("inf"))
    w = torch.softmax(s, -1).nan_to_num(0.0)
    return torch.einsum("rhv,rvhd->rhd", w, U)


CASES = [  # B, S, n, V, N, H, prefix, rounds, dtype, mode
    (1, 1, 1, 40, 8, 1, 0, 6, torch.float32, None),              # nothing before the branches
    (2, 3, 2, 60, 16, 2, 25, 6, torch.float32, None),
    (3, 2, 5, 50, 64, 1, 40, 4, torch.float32, "fp32"),
    (1, 70, 1, 300, 32, 1, 150, 2, torch.float32, None),         # more branches than a CTA takes
    (2, 2, 3, 400, 128, 2, 330, 3, torch.float32, None),         # several tiles, 128 channels
    (1, 1, 32, 90, 24, 1, 30, 2, torch.float32, None),           # the most staged tokens
    (2, 1, 1, 30, 7, 3, 12, 4, torch.float32, None),             # odd channels and heads
    (2, 3, 2, 60, 16, 2, 25, 4, torch.bfloat16, None),
    (1, 1, 1, 40, 64, 1, 0, 6, torch.bfloat16, None),
    (2, 1, 6, 400, 64, 2, 300, 3, torch.bfloat16, None),
    (2, 5, 3, 300, 64, 2, 140, 3, torch.bfloat16, None),
    (1, 17, 1, 300, 64, 1, 200, 4, torch.bfloat16, None),
    (1, 64, 1, 500, 64, 2, 333, 2, torch.bfloat16, None),
    (2, 33, 2, 200, 128, 1, 129, 2, torch.bfloat16, None),
    (1, 1, 11, 200, 128, 3, 60, 2, torch.bfloat16, None),
    (2, 2, 3, 200, 64, 1, 90, 2, torch.bfloat16, "fp32"),
]


@pytest.mark.parametrize("B,S,n,V,N,H,prefix,rounds,dt,mode", CASES)
def test_branches_match_dense_decode(B, S, n, V, N, H, prefix, rounds, dt, mode):
    g, rhos, E_k, E_v, W, st, state, last = _setup(B, V, N, H, prefix, dt, 1000 * B + 10 * S + n)
    br = st.fork(S, prefix, capacity=n * rounds, max_new=n)
    state, last = state.repeat_interleave(S, 0), last.repeat_interleave(S, 0)
    t = torch.full((B * S,), prefix)
    Ed = E_k.double(), E_v.double(), W.double()
    tabs = E_k.cuda(), E_v.cuda(), W.cuda()
    before = {k: getattr(st, k).clone() for k in ("state", "last_t", "active", "n_active")}
    for rnd in range(rounds):
        tok = torch.randint(0, V, (B, S, n), generator=g)
        tok = torch.where(torch.rand(B, S, n, generator=g) < 0.4, tok % 5, tok)            # repeats, inside a call too
        tok = torch.where(torch.rand(B, S, n, generator=g) < 0.1, torch.full_like(tok, -1), tok)
        q = torch.randn(B, S, n, H, 64, generator=g).to(dt)
        C_q = br.extend(tok.cuda())
        O = br.attend(q.cuda(), *tabs, mode=mode)
        assert O.dtype == dt and O.shape == q.shape
        flat = tok.view(B * S, n)
        s2, l2 = state.clone(), last.clone()
        O_ref, C_ref = _rows(s2, l2, t, flat, q.view(B * S, n, H, 64).double(), *Ed, rhos, V)
        assert rel_err(C_q.cpu().view(B * S, n, N), C_ref) < 1e-5 or float(C_ref.abs().max()) == 0.0, rnd
        assert rel_err(O.cpu().view(B * S, n, H, 64), O_ref) < TOL[dt], rnd
        if rnd % 3 == 2:
            state, last, t = s2, l2, t + n                                                # kept by the next extend
            continue
        counts = torch.randint(0, n + 1, (B,), generator=g)
        br.keep(counts.cuda())
        per = counts.repeat_interleave(S)
        for c in range(1, n + 1):
            rows = per >= c
            s1, l1 = state[rows], last[rows]
            if len(s1):
                _rows(s1, l1, t[rows], flat[rows][:, c - 1:c], torch.zeros(len(s1), 1, H, 64, dtype=torch.float64), *Ed, rhos, V)
                state[rows], last[rows] = s1, l1
                t = torch.where(rows, t + 1, t)
        assert torch.equal(br.lengths.cpu().view(-1).long(), t - prefix), rnd
    br.check_overflow()
    for k, x in before.items():
        assert torch.equal(getattr(st, k), x), k


@pytest.mark.parametrize("dt,N", [(torch.float32, 16), (torch.bfloat16, 64)])
@pytest.mark.parametrize("silu", [True, False])
def test_listed_slots_only_and_a_row_that_sees_none(dt, N, silu):
    B, S, n, V, H, prefix = 2, 3, 2, 40, 2, 6
    g, rhos, E_k, E_v, W, st, state, last = _setup(B, V, N, H, prefix, dt, 7)
    Ed = E_k.double(), E_v.double(), W.double()
    for t0, st_, s_, l_ in ((prefix, st, state, last), (0, type(st)(B, V, rhos.cuda(), capacity=8), torch.zeros_like(state), torch.full_like(last, -1))):
        br = st_.fork(S, t0, capacity=8, max_new=n)
        tok = torch.randint(0, V, (B, S, n), generator=g)
        tok[0, 0, 0] = -1
        q = torch.randn(B, S, n, H, 64, generator=g).to(dt)
        br.extend(tok.cuda())
        O = br.attend(q.cuda(), E_k.cuda(), E_v.cuda(), W.cuda(), listed_only=True, use_silu=silu).cpu()
        ref, _ = _rows(s_.repeat_interleave(S, 0), l_.repeat_interleave(S, 0), torch.full((B * S,), t0), tok.view(-1, n),
                       q.view(-1, n, H, 64).double(), *Ed, rhos, V, use_silu=silu, listed_only=True)
        assert rel_err(O.view(-1, n, H, 64), ref) < TOL[dt]
        if t0 == 0:
            assert (O[:, :, 0] == 0).all() and (O[0, 0, 1] == 0).all()          # the first rows see no slot at all


def test_adopted_branch_goes_on_as_the_sequence():
    """Branches of different lengths (sequences that kept different counts) adopted, then decoded and forked on."""
    B, S, V, N, H, prefix, n = 3, 2, 60, 16, 1, 20, 3
    g, rhos, E_k, E_v, W, st, state, last = _setup(B, V, N, H, prefix, torch.float32, 3)
    br = st.fork(S, prefix, capacity=32, max_new=n)
    hist = [[[] for _ in range(S)] for _ in range(B)]
    for _ in range(4):
        tok = torch.randint(0, V, (B, S, n), generator=g)
        counts = torch.randint(0, n + 1, (B,), generator=g)
        br.extend(tok.cuda())
        br.keep(counts.cuda())
        for b in range(B):
            for s in range(S):
                hist[b][s] += tok[b, s, :counts[b]].tolist()
    branch = torch.tensor([1, 0, 1])
    t_next = prefix + 4 * n + 5
    br.adopt(branch.cuda(), t_next)
    Ed = E_k.double(), E_v.double(), W.double()
    zero = torch.zeros(1, H, 64, dtype=torch.float64)
    for b in range(B):
        for i, v in enumerate(hist[b][branch[b]]):
            orc.decode_step(state[b:b + 1], last[b:b + 1], prefix + i, torch.tensor([v]), zero, *Ed, rhos, V, dtype=torch.float64)
        shift = t_next - (prefix + len(hist[b][branch[b]]))
        last[b] = torch.where(last[b] >= 0, last[b] + shift, last[b])
    assert torch.equal(st.last_t.cpu().long(), last)
    assert rel_err(st.state.cpu(), state) < 1e-5
    for b in range(B):
        assert set(st.active[b, :int(st.n_active[b])].tolist()) == set((last[b] >= 0).nonzero().flatten().tolist())
        assert int(st.n_active[b]) == int((last[b] >= 0).sum())
    q = torch.randn(B, H, 64, generator=g)
    tok = torch.randint(0, V, (B,), generator=g)
    br2 = st.fork(1, t_next, capacity=4, max_new=1)
    C2 = br2.extend(tok.cuda().view(B, 1, 1))
    O2 = br2.attend(q.view(B, 1, 1, H, 64).cuda(), E_k.cuda(), E_v.cuda(), W.cuda())
    O = st.attend(q.cuda(), E_k.cuda(), E_v.cuda(), W.cuda(), t_next, mode="fp32")
    C = st.update(tok.cuda(), t_next)
    O_ref, C_ref = orc.decode_step(state, last, t_next, tok, q.double(), *Ed, rhos, V, dtype=torch.float64)
    assert rel_err(O.cpu(), O_ref) < 1e-4 and rel_err(O2.cpu().view_as(O_ref), O_ref) < 1e-4
    assert rel_err(C.cpu(), C_ref) < 1e-5 and rel_err(C2.cpu().view_as(C_ref), C_ref) < 1e-5
    st.check_overflow()
    from mathbrain_b200 import _lib
    with pytest.raises(_lib.MbemaError, match="updated"):
        br2.extend(tok.cuda().view(B, 1, 1))
    with pytest.raises(_lib.MbemaError, match="adopted"):
        br.extend(tok.cuda().view(B, 1, 1).expand(B, S, 1))


def test_reports_of_full_lists_and_bad_values():
    from mathbrain_b200 import _lib
    _, _, _, _, _, st, _, _ = _setup(1, 30, 8, 1, 4, torch.float32, 5, cap=6)
    one = torch.tensor([0]).cuda()
    br = st.fork(1, 4, capacity=2, max_new=3)
    br.extend(torch.tensor([[[10, 11, 12]]]).cuda())
    br.check_overflow()
    br.keep(torch.tensor([3]).cuda())
    with pytest.raises(_lib.MbemaError, match="full"):
        br.check_overflow()
    br = st.fork(1, 4, capacity=8, max_new=3)
    br.extend(torch.tensor([[[3, 30, -1]]]).cuda())
    with pytest.raises(_lib.MbemaError, match="vocabulary"):
        br.check_overflow()
    for branch, t_next, what in ((torch.tensor([1]), 99, "branch"), (one.cpu(), 4, "t_next")):
        br = st.fork(1, 4, capacity=8, max_new=3)
        keep = st.state.clone(), st.last_t.clone(), st.n_active.clone()
        br.extend(torch.tensor([[[20]]]).cuda())
        br.adopt(branch.cuda(), t_next)
        with pytest.raises(_lib.MbemaError, match=what):
            br.check_overflow()
        assert all(torch.equal(a, b) for a, b in zip(keep, (st.state, st.last_t, st.n_active)))
    br = st.fork(1, 4, capacity=8, max_new=3)               # the state's own list is too short for what the branch brings
    br.extend(torch.tensor([[[20, 21, 22]]]).cuda())
    br.extend(torch.tensor([[[23, 24, 25]]]).cuda())
    br.adopt(one, 99)
    with pytest.raises(_lib.MbemaError):
        st.check_overflow()


def test_refusals():
    from mathbrain_b200 import _lib
    _, _, E_k, E_v, W, st, _, _ = _setup(2, 30, 8, 1, 4, torch.float32, 5)
    E_k, E_v, W = E_k.cuda(), E_v.cuda(), W.cuda()
    E = _lib.MbemaError
    for kw in (dict(branches=0), dict(branches=1, capacity=0), dict(branches=1, max_new=0), dict(branches=1, max_new=33)):
        with pytest.raises(E):
            st.fork(t_now=4, **kw)
    br = st.fork(3, 4, capacity=8, max_new=2)
    q = torch.zeros(2, 3, 1, 1, 64).cuda()
    with pytest.raises(E, match="extend first"):
        br.attend(q, E_k, E_v, W)
    for tok in (torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3, 3, dtype=torch.int64), torch.zeros(2, 3, 0, dtype=torch.int64),
                torch.zeros(3, 2, 1, dtype=torch.int64), torch.zeros(2, 3, 1, dtype=torch.int32)):
        with pytest.raises(E):
            br.extend(tok.cuda())
    with pytest.raises(E):
        br.extend(torch.zeros(2, 3, 1, dtype=torch.int64))              # on the CPU
    br.extend(torch.zeros(2, 3, 1, dtype=torch.int64).cuda())
    for bad in ((q[:, :2], E_k, E_v, W), (q[..., :32], E_k, E_v, W), (q, E_k[:5], E_v, W), (q, E_k, E_v[:, :32], W), (q, E_k, E_v, W[:4]),
                (q.half(), E_k, E_v, W), (q, E_k.half(), E_v, W), (q.cpu(), E_k, E_v, W)):
        with pytest.raises(E):
            br.attend(*bad)
    with pytest.raises(ValueError):
        br.attend(q, E_k, E_v, W, mode="exact")
    for counts in (torch.zeros(3, dtype=torch.int64), torch.zeros(2), torch.zeros(2, dtype=torch.bool)):
        with pytest.raises(E):
            br.keep(counts.cuda())
    with pytest.raises(E):
        br.adopt(torch.zeros(3, dtype=torch.int64).cuda(), 9)
    st.state = st.state[:, :, ::2].contiguous()
    with pytest.raises(E):
        st.fork(1, 4)


def test_one_round_captured_and_replayed():
    """extend, two attends and keep captured once, replayed with other tokens, queries and counts; another branch set run
    eagerly beside it."""
    B, S, n, V, N, H, prefix, dt = 2, 3, 2, 200, 64, 2, 120, torch.bfloat16
    g, rhos, E_k, E_v, W, st, _, _ = _setup(B, V, N, H, prefix, dt, 11)
    tabs = E_k.cuda(), E_v.cuda(), W.cuda()
    br, ref = (st.fork(S, prefix, capacity=32, max_new=n) for _ in range(2))
    toks = torch.randint(0, V, (5, B, S, n), generator=g).cuda()
    counts = torch.randint(0, n + 1, (5, B), generator=g).cuda()
    qs = torch.randn(5, 2, B, S, n, H, 64, generator=g).to(dt).cuda()
    tok, cnt, q = toks[0].clone(), counts[0].clone(), qs[0].clone()

    def round_(which, tok, cnt, q):
        C = which.extend(tok)
        O = [which.attend(q[l], *tabs) for l in range(2)]
        which.keep(cnt)
        return C, O

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        round_(br, tok, torch.zeros_like(cnt), q)            # dropped again
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        C, O = round_(br, tok, cnt, q)
    for i in range(5):
        tok.copy_(toks[i]); cnt.copy_(counts[i]); q.copy_(qs[i])
        graph.replay()
        C_ref, O_ref = round_(ref, toks[i], counts[i], qs[i])
        assert torch.equal(C, C_ref) and all(torch.equal(a, b) for a, b in zip(O, O_ref)), i
    assert torch.equal(br.lengths, ref.lengths)
    br.check_overflow()
