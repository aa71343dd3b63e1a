"""Branches as they are used (drafts verified, samples drawn), over long lists, and in calls from unusual places.

Tolerances as in test_gpu_branches.py, norm-wise: fp32 arithmetic 1e-4, bf16 2e-2 (half a step of bf16, 2^-8, for each of the output,
the values, the weights and the scores' operands)."""
import pytest
import torch

from helpers import rel_err
from test_gpu_branches import TOL, _rows

pytestmark = pytest.mark.gpu


def _made_up(B, V, N, H, listed, dt, seed, t0=5000, hl=(2.0, 400.0)):
    """A decode state with listed[b] slots, filled in rather than run; its dense double; tables."""
    from mathbrain_b200 import synth
    from mathbrain_b200.decode import DecodeState
    g = torch.Generator().manual_seed(seed)
    rhos = synth.make_rhos(N, *hl)
    D = 64 * H
    E_k, E_v = ((torch.randn(V, D, generator=g) * 0.2).to(dt) for _ in range(2))
    W = torch.randn(N, D, generator=g) * 0.1
    st = DecodeState(B, V, rhos.cuda(), capacity=V)
    state, last = torch.zeros(B, V, N), torch.full((B, V), -1, dtype=torch.long)
    active = torch.zeros(B, V, dtype=torch.int32)
    for b, count in enumerate(listed):
        slots = torch.randperm(V, generator=g)[:count]
        active[b, :count] = slots.int()
        state[b, slots] = 1.0 + 3.0 * torch.rand(count, N, generator=g)
        last[b, slots] = torch.randint(t0 - 300, t0, (count,), generator=g)
    st.state.copy_(state)
    st.last_t.copy_(last.int())
    st.active.copy_(active)
    st.n_active.copy_(torch.tensor(listed, dtype=torch.int32))
    return g, rhos, E_k, E_v, W, st, state.double(), last, t0


LONG = [  # B, S, n, V, N, H, listed slots, own rounds (of 32 tokens), dtype
    (2, 1, 1, 5000, 64, 2, [5000, 129], 0, torch.bfloat16),
    (3, 1, 6, 1500, 64, 2, [1300, 0, 1], 5, torch.bfloat16),
    (1, 1, 32, 900, 64, 3, [640], 6, torch.bfloat16),
    (2, 1, 5, 1200, 128, 2, [1111, 256], 5, torch.bfloat16),
    (70, 1, 2, 150, 64, 1, [i * 2 for i in range(70)], 1, torch.bfloat16),
    (2, 2, 3, 2000, 64, 2, [1999, 15], 6, torch.bfloat16),
    (1, 40, 1, 3000, 64, 1, [2900], 1, torch.bfloat16),
    (2, 3, 9, 800, 128, 1, [700, 17], 4, torch.bfloat16),
    (1, 2, 32, 600, 64, 1, [500], 2, torch.bfloat16),
    (3, 2, 4, 900, 24, 2, [700, 0, 65], 3, torch.float32),
    (1, 1, 32, 1500, 64, 1, [1400], 4, torch.float32),
    (230, 1, 9, 60, 64, 2, [i % 61 for i in range(230)], 0, torch.bfloat16),     # many rows: several steps to a merging CTA
    (80, 3, 3, 50, 64, 2, [i % 51 for i in range(80)], 1, torch.bfloat16),
    (80, 3, 10, 40, 16, 2, [i % 41 for i in range(80)], 1, torch.float32),
]


@pytest.mark.parametrize("B,S,n,V,N,H,listed,own,dt", LONG)
def test_long_lists(B, S, n, V, N, H, listed, own, dt):
    """Lists over many tiles, pieces and workers, and ones that are empty or end inside a tile; capacities far above their use."""
    g, rhos, E_k, E_v, W, st, state, last, t0 = _made_up(B, V, N, H, listed, dt, B * 1000 + S * 10 + n)
    br = st.fork(S, t0, capacity=own * 32 + n + 1000, max_new=32)
    state, last = state.repeat_interleave(S, 0), last.repeat_interleave(S, 0)
    perm = torch.stack([torch.randperm(V, generator=g)[:max(own * 32, 1)] for _ in range(B * S)])
    rh = rhos.double()
    for i in range(own):                                             # (the tokens of a branch are distinct: one addition each)
        br.extend(perm[:, i * 32:(i + 1) * 32].reshape(B, S, 32).contiguous().cuda())
    for i in range(own * 32):
        rows, v = torch.arange(B * S), perm[:, i]
        dt_ = (t0 + i - last[rows, v]).double()[:, None]
        state[rows, v] = torch.where(last[rows, v][:, None] >= 0, state[rows, v] * rh ** dt_, 0.0) + 1.0
        last[rows, v] = t0 + i
    tok = torch.randint(0, V, (B, S, n), generator=g)
    q = torch.randn(B, S, n, H, 64, generator=g).to(dt)
    C_q = br.extend(tok.cuda())
    O = br.attend(q.cuda(), E_k.cuda(), E_v.cuda(), W.cuda())
    O_ref, C_ref = _rows(state, last, torch.full((B * S,), t0 + own * 32), tok.view(-1, n), q.view(-1, n, H, 64).double(),
                         E_k.double(), E_v.double(), W.double(), rhos, V)
    assert rel_err(C_q.cpu().view(-1, n, N), C_ref) < 1e-5
    assert rel_err(O.cpu().view(-1, n, H, 64), O_ref) < TOL[dt]
    assert br.device_status() == 0
    br.check_overflow()


def _toy(V, N, H, layers, seed):
    """A next-token rule on top of the attention: q from the token and its state, logits from the layers' outputs."""
    g = torch.Generator().manual_seed(seed)
    emb = torch.randn(V, H * 64, generator=g).cuda()
    mix = (torch.randn(layers, N, H * 64, generator=g) * 0.3).cuda()
    head = torch.randn(layers * H * 64, V, generator=g).cuda()
    tabs = [tuple((torch.randn(V, H * 64, generator=g) * 0.5).cuda() for _ in range(2)) +
            ((torch.randn(N, H * 64, generator=g) * 0.2).cuda(),) for _ in range(layers)]

    def queries(l, tok, C):
        return (emb[tok.clamp_min(0)] + C @ mix[l]).unflatten(-1, (H, 64))

    def logits(outs):
        return torch.cat([o.flatten(-2) for o in outs], -1) @ head
    return tabs, queries, logits


def test_drafts_verified_round_by_round_give_the_plain_decode():
    """extend, attends, verify_drafts, keep in a loop, with drafts that are right now and then, against one token at a time: a
    target that is sure of its token makes the drafts' tokens the very ones of the plain loop."""
    from mathbrain_b200 import synth
    from mathbrain_b200.decode import DecodeState
    from mathbrain_b200.verify import verify_drafts
    B, V, N, H, layers, G, steps = 3, 80, 16, 2, 2, 4, 24
    tabs, queries, logits = _toy(V, N, H, layers, 1)
    rhos = synth.make_rhos(N, 2.0, 50.0).cuda()
    first = torch.tensor([3, 70, 11]).cuda()
    # plain: one token at a time; the token's own state is read by a fork that is thrown away, as a query needs it first
    st = DecodeState(B, V, rhos, capacity=V)
    tok, plain = first, [first]
    for t in range(steps):
        look = st.fork(1, t, capacity=1, max_new=1)
        C = look.extend(tok.view(B, 1, 1))[:, 0, 0]
        outs = [st.attend(queries(l, tok, C), *tabs[l], t, mode="fp32") for l in range(layers)]
        st.update(tok, t)
        tok = logits(outs).argmax(-1)
        plain.append(tok)
    plain = torch.stack(plain, 1)                                     # [B, steps + 1]
    # drafts: the plain tokens, some of them wrong
    g = torch.Generator().manual_seed(5)
    st = DecodeState(B, V, rhos, capacity=V)
    br = st.fork(1, 0, capacity=V, max_new=G + 1)
    done = [[int(v)] for v in first.cpu()]
    rounds = accepted = 0
    while min(len(d) for d in done) <= steps:
        at = torch.tensor([len(d) for d in done]) - 1
        drafts = torch.stack([plain[b].cpu()[(at[b] + 1 + torch.arange(G)).clamp(max=steps)] for b in range(B)])
        drafts = torch.where(torch.rand(B, G, generator=g) < 0.3, torch.randint(0, V, (B, G), generator=g), drafts).cuda()
        tok = torch.cat([torch.tensor([[d[-1]] for d in done]).cuda(), drafts], 1)
        C = br.extend(tok.view(B, 1, G + 1))[:, 0]
        outs = [br.attend(queries(l, tok, C)[:, None], *tabs[l], mode="fp32")[:, 0] for l in range(layers)]
        p = torch.nn.functional.one_hot(logits(outs).argmax(-1), V).float()
        n_acc, out = verify_drafts(p, drafts, torch.rand(B, G + 1, generator=g).cuda())
        br.keep(n_acc + 1)
        for b in range(B):
            n = int(n_acc[b])
            assert out[b, n + 1:].eq(-1).all()
            done[b] += out[b, :n + 1].tolist()
            accepted += n
        rounds += 1
    assert accepted > 0 and rounds < steps                             # (drafts were of use)
    for b in range(B):
        assert done[b][:steps + 1] == plain[b].tolist()
    assert br.lengths.cpu().view(-1).tolist() == [len(d) - 1 for d in done]
    br.check_overflow()


@pytest.mark.parametrize("dt,N,S", [(torch.float32, 16, 3), (torch.bfloat16, 64, 5)])
def test_samples_drawn_and_the_best_adopted(dt, N, S):
    """S samples of a prompt drawn with given numbers (no drafts), one of them adopted; then the state as if it had been decoded so."""
    from mathbrain_b200.verify import verify_drafts
    B, V, H, steps = 2, 300, 1, 6
    g, rhos, E_k, E_v, W, st, state, last, t0 = _made_up(B, V, N, H, [200, 77], dt, 9)
    tabs = E_k.cuda(), E_v.cuda(), W.cuda()
    head = torch.randn(H * 64, V, generator=g).cuda()
    br = st.fork(S, t0, capacity=steps, max_new=1)
    state, last = state.repeat_interleave(S, 0), last.repeat_interleave(S, 0)
    tok = torch.randint(0, V, (B * S,), generator=g).cuda()
    history = []
    for i in range(steps):
        q = torch.randn(B, S, 1, H, 64, generator=g).to(dt)
        history.append(tok.cpu())
        br.extend(tok.view(B, S, 1))
        O = br.attend(q.cuda(), *tabs)
        O_ref, _ = _rows(state, last, torch.full((B * S,), t0 + i), history[-1][:, None], q.view(-1, 1, H, 64).double(),
                         E_k.double(), E_v.double(), W.double(), rhos, V)
        assert rel_err(O.cpu().view_as(O_ref), O_ref) < TOL[dt], i
        p = torch.softmax(O.float().view(B * S, 1, H * 64) @ head, -1)
        u = torch.rand(B * S, 1, generator=g)
        n_acc, out = verify_drafts(p, torch.empty(B * S, 0, dtype=torch.int64).cuda(), u.cuda())
        assert (n_acc == 0).all()
        tok = out[:, 0]
        cum = p[:, 0].double().cumsum(-1)
        assert (cum.gather(1, tok[:, None])[:, 0] > u.cuda()[:, 0].double() * cum[:, -1] - 1e-9).all()
    pick = torch.tensor([S - 1, 1])
    br.adopt(pick.cuda(), t0 + steps)
    rows = pick + S * torch.arange(B)
    assert torch.equal(st.last_t.cpu().long(), last[rows])
    assert rel_err(st.state.cpu(), state[rows]) < 1e-5


@pytest.mark.parametrize("S,dt,N,mode", [(1, torch.bfloat16, 64, None), (3, torch.bfloat16, 64, None), (2, torch.float32, 20, None),
                                         (1, torch.bfloat16, 128, None), (3, torch.bfloat16, 64, "fp32")])
def test_scores_below_fp32_and_values_that_are_not_finite(S, dt, N, mode):
    B, n, V, H = 1, 3, 120, 1
    g, rhos, E_k, E_v, W, st, state, last, t0 = _made_up(B, V, N, H, [50], dt, 21)
    W = W.abs() + 0.01                                                # (gates above 0: the score of a slot has the sign of q.E_k)
    listed = st.active[0, :50].cpu().long()
    new = torch.tensor([v for v in range(V) if v not in set(listed.tolist())])
    q = torch.randn(B, S, n, H, 64, generator=g).to(dt)

    def run(E_k, E_v, tok, q):
        br = st.fork(S, t0, capacity=8, max_new=n)
        br.extend(tok.cuda())
        return br.attend(q.cuda(), E_k.cuda(), E_v.cuda(), W.cuda(), mode=mode).cpu().view(S, n, H, 64)

    def ref(E_k, E_v, tok, q):
        return _rows(state.repeat_interleave(S, 0), last.repeat_interleave(S, 0), torch.full((B * S,), t0), tok.view(-1, n),
                     q.view(-1, n, H, 64).double(), E_k.double(), E_v.double(), W.double(), rhos, V)[0]

    # products of -1e38 and 1e38: below fp32's range in every listed slot, a weight of zero in the plain form
    low_k, big_q = E_k.clone(), q.clone()
    low_k[:, 0] = -1e38
    big_q[..., 0] = 1e38
    tok = new[:n].repeat(S).view(1, S, n)
    out, plain = run(low_k, E_v, tok, big_q), ref(low_k, E_v, tok, big_q)
    assert (plain == 0).all() and (out == 0).all()                    # all of the weight lies on slots that are not listed
    # tokens that no row sees may hold anything
    odd_k, odd_v = E_k.clone(), E_v.clone()
    odd_k[new[n:]], odd_v[new[n:]] = float("nan"), float("inf")
    assert torch.equal(run(odd_k, odd_v, tok, q), run(E_k, E_v, tok, q))
    # a NaN in a query stays in its row, one in a staged token's value in the rows behind it
    nan_q = q.clone()
    nan_q[0, S - 1, 1] = float("nan")
    out = run(E_k, E_v, tok, nan_q)
    assert out[S - 1, 1].isnan().all() and out[S - 1, 0].isfinite().all() and out[S - 1, 2].isfinite().all()
    assert out[:S - 1].isfinite().all()
    nan_v = E_v.clone()
    nan_v[new[0]] = float("nan")
    tok2 = new[1:n + 1].repeat(S).view(1, S, n).clone()
    tok2[0, 0, 1] = new[0]
    out = run(E_k, nan_v, tok2, q)
    assert out[0, 2].isnan().all() and out[0, :2].isfinite().all() and out[1:].isfinite().all()
    # one in the prefix reaches all rows
    nan_v = E_v.clone()
    nan_v[listed[49]] = float("nan")
    assert run(E_k, nan_v, tok, q).isnan().all()


@pytest.mark.parametrize("S,dt,N", [(1, torch.bfloat16, 64), (4, torch.bfloat16, 64), (2, torch.float32, 64)])
def test_channels_that_forget_at_once_and_never(S, dt, N):
    """Decay 0 (a half-life too short for fp32) and 1, and steps far apart."""
    B, n, V, H = 2, 4, 90, 1
    g, rhos, E_k, E_v, W, st, state, last, t0 = _made_up(B, V, N, H, [60, 33], dt, 31)
    rhos = rhos.clone()
    rhos[::3], rhos[1::3] = 0.0, 1.0
    st.rhos = rhos.cuda()
    last = torch.where(last >= 0, last - 4600, last)                  # ages up to 5000 steps
    st.last_t.copy_(last.int())
    br = st.fork(S, t0, capacity=16, max_new=n)
    state, last = state.repeat_interleave(S, 0), last.repeat_interleave(S, 0)
    for rnd in range(2):
        tok = torch.randint(0, 40, (B, S, n), generator=g)
        q = torch.randn(B, S, n, H, 64, generator=g).to(dt)
        C = br.extend(tok.cuda())
        O = br.attend(q.cuda(), E_k.cuda(), E_v.cuda(), W.cuda())
        O_ref, C_ref = _rows(state, last, torch.full((B * S,), t0 + rnd * n), tok.view(-1, n), q.view(-1, n, H, 64).double(),
                             E_k.double(), E_v.double(), W.double(), rhos, V)
        assert rel_err(C.cpu().view_as(C_ref), C_ref) < 1e-5
        assert rel_err(O.cpu().view_as(O_ref), O_ref) < TOL[dt]


@pytest.mark.parametrize("S", [1, 3])
def test_strided_operands_other_integers_and_tables_of_other_types(S):
    B, n, V, N, H = 2, 2, 200, 64, 2
    g, rhos, E_k, E_v, W, st, state, last, t0 = _made_up(B, V, N, H, [150, 20], torch.bfloat16, 41)
    a, b = (st.fork(S, t0, capacity=64, max_new=n) for _ in range(2))
    tok = torch.randint(0, V, (B, S, n), generator=g)
    q = torch.randn(B, S, n, H, 64, generator=g).bfloat16()
    tabs = E_k.cuda(), E_v.cuda(), W.cuda()
    wide = torch.zeros(B, S, 2 * n, dtype=torch.int64).cuda()
    wide[..., ::2] = tok.cuda()
    assert torch.equal(a.extend(tok.cuda()), b.extend(wide[..., ::2]))
    O = a.attend(q.cuda(), *tabs)
    q2 = q.cuda().transpose(2, 3).contiguous().transpose(2, 3)
    E2 = torch.zeros(V, 2 * H * 64, dtype=torch.bfloat16).cuda()
    E2[:, ::2] = tabs[0]
    W2 = tabs[2].t().contiguous().t()
    assert torch.equal(O, b.attend(q2, E2[:, ::2], tabs[1].float(), W2))          # (E_v is taken in E_k's type)
    a.keep(torch.tensor([1, 2]).cuda())
    b.keep(torch.tensor([1, 2], dtype=torch.uint8).cuda())
    assert torch.equal(a.lengths, b.lengths)
    a.extend(tok.cuda()), b.extend(tok.cuda())
    assert torch.equal(a.attend(q.cuda(), *tabs), b.attend(q.cuda(), *tabs))
    # fp32 queries with bf16 tables, and the other way round: fp32 arithmetic
    for qd, ed in ((torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)):
        x = a.attend(q.to(qd).cuda(), tabs[0].to(ed), tabs[1].to(ed), tabs[2])
        y = a.attend(q.cuda(), *tabs, mode="fp32")
        assert x.dtype == qd and rel_err(x.float().cpu(), y.float().cpu()) < 2 ** -7          # one rounding to bf16 on either side
        with pytest.raises(Exception, match="tc_bf16"):
            a.attend(q.to(qd).cuda(), tabs[0].to(ed), tabs[1].to(ed), tabs[2], mode="tc_bf16")


@pytest.mark.parametrize("S,n", [(1, 3), (1, 1), (4, 2)])
def test_two_sets_at_once_on_two_streams(S, n):
    """Two sets of branches of one state worked on at once on two streams, against the same work in turn; a repeated call gives the
    same bits."""
    B, V, N, H, rounds = 2, 1000, 64, 2, 6
    g, rhos, E_k, E_v, W, st, *_, t0 = _made_up(B, V, N, H, [900, 400], torch.bfloat16, 51)
    tabs = E_k.cuda(), E_v.cuda(), W.cuda()
    toks = torch.randint(0, V, (2, rounds, B, S, n), generator=g).cuda()
    qs = torch.randn(2, rounds, B, S, n, H, 64, generator=g).bfloat16().cuda()
    sets = [[st.fork(S, t0, capacity=64, max_new=n) for _ in range(2)] for _ in range(2)]

    def work(br, x, i):
        C = br.extend(toks[x, i])
        return C, br.attend(qs[x, i], *tabs), br.attend(qs[x, i], *tabs)

    in_turn = [[work(sets[0][x], x, i) for i in range(rounds)] for x in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    at_once = [[], []]
    for i in range(rounds):
        for x in range(2):
            with torch.cuda.stream(streams[x]):
                at_once[x].append(work(sets[1][x], x, i))
    torch.cuda.synchronize()
    for x in range(2):
        for u, v in zip(in_turn[x], at_once[x]):
            assert all(torch.equal(p, q) for p, q in zip(u, v)) and torch.equal(v[1], v[2])
    assert all(br.device_status() == 0 for pair in sets for br in pair)


@pytest.mark.parametrize("S", [1, 4])
def test_a_sampling_step_replayed_while_the_lists_grow(S):
    """extend (which keeps the call before's tokens) and attend captured after one eager call; replayed, the own lists grow past
    several tiles."""
    B, V, N, H, n, steps = 2, 700, 64, 1, 4, 90
    g, rhos, E_k, E_v, W, st, *_, t0 = _made_up(B, V, N, H, [300, 0], torch.bfloat16, 61)
    tabs = E_k.cuda(), E_v.cuda(), W.cuda()
    toks = torch.randint(0, V, (steps, B, S, n), generator=g).cuda()
    qs = torch.randn(steps, B, S, n, H, 64, generator=g).bfloat16().cuda()
    br, ref = (st.fork(S, t0, capacity=steps * n, max_new=n) for _ in range(2))
    tok, q = toks[0].clone(), qs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        br.extend(tok)
        br.attend(q, *tabs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        C = br.extend(tok)
        O = br.attend(q, *tabs)
    ref.extend(toks[0])
    for i in range(1, steps):
        tok.copy_(toks[i]); q.copy_(qs[i])
        graph.replay()
        C_ref, O_ref = ref.extend(toks[i]), ref.attend(qs[i], *tabs)
        assert torch.equal(C, C_ref) and torch.equal(O, O_ref), i
    assert torch.equal(br.lengths, ref.lengths) and int(br.lengths.min()) == (steps - 1) * n
    br.check_overflow()


def test_no_sequences():
    from mathbrain_b200 import synth
    from mathbrain_b200.decode import DecodeState
    from mathbrain_b200.verify import verify_drafts
    rhos = synth.make_rhos(64, 2.0, 64.0).cuda()
    st = DecodeState(0, 30, rhos, capacity=8)
    br = st.fork(2, 0, capacity=4, max_new=2)
    C = br.extend(torch.zeros(0, 2, 1, dtype=torch.int64).cuda())
    O = br.attend(torch.zeros(0, 2, 1, 1, 64).bfloat16().cuda(), *(torch.zeros(30, 64).bfloat16().cuda() for _ in range(2)), torch.zeros(64, 64).cuda())
    br.keep(torch.zeros(0, dtype=torch.int64).cuda())
    assert C.shape == (0, 2, 1, 64) and O.shape == (0, 2, 1, 1, 64)
    n, out = verify_drafts(torch.zeros(0, 3, 30).cuda(), torch.zeros(0, 2, dtype=torch.int64).cuda(), torch.zeros(0, 3).cuda())
    assert n.shape == (0,) and out.shape == (0, 3)


@pytest.mark.parametrize("S,dt", [(1, torch.bfloat16), (3, torch.bfloat16), (2, torch.float32)])
def test_captured_behind_copies_and_joined_streams(S, dt):
    """A graph in which copies, another stream's work and library kernels stand between the calls; replayed back to back."""
    from mathbrain_b200.verify import verify_drafts
    B, V, N, H, n, rounds = 2, 400, 64, 2, 3, 5
    g, rhos, E_k, E_v, W, st, *_, t0 = _made_up(B, V, N, H, [350, 40], dt, 71)
    tabs = E_k.cuda(), E_v.cuda(), W.cuda()
    toks = torch.randint(0, V, (rounds, B, S, n), generator=g).cuda()
    qs = torch.randn(rounds, B, S, n, H, 64, generator=g).to(dt).cuda()
    us = torch.rand(rounds, B * S, n, generator=g).cuda()
    head = torch.randn(H * 64, V, generator=g).cuda()
    br, ref = (st.fork(S, t0, capacity=rounds * n + n, max_new=n) for _ in range(2))
    side = torch.cuda.Stream()

    def round_(which, tok, q, u, other=None):
        held = torch.empty_like(tok)
        held.copy_(tok)
        if other is not None:                                        # the query comes from another stream
            other.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(other):
                q2 = q * 1.0
        C = which.extend(held)
        if other is not None:
            torch.cuda.current_stream().wait_stream(other)
        O = which.attend(q2 if other is not None else q * 1.0, *tabs)
        p = torch.softmax(O.float().view(B * S, n, H * 64) @ head, -1)
        n_acc, out = verify_drafts(p, held.view(B * S, n)[:, 1:], u)
        which.keep(n_acc.view(B, S).min(1).values + 1)
        return C, O, n_acc, out

    tok, q, u = toks[0].clone(), qs[0].clone(), us[0].clone()
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        spare = st.fork(S, t0, capacity=8, max_new=n)
        round_(spare, tok, q, u)
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = round_(br, tok, q, u, side)
    for i in range(rounds):
        tok.copy_(toks[i]); q.copy_(qs[i]); u.copy_(us[i])
        graph.replay()
        want = round_(ref, toks[i], qs[i], us[i])
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i
    assert torch.equal(br.lengths, ref.lengths)
    br.check_overflow()


@pytest.mark.parametrize("B,S,n,V,N,H", [(5000, 1, 2, 40, 64, 1), (1500, 1, 4, 50, 128, 1), (2000, 3, 2, 40, 64, 1),
                                         (1, 4000, 1, 300, 64, 1), (1, 1, 1, 50257, 64, 1), (1, 3, 1, 50257, 64, 1)])
def test_many_sequences_many_branches_and_the_whole_vocabulary(B, S, n, V, N, H):
    """Thousands of short lists and the longest list there is: the tensor cores against fp32 arithmetic (2e-2 and 1e-4 of the exact)."""
    listed = [(0, V, 7 * i % (V + 1))[i % 3] for i in range(B)] if B > 1 else [V]
    g, rhos, E_k, E_v, W, st, *_, t0 = _made_up(B, V, N, H, listed, torch.bfloat16, 81)
    br = st.fork(S, t0, capacity=64, max_new=8)
    br.extend(torch.randint(0, V, (B, S, 8), generator=g).cuda())
    br.extend(torch.randint(0, V, (B, S, n), generator=g).cuda())
    q = torch.randn(B, S, n, H, 64, generator=g).bfloat16().cuda()
    tabs = E_k.cuda(), E_v.cuda(), W.cuda()
    O, exact = br.attend(q, *tabs), br.attend(q, *tabs, mode="fp32")
    assert rel_err(O.float().cpu(), exact.float().cpu()) < 2e-2 + 1e-4 + 2 ** -8
    assert br.device_status() == 0
    br.check_overflow()
