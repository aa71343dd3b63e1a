"""Branches of a decode state where values, options and reports are unusual; results are equal, or NaN, or not."""
import pytest
import torch

from test_gpu_branches_use import _made_up

pytestmark = pytest.mark.gpu

FORMS = [(1, torch.bfloat16, 64, None), (3, torch.bfloat16, 64, None), (1, torch.bfloat16, 128, None), (3, torch.bfloat16, 128, None),
         (1, torch.bfloat16, 64, "fp32"), (3, torch.float32, 20, None)]


@pytest.mark.parametrize("S,dt,N,mode", FORMS)
def test_a_state_that_is_nan_reaches_the_rows_that_see_it(S, dt, N, mode):
    """In a prefix slot: every row of the sequence, not the other sequence's.  In an own slot: the rows of its branch."""
    B, n, V, H = 2, 2, 300, 2
    g, rhos, E_k, E_v, W, st, *_, t0 = _made_up(B, V, N, H, [200, 40], dt, 91)
    tabs = E_k.cuda(), E_v.cuda(), W.cuda()
    q = torch.randn(B, S, n, H, 64, generator=g).to(dt).cuda()
    first = torch.randint(0, V, (B, S, n), generator=g).cuda()
    tok = torch.randint(0, V, (B, S, n), generator=g).cuda()

    def run(into):
        br = st.fork(S, t0, capacity=8, max_new=n)
        br.extend(first)
        br.keep(torch.full((B,), n).cuda())
        into(br)
        br.extend(tok)
        return br.attend(q, *tabs, mode=mode).isnan()

    assert not run(lambda br: None).any()

    def own(br):
        br._hold["own_state"][1, S - 1, 0, N // 2] = float("nan")
    seen = run(own)
    assert seen[1, S - 1].all() and not seen[0].any() and not seen[1, :S - 1].any()
    slot = next(v for v in st.active[0, :200].tolist() if v not in first[0].flatten().tolist() + tok[0].flatten().tolist())
    st.state[0, slot, 5] = float("nan")
    seen = run(lambda br: None)
    assert seen[0].all() and not seen[1].any()


@pytest.mark.parametrize("S,dt,N,mode", FORMS)
def test_a_gate_weight_that_is_nan_reaches_its_head(S, dt, N, mode):
    B, n, V, H = 1, 2, 100, 2
    g, rhos, E_k, E_v, W, st, *_, t0 = _made_up(B, V, N, H, [60], dt, 92)
    W[N - 1, 64 + 7] = float("nan")
    br = st.fork(S, t0, capacity=8, max_new=n)
    br.extend(torch.randint(0, V, (B, S, n), generator=g).cuda())
    q = torch.randn(B, S, n, H, 64, generator=g).to(dt).cuda()
    O = br.attend(q, E_k.cuda(), E_v.cuda(), W.cuda(), mode=mode)
    assert O[..., 1, :].isnan().all() and O[..., 0, :].isfinite().all()


@pytest.mark.parametrize("N,S,offset", [(32, 3, 1), (96, 1, 2), (4, 2, 3), (20, 1, 1)])
def test_a_state_at_any_offset(N, S, offset):
    """A contiguous view that starts between two 16-byte pieces: the same results."""
    B, n, V, H = 2, 2, 90, 1
    g, rhos, E_k, E_v, W, st, *_, t0 = _made_up(B, V, N, H, [70, 12], torch.float32, 90)
    tabs = E_k.cuda(), E_v.cuda(), W.cuda()
    tok = torch.randint(0, V, (2, B, S, n), generator=g).cuda()
    q = torch.randn(B, S, n, H, 64, generator=g).cuda()

    def run():
        br = st.fork(S, t0, capacity=8, max_new=n)
        br.extend(tok[0])
        return br.extend(tok[1]), br.attend(q, *tabs)

    want = run()
    buf = torch.empty(st.state.numel() + 4, device="cuda")
    view = buf[offset:offset + st.state.numel()].view_as(st.state)
    view.copy_(st.state)
    st.state = view
    assert view.data_ptr() % 16 != 0 and all(torch.equal(a, b) for a, b in zip(run(), want))


def test_reports_do_not_replace_one_another():
    """A full own list, then a token outside the vocabulary: both are reported, by the branches and, after adopt, by the state."""
    from mathbrain_b200 import _lib
    B, V, N, H = 1, 60, 16, 1
    g, rhos, E_k, E_v, W, st, *_, t0 = _made_up(B, V, N, H, [20], torch.float32, 95)
    br = st.fork(1, t0, capacity=2, max_new=3)
    br.extend(torch.tensor([[[10, 11, 12]]]).cuda())
    br.keep(torch.tensor([3]).cuda())
    br.extend(torch.tensor([[[V, 11, -1]]]).cuda())
    br.adopt(torch.tensor([0]).cuda(), t0 + 6)
    for who in (br, st):
        for what in ("full", "vocabulary"):
            with pytest.raises(_lib.MbemaError, match=what):
                who.check_overflow()
    other = type(st)(B, V, rhos.cuda(), capacity=1)                   # the state's own reports
    for t, tok in enumerate((3, 4, V, 5, -2)):
        other.update(torch.tensor([tok]).cuda(), t)
    for what in ("full", "vocabulary"):
        with pytest.raises(_lib.MbemaError, match=what):
            other.check_overflow()


def _state_of(st):
    return [getattr(st, k).clone() for k in ("state", "last_t", "active", "n_active")]


@pytest.mark.parametrize("what", ["branch", "t_next"])
@pytest.mark.parametrize("device_step", [False, True])
def test_a_refused_adopt_moves_no_sequence_and_is_reported(what, device_step):
    """One sequence's branch (or end) cannot be taken: the whole batch stays where it was, step number included, and the state says so."""
    from mathbrain_b200 import _lib
    B, S, V, N, H = 3, 2, 50, 16, 1
    g, rhos, E_k, E_v, W, st, *_, t0 = _made_up(B, V, N, H, [20, 5, 0], torch.float32, 93)
    if device_step:
        st.use_device_step(t0)
    br = st.fork(S, t0, capacity=8, max_new=3)
    br.extend(torch.randint(0, V, (B, S, 3), generator=g).cuda())
    br.keep(torch.tensor([1, 3, 2]).cuda())
    before = _state_of(st)
    branch, t_next = (torch.tensor([0, 1, S]), t0 + 3) if what == "branch" else (torch.tensor([0, 1, 1]), t0 + 2)
    br.adopt(branch.cuda(), t_next)
    assert all(torch.equal(a, b) for a, b in zip(before, _state_of(st)))
    if device_step:
        assert int(st.t_dev) == t0
    for who in (br, st):
        with pytest.raises(_lib.MbemaError, match=what):
            who.check_overflow()
    # the state goes on from where it stands, and the report stays
    st.update(torch.tensor([1, 2, V + 3]).cuda(), t0)
    with pytest.raises(_lib.MbemaError, match=what):
        st.check_overflow()
    with pytest.raises(_lib.MbemaError, match="vocabulary"):
        st.check_overflow()


def test_an_adopt_moves_the_device_step():
    B, S, V, N, H = 2, 2, 50, 16, 1
    g, rhos, E_k, E_v, W, st, *_, t0 = _made_up(B, V, N, H, [20, 5], torch.float32, 94)
    st.use_device_step(t0)
    br = st.fork(S, 0, capacity=8, max_new=3)
    br.extend(torch.randint(0, V, (B, S, 3), generator=g).cuda())
    br.keep(torch.tensor([1, 3]).cuda())
    before = _state_of(st)
    br.adopt(torch.tensor([1, 0]).cuda(), t0 + 9)
    assert int(st.t_dev) == t0 + 9 and not torch.equal(before[1], st.last_t)
    st.check_overflow()
    br.check_overflow()


def test_branches_of_no_sequences_report_nothing():
    from mathbrain_b200 import synth
    from mathbrain_b200.decode import DecodeState
    rhos = synth.make_rhos(64, 2.0, 64.0).cuda()
    junk = [torch.full((1,), 5, dtype=torch.int32).cuda() for _ in range(64)]          # small blocks that the next allocations get
    del junk
    st = DecodeState(0, 30, rhos, capacity=8)
    br = st.fork(2, 0, capacity=4, max_new=2)
    br.extend(torch.zeros(0, 2, 1, dtype=torch.int64).cuda())
    br.check_overflow()
    br.adopt(torch.zeros(0, dtype=torch.int64).cuda(), 3)
    br.check_overflow()
    st.check_overflow()


@pytest.mark.parametrize("N,dt,qd", [(64, torch.float32, torch.float32), (64, torch.bfloat16, torch.float32), (20, torch.bfloat16, torch.bfloat16)])
def test_the_package_option_is_a_preference(N, dt, qd):
    """mode 'tc_bf16' as the package option: operands that the tensor cores do not take go through fp32 arithmetic, as a decode step
    does; asked for in the call it is refused."""
    import mathbrain_b200 as mb
    from mathbrain_b200 import _lib
    B, S, n, V, H = 1, 2, 2, 60, 1
    g, rhos, E_k, E_v, W, st, *_, t0 = _made_up(B, V, N, H, [30], dt, 96)
    tabs = E_k.cuda(), E_v.cuda(), W.cuda()
    q = torch.randn(B, S, n, H, 64, generator=g).to(qd).cuda()
    br = st.fork(S, t0, capacity=8, max_new=n)
    br.extend(torch.randint(0, V, (B, S, n), generator=g).cuda())
    exact = br.attend(q, *tabs, mode="fp32")
    was = mb.get_options()["mode"]
    try:
        mb.set_options(mode="tc_bf16")
        assert torch.equal(br.attend(q, *tabs), exact)
        with pytest.raises(_lib.MbemaError, match="tc_bf16"):
            br.attend(q, *tabs, mode="tc_bf16")
    finally:
        mb.set_options(mode=was)


def test_the_number_of_slots_is_read_at_every_call():
    B, S, n, V, N, H = 1, 2, 1, 60, 16, 1
    g, rhos, E_k, E_v, W, st, *_, t0 = _made_up(B, V, N, H, [30], torch.float32, 97)
    tabs = E_k.cuda(), E_v.cuda(), W.cuda()
    q = torch.randn(B, S, n, H, 64, generator=g).cuda()
    br = st.fork(S, t0, capacity=8, max_new=n)
    br.extend(torch.randint(0, V, (B, S, n), generator=g).cuda())
    total = torch.tensor(V)
    for v in (V, 4 * V, 40):
        total.fill_(v)
        assert torch.equal(br.attend(q, *tabs, V_total=total), br.attend(q, *tabs, V_total=v)), v


@pytest.mark.parametrize("B,S,n,N,H,dt", [(1, 1, 5, 64, 2, torch.bfloat16), (1, 3, 4, 64, 1, torch.bfloat16), (20, 1, 9, 128, 2, torch.bfloat16),
                                          (2, 2, 6, 24, 2, torch.float32)])
def test_every_call_sees_what_was_written_before_it(B, S, n, N, H, dt):
    """Tables, weights, queries and tokens rewritten in place between calls that follow one another without a pause, tokens kept and
    dropped in turn, against the same calls with the device at rest between them."""
    V, rounds = 200, 12
    g, rhos, E_k, E_v, W, st, *_, t0 = _made_up(B, V, N, H, [150 - i for i in range(B)], dt, 98)
    toks = torch.randint(0, V, (rounds, B, S, n), generator=g).cuda()
    qs = torch.randn(rounds, B, S, n, H, 64, generator=g).to(dt).cuda()
    Es = (torch.randn(rounds, 2, V, 64 * H, generator=g) * 0.2).to(dt).cuda()
    Ws = (torch.randn(rounds, N, 64 * H, generator=g) * 0.1).cuda()
    counts = torch.randint(0, n + 1, (rounds, B), generator=g).cuda()

    def run(pause):
        br = st.fork(S, t0, capacity=rounds * n, max_new=n)
        tok, q, E, w = toks[0].clone(), qs[0].clone(), Es[0].clone(), Ws[0].clone()
        out = []
        for i in range(rounds):
            for dst, src in ((tok, toks), (E, Es), (q, qs), (w, Ws)):
                dst.copy_(src[i])
            pause()
            C = br.extend(tok)
            pause()
            O = br.attend(q, E[0], E[1], w)
            w.mul_(0.5)
            q.mul_(2.0)
            pause()
            O2 = br.attend(q, E[0], E[1], w)
            pause()
            if i % 3:
                br.keep(counts[i])
                pause()
            out += [C, O, O2]
        br.check_overflow()
        return out

    assert all(torch.equal(a, b) for a, b in zip(run(lambda: None), run(torch.cuda.synchronize)))
