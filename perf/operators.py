"""Decoding several rows at once against resident slot state, as cases that can be timed and compared: attention of a batch
of continuations or drafted tokens that share their sequence's prefix, the states of the tokens staged for it, and the
verification of drafted tokens.

A case is a dict with a "kind" and its sizes.  prepare(case, seed) makes what a serving program holds before the call,
run(state) is one pass: with `own` through the library's operators, without it in elementary torch operations.

B sequences hold K seen slots each (ragged, the longest K); S branches continue every sequence with L tokens of their own; n new
tokens are staged per branch.  Row j of a branch sees the prefix, the branch's L tokens and its staged tokens before j.
"""
import math

import numpy as np
import torch

own = False

HD = 64                     # head width of every configuration of the model
VOCAB = 50257


def listed():
    return [
        # four samples of a short prompt, the smallest serving call: one new token each
        dict(name="4 samples short prompt", kind="attend", B=1, S=4, n=1, K=150, L=20, H=8, N=64, V=VOCAB, bf16=True),
        # 64 samples of one long document
        dict(name="64 samples long prompt", kind="attend", B=1, S=64, n=1, K=3400, L=300, H=8, N=64, V=VOCAB, bf16=True),
        # four prompts with sixteen long continuations each: the branches' own slots are the larger part
        dict(name="4x16 long answers", kind="attend", B=4, S=16, n=1, K=2000, L=700, H=8, N=64, V=VOCAB, bf16=True),
        # eight rows of one sequence: seven drafted tokens verified at once
        dict(name="8 drafted rows", kind="attend", B=1, S=1, n=8, K=1333, L=5, H=8, N=64, V=VOCAB, bf16=True),
        # a serving batch of 64 sequences with five drafts each: the largest
        dict(name="64 sequences 6 rows", kind="attend", B=64, S=1, n=6, K=3400, L=90, H=8, N=64, V=VOCAB, bf16=True),
        # 128 channels, an odd number of seen slots and branches
        dict(name="24 samples 128 channels", kind="attend", B=2, S=23, n=1, K=4001, L=150, H=8, N=128, V=VOCAB, bf16=True),
        # the exact mode: fp32 tables and queries, drafts in several branches
        dict(name="fp32 drafts in branches", kind="attend", B=2, S=5, n=3, K=701, L=33, H=8, N=64, V=VOCAB, bf16=False),
        # one interactive sequence: the next token's state
        dict(name="stage one token", kind="stage", B=1, S=1, n=1, K=300, L=50, H=8, N=64, V=VOCAB),
        # the states of a serving batch's drafted tokens, all dropped again
        dict(name="stage 64x6 drafts", kind="stage", B=64, S=1, n=6, K=3400, L=90, H=8, N=64, V=VOCAB),
        # one sequence, four drafts
        dict(name="verify one sequence", kind="verify", R=1, G=4, V=VOCAB, bf16=False, draft=True),
        # a large serving batch, seven drafts with the draft model's probabilities
        dict(name="verify 256 sequences", kind="verify", R=256, G=7, V=VOCAB, bf16=False, draft=True),
        # drafts without probabilities (looked up in the text), 16-bit probabilities
        dict(name="verify lookup drafts", kind="verify", R=100, G=3, V=VOCAB, bf16=True, draft=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "attend", "stage", "verify", "verify"])
    V = rng.choice([VOCAB, VOCAB, 32000])
    if kind == "verify":
        return dict(kind="verify", R=_log(rng, 1, 256), G=rng.randint(1, 7), V=V, bf16=rng.random() < 0.4, draft=rng.random() < 0.6)
    N = rng.choice([64, 64, 64, 128])
    K = _log(rng, 40, 4000)
    if rng.random() < 0.5:                  # continuations of shared prompts, a token at a time
        S, n, B = _log(rng, 2, 64), rng.choice([1, 1, 2]), rng.randint(1, 4)
        S = max(1, min(S, 64 // B))
        L = _log(rng, 1, 700)
    else:                                   # drafted tokens
        S, n, B = rng.choice([1, 1, 2]), rng.randint(2, 8), _log(rng, 1, 40)
        L = rng.randint(0, 100)
    bf16 = kind == "stage" or rng.random() < 0.75
    if not bf16:                            # the exact mode, smaller
        B, S, n, K, L, N = min(B, 3), min(S, 8), min(n, 4), min(K, 900), min(L, 60), rng.choice([32, 64, 96, 128])
    B = max(1, min(B, 80_000_000 // (n * K * N)))                             # no more than the largest listed batch
    case = dict(kind=kind, B=B, S=S, n=n, K=K, L=L, H=rng.choice([4, 8, 8]), N=N, V=V)
    return case if kind == "stage" else dict(case, bf16=bf16)


# ------------------------------------------------------------------------------------------------ inputs
def _zipf(V):
    p = torch.arange(1, V + 1, dtype=torch.float64) ** -1.1
    return p / p.sum()


def _rhos(N):
    h = torch.logspace(math.log10(1024.0), math.log10(4096.0), N)          # half-lives of the model's default configuration
    return torch.exp(-math.log(2.0) / h)


def _slots(c, seed):
    """Resident state of B sequences after T0 tokens, their branches' tokens and the staged ones, on the GPU."""
    B, S, n, K, L, N, V = (c[k] for k in ("B", "S", "n", "K", "L", "N", "V"))
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = dict(device="cuda")
    p = _zipf(V).to(**dev)
    rhos = _rhos(N).to(**dev)
    T0 = 4 * K + 7
    race = torch.empty(B, V, **dev).exponential_(generator=g) / p.float()
    active = race.topk(K, dim=1, largest=False).indices                      # a prefix of tokens drawn by their frequency
    active = active.gather(1, torch.rand(B, K, generator=g, **dev).argsort(1)).int()
    n_active = (K - (torch.rand(B, generator=g, **dev) * (K // 3 + 1)).long()).int()
    n_active[0] = K
    state = torch.zeros(B, V, N, **dev)
    last_t = torch.full((B, V), -1, dtype=torch.int32, **dev)
    listed_ = torch.arange(K, **dev) < n_active[:, None]
    rows = torch.arange(B, **dev)[:, None].expand(B, K)[listed_]
    slots = active[listed_].long()
    expect = torch.minimum(p[slots].float()[:, None] / (1 - rhos), torch.tensor(float(T0), **dev))
    state[rows, slots] = 1 + expect * (0.5 + torch.rand(len(slots), 1, generator=g, **dev))
    last_t[rows, slots] = (T0 - 1 - (torch.rand(len(slots), generator=g, **dev) ** 2 * (T0 - 1)).long()).int()
    hist = torch.multinomial(p.float().expand(B * S, V), L + n, replacement=True, generator=g).view(B, S, L + n)
    again = torch.rand(B, S, L + n, generator=g, **dev) < 0.3                 # a continuation takes up words of its document
    pick = (torch.rand(B, S, L + n, generator=g, **dev) * n_active[:, None, None]).long()
    doc = active.long().gather(1, pick.view(B, -1)).view(B, S, L + n)
    hist = torch.where(again, doc, hist)
    return dict(state=state, last_t=last_t, active=active, n_active=n_active, rhos=rhos, T0=T0,
                hist=hist[:, :, :L].contiguous(), tok=hist[:, :, L:].contiguous())


def _branch_tables(s):
    """The slots that every branch has touched so far, with their state right after the last update: [B, S, U]."""
    B, S, L = s["hist"].shape
    V, N = s["state"].shape[1:]
    dev = s["state"].device
    R = B * S
    seq = torch.arange(R, device=dev) // S
    row = torch.arange(R, device=dev)
    index = torch.full((R, V), -1, dtype=torch.long, device=dev)
    slot = torch.zeros(R, max(L, 1), dtype=torch.long, device=dev)
    step = torch.zeros(R, max(L, 1), dtype=torch.long, device=dev)
    value = torch.zeros(R, max(L, 1), N, dtype=torch.float64, device=dev)
    count = torch.zeros(R, dtype=torch.long, device=dev)
    rh = s["rhos"].double()
    for i in range(L):
        v, t = s["hist"][:, :, i].reshape(R), s["T0"] + i
        at = index[row, v]
        fresh = at < 0
        at = torch.where(fresh, count, at)
        last = s["last_t"][seq, v].long()
        from_prefix = s["state"][seq, v].double() * rh ** (t - last)[:, None].double() * (last >= 0)[:, None]
        from_branch = value[row, at] * rh ** (t - step[row, at])[:, None].double()
        value[row, at] = torch.where(fresh[:, None], from_prefix, from_branch) + 1
        index[row, v], slot[row, at], step[row, at] = at, v, t
        count += fresh
    U = max(1, int(count.max())) if L else 1
    return dict(o_slot=slot[:, :U].view(B, S, U), o_step=step[:, :U].view(B, S, U), o_state=value[:, :U].float().view(B, S, U, N),
                o_n=count.view(B, S), index=index.view(B, S, V))


def _rows(s):
    """What the staged rows see, from the tokens alone: masks over the prefix's slots, the branches' and the staged ones, and
    the number of listed slots; what a program's bookkeeping holds beside the state."""
    B, S, n = s["tok"].shape
    V = s["state"].shape[1]
    K = s["active"].shape[1]
    U = s["o_slot"].shape[2]
    dev = s["tok"].device
    act = s["active"].long()
    inside = (torch.arange(K, device=dev) < s["n_active"][:, None])[:, None, None, :]
    touched = s["index"].gather(2, act[:, None].expand(B, S, K)) >= 0
    before = torch.ones(n, n, dtype=torch.bool, device=dev).tril(-1)                 # [row j, staged i]
    hit = torch.zeros(B, S, n, K, dtype=torch.bool, device=dev)
    gone = torch.zeros(B, S, n, U, dtype=torch.bool, device=dev)
    for i in range(n):
        same = act[:, None] == s["tok"][:, :, i:i + 1]
        hit |= same[:, :, None] & before[:, i][None, None, :, None]
        gone |= (s["o_slot"] == s["tok"][:, :, i:i + 1])[:, :, None] & before[:, i][None, None, :, None]
    eq = s["tok"][:, :, :, None] == s["tok"][:, :, None, :]                          # [i, i']
    later = torch.stack([(eq & before[j][None, None, None, :] & before.t()[None, None]).any(-1) for j in range(n)], 2)
    see_staged = before[None, None] & ~later
    first = ~(eq & before[None, None]).any(-1)                                       # not staged before in this call
    new = first & (s["index"].gather(2, s["tok"]) < 0) & (s["last_t"][:, None].expand(B, S, V).gather(2, s["tok"]) < 0)
    o_new = ((s["last_t"][:, None].expand(B, S, V).gather(2, s["o_slot"]) < 0)
             & (torch.arange(U, device=dev) < s["o_n"][:, :, None])).sum(-1)
    listed_ = s["n_active"].long()[:, None, None] + o_new[:, :, None] + (new[:, :, None] & before[None, None]).sum(-1)
    return dict(see_prefix=inside & ~touched[:, :, None] & ~hit, see_staged=see_staged, n_listed=listed_,
                see_branch=(torch.arange(U, device=dev) < s["o_n"][:, :, None])[:, :, None] & ~gone)


def _tables(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed + 500009)
    D, dt = c["H"] * HD, torch.bfloat16 if c["bf16"] else torch.float32
    E_k = (torch.randn(c["V"], D, generator=g, device="cuda") * 0.2).to(dt)
    E_v = (torch.randn(c["V"], D, generator=g, device="cuda") * 0.2).to(dt)
    W = torch.randn(c["N"], D, generator=g, device="cuda") * 0.02
    q = torch.randn(c["B"], c["S"], c["n"], c["H"], HD, generator=g, device="cuda").to(dt)
    return dict(E_k=E_k, E_v=E_v, W=W, q=q)


def _handle(c, s):
    """The handle a program keeps: the sequences' resident state and their branches, brought up to the last kept token."""
    from mathbrain_b200.decode import DecodeState
    B, S, n, L = c["B"], c["S"], c["n"], c["L"]
    st = DecodeState(B, c["V"], s["rhos"], capacity=c["K"])
    st.state, st.last_t, st.active, st.n_active = s["state"], s["last_t"], s["active"], s["n_active"]
    br = st.fork(S, s["T0"], capacity=L + n, max_new=32)
    for i in range(0, L, br.max_new):
        br.extend(s["hist"][:, :, i:i + br.max_new].contiguous())
    if L:
        br.keep(torch.full((B,), (L - 1) % br.max_new + 1, device="cuda"))
    return br


def _probabilities(c, seed):
    """Target and draft distributions that agree more or less, drafts drawn from the draft's, uniform numbers."""
    R, G, V = c["R"], c["G"], c["V"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = torch.bfloat16 if c["bf16"] else torch.float32
    base = torch.randn(R, G + 1, V, generator=g, device="cuda").mul_(2.5)
    p = (base + 0.3 * torch.randn(R, G + 1, V, generator=g, device="cuda")).softmax(-1).to(dt)
    q = (base[:, :G] + 0.5 * torch.randn(R, G, V, generator=g, device="cuda")).softmax(-1).to(dt)
    del base
    drafted = torch.multinomial(q.float().view(R * G, V), 1, generator=g).view(R, G)
    u = torch.rand(R, G + 1, generator=g, device="cuda")
    return dict(p=p, q=q if c["draft"] else None, drafted=drafted, u=u)


def prepare(case, seed):
    c = dict(case)
    if c["kind"] == "verify":
        return dict(kind="verify", **_probabilities(c, seed))
    s = _slots(c, seed)
    none = torch.zeros(c["B"], dtype=torch.long, device="cuda")
    out = dict(kind=c["kind"], V=c["V"], none=none, **s)
    if c["kind"] == "attend":
        out.update(_tables(c, seed))
    if own:
        out["br"] = _handle(c, s)
        if c["kind"] == "attend":
            out["br"].extend(s["tok"])
        return out
    out.update(_branch_tables(s))
    if c["kind"] == "attend":
        out.update(_rows(out))
        out["C_q"] = _staged_states(out)
    return out


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if state["kind"] == "verify":
        return _verify(state)
    return _stage(state) if state["kind"] == "stage" else _attend(state)


def _staged_states(s):
    """State of every staged token just before its own step: the kept state decayed to that step, and the tokens staged before
    it.  Powers of far steps in 64 bits."""
    B, S, n = s["tok"].shape
    N = s["rhos"].shape[0]
    U, L = s["o_slot"].shape[2], s["hist"].shape[2]
    rh = s["rhos"].double()
    tau = s["T0"] + L + torch.arange(n, device=rh.device)
    at = s["index"].gather(2, s["tok"])                                              # [B, S, n]: the branch's slot, or -1
    seq = torch.arange(B, device=rh.device)[:, None, None]
    last = s["last_t"].long()[seq, s["tok"]]
    kept_t = torch.where(at >= 0, s["o_step"].gather(2, at.clamp_min(0)), last)
    kept = torch.where((at >= 0)[..., None], s["o_state"].gather(2, at.clamp_min(0)[..., None].expand(B, S, n, N)), s["state"][seq, s["tok"]])
    C = kept.double() * rh ** (tau - kept_t)[..., None].double() * ((at >= 0) | (last >= 0))[..., None]
    age = (tau[:, None] - tau[None, :])
    same = (s["tok"][:, :, :, None] == s["tok"][:, :, None, :]) & (age > 0)
    C = C + torch.einsum("bsij,ijn->bsin", same.double(), rh ** age.clamp_min(0)[..., None].double())
    return C.float()


def _stage(s):
    if own:
        C_q = s["br"].extend(s["tok"])
        s["br"].keep(s["none"])
        return C_q
    return _staged_states(s)


def _scores(q, E, W, M):
    """Gate of the slots, and their scores and values: M [..., items, N], E (k and v) [..., items, D], q [..., rows, H, 64]."""
    x = M @ W
    gate = x * torch.sigmoid(x)
    k = (E[0].float() * gate).unflatten(-1, (-1, HD))
    v = (E[1].float() * gate).unflatten(-1, (-1, HD))
    return torch.einsum("...rhd,...khd->...rhk", q, k) * HD ** -0.5, v


def _attend(s):
    if own:
        return s["br"].attend(s["q"], s["E_k"], s["E_v"], s["W"])
    B, S, n, H, _ = s["q"].shape
    L = s["hist"].shape[2]
    rh, W, q = s["rhos"].double(), s["W"].float(), s["q"].float()
    E = (s["E_k"], s["E_v"])
    tau = s["T0"] + L + torch.arange(n, device=rh.device)
    act = s["active"].long()
    seq = torch.arange(B, device=rh.device)[:, None]
    age = (tau[None, :, None] - s["last_t"].long()[seq, act][:, None]).clamp_min(0)               # [B, n, K]
    M = (s["state"][seq, act][:, None] * torch.exp(age[..., None].double() * rh.log()).float())   # [B, n, K, N]
    sc, v = _scores(q.transpose(1, 2), [e[act][:, None] for e in E], W, M)                        # rows: the branches at one step
    sc = sc.transpose(1, 2).masked_fill(~s["see_prefix"][:, :, :, None], -math.inf)               # [B, S, n, H, K]
    age = tau[:, None] - s["o_step"][:, :, None]                                                  # [B, S, n, U]
    M = s["o_state"][:, :, None] * torch.exp(age[..., None].double() * rh.log()).float()
    sb, vb = _scores(q[:, :, :, None], [e[s["o_slot"]][:, :, None] for e in E], W, M)
    sb = sb[:, :, :, 0].masked_fill(~s["see_branch"][:, :, :, None], -math.inf)
    age = (tau[:, None] - tau[None, :]).clamp_min(0)                                              # [row, staged]
    M = (s["C_q"] + 1)[:, :, None] * torch.exp(age[..., None].double() * rh.log()).float()
    ss, vs = _scores(q[:, :, :, None], [e[s["tok"]][:, :, None] for e in E], W, M)
    ss = ss[:, :, :, 0].masked_fill(~s["see_staged"][:, :, :, None], -math.inf)
    rest = (s["V"] - s["n_listed"]).float()[..., None]                                            # slots with score 0 and value 0
    m = torch.cat([sc, sb, ss], -1).amax(-1).clamp_min(0)
    a, b, c = (torch.exp(t - m[..., None]) for t in (sc, sb, ss))
    total = a.sum(-1) + b.sum(-1) + c.sum(-1) + rest * torch.exp(-m)
    out = (torch.einsum("bsnhk,bnkhd->bsnhd", a, v) + torch.einsum("bsnhk,bsnkhd->bsnhd", b, vb)
           + torch.einsum("bsnhk,bsnkhd->bsnhd", c, vs))
    return (out / total[..., None]).to(s["q"].dtype)


def _verify(s):
    if own:
        from mathbrain_b200.verify import verify_drafts
        return verify_drafts(s["p"], s["drafted"], s["u"], p_draft=s["q"])
    p, q, x, u = s["p"], s["q"], s["drafted"], s["u"].double()
    R, G = x.shape
    V = p.shape[-1]
    px = p[:, :G].gather(2, x[..., None])[..., 0].double()
    qx = torch.ones_like(px) if q is None else q.gather(2, x[..., None])[..., 0].double()
    accepted = (u[:, :G] * qx < px).long().cumprod(1).sum(1)
    row = torch.arange(R, device=p.device)
    pa = p[row, accepted].double()
    at = accepted.clamp_max(G - 1)
    if q is None:
        qa = torch.zeros_like(pa).scatter_(1, x[row, at][:, None], 1.0)
    else:
        qa = q[row, at].double()
    w = torch.where((accepted == G)[:, None], pa, (pa - qa).clamp_min(0))
    w = torch.where(w.sum(1, keepdim=True) > 0, w, pa)
    cum = w.cumsum(1)
    nxt = (cum <= u[:, G:] * cum[:, -1:]).sum(1).clamp_max(V - 1)
    place = torch.arange(G + 1, device=p.device)
    tokens = torch.cat([x, x[:, :1]], 1)
    tokens = torch.where(place < accepted[:, None], tokens, torch.where(place == accepted[:, None], nxt[:, None], -1))
    return accepted, tokens


# ------------------------------------------------------------------------------------------------ what a pass costs
def _distinct(c, lists):
    """Distinct tokens expected in `lists` prefixes of K frequent-first tokens."""
    p = _zipf(c["V"]).numpy()
    lo, hi = 0.0, 1e12
    for _ in range(80):
        mid = math.sqrt(max(lo, 1e-6) * hi)
        lo, hi = (mid, hi) if (1 - np.exp(-mid * p)).sum() < c["K"] else (lo, mid)
    seen = 1 - np.exp(-hi * p)
    return float((1 - (1 - seen) ** lists).sum())


def work(case):
    c = case
    if c["kind"] == "verify":       # the drafts' probabilities, one distribution for the next token (and the draft's after a rejection)
        size = 2 if c["bf16"] else 4
        rows = c["V"] * size * (2 if c["draft"] else 1)
        return {"bytes": c["R"] * (rows + (c["G"] + 1) * 16 + c["G"] * (8 + 64) + 8), "flops": 2 * c["R"] * c["V"]}
    B, S, n, K, L, N, D = c["B"], c["S"], c["n"], c["K"], c["L"], c["N"], c["H"] * HD
    if c["kind"] == "stage":        # the tokens, the kept state of each, the states of the rows
        return {"bytes": B * S * n * (8 + 4 + 2 * 4 * N), "flops": B * S * n * 3 * N}
    size = 2 if c["bf16"] else 4
    K = K * 5 / 6                   # ragged: mean number of seen slots
    U = 0.6 * L                     # distinct tokens of a branch, about
    bytes_ = (_distinct(c, B) * 2 * D * size                                     # rows of E_k and E_v, once
              + B * K * (4 * N + 8) + B * S * U * (4 * N + 8)                    # states, slots, steps
              + B * S * n * D * 2 * size + N * D * 4)
    pairs = B * S * n * (K + U)                                                  # (row, slot)
    gates = B * n * K + B * S * n * U                                            # (step, slot) of the prefix once for all branches
    return {"bytes": bytes_, "flops": gates * 2 * N * D + pairs * 4 * D}


# ------------------------------------------------------------------------------------------------ in 64 bits, from the definition
def _exact_state(s, b, br, j, slots):
    """M [slots, N] of the slots at row j: the prefix's state decayed, and a power for every occurrence in the branch."""
    L = s["hist"].shape[2]
    rh = s["rhos"].double()
    now = s["T0"] + L + j
    last = s["last_t"][b, slots].double()
    M = torch.where(last[:, None] >= 0, s["state"][b, slots].double() * rh ** (now - last)[:, None], 0.0)
    seen = torch.cat([s["hist"][b, br], s["tok"][b, br, :j]])
    where = torch.full((s["last_t"].shape[1],), -1, dtype=torch.long, device=rh.device)
    where[slots] = torch.arange(len(slots), device=rh.device)
    age = (now - s["T0"] - torch.arange(len(seen), device=rh.device)).double()
    keep = where[seen] >= 0
    return M.index_add(0, where[seen][keep], (rh ** age[:, None])[keep])


def exact(case, seed):
    c = dict(case)
    if c["kind"] == "verify":
        s = _probabilities(c, seed)
        accepted, tokens = [], []
        x, u = s["drafted"].cpu().numpy(), s["u"].double().cpu().numpy()
        for r in range(c["R"]):
            out, nxt = [], None
            for j in range(c["G"]):
                t = x[r, j]
                q_of = 1.0 if s["q"] is None else float(s["q"][r, j, t])
                if u[r, j] * q_of < float(s["p"][r, j, t]):
                    out.append(int(t))
                    continue
                w = s["p"][r, j].double().cpu().numpy()
                if s["q"] is None:
                    d = w.copy()
                    d[t] = max(d[t] - 1.0, 0.0)
                else:
                    d = np.maximum(w - s["q"][r, j].double().cpu().numpy(), 0.0)
                nxt = d if d.sum() > 0 else w
                break
            if nxt is None:
                nxt = s["p"][r, c["G"]].double().cpu().numpy()
            run_ = np.cumsum(nxt)
            out.append(int(np.searchsorted(run_, u[r, c["G"]] * run_[-1], side="right")))
            accepted.append(len(out) - 1)
            tokens.append(out + [-1] * (c["G"] + 1 - len(out)))
        return torch.tensor(accepted), torch.tensor(tokens)
    s = _slots(c, seed)
    B, S, n, H = c["B"], c["S"], c["n"], c["H"]
    if c["kind"] == "stage":
        return torch.stack([torch.stack([torch.cat([_exact_state(s, b, r, j, s["tok"][b, r, j:j + 1]) for j in range(n)])
                                         for r in range(S)]) for b in range(B)])
    t = _tables(c, seed)
    out = torch.zeros(B, S, n, H, HD, dtype=torch.float64, device="cuda")
    for b in range(B):
        seen_b = s["active"][b, :s["n_active"][b]].long()
        for r in range(S):
            for j in range(n):
                slots = torch.unique(torch.cat([seen_b, s["hist"][b, r], s["tok"][b, r, :j]]))
                x = _exact_state(s, b, r, j, slots) @ t["W"].double()
                gate = (x / (1 + torch.exp(-x))).view(-1, H, HD)
                k = t["E_k"][slots].double().view(-1, H, HD) * gate
                v = t["E_v"][slots].double().view(-1, H, HD) * gate
                z = (k * t["q"][b, r, j].double()).sum(-1) / 8.0                 # [slots, H]
                top = z.amax(0).clamp_min(0)
                e = torch.exp(z - top)
                out[b, r, j] = (e[..., None] * v).sum(0) / (e.sum(0) + (c["V"] - len(slots)) * torch.exp(-top))[:, None]
    return out
