"""Branches of a decode state: several continuations or drafted tokens of every sequence, attended together.

    br = st.fork(S, t_now)                       # st: DecodeState of B sequences, at step t_now
    C_q = br.extend(tok)                         # tok int64 [B, S, n]: n new tokens a branch; C_q [B, S, n, N] for the query gate
    O = br.attend(q, E_k, E_v, W_pe)             # q [B, S, n, H, 64] -> O, once a layer
    br.keep(counts)                              # counts [B]: the first counts[b] of the n tokens stay
    br.adopt(branch, t_next)                     # branch [B]: one branch of every sequence becomes the state of `st`

Row j of a branch is one iteration of the reference's loop body (mathbrain/flash_ema_attention.py:46-82), as a decode step is: it
sees the slots of the sequence's prefix, the branch's kept tokens and its staged tokens before j.  The prefix stays where it is
and is read by all branches; a branch holds only the slots that it has touched.

Sampling: S continuations of a prompt, `extend` with one token each; the tokens of the call before are kept by themselves.
Drafts:   S = 1, `extend` with the last token and G drafted ones; `verify_drafts` (mathbrain_b200/verify.py) says how many stand,
          `keep(n_accepted + 1)` drops the others.
Scoring candidates: `extend`, `attend`, `keep` of zeros.

The calls can be captured in CUDA graphs.  A captured `extend` keeps as many tokens at every replay as were staged when it was captured:
capture a sampling step after one eager `extend`, a drafting round from `extend` to `keep`.
"""
import ctypes

import torch

from . import _lib
from .decode import raise_reports
from .ops import _OPTIONS, _current_device, _dt, _ptr, _raw_stream, _require_cuda

_INTEGERS = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)


class Branches:
    """Made by DecodeState.fork.  While the branches live the state must not be updated (its own tokens are the branches'
    prefix); a call on them after an update raises (one by a replayed graph is not noticed).  Memory: 4 bytes for each token of the
    vocabulary a sequence, 4 N (with 64 or 128 channels 6 N) for each of capacity slots a branch, and, with 64 or 128 channels, 2 N for
    each slot of the state's capacity."""

    def __init__(self, prefix, branches, t_now, capacity=1024, max_new=16):
        B, V, N, Kcap = prefix.B, prefix.V, prefix.N, prefix.cap
        S, cap, max_new = int(branches), int(capacity), int(max_new)
        if S < 1 or cap < 1 or not 1 <= max_new <= 32:
            raise _lib.MbemaError("fork: %d branches of capacity %d with %d new tokens at most (1 to 32)" % (S, cap, max_new))
        self.prefix, self.B, self.S, self.V, self.N = prefix, B, S, V, N
        self.capacity, self.max_new = cap, max_new
        self._epoch = prefix._epoch
        self._staged = 0             # tokens of the last extend that keep has not decided on
        dev = prefix.state.device
        expected = (("state", torch.float32, (B, V, N)), ("last_t", torch.int32, (B, V)), ("active", torch.int32, (B, Kcap)),
                    ("n_active", torch.int32, (B,)), ("rhos", torch.float32, (N,)))
        for name, dtype, shape in expected:
            t = getattr(prefix, name)
            if t.device != dev or t.dtype != dtype or t.shape != shape or not t.is_contiguous():
                raise _lib.MbemaError("fork: the state's %s is %s %s on %s, expected contiguous %s %s on %s"
                                      % (name, t.dtype, tuple(t.shape), t.device, dtype, shape, dev))
        _require_cuda(prefix.state)
        i32, f32 = dict(dtype=torch.int32, device=dev), dict(dtype=torch.float32, device=dev)
        self._hold = dict(
            rhos=prefix.rhos, state=prefix.state, last_t=prefix.last_t, active=prefix.active, n_active=prefix.n_active,
            pos=torch.empty(B, V, **i32), t0=torch.empty(1, **i32), len=torch.empty(B, S, **i32), own_n=torch.empty(B, S, **i32),
            own_new=torch.empty(B, S, **i32), own_slot=torch.empty(B, S, cap, **i32), own_t=torch.empty(B, S, cap, **i32),
            own_state=torch.empty(B, S, cap, N, **f32), touched=torch.empty(B, S, (Kcap + 31) // 32, **i32),
            st_tok=torch.empty(B, S, max_new, **i32), st_own=torch.empty(B, S, max_new, **i32),
            st_pos=torch.empty(B, S, max_new, **i32), st_same=torch.empty(B, S, max_new, **i32),
            st_new=torch.empty(B, S, max_new, **i32), st_state=torch.empty(B, S, max_new, N, **f32), overflow=torch.zeros(1, **i32))
        self._tensor_cores = N in (64, 128)
        if self._tensor_cores:
            self._hold.update(pre_op=torch.empty(B, (Kcap + 127) // 128 * 128, N, dtype=torch.float16, device=dev),
                              own_op=torch.empty(B, S, (cap + 127) // 128 * 128, N, dtype=torch.float16, device=dev),
                              work=torch.empty(B * ((S + 15) // 16 + S) + 1, 2, **i32), status=torch.zeros(1, **i32))
        self._c = _lib.BranchesStruct(**{k: _ptr(t) for k, t in self._hold.items()}, B=B, S=S, V=V, N=N, Kcap=Kcap, cap=cap,
                                      max_new=max_new)
        self._ref = ctypes.byref(self._c)
        self._lib = _lib.load()
        self._device, self._dev = dev, prefix.state.get_device()
        self._plans = {}
        with torch.cuda.device(dev):
            rc = self._lib.mbema_branches_init(self._ref, int(t_now), _ptr(prefix.t_dev), _raw_stream(self._dev))
        _lib.check(rc, "mbema_branches_init")

    def _alive(self):
        if self.prefix is None:
            raise _lib.MbemaError("branches: adopted already")
        if self.prefix._epoch != self._epoch:
            raise _lib.MbemaError("branches: the state they were forked from has been updated since")

    def _refuse(self, *operands):
        for t in operands:
            if t.get_device() != self._dev:
                raise _lib.MbemaError("branches: operand on %s, state on %s" % (t.device, self._hold["state"].device))

    def _on_device(self, fn, *args):
        if self._dev == _current_device():
            return fn(*args)
        with torch.cuda.device(self._dev):
            return fn(*args)

    def extend(self, tok):
        """Stage n <= max_new new tokens of every branch (int64 [B, S, n]; -1: this branch has none at this step) and return
        C_q [B, S, n, N] float32, the state of each token just before its own step (0 if never seen).  Tokens staged by the
        call before are kept unless `keep` has decided on them."""
        self._alive()
        if tok.get_device() != self._dev:
            self._refuse(tok)
        shape = tok.shape
        if len(shape) != 3 or shape[0] != self.B or shape[1] != self.S or not 1 <= shape[2] <= self.max_new:
            raise _lib.MbemaError("extend: tokens %s, expected [%d, %d, 1 to %d]" % (tuple(shape), self.B, self.S, self.max_new))
        if tok.dtype != torch.int64:
            raise _lib.MbemaError("extend: tokens of %s, expected int64" % tok.dtype)
        if self._dev == _current_device():
            return self._extend(tok.contiguous())
        with torch.cuda.device(self._dev):
            return self._extend(tok.contiguous())

    def _extend(self, tok):
        n = tok.shape[2]
        C_q = torch.empty((self.B, self.S, n, self.N), dtype=torch.float32, device=self._device)
        rc = self._lib.mbema_branches_extend(self._ref, tok.data_ptr(), n, self._staged, C_q.data_ptr(), _raw_stream(self._dev))
        if rc:
            _lib.check(rc, "mbema_branches_extend")
        self._staged = n
        return C_q

    def keep(self, counts):
        """Keep the first counts[b] of the staged tokens in every branch of sequence b and drop the others (integers [B] on
        the GPU; clamped to 0..n).  The branches then have no staged tokens until the next `extend`."""
        self._alive()
        if counts.get_device() != self._dev:
            self._refuse(counts)
        if counts.dim() != 1 or counts.shape[0] != self.B or counts.dtype not in _INTEGERS:
            raise _lib.MbemaError("keep: counts %s of %s, expected [%d] integers" % (tuple(counts.shape), counts.dtype, self.B))
        if counts.dtype != torch.int64:
            counts = counts.long()
        return self._on_device(self._keep, counts.contiguous())

    def _keep(self, counts):
        rc = self._lib.mbema_branches_keep(self._ref, counts.data_ptr(), self._staged, _raw_stream(self._dev))
        if rc:
            _lib.check(rc, "mbema_branches_keep")
        self._staged = 0

    def attend(self, q, E_k, E_v, W_pe, V_total=None, use_silu=True, listed_only=False, mode=None):
        """O [B, S, n, H, 64] of q's dtype for the n staged rows of every branch.  q [B, S, n, H, 64] float32 or bfloat16;
        E_k, E_v [V, H*64] projected slot embeddings; W_pe [N, H*64].  Softmax over all V_total slots (the vocabulary by
        default), those that a row does not see with score 0 and value 0; listed_only: over the seen ones alone (a row that
        has seen none gets 0).  E_v is taken in E_k's type.  mode: "fp32", "tc_bf16" or "auto".  The tensor cores take
        bfloat16 q and tables with 64 or 128 channels; "auto" runs anything else in fp32 arithmetic, "tc_bf16" refuses it.
        Without one the package option `mode` decides: "fp32" as such, the others as "auto".
        On the tensor cores states and W_pe are fp16 operands: states above 4.19 million and |W_pe| above 1023 count as that."""
        self._alive()
        dev = self._dev
        if q.get_device() != dev or E_k.get_device() != dev or E_v.get_device() != dev or W_pe.get_device() != dev:
            self._refuse(q, E_k, E_v, W_pe)
        if mode is None:                       # (the option is a preference, as for a decode step: it refuses nothing)
            mode = "fp32" if _OPTIONS["mode"] == "fp32" else "auto"
        if V_total is not None:                # (numbers: a tensor's value may change between calls)
            V_total = int(V_total)
        use_silu, listed_only = bool(use_silu), bool(listed_only)
        # checked and sized once for operands of the same shapes, types and options
        key = (q.shape, q.dtype, E_k.shape, E_k.dtype, E_v.shape, E_v.dtype, W_pe.shape, W_pe.dtype, self._staged, V_total, use_silu,
               listed_only, mode)
        plan = self._plans.get(key)
        if plan is None:
            plan = self._plan(q, E_k, E_v, W_pe, V_total, use_silu, listed_only, mode)
            if len(self._plans) >= 64:
                self._plans.clear()
            self._plans[key] = plan
        if dev == _current_device():
            return self._attend(q, E_k, E_v, W_pe, plan)
        with torch.cuda.device(dev):
            return self._attend(q, E_k, E_v, W_pe, plan)

    def _plan(self, q, E_k, E_v, W_pe, V_total, use_silu, listed_only, mode):
        """(arguments of the C call behind O, workspace bytes, whether E_v or W_pe have to be cast)."""
        n = self._staged
        if n == 0:
            raise _lib.MbemaError("attend: no staged tokens (call extend first)")
        if q.dim() != 5 or q.shape[:3] != (self.B, self.S, n) or q.shape[4] != 64 or q.shape[3] < 1:
            raise _lib.MbemaError("attend: q %s, expected [%d, %d, %d, H, 64]" % (tuple(q.shape), self.B, self.S, n))
        H = q.shape[3]
        D = H * 64
        if E_k.shape != (self.V, D) or E_v.shape != (self.V, D) or W_pe.shape != (self.N, D):
            raise _lib.MbemaError("attend: E_k %s, E_v %s, W_pe %s, expected [%d, %d] twice and [%d, %d]"
                                  % (tuple(E_k.shape), tuple(E_v.shape), tuple(W_pe.shape), self.V, D, self.N, D))
        q_dt, e_dt = _dt(q), _dt(E_k)
        if mode not in ("fp32", "tc_bf16", "auto"):
            raise ValueError("mode must be 'fp32', 'tc_bf16' or 'auto'")
        fits = self._tensor_cores and q_dt == _lib.BF16 and e_dt == _lib.BF16
        if mode == "tc_bf16" and not fits:
            raise _lib.MbemaError("attend: mode 'tc_bf16' needs bfloat16 q and tables and 64 or 128 channels (%s, %s, %d)"
                                  % (q.dtype, E_k.dtype, self.N))
        code = _lib.MODE_TC_BF16 if fits and mode != "fp32" else _lib.MODE_FP32
        flags = (_lib.FLAG_SILU if use_silu else 0) | (_lib.FLAG_LISTED_ONLY if listed_only else 0)
        need = self._lib.mbema_branches_attend_workspace_bytes(self.B, self.S, n, H, self.prefix.cap, self.capacity, code)
        cast = E_v.dtype != E_k.dtype or W_pe.dtype != torch.float32
        return q_dt, e_dt, n, H, self.V if V_total is None else V_total, flags, code, need, cast

    def _attend(self, q, E_k, E_v, W_pe, plan):
        q_dt, e_dt, n, H, V_total, flags, code, need, cast = plan
        if cast:
            E_v, W_pe = E_v.to(E_k.dtype), W_pe.float()
        q, E_k, E_v, W = q.contiguous(), E_k.contiguous(), E_v.contiguous(), W_pe.contiguous()
        O = torch.empty_like(q)
        ws = torch.empty(need, dtype=torch.uint8, device=self._device)
        rc = self._lib.mbema_branches_attend(self._ref, q.data_ptr(), q_dt, E_k.data_ptr(), E_v.data_ptr(), e_dt, W.data_ptr(), O.data_ptr(),
                                             n, H, 64, V_total, flags, code, ws.data_ptr(), need, _raw_stream(self._dev))
        if rc:
            _lib.check(rc, "mbema_branches_attend")
        return O

    def adopt(self, branch, t_next):
        """Branch branch[b] (integers [B] on the GPU) of every sequence becomes the state's own: its tokens join the resident
        state and the active list.  Staged tokens are kept unless `keep` has decided on them.  The next step of every sequence
        is t_next afterwards, whatever the branches' lengths (not before the longest one's end).  A branch that does
        not exist or ends behind t_next, in any sequence, leaves the whole state and its step as they were.  Ends these branches
        in either case; what they have to report goes to the state's overflow word."""
        self._alive()
        self._refuse(branch)
        if branch.shape != (self.B,) or branch.dtype not in _INTEGERS:
            raise _lib.MbemaError("adopt: branch %s of %s, expected [%d] integers" % (tuple(branch.shape), branch.dtype, self.B))
        return self._on_device(self._adopt, branch.long().contiguous(), int(t_next))

    def _adopt(self, branch, t_next):
        st = self.prefix
        if self._staged:
            self._keep(torch.full((self.B,), self._staged, dtype=torch.int64, device=branch.device))
        _lib.check(self._lib.mbema_branches_adopt(self._ref, _ptr(branch), t_next, _raw_stream(self._dev)), "mbema_branches_adopt")
        st._epoch += 1
        st.overflow.bitwise_or_(self._hold["overflow"])
        if st.t_dev is not None:
            st.t_dev.copy_(torch.where(self._hold["overflow"] >= 4, st.t_dev, t_next))
        self.prefix = None

    @property
    def lengths(self):
        """Kept tokens of the branches, int32 [B, S] on the GPU."""
        return self._hold["len"]

    def device_status(self):
        """Status word of the tensor-core attends of these branches (synchronises): 0 = ok, else a bounded wait inside a kernel
        gave up and the outputs since then are invalid."""
        return int(self._hold["status"].item()) if self._tensor_cores else 0

    def check_overflow(self):
        """Synchronises; raises if a list overflowed, a token was out of range, or adopt was given a branch or a step that it
        cannot take."""
        raise_reports(self._hold["overflow"], "branches")
