"""Verification of drafted tokens: which of them stand, and the token behind them.

The reference has no decode loop.  For rows that were drafted by a cheaper model, by another branch or by looking the text up,
`verify_drafts` decides from given uniform numbers so that the tokens which come out have the target's distribution:
draft j, drawn from q_j, stands with probability min(1, p_j / q_j); the first that does not is replaced by a draw from
max(p_j - q_j, 0), and behind drafts that all stand one more token is drawn from the target.
"""
import torch

from . import _lib
from .ops import _dt, _on_tensor_device, _ptr, _require_cuda, _stream


@_on_tensor_device
def verify_drafts(p_target, drafted, uniforms, p_draft=None):
    """(n_accepted int64 [R], tokens int64 [R, G + 1]): the drafts that stand, the next token, then -1.

    p_target [R, G + 1, V] probabilities of the target at every draft and behind the last, float32 or bfloat16 (rows need not
        be contiguous, the vocabulary axis must be); drafted [R, G] int64 (a value outside [0, V), -1 say, ends the drafts of its
        row: the next token is drawn from the target there); uniforms [R, G + 1] float32 in [0, 1): one for each draft, the last
        for the draw;
    p_draft [R, G, V] probabilities the drafts were drawn from (p_target's dtype), or None for drafts that were not drawn: draft
        j then stands with probability p_j and its token is left out of the draw otherwise.

    A draw takes the smallest i whose running sum of weights passes uniform * their total; probabilities that are negative or
    not finite count as 0 there.  G = 0 draws from p_target alone."""
    _require_cuda(p_target, drafted, uniforms, p_draft)
    if p_target.dim() != 3 or p_target.shape[1] < 1 or p_target.shape[2] < 1:
        raise _lib.MbemaError("verify_drafts: p_target %s, expected [R, G + 1, V]" % (tuple(p_target.shape),))
    R, G, V = p_target.shape[0], p_target.shape[1] - 1, p_target.shape[2]
    if drafted.shape != (R, G) or drafted.dtype != torch.int64:
        raise _lib.MbemaError("verify_drafts: drafted %s of %s, expected [%d, %d] int64" % (tuple(drafted.shape), drafted.dtype, R, G))
    if uniforms.shape != (R, G + 1) or uniforms.dtype != torch.float32:
        raise _lib.MbemaError("verify_drafts: uniforms %s of %s, expected [%d, %d] float32"
                              % (tuple(uniforms.shape), uniforms.dtype, R, G + 1))
    if p_draft is not None and (p_draft.shape != (R, G, V) or p_draft.dtype != p_target.dtype):
        raise _lib.MbemaError("verify_drafts: p_draft %s of %s, expected [%d, %d, %d] %s"
                              % (tuple(p_draft.shape), p_draft.dtype, R, G, V, p_target.dtype))
    dt = _dt(p_target)
    if V > 1 and p_target.stride(2) != 1:
        p_target = p_target.contiguous()
    if p_draft is not None and V > 1 and p_draft.stride(2) != 1:
        p_draft = p_draft.contiguous()
    drafted, uniforms = drafted.contiguous(), uniforms.contiguous()
    n_accepted = torch.empty(R, dtype=torch.int64, device=p_target.device)
    tokens = torch.empty(R, G + 1, dtype=torch.int64, device=p_target.device)
    q_row, q_pos = (p_draft.stride(0), p_draft.stride(1)) if p_draft is not None else (0, 0)
    rc = _lib.load().mbema_verify_drafts(_ptr(p_target), p_target.stride(0), p_target.stride(1), _ptr(p_draft), q_row, q_pos, dt,
                                         _ptr(drafted), _ptr(uniforms), _ptr(n_accepted), _ptr(tokens), R, G, V, _stream())
    _lib.check(rc, "mbema_verify_drafts")
    return n_accepted, tokens
