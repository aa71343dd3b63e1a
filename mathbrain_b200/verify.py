"""Verification of drafted tokens: which of them stand, and the token behind them.

The reference has no decode loop.  For rows that were drafted by a cheaper model, by another branch or by looking the text up,
`verify_drafts` decides from given uniform numbers so that the tokens which come out have the target's distribution:
draft j, drawn from q_j, stands with probability min(1, p_j / q_j); the first that does not is replaced by a draw from
max(p_j - q_j, 0), and behind drafts that all stand one more token is drawn from the target.
"""
import torch

from . import _lib
from .ops import _current_device, _dt, _raw_stream, _require_cuda


def verify_drafts(p_target, drafted, uniforms, p_draft=None):
    """(n_accepted int64 [R], tokens int64 [R, G + 1]): the drafts that stand, the next token, then -1.

    p_target [R, G + 1, V] probabilities of the target at every draft and behind the last, float32 or bfloat16 (rows need not
        be contiguous, the vocabulary axis must be); drafted [R, G] int64 (a value outside [0, V), -1 say, ends the drafts of its
        row: the next token is drawn from the target there); uniforms [R, G + 1] float32 in [0, 1): one for each draft, the last
        for the draw;
    p_draft [R, G, V] probabilities the drafts were drawn from (p_target's dtype), or None for drafts that were not drawn: draft
        j then stands with probability p_j and its token is left out of the draw otherwise.

    A draw takes the smallest i whose running sum of weights (p, or p - q where a draft was rejected) passes uniform * their total;
    weights that are negative, not finite or beyond fp32 count as 0.  G = 0 draws from p_target alone."""
    dev = p_target.get_device()
    if dev < 0 or drafted.get_device() != dev or uniforms.get_device() != dev or (p_draft is not None and p_draft.get_device() != dev):
        _require_cuda(p_target, drafted, uniforms, p_draft)
        raise _lib.MbemaError("verify_drafts: operands live on different devices")
    shape, dtype = p_target.shape, p_target.dtype
    if len(shape) != 3 or shape[1] < 1 or shape[2] < 1:
        raise _lib.MbemaError("verify_drafts: p_target %s, expected [R, G + 1, V]" % (tuple(shape),))
    R, places, V = shape
    G = places - 1
    if drafted.shape != (R, G) or drafted.dtype != torch.int64:
        raise _lib.MbemaError("verify_drafts: drafted %s of %s, expected [%d, %d] int64" % (tuple(drafted.shape), drafted.dtype, R, G))
    if uniforms.shape != (R, places) or uniforms.dtype != torch.float32:
        raise _lib.MbemaError("verify_drafts: uniforms %s of %s, expected [%d, %d] float32"
                              % (tuple(uniforms.shape), uniforms.dtype, R, places))
    if p_draft is not None and (p_draft.shape != (R, G, V) or p_draft.dtype != dtype):
        raise _lib.MbemaError("verify_drafts: p_draft %s of %s, expected [%d, %d, %d] %s"
                              % (tuple(p_draft.shape), p_draft.dtype, R, G, V, dtype))
    dt = _dt(p_target)
    if dev != _current_device():
        with torch.cuda.device(dev):
            return _verify(p_target, drafted, uniforms, p_draft, dt, dev, R, G, V)
    return _verify(p_target, drafted, uniforms, p_draft, dt, dev, R, G, V)


def _verify(p, drafted, uniforms, q, dt, dev, R, G, V):
    p_row, p_pos, one = p.stride()
    if one != 1 and V > 1:
        p = p.contiguous()
        p_row, p_pos, _ = p.stride()
    q_ptr, q_row, q_pos = None, 0, 0
    if q is not None:
        q_row, q_pos, one = q.stride()
        if one != 1 and V > 1:
            q = q.contiguous()
            q_row, q_pos, _ = q.stride()
        q_ptr = q.data_ptr()
    drafted, uniforms = drafted.contiguous(), uniforms.contiguous()
    n_accepted = torch.empty(R, dtype=torch.int64, device=p.device)
    tokens = torch.empty((R, G + 1), dtype=torch.int64, device=p.device)
    rc = _lib.load().mbema_verify_drafts(p.data_ptr(), p_row, p_pos, q_ptr, q_row, q_pos, dt, drafted.data_ptr(), uniforms.data_ptr(),
                                         n_accepted.data_ptr(), tokens.data_ptr(), R, G, V, _raw_stream(dev))
    if rc:
        _lib.check(rc, "mbema_verify_drafts")
    return n_accepted, tokens
