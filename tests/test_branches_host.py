"""What the C entry points of the branches and of the drafts' verification refuse before anything is launched (no GPU needed)."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from mathbrain_b200 import build, _lib
    build.build()
    return _lib.load()


def _branches(**kw):
    from mathbrain_b200 import _lib
    buf = ctypes.create_string_buffer(64)
    addr = (ctypes.addressof(buf) + 15) // 16 * 16
    sizes = dict(B=2, S=3, V=50, N=64, Kcap=40, cap=20, max_new=8)
    sizes.update({k: v for k, v in kw.items() if k in sizes})
    c = _lib.BranchesStruct(**{n: kw.get(n, addr) for n, t in _lib.BranchesStruct._fields_ if t is ctypes.c_void_p}, **sizes)
    return c, buf, addr


BAD = [(dict(S=0), 2), (dict(N=0), 2), (dict(Kcap=0), 2), (dict(cap=0), 2), (dict(max_new=0), 2), (dict(V=0), 2), (dict(N=129), 3),
       (dict(max_new=33), 3), (dict(state=None), 1), (dict(own_state=None), 1), (dict(overflow=None), 1)]


@pytest.mark.parametrize("kw,code", BAD)
def test_branch_calls_refuse(lib, kw, code):
    c, _, addr = _branches(**kw)
    ref = ctypes.byref(c)
    assert lib.mbema_branches_init(ref, 0, None, None) == code
    assert lib.mbema_branches_extend(ref, addr, 1, 0, addr, None) == code
    assert lib.mbema_branches_keep(ref, addr, 1, None) == code
    assert lib.mbema_branches_adopt(ref, addr, 5, None) == code


def test_branch_argument_errors(lib):
    c, _, addr = _branches()
    ref = ctypes.byref(c)
    assert lib.mbema_branches_init(None, 0, None, None) == 1
    for n, pending in ((0, 0), (9, 0), (1, -1), (1, 9)):
        assert lib.mbema_branches_extend(ref, addr, n, pending, addr, None) == 2
    assert lib.mbema_branches_extend(ref, None, 1, 0, addr, None) == 1
    assert lib.mbema_branches_keep(ref, addr, 9, None) == 2
    assert lib.mbema_branches_keep(ref, None, 1, None) == 1
    assert lib.mbema_branches_adopt(ref, None, 5, None) == 1
    assert lib.mbema_branches_adopt(ref, addr, -1, None) == 2
    assert lib.mbema_branches_adopt(ref, addr, 1 << 31, None) == 2

    def attend(br=ref, q=addr, qd=0, ed=0, O=addr, n=1, H=8, hd=64, mode=0, ws=addr, nbytes=1 << 40):
        return lib.mbema_branches_attend(br, q, qd, addr, addr, ed, addr, O, n, H, hd, 50, 1, mode, ws, nbytes, None)

    assert attend(br=None) == 1 and attend(n=0) == 2 and attend(n=9) == 2 and attend(H=0) == 2 and attend(hd=32) == 3
    assert attend(q=None) == 1 and attend(qd=2) == 6 and attend(ed=7) == 6 and attend(q=addr + 4) == 7 and attend(O=addr + 2) == 7
    assert attend(nbytes=64) == 4 and attend(ws=None) == 1
    assert lib.mbema_branches_attend_workspace_bytes(0, 1, 1, 8, 40, 20, 0) > 0
    for bad in ((-1, 1, 1, 8, 40, 20), (1, 0, 1, 8, 40, 20), (1, 1, 33, 8, 40, 20), (1, 1, 1, 0, 40, 20), (1, 1, 1, 8, 0, 20)):
        assert lib.mbema_branches_attend_workspace_bytes(*bad, 0) == 0
    empty, _, _ = _branches(B=0, state=None, overflow=None)
    assert lib.mbema_branches_init(ctypes.byref(empty), 0, None, None) == 0
    assert lib.mbema_branches_extend(ctypes.byref(empty), None, 1, 0, None, None) == 0
    assert attend(br=ctypes.byref(empty), q=None) == 0


def test_verify_argument_errors(lib):
    buf = ctypes.create_string_buffer(64)
    a = ctypes.addressof(buf)

    def verify(p=a, q=a, dt=0, x=a, u=a, n=a, t=a, R=1, G=1, V=5):
        return lib.mbema_verify_drafts(p, V, V, q, V, V, dt, x, u, n, t, R, G, V, None)

    assert verify(R=-1) == 2 and verify(G=-1) == 2 and verify(V=0) == 2 and verify(dt=3) == 6
    assert verify(V=1 << 30) == 3 and verify(G=4097) == 3 and verify(R=1 << 30) == 3
    for name in "pxunt":
        assert verify(**{name: None}) == 1
    assert verify(p=None, R=0) == 0


def test_operands_on_the_cpu_are_refused():
    import torch
    import mathbrain_b200 as mb
    from mathbrain_b200.verify import verify_drafts
    with pytest.raises(mb._lib.MbemaError):
        verify_drafts(torch.zeros(1, 2, 5), torch.zeros(1, 1, dtype=torch.long), torch.zeros(1, 2))
