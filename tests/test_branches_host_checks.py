"""What the C entry points of the branches refuse before anything is launched, pointer by pointer (no GPU needed)."""
import ctypes

import pytest

from test_branches_host import BAD, _branches, lib  # noqa: F401  (a fixture)

POINTERS = ("rhos state last_t active n_active pos t0 len own_n own_new own_slot own_t own_state touched st_tok st_own st_pos st_same "
            "st_new st_state pre_op own_op work status overflow").split()


def _attend(lib, c, addr, n=1, H=8, mode=0, dt=0, nbytes=1 << 40):
    return lib.mbema_branches_attend(ctypes.byref(c), addr, dt, addr, addr, dt, addr, addr, n, H, 64, 50, 1, mode, addr, nbytes, None)


@pytest.mark.parametrize("kw,code", BAD)
def test_attend_refuses_what_the_other_calls_refuse(lib, kw, code):
    c, _, addr = _branches(**kw)
    assert _attend(lib, c, addr) == code


@pytest.mark.parametrize("name", POINTERS)
@pytest.mark.parametrize("mode,dt", [(0, 0), (1, 1)])
def test_attend_refuses_a_missing_buffer(lib, name, mode, dt):
    c, _, addr = _branches(**{name: None})
    assert _attend(lib, c, addr, mode=mode, dt=dt) == 1


@pytest.mark.parametrize("name", ["state", "own_state", "pre_op", "own_op", "work"])
def test_buffers_of_the_tensor_cores_are_aligned(lib, name):
    c, _, addr = _branches()
    setattr(c, name, addr + 4)
    assert _attend(lib, c, addr, mode=1, dt=1) == 7
    assert lib.mbema_branches_extend(ctypes.byref(c), addr, 1, 0, addr, None) == 7


@pytest.mark.parametrize("t_now", [-1, 1 << 31, 1 << 32])
def test_a_step_outside_its_type_is_refused(lib, t_now):
    c, _, addr = _branches()
    assert lib.mbema_branches_init(ctypes.byref(c), t_now, None, None) == 2


@pytest.mark.parametrize("H", [65536, (1 << 32) + 8])
@pytest.mark.parametrize("S,mode,dt", [(3, 0, 0), (3, 1, 1), (1, 1, 1)])
def test_more_heads_than_a_grid_holds_are_refused(lib, H, S, mode, dt):
    c, _, addr = _branches(S=S)
    assert _attend(lib, c, addr, H=H, mode=mode, dt=dt, nbytes=1 << 62) == 3
