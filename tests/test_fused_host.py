"""What the feed-forward and orthogonalising entry points refuse before they touch a device, and the
Python layer's checks of tensors (meta data only, so CPU tensors do)."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from mlir_roller_b200 import _lib  # noqa: E402
from mlir_roller_b200.ffn import check_matrix  # noqa: E402


def test_ffn_create_refuses_bad_arguments():
    lib, h = _lib.load(), C.c_void_p()
    for args in ((0, 8, 8, 16, 0, 0), (8, 0, 8, 16, 0, 0), (8, 8, -1, 16, 0, 0), ((1 << 20) + 1, 8, 8, 16, 0, 0),
                 (8, 8, 8, _lib.MODE_3XTF32, 0, 0), (8, 8, 8, 16, 3, 0), (8, 8, 8, 16, -1, 0), (8, 8, 8, 16, 0, 2)):
        assert lib.roller_b200_ffn_create(*args, C.byref(h)) == _lib.ERR_INVALID, args
        assert not h
    assert lib.roller_b200_ffn_create(8, 8, 8, 16, 0, 0, None) == _lib.ERR_INVALID


def test_ffn_calls_refuse_null():
    lib, io = _lib.load(), _lib.FfnIo()
    assert lib.roller_b200_ffn_forward(None, C.byref(io), None) == _lib.ERR_INVALID
    assert lib.roller_b200_ffn_backward(None, C.byref(io), None) == _lib.ERR_INVALID
    assert lib.roller_b200_ffn_status(None, None) == _lib.ERR_INVALID
    assert lib.roller_b200_ffn_destroy(None) == _lib.OK


def test_ortho_create_refuses_bad_arguments():
    lib, h = _lib.load(), C.c_void_p()
    muon = (3.4445, -4.7750, 2.0315, 1e-7)
    for args in ((0, 8, 8, 0, 5), (4097, 8, 8, 0, 5), (1, 0, 8, 0, 5), (1, 8, 65537, 0, 5), (1, 8, 8, 3, 5), (1, 8, 8, -1, 5),
                 (1, 8, 8, 0, 0), (1, 8, 8, 0, 33)):
        assert lib.roller_b200_ortho_create(*args, *muon, C.byref(h)) == _lib.ERR_INVALID, args
    inf, nan = float("inf"), float("nan")
    for coef in ((inf, 0, 0, 0), (1, nan, 0, 0), (1, 0, 0, -1), (1, 0, 0, nan), (4.5, 0, 0, 0), (1, 40, -40, 0),
                 (3.9, -4.775, 2.0315, 0)):
        assert lib.roller_b200_ortho_create(1, 8, 8, 0, 8, *coef, C.byref(h)) == _lib.ERR_INVALID, coef
    assert lib.roller_b200_ortho_create(1, 16385, 16385, 0, 5, *muon, C.byref(h)) == _lib.ERR_TOO_LARGE
    assert lib.roller_b200_ortho_run(None, None, 8, 8, None, 8, 8, None) == _lib.ERR_INVALID
    assert lib.roller_b200_ortho_status(None, None) == _lib.ERR_INVALID
    assert lib.roller_b200_ortho_destroy(None) == _lib.OK
    assert not h


def test_packed_operands_match_the_structure():
    from mlir_roller_b200 import ffn
    io = _lib.FfnIo()
    assert ffn._BACKWARD.size == C.sizeof(io)
    ffn._BACKWARD.pack_into(io, 0, 7, *range(100, 124))
    assert io.tokens == 7
    names = [n for n, _ in _lib.FfnIo._fields_[1:]]
    for i, n in enumerate(names):
        assert (getattr(io, n).ptr, getattr(io, n).ld) == (100 + 2 * i, 101 + 2 * i), n
    ffn._FORWARD.pack_into(io, 0, 3, *range(200, 214))
    assert io.tokens == 3 and names[6] == "u" and io.u.ld == 213 and io.dy.ptr == 114


def test_tensor_checks():
    cpu, bf16 = torch.device("cpu"), torch.bfloat16
    t = torch.zeros(6, 10, dtype=bf16)
    assert check_matrix(t, "x", bf16, cpu, 6, 10) == 10
    assert check_matrix(t[:, 2:9], "x", bf16, cpu, 6, 7) == 10
    assert check_matrix(t[::2], "x", bf16, cpu, 3, 10) == 20
    assert check_matrix(t[:1].expand(1, 10), "x", bf16, cpu, 1, 10) == 16
    assert check_matrix(t[:0], "x", bf16, cpu, 0, 10) == 16
    assert check_matrix(t[:, :1], "x", bf16, cpu, 6, 1) == 10
    with pytest.raises(TypeError):
        check_matrix(t.half(), "x", bf16, cpu, 6, 10)
    with pytest.raises(ValueError, match="bound to"):
        check_matrix(t, "x", bf16, torch.device("cuda", 0), 6, 10)
    with pytest.raises(ValueError, match="shape"):
        check_matrix(t, "x", bf16, cpu, 10, 6)
    with pytest.raises(ValueError, match="shape"):
        check_matrix(t[0], "x", bf16, cpu, 1, 10)
    with pytest.raises(ValueError, match="contiguous rows"):
        check_matrix(t.T, "x", bf16, cpu, 10, 6)
    with pytest.raises(ValueError, match="overlapping"):
        check_matrix(t[:1].expand(6, 10), "x", bf16, cpu, 6, 10)
    with pytest.raises(ValueError, match="overlapping"):
        check_matrix(torch.zeros(60, dtype=bf16).as_strided((6, 10), (4, 1)), "x", bf16, cpu, 6, 10)


def test_plans_name_what_they_do_not_take():
    from mlir_roller_b200 import GatedFfnPlan, OrthogonalPlan
    with pytest.raises(TypeError):
        GatedFfnPlan(4, 8, 8, dtype=torch.float32)
    with pytest.raises(ValueError):
        GatedFfnPlan(4, 8, 8, activation="relu")
    with pytest.raises(TypeError):
        OrthogonalPlan(4, 4, dtype=torch.float64)
    with pytest.raises(_lib.RollerError) as e:
        OrthogonalPlan(4, 4, steps=0)
    assert e.value.status == _lib.ERR_INVALID


def test_sizes_beyond_a_c_int_are_refused():
    from mlir_roller_b200 import GatedFfnPlan, OrthogonalPlan
    wrap = (1 << 32) + 8          # modulo 2^32 an ordinary size
    for make in (lambda: GatedFfnPlan(wrap, 8, 8), lambda: GatedFfnPlan(8, wrap, 8), lambda: GatedFfnPlan(8, 8, wrap),
                 lambda: OrthogonalPlan(wrap, 8), lambda: OrthogonalPlan(8, wrap), lambda: OrthogonalPlan(8, 8, batch=wrap),
                 lambda: OrthogonalPlan(8, 8, steps=wrap)):
        with pytest.raises(_lib.RollerError) as e:
            make()
        assert e.value.status == _lib.ERR_INVALID


@pytest.mark.parametrize("kind", ["block", "update"])
def test_status_is_read_on_the_plan_s_own_device(monkeypatch, kind):
    """Two devices, in imitation: a plan of the second one, asked while the first one is current."""
    from contextlib import contextmanager

    from mlir_roller_b200 import GatedFfnPlan, OrthogonalPlan
    current = [0]

    @contextmanager
    def device(d):
        before, current[0] = current[0], torch.device(d).index
        yield
        current[0] = before

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    seen = []

    class Library:
        def status(self, handle, word):
            seen.append(current[0])
            word._obj.value = 6
            return _lib.ERR_TIMEOUT

        roller_b200_ffn_status = roller_b200_ortho_status = status

        def destroy(self, handle):
            return _lib.OK

        roller_b200_ffn_destroy = roller_b200_ortho_destroy = destroy

    cls = GatedFfnPlan if kind == "block" else OrthogonalPlan
    plan = cls.__new__(cls)
    plan._lib, plan._h, plan.device = Library(), C.c_void_p(1), torch.device("cuda", 1)
    with pytest.raises(_lib.RollerError, match="= 6") as e:
        plan.check_status()
    assert e.value.status == _lib.ERR_TIMEOUT
    assert seen == [1] and current == [0]
    plan.destroy()
