"""Run as a process of its own by tests/test_muon.py: md2_broadcast_state with a stand-in for RCCL (tests/native/fake_rccl.cpp), without torch, whose own librccl would be found first.
Prints one line per case: name, status, broadcasts, reductions, this rank's answer, the handle's Muon state count, the error."""
import ctypes as C
import importlib.util
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
fake = C.CDLL(os.path.join(ROOT, "tests", "native", "libfake_rccl.so"), mode=C.RTLD_GLOBAL)      # (before the library: its hipMalloc is found first, and "librccl.so.1" is this one)
spec = importlib.util.spec_from_file_location("md2lib", os.path.join(ROOT, "monodepth2.jl_amd", "_lib.py")); m = importlib.util.module_from_spec(spec); spec.loader.exec_module(m)
L = m.lib()
assert "torch" not in sys.modules

cfg = m.Md2Config(1, 1, 64, 96, 0, 0, 0.1, 100.0, 1e-3, 1e-4, 18, 0, 2, (C.c_int32 * 2)(1, 3), (C.c_int32 * 5)(2, 3, 4, 5), (C.c_double * 5)())
D, I, S = C.c_double, C.c_int, C.c_size_t


def case(name, has_muon, root_has, others_can, fail_above):
    h = C.c_void_p(); assert L.md2_create(C.byref(cfg), C.byref(h)) == 0, L.md2_last_error(None)
    n = L.md2_params_count(h)
    if has_muon:
        assert L.md2_muon_state_set(h, (C.c_float * n)(), n) == 0, L.md2_last_error(h)
    assert L.md2_comm_init(h, 0, 2, (C.c_char * 128)()) == 0, L.md2_last_error(h)
    D.in_dll(fake, "fake_root_has_muon").value = root_has; D.in_dll(fake, "fake_others_can").value = others_can; I.in_dll(fake, "fake_fail_above").value = fail_above
    for k in ("fake_broadcasts", "fake_reduces"):
        I.in_dll(fake, k).value = 0
    D.in_dll(fake, "fake_mine").value = -1
    r = L.md2_broadcast_state(h, 1)
    I.in_dll(fake, "fake_fail_above").value = 0
    print(name, r, I.in_dll(fake, "fake_broadcasts").value, I.in_dll(fake, "fake_reduces").value, D.in_dll(fake, "fake_mine").value, int(L.md2_muon_state_count(h) == n), repr(L.md2_last_error(h).decode()), flush=True)
    assert L.md2_comm_destroy(h) == 0 and L.md2_destroy(h) == 0


case("nobody", 0, 0.0, 1.0, 0)
case("dropped", 1, 0.0, 1.0, 0)
case("given", 0, 1.0, 1.0, 0)
case("kept", 1, 1.0, 1.0, 0)
case("other_cannot", 0, 1.0, 0.0, 0)
case("other_cannot_kept", 1, 1.0, 0.0, 0)
case("cannot", 0, 1.0, 1.0, 4096)
