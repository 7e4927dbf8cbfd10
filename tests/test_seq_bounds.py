"""CPU: sizes and pointers that the sequence operators refuse because a kernel could not take them."""
from test_seq_checks import INVALID, P, UNSUPPORTED, append, attend, call, desc, load


def test_more_columns_than_the_kernels_count():
    """Kernels step past the last column in 32 bits."""
    for cols in ((1 << 30) + 1, (1 << 31) - 1):
        assert call("vdt_quantize_rows", P, 0, 1, cols, cols, P, cols, P, None) == UNSUPPORTED
        assert call("vdt_int8_matmul", P, 32, P, P, 32, P, None, 3, cols, 20, 2, P, cols, None) == UNSUPPORTED
        assert call("vdt_int8_linear", P, 1, 20, P, 32, P, None, 3, cols, 20, 1, P, cols, P, 1 << 20, None) == UNSUPPORTED


def test_scales_and_lengths_off_their_alignment():
    """A kernel's 32-bit load from such an address would fault."""
    def matmul(a_scale=P, w_scale=P, bias=P):
        return call("vdt_int8_matmul", P, 32, a_scale, P, 32, w_scale, bias, 3, 5, 20, 2, P, 5, None)

    def linear(w_scale=P, bias=P):
        return call("vdt_int8_linear", P, 1, 20, P, 32, w_scale, bias, 3, 5, 20, 1, P, 5, P, 1 << 20, None)

    for off in (1, 2, 3):
        for over in (dict(a_scale=P + off), dict(w_scale=P + off), dict(bias=P + off)):
            assert matmul(**over) == INVALID, over
            if "a_scale" not in over:
                assert linear(**over) == INVALID, over
        for go in (append, load, attend):
            for over in (dict(k_scale=P + off), dict(v_scale=P + off)):
                assert go(desc(**over)) == INVALID, over
            for over in (dict(table=P + off), dict(held=P + off), dict(starts=P + off)):
                assert go(desc(), **over) == INVALID, over


def test_the_module_has_no_standard_library_of_its_own():
    """A second libstdc++ in the process: its streams ended it when they met the first one's locales."""
    import os
    from conftest import ROOT
    with open(os.path.join(ROOT, "vd-ttfs_b200", "vdttfs", "_seq.so"), "rb") as f:
        built = f.read()
    assert b"libstdc++.so.6\0" in built and b"_ZNSt6locale5facet" not in built


def test_the_library_is_built_without_torch():
    """The default target is a C integrator's: nvcc alone.  The module for torch tensors has a target of its own."""
    import os
    import subprocess
    from conftest import ROOT

    def steps(*target):
        return subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "vd-ttfs_b200"), "PYTHON=no-such-python", *target], check=True,
                              capture_output=True, text=True).stdout

    assert "libvdttfs.so" in steps() and "seq_torch" not in steps() and "no-such-python" not in steps()
    assert "seq_torch" in steps("seq") and "libvdttfs.so" in steps("seq")
