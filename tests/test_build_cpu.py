"""What `make -C slam_amd/csrc` asks for: the C library needs hipcc alone, the binding of the sequence layers a Python with torch, and both are
built again when what they are built from or for has changed."""
import os
import subprocess
import sys

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "slam_amd", "csrc")


def make(*args):
    r = subprocess.run(["make", "--no-print-directory", "-C", CSRC, *args], capture_output=True, text=True)
    return r.returncode, r.stdout, r.stderr


def test_the_library_needs_no_python():
    rc, out, err = make("-n", "-B", "PYTHON=false")
    assert rc == 0, err
    assert "-o ../_lib/libslamhip.so" in out and "_sequence" not in out


def test_the_binding_says_what_it_needs():
    rc, out, err = make("-n", "binding", "PYTHON=false")
    assert rc != 0 and "torch" in err, (out, err)


def test_with_torch_both_are_built():
    rc, out, err = make("-n", "-B", "PYTHON=" + sys.executable)
    assert rc == 0, err
    assert "-o ../_lib/libslamhip.so" in out and "-o ../_lib/_sequence.so" in out


def test_other_flags_mean_other_objects(tmp_path):
    """The compiler's flags are in the Makefile: when it changes, every object is compiled again."""
    lib = str(tmp_path / "lib")
    compiler = tmp_path / "compiler"
    compiler.write_text("while [ \"$1\" != -o ]; do shift; done; : > \"$2\"\n")
    stub = "HIPCC=sh " + str(compiler)
    rc, out, err = make("OUT=" + lib, stub, "PYTHON=false")
    assert rc == 0, err
    objects = [f for f in os.listdir(lib) if f.endswith(".o")]
    assert len(objects) >= 12
    _, out, _ = make("-n", "OUT=" + lib, stub, "PYTHON=false")
    assert ".o" not in out
    _, out, _ = make("-n", "-W", "Makefile", "OUT=" + lib, stub, "PYTHON=false")
    assert all("-o " + os.path.join(lib, f) in out for f in objects)


def test_another_torch_means_another_binding(tmp_path):
    lib = tmp_path / "lib"
    stub = ["OUT=" + str(lib), "PYTHON=" + sys.executable, "CXX=touch %s; true" % (lib / "_sequence.so"), "binding"]
    assert make(*stub)[0] == 0 and (lib / "_sequence.so").exists()
    assert "true" not in make(*stub)[1]          # nothing has changed
    (lib / "torch.stamp").write_text("/elsewhere 0.0\n")
    rc, out, err = make(*stub)
    assert rc == 0 and "true" in out, (out, err)
