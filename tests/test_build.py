"""The package's Makefile, dry: what is built where torch or Python's headers are missing, and after
another torch has been installed."""
import subprocess

from conftest import PKG_DIR


def _dry(*args):
    run = subprocess.run(["make", "-n", "-C", str(PKG_DIR), *args], capture_output=True, text=True)
    return run.returncode, run.stdout


def _python(tmp_path, text):
    """A PYTHON that answers every question with `text`."""
    fake = tmp_path / "python"
    fake.write_text(f"#!/bin/sh\n{text}\n")
    fake.chmod(0o755)
    return f"PYTHON={fake}"


def test_the_c_library_needs_no_torch(tmp_path):
    rc, out = _dry("-B", _python(tmp_path, "exit 1"))
    assert rc == 0 and "int8_gemm.cu" in out and "-o lib/libgemm_sm100a.so" in out
    assert "torch_host.cpp" not in out and "is not built" in out


def test_another_torch_builds_the_extension_again(tmp_path):
    for answer in ("/a/torch /a/include py3.99-torch9.9", "/a/torch /a/include py3.99-torch9.8"):
        rc, out = _dry(_python(tmp_path, f"echo {answer}"))
        assert rc == 0 and "csrc/torch_host.cpp" in out and "-I/a/torch/include" in out
