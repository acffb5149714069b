"""The C++ face of the calls on a 4- or 8-bit cache (no GPU): it compiles, sizes
agree and refusals are std::invalid_argument with the C ABI's messages."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_cpp_face(tmp_path):
    exe = tmp_path / "scored_api_test"
    lib = os.path.join(ROOT, "kvbridge_amd")
    r = subprocess.run(["hipcc", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "include"),
                        os.path.join(ROOT, "tests", "cpp", "scored_api_test.cpp"), "-L", lib, "-lkvbridge_amd",
                        f"-Wl,-rpath,{lib}", "-o", str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "PASS" in r.stdout
