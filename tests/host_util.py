"""Programs of the library's host code on tests/shims/fake_cuda.h: failures of CUDA's calls without a GPU."""
import os
import subprocess

from densecore_b200 import build as B

TESTS = os.path.dirname(os.path.abspath(__file__))


def program(tmp_path, parts, text):
    """Compiles `text` (a main() behind fake_cuda.h) and the library's sources `parts`, links them without CUDA's runtime; the executable's path."""
    src = tmp_path / "p.cpp"
    src.write_text('#include "fake_cuda.h"\n' + text)
    common = ["-std=c++17", "-I", os.path.join(B.ROOT, "include"), "-I", B.CSRC]
    jobs = [(tmp_path / f"{n}.o", [B.nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-Xcicc", "-O0", "-Xptxas", "-O0", "--expt-relaxed-constexpr", *common, "-c",
                                   os.path.join(B.CSRC, f"{n}.cu")]) for n in parts]
    jobs.append((tmp_path / "p.o", [B.nvcc(), "-Xcompiler", "-Wall", *common, "-I", os.path.join(TESTS, "shims"), "-c", str(src)]))
    running = [subprocess.Popen([*cmd, "-o", str(obj)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True) for obj, cmd in jobs]
    for r in running:
        out, _ = r.communicate()
        assert r.returncode == 0, out
    exe = str(tmp_path / "p")
    subprocess.check_call(["g++", *(str(obj) for obj, _ in jobs), "-o", exe])
    return exe


def run(exe, *args):
    return subprocess.run([exe, *map(str, args)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=60)
