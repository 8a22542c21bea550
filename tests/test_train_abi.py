"""include/rgb200_train.h as C: it compiles, every function it declares is in the library, and its structs have the sizes that the
ctypes mirrors have."""
import ctypes as C
import os
import re
import shutil
import subprocess

import pytest

from bit_reproducible_training_b200 import _lib, repro_optim

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "rgb200_train.h")
needs_lib = pytest.mark.skipif(not os.path.exists(_lib._build.LIB), reason="librgb200.so is not built")
needs_cc = pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler")


def functions():
    with open(HEADER) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    return re.findall(r"^(?:int|size_t) (rgb200_\w+)\(", text, re.M)


@needs_lib
def test_every_declared_function_is_exported():
    names = functions()
    assert len(names) >= 14
    for name in names:
        assert hasattr(_lib.lib(), name), name


@needs_lib
@needs_cc
def test_header_is_c_and_its_structs_match(tmp_path):
    source = tmp_path / "t.c"
    source.write_text("""#include <stdio.h>
#include "rgb200_train.h"
int main(void) {
    printf("%%zu %%zu %%zu %%zu\\n", sizeof(rgb200_epilogue), sizeof(rgb200_block_norm), sizeof(rgb200_adamw_tensor), sizeof(rgb200_adamw_hyper));
    return rgb200_linear_xent_workspace(0, 1, 1, 3, 0) != 0 || rgb200_block_norm_forward(NULL, NULL) != 1;
}
""".replace("%%", "%").replace("\\\\", "\\"))
    exe = str(tmp_path / "t")
    lib = os.path.dirname(_lib._build.LIB)
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-o", exe, str(source), "-L", lib, "-lrgb200", "-Wl,-rpath," + lib], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0
    assert [int(v) for v in out.stdout.split()] == [C.sizeof(_lib.Epilogue), C.sizeof(_lib.BlockNorm), repro_optim._ROW.itemsize, C.sizeof(_lib.AdamwHyper)]


def test_the_build_notices_an_edited_input(tmp_path, monkeypatch):
    """An object older than a header it includes makes the library stale even when the library itself is newer."""
    build = _lib._build
    src = tmp_path / "a.cu"
    (tmp_path / "a.cuh").write_text("")
    src.write_text('#include "a.cuh"\n')
    (tmp_path / "obj").mkdir()
    obj, lib = tmp_path / "obj" / "a.o", tmp_path / "lib.so"
    for f in (obj, lib):
        f.write_text("")
    monkeypatch.setattr(build, "CSRC", str(tmp_path))
    monkeypatch.setattr(build, "OBJ", str(tmp_path / "obj"))
    monkeypatch.setattr(build, "LIB", str(lib))
    monkeypatch.setattr(build, "SOURCES", ["a.cu"])
    for path, when in ((src, 100), (tmp_path / "a.cuh", 100), (obj, 200), (lib, 300)):
        os.utime(path, (when, when))
    assert not build.stale()
    os.utime(tmp_path / "a.cuh", (250, 250))
    assert build.stale()
    os.utime(obj, (260, 260))
    assert not build.stale()
    os.utime(src, (400, 400))
    assert build.stale()
