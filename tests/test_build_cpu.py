"""What build() makes where torch or its compiler is missing: the library, which programs without torch use through its C ABI.
The compilers are stand-ins that write the file they are asked for; build.py is loaded by its path, as a program without torch runs it."""
import pathlib
import subprocess
import sys

ROOT = pathlib.Path(__file__).resolve().parent.parent
STAND_IN = '''#!/bin/sh
while [ $# -gt 0 ]; do [ "$1" = -o ] && { echo made > "$2"; exit 0; }; shift; done
exit 1
'''
BUILD = '''
import importlib.util, pathlib, sys
if {torch} is None:
    sys.modules["torch"] = None
spec = importlib.util.spec_from_file_location("build_by_path", {path!r})
b = importlib.util.module_from_spec(spec)
spec.loader.exec_module(b)
b.LIB_DIR = pathlib.Path({lib!r})
b.LIB_PATH, b.BINDING_PATH = b.LIB_DIR / "libngpt_fp8.so", b.LIB_DIR / "_ngpt_torch.so"
{more}
print("built", b.build().name)
'''


def run(tmp_path, torch, more=""):
    hipcc = tmp_path / "hipcc"
    hipcc.write_text(STAND_IN)
    hipcc.chmod(0o755)
    lib = tmp_path / "lib"
    code = BUILD.format(torch=torch, path=str(ROOT / "modded-nanogpt_amd" / "build.py"), lib=str(lib), more=more)
    p = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=tmp_path,
                       env={"PATH": "/usr/bin:/bin", "HIPCC": str(hipcc), "HOME": str(tmp_path)})
    return p, sorted(f.name for f in lib.iterdir())


def test_the_library_is_built_without_torch(tmp_path):
    p, files = run(tmp_path, "None")
    assert p.returncode == 0 and "built libngpt_fp8.so" in p.stdout and "no torch" in p.stdout, p.stderr
    assert files == ["libngpt_fp8.so"]


def test_the_library_is_in_place_when_its_binding_fails(tmp_path):
    p, files = run(tmp_path, "1", 'b._binding_commands = lambda obj, lib_dir: (["false"], [])')
    assert p.returncode != 0 and "false failed" in p.stderr
    assert files == ["libngpt_fp8.so"]


def test_the_binding_is_made_beside_the_library(tmp_path):
    p, files = run(tmp_path, "1", 'b._binding_commands = lambda obj, lib_dir: (["touch", obj], ["touch", str(b.BINDING_PATH) + ".tmp"])')
    assert p.returncode == 0, p.stderr
    assert files == ["_ngpt_torch.so", "libngpt_fp8.so"]
