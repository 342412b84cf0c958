"""The build recipe with stand-ins for the compilers: what it needs, and what is
left when a part of it fails."""

import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parents[1]
LIBRARY = "libfds_b200.so"

# "compiles" by writing its sources' names to the output, and reports what the register check reads
NVCC = """#!/bin/sh
out=; srcs=
while [ $# -gt 0 ]; do
  case "$1" in -o) out="$2"; shift;; *.cu) srcs="$srcs $1";; *.o) srcs="$srcs $(cat "$1")";; esac
  shift
done
echo "$srcs" > "$out"
for k in "attn_fwd_kernel 168" "window_tile_kernel 128"; do
  set -- $k
  echo "ptxas info    : Compiling entry function '$1' for 'sm_100a'"
  echo "ptxas info    : Used $2 registers"
done
"""
FAILS = "#!/bin/sh\necho 'no such compiler' >&2\nexit 1\n"
WORKS = '#!/bin/sh\nwhile [ "$1" != -o ]; do shift; done\necho extension > "$2"\n'


@pytest.fixture
def tree(tmp_path):
    """A copy of what the recipe reads, without built files; bin/ first on the PATH."""
    pkg = tmp_path / "fastdialoguesidon_b200"
    shutil.copytree(REPO / "fastdialoguesidon_b200" / "csrc", pkg / "csrc")
    shutil.copy(REPO / "fastdialoguesidon_b200" / "build.py", pkg / "build.py")
    shutil.copytree(REPO / "include", tmp_path / "include")
    (tmp_path / "bin").mkdir()
    _tool(tmp_path, "nvcc", NVCC)
    _tool(tmp_path, "g++", WORKS)
    return tmp_path


def _tool(tree, name, text):
    path = tree / "bin" / name
    path.write_text(text)
    path.chmod(0o755)


def _start(tree, code="", args=()):
    """The recipe as a script, after `code`."""
    text = f"import sys, runpy; sys.argv[1:] = {list(args)!r}\n{code}\nrunpy.run_path('fastdialoguesidon_b200/build.py', run_name='__main__')"
    env = dict(os.environ, PATH=f"{tree / 'bin'}:{os.environ['PATH']}")
    return subprocess.Popen([sys.executable, "-c", text], cwd=tree, env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)


def _run(tree, code="", args=()):
    p = _start(tree, code, args)
    out = p.communicate(timeout=120)[0]
    return p.returncode, out


def _built(tree):
    return sorted(p.name for p in (tree / "fastdialoguesidon_b200" / "_lib").iterdir() if not p.name.endswith(".lock"))


def test_both_are_built(tree):
    rc, out = _run(tree)
    assert rc == 0, out
    assert LIBRARY in _built(tree) and len([n for n in _built(tree) if n.startswith("_fds_torch")]) == 1
    text = (tree / "fastdialoguesidon_b200" / "_lib" / LIBRARY).read_text()
    for src in ("fds_capi.cu", "fds_rope_static.cu", "fds_int8.cu", "fds_norm.cu", "fds_window.cu"):
        assert src in text


def test_the_library_needs_no_torch(tree):
    rc, out = _run(tree, "sys.modules['torch'] = None")
    assert rc == 0, out
    assert _built(tree) == [LIBRARY]


def test_the_library_stays_when_the_extension_fails(tree):
    _tool(tree, "g++", FAILS)
    rc, out = _run(tree)
    assert rc != 0 and "g++ failed" in out and "no such compiler" in out, out
    assert LIBRARY in _built(tree)


def test_an_extension_of_another_torch_is_not_taken(tree):
    """The extension is built again for the torch (or Python) that is there, whatever the files' times."""
    assert _run(tree)[0] == 0
    before = _built(tree)
    rc, out = _run(tree, "import torch; torch.__version__ = '99.1'")
    assert rc == 0, out
    new = set(_built(tree)) - set(before)
    assert len(new) == 1 and "99.1" in new.pop()
    rc, out = _run(tree, "sys.implementation.cache_tag = 'cpython-399'")
    assert rc == 0 and any("cpython-399" in n for n in _built(tree)), out


def test_processes_that_build_at_once(tree):
    """Four, on a fresh tree, each step of which takes a while: one builds, every one
    succeeds, and nothing but the results is left."""
    _tool(tree, "nvcc", NVCC.replace("out=; srcs=", "out=; srcs=; echo call >> calls; sleep 0.2"))
    procs = [_start(tree, "sys.modules['torch'] = None") for _ in range(4)]
    outs = [(p.communicate(timeout=120)[0], p.returncode) for p in procs]
    assert all(rc == 0 for _, rc in outs), outs
    assert _built(tree) == [LIBRARY]
    assert len((tree / "calls").read_text().split()) == 6  # five sources and a link
    procs = [_start(tree, "sys.modules['torch'] = None", ["--force"]) for _ in range(3)]
    outs = [(p.communicate(timeout=120)[0], p.returncode) for p in procs]
    assert all(rc == 0 for _, rc in outs), outs
    text = (tree / "fastdialoguesidon_b200" / "_lib" / LIBRARY).read_text()
    assert _built(tree) == [LIBRARY] and text.count(".cu") == 5


def test_nothing_is_replaced_by_a_library_with_other_registers(tree):
    _tool(tree, "nvcc", NVCC.replace("window_tile_kernel 128", "window_tile_kernel 126"))
    rc, out = _run(tree)
    assert rc != 0 and "126 registers" in out, out
    assert LIBRARY not in _built(tree)


def test_a_library_of_another_abi_is_refused(tmp_path, monkeypatch):
    """By its version, although it lacks entry points of this one."""
    from fastdialoguesidon_b200 import _native as N

    src = tmp_path / "old.c"
    src.write_text("int fds_abi_version(void) { return 4; }\nint fds_linear_fwd(void *a, void *s) { return 0; }\n")
    lib = tmp_path / "libold.so"
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(lib), str(src)], check=True)
    monkeypatch.setattr(N, "_lib", None)
    monkeypatch.setattr(N._build, "LIB_PATH", lib)
    with pytest.raises(RuntimeError, match="ABI version 4"):
        N.load()
