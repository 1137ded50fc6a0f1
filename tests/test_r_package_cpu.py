"""The R package's build, without R: what `configure` compiles links completely, with the flags of the library's own build.  The compiler it
calls is a stand-in that hands out the objects which the library was linked from."""
import os
import re
import shutil
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "chatterbox_amd", "csrc")


def makefile_flags():
    text = open(os.path.join(CSRC, "Makefile")).read()
    flags = re.search(r"^CXXFLAGS := (.*)$", text, re.M).group(1).replace("$(ARCH)", "gfx950").split()
    return [f for f in flags if not f.startswith(("-I", "-W"))]


def test_what_configure_compiles_links(tmp_path):
    objects = re.search(r"^OBJS := (.*)$", open(os.path.join(CSRC, "Makefile")).read(), re.M).group(1).split()
    if not all(os.path.exists(os.path.join(CSRC, o)) for o in objects):
        subprocess.check_call(["make", "-C", CSRC, "-j8"] + objects)
    pkg = tmp_path / "pkg"
    shutil.copytree(os.path.join(ROOT, "r-package"), pkg)
    shutil.copytree(CSRC, pkg / "src" / "t3mi", ignore=shutil.ignore_patterns("*.o"))
    (pkg / "inst" / "include").mkdir(parents=True)
    shutil.copy(os.path.join(ROOT, "include", "t3mi.h"), pkg / "inst" / "include")
    log, hipcc = tmp_path / "log", tmp_path / "hipcc"
    hipcc.write_text(f"""#!/bin/sh
echo "$@" >> {log}
while [ $# -gt 0 ]; do
  case "$1" in -c) in="$2" ;; -o) out="$2" ;; esac
  shift
done
name=$(basename "$in")
cp {CSRC}/"${{name%.*}}".o "$out"
""")
    hipcc.chmod(0o755)
    subprocess.check_call(["sh", "configure"], cwd=pkg, env={**os.environ, "HIPCC": str(hipcc)})
    for line in log.read_text().splitlines():
        used = line.split()
        for f in makefile_flags():
            assert f in used, (f, line)
    makevars = (pkg / "src" / "Makevars").read_text()
    cpp, libs = (re.search(rf"^{n} = ?(.*)$", makevars, re.M).group(1).split() for n in ("PKG_CPPFLAGS", "PKG_LIBS"))
    mock = os.path.join(ROOT, "tests", "r_mock")
    glue = ["r_glue.c", "r_glue_s3gen.c", os.path.join(mock, "r_mock.c")]
    subprocess.check_call(["gcc", "-O1", "-fPIC", "-shared", "-Wl,--no-undefined", "-Wno-cast-function-type", *cpp, f"-I{mock}/include", *glue, *libs, "-o", "chatterbox.so"],
                          cwd=pkg / "src")
    names = subprocess.run(["nm", "-D", "--defined-only", "chatterbox.so"], cwd=pkg / "src", check=True, capture_output=True, text=True).stdout
    assert "t3mi_paged_attention" in names and "t3mi_hift_inference" in names


def test_the_library_builds_without_python_headers():
    """A C or R user needs no Python.h: the library is made, the Python side left out and named."""
    plan = lambda *a: subprocess.run(["make", "-n", "-B", "-C", CSRC, *a], check=True, capture_output=True, text=True).stdout  # noqa: E731
    assert "py_ops.c" in plan()
    out = plan("PYINC=/nonexistent")
    assert "py_ops.c" not in out and "-o ../libt3mi.so" in out and "no Python.h" in out
