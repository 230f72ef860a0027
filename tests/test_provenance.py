"""A deployment's source digest covers the files that its own library is compiled from, no others."""
import os
import shutil
import subprocess

import pytest

from custom_ops_amd import FAOps, ServeOps, build


@pytest.mark.parametrize("src", [build.SRC, build.SERVE_SRC])
def test_sources_are_the_compilers(src):
    """The compiler's own list of what it reads, as far as it is this package's."""
    res = subprocess.run([build.hipcc(), "--offload-arch=gfx950", "-std=c++17", "--cuda-host-only", f"-I{build.INCLUDE}", "-M", src],
                         capture_output=True, text=True, check=True)
    root = os.path.dirname(build.PKG_DIR)
    used = {os.path.realpath(w) for w in res.stdout.partition(":")[2].replace("\\\n", " ").split()}
    mine = {p for p in used if p.startswith(os.path.realpath(root) + os.sep)}
    assert {os.path.realpath(p) for p in build.sources_of(src)} == mine


def test_a_header_counts_for_its_own_library(tmp_path, monkeypatch):
    """Of a copy of the sources: one of the serving operators' headers, then a shared one."""
    pkg = tmp_path / "pkg"
    shutil.copytree(os.path.dirname(build.SRC), pkg / "csrc")
    shutil.copytree(build.INCLUDE, tmp_path / "include")
    monkeypatch.setattr(build, "INCLUDE", str(tmp_path / "include"))
    monkeypatch.setattr(build, "SRC", str(pkg / "csrc" / os.path.basename(build.SRC)))
    monkeypatch.setattr(build, "SERVE_SRC", str(pkg / "csrc" / os.path.basename(build.SERVE_SRC)))

    def digests():
        return [g()._provenance(["gfx950"], [])["sources_sha256"] for g in (FAOps, ServeOps)]

    fa, serve = digests()
    for name in ("packed_fwd.h", "serve_sched.h"):
        with open(pkg / "csrc" / name, "a") as f:
            f.write("// changed\n")
        now = digests()
        assert now[0] == fa and now[1] != serve
        serve = now[1]
    with open(tmp_path / "include" / "mi355_fa.h", "a") as f:
        f.write("/* changed */\n")
    now = digests()
    assert now[0] != fa and now[1] == serve
    with open(pkg / "csrc" / "gfx950.h", "a") as f:
        f.write("// changed\n")
    assert digests()[0] != now[0] and digests()[1] != now[1]
