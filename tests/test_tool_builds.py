"""CPU: the scripts that build variants of the library take its sources and flags from where build() has them."""
import os
import shutil
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

COMPILER = """#!%s
import os, sys
out = sys.argv[sys.argv.index("-o") + 1]
missing = [a for a in sys.argv[1:] if a.endswith((".o", ".hip")) and a != out and not os.path.exists(a)]
open(out, "w").write("x")
open(%r, "a").write(" ".join(sys.argv[1:]) + "\\n")
sys.exit(bool(missing))
"""


def _tree(tmp_path):
    """A copy of what the scripts read, and a compiler that writes down its arguments."""
    root = tmp_path / "repo"
    for d in ("distgcn_amd/csrc", "include", "tools"):
        shutil.copytree(os.path.join(ROOT, d), root / d, ignore=shutil.ignore_patterns("*.so", "*.o", "runs", "__pycache__"))
    shutil.copy(os.path.join(ROOT, "__graft_entry__.py"), root)
    log, cc = tmp_path / "log", tmp_path / "cc"
    cc.write_text(COMPILER % (sys.executable, str(log)))
    cc.chmod(0o755)

    def run(script, *args):
        log.write_text("")
        subprocess.run(["bash", str(root / "tools" / script)] + list(args), check=True, env={**os.environ, "HIPCC": str(cc)}, cwd=str(tmp_path), timeout=60)
        return [line.split() for line in log.read_text().splitlines()]
    return root, run


def _entry():
    sys.path.insert(0, ROOT)
    import __graft_entry__
    return __graft_entry__


def _names(args, suffix):
    return sorted(os.path.basename(a)[:-len(suffix)] for a in args if a.endswith(suffix))


def test_diag_build_has_every_source_and_flag(tmp_path):
    g = _entry()
    root, run = _tree(tmp_path)
    calls = run("build_diag.sh")
    sources = sorted(s[:-4] for s in g.HIP_SOURCES)
    assert sorted(n for c in calls for n in _names(c, ".hip")) == sources
    for c in calls:
        assert c[:len(g.HIP_FLAGS)] == g.HIP_FLAGS
        assert "-shared" in c or "-DDGCN_DIAG" in c
    assert _names([a for a in calls[-1] if a != "-o"], ".o") == sources and (root / "distgcn_amd" / "libdgcn_diag.so").exists()
    assert len(run("build_diag.sh")) == 1  # nothing changed: the link alone
    entry = root / "__graft_entry__.py"
    entry.write_text(entry.read_text().replace('"-O3"', '"-O2"'))
    os.utime(entry, (2e9, 2e9))  # other flags: every object anew
    calls = run("build_diag.sh")
    assert len(calls) == len(sources) + 1 and all("-O2" in c for c in calls)


def test_placement_sweep_links_every_object(tmp_path):
    g = _entry()
    root, run = _tree(tmp_path)
    obj = root / "build" / "obj"
    obj.mkdir(parents=True)
    for s in g.HIP_SOURCES:
        (obj / (s[:-4] + ".o")).write_text("x")
    compile_, link = run("placement_sweep.sh", "a", "-mllvm -x")
    assert compile_[:len(g.HIP_FLAGS)] == g.HIP_FLAGS and "-mllvm" in compile_ and _names(compile_, ".hip") == ["fused"]
    objs = [a for a in link if a.endswith(".o")]
    assert sorted(os.path.basename(a) for a in objs) == sorted([s[:-4] + ".o" for s in g.HIP_SOURCES if s != "fused.hip"] + ["fused_a.o"])
    assert link[:len(g.HIP_FLAGS)] == g.HIP_FLAGS
