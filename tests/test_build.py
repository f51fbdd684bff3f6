"""What the build makes, from what, and in which order (no compiler runs here)."""
import os
import subprocess
import sys

import pytest

from pybgmm_amd import _build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def made(monkeypatch, fails=None):
    """Records what a build makes; `fails`: a target whose compiler fails."""
    log = []

    def one(lib, *args):
        log.append(lib)
        return lib

    def run(cmd, verbose):
        log.append(cmd[cmd.index("-o") + 1])
        if log[-1] == fails:
            raise RuntimeError("no compiler")
    monkeypatch.setattr(_build, "_build_one", one)
    monkeypatch.setattr(_build, "_run", run)
    return log


def test_a_binding_that_cannot_be_built_leaves_the_samplers_library(monkeypatch):
    log = made(monkeypatch, fails=_build.OPS_BINDING)
    monkeypatch.setattr(_build, "_stale", lambda target, deps: True)
    with pytest.raises(RuntimeError):
        _build.build()
    assert log[0] == _build.LIB


def test_a_missing_library_is_built_by_itself(monkeypatch, tmp_path):
    from pybgmm_amd import _lib
    log = made(monkeypatch)
    monkeypatch.setattr(_lib, "_lib", None)
    missing = str(tmp_path / "libbgmm_hip.so")
    monkeypatch.setattr(_build, "LIB", missing)
    with pytest.raises(OSError):                # (nothing was really built)
        _lib.load()
    assert log == [missing]


@pytest.mark.parametrize("without", ["torch", "hip"])
def test_the_entry_point_builds_without_a_torch_that_has_hip(without, tmp_path):
    """In a process of its own: no torch at all, or one without HIP."""
    code = """if 1:
        import sys
        if %r == "torch":
            sys.modules["torch"] = None
        else:
            sys.path.insert(0, %r)
        import __graft_entry__ as entry
        from pybgmm_amd import _build
        forced = []
        _build.build = lambda force=False, **k: forced.append(force) or _build.LIB
        entry.build()
        assert forced == [True]
        assert "pybgmm_amd.ops" not in sys.modules
    """ % (without, str(tmp_path))
    os.makedirs(str(tmp_path / "torch" / "lib"))
    (tmp_path / "torch" / "__init__.py").write_text("raise ImportError('a torch without HIP')")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert r.returncode == 0, r.stdout


def test_another_torch_gets_another_binding(monkeypatch, tmp_path):
    if not _build.bindable():
        pytest.skip("no torch with HIP")
    log = made(monkeypatch)
    monkeypatch.setattr(_build, "_stale", lambda target, deps: False)
    monkeypatch.setattr(_build, "BOUND_TO", str(tmp_path / "torch.txt"), raising=False)
    _build.build_ops()
    assert log == [_build.OPS_LIB, _build.OPS_BINDING]
    _build.build_ops()
    assert log[2:] == [_build.OPS_LIB]                               # (the same torch: up to date)
    version = _build.importlib.metadata.version
    monkeypatch.setattr(_build.importlib.metadata, "version", lambda name: version(name) + ".1")
    _build.build_ops()
    assert log[3:] == [_build.OPS_LIB, _build.OPS_BINDING]


@pytest.mark.parametrize("script,own", [("build_prof.sh", "kernels_home"), ("build_prof_gram.sh", "kernels_gram"), ("build_prof_seq.sh", "kernels_seq"),
                                        ("build_variant.sh", "kernels_home"), ("build_tsan.sh", None)])
def test_variants_of_the_samplers_library_hold_its_own_objects(script, own, tmp_path):
    """The objects a script of tools/ links besides what it compiles itself."""
    os.makedirs(str(tmp_path / "_obj"))
    for src in _build.SOURCES + _build.OPS_SOURCES:
        (tmp_path / "_obj" / (src + ".o")).write_text("")
    line, = [a for a in open(os.path.join(ROOT, "tools", script)).read().splitlines() if a.startswith("OBJS=")]
    out = subprocess.run(["bash", "-c", "FILE=kernels_home.hip; %s; echo $OBJS" % line], cwd=str(tmp_path), stdout=subprocess.PIPE, text=True, check=True).stdout
    want = set(s for s in _build.SOURCES if s != "%s.hip" % own and (own or s.startswith("kernels_")))
    assert set(os.path.basename(o)[:-2] for o in out.split()) == want


def test_a_torch_without_package_metadata_has_a_name(monkeypatch):
    if not _build.bindable():
        pytest.skip("no torch with HIP")

    def version(name):
        raise _build.importlib.metadata.PackageNotFoundError(name)
    monkeypatch.setattr(_build.importlib.metadata, "version", version)
    assert _build._torch_here().endswith("__init__.py")
