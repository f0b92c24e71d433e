"""The extension module is bound to one Python and one torch: a build for another is made again, and an import
of it says what is wrong."""
import pytest


def test_a_build_for_another_torch_is_stale(tmp_path, monkeypatch):
    from mole_b200 import build
    for name in ("LIB", "HOST_LIB", "HOST_STAMP"):        # newer than every source
        monkeypatch.setattr(build, name, tmp_path / name)
        (tmp_path / name).write_text("")
    assert build._stale()
    build.HOST_STAMP.write_text(build.host_abi())
    assert not build._stale()
    build.HOST_STAMP.write_text("cpython-399, torch 0.0")
    assert build._stale()
    build.HOST_STAMP.unlink()                             # built by something that left no word of it
    assert build._stale()


def test_an_import_says_what_the_module_was_built_for(tmp_path):
    from mole_b200 import _host, build
    with pytest.raises(ImportError, match=r"is missing.*mole_b200/build\.py"):
        _host._load(tmp_path / "none.so")
    lib, stamp = tmp_path / "_host.so", tmp_path / "_host.built_for"
    lib.write_bytes(b"no shared object")
    stamp.write_text("cpython-399, torch 0.0")
    with pytest.raises(ImportError, match=r"built for cpython-399, torch 0\.0; here is .*torch.*mole_b200/build\.py"):
        _host._load(lib, stamp)
    stamp.write_text(build.host_abi())
    with pytest.raises(ImportError, match=r"does not load with .*torch.*mole_b200/build\.py"):
        _host._load(lib, stamp)
