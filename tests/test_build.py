"""The build script on a machine without torch: libkmc.so needs none, and the torch binding is left out."""
import importlib.util
import os
import sys

from conftest import ROOT


def test_build_without_torch(tmp_path, monkeypatch, capsys):
    spec = importlib.util.spec_from_file_location("kmc_build", os.path.join(ROOT, "mlx_kmeans_b200", "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    monkeypatch.setattr(build, "BIND", str(tmp_path / "_experts.so"))
    monkeypatch.setattr(build, "up_to_date", lambda: True)
    monkeypatch.setitem(sys.modules, "torch", None)            # importing it raises ImportError
    assert build.build() == build.LIB
    assert not os.path.exists(build.BIND)
    assert "torch" in capsys.readouterr().err
