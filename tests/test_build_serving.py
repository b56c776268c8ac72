"""The tensor front end is built again when the torch or the interpreter that it was built for has changed."""
import importlib.metadata
import os

from bitstack_b200 import build


def test_front_end_follows_torch_and_interpreter(tmp_path, monkeypatch):
    runs = []

    def compile_(cmd, **_):
        runs.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
    monkeypatch.setattr(build, "HERE", str(tmp_path))
    monkeypatch.setattr(build, "SERVING_LIB", os.path.join(str(tmp_path), "_serving.so"))
    monkeypatch.setattr(build.subprocess, "check_call", compile_)
    version = importlib.metadata.version
    build.build_serving()
    build.build_serving()
    assert len(runs) == 1
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "0.0.1" if name == "torch" else version(name))
    build.build_serving()
    build.build_serving()
    assert len(runs) == 2
    monkeypatch.setattr(build.sysconfig, "get_config_var", lambda name: "cpython-300")
    build.build_serving()
    assert len(runs) == 3
    build.build_serving(force=True)
    assert len(runs) == 4
