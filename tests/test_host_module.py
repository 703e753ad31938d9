"""The native host module (t3st_b200._dfc_host) is handed out only once its
kernel addresses are set."""

import os
import subprocess
import sys
import threading

import pytest

from t3st_b200 import _lib

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def unbound(monkeypatch):
    """As in a process that has not called host() yet; counts the bindings."""
    module = _lib.host()
    calls = []
    monkeypatch.setattr(_lib, "_host", None)
    bind = module.bind
    monkeypatch.setattr(module, "bind", lambda *a: (calls.append(len(a)), bind(*a))[1])
    return module, calls


def test_a_failed_load_leaves_no_module_behind(unbound, monkeypatch):
    module, calls = unbound
    load = _lib.lib

    def fail():
        raise ImportError("no library")

    monkeypatch.setattr(_lib, "lib", fail)
    for _ in range(2):
        with pytest.raises(ImportError):
            _lib.host()
    assert not calls
    monkeypatch.setattr(_lib, "lib", load)
    assert _lib.host() is module and calls == [5]
    assert _lib.host() is module and calls == [5]  # once


def test_threads_wait_for_the_first_call(unbound, monkeypatch):
    module, calls = unbound
    load = _lib.lib
    loading, go = threading.Event(), threading.Event()

    def slow():
        loading.set()
        assert go.wait(60)
        return load()

    monkeypatch.setattr(_lib, "lib", slow)
    seen = []

    def call():
        m = _lib.host()
        seen.append((m, list(calls)))

    first = threading.Thread(target=call)
    first.start()
    assert loading.wait(60)
    second = threading.Thread(target=call)
    second.start()
    second.join(0.3)  # cannot return before the addresses are set
    early = not second.is_alive()
    go.set()
    first.join(60), second.join(60)
    assert not early and seen == [(module, [5])] * 2


def test_an_unbound_module_refuses_its_calls():
    code = """
import importlib
import torch
m = importlib.import_module("t3st_b200._dfc_host")
x, t = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
for call in (lambda: m.dropout(x, x, 0.5, 0, 0, None, None),
             lambda: m.embedding(t, x, x, 1.0, 0.0, 0, 0, None),
             lambda: m.embedding_grad(t, x, x, 1.0, None, 0.0, 0, 0, None, False),
             lambda: m.nn_dropout(x, 0.5, 0, 0, None, None),
             lambda: m.nn_embedding(t, x, 1.0, None, 0.0, 0, 0, None, None, False)):
    try:
        call()
    except RuntimeError as e:
        assert "not bound" in str(e), e
    else:
        raise SystemExit("not refused")
print("refused")
"""
    out = subprocess.run([sys.executable, "-c", code], cwd=REPO, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "refused", out.stderr


def test_a_host_module_of_another_version_is_rebuilt(monkeypatch, tmp_path):
    """An extension left by an earlier version of the sources is found out
    before it is imported, and built again."""
    from t3st_b200 import build

    real, stale = build.HOST_PATH, tmp_path / "old.so"
    source = tmp_path / "old.c"
    builds = []

    def rebuild(force=False):
        builds.append(force)
        stale.unlink()
        stale.symlink_to(real)
        return str(stale)

    for text, want in (("int some_other_symbol;", [True]),
                       ('const char* v(void) { return "t3st_b200._dfc_host version 0"; }', [True])):
        source.write_text(text)
        if stale.is_symlink():
            stale.unlink()
        subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(stale), str(source)], check=True)
        builds.clear()
        monkeypatch.setattr(build, "HOST_PATH", str(stale))
        monkeypatch.setattr(build, "build_host", rebuild)
        monkeypatch.setattr(_lib, "_host", None)
        assert _lib.host().__name__ == "t3st_b200._dfc_host"
        assert builds == want


def test_a_current_host_module_is_not_rebuilt(monkeypatch):
    from t3st_b200 import build

    def rebuild(force=False):
        raise AssertionError("built again")

    monkeypatch.setattr(build, "build_host", rebuild)
    monkeypatch.setattr(_lib, "_host", None)
    assert hasattr(_lib.host(), "StepPlan")


def test_a_host_module_that_stays_wrong_raises(monkeypatch, tmp_path):
    from t3st_b200 import build

    source, other = tmp_path / "old.c", tmp_path / "old.so"
    source.write_text("int some_other_symbol;")
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(other), str(source)], check=True)
    monkeypatch.setattr(build, "HOST_PATH", str(other))
    monkeypatch.setattr(build, "build_host", lambda force=False: str(other))
    monkeypatch.setattr(_lib, "_host", None)
    with pytest.raises(ImportError):
        _lib.host()
    assert _lib._host is None
