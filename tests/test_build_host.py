"""The build's host side: what one part's failure means for the other, and builders that come at the same time.  Compilers are stood in
for: nothing is compiled here."""
import os
import subprocess
import threading
import time
import types
import warnings

import pytest
import torch

from convnn_b200 import build as B


def output_of(cmd):
    return cmd[cmd.index("-o") + 1]


@pytest.fixture
def elsewhere(monkeypatch, tmp_path):
    """The build's products in a folder of their own, all of them missing."""
    for name in ("LIB", "STAMP", "CALL_LIB", "CALL_STAMP"):
        monkeypatch.setattr(B, name, str(tmp_path / os.path.basename(getattr(B, name))))
    monkeypatch.setattr(B, "OBJ", str(tmp_path / "build"))
    return tmp_path


def compilers(monkeypatch, gpp_works):
    ran = []

    def run(cmd, **kw):
        tool = os.path.basename(cmd[0])
        ran.append(tool)
        if tool == "g++" and gpp_works is None:
            raise FileNotFoundError(2, "Python.h: no such file, nor a compiler")
        if tool == "g++" and not gpp_works:
            return types.SimpleNamespace(returncode=1, stdout="", stderr="Python.h: no such file")
        with open(output_of(cmd), "w") as f:
            f.write(tool)
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(subprocess, "run", run)
    return ran


@pytest.mark.parametrize("force", [False, True])
@pytest.mark.parametrize("gpp_works", [False, None])
def test_the_library_is_built_where_the_host_module_cannot_be(elsewhere, monkeypatch, force, gpp_works):
    ran = compilers(monkeypatch, gpp_works)
    with pytest.warns(RuntimeWarning, match="Python.h"):
        assert B.build(force=force) == B.LIB
    assert os.path.exists(B.LIB) and not B.stale() and not os.path.exists(B.CALL_LIB) and B.call_stale()
    assert "nvcc" in ran


def test_both_are_built(elsewhere, monkeypatch, recwarn):
    ran = compilers(monkeypatch, gpp_works=True)
    B.build()
    assert os.path.exists(B.LIB) and os.path.exists(B.CALL_LIB) and not B.stale() and not B.call_stale()
    assert not [w for w in recwarn if issubclass(w.category, RuntimeWarning)]
    del ran[:]
    B.build()
    assert not ran


@pytest.fixture
def no_calls(monkeypatch):
    """ops as it is before its first 8-bit call."""
    from convnn_b200 import ops
    monkeypatch.setattr(ops, "_calls", None)
    return ops


def test_calls_go_through_python_where_the_module_cannot_be_built(no_calls, monkeypatch):
    def build_call():
        raise RuntimeError("g++ failed")

    monkeypatch.delenv("CONVNN_B200_NO_BUILD", raising=False)
    monkeypatch.setattr(B, "call_stale", lambda: True)
    monkeypatch.setattr(B, "build_call", build_call)
    x, w = torch.zeros(2, 8), torch.zeros(8)
    with torch.no_grad():
        with pytest.warns(RuntimeWarning, match="through Python"), pytest.raises(RuntimeError, match="no CPU path"):
            no_calls.rms_norm(x, w)
        with warnings.catch_warnings(), pytest.raises(RuntimeError, match="no CPU path"):
            warnings.simplefilter("error")                   # (once is enough)
            no_calls.quantize_fp8(x)


def test_a_module_of_another_source_is_not_loaded(no_calls, monkeypatch):
    """Where nothing may be built: its signatures need not be the library's."""
    monkeypatch.setenv("CONVNN_B200_NO_BUILD", "1")
    monkeypatch.setattr(B, "call_stale", lambda: True)
    monkeypatch.setattr(B, "build_call", lambda: pytest.fail("built"))
    with torch.no_grad(), pytest.warns(RuntimeWarning, match="out of date"), pytest.raises(RuntimeError, match="no CPU path"):
        no_calls.rms_norm(torch.zeros(2, 8), torch.zeros(8))
    assert not hasattr(no_calls._calls, "bind")


def test_builders_at_the_same_time_do_not_share_a_file(elsewhere, monkeypatch):
    """Ranks that come first together: each puts a whole file in place."""
    both = threading.Barrier(2)

    def run(cmd, **kw):
        with open(output_of(cmd), "w") as f:
            f.write("first half")
            f.flush()
            both.wait(10)
            f.write(", second half")
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(subprocess, "run", run)
    failed = []

    def build():
        try:
            B.build_call()
        except Exception as e:
            failed.append(e)

    threads = [threading.Thread(target=build) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    with open(B.CALL_LIB) as f:
        assert f.read() == "first half, second half"
    assert not B.call_stale()
    assert sorted(os.listdir(elsewhere)) == sorted(os.path.basename(p) for p in (B.CALL_LIB, B.CALL_STAMP))


def test_a_failed_build_leaves_nothing_behind(elsewhere, monkeypatch):
    def run(cmd, **kw):
        open(output_of(cmd), "w").close()
        return types.SimpleNamespace(returncode=1, stdout="", stderr="no space left")

    monkeypatch.setattr(subprocess, "run", run)
    with pytest.raises(RuntimeError, match="no space left"):
        B.build_call()
    assert os.listdir(elsewhere) == []


def test_threads_that_come_first_together_bind_once(no_calls, monkeypatch):
    bound, calls = [], no_calls._GeneralCalls

    def ordinary():
        bound.append(threading.get_ident())
        time.sleep(0.2)
        return calls

    monkeypatch.setattr(no_calls, "_ordinary_calls", ordinary)
    got = []
    threads = [threading.Thread(target=lambda: got.append(no_calls._calls or no_calls._bind_calls())) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(bound) == 1 and got == [calls] * 4


def test_a_changed_header_rebuilds_the_host_module(elsewhere, monkeypatch):
    """The module calls the library by address with the signatures of the header."""
    compilers(monkeypatch, True)
    header = elsewhere / "include" / "convnn_b200.h"
    header.parent.mkdir()
    with open(os.path.join(B.INCLUDE, header.name)) as f:
        header.write_text(f.read())
    monkeypatch.setattr(B, "INCLUDE", str(header.parent))
    B.build_call()
    assert not B.call_stale()
    header.write_text(header.read_text() + "/* another signature */")
    assert B.call_stale()


def test_the_host_module_takes_the_signatures_from_the_header():
    """A signature that is written down twice can differ."""
    with open(B.CALL_SRC) as f:
        source = f.read()
    for name in ("rms_norm", "rms_norm_fp8", "quantize_fp8", "linear_fp8"):
        assert f"decltype(&convnn_b200_{name})" in source
