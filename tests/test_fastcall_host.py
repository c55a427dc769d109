"""The argument-conversion module of the hot entry points among threads, and its build: on the host."""

from __future__ import annotations

import ctypes
import threading
import time

import pytest

from qtts_b200 import _native as nat

NORM = [16, 64, 16, 64, 16, 1e-6, 16, 64, nat.BF16, 16, 64, nat.E4M3, 16, 4, 64, 0, None]


def addresses():
    return [ctypes.cast(getattr(nat.lib(), name), ctypes.c_void_p).value for name in nat._LAUNCHED]


def test_other_threads_run_during_a_call():
    # A launch may block (a full queue, a module's first load). Threads that run Python must not stand
    # still for it: the work that it waits for may need one of them.
    fast = nat._fastcall()
    if fast is None:
        pytest.skip("csrc/fastcall.c is not built here")
    libc = ctypes.CDLL(None)
    seen, stop = [], threading.Event()

    def other():
        while not stop.is_set():
            seen.append(time.monotonic())
            time.sleep(0.002)

    thread = threading.Thread(target=other)
    thread.start()
    try:
        # usleep in the place of an entry point: its first argument is the time.
        fast.bind(ctypes.cast(libc.usleep, ctypes.c_void_p).value, *addresses()[1:])
        time.sleep(0.02)
        began = time.monotonic()
        fast.qtts_add_rms_norm_quant(400_000, *NORM[1:])
        ended = time.monotonic()
    finally:
        fast.bind(*addresses())
        stop.set()
        thread.join()
    assert ended - began >= 0.35
    assert sum(began + 0.05 < t < ended - 0.05 for t in seen) >= 10


def test_first_calls_of_two_threads(monkeypatch):
    # The second thread arrives while the first is still looking entry points up.
    half_done, go_on = threading.Event(), threading.Event()

    class Slow:
        def __getattr__(self, name):
            if name == nat._LAUNCHED[-1]:
                half_done.set()
                assert go_on.wait(10)
            return lambda *args: nat.OK

    monkeypatch.setattr(nat, "_calls", {})
    monkeypatch.setattr(nat, "_fastcall", Slow)
    monkeypatch.setattr(nat, "_raw_device", lambda: 0)
    monkeypatch.setattr(nat, "_raw_stream", lambda index: None)
    failed = []

    def call(name):
        try:
            nat.launch(name, 0)
        except BaseException as e:  # noqa: BLE001 - the test's result
            failed.append(e)

    threads = [threading.Thread(target=call, args=(name,)) for name in (nat._LAUNCHED[0], nat._LAUNCHED[-1])]
    threads[0].start()
    assert half_done.wait(10)
    threads[1].start()
    time.sleep(0.1)
    go_on.set()
    for t in threads:
        t.join(10)
    assert not failed and set(nat._calls) == set(nat._LAUNCHED)


@pytest.fixture
def build_dir(monkeypatch, tmp_path):
    from qtts_b200 import build

    monkeypatch.setattr(build, "LIB_DIR", tmp_path)
    monkeypatch.setattr(build, "LIB_PATH", tmp_path / "libqtts_b200.so")
    monkeypatch.setattr(build, "FAST_PATH", tmp_path / "_qtts_fastcall.so")
    monkeypatch.setattr(build, "nvcc_path", lambda: "nvcc")
    monkeypatch.setattr(build, "PKG_DIR", tmp_path / "pkg")
    return build


def runs(monkeypatch, build, fails):
    """Commands as build._run sees them: the output file appears, or the command fails."""
    seen = []

    def run(cmd, verbose):
        what = "nvcc" if cmd[0] == "nvcc" else "cc"
        seen.append(what)
        if what in fails:
            raise RuntimeError(f"{what} failed")
        out = cmd[cmd.index("-o") + 1]
        with open(out, "w") as f:
            f.write("new")

    monkeypatch.setattr(build, "_run", run)
    return seen


def test_a_failed_compile_of_the_module_leaves_the_library(build_dir, monkeypatch):
    # The module is optional: without it the calls go through ctypes.
    build_dir.FAST_PATH.write_text("old")
    runs(monkeypatch, build_dir, {"cc"})
    assert build_dir.build(force=True) == build_dir.LIB_PATH and build_dir.LIB_PATH.read_text() == "new"
    assert not build_dir.FAST_PATH.exists()  # one of an earlier library would pass its old argument lists


@pytest.mark.parametrize("gone", ["cc", "header"])
def test_no_compiler_leaves_no_old_module(build_dir, monkeypatch, gone):
    build_dir.FAST_PATH.write_text("old")
    runs(monkeypatch, build_dir, set())
    if gone == "cc":
        monkeypatch.setattr(build_dir.shutil, "which", lambda name: None)
    else:
        monkeypatch.setattr(build_dir.sysconfig, "get_paths", lambda: {"include": "/nowhere"})
    build_dir.build(force=True)
    assert build_dir.LIB_PATH.read_text() == "new" and not build_dir.FAST_PATH.exists()


def test_a_failed_library_leaves_library_and_module_as_they_were(build_dir, monkeypatch):
    build_dir.LIB_PATH.write_text("old")
    build_dir.FAST_PATH.write_text("old")
    runs(monkeypatch, build_dir, {"nvcc"})
    with pytest.raises(RuntimeError):
        build_dir.build(force=True)
    assert build_dir.LIB_PATH.read_text() == build_dir.FAST_PATH.read_text() == "old"


def test_the_module_is_built_behind_the_library(build_dir, monkeypatch):
    seen = runs(monkeypatch, build_dir, set())
    build_dir.build(force=True)
    assert seen[-2:] == ["nvcc", "cc"] and build_dir.FAST_PATH.read_text() == "new"
