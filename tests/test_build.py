"""The build's own rules, with nothing compiled: what every library is made of, and when it is made again."""
import os
import re
import subprocess

import pytest

from streamvbyte_amd import build as b


class Recorder:
    """Stands for the compiler: writes down the commands and makes their outputs."""

    def __init__(self, monkeypatch):
        self.commands = []
        monkeypatch.setattr(b.subprocess, "Popen", self._popen)

    def _popen(self, cmd, **kw):
        self.commands.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return type("Job", (), {"wait": lambda self: 0, "args": cmd})()

    def units(self):
        return [os.path.basename(c[c.index("-c") + 1]) for c in self.commands if "-c" in c]


@pytest.fixture
def recorder(monkeypatch, tmp_path):
    for name in ("LIB", "STRESS_LIB", "LINK", "OBJ"):
        monkeypatch.setattr(b, name, str(tmp_path / os.path.basename(getattr(b, name))))
    return Recorder(monkeypatch)


HIP = sorted(f for f in os.listdir(b.CSRC) if f.endswith(".hip"))


def test_variant_libraries_are_whole(recorder, tmp_path):
    """A library for an A/B comparison is every unit with the product's flags and its own: _lib.load() asks for every entry
    point of the headers."""
    out = str(tmp_path / "libvariant.so")
    b.build_variant(out, ["-DSOMETHING"], verbose=False)
    assert sorted(recorder.units()) == HIP
    compiles, link = recorder.commands[:-1], recorder.commands[-1]
    for c in compiles:
        assert "-DSOMETHING" in c and all(f in c for f in b.DEVICE_FLAGS)
        assert c[c.index("-o") + 1] in link
    assert link[link.index("-o") + 1] == out and os.path.exists(out)
    assert not os.path.exists(b.LIB) and not os.path.exists(b.LINK)


def test_tools_compile_through_the_build():
    """No tool has units or device flags of its own to fall behind with."""
    tools = os.path.join(b.ROOT, "tools")
    for name in sorted(os.listdir(tools)):
        path = os.path.join(tools, name)
        if os.path.isfile(path) and name.endswith((".py", ".sh")):
            text = open(path).read()
            assert "svb_api.hip" not in text and "packed-fp32" not in text, name
            if re.search(r"SVB_\w+ -shared|-shared .*-DSVB_", text):
                assert "build_variant" in text, name
    text = open(os.path.join(tools, "ab_length_table.sh")).read()
    assert "streamvbyte_amd.build --variant" in text and "-DSVB_LENGTH_TABLE_LDS" in text
    subprocess.check_call(["bash", "-n", os.path.join(tools, "ab_length_table.sh")])


def test_only_what_is_out_of_date_is_made(recorder):
    b.build(verbose=False)
    assert sorted(recorder.units()) == sorted(2 * HIP) and os.readlink(b.LINK) == os.path.basename(b.LIB)
    later = max(os.path.getmtime(p) for p in (b.LIB, b.STRESS_LIB)) + 10

    def commands(force=False):
        recorder.commands.clear()
        b.build(force=force, verbose=False)
        return len(recorder.commands)
    assert commands() == 0
    # libraries that travelled without their objects are as good as they were
    for f in os.listdir(b.OBJ):
        os.remove(os.path.join(b.OBJ, f))
    assert commands() == 0
    # ... until a library is missing or older than a source, or everything is asked for
    os.remove(b.STRESS_LIB)
    assert commands() == len(HIP) + 1
    for f in os.listdir(b.OBJ):
        os.utime(os.path.join(b.OBJ, f), (0, 0))
    os.utime(b.LIB, (0, 0))
    assert commands() == len(HIP) + 1
    # a link that did not happen is made up for
    for f in os.listdir(b.OBJ):
        os.utime(os.path.join(b.OBJ, f), (later, later))
    os.utime(b.LIB, (0, 0))
    assert commands() == 1
    assert commands(force=True) == 2 * len(HIP) + 2
