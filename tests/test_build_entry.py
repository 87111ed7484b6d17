"""What build() makes: the library, the oracle and the first mirror driver.  Programs of single tests are those tests' own to build."""
import os
import subprocess

import __graft_entry__ as entry


def test_build_asks_the_test_directory_for_one_program(monkeypatch):
    """build() has to work beside a test directory that knows no other program than the engine mirror's driver."""
    asked = []
    monkeypatch.setattr(subprocess, "check_call", lambda command, *a, **k: asked.append(command))
    entry.build()
    here = os.path.dirname(os.path.abspath(__file__))
    directories = [os.path.realpath(c[c.index("-C") + 1]) for c in asked]
    assert len(asked) == 3 and directories.count(os.path.realpath(here)) == 1
    command = asked[directories.index(os.path.realpath(here))]
    options = command[command.index("-C") + 2:]
    assert options == ["-B", "vmath_mirror_driver"]
