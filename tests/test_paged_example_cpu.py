"""examples/paged_generate.py refuses what it cannot serve before it touches a GPU."""

import os
import sys

import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("args", [["--new", "0"], ["--prompts", "5,0"], ["--chunk", "0"], ["--budget", "8", "--recent", "9"],
                                  ["--budget", "-1"]])
def test_arguments_that_leave_nothing_to_serve(monkeypatch, args):
    import paged_generate as pg

    def no_model(*a):
        raise AssertionError("a model was made")

    monkeypatch.setattr(pg, "Decoder", no_model)
    monkeypatch.setattr(sys, "argv", ["paged_generate.py", *args])
    with pytest.raises(SystemExit) as e:
        pg.main()
    assert e.value.code == 2
