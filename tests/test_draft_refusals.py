"""CPU checks of calls that the draft operators refuse before any device work."""
import os
import subprocess

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "test_draft_refusals")


def test_cpp_refusals():
    """The C++ forms (tests/cpp/test_draft_refusals.cpp), which need no device."""
    assert os.path.exists(CPP), "build first: python -c 'import __graft_entry__ as g; g.build()'"
    r = subprocess.run([CPP], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr
