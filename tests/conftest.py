"""pytest configuration: the ``gpu`` marker and import paths."""
import os
import random
import socket
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
GOLDEN = os.path.join(ROOT, "tests", "golden")
for p in (ROOT, GOLDEN):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


_choice = random.Random()          # of its own: tests seed the global one


def _port_below_the_ephemeral_ones() -> int:
    """A free port that no outgoing connection is given (those start at 32768): one from bind(0) can be taken again in the
    seconds between its choice and a rank's listening on it (EADDRINUSE in init_process_group)."""
    for _ in range(1000):
        port = _choice.randrange(20000, 32000)
        with socket.socket() as s:
            try:
                s.bind(("0.0.0.0", port))
                return port
            except OSError:
                pass
    raise RuntimeError("no free port below 32000")


@pytest.fixture(autouse=True)
def _ports_for_ranks(request, monkeypatch):
    if hasattr(getattr(request, "module", None), "_free_port"):
        monkeypatch.setattr(request.module, "_free_port", _port_below_the_ephemeral_ones)
