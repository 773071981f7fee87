import os
import sys

import pytest

# torch brings a HIP runtime of its own.  Loaded first, it is the library's as well; behind the library, which then has the system's, it is a second one, and the streams,
# graphs and events of one are none to the other.
try:
    import torch  # noqa: F401
except ImportError:
    pass

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu)")
