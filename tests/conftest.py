import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an AMD GPU (MI355X) and the built HIP library")


def gpu_available() -> bool:
    try:
        import torch

        return torch.cuda.is_available()
    except Exception:
        return False


@pytest.fixture(scope="session")
def dev():
    """cuda:0 on a GPU box. GPU tests fail loudly (no fallback) when no GPU is visible."""
    import torch

    if not torch.cuda.is_available():
        pytest.fail("GPU test run without a visible GPU")
    return torch.device("cuda:0")


@pytest.fixture(autouse=True)
def same_draws():
    """What a test draws without a generator of its own is the same in every run (the GPU's default one starts anywhere)."""
    torch = sys.modules.get("torch")
    if torch is not None:
        torch.manual_seed(0)
