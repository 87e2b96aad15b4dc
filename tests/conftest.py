import gc
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an AMD GPU and the built HIP kernels")


@pytest.fixture(scope="session")
def gpu_device():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


@pytest.fixture(scope="module", autouse=True)
def garbage_of_earlier_modules():
    """What earlier modules' tests left in reference cycles is freed before a module begins, not
    whenever Python next looks for it: a test that reads the device's memory before and after a
    call must not find an earlier test's tensors freed in between."""
    gc.collect()
