import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "tests")):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a B200 (sm_100a) GPU; parity tests of the CUDA path")


# CPU tests that pass made-up addresses to calls that the library accepts: without a device they end in an error.
NEEDS_NO_DEVICE = {"test_gradient_that_overlaps_its_logits_is_refused"}


def pytest_runtest_setup(item):
    if item.name in NEEDS_NO_DEVICE:
        import torch

        if torch.cuda.is_available():
            pytest.skip("its addresses are not memory: only where there is no CUDA device")


@pytest.fixture(scope="session")
def cuda():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    major, minor = torch.cuda.get_device_capability(0)
    if major != 10:
        pytest.skip(f"needs sm_100 (found sm_{major}{minor})")
    import dirktensor_b200  # noqa: F401  (fails loudly if the library is missing)

    return torch.device("cuda:0")
