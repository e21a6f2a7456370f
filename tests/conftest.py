import os
import sys

import pytest

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for _p in (os.path.join(_ROOT, "flash-model-architectures_b200"), _ROOT, os.path.dirname(os.path.abspath(__file__))):
    if _p not in sys.path:
        sys.path.insert(0, _p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200)")


@pytest.fixture(scope="session", autouse=True)
def _library_products_are_summed_in_float32():
    """The products that tests compare with, and the router's gate where it is a library product, are rounded once. By default
    the library may add up 16-bit partial sums where it splits the reduction, and whether it does differs from machine to
    machine (7 tokens, 6 experts, H=2048: 25 of 42 logits off the rounded product on one, by up to a step)."""
    import torch

    matmul = torch.backends.cuda.matmul
    before = matmul.allow_bf16_reduced_precision_reduction, matmul.allow_fp16_reduced_precision_reduction
    matmul.allow_bf16_reduced_precision_reduction = matmul.allow_fp16_reduced_precision_reduction = False
    yield
    matmul.allow_bf16_reduced_precision_reduction, matmul.allow_fp16_reduced_precision_reduction = before


@pytest.fixture(scope="session", autouse=True)
def _native_library_is_built():
    """The shared library is built once per session (nvcc cross-compiles without a GPU)."""
    sys.path.insert(0, os.path.join(_ROOT, "flash-model-architectures_b200"))
    import build as xma_build

    xma_build.build()


@pytest.fixture()
def device():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)
