"""pytest configuration: the ``gpu`` marker and import paths.

``-m "not gpu"`` runs on a host without a GPU (oracle, golden fixtures, C-ABI
exports and argument checks, host logic, gloo multi-rank tests);
``-m gpu`` runs the parity tests through the C-ABI on a B200.
"""

from __future__ import annotations

import os
import sys

import pytest

# The float64 products of the CPU checks must not depend on a column's place in the matrix (equal
# centroids tie exactly); some of MKL's kernels round the edge columns differently (seen with AVX-512 on AMD EPYC).
os.environ.setdefault("MKL_CBWR", "COMPATIBLE")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "flash-kmeans-cuda_b200")
for p in (PKG, ROOT):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200); runs the CUDA kernels")


@pytest.fixture(scope="session")
def cuda_device():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("CUDA not available")
    return torch.device("cuda", 0)
