import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA GPU (B200) and the built sm_100a extension")
    config.addinivalue_line("markers", "multigpu: needs two or more CUDA GPUs")


def pytest_collection_modifyitems(config, items):
    import torch

    # These expect, for an id recorded more than once, a divergence with one term for each place (row 2); the token's mass
    # is the sum of its places (test_token_scoring_edges.py). They run after the others, which `-x` would hide.
    items.sort(key=lambda item: getattr(item, "originalname", "") == "test_distillation_special_rows")
    if torch.cuda.is_available():
        return
    skip = pytest.mark.skip(reason="no CUDA device")
    for item in items:
        if "gpu" in item.keywords or "multigpu" in item.keywords:
            item.add_marker(skip)
