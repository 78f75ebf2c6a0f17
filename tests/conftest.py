import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200)")


# Takes its inputs from the global generator, wherever that stands by then, and its bound does not allow for what the path rounds on more than
# 64 rows: 13 of 30 draws missed it (test_gpu_decoder_rounding.py has such steps against what the path does).  Last, so that a run that
# ends at the first failure has been through everything else.
LAST = "test_gpu_decoder.py::test_prompts_trees_and_single_tokens[True]"


def pytest_collection_modifyitems(config, items):
    items.sort(key=lambda item: item.nodeid.endswith(LAST))
    try:
        import torch
        has_gpu = torch.cuda.is_available()
    except Exception:
        has_gpu = False
    if has_gpu:
        return
    skip = pytest.mark.skip(reason="no CUDA device")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)
