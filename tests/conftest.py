"""pytest configuration: the ``gpu`` marker and import paths.

``-m "not gpu"`` runs on any host (oracle, host logic, library symbols);
``-m gpu`` needs a ROCm device and the built ``libnmce.so``.
"""

import pathlib
import sys

import pytest

ROOT = pathlib.Path(__file__).resolve().parent.parent
for p in (ROOT, ROOT / "nano-megatron_amd"):
    if str(p) not in sys.path:
        sys.path.insert(0, str(p))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a ROCm GPU and the built libnmce.so")


# Tests whose own reference is wrong. They run as they are, and have to fail: test_distill_gpu's
# _reference adds p log p for every place of a list, where an id that comes several times has
# (sum of its p) log (sum of its p). Of the list [5, 5] of equal logits and a student that is
# certain of 5 it makes the divergence -log 2. (Lists that name an id once are not touched by it,
# and test_distill_again_gpu has the same inputs with lists that are merged first.)
_WRONG_REFERENCE = ("test_distill_gpu.py::test_an_id_that_comes_again[",
                    "test_distill_gpu.py::test_long_lists_of_few_ids[")


def pytest_collection_modifyitems(items):
    for item in items:
        if any(name in item.nodeid for name in _WRONG_REFERENCE):
            item.add_marker(pytest.mark.xfail(
                strict=True, raises=AssertionError,
                reason="its reference sums p log p by places of the list, not by ids"))
