import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "oracle"), os.path.dirname(os.path.abspath(__file__))):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (gfx950) GPU and the built HIP library")


# Cases that hold a wrong value, and where the right one is tested.
_ONE_CALL = ("its float64 decoder takes a step's drafts in one call, so that the rows before a block's end see the block in codes whose "
             "scale has the drafts after them; the rows are those of single steps (test_drafts_rows.py)")
WRONG = {"test_serving_step.py::test_decoder_by_drafts[False-True-True]": _ONE_CALL,
         "test_serving_step.py::test_decoder_by_drafts[True-True-True]": _ONE_CALL}


def pytest_collection_modifyitems(items):
    for item in items:
        reason = WRONG.get(item.nodeid.rsplit("/", 1)[-1])
        if reason:
            item.add_marker(pytest.mark.xfail(reason=reason, raises=AssertionError, strict=True))


@pytest.fixture(scope="session")
def orc():
    import oracle as orc_mod
    orc_mod.lib()
    return orc_mod
