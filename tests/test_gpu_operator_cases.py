"""The ordering of perf/operators.py's calls with torch's: the library's stream does not wait for torch's, so the inputs that
prepare makes have to be there when it returns."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")


def test_inputs_are_complete_when_prepare_returns():
    import torch
    spec = importlib.util.spec_from_file_location("operator_cases", PATH)
    cases = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(cases)
    cases.own = True
    try:
        for case in cases.listed():
            state = cases.prepare(case, 1)
            assert torch.cuda.current_stream().query(), case["name"]
            del state
    finally:
        if cases._context is not None:
            cases._context.close()
        torch.cuda.empty_cache()
