"""Cases whose expected values are known to be wrong: they run, and have to fail."""
import pytest

TWICE = ("expects bfloat16 logits rounded to float32 first, which a few of its tokens show; "
         "tests/test_logits_rounding_gpu.py holds the values rounded once")
WRONG = {
    "test_paged_edges_gpu.py::test_most_of_a_vocabulary_is_touched[50-8191-16000-1100-dtype1]": TWICE,
    "test_paged_edges_gpu.py::test_most_of_a_vocabulary_is_touched[1100-4000-6000-600-dtype4]": TWICE,
}


def pytest_collection_modifyitems(items):
    for item in items:
        why = WRONG.get(item.nodeid.split("/")[-1])
        if why:
            item.add_marker(pytest.mark.xfail(reason=why, strict=True, raises=AssertionError))
