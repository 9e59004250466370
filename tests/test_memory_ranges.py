"""tests/cpp/test_memory_ranges.cpp: the arithmetic by which calls refuse buffers that share memory."""
import pytest

from test_frontend import case_names, check_case, run_program

PROGRAM = "test_memory_ranges"


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    return run_program(PROGRAM, tmp_path_factory.mktemp(PROGRAM))


@pytest.mark.parametrize("name", case_names(PROGRAM))
def test_memory_ranges(run, name):
    check_case(run, name)
