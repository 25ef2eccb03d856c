"""The serving operators' calls at the ends of what include/moe_serve.h allows, on the host (tests/cpp/serve_bounds_test.cpp)."""
import subprocess

import pytest

from tests.test_dense_calls import build


@pytest.fixture(scope="module")
def bounds(tmp_path_factory):
    return build(tmp_path_factory.mktemp("bounds"), "serve_bounds_test", "serve_api.cpp")


def run(bounds, what):
    r = subprocess.run([bounds, what], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout


def test_masses_of_a_row_fit_64_bits(bounds):
    run(bounds, "shift")


def test_launches_of_wide_rows(bounds):
    run(bounds, "rows")


def test_workspace_of_wide_products(bounds):
    run(bounds, "terms")


def test_products_without_a_workspace(bounds):
    run(bounds, "alone")
