"""Shared test setup.

The package directory is ``yolo11.cu_b200/`` (a dotted name), so it is loaded by path as
``yolo11_cu_b200``.  The oracle (``oracle/``) is test infrastructure and is imported only
from here and the test files.
"""
import importlib.util
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG_DIR = os.path.join(ROOT, "yolo11.cu_b200")
GOLDEN = os.path.join(ROOT, "tests", "golden")
MODELS = os.path.join(ROOT, "models")


def load_pkg():
    if "yolo11_cu_b200" in sys.modules:
        return sys.modules["yolo11_cu_b200"]
    spec = importlib.util.spec_from_file_location(
        "yolo11_cu_b200", os.path.join(PKG_DIR, "__init__.py"), submodule_search_locations=[PKG_DIR])
    mod = importlib.util.module_from_spec(spec)
    sys.modules["yolo11_cu_b200"] = mod
    spec.loader.exec_module(mod)
    return mod


load_pkg()
if os.path.join(ROOT, "oracle") not in sys.path:
    sys.path.insert(0, os.path.join(ROOT, "oracle"))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA GPU (B200, sm_100a)")


@pytest.fixture(scope="session")
def pkg():
    return load_pkg()


@pytest.fixture(scope="session")
def lib(pkg):
    from yolo11_cu_b200 import build, runtime
    build.build()
    return runtime.load()


def release_hooks(lib):
    """The library's own rules again, whatever a test forced (yk_test_inject, which takes a GPU, is its test's own to release)."""
    lib.yk_test_nms_cluster(0)
    lib.yk_test_attn_kv8(0)
    lib.yk_test_gemm_fp4(0, 0)
    lib.yk_test_sample(0)
    lib.yk_test_sample_kernel(0)


@pytest.fixture(autouse=True)
def hooks_end_with_their_test():
    yield
    from yolo11_cu_b200 import runtime
    if runtime._lib is not None:
        release_hooks(runtime._lib)


@pytest.fixture(scope="session")
def cuda():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.init()
    return torch.device("cuda:0")


def golden_cases():
    return sorted(d for d in os.listdir(GOLDEN) if os.path.isdir(os.path.join(GOLDEN, d)))


def split_case(case):
    name, S = case.rsplit("-", 1)
    return name, int(S)


@pytest.fixture(scope="session")
def golden_dirs(pkg, tmp_path_factory):
    """Model directories regenerated by this package's exporter for every golden case."""
    from yolo11_cu_b200 import export
    base = tmp_path_factory.mktemp("golden_models")
    out = {}
    for case in golden_cases():
        name, S = split_case(case)
        d = str(base / case)
        export.export_model(name, d, S)
        out[case] = d
    return out
