"""What the compiler made of the kernels of libbattgp_products.so (CPU suite; hipcc cross-compiles gfx950): read from the
assembly of the sources as battgp_amd/build.py compiles them."""

import os
import re
import sys
from concurrent.futures import ThreadPoolExecutor

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tools"))

pytestmark = pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")


@pytest.fixture(scope="module")
def code(tmp_path_factory):
    import kernel_resources as kr

    from battgp_amd import build

    tmp = tmp_path_factory.mktemp("asm")
    os.mkdir(tmp / "products")
    own = [f for f in build.PRODUCTS_FLAGS if f not in build.FLAGS or f == "-Xclang"]
    with ThreadPoolExecutor(2) as pool:
        texts = list(pool.map(lambda s: kr.compile_asm("products/" + s, str(tmp), own), build.PRODUCTS_SOURCES))
    rows = {}
    for text in texts:
        found = kr.resources(text)
        for r, name in zip(found, kr.demangle([r["name"] for r in found])):
            rows[name] = dict(r, text=text)
    return rows


def test_no_kernel_spills(code):
    assert len(code) > 80  # the table really was parsed
    for name, r in code.items():
        assert r["scratch"] == 0, name


def test_no_packed_fp32_arithmetic(code):
    for text in {r["text"] for r in code.values()}:
        assert not re.search(r"v_pk_(add|mul|fma)_f32", text)


def test_workgroups_fit_a_cu_as_their_launches_assume(code):
    """160 KB of LDS and 512 registers for each lane of a SIMD: two workgroups of 4 waves, one of 8"""
    for name, r in code.items():
        if r["wg"] == 256 and "quantize" not in name:
            assert 2 * r["lds"] <= 160 * 1024 and 2 * r["vgpr"] <= 512, name
        else:
            assert r["lds"] <= 160 * 1024 and r["wg"] // 256 * r["vgpr"] <= 512, name


def test_nothing_but_the_loads_into_lds_uses_m0(code):
    """The inline assembly of those loads sets m0 and can not say so: it is a reserved register, which a clobber list may
    not name.  The compiler keeps no value of its own in it, but may use it for an instruction that takes it unnamed."""
    unnamed = re.compile(r"movrel|s_set_gpr_idx|gws|sendmsg|ttrace|addtid|\blds\b|_interp_")
    for text in {r["text"] for r in code.values()}:
        lines = [line.split(";")[0].strip() for line in text.split("\n")]
        sets = [i for i, line in enumerate(lines) if re.search(r"\bm0\b", line)]
        assert len(sets) > 100
        for i in sets:
            assert re.fullmatch(r"s_mov_b32 m0, s\d+", lines[i]) and lines[i + 1] == "s_nop 0" and lines[i + 2].startswith("global_load_lds_dwordx4 "), lines[i]
        loads = [line for line in lines if "global_load_lds" in line]
        assert len(loads) == len(sets)
        assert not [line for line in lines if unnamed.search(line) and not line.startswith(".")]
