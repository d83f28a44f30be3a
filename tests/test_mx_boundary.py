"""The C ABI of include/scmx_mx.h without a GPU: every entry point exported, bound and driven, its host code under AddressSanitizer and
UBSan; what the Python entry points refuse."""
import importlib.util
import os
import re
import shutil
import subprocess

import pytest
import torch

from tests.conftest import ROOT

BF = torch.bfloat16


@pytest.fixture(scope="module")
def pkg():
    import mxfp4_int8_m5_amd as p
    if not os.path.exists(p._lib.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return p


def header_entries():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "scmx_mx.h")).read(), flags=re.S)
    return {m.group(1): m.group(2).count(",") + 1 for m in re.finditer(r"\b(scmx_\w+)\s*\(([^;{]*?)\)\s*;", text, flags=re.S)}


def test_every_declared_entry_point_is_exported_bound_and_driven(pkg):
    decl, lib, sigs = header_entries(), pkg._lib.load(), pkg._lib.MX_SIGNATURES
    assert set(decl) == set(sigs) and not set(decl) & (set(pkg._lib.SIGNATURES) | set(pkg._lib.CACHE_SIGNATURES))
    with open(os.path.join(ROOT, "tests", "boundary_driver_mx.cpp")) as f:
        calls = f.read()
    for name, nargs in decl.items():
        assert hasattr(lib, name) and len(sigs[name][1]) == nargs and hasattr(pkg._lib.native(), name) and name + "(" in calls


def test_the_ranges_of_a_cache(pkg):
    """Whole up to 512 rows; as many as the CUs hold, twice as many behind long contexts; never more than 64."""
    s = lambda T, n, hq, hk, d: pkg.sc_cache.attn_tree_splits(T, n, hq, hk, d, 4)   # noqa: E731
    assert s(1, 500, 16, 8, 128) == 1 and s(1, 40000, 16, 8, 128) == 64 and s(1, 2 ** 31 - 1, 1, 1, 64) == 64
    assert all(1 <= s(T, n, hq, hk, d) <= 64 for T in (1, 17, 64) for n in (1, 32, 700, 5000, 10 ** 6) for hq, hk in ((1, 1), (16, 8), (4096, 4096)) for d in (64, 128, 256))


def test_cpu_tensors_and_bad_operands_are_refused(pkg):
    X, C = pkg.sc_mx, pkg.sc_cache
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)   # noqa: E731
    bf = lambda *s: torch.zeros(*s, dtype=BF)            # noqa: E731
    w = u8(8, 32), u8(8, 2)
    for bad in (lambda: X.quantize(bf(2, 64)), lambda: X.quantize(bf(2, 63)), lambda: X.quantize(u8(2, 64)), lambda: X.dequantize(u8(2, 32), u8(2, 2)),
                lambda: X.dequantize(u8(2, 32), u8(2, 3)), lambda: X.mm(u8(2, 32), u8(2, 2), *w), lambda: X.mm(u8(2, 16), u8(2, 1), *w),
                lambda: X.linear(bf(2, 64), *w), lambda: X.linear(bf(2, 96), *w), lambda: X.linear(bf(2, 64), *w, 2), lambda: X.linear(bf(2, 64), *w, 4),
                lambda: C.attn_tree(bf(2, 1, 64), u8(1, 8, 32), u8(1, 8, 32), 0, None, u8(1, 8, 2), u8(1, 8, 2)),
                lambda: C.attn_tree(bf(2, 1, 64), u8(1, 8, 32), u8(1, 8, 32), 0, None, u8(1, 8, 4), u8(1, 8, 4)),
                lambda: C.cache_read(u8(1, 8, 32), u8(1, 8, 32), u8(1, 8, 2), u8(1, 8, 2), 4),
                lambda: C.cache_keep([(u8(1, 8, 32), u8(1, 8, 32), u8(1, 8, 2), u8(1, 8, 2))], torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 0),
                lambda: C.cache_write(bf(1, 192), bf(64), bf(64), 1e-6, 1, 1, 1, 64, u8(1, 8, 32), u8(1, 8, 32), 0, torch.zeros(32), u8(1, 8, 2), u8(1, 8, 2))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.skipif(shutil.which(os.environ.get("HIPCC", "hipcc")) is None, reason="needs hipcc to build the instrumented library")
def test_host_code_under_address_and_undefined_behaviour_sanitizers():
    """As tests/test_boundary.py does for scmx.h, with the sources of these entry points alone."""
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    spec = importlib.util.spec_from_file_location("scmx_build", os.path.join(ROOT, "mxfp4-int8-m5_amd", "build.py"))
    builder = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(builder)
    out = os.path.join(builder.HERE, "build", "host_check", "boundary_check_mx")
    exe = builder.build_host_check(os.path.join(ROOT, "tests", "boundary_driver_mx.cpp"), out,
                                   ["api.hip", "silu_table.hip", "mx_quant.hip", "mx_gemm.hip", "cache4.hip", "attn_tree4.hip"])
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:abort_on_error=0", UBSAN_OPTIONS="print_stacktrace=1")
    run = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=600, env=env)
    if run.returncode == 77:
        pytest.skip("a GPU is present")
    assert run.returncode == 0, run.stdout[-4000:]
    assert "0 failure(s)" in run.stdout and "runtime error" not in run.stdout and "AddressSanitizer" not in run.stdout
