"""The C ABI of include/scmx_cache.h without a GPU: every entry point exported, bound and driven, its host code under AddressSanitizer and
UBSan."""
import importlib.util
import os
import re
import shutil
import subprocess

import pytest
import torch

from tests.conftest import ROOT


@pytest.fixture(scope="module")
def pkg():
    import mxfp4_int8_m5_amd as p
    if not os.path.exists(p._lib.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return p


def header_entries():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "scmx_cache.h")).read(), flags=re.S)
    return {m.group(1): m.group(2).count(",") + 1 for m in re.finditer(r"\b(scmx_\w+)\s*\(([^;{]*?)\)\s*;", text, flags=re.S)}


def test_every_declared_entry_point_is_exported_bound_and_driven(pkg):
    decl, lib = header_entries(), pkg._lib.load()
    assert set(decl) == set(pkg._lib.CACHE_SIGNATURES) and not set(decl) & set(pkg._lib.SIGNATURES)
    with open(os.path.join(ROOT, "tests", "boundary_driver_cache.cpp")) as f:
        calls = f.read()
    for name, nargs in decl.items():
        assert hasattr(lib, name) and len(pkg._lib.CACHE_SIGNATURES[name][1]) == nargs and hasattr(pkg._lib.native(), name) and name + "(" in calls


def test_workspace_sizes(pkg):
    ws = pkg._lib.load().scmx_verify_workspace
    assert ws(8, 151936, 0) == 8 * 38 * 12 and ws(8, 151936, 3) == 8 * 38 * 36 and ws(1, 1, 0) == 12
    assert not any((ws(0, 10, 0), ws(65, 10, 0), ws(1, 0, 0), ws(1, 4194305, 0), ws(1, 10, -1), ws(1, 10, 17)))


def test_cpu_tensors_are_refused(pkg):
    C, D = pkg.sc_cache, pkg.sc_draft
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t)   # noqa: E731
    with pytest.raises(ValueError):
        C.attn_tree(z(2, 1, 64), z(1, 8, 64), z(1, 8, 64), 0)
    with pytest.raises(ValueError):
        C.cache_read(z(1, 8, 64, t=torch.int8), z(1, 8, 64, t=torch.int8), z(1, 8, t=torch.float32), z(1, 8, t=torch.float32), 4)
    with pytest.raises(ValueError):
        C.cache_keep([(z(1, 8, 64), z(1, 8, 64), None, None)], z(2, t=torch.int32), z(1, t=torch.int32), 0)
    with pytest.raises(ValueError):
        D.verify_drafts(z(2, 10), z(2, t=torch.int64), z(2, t=torch.int32))
    with pytest.raises(ValueError):
        C.cache_write(z(1, 192), z(64), z(64), 1e-6, 1, 1, 1, 64, z(1, 8, 64), z(1, 8, 64), 0, z(32, t=torch.float32))


@pytest.mark.skipif(shutil.which(os.environ.get("HIPCC", "hipcc")) is None, reason="needs hipcc to build the instrumented library")
def test_host_code_under_address_and_undefined_behaviour_sanitizers():
    """As tests/test_boundary.py does for scmx.h, with the sources of these entry points alone."""
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    spec = importlib.util.spec_from_file_location("scmx_build", os.path.join(ROOT, "mxfp4-int8-m5_amd", "build.py"))
    builder = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(builder)
    out = os.path.join(builder.HERE, "build", "host_check", "boundary_check_cache")
    exe = builder.build_host_check(os.path.join(ROOT, "tests", "boundary_driver_cache.cpp"), out,
                                   ["api.hip", "silu_table.hip", "cache.hip", "attn_tree.hip", "verify.hip"])
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:abort_on_error=0", UBSAN_OPTIONS="print_stacktrace=1")
    run = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=600, env=env)
    if run.returncode == 77:
        pytest.skip("a GPU is present")
    assert run.returncode == 0, run.stdout[-4000:]
    assert "0 failure(s)" in run.stdout and "runtime error" not in run.stdout and "AddressSanitizer" not in run.stdout
