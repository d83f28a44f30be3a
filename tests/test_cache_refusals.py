"""What the entry points of include/scmx_cache.h refuse before anything is launched, by their status (no GPU: the addresses are none)."""
import pytest
import torch


@pytest.mark.skipif(torch.cuda.is_available(), reason="the calls that are accepted would be launched")
@pytest.mark.parametrize("scale,refused", [(2.4e38, True), (-2.4e38, True), (3.0e38, True), (float("inf"), True), (float("nan"), True),
                                           (2.3e38, False), (-2.3e38, False), (0.0, False)])
def test_attention_scales(scale, refused):
    """The scale is taken in powers of two, so that it has to be finite times log2 e."""
    import mxfp4_int8_m5_amd as scmx
    lib, at = scmx._lib.load(), 4096
    rc = lib.scmx_attn_tree(at, at, at, None, None, None, None, 0, at, 1, 1, 1, 64, 8, scale, None, 1, None)
    assert rc < 0 and (b"scale" in lib.scmx_last_error()) == refused
