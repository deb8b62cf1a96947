"""Addresses that no 32-bit value can have are refused by the calls of a paged cache: a kernel that read from them would fault.  No GPU: argument checks come first."""
import ctypes as C

import pytest

from test_paged_refusals import P, attention, cache, pkg, refused, verification


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("name", ["k_scale", "v_scale", "table", "lens", "starts"])
def test_arrays_of_a_cache(name, off):
    lib, c = pkg.load_kernels(), cache(**{name: P + off})
    refused(lib.lv_paged_append(None, C.byref(c), P, P, pkg.TYPE_F32, 256, None, 0, 0, 3), "4-byte")
    refused(lib.lv_paged_read(None, C.byref(c), P, P, pkg.TYPE_F32, 0, 0, 0, 0, 3), "4-byte")
    a = attention(c)
    refused(lib.lv_paged_attention(None, C.byref(a), P, 1 << 30), "4-byte")
    assert lib.lv_paged_attention_scratch_bytes(None, C.byref(a)) == 0


def test_scales_that_nothing_reads():
    lib, c = pkg.load_kernels(), cache(type=pkg.TYPE_F16, k_scale=P + 1, v_scale=None)
    refused(lib.lv_paged_append(None, C.byref(c), P, P, pkg.TYPE_F32, 256, None, 0, 0, 3), "null context")


def test_sinks():
    refused(pkg.load_kernels().lv_paged_attention(None, C.byref(attention(sink=P + 2)), P, 1 << 30), "4-byte")


@pytest.mark.parametrize("out,logits,temperature", [(P + 2, P, P), (P, P + 1, P), (P, P, P + 3)])
def test_probabilities(out, logits, temperature):
    refused(pkg.load_kernels().lv_probabilities(None, out, 10, logits, 10, 10, 2, temperature), "4-byte")


@pytest.mark.parametrize("name", ["target", "draft", "drafted", "starts", "accept", "pick", "tokens", "accepted", "lens"])
def test_verification(name):
    refused(pkg.load_kernels().lv_verify_drafts(None, C.byref(verification(**{name: P + 2}))), "4-byte")
