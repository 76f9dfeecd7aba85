"""Null and impossible arguments of the operators between a token's projections are refused on the host, with no GPU."""
import ctypes

from apeiron_amd import _lib

INVALID = 21


def test_null_context_and_handles():
    L = _lib.load()
    out = ctypes.c_void_p(5)
    tokens, attn, spec, params = _lib.Kv4Tokens(), _lib.Kv4Attn(), _lib.RopeSpec(64, 64, 0, 0, 1e4), _lib.SampleParams()
    assert L.ah_norm_quant_dev(None, 1, None, 1, 1e-6, 1, 64, None, 1, None, None, None, None) == INVALID
    assert L.ah_rope_create(None, ctypes.byref(spec), ctypes.byref(out)) == INVALID
    assert L.ah_rope_free(None, None) == INVALID and L.ah_rope_info(None, None, None) == INVALID
    assert L.ah_rope_dev(None, None, 1, 64, 1, 1, 1, 1, 64, None) == INVALID
    assert L.ah_kv4_create(None, 1, 32, 1, 64, ctypes.byref(out)) == INVALID
    assert L.ah_kv4_free(None, None) == INVALID and L.ah_kv4_info(None, *[None] * 5) == INVALID
    assert L.ah_kv4_append_dev(None, None, None, ctypes.byref(tokens), *[None, 0, 0, None, 0, None, 0, None, 0], None) == INVALID
    assert L.ah_kv4_read_dev(None, None, ctypes.byref(tokens), None, None, None) == INVALID
    assert L.ah_kv4_attn_dev(None, None, ctypes.byref(attn), None, 0, None, 0, None) == INVALID
    assert L.ah_sample_dev(None, 1, 8, 1, 8, ctypes.byref(params), 1, 1, None, None) == INVALID


def test_struct_sizes_match_the_header():
    assert ctypes.sizeof(_lib.RopeSpec) == 2 * 8 + 2 * 4 + 6 * 8
    assert ctypes.sizeof(_lib.Kv4Tokens) == 6 * 8
    assert ctypes.sizeof(_lib.Kv4Attn) == 5 * 8 + 3 * 8 + 8 + 8 + 2 * 8
    assert ctypes.sizeof(_lib.SampleParams) == 4 * 8
