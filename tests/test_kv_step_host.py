"""What of the 4-bit cache, the head norms and the pages' step needs no GPU: the structs' layout, the refusals of the C ABI, and the
reference's own rounding."""
import ctypes
import re

import pytest
import torch

import candelora_metal_kernels_b200 as c
import kv_step_reference as ref
from candelora_metal_kernels_b200 import _lib
from candelora_metal_kernels_b200.build import build
from conftest import ROOT
from test_attention_host import _SIZES, _fields


@pytest.fixture(scope="module")
def lib():
    build()
    return _lib.load()


@pytest.mark.parametrize("name,packed", [("iq2_head_norms", _lib.HEAD_NORMS), ("iq2_kv_step", _lib.KV_STEP)])
def test_packed_structs_have_the_headers_fields(name, packed):
    fields = [(f, _SIZES[t]) for f, t in _fields(name)]
    struct = type("S", (ctypes.Structure,), {"_fields_": fields})
    assert packed.size == ctypes.sizeof(struct)
    assert re.sub(r"0q$", "", packed.format.strip("@")) == "".join(t for _, t in _fields(name))


def test_pages_struct_matches_the_header():
    kinds = {ctypes.c_void_p: "P", ctypes.c_uint32: "I"}
    assert [(n, kinds[t]) for n, t in _lib.KvPagesStruct._fields_] == _fields("iq2_kv_pages")


def test_rust_structs_have_the_headers_fields():
    ffi = (ROOT / "candelora_metal_kernels_b200" / "rust" / "src" / "iq2_cuda_ffi.rs").read_text()
    kinds = {"u32": "I", "c_int": "i", "f32": "f"}
    for rust, name in (("Iq2HeadNorms", "iq2_head_norms"), ("Iq2KvPages", "iq2_kv_pages"), ("Iq2KvStep", "iq2_kv_step")):
        body = re.search(r"pub struct %s \{(.*?)\}" % rust, ffi, re.S).group(1)
        assert [(f, "P" if t.startswith("*") else kinds[t]) for f, t in re.findall(r"pub (\w+): ([^,]+),", body)] == _fields(name)
    assert "pub const IQ2_KV_INT4: c_int = %d;" % _lib.KV_INT4 in ffi


def _pages(lib, sequences=2, width=3, pages=8, page=4, total=5, step=True):
    struct = _lib.KvPagesStruct(1 << 12, 1 << 12, 1 << 12, 1 << 12, sequences, width, pages, page)
    args = _lib.KV_STEP.pack(0, 1 << 12, total, *[1 << 12] * 5)
    return lib.iq2_kv_pages_step(ctypes.addressof(struct), args if step else None, None)


def test_pages_refusals_without_a_device(lib):
    assert _pages(lib, step=False) == _lib.IQ2_ERR_INVALID_ARGUMENT
    assert lib.iq2_kv_pages_step(None, _lib.KV_STEP.pack(*[0] * 8), None) == _lib.IQ2_ERR_INVALID_ARGUMENT
    for zero in ("sequences", "width", "pages", "page"):
        assert _pages(lib, **{zero: 0}) == _lib.IQ2_ERR_ZERO_DIM
    assert _pages(lib, sequences=8193) == _lib.IQ2_ERR_UNSUPPORTED and b"8193" in lib.iq2_last_error()
    assert _pages(lib, pages=1 << 20, page=1 << 11) == _lib.IQ2_ERR_OVERFLOW
    assert _pages(lib, total=1 << 31) == _lib.IQ2_ERR_OVERFLOW


def _write(lib, dtype=_lib.KV_INT4, d=64, q=True, norms=None):
    cache = _lib.KvCacheStruct(1 << 12, 1 << 12, 1 << 12, 1 << 12, 4, 2, 16, d, dtype, 1 << 12, 1 << 12)
    args = _lib.KV_TOKENS.pack(1 << 12, 128, 64, 1 << 12, 128, 64, (1 << 12) if q else 0, 256, 64, 0, 3, 4, 1 << 12, 0, 0, 0, 0, 0, 1 << 12, 0)
    return lib.iq2_kv_cache_write_normed(ctypes.addressof(cache), args, norms, None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up pointers: only where there is no device to look them up on")
def test_write_refusals_without_a_device(lib):
    assert _write(lib) == _lib.IQ2_ERR_DEVICE  # all of the rest fits
    assert _write(lib, d=48) == _lib.IQ2_ERR_UNSUPPORTED and b"4-bit" in lib.iq2_last_error()
    assert _write(lib, dtype=5) == _lib.IQ2_ERR_DTYPE


def test_tensor_level_refusals_without_a_device():
    t = torch.zeros((2, 3), dtype=torch.int32)
    with pytest.raises(c.Iq2Error, match="requires a CUDA device"):
        c.KvPages(t, t[0], t[0], t[0, :1], 4)
    with pytest.raises(c.Iq2Error, match="not a multiple of 32"):
        c.KvCache.empty(2, 2, 4, 48, torch.uint8, device="cpu")


def test_reference_rounds_group_scales_as_the_type_does():
    x = torch.cat([ref.E4M3, (ref.E4M3[1:] + ref.E4M3[:-1]) / 2, torch.rand(2000, dtype=torch.float64) * 448])
    assert torch.equal(ref.nearest_e4m3(x).to(torch.uint8), x.float().to(torch.float8_e4m3fn).view(torch.uint8))
    assert torch.equal(ref.E4M3, torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("d", [32, 64, 96, 128])
def test_reference_values_are_within_half_a_step(d):
    """A value is off by half of s g at most, which is m_g / 7 and up to 2^-4 of that more."""
    x = torch.randn((50, d), generator=torch.Generator().manual_seed(d), dtype=torch.float64)
    y = ref.values4(*ref.quantised4(x))
    most = x.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True)
    assert ((x - y).unflatten(-1, (-1, 32)).abs() <= most / 14 * (1 + 2.0 ** -4)).all()
    assert torch.equal(y, y.bfloat16().double())  # eight significant bits
