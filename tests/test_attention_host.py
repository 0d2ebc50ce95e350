"""The attention operators' checks that need no GPU: the argument structs' layout, and the C ABI's refusals in their order
(dimensions and types before the device)."""
import ctypes
import re

import pytest
import torch

import candelora_metal_kernels_b200 as c
from candelora_metal_kernels_b200 import _lib
from candelora_metal_kernels_b200.build import build
from conftest import HEADER, ROOT

_SIZES = {"P": ctypes.c_void_p, "q": ctypes.c_int64, "i": ctypes.c_int, "I": ctypes.c_uint32, "f": ctypes.c_float}


@pytest.fixture(scope="module")
def lib():
    build()
    return _lib.load()


def _fields(name):
    """[(field, C type)] of a struct of the header, iq2_rows spread out."""
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
    out = []
    for decl in (" ".join(d.split()) for d in body.split(";") if d.strip()):
        pointer = "*" in decl
        typ, names = re.match(r"(?:const )?(\w+)(?: \*|\* | )\s*(.*)$", decl).groups()
        for field in names.split(","):
            field = field.strip(" *")
            if typ == "iq2_rows":
                out += [(field + ".data", "P"), (field + ".token_stride", "q"), (field + ".head_stride", "q")]
            else:
                out.append((field, "P" if pointer else {"int": "i", "uint32_t": "I", "int64_t": "q", "float": "f"}[typ]))
    return out


@pytest.mark.parametrize("name,packed", [("iq2_kv_tokens", _lib.KV_TOKENS), ("iq2_attention_prompts", _lib.ATTENTION_PROMPTS),
                                         ("iq2_attention_tokens", _lib.ATTENTION_TOKENS)])
def test_packed_structs_have_the_headers_fields(name, packed):
    fields = [(f.replace(".", "_"), _SIZES[t]) for f, t in _fields(name)]
    struct = type("S", (ctypes.Structure,), {"_fields_": fields})
    assert packed.size == ctypes.sizeof(struct)
    assert re.sub(r"0q$", "", packed.format.strip("@")) == "".join(t for _, t in _fields(name))


def test_cache_struct_matches_the_header():
    kinds = {ctypes.c_void_p: "P", ctypes.c_uint32: "I", ctypes.c_int: "i"}
    assert [(n, kinds[t]) for n, t in _lib.KvCacheStruct._fields_] == _fields("iq2_kv_cache")


def test_rust_structs_have_the_headers_fields():
    ffi = (ROOT / "candelora_metal_kernels_b200" / "rust" / "src" / "iq2_cuda_ffi.rs").read_text()
    kinds = {"u32": "I", "i64": "q", "c_int": "i", "f32": "f"}
    for rust, name in (("Iq2KvCache", "iq2_kv_cache"), ("Iq2KvTokens", "iq2_kv_tokens"), ("Iq2AttentionPrompts", "iq2_attention_prompts"),
                       ("Iq2AttentionTokens", "iq2_attention_tokens")):
        body = re.search(r"pub struct %s \{(.*?)\}" % rust, ffi, re.S).group(1)
        got = []
        for field, typ in re.findall(r"pub (\w+): ([^,]+),", body):
            if typ == "Iq2Rows":
                got += [(field + ".data", "P"), (field + ".token_stride", "q"), (field + ".head_stride", "q")]
            else:
                got.append((field, "P" if typ.startswith("*") else kinds[typ]))
        assert got == _fields(name), rust


def _cache(pages=4, heads=2, page=16, d=64, dtype=2):
    return _lib.KvCacheStruct(1 << 12, 1 << 12, None, None, pages, heads, page, d, dtype)


def _decode(lib, cache, dtype=2, batch=1, q_heads=4, width=1, scale=0.0):
    args = _lib.ATTENTION_TOKENS.pack(1 << 12, 64, 64, dtype, batch, q_heads, width, 1 << 12, 1 << 12, scale, 1 << 12)
    return lib.iq2_attention_decode(ctypes.addressof(cache), args, None, 0, None)


def _prefill(lib, dtype=2, seqs=1, tq=4, tk=4, hq=4, hkv=2, d=64, scale=0.0):
    args = _lib.ATTENTION_PROMPTS.pack(1 << 12, 256, 64, 1 << 12, 128, 64, 1 << 12, 128, 64, dtype, seqs, tq, tk, hq, hkv, d,
                                       1 << 12, 1 << 12, 1, scale, 1 << 12)
    return lib.iq2_attention_prefill(args, None, 0, None)


def test_refusals_without_a_device(lib):
    assert lib.iq2_attention_prefill(None, None, 0, None) == _lib.IQ2_ERR_INVALID_ARGUMENT
    assert _prefill(lib, hq=0) == _lib.IQ2_ERR_ZERO_DIM
    assert _prefill(lib, hq=3) == _lib.IQ2_ERR_UNSUPPORTED and b"not a multiple" in lib.iq2_last_error()
    assert _prefill(lib, d=72) == _lib.IQ2_ERR_UNSUPPORTED and b"head_dim=72" in lib.iq2_last_error()
    assert _prefill(lib, dtype=0) == _lib.IQ2_ERR_DTYPE
    assert _prefill(lib, scale=float("nan")) == _lib.IQ2_ERR_INVALID_ARGUMENT
    assert _prefill(lib, seqs=0) == _lib.IQ2_ERR_ZERO_DIM
    assert _prefill(lib, tq=2 ** 31 - 1, hq=128, hkv=2) == _lib.IQ2_ERR_OVERFLOW
    assert _prefill(lib, tq=0) == _lib.IQ2_OK  # nothing to do
    assert lib.iq2_attention_decode(None, _lib.ATTENTION_TOKENS.pack(*[0] * 9, 0.0, 0), None, 0, None) == _lib.IQ2_ERR_INVALID_ARGUMENT
    assert _decode(lib, _cache(pages=0)) == _lib.IQ2_ERR_ZERO_DIM
    assert _decode(lib, _cache(dtype=7)) == _lib.IQ2_ERR_DTYPE and b"cache dtype" in lib.iq2_last_error()
    assert _decode(lib, _cache(pages=2 ** 31, page=2)) == _lib.IQ2_ERR_OVERFLOW
    assert lib.iq2_kv_cache_write(ctypes.addressof(_cache()), None, None) == _lib.IQ2_ERR_INVALID_ARGUMENT
    assert lib.iq2_kv_cache_read(None, None, 1, 1, None, None, 1, None, None, 2, None) == _lib.IQ2_ERR_INVALID_ARGUMENT


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-device path")
def test_no_device_is_a_device_error(lib):
    assert _prefill(lib) == _lib.IQ2_ERR_DEVICE
    assert _decode(lib, _cache()) == _lib.IQ2_ERR_DEVICE


def test_workspace_queries_need_no_device(lib):
    args = _lib.ATTENTION_PROMPTS.pack(*[0] * 9, 2, 1, 4, 4, 4, 2, 64, 0, 0, 1, 0.0, 0)
    assert lib.iq2_attention_prefill_workspace_size(args) > 0
    assert lib.iq2_attention_prefill_workspace_size(None) == 0
    assert lib.iq2_attention_decode_workspace_size(ctypes.addressof(_cache()), 1, 4) > 0
    assert lib.iq2_attention_decode_workspace_size(ctypes.addressof(_cache()), 0, 4) == 0


def test_tensor_level_refusals_without_a_device():
    k = torch.zeros((2, 2, 16, 64), dtype=torch.float16)
    with pytest.raises(c.Iq2Error, match="requires a CUDA device"):
        c.KvCache(k, k)
    with pytest.raises(c.Iq2Error, match="of one shape"):
        c.KvCache(k, k[:1])
    x = torch.zeros((3, 2, 64), dtype=torch.float16)
    with pytest.raises(c.Iq2Error, match="requires a CUDA device"):
        c.attention_prefill(x, x, x, torch.tensor([0, 3], dtype=torch.int32))
