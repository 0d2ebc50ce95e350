"""Which GPU the attention operators' host side asks: the tensors' own, whichever is the current one. On the CPU, with two
devices made up."""
import contextlib
import types

import pytest
import torch

import candelora_metal_kernels_b200 as c
from candelora_metal_kernels_b200 import _lib


class Tensor:
    """What the host side looks at of a contiguous tensor on cuda:1."""

    is_cuda = True

    def __init__(self, shape, dtype):
        self.shape, self.dtype = tuple(shape), dtype

    def dim(self):
        return len(self.shape)

    def stride(self):
        return tuple(int(torch.tensor(self.shape[i + 1:]).prod()) for i in range(len(self.shape)))

    def numel(self):
        return int(torch.tensor(self.shape).prod())

    def get_device(self):
        return 1

    def data_ptr(self):
        return 1 << 12

    def is_contiguous(self):
        return True

    def new_empty(self, shape, dtype):
        return Tensor((shape,) if isinstance(shape, int) else shape, dtype)


@pytest.mark.parametrize("current", [0, 1])
def test_prefill_asks_the_tensors_device(monkeypatch, current):
    state, asked = {"device": current}, []

    @contextlib.contextmanager
    def device(index):
        before, state["device"] = state["device"], index
        yield
        state["device"] = before

    def query(args):
        asked.append(("workspace", state["device"]))
        return 64

    def run(*args):
        asked.append(("call", state["device"]))
        return _lib.IQ2_OK

    fake = types.SimpleNamespace(iq2_attention_prefill_workspace_size=query, iq2_attention_prefill=run)
    monkeypatch.setattr(_lib, "load", lambda: fake)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: state["device"], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    q, kv = Tensor((3, 4, 64), torch.bfloat16), Tensor((3, 2, 64), torch.bfloat16)
    c.attention_prefill(q, kv, kv, Tensor((2,), torch.int32), out=Tensor((3, 4, 64), torch.bfloat16))
    assert asked == [("workspace", 1), ("call", 1)] and state["device"] == current
