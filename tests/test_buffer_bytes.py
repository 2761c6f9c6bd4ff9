"""A buffer of narrower elements than the kernels' is refused by its bytes, before the launch."""
import numpy as np
import pytest

from aurora_amd.gpu import GemmKernel, GpuBuffer, PagedBatch, SampleKernel

PTR = 0x10000  # an address that nothing here reads


class Nothing:
    def call(self, *args):
        raise AssertionError(args)


def _sample(**other):
    x = dict(logits=GpuBuffer(None, PTR, 20), u=GpuBuffer(None, PTR, 2), tokens=GpuBuffer(None, PTR, 2, np.int32),
             logprob=GpuBuffer(None, PTR, 2), top_k=GpuBuffer(None, PTR, 2, np.int32))
    x.update(other)
    SampleKernel().dispatch_into(Nothing(), x["logits"], 10, x["u"], x["tokens"], x["logprob"], 2, 10, 0, x["top_k"])


@pytest.mark.parametrize("name", ["logits", "u", "tokens", "logprob", "top_k"])
@pytest.mark.parametrize("dtype", [np.uint8, np.float16])
def test_choice(name, dtype):
    n = 20 if name == "logits" else 2
    with pytest.raises(ValueError, match=f"{n} of 4 needed"):
        _sample(**{name: GpuBuffer(None, PTR, n, dtype)})
    with pytest.raises(AssertionError, match="aur_sample"):  # bytes enough: the call is made
        _sample(**{name: GpuBuffer(None, PTR, 4 * n, dtype)})


def test_others():
    f32, f16 = (lambda n: GpuBuffer(None, PTR, n)), (lambda n: GpuBuffer(None, PTR, n, np.float16))
    with pytest.raises(ValueError, match="GemmKernel c"):
        GemmKernel().dispatch_into(Nothing(), f32(16), f32(16), f16(16), 4, 4, 4)
    with pytest.raises(ValueError, match="PagedBatch own_len"):
        PagedBatch(PTR, GpuBuffer(None, PTR, 4, np.int16), PTR, 4, 2, 4, 1, 32)
