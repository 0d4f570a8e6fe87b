"""Calls of the operators over the paged cache and of the 4-bit products that were once taken, refused before anything is launched."""
import pytest

from flexllm_b200 import _lib

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops():
    from flexllm_b200 import build, ops
    build.build()
    return ops


class OnDevice:
    """What the checks look at of a dense tensor on a device that this machine need not have."""

    is_cuda = True

    def __init__(self, shape, dtype, device=0):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, torch.device("cuda", device)

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def stride(self, i=None):
        s = [self.shape[d + 1:].numel() for d in range(len(self.shape))]
        return s if i is None else s[i]

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 1 << 20


@pytest.fixture
def called(ops, monkeypatch):
    """The arguments of calls that pass the checks."""
    seen = []
    monkeypatch.setattr(ops, "_front", False)
    monkeypatch.setattr(ops, "_bind_front_end", lambda: False)
    monkeypatch.setattr(ops, "_call_on", lambda device, name, *args: seen.append((name, args)))
    return seen


def test_four_bit_products_want_their_output_on_their_inputs_device(ops, called):
    BF, F32, U8 = torch.bfloat16, torch.float32, torch.uint8
    x, w, s = OnDevice((2, 64), BF), OnDevice((8, 32), U8), OnDevice((8, 2), BF)
    y = OnDevice((2, 8), BF)
    assert ops.linear_w4(x, w, s, out=y) is y and len(called) == 1
    assert ops.linear_w4(x, w, s, out_f32=True, out=OnDevice((2, 8), F32)).dtype is F32 and len(called) == 2
    for out_f32, dtype in ((False, BF), (True, F32)):
        with pytest.raises(ValueError):
            ops.linear_w4(x, w, s, out_f32=out_f32, out=OnDevice((2, 8), dtype, 1))
    assert len(called) == 2


def test_sections_of_one_axis_have_to_add_up():
    import test_paged_cpu as c
    from flexllm_b200 import build
    build.build()
    lib = _lib.load()
    assert c.rope(lib, sec=[32]) == _lib.OK and c.rope(lib) == _lib.OK
    for bad in (31, 33, 0, -32):
        assert c.rope(lib, sec=[bad]) == _lib.EINVAL
