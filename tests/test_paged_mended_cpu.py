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


def test_positions_and_sections_of_more_than_32_bits(ops, called):
    """ctypes passes the low 32 bits on; sections of one axis were not looked at."""
    I32, F32 = torch.int32, torch.float32
    k, v, q = OnDevice((2, 2, 64, 64), F32), OnDevice((2, 2, 64, 64), F32), OnDevice((3, 4, 64), F32)
    table, cu, ctx, mask = OnDevice((1, 2), I32), OnDevice((2,), I32), OnDevice((1,), I32), OnDevice((3,), torch.int64)
    keep, count, out = OnDevice((1, 4), I32), OnDevice((1,), I32), OnDevice((3, 256), F32)
    proj, pos, cos = OnDevice((3, 512), F32), OnDevice((3,), I32), OnDevice((9, 32), F32)
    rope = lambda **a: ops.qk_norm_rope(proj, 4, pos, cos, cos, k, v, table, cu, ctx, out=out, **a)
    ops.attn_packed(q, k, v, table, cu, ctx, max_ctx=127, out=out), ops.kv_keep([(k, v)], table, ctx, keep, count, max_ctx=127), rope(max_ctx=127, sections=[32])
    assert len(called) == 3
    for wide in ((1 << 32) + 127, 1 << 31, -(1 << 32) + 100):
        for call in (lambda: ops.attn_packed(q, k, v, table, cu, ctx, max_ctx=wide, out=out), lambda: ops.attn_tree(q, mask, k, v, table, cu, ctx, max_ctx=wide, out=out),
                     lambda: ops.kv_keep([(k, v)], table, ctx, keep, count, max_ctx=wide), lambda: rope(max_ctx=wide)):
            with pytest.raises(ValueError):
                call()
    for sections in ([16, 16], [], [(1 << 32) + 32], [-1], [33]):
        with pytest.raises(ValueError):
            rope(sections=sections)
    assert len(called) == 3


def test_sections_of_one_axis_have_to_add_up():
    import test_paged_cpu as c
    from flexllm_b200 import build
    build.build()
    lib = _lib.load()
    assert c.rope(lib, sec=[32]) == _lib.OK and c.rope(lib) == _lib.OK
    for bad in (31, 33, 0, -32):
        assert c.rope(lib, sec=[bad]) == _lib.EINVAL


def test_four_bit_products_count_rows_in_31_bits():
    """The row numbers behind the last tile of 2^31 - 1 rows would wrap and be read."""
    from flexllm_b200 import build
    build.build()
    lib, P = _lib.load(), 1 << 20
    call = lambda M, N: lib.flexllm_linear_w4(_lib.BF16, P, 32, P, P, _lib.BF16, None, 32, None, M, N, 32, P, N, 0, None)
    assert call(0, 1 << 30) == _lib.OK
    for M, N in ((0, (1 << 30) + 1), (0, (1 << 31) - 1), (0, (1 << 31) - 500)):
        assert call(M, N) == _lib.ENOTSUP
