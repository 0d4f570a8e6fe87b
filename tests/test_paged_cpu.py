"""What the operators over packed sequences and the 4-bit products refuse, and what they take without a GPU (nothing is launched)."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest

from flexllm_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, EINVAL, ENOTSUP = _lib.OK, _lib.EINVAL, _lib.ENOTSUP
P = C.c_void_p(1 << 20)                          # aligned, and never followed


@pytest.fixture(scope="module")
def lib():
    from flexllm_b200 import build
    build.build()
    return _lib.load()


def pages(k=1 << 20, v=1 << 21, n_pages=8, hkv=2, kdim=64, vdim=64):
    return _lib.KvPages(k, v, n_pages, hkv, kdim, vdim)


def attention(lib, mask=None, **change):
    a = dict(dtype=_lib.BF16, kv=pages(), heads=4, scale=0.125, q=P, ldq=256, cu=P, ctx=P, table=P, max_pages=4, max_ctx=255, B=2, T=0, out=P, ldo=256)
    a.update(change)
    head = [a["dtype"], C.byref(a["kv"]) if a["kv"] is not None else None, a["heads"], a["scale"], a["q"], a["ldq"]]
    tail = [a["cu"], a["ctx"], a["table"], a["max_pages"], a["max_ctx"], a["B"], a["T"], a["out"], a["ldo"], None]
    if mask is None:
        return lib.flexllm_attn_packed(*head, *tail)
    return lib.flexllm_attn_tree(*head, mask, *tail)


BAD_ATTENTION = [dict(dtype=2), dict(kv=None), dict(kv=pages(k=0)), dict(kv=pages(hkv=0)), dict(kv=pages(hkv=3)), dict(heads=0), dict(heads=5), dict(scale=-0.1),
                 dict(scale=float("nan")), dict(scale=float("inf")), dict(cu=None), dict(ctx=None), dict(table=None), dict(max_pages=0), dict(max_ctx=256), dict(max_ctx=-1),
                 dict(B=0), dict(T=-1), dict(ldq=255), dict(ldq=260), dict(ldo=255), dict(T=3, q=None), dict(T=3, out=None), dict(T=3, q=C.c_void_p((1 << 20) + 8)),
                 dict(T=3, kv=pages(k=(1 << 20) + 8)), dict(T=3, out=C.c_void_p((1 << 20) + 1)), dict(dtype=_lib.F32, ldq=258), dict(kv=pages(n_pages=0)), dict(max_pages=1 << 25, max_ctx=1 << 30),
                 dict(cu=C.c_void_p(6)), dict(ctx=C.c_void_p(6)), dict(table=C.c_void_p(6)), dict(heads=1 << 17, ldq=1 << 23, ldo=1 << 23)]


@pytest.mark.parametrize("change", BAD_ATTENTION, ids=lambda c: ",".join(c))
def test_attention_refuses(lib, change):
    assert attention(lib, **change) == EINVAL
    assert attention(lib, mask=P, **change) == EINVAL


def test_attention_sizes(lib):
    assert attention(lib) == OK and attention(lib, mask=P) == OK                       # no rows: nothing to do
    assert attention(lib, T=3, mask=C.c_void_p(12)) == EINVAL                          # masks are 64-bit words
    assert lib.flexllm_attn_tree(_lib.BF16, C.byref(pages()), 4, 0.125, P, 256, None, P, P, P, 4, 255, 2, 3, P, 256, None) == EINVAL
    for kdim, vdim in ((60, 64), (64, 60), (264, 64), (64, 264)):
        assert attention(lib, kv=pages(kdim=kdim, vdim=vdim), ldq=4096, ldo=4096) == ENOTSUP
    assert attention(lib, T=3, kv=pages(n_pages=1 << 26)) == ENOTSUP                   # rows of pages beyond 31 bits


def rope(lib, **change):
    a = dict(dtype=_lib.BF16, kv=pages(), heads=4, proj=P, ldp=512, qg=P, kg=P, eps=1e-6, pos=P, axes=1, sec=None, cos=P, sin=P, rot=64, table_len=100, cu=P, ctx=P,
             table=P, max_pages=4, max_ctx=255, B=2, T=0, q=P, ldq=256)
    a.update(change)
    sec = None if a["sec"] is None else (C.c_int * len(a["sec"]))(*a["sec"])
    return lib.flexllm_qk_norm_rope(a["dtype"], C.byref(a["kv"]), a["heads"], a["proj"], a["ldp"], a["qg"], a["kg"], a["eps"], a["pos"], a["axes"], sec, a["cos"], a["sin"],
                                    a["rot"], a["table_len"], a["cu"], a["ctx"], a["table"], a["max_pages"], a["max_ctx"], a["B"], a["T"], a["q"], a["ldq"], None)


def test_norm_rotation_refuses(lib):
    assert rope(lib) == OK and rope(lib, axes=3, sec=[8, 12, 12]) == OK and rope(lib, rot=0, cos=None, sin=None) == OK
    for change in (dict(dtype=3), dict(kv=pages(v=0)), dict(heads=0), dict(ldp=511), dict(ldp=516), dict(ldq=248), dict(eps=-1.0), dict(axes=0), dict(axes=5, sec=[8] * 5),
                   dict(axes=3), dict(axes=3, sec=[8, 12, 11]), dict(axes=2, sec=[40, -8]), dict(cos=None), dict(sin=None), dict(table_len=0), dict(rot=72), dict(rot=-8),
                   dict(cu=None), dict(max_ctx=256), dict(B=0), dict(T=-1), dict(T=2, proj=None), dict(T=2, q=None), dict(T=2, pos=None),
                   dict(T=2, qg=C.c_void_p(8)), dict(T=2, proj=C.c_void_p((1 << 20) + 4))):
        assert rope(lib, **change) == EINVAL, change
    assert rope(lib, rot=36) == ENOTSUP and rope(lib, kv=pages(kdim=60), ldp=4096, ldq=4096, rot=8) == ENOTSUP


def test_accepted_paths_refuse(lib):
    layers = (_lib.KvPages * 2)(pages(), pages(hkv=1))
    call = lambda dtype=_lib.BF16, kv=layers, n=2, table=P, max_pages=4, ctx=P, max_ctx=255, keep=P, count=P, most=0, B=3: lib.flexllm_kv_keep(
        dtype, kv, n, table, max_pages, ctx, max_ctx, keep, count, most, B, None)
    assert call() == OK
    for change in (dict(dtype=5), dict(kv=None), dict(n=0), dict(table=None), dict(ctx=None), dict(max_pages=0), dict(max_ctx=256), dict(most=-1), dict(B=0),
                   dict(most=2, keep=None), dict(most=2, count=None), dict(kv=(_lib.KvPages * 2)(pages(), pages(k=8)))):
        assert call(**change) == EINVAL, change
    assert call(max_pages=1 << 25, max_ctx=(1 << 30)) == EINVAL and call(most=2, keep=C.c_void_p(6)) == EINVAL
    assert call(most=65) == ENOTSUP and call(kv=(_lib.KvPages * 2)(pages(), pages(vdim=4))) == ENOTSUP


def test_four_bit_products_refuse(lib):
    call = lambda dtype=_lib.BF16, a=P, lda=128, w=P, scale=P, st=_lib.BF16, zero=None, group=64, M=0, N=8, K=128, y=P, ldy=8: lib.flexllm_linear_w4(
        dtype, a, lda, w, scale, st, zero, group, None, M, N, K, y, ldy, 0, None)
    assert call() == OK
    for change in (dict(dtype=2), dict(st=3), dict(group=0), dict(group=48), dict(group=96), dict(lda=120), dict(lda=132), dict(M=-1), dict(N=0), dict(K=0), dict(ldy=7),
                   dict(M=1, a=None), dict(M=1, w=None), dict(M=1, scale=None), dict(M=1, y=None), dict(M=1, w=C.c_void_p(24)), dict(M=1, a=C.c_void_p(8)),
                   dict(M=1, scale=C.c_void_p(17)), dict(M=1, y=C.c_void_p(17)), dict(M=1, st=_lib.F32, scale=C.c_void_p(18))):
        assert call(**change) == EINVAL, change
    assert call(K=1 << 21, lda=1 << 21) == ENOTSUP and call(M=64 * 65536, N=8) == ENOTSUP


def test_pages_of_a_cache(lib):
    out = _lib.KvPages()
    assert lib.flexllm_kv_cache_pages(None, 0, C.byref(out)) == EINVAL


def test_python_refusals():
    """Wrong types, shapes and devices raise before anything is called."""
    torch = pytest.importorskip("torch")
    from flexllm_b200 import build, ops
    build.build()
    q, k, v = torch.zeros(3, 4, 64), torch.zeros(2, 2, 64, 64), torch.zeros(2, 2, 64, 64)
    i = lambda *n: torch.zeros(n, dtype=torch.int32)
    for call in (lambda: ops.attn_packed(q, k, v, i(1, 2), i(2), i(1)), lambda: ops.attn_tree(q, torch.zeros(3, dtype=torch.int64), k, v, i(1, 2), i(2), i(1)),
                 lambda: ops.attn_tree(q, None, k, v, i(1, 2), i(2), i(1)), lambda: ops.linear_w4(torch.zeros(1, 64), torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2)),
                 lambda: ops.qk_norm_rope(torch.zeros(3, 512), 4, i(3), torch.zeros(9, 32), torch.zeros(9, 32), k, v, i(1, 2), i(2), i(1)),
                 lambda: ops.kv_keep([(k, v)], i(1, 2), i(1), i(1, 4), i(1)), lambda: ops.kv_keep([], i(1, 2), i(1), i(1, 4), i(1))):
        with pytest.raises(ValueError):
            call()


SRC = r'''
#include <flexllm/flexllm.hpp>
int main() {
    using namespace flexllm;
    FloatKVCache cache;
    flexllm_kv_pages p = {};
    PackedSequences s = {};
    if (cache.pages(0, &p) != FLEXLLM_EINVAL) return 1;
    if (qk_norm_rope(FLEXLLM_BF16, p, 4, nullptr, 0, nullptr, nullptr, 0.0f, nullptr, 1, nullptr, nullptr, nullptr, 0, 0, s, nullptr, 0) != FLEXLLM_EINVAL) return 2;
    if (attn_packed(FLEXLLM_BF16, p, 4, 1.0f, nullptr, 0, s, nullptr, 0) != FLEXLLM_EINVAL) return 3;
    if (attn_tree(FLEXLLM_F32, p, 4, 1.0f, nullptr, 0, nullptr, s, nullptr, 0) != FLEXLLM_EINVAL) return 4;
    if (kv_keep(FLEXLLM_BF16, &p, 1, s, nullptr, nullptr, 4) != FLEXLLM_EINVAL) return 5;
    if (linear_w4(FLEXLLM_BF16, nullptr, 64, nullptr, nullptr, FLEXLLM_BF16, nullptr, 64, nullptr, 1, 8, 64, nullptr, 8) != FLEXLLM_EINVAL) return 6;
    return 0;
}
'''


def test_cpp_wrappers():
    from flexllm_b200 import build
    lib = build.build()
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "t.cpp"), os.path.join(d, "t")
        open(src, "w").write(SRC)
        r = subprocess.run(["/usr/bin/g++", "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "include"), src, "-o", exe, lib, "-Wl,-rpath," + os.path.dirname(lib)],
                           capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
        assert subprocess.run([exe]).returncode == 0
