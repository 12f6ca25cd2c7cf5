"""CPU tests of the 8-bit layer operators' host side at its edges."""
import subprocess
import sys

import pytest
from conftest import ROOT

# Arrays of exactly the inputs' descriptors, right before a page that cannot be read.
GUARDED = """
import ctypes, mmap, sys
from whirlwind_trt_plugins_b200 import plugins as pl
T = pl.TensorDesc
libc = ctypes.CDLL(None, use_errno=True)
libc.mmap.restype = ctypes.c_void_p
libc.mmap.argtypes = [ctypes.c_void_p, ctypes.c_size_t] + [ctypes.c_int] * 3 + [ctypes.c_long]
libc.mprotect.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int]
page, anonymous = mmap.PAGESIZE, mmap.MAP_PRIVATE | mmap.MAP_ANONYMOUS
plain = pl._descs
def guarded(descs):
    a = plain(descs)
    n = ctypes.sizeof(a)
    pages = (n + page - 1) // page
    at = libc.mmap(None, (pages + 1) * page, mmap.PROT_READ | mmap.PROT_WRITE, anonymous, -1, 0)
    assert at not in (None, ctypes.c_void_p(-1).value) and libc.mprotect(at + pages * page, page, 0) == 0
    ctypes.memmove(at + pages * page - n, a, n)
    return type(a).from_address(at + pages * page - n)
pl._descs = guarded
I8, F, I32, B = pl.DTYPE_INT8, pl.DTYPE_FLOAT, 3, 4
q, kv, s = T((2, 1, 6, 32)), T((2, 7, 3, 32), I8), T((2, 3, 7), F)
for lens in (0, 1):
    for mask in (0, 1):
        for bias in (0, 1):
            ins = [q, kv, kv, s, s] + [T((2,), I32)] * lens + [T((2, 7), B)] * mask + [T((6, 16))] * bias
            p = pl.CrossAttentionInt8Plugin(lens, mask, bias)
            assert p.get_workspace_size(ins) > 0 and p.get_output_shapes(ins) == [q.dims]
            assert all(p.supports_format_combination(i, ins, len(ins), 1) for i in range(len(ins)))
            assert p.supports_format_combination(len(ins), ins + [q], len(ins), 1)
            assert p.enqueue(ins, [0] * len(ins), [0], stream=0) == 1
x, w = T((4, 64)), T((64,))
assert pl.LayerNormPlugin(1).enqueue([x, w, w, x], [0] * 4, [0] * 2, stream=0) == 1
lin = [x, T((33, 64), I8), T((33,), F), T((33,))]
assert pl.Int8LinearPlugin(1).get_workspace_size(lin) >= 0 and pl.Int8LinearPlugin(1).enqueue(lin, [0] * 4, [0], stream=0) == 1
k = T((2, 7, 3, 32))
assert pl.QuantizeKvPlugin().enqueue([k, k], [0] * 2, [0] * 4, stream=0) == 1
print("done")
"""


def test_plugins_read_the_inputs_descriptors_only():
    if not sys.platform.startswith("linux"):
        pytest.skip("mmap")
    r = subprocess.run([sys.executable, "-c", GUARDED], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "done", (r.returncode, r.stderr[-500:])


def test_linear_plugin_workspace_holds_for_smaller_sizes():
    """What the plugin asks for its largest sizes is enough for every smaller one, whichever form that takes."""
    from whirlwind_trt_plugins_b200 import layers, plugins as pl
    T = pl.TensorDesc

    def needed(M, K, N):
        return layers._lib.ww_int8_matmul_workspace(layers._MATMUL.pack(16, 0, 0, 16, 16, 0, 16, 0, 0, K, K, K, pl.DTYPE_HALF, M, K, N))

    assert needed(4, 4096, 9473) == 0 and needed(4, 4096, 9472) > 0
    for M, K, N in ((4, 4096, 9473), (8, 2048, 9473), (1, 4096, 64), (1, 20000, 64), (300, 64, 33)):
        have = pl.Int8LinearPlugin().get_workspace_size([T((M, K)), T((N, K), pl.DTYPE_INT8), T((N,), pl.DTYPE_FLOAT)])
        for m in {1, 2, M // 2 or 1, max(1, M - 1), M}:
            for k in {16, K // 32 * 16, K}:
                for n in {1, N // 2, N - 1, N}:
                    assert m > M or needed(m, k, n) <= have, (m, k, n)


def test_attention_copies_of_the_least_memory():
    """Many rows take the copies' bytes alone, as the header says; the size asked for holds the heads' powers in fp16 as well."""
    import test_layers as t
    import torch
    layers, L = t._layers()
    copies, powers = 2 * 2 * 8 * 4 * 64 * 2, 256
    assert L.ww_cross_attention_int8_workspace(t._attention(Lq=129)) >= copies + powers

    def status(have):
        from whirlwind_trt_plugins_b200.attention import _ATTN
        a = _ATTN.pack(*[0x1000] * 4, *[0] * 9, 0x10000, have, *[4 * 64 * 8, 4 * 64, 64] * 4, 1, 2, 129, 8, 4, 4, 64, 0, 128, 1, 0, 0.125)
        return L.ww_cross_attention_int8(a + layers._SCALES.pack(0x1000, 0x1000, 32, 8, 32, 8), None)

    assert status(copies - 1) == t.LIMIT
    if not torch.cuda.is_available():  # past the checks a call asks for its device (the addresses are none: only where there is none)
        assert status(copies) not in (t.OK, t.LIMIT)
