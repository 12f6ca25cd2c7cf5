"""CPU tests of the attention operators' host side: the relative-position
buckets against the formula in whole numbers, and what the C ABI and the
wrappers refuse before any GPU work."""
import ctypes

import pytest


def _bucket(rel, num, dist, bi):
    """The formula, its comparison made exact: (d / e)^(n - e) >= (dist / e)^t in whole numbers."""
    n = num // 2 if bi else num
    e = n // 2
    first = n if bi and rel > 0 else 0
    d = abs(rel) if bi else max(0, -rel)
    if d < e:
        return first + d
    m = n - e
    return first + e + sum(d ** m >= e ** (m - t) * dist ** t for t in range(1, m))


@pytest.mark.parametrize("num,dist,bi", [(32, 128, True), (32, 128, False), (8, 20, False), (4, 2, True), (2, 2, False),
                                         (128, 500, True), (128, 640, False), (64, 16384, False), (16, 4096, True)])
def test_buckets_are_the_formula(num, dist, bi):
    import whirlwind_trt_plugins_b200 as ww
    rels = list(range(-300, 301)) + [s * (dist + d) for s in (1, -1) for d in (-1, 0, 1)] + [10 ** 6, -10 ** 6]
    for rel in rels:
        assert ww.relative_position_bucket(rel, num, dist, bi) == _bucket(rel, num, dist, bi), rel
    assert max(ww.relative_position_bucket(r, num, dist, bi) for r in rels) <= num - 1


def test_bucket_refusals():
    import whirlwind_trt_plugins_b200 as ww
    for args in ((0, 128, True), (7, 128, True), (32, 8, True), (1, 8, False)):
        with pytest.raises(ww.WWError) as e:
            ww.relative_position_bucket(1, *args)
        assert e.value.status == 2
    with pytest.raises(ww.WWError) as e:
        ww.relative_position_bucket(1, 256, 1024, True)
    assert e.value.status == 5


def _attention(**kw):
    from whirlwind_trt_plugins_b200 import attention
    f = dict(ptrs=[0x1000] * 4 + [0] * 10, bytes=0, strides=[4 * 64 * 8, 4 * 64, 64] * 4,
             sizes=[1, 2, 8, 8, 4, 4, 64, 0, 128, 1, 0], scale=0.125)
    f.update(kw)
    return attention._ATTN.pack(*f["ptrs"], f["bytes"], *f["strides"], *f["sizes"], f["scale"])


def test_attention_arguments():
    import whirlwind_trt_plugins_b200 as ww
    L = ww.lib()

    def status(**kw):
        return L.ww_cross_attention(_attention(**kw), None)

    def sized(**at):
        names = ("dtype", "B", "Lq", "Lk", "Hq", "Hk", "D", "buckets", "distance", "bi", "off")
        base = dict(zip(names, [1, 2, 8, 8, 4, 4, 64, 0, 128, 1, 0]))
        base.update(at)
        return [base[n] for n in names]

    assert L.ww_cross_attention(None, None) == 4
    assert status(sizes=sized(dtype=0)) == 3 and status(sizes=sized(dtype=2)) == 3
    assert status(sizes=sized(B=-1)) == 2 and status(sizes=sized(Hk=3)) == 2 and status(sizes=sized(Hk=0)) == 2
    assert status(sizes=sized(D=60)) == 5 and status(sizes=sized(D=136)) == 5
    assert status(scale=float("nan")) == 2
    for n in range(4):
        ptrs = [0x1000] * 4 + [0] * 10
        ptrs[n] = 0
        assert status(ptrs=ptrs) == 4
        ptrs[n] = 0x1008
        assert status(ptrs=ptrs) == 6
    assert status(strides=[4 * 64 * 8, 4 * 64, 60] * 4) == 6
    assert status(strides=[4 * 64 * 8, -64, 64] * 4) == 6
    table = [0x1000] * 4 + [0, 0, 0, 0x1000] + [0] * 6
    assert status(ptrs=table, sizes=sized(buckets=9)) == 2
    assert status(ptrs=table, sizes=sized(buckets=32, distance=8)) == 2
    assert status(ptrs=table, sizes=sized(buckets=130)) == 5
    # nothing to do: success without a device
    assert status(sizes=sized(B=0)) == 0 and status(sizes=sized(Lq=0)) == 0
    # the gradient needs lse, dout, its outputs and its workspace
    assert L.ww_cross_attention_backward(_attention(), None) == 4
    full = [0x1000] * 5 + [0, 0, 0] + [0x1000] * 4 + [0, 0]
    assert L.ww_cross_attention_backward(_attention(ptrs=full), None) == 4
    full[13] = 0x1000
    assert L.ww_cross_attention_backward(_attention(ptrs=full), None) == 5
    assert L.ww_cross_attention_backward_workspace(_attention(ptrs=full)) > 0


def test_norm_rope_arguments():
    import whirlwind_trt_plugins_b200 as ww
    from whirlwind_trt_plugins_b200 import attention
    L = ww.lib()
    names = ("qs", "ks", "dtype", "B", "Lq", "Lk", "Hq", "Hk", "D", "R", "P", "inter")

    def status(fn=L.ww_qk_norm_rope, ptrs=None, strides=None, eps=1e-6, **at):
        base = dict(zip(names, [0, 0, 1, 2, 8, 8, 4, 4, 64, 64, 8, 0]))
        base.update(at)
        return fn(attention._ROPE.pack(*(ptrs or [0x1000] * 6 + [0, 0, 0x1000, 0x1000] + [0] * 7), 0,
                                       *(strides or [4 * 64 * 8, 4 * 64, 64] * 4), *[base[n] for n in names], eps),
                  None)

    assert L.ww_qk_norm_rope(None, None) == 4
    assert status(dtype=2) == 3 and status(B=-1) == 2 and status(R=66) == 2 and status(R=7) == 2
    assert status(D=60, R=0) == 5 and status(R=12) == 5 and status(D=264) == 5
    assert status(P=0) == 2 and status(eps=-1.0) == 2 and status(eps=float("nan")) == 2
    for n in (0, 1, 2, 3, 4, 5, 8, 9):
        ptrs = [0x1000] * 6 + [0, 0, 0x1000, 0x1000] + [0] * 7
        ptrs[n] = 0
        assert status(ptrs=ptrs) == 4
    assert status(strides=[4 * 64 * 8, 4 * 64, 60] * 4) == 6
    assert status(B=0) == 0 and status(Lq=0, Lk=0) == 0
    assert status(fn=L.ww_qk_norm_rope_backward) == 4


def test_structs_match_the_header(tmp_path):
    """The wrappers pack the parameter structs by hand: sizes and the last fields' places from the header."""
    import shutil
    import subprocess

    from conftest import ROOT
    from whirlwind_trt_plugins_b200 import attention
    if shutil.which("gcc") is None:
        pytest.skip("needs gcc")
    src = tmp_path / "s.c"
    src.write_text('#include "ww_trt_plugins.h"\n#include <stdio.h>\nint main(void) { printf("%zu %zu %zu %zu", '
                   "sizeof(ww_attention_t), offsetof(ww_attention_t, scale), sizeof(ww_qk_norm_rope_t), "
                   "offsetof(ww_qk_norm_rope_t, eps)); return 0; }\n")
    exe = tmp_path / "s"
    subprocess.run(["gcc", f"-I{ROOT}/include", str(src), "-o", str(exe)], check=True)
    a, s, r, e = map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split())
    assert (attention._ATTN.size, attention._ROPE.size) == (a, r)
    assert s == 14 * 8 + 8 + 12 * 8 + 11 * 4 and e == 17 * 8 + 8 + 12 * 8 + 12 * 4
    assert ctypes.sizeof(ctypes.c_void_p) == 8


def test_wrappers_refuse_host_tensors():
    import torch
    import whirlwind_trt_plugins_b200 as ww
    x = torch.zeros((1, 2, 2, 32), dtype=torch.float16)
    with pytest.raises(TypeError):
        ww.cross_attention(x, x, x)
    with pytest.raises(TypeError):
        ww.qk_norm_rope(x, x, x[0, 0, 0], x[0, 0, 0], torch.zeros(2, 16), torch.zeros(2, 16))


def test_plugins_shapes_formats_fields():
    from whirlwind_trt_plugins_b200 import plugins as pl
    T = pl.TensorDesc
    cr = pl.get_plugin_creator("CrossAttention", "1")
    p = cr.create_plugin({"use_lens": 1, "use_bias": 1, "q_offset": 3})
    assert p.clone().get_fields_to_serialize() == {"use_lens": 1, "use_mask": 0, "use_bias": 1, "max_distance": 128,
                                                   "bidirectional": 1, "q_offset": 3}
    q, k, lens, table = T((2, 5, 8, 64)), T((2, 7, 4, 64)), T((2,), 3), T((8, 32))
    assert p.get_output_shapes([q, k, k, lens, table]) == [(2, 5, 8, 64)]
    for bad in ([q, k, k, lens], [q, k, T((2, 6, 4, 64)), lens, table], [q, T((2, 7, 3, 64))] + [T((2, 7, 3, 64)), lens, table],
                [q, k, k, T((3,), 3), table], [q, k, k, lens, T((4, 32))]):
        with pytest.raises(ValueError):
            p.get_output_shapes(bad)
    io = [q, k, k, lens, table, q]
    assert all(p.supports_format_combination(i, io, 5, 1) for i in range(6))
    assert not p.supports_format_combination(3, [q, k, k, T((2,), 1), table, q], 5, 1)
    assert not p.supports_format_combination(0, [T((2, 5, 8, 64), 0)] + io[1:], 5, 1)
    m = cr.create_plugin({"use_mask": 1})
    assert m.supports_format_combination(3, [q, k, k, T((2, 7), 4), q], 4, 1)
    assert m.get_workspace_size() == 64 << 20 and m.get_nb_outputs() == 1
    # refused before any GPU work
    assert p.enqueue([q, k, k, lens, T((4, 32))], [0] * 5, [0], stream=0) == 1
    assert p.enqueue([q, k, k, lens, table], [0] * 5, [0], stream=0) == 1

    cr = pl.get_plugin_creator("QkNormRope", "1")
    r = cr.create_plugin({"use_positions": 1})
    assert r.get_nb_outputs() == 2 and r.get_output_data_types([7] * 8) == [7, 7]
    w, c = T((64,)), T((100, 16), 0)
    ins = [q, k, w, w, c, c, T((5,), 3), T((2, 7), 3)]
    assert r.get_output_shapes(ins) == [(2, 5, 8, 64), (2, 7, 4, 64)]
    assert all(r.supports_format_combination(i, ins + [q, k], 8, 2) for i in range(10))
    assert not r.supports_format_combination(4, [q, k, w, w, T((100, 16), 1)] + ins[5:] + [q, k], 8, 2)
    with pytest.raises(ValueError):
        r.get_output_shapes(ins[:6])
    with pytest.raises(ValueError):
        r.get_output_shapes(ins[:6] + [T((6,), 3), T((2, 7), 3)])
    assert r.enqueue(ins, [0] * 8, [0, 0], stream=0) == 1
