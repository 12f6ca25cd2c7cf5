"""CPU tests of the 8-bit layer operators' host side: what the C ABI and the
wrappers refuse before any GPU work."""
import pytest

OK, SHAPE, DTYPE, NULL, LIMIT, ALIGN = 0, 2, 3, 4, 5, 6


def _layers():
    from whirlwind_trt_plugins_b200 import layers
    return layers, layers._lib


def _pack(struct, names, base, changes):
    assert set(changes) <= set(names), changes
    return struct.pack(*[{**base, **changes}[n] for n in names])


NORM = ("x residual weight bias y sum y_q y_scale mean rstd dy dsum dx dweight dbias workspace workspace_bytes "
        "x_stride residual_stride y_q_stride dy_stride dsum_stride dtype rows N eps").split()


def _norm(**kw):
    base = {**dict.fromkeys(NORM, 0), "x": 0x1000, "y": 0x2000, "x_stride": 64, "dtype": 1, "rows": 4, "N": 64, "eps": 1e-5}
    return _pack(_layers()[0]._NORM, NORM, base, kw)


def test_layer_norm_arguments():
    _, L = _layers()
    status = lambda **kw: L.ww_layer_norm(_norm(**kw), None)  # noqa: E731
    assert L.ww_layer_norm(None, None) == NULL
    assert status(dtype=2) == DTYPE and status(rows=-1) == SHAPE and status(N=0) == SHAPE and status(N=1 << 25) == LIMIT
    assert status(eps=-1.0) == SHAPE and status(eps=float("nan")) == SHAPE and status(x_stride=-64) == SHAPE
    assert status(x=0) == NULL and status(y=0) == NULL and status(bias=0x1000) == NULL and status(sum=0x1000) == NULL
    assert status(y_q=0x3000, y_q_stride=64) == NULL  # both results
    assert status(y=0, y_q=0x3000, y_q_stride=64) == NULL and status(y=0, y_q=0x3000, y_scale=0x4000, y_q_stride=63) == SHAPE
    assert status(x=0x1001) == ALIGN and status(x=0x1002, dtype=0) == ALIGN and status(mean=0x1002) == ALIGN
    assert status(rows=0, x=0, y=0) == OK  # nothing to do: success without a device
    quant = lambda **kw: L.ww_quantize_tokens(_norm(**{**dict(y=0, y_q=0x3000, y_scale=0x4000, y_q_stride=64), **kw}), None)  # noqa: E731
    assert L.ww_quantize_tokens(None, None) == NULL
    assert quant(y=0x2000, y_q=0) == NULL and quant(weight=0x1000) == NULL and quant(residual=0x1000) == NULL
    assert quant(rows=0, x=0) == OK


def test_layer_norm_backward_arguments():
    _, L = _layers()
    full = dict(y=0, mean=0x5000, rstd=0x6000, dy=0x7000, dx=0x8000, dy_stride=64)
    status = lambda **kw: L.ww_layer_norm_backward(_norm(**{**full, **kw}), None)  # noqa: E731
    assert L.ww_layer_norm_backward(None, None) == NULL and L.ww_layer_norm_backward_workspace(None) == 0
    for name in ("mean", "rstd", "dy", "dx"):
        assert status(**{name: 0}) == NULL
    assert status(dweight=0x9000) == NULL and status(dbias=0x9000) == NULL  # both or neither
    assert status(dy_stride=-1) == SHAPE and status(dx=0x8001) == ALIGN and status(dtype=9) == DTYPE
    assert status(rows=0, x=0, mean=0, rstd=0, dy=0, dx=0) == OK
    both = dict(dweight=0x9000, dbias=0xa000)
    need = L.ww_layer_norm_backward_workspace(_norm(**full, **both))
    assert need >= 2 * 64 * 4 and L.ww_layer_norm_backward_workspace(_norm(**full)) == 0


MATMUL = "x x_q x_scale w_q w_scale bias out workspace workspace_bytes x_stride x_q_stride w_stride dtype M K N".split()


def _matmul(**kw):
    base = {**dict.fromkeys(MATMUL, 0), "x_q": 0x1000, "x_scale": 0x2000, "w_q": 0x3000, "w_scale": 0x4000, "out": 0x5000,
            "x_q_stride": 64, "w_stride": 64, "dtype": 1, "M": 40, "K": 64, "N": 32}
    return _pack(_layers()[0]._MATMUL, MATMUL, base, kw)


def test_matmul_arguments():
    _, L = _layers()
    status = lambda **kw: L.ww_int8_matmul(_matmul(**kw), None)  # noqa: E731
    assert L.ww_int8_matmul(None, None) == NULL and L.ww_int8_matmul_workspace(None) == 0
    assert status(dtype=2) == DTYPE and status(M=-1) == SHAPE and status(K=0) == SHAPE and status(N=-1) == SHAPE
    assert status(K=1 << 17, w_stride=1 << 17, x_q_stride=1 << 17) == LIMIT
    for name in ("x_q", "x_scale", "w_q", "w_scale", "out"):
        assert status(**{name: 0}) == NULL
    assert status(x=0x6000) == NULL  # both forms of the activations
    assert status(w_stride=48) == SHAPE and status(x_q_stride=48) == SHAPE and status(w_stride=72) == ALIGN and status(x_q_stride=72) == ALIGN
    assert status(w_q=0x3008) == ALIGN and status(x_q=0x1008) == ALIGN and status(out=0x5001) == ALIGN and status(bias=0x5001) == ALIGN
    assert status(w_scale=0x4002) == ALIGN and status(x_scale=0x2001) == ALIGN
    assert status(M=0, x_q=0) == OK and status(N=0, w_q=0) == OK
    wide = dict(x=0x6000, x_q=0, x_scale=0, x_stride=64)
    assert L.ww_int8_matmul_workspace(_matmul(**wide)) == 40 * 64 + 40 * 4
    assert L.ww_int8_matmul_workspace(_matmul(**wide, M=4)) == 0 and L.ww_int8_matmul_workspace(_matmul()) == 0
    assert status(**wide) == NULL and status(**wide, workspace=0x7008, workspace_bytes=1 << 20) == ALIGN
    assert status(**wide, workspace=0x7000, workspace_bytes=100) == LIMIT


CACHE = (["k", "v", "k_cache", "v_cache", "k_scale", "v_scale", "start", "lens", "k_out", "v_out"] +
         [f"{n}{i}" for n in ("ks", "vs", "kc", "vc") for i in range(3)] + [f"{n}{i}" for n in ("kss", "vss") for i in range(2)] +
         ["dtype", "B", "L", "places", "H", "D"])


def _cache(**kw):
    base = {**dict.fromkeys(CACHE, 0), **{n: 0x1000 for n in CACHE[:6]}, "k_out": 0x2000, "v_out": 0x3000,
            **{f"{n}{i}": s for n in ("ks", "vs", "kc", "vc") for i, s in enumerate((8 * 4 * 32, 4 * 32, 32))},
            **{f"{n}{i}": s for n in ("kss", "vss") for i, s in enumerate((32, 8))}, "dtype": 1, "B": 2, "L": 8, "places": 8, "H": 4, "D": 32}
    return _pack(_layers()[0]._CACHE, CACHE, base, kw)


def test_cache_arguments():
    _, L = _layers()
    for call, inputs in ((L.ww_quantize_kv, ("k", "v")), (L.ww_dequantize_kv, ("k_out", "v_out"))):
        status = lambda call=call, **kw: call(_cache(**kw), None)  # noqa: E731
        assert call(None, None) == NULL
        assert status(dtype=0) == DTYPE and status(B=-1) == SHAPE and status(H=0) == SHAPE and status(D=0) == SHAPE
        assert status(D=40) == LIMIT and status(D=144) == LIMIT and status(B=1 << 20, L=1 << 12, places=1 << 12) == LIMIT
        for name in (*inputs, "k_cache", "v_cache", "k_scale", "v_scale"):
            assert status(**{name: 0}) == NULL
            assert status(**{name: 0x1002 if "scale" in name else 0x1008}) == ALIGN
        assert status(kc1=120) == ALIGN and status(vc0=-1024) == ALIGN and status(vss1=-1) == SHAPE
        assert status(start=0x1001) == ALIGN and status(lens=0x1002) == ALIGN
        assert status(B=0) == OK and status(places=0) == OK
    write = lambda **kw: L.ww_quantize_kv(_cache(**kw), None)  # noqa: E731
    assert write(kc1=0) == SHAPE and write(vc0=0) == SHAPE and write(kss1=0) == SHAPE and write(vss0=4) == SHAPE  # two places in one
    assert write(ks1=100) == ALIGN and write(vs2=-32) == ALIGN and write(L=0) == OK


def _attention(scales=(0x1000, 0x1000, 32, 8, 32, 8), **kw):
    from whirlwind_trt_plugins_b200 import attention, layers
    names = ("dtype", "B", "Lq", "Lk", "Hq", "Hk", "D", "buckets", "distance", "bi", "off")
    sizes = dict(zip(names, [1, 2, 1, 8, 4, 4, 64, 0, 128, 1, 0]))
    ptrs, strides = kw.pop("ptrs", [0x1000] * 4 + [0] * 10), kw.pop("strides", [4 * 64 * 8, 4 * 64, 64] * 4)
    assert set(kw) <= set(names)
    return attention._ATTN.pack(*ptrs, 0, *strides, *[{**sizes, **kw}[n] for n in names], 0.125) + layers._SCALES.pack(*scales)


def test_attention_int8_arguments():
    _, L = _layers()
    status = lambda **kw: L.ww_cross_attention_int8(_attention(**kw), None)  # noqa: E731
    assert L.ww_cross_attention_int8(None, None) == NULL and L.ww_cross_attention_int8_workspace(None) == 0
    assert status(dtype=0) == DTYPE and status(B=-1) == SHAPE and status(Hk=3) == SHAPE and status(D=56) == LIMIT and status(D=144) == LIMIT
    for n in range(4):
        for p, want in ((0, NULL), (0x1008, ALIGN)):
            ptrs = [0x1000] * 4 + [0] * 10
            ptrs[n] = p
            assert status(ptrs=ptrs) == want
    good = [4 * 64 * 8, 4 * 64, 64]
    assert status(strides=good + [4 * 64 * 8, 4 * 64, 24] + good * 2) == ALIGN and status(strides=good * 2 + [4 * 64 * 8, -64, 64] + good) == ALIGN
    assert status(strides=good + [4 * 64 * 8, 0, 64] + good * 2) == ALIGN  # broadcast along the keys
    assert status(scales=(0, 0x1000, 32, 8, 32, 8)) == NULL and status(scales=(0x1000, 0x1002, 32, 8, 32, 8)) == ALIGN
    assert status(scales=(0x1000, 0x1000, 32, -8, 32, 8)) == SHAPE
    assert status(B=1 << 12, Lk=1 << 20) == LIMIT
    assert status(Lq=0) == OK and status(B=0) == OK
    many = L.ww_cross_attention_int8_workspace(_attention(Lq=129))
    assert many >= 2 * 2 * 8 * 4 * 64 * 2 and status(Lq=129) == NULL  # copies in 16 bits need their memory


def test_wrappers_refuse():
    import torch
    import whirlwind_trt_plugins_b200 as ww
    x = torch.zeros(4, 64)
    for call in (lambda: ww.layer_norm(x), lambda: ww.layer_norm_int8(x), lambda: ww.quantize_tokens(x),
                 lambda: ww.layer_norm_backward(x, x, None, x, x), lambda: ww.int8_linear(x, x, x), lambda: ww.int8_matmul(x, x, x, x),
                 lambda: ww.quantize_kv(x, x, x, x, x, x), lambda: ww.dequantize_kv(x, x, x, x),
                 lambda: ww.cross_attention_int8(x, x, x, x, x), lambda: ww.layer_norm(None)):
        with pytest.raises(TypeError, match="CUDA tensor"):
            call()


@pytest.fixture(scope="module")
def pl():
    from whirlwind_trt_plugins_b200 import plugins
    return plugins


def test_struct_layouts(tmp_path):
    import shutil
    import subprocess

    from conftest import ROOT
    layers, _ = _layers()
    if shutil.which("gcc") is None:
        pytest.skip("needs gcc")
    src, exe = tmp_path / "s.c", tmp_path / "s"
    names = "ww_layer_norm_t ww_int8_matmul_t ww_kv_cache_t ww_attention_int8_t".split()
    at = "ww_layer_norm_t, workspace|ww_int8_matmul_t, workspace|ww_attention_t, workspace|ww_attention_int8_t, k_scale".split("|")
    values = ", ".join([f"sizeof({n})" for n in names] + [f"offsetof({n})" for n in at])
    src.write_text(f'#include "ww_trt_plugins.h"\n#include <stdio.h>\nint main(void) {{ size_t v[] = {{{values}}}; '
                   'for (int i = 0; i < 8; ++i) printf("%zu ", v[i]); return 0; }\n')
    subprocess.run(["gcc", f"-I{ROOT}/include", str(src), "-o", str(exe)], check=True)
    got = list(map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()))
    from whirlwind_trt_plugins_b200.attention import _ATTN
    assert got == [layers._NORM.size, layers._MATMUL.size, layers._CACHE.size, _ATTN.size + layers._SCALES.size,
                   layers._NORM_WS, layers._MATMUL_WS, layers._ATTN_WS, _ATTN.size]


def test_plugin_shapes_and_formats(pl):
    T = pl.TensorDesc
    H, I8, F = pl.DTYPE_HALF, pl.DTYPE_INT8, pl.DTYPE_FLOAT
    norm = pl.get_plugin_creator("LayerNorm").create_plugin({"use_residual": 1})
    x, w = T((2, 5, 64)), T((64,))
    assert norm.get_nb_outputs() == 2 and norm.eps_nano == 10000 and norm.clone().use_residual == 1
    assert norm.get_output_shapes([x, w, w, x]) == [(2, 5, 64)] * 2 and norm.get_output_data_types([H] * 4) == [H, H]
    assert all(norm.supports_format_combination(i, [x, w, w, x, x, x], 4, 2) for i in range(6))
    assert not norm.supports_format_combination(1, [x, T((64,), F), w, x, x, x], 4, 2)
    assert not norm.supports_format_combination(0, [T((2, 64), I8)] * 6, 4, 2) and not norm.supports_format_combination(6, [x] * 6, 4, 2)
    for bad in ([x, w, w], [x, T((32,)), w, x], [x, w, w, T((2, 4, 64))], [T(()), w, w, T(())]):
        with pytest.raises(ValueError):
            norm.get_output_shapes(bad)
    lin = pl.get_plugin_creator("Int8Linear").create_plugin({"use_bias": 1})
    ins = [x, T((33, 64), I8), T((33,), F), T((33,))]
    assert lin.get_output_shapes(ins) == [(2, 5, 33)]
    assert all(lin.supports_format_combination(i, ins + [T((2, 5, 33))], 4, 1) for i in range(5))
    assert not lin.supports_format_combination(1, [x, T((33, 64)), *ins[2:], x], 4, 1)
    assert lin.get_workspace_size([T((700, 64)), *ins[1:]]) == 700 * 64 + 700 * 4 and lin.get_workspace_size(ins[:1] * 4) == -1
    for bad in ([x, T((33, 72), I8), *ins[2:]], [T((2, 24)), T((33, 24), I8), *ins[2:]], ins[:3], [*ins[:3], T((32,))]):
        with pytest.raises(ValueError):
            lin.get_output_shapes(bad)
    quant = pl.get_plugin_creator("QuantizeKv").create_plugin()
    k = T((2, 7, 3, 32))
    assert quant.get_output_shapes([k, k]) == [(2, 7, 3, 32)] * 2 + [(2, 3, 7)] * 2 and quant.get_output_data_types([H, H]) == [I8, I8, F, F]
    outs = [T((2, 7, 3, 32), I8)] * 2 + [T((2, 3, 7), F)] * 2
    assert all(quant.supports_format_combination(i, [k, k, *outs], 2, 4) for i in range(6))
    for bad in ([k], [k, T((2, 7, 3, 16))], [T((2, 7, 3, 40))] * 2, [T((2, 7, 96))] * 2):
        with pytest.raises(ValueError):
            quant.get_output_shapes(bad)
    attn = pl.get_plugin_creator("CrossAttentionInt8").create_plugin({"use_lens": 1, "use_bias": 1})
    q = T((2, 1, 6, 32))
    ins = [q, *outs, T((2,), pl.DTYPE_INT32), T((6, 16))]
    assert attn.get_output_shapes(ins) == [(2, 1, 6, 32)] and attn.clone().use_bias == 1
    assert all(attn.supports_format_combination(i, ins + [q], 7, 1) for i in range(8))
    assert not attn.supports_format_combination(1, [q, k, *ins[2:], q], 7, 1) and not attn.supports_format_combination(3, ins[:3] + [q] * 5, 7, 1)
    assert attn.get_workspace_size(ins) >= 2 * 2 * 7 * 3 * 32 * 2 and attn.get_workspace_size([q] * 7) == -1
    for bad in (ins[:5], [q, *outs[:2], T((2, 7, 3), F), *ins[4:]], [T((2, 1, 6, 16)), *ins[1:]]):
        with pytest.raises(ValueError):
            attn.get_output_shapes(bad)


def test_plugin_enqueue_refuses(pl):
    """A rejected request gives 1, as IPluginV3OneRuntime::enqueue does, before any GPU work."""
    T = pl.TensorDesc
    x, w = T((4, 64)), T((64,))
    norm = pl.LayerNormPlugin()
    assert norm.enqueue([x, w, T((32,))], [0x1000] * 3, [0x2000], stream=0) == 1
    assert norm.enqueue([x, w, w], [0x1000, 0x1000, 0], [0x2000], stream=0) == 1
    lin = pl.Int8LinearPlugin()
    ins = [T((400, 64)), T((33, 64), pl.DTYPE_INT8), T((33,), pl.DTYPE_FLOAT)]
    assert lin.enqueue(ins, [0x1000] * 3, [0x2000], stream=0) == 1  # its workspace is missing
    k = T((2, 7, 3, 32))
    assert pl.QuantizeKvPlugin().enqueue([k, T((2, 7, 3, 32), pl.DTYPE_FLOAT)], [0x1000] * 2, [0x2000] * 4, stream=0) == 1
    attn = pl.CrossAttentionInt8Plugin()
    i8, sc = T((2, 7, 3, 32), pl.DTYPE_INT8), T((2, 3, 7), pl.DTYPE_FLOAT)
    assert attn.enqueue([T((2, 200, 6, 32)), i8, i8, sc, sc], [0x1000] * 5, [0x2000], stream=0) == 1  # copies need their memory
    assert attn.enqueue([T((2, 1, 6, 32)), i8, i8, sc, k], [0x1000] * 5, [0x2000], stream=0) == 1
