// plugin_core.cpp -- the logic of the reference's IPluginV3 methods for
// CorrVolume and CostStem3D (and the fused CorrCostStem3D extension), written
// against plain descriptors (ww_tensor_desc_t) instead of TensorRT types.
// The TensorRT shim in trt/ forwards each IPluginV3 method here; the tests
// call these directly.  Nothing here touches the GPU except the *_enqueue
// functions, and those only after every check has passed.
#include "../../include/ww_trt_plugins.h"

#include <cmath>
#include <cstring>

namespace {

bool is_linear_half(const ww_tensor_desc_t& d)
{
    return d.format == WW_FORMAT_LINEAR && d.dtype == WW_DTYPE_HALF;
}

bool fits_int(int64_t v) { return v >= 0 && v <= 0x7fffffff; }

bool same_shape(const ww_tensor_desc_t& a, const ww_tensor_desc_t& b)
{
    if (a.nb_dims != b.nb_dims || a.nb_dims < 0 || a.nb_dims > 8) return false;
    for (int i = 0; i < a.nb_dims; ++i)
        if (a.dims[i] != b.dims[i]) return false;
    return true;
}

// Element count of a descriptor; -1 for a negative (unknown) or invalid shape.
int64_t numel(const ww_tensor_desc_t& d)
{
    if (d.nb_dims < 0 || d.nb_dims > 8) return -1;
    int64_t n = 1;
    for (int i = 0; i < d.nb_dims; ++i) {
        if (d.dims[i] < 0) return -1;
        n *= d.dims[i];
    }
    return n;
}

// Inputs of CrossAttention with these flags, and what input i >= 3 is.
int attention_inputs(int flags)
{
    return 3 + ((flags & WW_PLUGIN_ATTENTION_LENS) != 0) + ((flags & WW_PLUGIN_ATTENTION_MASK) != 0) +
           ((flags & WW_PLUGIN_ATTENTION_BIAS) != 0);
}

int attention_role(int flags, int i)
{
    for (int role = WW_PLUGIN_ATTENTION_LENS; role <= WW_PLUGIN_ATTENTION_BIAS; role <<= 1)
        if ((flags & role) != 0 && i-- == 3) return role;
    return 0;
}

// {b, l, h} strides of a contiguous [B, L, H, D].
void contiguous_strides(const ww_tensor_desc_t& d, int64_t (&s)[3])
{
    s[2] = d.dims[3];
    s[1] = s[2] * d.dims[2];
    s[0] = s[1] * d.dims[1];
}

bool is_float_type(int32_t t) { return t == WW_DTYPE_HALF || t == WW_DTYPE_BF16 || t == WW_DTYPE_FLOAT; }

// Rows (all dims but the last) and their length; false where they do not fit.
bool rows_of(const ww_tensor_desc_t& d, int32_t* rows, int32_t* n)
{
    const int64_t all = numel(d);
    if (d.nb_dims < 1 || all < 0) return false;
    const int64_t last = d.dims[d.nb_dims - 1], count = last > 0 ? all / last : 0;
    if (!fits_int(last) || !fits_int(count)) return false;
    *rows = static_cast<int32_t>(count);
    *n = static_cast<int32_t>(last);
    return true;
}

// Sizes of an Int8Linear call, pointers that are there (not these) for the workspace's size.
bool int8_linear(int use_bias, const ww_tensor_desc_t* in, ww_int8_matmul_t* p)
{
    ww_tensor_desc_t out;
    const int n = use_bias ? 4 : 3;
    if (in == nullptr || ww_plugin_int8_linear_output_dims(use_bias, n, in, &out) != 0) return false;
    for (int i = 0; i < n; ++i)
        if (!ww_plugin_int8_linear_supports_format(use_bias, i, in, n, 1)) return false;
    std::memset(p, 0, sizeof(*p));
    if (!rows_of(in[0], &p->M, &p->K) || !fits_int(in[1].dims[0])) return false;
    p->N = static_cast<int32_t>(in[1].dims[0]);
    p->x_stride = p->w_stride = p->K;
    p->dtype = in[0].dtype;
    static const uint64_t kThere[2] = {};
    p->x = p->w_scale = reinterpret_cast<const float*>(kThere);
    p->w_q = reinterpret_cast<const int8_t*>((reinterpret_cast<uintptr_t>(kThere) + 15) / 16 * 16);
    p->out = const_cast<uint64_t*>(kThere);
    return true;
}

// The first n descriptors without the two scales behind v.
void without_scales(const ww_tensor_desc_t* in, int n, ww_tensor_desc_t* out)
{
    for (int i = 0; i < n; ++i)
        if (i < 3) out[i] = in[i];
        else if (i >= 5) out[i - 2] = in[i];
}

// Sizes and strides of a CrossAttentionInt8 call.
bool attention_int8(int flags, const ww_tensor_desc_t* in, ww_attention_int8_t* p)
{
    ww_tensor_desc_t out;
    const int n = attention_inputs(flags) + 2;
    if (in == nullptr || ww_plugin_cross_attention_int8_output_dims(flags, n, in, &out) != 0) return false;
    for (int i = 0; i < n; ++i) {
        if (!ww_plugin_cross_attention_int8_supports_format(flags, i, in, n, 1)) return false;
        for (int j = 0; j < in[i].nb_dims; ++j)
            if (!fits_int(in[i].dims[j])) return false;
    }
    std::memset(p, 0, sizeof(*p));
    ww_attention_t& a = p->attention;
    const ww_tensor_desc_t &q = in[0], &k = in[1];
    a.dtype = q.dtype;
    a.B = static_cast<int32_t>(q.dims[0]);
    a.Lq = static_cast<int32_t>(q.dims[1]);
    a.Hq = static_cast<int32_t>(q.dims[2]);
    a.D = static_cast<int32_t>(q.dims[3]);
    a.Lk = static_cast<int32_t>(k.dims[1]);
    a.Hk = static_cast<int32_t>(k.dims[2]);
    contiguous_strides(q, a.q_strides);
    contiguous_strides(k, a.k_strides);
    contiguous_strides(k, a.v_strides);
    p->k_scale_strides[0] = p->v_scale_strides[0] = k.dims[1] * k.dims[2];
    p->k_scale_strides[1] = p->v_scale_strides[1] = k.dims[1];
    a.scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(a.D)));
    return true;
}

// Bytes of the 16-bit copies that ww_cross_attention_int8 makes for many rows, with their powers of two.
int64_t attention_copies(const ww_attention_t& a)
{
    const int64_t heads = static_cast<int64_t>(a.B) * a.Hk, one = heads * a.Lk * a.D * 2;
    return 2 * ((one + 255) / 256 * 256) + (heads * 8 + 255) / 256 * 256;
}

}  // namespace

extern "C" {

// plugin_fields.hpp:17-31: first field named `name` whose data is non-null.
int ww_plugin_get_int_field(int nb_fields, const char* const* names, const int32_t* const* values,
                            const char* name, int fallback)
{
    if (names == nullptr || values == nullptr || name == nullptr) return fallback;
    for (int i = 0; i < nb_fields; ++i) {
        if (values[i] == nullptr || names[i] == nullptr) continue;
        if (std::strcmp(names[i], name) == 0) return *values[i];
    }
    return fallback;
}

// ---------------------------------------------------------------- CorrVolume

// corr_volume.cpp:28-37: output type = input 0 type.
int ww_plugin_corr_volume_output_dtype(int nb_inputs, const int32_t* in_dtypes, int32_t* out_dtype)
{
    if (nb_inputs < 1 || in_dtypes == nullptr || out_dtype == nullptr) return 1;
    *out_dtype = in_dtypes[0];
    return 0;
}

// corr_volume.cpp:39-58: [B, max_disp, H, W]; with the num_groups extension
// and G > 1: [B, G, max_disp, H, W].
int ww_plugin_corr_volume_output_dims(int max_disp, int num_groups, int nb_inputs,
                                      const ww_tensor_desc_t* inputs, ww_tensor_desc_t* out)
{
    if (nb_inputs != 2 || inputs == nullptr || out == nullptr) return 1;
    const ww_tensor_desc_t& in = inputs[0];
    if (in.nb_dims != 4) return 1;
    *out = in;
    if (num_groups <= 1) {
        out->nb_dims = 4;
        out->dims[0] = in.dims[0];
        out->dims[1] = max_disp;
        out->dims[2] = in.dims[2];
        out->dims[3] = in.dims[3];
    } else {
        out->nb_dims = 5;
        out->dims[0] = in.dims[0];
        out->dims[1] = num_groups;
        out->dims[2] = max_disp;
        out->dims[3] = in.dims[2];
        out->dims[4] = in.dims[3];
    }
    return 0;
}

// corr_volume.cpp:60-82: LINEAR only; position 0 fp16 only (advertising
// fp32 would let TensorRT insert a reformat in front of the fast path); the
// other input and the output must match position 0.
int ww_plugin_corr_volume_supports_format(int pos, const ww_tensor_desc_t* in_out, int nb_inputs,
                                          int nb_outputs)
{
    if (in_out == nullptr || nb_inputs != 2 || nb_outputs != 1) return 0;
    if (pos < 0 || pos >= nb_inputs + nb_outputs) return 0;
    const ww_tensor_desc_t& d = in_out[pos];
    if (d.format != WW_FORMAT_LINEAR) return 0;
    if (pos == 0) return d.dtype == WW_DTYPE_HALF;
    return d.dtype == in_out[0].dtype;
}

// corr_volume.cpp:84-111: rank-4 input, fp16 or fp32, launch; 0 or 1.
int ww_plugin_corr_volume_enqueue(int max_disp, int num_groups, const ww_tensor_desc_t* in_desc,
                                  const void* const* inputs, void* const* outputs, void* stream)
{
    if (in_desc == nullptr || inputs == nullptr || outputs == nullptr) return 1;
    const ww_tensor_desc_t& d = in_desc[0];
    if (d.nb_dims != 4) return 1;
    for (int i = 0; i < 4; ++i)
        if (!fits_int(d.dims[i])) return 1;
    if (d.dtype != WW_DTYPE_HALF && d.dtype != WW_DTYPE_FLOAT) return 1;
    const int G = num_groups <= 0 ? 1 : num_groups;
    const int st = ww_corr_volume(inputs[0], inputs[1], outputs[0], d.dtype, static_cast<int>(d.dims[0]),
                                  static_cast<int>(d.dims[1]), static_cast<int>(d.dims[2]),
                                  static_cast<int>(d.dims[3]), max_disp, G, stream);
    return st == WW_SUCCESS ? 0 : 1;
}

// ---------------------------------------------------------------- CostStem3D

// cost_stem_3d.cpp:28-37 (7 inputs: output = input 0 shape) plus the 3-input
// generalised form (output [B, Cout, D, H, W], Cout = w.dims[0]).
int ww_plugin_cost_stem3d_output_dims(int nb_inputs, const ww_tensor_desc_t* inputs, ww_tensor_desc_t* out)
{
    if (inputs == nullptr || out == nullptr) return 1;
    if (nb_inputs == 7) {
        *out = inputs[0];
        return 0;
    }
    if (nb_inputs == 3) {
        if (inputs[0].nb_dims != 5 || inputs[1].nb_dims != 5) return 1;
        // the generalised stem's limits (ww_cost_stem3d_supported), where known
        const int64_t Cin = inputs[0].dims[1], D = inputs[0].dims[2], Cout = inputs[1].dims[0];
        if (Cin > 0 && D > 0 && Cout > 0 && fits_int(Cin) && fits_int(D) && fits_int(Cout) &&
            ww_cost_stem3d_supported(static_cast<int>(Cin), static_cast<int>(D), static_cast<int>(Cout)) != WW_SUCCESS)
            return 1;
        *out = inputs[0];
        out->dims[1] = inputs[1].dims[0];
        return 0;
    }
    return 1;
}

// cost_stem_3d.cpp:39-48: every position fp16 LINEAR.
int ww_plugin_cost_stem3d_supports_format(int pos, const ww_tensor_desc_t* in_out, int nb_inputs,
                                          int nb_outputs)
{
    if (in_out == nullptr || (nb_inputs != 7 && nb_inputs != 3) || nb_outputs != 1) return 0;
    if (pos < 0 || pos >= nb_inputs + nb_outputs) return 0;
    return is_linear_half(in_out[pos]);
}

// cost_stem_3d.cpp:50-73 (rank-5 input 0, B = d[0], D = d[2], H = d[3],
// W = d[4]) and the 3-input form (w [Cout, Cin, 3, 3, 3], b [Cout]).
int ww_plugin_cost_stem3d_enqueue(int nb_inputs, int act, const ww_tensor_desc_t* in_desc,
                                  const void* const* inputs, void* const* outputs, void* stream)
{
    if (in_desc == nullptr || inputs == nullptr || outputs == nullptr) return 1;
    const ww_tensor_desc_t& d = in_desc[0];
    if (d.nb_dims != 5) return 1;
    for (int i = 0; i < 5; ++i)
        if (!fits_int(d.dims[i])) return 1;
    const int B = static_cast<int>(d.dims[0]), D = static_cast<int>(d.dims[2]);
    const int H = static_cast<int>(d.dims[3]), W = static_cast<int>(d.dims[4]);
    int st;
    if (nb_inputs == 7) {
        st = ww_cost_stem3d_ref3(inputs[0], outputs[0], inputs[1], inputs[2], inputs[3], inputs[4], inputs[5],
                                 inputs[6], B, D, H, W, stream);
    } else if (nb_inputs == 3) {
        const ww_tensor_desc_t& wd = in_desc[1];
        if (wd.nb_dims != 5 || wd.dims[1] != d.dims[1] || wd.dims[2] != 3 || wd.dims[3] != 3 || wd.dims[4] != 3)
            return 1;
        if (!fits_int(wd.dims[0])) return 1;
        st = ww_cost_stem3d(inputs[0], inputs[1], inputs[2], outputs[0], B, static_cast<int>(d.dims[1]),
                            static_cast<int>(wd.dims[0]), D, H, W, act, stream);
    } else {
        return 1;
    }
    return st == WW_SUCCESS ? 0 : 1;
}

// ------------------------------------------------------- CorrCostStem3D (new)

int ww_plugin_corr_cost_stem3d_output_dims(int max_disp, int num_groups, int nb_inputs,
                                           const ww_tensor_desc_t* inputs, ww_tensor_desc_t* out)
{
    if ((nb_inputs != 4 && nb_inputs != 8) || inputs == nullptr || out == nullptr) return 1;
    if (inputs[0].nb_dims != 4) return 1;
    if (nb_inputs == 4) {
        // The fused kernel's limits, checked here so that an engine build
        // fails rather than the enqueue (C may be unknown, -1, for a dynamic
        // shape: then the group-size dependent part is left to the enqueue).
        if (inputs[2].nb_dims != 5) return 1;
        const int G = num_groups <= 0 ? 1 : num_groups;
        if (inputs[2].dims[1] != G || !fits_int(inputs[2].dims[0])) return 1;
        const int Cout = static_cast<int>(inputs[2].dims[0]);
        const int64_t C = inputs[0].dims[1];
        const int lim = C > 0 && fits_int(C) ? ww_corr_cost_stem3d_supported(static_cast<int>(C), G, max_disp, Cout)
                                             : ww_corr_cost_stem3d_supported(8 * G, G, max_disp, Cout);
        if (lim != WW_SUCCESS) return 1;
    }
    *out = inputs[0];
    out->nb_dims = 5;
    out->dims[0] = inputs[0].dims[0];
    // 8 inputs: the reference's 3-stage stem (w0, b0, w1, b1, w2, b2), one
    // output channel
    out->dims[1] = nb_inputs == 8 ? 1 : inputs[2].dims[0];
    out->dims[2] = max_disp;
    out->dims[3] = inputs[0].dims[2];
    out->dims[4] = inputs[0].dims[3];
    return 0;
}

int ww_plugin_corr_cost_stem3d_supports_format(int pos, const ww_tensor_desc_t* in_out, int nb_inputs,
                                               int nb_outputs)
{
    if (in_out == nullptr || (nb_inputs != 4 && nb_inputs != 8) || nb_outputs != 1) return 0;
    if (pos < 0 || pos >= nb_inputs + nb_outputs) return 0;
    return is_linear_half(in_out[pos]);
}

int ww_plugin_corr_cost_stem3d_enqueue(int nb_inputs, int max_disp, int num_groups, int act,
                                       const ww_tensor_desc_t* in_desc, const void* const* inputs,
                                       void* const* outputs, void* stream)
{
    if (in_desc == nullptr || inputs == nullptr || outputs == nullptr) return 1;
    if (nb_inputs != 4 && nb_inputs != 8) return 1;
    const ww_tensor_desc_t& d = in_desc[0];
    if (d.nb_dims != 4 || !same_shape(d, in_desc[1])) return 1;
    for (int i = 0; i < 4; ++i)
        if (!fits_int(d.dims[i])) return 1;
    for (int i = 0; i < nb_inputs; ++i)
        if (in_desc[i].dtype != WW_DTYPE_HALF) return 1;
    if (nb_inputs == 8) {
        // CorrVolume (G = 1) fused with the reference's 3-stage CostStem3D:
        // w0 [4,1,3,3,3] b0 [4] w1 [4,4,3,3,3] b1 [4] w2 [1,4,3,3,3] b2 [1]
        // (cost_stem_3d_kernel.hpp:8-15), any rank with those element
        // counts; num_groups must be 1 and the activation is ReLU6.
        static const int64_t kCounts[6] = {108, 4, 432, 4, 108, 1};
        if (num_groups > 1) return 1;
        for (int i = 0; i < 6; ++i)
            if (numel(in_desc[2 + i]) != kCounts[i]) return 1;
        const int st = ww_corr_cost_stem3d_ref3(inputs[0], inputs[1], outputs[0], inputs[2], inputs[3], inputs[4],
                                                inputs[5], inputs[6], inputs[7], static_cast<int>(d.dims[0]),
                                                static_cast<int>(d.dims[1]), static_cast<int>(d.dims[2]),
                                                static_cast<int>(d.dims[3]), max_disp, stream);
        return st == WW_SUCCESS ? 0 : 1;
    }
    const ww_tensor_desc_t& wd = in_desc[2];
    const int G = num_groups <= 0 ? 1 : num_groups;
    if (wd.nb_dims != 5 || wd.dims[1] != G || wd.dims[2] != 3 || wd.dims[3] != 3 || wd.dims[4] != 3 ||
        !fits_int(wd.dims[0]))
        return 1;
    if (numel(in_desc[3]) != wd.dims[0]) return 1;  // one bias per output channel
    const int st = ww_corr_cost_stem3d(inputs[0], inputs[1], inputs[2], inputs[3], outputs[0],
                                       static_cast<int>(d.dims[0]), static_cast<int>(d.dims[1]), G,
                                       static_cast<int>(d.dims[2]), static_cast<int>(d.dims[3]), max_disp,
                                       static_cast<int>(wd.dims[0]), act, stream);
    return st == WW_SUCCESS ? 0 : 1;
}

// ------------------------------------------------------------- Nv12Decode

// nv12_decode.cpp:26-39: the output is declared fp32 whatever the input
// (TensorRT picks fp16 or fp32 through supportsFormatCombination).
int ww_plugin_nv12_decode_output_dtype(int nb_inputs, int32_t* out_dtype)
{
    (void)nb_inputs;
    if (out_dtype == nullptr) return 1;
    *out_dtype = WW_DTYPE_FLOAT;
    return 0;
}

// nv12_decode.cpp:41-60: [B, H_IN * 3 / 2, W_IN] -> [B, 3, out_h, out_w].
int ww_plugin_nv12_decode_output_dims(int out_h, int out_w, int nb_inputs, const ww_tensor_desc_t* inputs,
                                      ww_tensor_desc_t* out)
{
    if (nb_inputs != 1 || inputs == nullptr || out == nullptr) return 1;
    *out = inputs[0];
    out->nb_dims = 4;
    out->dims[0] = inputs[0].dims[0];
    out->dims[1] = 3;
    out->dims[2] = out_h;
    out->dims[3] = out_w;
    out->dtype = WW_DTYPE_FLOAT;
    return 0;
}

// nv12_decode.cpp:62-86: LINEAR; position 0 INT8 only (the bytes are uint8
// NV12 values; accepting fp32 would let TensorRT insert a sign-extending
// cast), the output fp16 or fp32.
int ww_plugin_nv12_decode_supports_format(int pos, const ww_tensor_desc_t* in_out, int nb_inputs, int nb_outputs)
{
    if (in_out == nullptr || nb_inputs != 1 || nb_outputs != 1) return 0;
    if (pos < 0 || pos >= nb_inputs + nb_outputs) return 0;
    const ww_tensor_desc_t& d = in_out[pos];
    if (d.format != WW_FORMAT_LINEAR) return 0;
    if (pos == 0) return d.dtype == WW_DTYPE_INT8;
    return d.dtype == WW_DTYPE_HALF || d.dtype == WW_DTYPE_FLOAT;
}

// nv12_decode.cpp:88-115: rank-3 input, H_IN = 2 d[1] / 3, W_IN = d[2]; the
// output dtype selects the kernel; 0 or 1.  Every batch item is decoded (the
// reference launches batch 0 only).
int ww_plugin_nv12_decode_enqueue(int out_h, int out_w, const ww_tensor_desc_t* in_desc,
                                  const ww_tensor_desc_t* out_desc, const void* const* inputs,
                                  void* const* outputs, void* stream)
{
    if (in_desc == nullptr || out_desc == nullptr || inputs == nullptr || outputs == nullptr) return 1;
    const ww_tensor_desc_t& d = in_desc[0];
    if (d.nb_dims != 3) return 1;
    for (int i = 0; i < 3; ++i)
        if (!fits_int(d.dims[i])) return 1;
    const int dt = out_desc[0].dtype;
    if (dt != WW_DTYPE_HALF && dt != WW_DTYPE_FLOAT) return 1;
    const int H_IN = static_cast<int>(d.dims[1] * 2 / 3);
    const int st = ww_nv12_decode(inputs[0], outputs[0], dt, static_cast<int>(d.dims[0]), H_IN,
                                  static_cast<int>(d.dims[2]), out_h, out_w, stream);
    return st == WW_SUCCESS ? 0 : 1;
}

// ------------------------------------------------------ DisparityRegression
// No reference counterpart (the reference pipeline ends at CostStem3D); the
// plugin follows the conventions of the ones above: LINEAR, output dtype =
// input dtype, 0 / 1 enqueue codes.

// [B, D, H, W] or [B, 1, D, H, W] -> [B, 1, H, W].
int ww_plugin_disparity_regression_output_dims(int nb_inputs, const ww_tensor_desc_t* inputs,
                                               ww_tensor_desc_t* out)
{
    if (nb_inputs != 1 || inputs == nullptr || out == nullptr) return 1;
    const ww_tensor_desc_t& d = inputs[0];
    if (d.nb_dims != 4 && !(d.nb_dims == 5 && d.dims[1] == 1)) return 1;
    *out = d;
    out->nb_dims = 4;
    out->dims[0] = d.dims[0];
    out->dims[1] = 1;
    out->dims[2] = d.dims[d.nb_dims - 2];
    out->dims[3] = d.dims[d.nb_dims - 1];
    return 0;
}

// Position 0 fp16 or fp32 LINEAR; the output matches the input's dtype.
int ww_plugin_disparity_regression_supports_format(int pos, const ww_tensor_desc_t* in_out, int nb_inputs,
                                                   int nb_outputs)
{
    if (in_out == nullptr || nb_inputs != 1 || nb_outputs != 1) return 0;
    if (pos < 0 || pos >= nb_inputs + nb_outputs) return 0;
    const ww_tensor_desc_t& d = in_out[pos];
    if (d.format != WW_FORMAT_LINEAR) return 0;
    if (d.dtype != WW_DTYPE_HALF && d.dtype != WW_DTYPE_FLOAT) return 0;
    return pos == 0 || d.dtype == in_out[0].dtype;
}

int ww_plugin_disparity_regression_enqueue(int mode, const ww_tensor_desc_t* in_desc,
                                           const ww_tensor_desc_t* out_desc, const void* const* inputs,
                                           void* const* outputs, void* stream)
{
    if (in_desc == nullptr || out_desc == nullptr || inputs == nullptr || outputs == nullptr) return 1;
    const ww_tensor_desc_t& d = in_desc[0];
    if (d.nb_dims != 4 && !(d.nb_dims == 5 && d.dims[1] == 1)) return 1;
    for (int i = 0; i < d.nb_dims; ++i)
        if (!fits_int(d.dims[i])) return 1;
    const int n = d.nb_dims;
    const int st = ww_disparity_regression(inputs[0], outputs[0], d.dtype, out_desc[0].dtype,
                                           static_cast<int>(d.dims[0]), static_cast<int>(d.dims[n - 3]),
                                           static_cast<int>(d.dims[n - 2]), static_cast<int>(d.dims[n - 1]), mode,
                                           stream);
    return st == WW_SUCCESS ? 0 : 1;
}

// ---------------------------------------------------------- CrossAttention
// No reference counterpart; LINEAR only, the type of q decides the others'.

int ww_plugin_cross_attention_output_dims(int flags, int nb_inputs, const ww_tensor_desc_t* inputs,
                                          ww_tensor_desc_t* out)
{
    if (inputs == nullptr || out == nullptr || nb_inputs != attention_inputs(flags)) return 1;
    const ww_tensor_desc_t &q = inputs[0], &k = inputs[1], &v = inputs[2];
    if (q.nb_dims != 4 || k.nb_dims != 4 || !same_shape(k, v)) return 1;
    if (k.dims[0] != q.dims[0] || k.dims[3] != q.dims[3]) return 1;
    if (q.dims[3] <= 0 || q.dims[3] % 8 != 0 || q.dims[3] > 128) return 1;
    if (k.dims[2] <= 0 || q.dims[2] <= 0 || q.dims[2] % k.dims[2] != 0) return 1;
    const int n = attention_inputs(flags);
    for (int i = 3; i < n; ++i) {
        const ww_tensor_desc_t& d = inputs[i];
        switch (attention_role(flags, i)) {
            case WW_PLUGIN_ATTENTION_LENS:
                if (d.nb_dims != 1 || d.dims[0] != q.dims[0]) return 1;
                break;
            case WW_PLUGIN_ATTENTION_MASK:
                if (d.nb_dims != 2 || d.dims[0] != q.dims[0] || d.dims[1] != k.dims[1]) return 1;
                break;
            default:
                if (d.nb_dims != 2 || d.dims[0] != q.dims[2]) return 1;
        }
    }
    *out = q;
    return 0;
}

int ww_plugin_cross_attention_supports_format(int flags, int pos, const ww_tensor_desc_t* in_out, int nb_inputs,
                                              int nb_outputs)
{
    if (in_out == nullptr || nb_outputs != 1 || nb_inputs != attention_inputs(flags)) return 0;
    if (pos < 0 || pos >= nb_inputs + nb_outputs) return 0;
    const ww_tensor_desc_t& d = in_out[pos];
    if (d.format != WW_FORMAT_LINEAR) return 0;
    if (pos == 0) return d.dtype == WW_DTYPE_HALF || d.dtype == WW_DTYPE_BF16;
    if (pos >= 3 && pos < nb_inputs) {
        const int role = attention_role(flags, pos);
        if (role == WW_PLUGIN_ATTENTION_LENS) return d.dtype == WW_DTYPE_INT32;
        // bytes, 0 or not; declared INT8 as NV12's are, too
        if (role == WW_PLUGIN_ATTENTION_MASK)
            return d.dtype == WW_DTYPE_BOOL || d.dtype == WW_DTYPE_UINT8 || d.dtype == WW_DTYPE_INT8;
    }
    return d.dtype == in_out[0].dtype;
}

int ww_plugin_cross_attention_enqueue(int flags, int max_distance, int bidirectional, int q_offset,
                                      const ww_tensor_desc_t* in_desc, const void* const* inputs,
                                      void* const* outputs, void* workspace, void* stream)
{
    if (in_desc == nullptr || inputs == nullptr || outputs == nullptr) return 1;
    ww_tensor_desc_t out;
    const int n = attention_inputs(flags);
    if (ww_plugin_cross_attention_output_dims(flags, n, in_desc, &out) != 0) return 1;
    for (int i = 0; i < n; ++i) {
        if (!ww_plugin_cross_attention_supports_format(flags, i, in_desc, n, 1)) return 1;
        for (int j = 0; j < in_desc[i].nb_dims; ++j)
            if (!fits_int(in_desc[i].dims[j])) return 1;
    }
    ww_attention_t p;
    std::memset(&p, 0, sizeof(p));
    p.q = inputs[0];
    p.k = inputs[1];
    p.v = inputs[2];
    p.out = outputs[0];
    for (int i = 3; i < n; ++i) {
        switch (attention_role(flags, i)) {
            case WW_PLUGIN_ATTENTION_LENS: p.k_lens = static_cast<const int32_t*>(inputs[i]); break;
            case WW_PLUGIN_ATTENTION_MASK: p.key_mask = static_cast<const uint8_t*>(inputs[i]); break;
            default:
                p.bias_table = inputs[i];
                p.num_buckets = static_cast<int32_t>(in_desc[i].dims[1]);
        }
        if (inputs[i] == nullptr && numel(in_desc[i]) != 0) return 1;
    }
    const ww_tensor_desc_t &q = in_desc[0], &k = in_desc[1];
    p.dtype = q.dtype;
    p.B = static_cast<int32_t>(q.dims[0]);
    p.Lq = static_cast<int32_t>(q.dims[1]);
    p.Hq = static_cast<int32_t>(q.dims[2]);
    p.D = static_cast<int32_t>(q.dims[3]);
    p.Lk = static_cast<int32_t>(k.dims[1]);
    p.Hk = static_cast<int32_t>(k.dims[2]);
    contiguous_strides(q, p.q_strides);
    contiguous_strides(k, p.k_strides);
    contiguous_strides(k, p.v_strides);
    p.max_distance = max_distance;
    p.bidirectional = bidirectional;
    p.q_offset = q_offset;
    p.scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(p.D)));
    if (workspace != nullptr && ww_cross_attention_workspace(&p) <= WW_PLUGIN_ATTENTION_WORKSPACE) {
        p.workspace = workspace;
        p.workspace_bytes = WW_PLUGIN_ATTENTION_WORKSPACE;
    }
    return ww_cross_attention(&p, stream) == WW_SUCCESS ? 0 : 1;
}

// --------------------------------------------------------------- QkNormRope

int ww_plugin_qk_norm_rope_output_dims(int use_positions, int which, int nb_inputs, const ww_tensor_desc_t* inputs,
                                       ww_tensor_desc_t* out)
{
    if (inputs == nullptr || out == nullptr || nb_inputs != (use_positions ? 8 : 6) || which < 0 || which > 1) return 1;
    const ww_tensor_desc_t &q = inputs[0], &k = inputs[1], &cs = inputs[4];
    if (q.nb_dims != 4 || k.nb_dims != 4 || q.dims[0] != k.dims[0] || q.dims[3] != k.dims[3]) return 1;
    for (int i = 2; i < 4; ++i)
        if (inputs[i].nb_dims != 1 || inputs[i].dims[0] != q.dims[3]) return 1;
    if (cs.nb_dims != 2 || !same_shape(cs, inputs[5]) || 2 * cs.dims[1] > q.dims[3]) return 1;
    for (int i = 6; i < nb_inputs; ++i) {  // [L] or [B, L]
        const ww_tensor_desc_t& d = inputs[i];
        const int64_t L = inputs[i - 6].dims[1];
        if (!(d.nb_dims == 1 && d.dims[0] == L) && !(d.nb_dims == 2 && d.dims[0] == q.dims[0] && d.dims[1] == L)) return 1;
    }
    *out = inputs[which];
    return 0;
}

int ww_plugin_qk_norm_rope_supports_format(int use_positions, int pos, const ww_tensor_desc_t* in_out, int nb_inputs,
                                           int nb_outputs)
{
    if (in_out == nullptr || nb_outputs != 2 || nb_inputs != (use_positions ? 8 : 6)) return 0;
    if (pos < 0 || pos >= nb_inputs + nb_outputs) return 0;
    const ww_tensor_desc_t& d = in_out[pos];
    if (d.format != WW_FORMAT_LINEAR) return 0;
    if (pos == 0) return d.dtype == WW_DTYPE_HALF || d.dtype == WW_DTYPE_BF16 || d.dtype == WW_DTYPE_FLOAT;
    if (pos == 4 || pos == 5) return d.dtype == WW_DTYPE_FLOAT;
    if (pos >= 6 && pos < nb_inputs) return d.dtype == WW_DTYPE_INT32;
    return d.dtype == in_out[0].dtype;
}

int ww_plugin_qk_norm_rope_enqueue(int use_positions, int eps_nano, int interleaved, const ww_tensor_desc_t* in_desc,
                                   const void* const* inputs, void* const* outputs, void* stream)
{
    if (in_desc == nullptr || inputs == nullptr || outputs == nullptr) return 1;
    const int n = use_positions ? 8 : 6;
    ww_tensor_desc_t out;
    if (ww_plugin_qk_norm_rope_output_dims(use_positions, 0, n, in_desc, &out) != 0) return 1;
    for (int i = 0; i < n; ++i) {
        if (!ww_plugin_qk_norm_rope_supports_format(use_positions, i, in_desc, n, 2)) return 1;
        for (int j = 0; j < in_desc[i].nb_dims; ++j)
            if (!fits_int(in_desc[i].dims[j])) return 1;
    }
    ww_qk_norm_rope_t p;
    std::memset(&p, 0, sizeof(p));
    p.q = inputs[0];
    p.k = inputs[1];
    p.q_weight = inputs[2];
    p.k_weight = inputs[3];
    p.cos = static_cast<const float*>(inputs[4]);
    p.sin = static_cast<const float*>(inputs[5]);
    p.q_out = outputs[0];
    p.k_out = outputs[1];
    const ww_tensor_desc_t &q = in_desc[0], &k = in_desc[1];
    if (use_positions) {
        p.q_pos = static_cast<const int32_t*>(inputs[6]);
        p.k_pos = static_cast<const int32_t*>(inputs[7]);
        p.q_pos_stride = in_desc[6].nb_dims == 2 ? static_cast<int32_t>(q.dims[1]) : 0;
        p.k_pos_stride = in_desc[7].nb_dims == 2 ? static_cast<int32_t>(k.dims[1]) : 0;
    }
    contiguous_strides(q, p.q_strides);
    contiguous_strides(k, p.k_strides);
    p.dtype = q.dtype;
    p.B = static_cast<int32_t>(q.dims[0]);
    p.Lq = static_cast<int32_t>(q.dims[1]);
    p.Lk = static_cast<int32_t>(k.dims[1]);
    p.Hq = static_cast<int32_t>(q.dims[2]);
    p.Hk = static_cast<int32_t>(k.dims[2]);
    p.D = static_cast<int32_t>(q.dims[3]);
    p.R = static_cast<int32_t>(2 * in_desc[4].dims[1]);
    p.P = static_cast<int32_t>(in_desc[4].dims[0]);
    p.interleaved = interleaved;
    p.eps = static_cast<float>(eps_nano * 1e-9);
    return ww_qk_norm_rope(&p, stream) == WW_SUCCESS ? 0 : 1;
}

// ---------------------------------------------------------------- LayerNorm

int ww_plugin_layer_norm_output_dims(int use_residual, int which, int nb_inputs, const ww_tensor_desc_t* inputs,
                                     ww_tensor_desc_t* out)
{
    if (inputs == nullptr || out == nullptr || nb_inputs != (use_residual ? 4 : 3) || which < 0 || which > (use_residual ? 1 : 0)) return 1;
    const ww_tensor_desc_t& x = inputs[0];
    if (x.nb_dims < 1 || x.nb_dims > 8) return 1;
    for (int i = 1; i < 3; ++i)
        if (inputs[i].nb_dims != 1 || inputs[i].dims[0] != x.dims[x.nb_dims - 1]) return 1;
    if (use_residual && !same_shape(inputs[3], x)) return 1;
    *out = x;
    return 0;
}

int ww_plugin_layer_norm_supports_format(int use_residual, int pos, const ww_tensor_desc_t* in_out, int nb_inputs,
                                         int nb_outputs)
{
    if (in_out == nullptr || nb_inputs != (use_residual ? 4 : 3) || nb_outputs != (use_residual ? 2 : 1)) return 0;
    if (pos < 0 || pos >= nb_inputs + nb_outputs || in_out[pos].format != WW_FORMAT_LINEAR) return 0;
    if (pos == 0) return is_float_type(in_out[0].dtype);
    return in_out[pos].dtype == in_out[0].dtype;
}

int ww_plugin_layer_norm_enqueue(int use_residual, int eps_nano, const ww_tensor_desc_t* in_desc,
                                 const void* const* inputs, void* const* outputs, void* stream)
{
    if (in_desc == nullptr || inputs == nullptr || outputs == nullptr) return 1;
    const int n = use_residual ? 4 : 3;
    ww_tensor_desc_t out;
    if (ww_plugin_layer_norm_output_dims(use_residual, 0, n, in_desc, &out) != 0) return 1;
    for (int i = 0; i < n; ++i)
        if (!ww_plugin_layer_norm_supports_format(use_residual, i, in_desc, n, use_residual ? 2 : 1)) return 1;
    ww_layer_norm_t p;
    std::memset(&p, 0, sizeof(p));
    if (!rows_of(in_desc[0], &p.rows, &p.N)) return 1;
    p.x = inputs[0];
    p.weight = inputs[1];
    p.bias = inputs[2];
    p.y = outputs[0];
    if (use_residual) {
        p.residual = inputs[3];
        p.sum = outputs[1];
        if (p.rows > 0 && (p.residual == nullptr || p.sum == nullptr)) return 1;
    }
    if (p.weight == nullptr || p.bias == nullptr) return 1;
    p.x_stride = p.residual_stride = p.N;
    p.dtype = in_desc[0].dtype;
    p.eps = static_cast<float>(eps_nano * 1e-9);
    return ww_layer_norm(&p, stream) == WW_SUCCESS ? 0 : 1;
}

// --------------------------------------------------------------- Int8Linear

int ww_plugin_int8_linear_output_dims(int use_bias, int nb_inputs, const ww_tensor_desc_t* inputs,
                                      ww_tensor_desc_t* out)
{
    if (inputs == nullptr || out == nullptr || nb_inputs != (use_bias ? 4 : 3)) return 1;
    const ww_tensor_desc_t &x = inputs[0], &w = inputs[1];
    if (x.nb_dims < 1 || x.nb_dims > 8 || w.nb_dims != 2 || w.dims[1] != x.dims[x.nb_dims - 1] || w.dims[1] % 16 != 0) return 1;
    for (int i = 2; i < nb_inputs; ++i)
        if (inputs[i].nb_dims != 1 || inputs[i].dims[0] != w.dims[0]) return 1;
    *out = x;
    out->dims[x.nb_dims - 1] = w.dims[0];
    return 0;
}

int ww_plugin_int8_linear_supports_format(int use_bias, int pos, const ww_tensor_desc_t* in_out, int nb_inputs,
                                          int nb_outputs)
{
    if (in_out == nullptr || nb_inputs != (use_bias ? 4 : 3) || nb_outputs != 1) return 0;
    if (pos < 0 || pos >= nb_inputs + nb_outputs || in_out[pos].format != WW_FORMAT_LINEAR) return 0;
    if (pos == 0) return is_float_type(in_out[0].dtype);
    if (pos == 1) return in_out[1].dtype == WW_DTYPE_INT8;
    if (pos == 2) return in_out[2].dtype == WW_DTYPE_FLOAT;
    return in_out[pos].dtype == in_out[0].dtype;
}

int64_t ww_plugin_int8_linear_workspace(int use_bias, const ww_tensor_desc_t* in_desc)
{
    // An engine asks for its largest sizes: the tokens in 8 bits and their scales, which grow with every size, even where
    // those sizes take a form without them -- smaller ones may take one with them (4 x 4096 x 9473 does not, 4 x 4096 x 9472 does).
    ww_int8_matmul_t p;
    return int8_linear(use_bias, in_desc, &p) ? static_cast<int64_t>(p.M) * (p.K + 4) : -1;
}

int ww_plugin_int8_linear_enqueue(int use_bias, const ww_tensor_desc_t* in_desc, const void* const* inputs,
                                  void* const* outputs, void* workspace, void* stream)
{
    ww_int8_matmul_t p;
    if (inputs == nullptr || outputs == nullptr || !int8_linear(use_bias, in_desc, &p)) return 1;
    const int64_t need = ww_int8_matmul_workspace(&p);
    p.x = inputs[0];
    p.w_q = static_cast<const int8_t*>(inputs[1]);
    p.w_scale = static_cast<const float*>(inputs[2]);
    p.bias = use_bias ? inputs[3] : nullptr;
    if (use_bias && p.bias == nullptr) return 1;
    p.out = outputs[0];
    p.workspace = workspace;
    p.workspace_bytes = workspace == nullptr ? 0 : need;
    return ww_int8_matmul(&p, stream) == WW_SUCCESS ? 0 : 1;
}

// --------------------------------------------------------------- QuantizeKv

int ww_plugin_quantize_kv_output_dims(int which, int nb_inputs, const ww_tensor_desc_t* inputs, ww_tensor_desc_t* out)
{
    if (inputs == nullptr || out == nullptr || nb_inputs != 2 || which < 0 || which > 3) return 1;
    const ww_tensor_desc_t& k = inputs[0];
    if (k.nb_dims != 4 || !same_shape(k, inputs[1]) || k.dims[3] <= 0 || k.dims[3] % 16 != 0 || k.dims[3] > 128) return 1;
    *out = k;
    out->dtype = WW_DTYPE_INT8;
    if (which >= 2) {
        out->dtype = WW_DTYPE_FLOAT;
        out->nb_dims = 3;
        out->dims[1] = k.dims[2];
        out->dims[2] = k.dims[1];
        out->dims[3] = 0;
    }
    return 0;
}

int ww_plugin_quantize_kv_supports_format(int pos, const ww_tensor_desc_t* in_out, int nb_inputs, int nb_outputs)
{
    if (in_out == nullptr || nb_inputs != 2 || nb_outputs != 4) return 0;
    if (pos < 0 || pos >= 6 || in_out[pos].format != WW_FORMAT_LINEAR) return 0;
    const int32_t t = in_out[pos].dtype;
    if (pos == 0) return t == WW_DTYPE_HALF || t == WW_DTYPE_BF16;
    return t == (pos == 1 ? in_out[0].dtype : pos < 4 ? WW_DTYPE_INT8 : WW_DTYPE_FLOAT);
}

int ww_plugin_quantize_kv_enqueue(const ww_tensor_desc_t* in_desc, const void* const* inputs, void* const* outputs,
                                  void* stream)
{
    if (in_desc == nullptr || inputs == nullptr || outputs == nullptr) return 1;
    ww_tensor_desc_t out;
    if (ww_plugin_quantize_kv_output_dims(0, 2, in_desc, &out) != 0) return 1;
    for (int i = 0; i < 2; ++i)
        if (!ww_plugin_quantize_kv_supports_format(i, in_desc, 2, 4)) return 1;
    const ww_tensor_desc_t& k = in_desc[0];
    for (int i = 0; i < 4; ++i)
        if (!fits_int(k.dims[i])) return 1;
    ww_kv_cache_t p;
    std::memset(&p, 0, sizeof(p));
    p.k = inputs[0];
    p.v = inputs[1];
    p.k_cache = static_cast<int8_t*>(outputs[0]);
    p.v_cache = static_cast<int8_t*>(outputs[1]);
    p.k_scale = static_cast<float*>(outputs[2]);
    p.v_scale = static_cast<float*>(outputs[3]);
    contiguous_strides(k, p.k_strides);
    contiguous_strides(k, p.v_strides);
    contiguous_strides(k, p.k_cache_strides);
    contiguous_strides(k, p.v_cache_strides);
    p.k_scale_strides[1] = p.v_scale_strides[1] = k.dims[1];
    p.k_scale_strides[0] = p.v_scale_strides[0] = k.dims[1] * k.dims[2];
    p.dtype = k.dtype;
    p.B = static_cast<int32_t>(k.dims[0]);
    p.L = p.places = static_cast<int32_t>(k.dims[1]);
    p.H = static_cast<int32_t>(k.dims[2]);
    p.D = static_cast<int32_t>(k.dims[3]);
    return ww_quantize_kv(&p, stream) == WW_SUCCESS ? 0 : 1;
}

// ------------------------------------------------------- CrossAttentionInt8
// CrossAttention with two scales behind v.

int ww_plugin_cross_attention_int8_output_dims(int flags, int nb_inputs, const ww_tensor_desc_t* inputs,
                                               ww_tensor_desc_t* out)
{
    if (inputs == nullptr || nb_inputs != attention_inputs(flags) + 2) return 1;
    ww_tensor_desc_t d[6];
    without_scales(inputs, nb_inputs, d);
    if (ww_plugin_cross_attention_output_dims(flags, nb_inputs - 2, d, out) != 0 || d[0].dims[3] % 16 != 0) return 1;
    for (int i = 3; i < 5; ++i) {
        const ww_tensor_desc_t& s = inputs[i];
        if (s.nb_dims != 3 || s.dims[0] != d[1].dims[0] || s.dims[1] != d[1].dims[2] || s.dims[2] != d[1].dims[1]) return 1;
    }
    return 0;
}

int ww_plugin_cross_attention_int8_supports_format(int flags, int pos, const ww_tensor_desc_t* in_out, int nb_inputs,
                                                   int nb_outputs)
{
    if (in_out == nullptr || nb_outputs != 1 || nb_inputs != attention_inputs(flags) + 2) return 0;
    if (pos < 0 || pos > nb_inputs || in_out[pos].format != WW_FORMAT_LINEAR) return 0;
    if (pos == 1 || pos == 2) return in_out[pos].dtype == WW_DTYPE_INT8;
    if (pos == 3 || pos == 4) return in_out[pos].dtype == WW_DTYPE_FLOAT;
    ww_tensor_desc_t d[7];
    without_scales(in_out, pos + 1, d);  // no further: callers that ask for the inputs alone have no output's descriptor
    return ww_plugin_cross_attention_supports_format(flags, pos < 3 ? pos : pos - 2, d, nb_inputs - 2, 1);
}

int64_t ww_plugin_cross_attention_int8_workspace(int flags, const ww_tensor_desc_t* in_desc)
{
    ww_attention_int8_t p;
    // the 16-bit copies, and what smaller calls may want to split their keys
    return attention_int8(flags, in_desc, &p) ? attention_copies(p.attention) + WW_PLUGIN_ATTENTION_WORKSPACE : -1;
}

int ww_plugin_cross_attention_int8_enqueue(int flags, int max_distance, int bidirectional, int q_offset,
                                           const ww_tensor_desc_t* in_desc, const void* const* inputs,
                                           void* const* outputs, void* workspace, void* stream)
{
    ww_attention_int8_t p;
    if (inputs == nullptr || outputs == nullptr || !attention_int8(flags, in_desc, &p)) return 1;
    ww_attention_t& a = p.attention;
    a.q = inputs[0];
    a.k = inputs[1];
    a.v = inputs[2];
    p.k_scale = static_cast<const float*>(inputs[3]);
    p.v_scale = static_cast<const float*>(inputs[4]);
    a.out = outputs[0];
    const int n = attention_inputs(flags);
    for (int i = 3; i < n; ++i) {
        const void* in = inputs[i + 2];
        switch (attention_role(flags, i)) {
            case WW_PLUGIN_ATTENTION_LENS: a.k_lens = static_cast<const int32_t*>(in); break;
            case WW_PLUGIN_ATTENTION_MASK: a.key_mask = static_cast<const uint8_t*>(in); break;
            default:
                a.bias_table = in;
                a.num_buckets = static_cast<int32_t>(in_desc[i + 2].dims[1]);
        }
        if (in == nullptr && numel(in_desc[i + 2]) != 0) return 1;
    }
    a.max_distance = max_distance;
    a.bidirectional = bidirectional;
    a.q_offset = q_offset;
    const int64_t have = attention_copies(a) + WW_PLUGIN_ATTENTION_WORKSPACE;
    a.workspace_bytes = have;
    a.workspace = workspace;
    // parts of few rows that do not fit: without them
    if (workspace != nullptr && static_cast<int64_t>(a.Hq / a.Hk) * a.Lq <= 128 && ww_cross_attention_int8_workspace(&p) > have) a.workspace = nullptr;
    return ww_cross_attention_int8(&p, stream) == WW_SUCCESS ? 0 : 1;
}

}  // extern "C"
