// attention_backward.cu -- ww_cross_attention_backward.
//
// One warp per query row (dq) or key row (dk, dv): 32 scores at a
// time, one per lane, with the running maximum and sum of the softmax; the
// second product runs over the 32 rows with the lanes across the head's dims.
#include "attention.cuh"

namespace ww {
namespace {

constexpr int kWarps = 4;

struct AttnParams {
    ww_attention_t a;
    RelBuckets rel;
    float* delta;   // [B, Hq, Lq] rowsum(dout * out)
    float* table_part;  // [B * Hq * row blocks][num_buckets]
    int row_blocks;
};

template <typename T>
__device__ __forceinline__ const T* row(const void* base, const int64_t* st, int b, int l, int h)
{
    return static_cast<const T*>(base) + b * st[0] + l * st[1] + h * st[2];
}

template <typename T>
__device__ __forceinline__ float dot(const T* x, const float* y, int D)
{
    float s = 0.0f;
    for (int d = 0; d < D; d += 8) {
        const uint4 u = *reinterpret_cast<const uint4*>(x + d);
        const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf(to_float(e[i]), y[d + i], s);
    }
    return s;
}

__device__ __forceinline__ bool valid_key(const ww_attention_t& a, int b, int j, int len)
{
    return j < len && (a.key_mask == nullptr || a.key_mask[static_cast<int64_t>(b) * a.Lk + j] != 0);
}

__device__ __forceinline__ int key_count(const ww_attention_t& a, int b)
{
    return a.k_lens == nullptr ? a.Lk : min(max(a.k_lens[b], 0), a.Lk);
}

template <typename T>
__device__ __forceinline__ float bias_of(const AttnParams& p, int h, int i, int j)
{
    if (p.rel.per_side == 0) return 0.0f;
    return bias_value<T>(static_cast<const T*>(p.a.bias_table)[h * p.rel.total + rel_bucket(p.rel, j - i - p.rel.q_offset)]);
}

template <typename T>
__global__ void __launch_bounds__(32 * kWarps) dq_kernel(const __grid_constant__ AttnParams p)
{
    __shared__ float qs[kWarps][128], gs[kWarps][128];
    __shared__ float db[kWarps][kMaxBuckets];
    const ww_attention_t& a = p.a;
    const int w = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rb = blockIdx.x % p.row_blocks, bh = blockIdx.x / p.row_blocks;
    const int b = bh / a.Hq, h = bh % a.Hq, g = h / (a.Hq / a.Hk);
    const int i = rb * kWarps + w;
    for (int t = threadIdx.x; t < kWarps * kMaxBuckets; t += 32 * kWarps) (&db[0][0])[t] = 0.0f;
    __syncthreads();
    if (i < a.Lq) {
        const int64_t at = ((static_cast<int64_t>(b) * a.Lq + i) * a.Hq + h) * a.D;
        const T* q = row<T>(a.q, a.q_strides, b, i, h);
        const T* go = row<T>(a.dout, a.dout_strides, b, i, h);
        const T* out = static_cast<const T*>(a.out) + at;
        float delta = 0.0f;
        for (int d = lane; d < a.D; d += 32) {
            qs[w][d] = to_float(q[d]);
            gs[w][d] = to_float(go[d]);
            delta += gs[w][d] * to_float(out[d]);
        }
        __syncwarp();
        for (int o = 16; o > 0; o >>= 1) delta += __shfl_xor_sync(~0u, delta, o);
        const int64_t r = (static_cast<int64_t>(b) * a.Hq + h) * a.Lq + i;
        if (lane == 0) p.delta[r] = delta;
        const float lse = a.lse[r];
        float acc[4] = {};
        const int len = lse == -INFINITY ? 0 : key_count(a, b);
        for (int j0 = 0; j0 < len; j0 += 32) {
            const int j = j0 + lane;
            float ds = 0.0f;
            if (valid_key(a, b, j, len)) {
                const float s = dot(row<T>(a.k, a.k_strides, b, j, g), qs[w], a.D) * a.scale + bias_of<T>(p, h, i, j);
                const float dp = dot(row<T>(a.v, a.v_strides, b, j, g), gs[w], a.D);
                ds = exp2_approx((s - lse) * kLog2eF) * (dp - delta);
            }
            for (int n = 0; n < 32; ++n) {
                const float x = __shfl_sync(~0u, ds, n);
                if (x == 0.0f) continue;
                if (p.rel.per_side != 0 && lane == 0) db[w][rel_bucket(p.rel, j0 + n - i - p.rel.q_offset)] += x;
                const T* k = row<T>(a.k, a.k_strides, b, j0 + n, g);
                for (int t = 0; t < 4; ++t)
                    if (lane + 32 * t < a.D) acc[t] += x * to_float(k[lane + 32 * t]);
            }
        }
        T* dq = static_cast<T*>(a.dq) + at;
        for (int t = 0; t < 4; ++t)
            if (lane + 32 * t < a.D) dq[lane + 32 * t] = from_float<T>(acc[t] * a.scale);
    }
    __syncthreads();
    if (p.rel.per_side != 0)
        for (int t = threadIdx.x; t < p.rel.total; t += 32 * kWarps)
            p.table_part[static_cast<int64_t>(blockIdx.x) * p.rel.total + t] =
                (db[0][t] + db[1][t]) + (db[2][t] + db[3][t]);
}

template <typename T>
__global__ void table_kernel(const __grid_constant__ AttnParams p)
{
    const ww_attention_t& a = p.a;
    const int t = threadIdx.x, h = blockIdx.x;
    if (t >= p.rel.total) return;
    float s = 0.0f;
    for (int b = 0; b < a.B; ++b)
        for (int n = 0; n < p.row_blocks; ++n)
            s += p.table_part[((static_cast<int64_t>(b) * a.Hq + h) * p.row_blocks + n) * p.rel.total + t];
    static_cast<T*>(a.dbias_table)[h * p.rel.total + t] = from_float<T>(s);
}

template <typename T>
__global__ void __launch_bounds__(32 * kWarps) dkv_kernel(const __grid_constant__ AttnParams p, int key_blocks)
{
    __shared__ float ks[kWarps][128], vs[kWarps][128];
    const ww_attention_t& a = p.a;
    const int w = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rb = blockIdx.x % key_blocks, bg = blockIdx.x / key_blocks;
    const int b = bg / a.Hk, g = bg % a.Hk;
    const int j = rb * kWarps + w;
    if (j >= a.Lk) return;
    const T* k = row<T>(a.k, a.k_strides, b, j, g);
    const T* v = row<T>(a.v, a.v_strides, b, j, g);
    for (int d = lane; d < a.D; d += 32) {
        ks[w][d] = to_float(k[d]);
        vs[w][d] = to_float(v[d]);
    }
    __syncwarp();
    float dk[4] = {}, dv[4] = {};
    const int G = a.Hq / a.Hk;
    const bool ok = valid_key(a, b, j, key_count(a, b));
    for (int h = g * G; ok && h < (g + 1) * G; ++h) {
        for (int i0 = 0; i0 < a.Lq; i0 += 32) {
            const int i = i0 + lane;
            float pr = 0.0f, ds = 0.0f;
            if (i < a.Lq) {
                const int64_t r = (static_cast<int64_t>(b) * a.Hq + h) * a.Lq + i;
                const float s = dot(row<T>(a.q, a.q_strides, b, i, h), ks[w], a.D) * a.scale + bias_of<T>(p, h, i, j);
                const float dp = dot(row<T>(a.dout, a.dout_strides, b, i, h), vs[w], a.D);
                if (a.lse[r] != -INFINITY) {
                    pr = exp2_approx((s - a.lse[r]) * kLog2eF);
                    ds = pr * (dp - p.delta[r]);
                }
            }
            for (int n = 0; n < 32 && i0 + n < a.Lq; ++n) {
                const float x = __shfl_sync(~0u, pr, n), y = __shfl_sync(~0u, ds, n);
                const T* go = row<T>(a.dout, a.dout_strides, b, i0 + n, h);
                const T* q = row<T>(a.q, a.q_strides, b, i0 + n, h);
                for (int t = 0; t < 4; ++t)
                    if (lane + 32 * t < a.D) {
                        dv[t] += x * to_float(go[lane + 32 * t]);
                        dk[t] += y * to_float(q[lane + 32 * t]);
                    }
            }
        }
    }
    const int64_t at = ((static_cast<int64_t>(b) * a.Lk + j) * a.Hk + g) * a.D;
    for (int t = 0; t < 4; ++t)
        if (lane + 32 * t < a.D) {
            static_cast<T*>(a.dk)[at + lane + 32 * t] = from_float<T>(dk[t] * a.scale);
            static_cast<T*>(a.dv)[at + lane + 32 * t] = from_float<T>(dv[t]);
        }
}

int64_t backward_workspace(const ww_attention_t& p)
{
    const int64_t rows = i64(p.B) * p.Hq * p.Lq;
    const int64_t blocks = i64(p.B) * p.Hq * ((p.Lq + kWarps - 1) / kWarps);
    return rows * 4 + (p.bias_table != nullptr ? blocks * p.num_buckets * 4 : 0);
}

void fill(const ww_attention_t& p, AttnParams* out)
{
    out->a = p;
    if (p.bias_table != nullptr) make_buckets(p.num_buckets, p.max_distance, p.bidirectional, p.q_offset, &out->rel);
    out->row_blocks = (p.Lq + kWarps - 1) / kWarps;
    out->delta = static_cast<float*>(p.workspace);
    out->table_part = out->delta + i64(p.B) * p.Hq * p.Lq;
}

template <typename T>
int backward(const ww_attention_t& p, cudaStream_t s)
{
    AttnParams r;
    fill(p, &r);
    const int kb = (p.Lk + kWarps - 1) / kWarps;
    if (r.row_blocks * p.B > 0) dq_kernel<T><<<r.row_blocks * p.B * p.Hq, 32 * kWarps, 0, s>>>(r);
    if (kb * p.B > 0) dkv_kernel<T><<<kb * p.B * p.Hk, 32 * kWarps, 0, s>>>(r, kb);
    if (p.bias_table != nullptr) table_kernel<T><<<p.Hq, kMaxBuckets, 0, s>>>(r);
    return launch_status("cross_attention_backward");
}

}  // namespace
}  // namespace ww

extern "C" {

int64_t ww_cross_attention_backward_workspace(const ww_attention_t* p)
{
    if (p == nullptr || ww::check_attention(*p) != WW_SUCCESS) return 0;
    return ww::backward_workspace(*p);
}

int ww_cross_attention_backward(const ww_attention_t* p, void* stream)
{
    if (p == nullptr) return WW_ERR_NULL_POINTER;
    int st = ww::check_attention(*p);
    if (st == WW_SUCCESS) st = ww::check_attention_backward(*p, ww::backward_workspace(*p));
    if (st != WW_SUCCESS) return st;
    ww::DeviceInfo d;
    if ((st = ww::current_device_info(&d)) != WW_SUCCESS) return st;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return p->dtype == WW_DTYPE_HALF ? ww::backward<__half>(*p, s) : ww::backward<__nv_bfloat16>(*p, s);
}

}  // extern "C"
